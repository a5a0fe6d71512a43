"""The loss's buffer sizes and refusals through the C ABI, without a GPU."""
import ctypes

import pytest
import torch

from sparsecore_b200 import _native as N


def _sizes(tokens=100, dim=64, vocab=300, dtype=torch.float32, reduction=0, train=1, x=0, w=0):
    lib = N.load_library()
    out = (ctypes.c_int64 * 3)()
    at = ctypes.addressof(out)
    a = N.XENT_ARGS.pack(x, w, 0, 0, 0, 0, 0, 0, 0, 0, tokens, dim, vocab, -100, N.DTYPES.get(dtype, dtype), reduction, train)
    return lib.sl_xent_sizes(a, at, at + 8, at + 16), tuple(out)


def test_shapes_that_the_calls_refuse_have_no_sizes():
    """Before a program allocates by them."""
    assert _sizes()[0] == N.SL_OK
    for bad in (dict(tokens=-1), dict(dim=0), dict(vocab=0), dict(dim=(1 << 20) + 1), dict(tokens=1 << 40), dict(vocab=1 << 40),
                dict(dtype=7), dict(reduction=3), dict(reduction=-1)):
        assert _sizes(**bad)[0] == N.SL_ERR_INVALID, bad


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_sizes_of_the_largest_shapes_do_not_wrap(dtype):
    """Operands of 2^30 rows and 2^20 columns: their sizes pass 32 bits and are still those of their parts."""
    planes = 2 if dtype == torch.float32 else 1
    for tokens, dim, vocab in (((1 << 30) - 1, 1 << 20, 300), (300, 1 << 20, (1 << 30) - 1), ((1 << 30) - 1, 64, (1 << 30) - 1)):
        rc, (kept, forward, backward) = _sizes(tokens, dim, vocab, dtype)
        assert rc == N.SL_OK
        assert kept >= planes * tokens * dim * 2 + 8 * tokens
        assert forward >= -(-vocab // 128) * tokens * 8
        assert backward >= planes * tokens * 256 * 2 + 4 * tokens * dim * (vocab > 256 and tokens > 1 << 20)
