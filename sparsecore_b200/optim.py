"""AdamW that updates only the live slots of SparseLinear weights.

The reference trains SparseLinear with a stock torch optimizer over the
aliased padded ``values`` tensor (``sparselab/nn.py:183-184``): every slot,
padding included, is read and written each step.  ``LiveAdamW`` keeps
torch's AdamW semantics (decoupled weight decay, per-slot state that stays
with the slot across topology rewrites) but runs one fused kernel per sparse
weight (``sl_adamw_live``) that skips padding slots -- their value stays
exactly 0 and their moments are never touched -- and a stock
``torch.optim.AdamW`` for every other parameter.

Values agree with ``torch.optim.AdamW`` to float rounding (rel 1e-6), not
bit for bit: torch's foreach kernels round some steps differently.  The step
counter lives on the host, so the optimizer is not CUDA-graph capturable;
use ``FusedAdamW(capturable=True)`` (or torch's) inside a captured step.

``FusedAdamW`` takes the whole list of tensors, sparse weights and dense
ones, in one launch (``sl_adamw_multi``), with the moments in 32 or in 8
bits; ``AdamWPlan`` is the same step over a caller's own lists.
"""
from __future__ import annotations

import functools
from operator import attrgetter

import numpy as np
import torch

from . import _native as N

__all__ = ["LiveAdamW", "FusedAdamW", "AdamWPlan", "adamw_step"]


class LiveAdamW(torch.optim.Optimizer):
    def __init__(self, model: torch.nn.Module, lr: float = 1e-3, betas=(0.9, 0.999),
                 eps: float = 1e-8, weight_decay: float = 1e-2):
        from .nn import SparseLinear

        if lr < 0.0 or eps < 0.0 or not (0.0 <= betas[0] < 1.0) or not (0.0 <= betas[1] < 1.0):
            raise ValueError(f"LiveAdamW: invalid hyper-parameters lr={lr}, betas={betas}, eps={eps}")
        self.sparse = [m for m in model.modules() if isinstance(m, SparseLinear)]
        sparse_ids = {id(m._values) for m in self.sparse}
        dense = [p for p in model.parameters() if p.requires_grad and id(p) not in sparse_ids]
        defaults = dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay)
        super().__init__([m._values for m in self.sparse] or [torch.zeros(0)], defaults)
        self.dense_opt = (torch.optim.AdamW(dense, lr=lr, betas=betas, eps=eps,
                                            weight_decay=weight_decay) if dense else None)

    @torch.no_grad()
    def step(self, closure=None):
        loss = closure() if closure is not None else None
        group = self.param_groups[0]
        b1, b2 = group["betas"]
        for m in self.sparse:
            p = m._values
            if p.grad is None:
                continue
            st = self.state[p]
            if not st:
                st["step"] = 0
                st["exp_avg"] = torch.zeros_like(p)
                st["exp_avg_sq"] = torch.zeros_like(p)
            st["step"] += 1
            csr = m._csr
            N.call("sl_adamw_live", csr._abi_ref(), N.ptr(p.grad), N.ptr(st["exp_avg"]),
                   N.ptr(st["exp_avg_sq"]), float(group["lr"]), float(b1), float(b2),
                   float(group["eps"]), float(group["weight_decay"]), int(st["step"]),
                   csr._stream())
        if self.dense_opt is not None:
            for g in self.dense_opt.param_groups:
                g["lr"] = group["lr"]
            self.dense_opt.step()
        return loss

    def zero_grad(self, set_to_none: bool = True):
        super().zero_grad(set_to_none=set_to_none)
        if self.dense_opt is not None:
            self.dense_opt.zero_grad(set_to_none=set_to_none)


#: Elements that share a scale where the moments are held in 8 bits.
BLOCK = 256

_ITEM = np.dtype([(n, np.uint64) for n in ("p", "g", "m", "v", "scale_m", "scale_v", "live")]
                 + [("n", np.int64), ("number", np.int64)])
_get_ptr, _get_numel, _get_device = torch.Tensor.data_ptr, torch.Tensor.numel, torch.Tensor.get_device
_is_contiguous, _get_dtype = torch.Tensor.is_contiguous, attrgetter("dtype")


def _check_hyper(fn, lr, betas, eps, weight_decay):
    if (lr < 0.0 or eps < 0.0 or weight_decay < 0.0 or not (0.0 <= betas[0] < 1.0) or not (0.0 <= betas[1] < 1.0)):
        raise ValueError(f"{fn}: invalid hyper-parameters lr={lr}, betas={betas}, eps={eps}, "
                         f"weight_decay={weight_decay}")


class AdamWPlan:
    """One AdamW step over many tensors in one launch per element type.

    ``params``: contiguous CUDA tensors of one device, each float32, bfloat16
    or float16.  ``exp_avgs`` / ``exp_avg_sqs``: their moments, all float32, or
    all float8_e4m3fn with ``scales``: a pair of float32 tensors per parameter,
    one value per 256 elements.  In 8 bits an element is its e4m3 value times
    its block's scale, and ``exp_avg_sqs`` hold the second moments' square
    roots, the byte 0xFF for an infinite one (see ``sl_adamw_multi``).  ``live``: per parameter None, or the int32
    column indices of a padded CSR whose slots below 0 are left alone, value
    and moments.  ``numbers``: the parameters' numbers that the 8-bit moments'
    dither depends on, where the list is part of a longer one (default: 0, 1, ...).

    The plan keeps the tensors and the table of their addresses; a tensor
    whose storage was replaced since is looked up again at the next step.
    """

    def __init__(self, params, exp_avgs, exp_avg_sqs, *, live=None, scales=None, numbers=None):
        self.params, self.exp_avgs, self.exp_avg_sqs = list(params), list(exp_avgs), list(exp_avg_sqs)
        n = len(self.params)
        self.live = [None] * n if live is None else list(live)
        self.scales = None if scales is None else [tuple(s) for s in scales]
        self.numbers = list(range(n) if numbers is None else numbers)
        for name, v in (("exp_avgs", self.exp_avgs), ("exp_avg_sqs", self.exp_avg_sqs), ("live", self.live),
                        ("scales", self.scales), ("numbers", self.numbers)):
            if v is not None and len(v) != n:
                raise ValueError(f"AdamWPlan: {name} has {len(v)} entries for {n} params")
        self._flat = self.params + self.exp_avgs + self.exp_avg_sqs + [t for t in self.live if t is not None]
        if self.scales is not None:
            self._flat += [t for s in self.scales for t in s]
        self._ptrs = None
        if n:
            self._build()

    def _build(self):
        for t in self._flat:
            if not isinstance(t, torch.Tensor):
                raise TypeError(f"AdamWPlan: expected torch.Tensor, got {type(t).__name__}")
        dev = self.params[0].device
        if dev.type != "cuda":
            raise RuntimeError(f"AdamWPlan: tensors must be on a CUDA device (got device={dev}). "
                               f"sparsecore_b200 has no CPU path.")
        for t in self._flat:
            if t.device != dev:
                raise RuntimeError(f"AdamWPlan: tensors are on {t.device} and {dev}; one plan serves one device")
            if not t.is_contiguous():
                raise ValueError("AdamWPlan: tensors must be contiguous")
        state = torch.float32 if self.scales is None else torch.float8_e4m3fn
        for i, (p, m, v, c) in enumerate(zip(self.params, self.exp_avgs, self.exp_avg_sqs, self.live)):
            n = p.numel()
            if p.dtype not in N.DTYPES:
                raise ValueError(f"AdamWPlan: params must be float32, bfloat16 or float16, got {p.dtype}")
            if m.dtype != state or v.dtype != state:
                raise ValueError(f"AdamWPlan: moments must be {state} {'without' if self.scales is None else 'with'} "
                                 f"scales, got {m.dtype} and {v.dtype}")
            if m.numel() != n or v.numel() != n:
                raise ValueError(f"AdamWPlan: moments of param {i} have {m.numel()} and {v.numel()} elements, not {n}")
            if c is not None and (c.dtype != torch.int32 or c.numel() != n):
                raise ValueError(f"AdamWPlan: live[{i}] must be int32 with {n} elements")
            if self.scales is not None:
                for s in self.scales[i]:
                    if s.dtype != torch.float32 or s.numel() != -(-n // BLOCK):
                        raise ValueError(f"AdamWPlan: scales[{i}] must be two float32 tensors of {-(-n // BLOCK)} elements")
        _no_overlap(self.params + self.exp_avgs + self.exp_avg_sqs
                    + ([t for s in self.scales for t in s] if self.scales is not None else []))
        self.device = dev
        ptr = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
        table = np.zeros(len(self.params), _ITEM)
        for i, p in enumerate(self.params):
            sm, sv = (None, None) if self.scales is None else self.scales[i]
            table[i] = (p.data_ptr(), 0, ptr(self.exp_avgs[i]), ptr(self.exp_avg_sqs[i]), ptr(sm), ptr(sv),
                        ptr(self.live[i]), p.numel(), self.numbers[i])
        self._sizes = list(map(_get_numel, self.params))
        self._dtypes = list(map(_get_dtype, self.params))
        kinds = sorted(set(self._dtypes), key=lambda d: N.DTYPES[d])
        # (type, its rows of the list, its part of the table)
        self._groups = [(N.DTYPES[d], np.array([i for i, e in enumerate(self._dtypes) if e == d]), None) for d in kinds]
        self._groups = [(d, rows, np.ascontiguousarray(table[rows])) for d, rows, _ in self._groups]
        self._ptrs = list(map(_get_ptr, self._flat))
        # While the table has an address its memory is kept: no other tensor's can be taken for it.
        self._kept = [t.untyped_storage() for t in self._flat]

    def step(self, grads, *, step: int | None = None, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8,
             weight_decay: float = 1e-2, seed: int = 0, hyper: torch.Tensor | None = None) -> None:
        """Updates params and moments in place from ``grads`` (a tensor of the
        parameter's type and size each, or None to leave a parameter alone).
        ``step`` counts from 1; ``seed`` shifts the 8-bit moments' dither.
        ``hyper``: these numbers made on the device (``sl_adamw_hyper``), for captured
        steps."""
        grads = list(grads)
        if len(grads) != len(self.params):
            raise ValueError(f"AdamWPlan: {len(grads)} grads for {len(self.params)} params")
        if hyper is None:
            _check_hyper("AdamWPlan", lr, betas, eps, weight_decay)
            if step is None or step < 1:
                raise ValueError(f"AdamWPlan: step must be at least 1, got {step}")
        if not grads:
            return
        if hyper is not None:
            _check_numbers(hyper, self.device)
        self._launch(*self._take(grads), lr, betas, eps, weight_decay, step, seed, hyper)

    def _take(self, grads):
        """(which parameters take the step, None for all; their gradients as the kernel reads them), checked."""
        if list(map(_get_ptr, self._flat)) != self._ptrs:
            self._build()
        given = grads
        if any(g is None for g in grads):
            on = [i for i, g in enumerate(grads) if g is not None]
            given = [grads[i] for i in on]
            sizes, dtypes = [self._sizes[i] for i in on], [self._dtypes[i] for i in on]
        else:
            on, sizes, dtypes = None, self._sizes, self._dtypes
        if list(map(_get_numel, given)) != sizes or list(map(_get_dtype, given)) != dtypes:
            self._build()  # maybe a parameter was cut or given another type where it lies
            every = range(len(grads)) if on is None else on
            given = self._fit(given, [self._sizes[i] for i in every], [self._dtypes[i] for i in every])
        elif not set(map(_get_device, given)) <= {self.device.index} or not all(map(_is_contiguous, given)):
            given = self._fit(given, sizes, dtypes)
        return on, given

    def _launch(self, on, given, lr, betas, eps, weight_decay, step, seed, hyper):
        ptrs = np.zeros(len(self.params), np.uint64)
        ptrs[slice(None) if on is None else on] = list(map(_get_ptr, given))
        bits = 32 if self.scales is None else 8
        with_step = (float(lr), float(betas[0]), float(betas[1]), float(eps), float(weight_decay),
                     0 if step is None else int(step), int(seed) & 0xFFFFFFFF, N.ptr(hyper))
        for dtype, rows, table in self._groups:
            table["g"] = ptrs[rows]
            t = table if on is None else np.ascontiguousarray(table[table["g"] != 0])
            if len(t):
                N.call_on(self.device, "sl_adamw_multi", t.ctypes.data, len(t), dtype, bits, *with_step)

    def _fit(self, grads, sizes, dtypes):
        """Gradients as the kernel reads them, or the reason why they cannot be."""
        for g, n, d in zip(grads, sizes, dtypes):
            if not isinstance(g, torch.Tensor):
                raise TypeError(f"AdamWPlan: grads must be torch.Tensor or None, got {type(g).__name__}")
            if g.is_sparse or g.layout != torch.strided:
                raise ValueError("AdamWPlan: grads must be dense")
            if g.device != self.device:
                raise RuntimeError(f"AdamWPlan: a grad is on {g.device} but its param on {self.device}")
            if g.numel() != n or g.dtype != d:
                raise ValueError(f"AdamWPlan: a grad has {g.numel()} elements of {g.dtype}; its param {n} of {d}")
        return [g.contiguous() for g in grads]


@functools.lru_cache(maxsize=None)
def _hyper_bytes():
    return int(N.lib().sl_adamw_hyper_bytes())


def _check_numbers(hyper, device):
    """Refuses what the kernel on `device` cannot read a step's numbers from."""
    if not isinstance(hyper, torch.Tensor):
        raise TypeError(f"AdamWPlan: hyper must be a torch.Tensor, got {type(hyper).__name__}")
    if (hyper.device != device or not hyper.is_contiguous() or hyper.numel() * hyper.element_size() < _hyper_bytes()
            or hyper.data_ptr() % 16):
        raise ValueError(f"AdamWPlan: hyper must be {_hyper_bytes()} contiguous bytes on {device}, 16-byte aligned")


def _check_counter(step, device):
    """Refuses a step count that the kernel on `device` must not write to."""
    if not isinstance(step, torch.Tensor) or step.device != device or step.dtype != torch.int64 or step.numel() != 1:
        raise ValueError(f"FusedAdamW: a step count on the device must be one int64 element on {device}, got {step!r}")


def _no_overlap(tensors):
    """Refuses tensors that are written and share memory (the same one twice, or views that overlap)."""
    spans = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for t in tensors if t.numel())
    for (_, end), (begin, _) in zip(spans, spans[1:]):
        if begin < end:
            raise ValueError("AdamWPlan: two of the tensors that the step writes share memory")


def adamw_step(params, grads, exp_avgs, exp_avg_sqs, *, step: int, lr: float = 1e-3, betas=(0.9, 0.999),
               eps: float = 1e-8, weight_decay: float = 1e-2, live=None, scales=None, seed: int = 0) -> None:
    """One AdamW step over lists of tensors, in place (``AdamWPlan`` for one step;
    a program that takes many steps keeps the plan)."""
    AdamWPlan(params, exp_avgs, exp_avg_sqs, live=live, scales=scales).step(
        grads, step=step, lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, seed=seed)


class FusedAdamW(torch.optim.Optimizer):
    """AdamW over a model's parameters, SparseLinear weights (padding slots left
    alone) and dense ones, in one launch per element type and group.

    ``model_or_params``: a module (its SparseLinears are found), parameters, or
    parameter groups; ``live`` maps further padded value arrays to their int32
    column indices.  ``state_bits``: 32, or 8 for e4m3 moments with a scale per
    256 elements (a quarter of the memory; ``state_values`` gives them back).
    ``capturable``: the step count is kept on the device, and a learning rate
    given as a float32 CUDA tensor is read there, so that a captured step
    replays correctly.  Before a capture, take one step with gradients on the
    same parameters: moments and counts that would begin inside it are refused,
    and so is a capture without ``capturable``.

    Each parameter's moments are corrected by the steps that it has taken itself,
    as in torch's AdamW: one that begins late, misses steps or is drawn again is
    stepped by its own count (in a launch of its own for each different count).
    Parameters are contiguous, and those of a group on one device.
    """

    def __init__(self, model_or_params, lr=1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2, *,
                 state_bits: int = 32, capturable: bool = False, seed: int = 0, live=None):
        from .nn import SparseLinear

        if not isinstance(lr, torch.Tensor):
            _check_hyper("FusedAdamW", lr, betas, eps, weight_decay)
        elif not capturable:
            raise ValueError("FusedAdamW: a tensor lr needs capturable=True")
        if state_bits not in (8, 32):
            raise ValueError(f"FusedAdamW: state_bits must be 8 or 32, got {state_bits}")
        self._sparse = []
        params = model_or_params
        if isinstance(params, torch.nn.Module):
            self._sparse = [m for m in params.modules() if isinstance(m, SparseLinear)]
            params = [p for p in params.parameters() if p.requires_grad]
        self._live = dict(live or {})
        self.state_bits, self.capturable, self.seed = state_bits, capturable, int(seed)
        self._plans: dict = {}
        self._hypers: dict = {}
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay))

    # torch's optimizers keep only their defaults, states and groups; a copy makes its own tables.  (SparseLinears hold
    # addresses and refuse to be copied, and so does an optimizer over them.)
    def __getstate__(self):
        return super().__getstate__() | {k: self.__dict__[k] for k in ("_sparse", "_live", "state_bits", "capturable", "seed")}

    def __setstate__(self, state):
        super().__setstate__(state)
        for k in ("_plans", "_hypers"):
            self.__dict__.setdefault(k, {})

    def _columns(self):
        cols = {m._values: m._csr.col_indices for m in self._sparse}
        cols.update(self._live)
        return cols

    def _init_state(self, p):
        st = self.state[p]
        if self.state_bits == 32:
            st["exp_avg"], st["exp_avg_sq"] = (torch.zeros_like(p, dtype=torch.float32, memory_format=torch.contiguous_format)
                                               for _ in range(2))
        else:
            for k in ("exp_avg", "exp_avg_sq_root"):
                st[k] = torch.zeros(p.numel(), dtype=torch.uint8, device=p.device).view(torch.float8_e4m3fn)
                st[k + "_scale"] = torch.zeros(-(-p.numel() // BLOCK), dtype=torch.float32, device=p.device)

    def _plan(self, k, group, params, cols):
        """The plan of a group's parameters of one count; made again where a tensor of it is another one."""
        live = [cols.get(p) for p in params]
        st = [self.state[p] for p in params]
        if self.state_bits == 32:
            ms, vs, scales = [s["exp_avg"] for s in st], [s["exp_avg_sq"] for s in st], None
        else:
            ms, vs = [s["exp_avg"] for s in st], [s["exp_avg_sq_root"] for s in st]
            scales = [(s["exp_avg_scale"], s["exp_avg_sq_root_scale"]) for s in st]
        kept = self._plans.get(k)
        if (kept is None or len(kept.params) != len(params)
                or any(a is not b for a, b in zip(kept.params + kept.exp_avgs + kept.exp_avg_sqs + kept.live,
                                                  params + ms + vs + live))):
            number = {p: i for i, p in enumerate(group["params"])}
            kept = self._plans[k] = AdamWPlan(params, ms, vs, live=live, scales=scales, numbers=[number[p] for p in params])
        return kept

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        cols = self._columns()
        used, stepped = set(), set()
        for k, group in enumerate(self.param_groups):
            params = [p for p in group["params"] if p.grad is not None]
            if not params:
                continue
            if not self.capturable and params[0].is_cuda and torch.cuda.is_current_stream_capturing():
                raise RuntimeError("FusedAdamW: a captured step needs capturable=True (its replays would repeat one step's numbers)")
            stepped.add(k)
            for j, (count, members, holders) in enumerate(self._counted(group, params)):
                used.add((k, j))
                plan = self._plan((k, j), group, members, cols)
                grads = [p.grad for p in members]
                if self.capturable:
                    taken = plan._take(grads)  # what is refused is refused before it is counted
                    plan._launch(*taken, 0.0, group["betas"], 0.0, 0.0, None, self.seed, self._advance((k, j), count, group, plan.device))
                    continue
                plan.step(grads, step=count + 1, lr=group["lr"], betas=group["betas"], eps=group["eps"],
                          weight_decay=group["weight_decay"], seed=self.seed)
                for h in holders:
                    h["step"] = count + 1
        if len(self._plans) > len(used):  # of counts that are no more
            self._plans = {key: plan for key, plan in self._plans.items() if key in used or key[0] not in stepped}
        return loss

    def _counted(self, group, params):
        """[(step count, the parameters of ``params`` that have it, the dictionaries that hold it)].  AdamW corrects
        a parameter's moments by its own steps: the group's "step" counts those of the parameters that have
        taken every one, and a parameter that began later, missed one or was drawn again has a "step" in
        its state.  On the device (capturable) parameters of one history share one tensor."""
        state = self.state
        at = group.get("step", 0)
        begun = isinstance(at, torch.Tensor) or at > 0
        if self.capturable and not isinstance(at, torch.Tensor):
            self._not_captured(params[0])
            at = group["step"] = torch.full((), at, dtype=torch.int64, device=params[0].device)
        late, zero = False, None
        for p in params:
            st = state[p]
            if not st or st["exp_avg"].numel() != p.numel():  # new, or a layer drawn again at another capacity
                self._not_captured(p)
                self._init_state(p)
                st.pop("step", None)
                if begun:
                    zero = (torch.zeros_like(at) if self.capturable else 0) if zero is None else zero
                    st["step"] = zero
            late = late or "step" in st
        if len(params) < len(group["params"]):
            self._set_apart(group, params, at)
            late = late or any("step" in state[p] for p in params)
        if not late:
            return [(at, params, [group])]
        by: dict = {}
        for p in params:
            count = state[p].get("step")
            key = None if count is None else id(count) if isinstance(count, torch.Tensor) else count
            by.setdefault(key, (at if count is None else count, []))[1].append(p)
        return [(count, ps, [group] if key is None else [state[p] for p in ps]) for key, (count, ps) in by.items()]

    def _set_apart(self, group, params, at):
        """Gives parameters that miss this step a count of their own where the one they share goes on without them."""
        state, copies = self.state, {}
        shared = {id(state[p].get("step", group)) for p in params}
        for p in group["params"]:
            st = state.get(p)
            if p.grad is not None or not st:
                continue
            count = st.get("step")
            if id(group if count is None else count) not in shared or isinstance(count, int):
                continue
            count = at if count is None else count
            if isinstance(count, torch.Tensor):
                self._not_captured(p)
                if id(count) not in copies:
                    copies[id(count)] = count.clone()
                count = copies[id(count)]
            st["step"] = count

    @staticmethod
    def _not_captured(p):
        if p.is_cuda and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("FusedAdamW: moments or step counts would begin inside a graph capture, and every replay would begin "
                               "them again; take one step with gradients on the same parameters before the capture")

    def _advance(self, key, count, group, dev):
        """Adds one to a step count on the device and makes the step's numbers there."""
        _check_counter(count, dev)
        hyper = self._hypers.get(key)
        if hyper is None or hyper.device != dev:
            hyper = self._hypers[key] = torch.empty(_hyper_bytes(), dtype=torch.uint8, device=dev)
        lr = group["lr"]
        on_device = isinstance(lr, torch.Tensor)
        if on_device and (lr.device != dev or lr.dtype != torch.float32 or lr.numel() != 1):
            raise ValueError(f"FusedAdamW: a tensor lr must be one float32 element on {dev}")
        N.call_on(dev, "sl_adamw_hyper", N.ptr(count), N.ptr(lr if on_device else None),
                  0.0 if on_device else float(lr), float(group["betas"][0]), float(group["betas"][1]),
                  float(group["eps"]), float(group["weight_decay"]), self.seed & 0xFFFFFFFF, N.ptr(hyper))
        return hyper

    def load_state_dict(self, state_dict):
        """As torch's, but the moments keep their own types (torch casts a state to its parameter's type)."""
        needed = "exp_avg_sq" if self.state_bits == 32 else "exp_avg_sq_root"
        if any(needed not in st for st in state_dict["state"].values()):
            raise ValueError(f"FusedAdamW: the state is not one of {self.state_bits}-bit moments")
        super().load_state_dict(state_dict)
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        for i, p in zip(ids, [p for g in self.param_groups for p in g["params"]]):
            for name, v in state_dict["state"].get(i, {}).items():
                keep = name == "step" or not isinstance(v, torch.Tensor)
                self.state[p][name] = v if keep else v.detach().to(p.device, copy=True)
        for group in self.param_groups:
            self._place_numbers(group)

    def _place_numbers(self, group):
        """A loaded group's step counts and learning rate came as they were saved, on the host maybe: they go where its
        parameters are, or become plain numbers where nothing is captured.  A state of ``torch.optim.AdamW`` has
        every count in its parameter's state."""
        if not group["params"]:
            return
        dev = group["params"][0].device
        put = lambda n: torch.full((), n, dtype=torch.int64, device=dev) if self.capturable else n  # noqa: E731
        held = [self.state[p] for p in group["params"] if self.state.get(p)]
        own = [int(st["step"]) if "step" in st else None for st in held]
        if "step" in group or any(n is not None for n in own):
            at = int(group["step"]) if "step" in group else max(n for n in own if n is not None)
            group["step"], counts = put(at), {}
            for st, n in zip(held, own):
                if n is None or n == at:
                    st.pop("step", None)
                else:
                    st["step"] = counts[n] = counts[n] if n in counts else put(n)
        if isinstance(group["lr"], torch.Tensor):
            group["lr"] = group["lr"].to(dev) if self.capturable else float(group["lr"])

    def state_values(self, p) -> tuple[torch.Tensor, torch.Tensor]:
        """The first and second moment of ``p`` in 32 bits, in its shape."""
        st = self.state[p]
        if self.state_bits == 32:
            return st["exp_avg"].clone(), st["exp_avg_sq"].clone()
        spread = lambda s: s.repeat_interleave(BLOCK)[:p.numel()]  # noqa: E731
        m = st["exp_avg"].float() * spread(st["exp_avg_scale"])
        root = st["exp_avg_sq_root"]
        r = root.float() * spread(st["exp_avg_sq_root_scale"])
        r.masked_fill_(root.view(torch.uint8) == 0xFF, float("inf"))
        return m.view(p.shape), r.square().view(p.shape)
