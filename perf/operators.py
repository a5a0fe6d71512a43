"""The cases that the training-step operators are measured on, and the operators in plain torch.

Three operators of a language model's training step stand around the sparse layers:

  xent   linear_cross_entropy: the softmax cross entropy of x . W^T against target tokens, taken over
         pieces of the vocabulary without keeping the logits, with the gradients of x and W
  norm   residual_norm: the norm after a block (optional), its gate and residual scale, the residual
         add and the norm before the next block in one pass, forward and backward
  adamw  AdamWPlan: one AdamW step over a list of tensors (dense ones and the padded value arrays of
         sparse weights, whose padding slots are left alone), with moments in 32 or in 8 bits

``own`` false: the plain form, elementary torch operations in 32 bits (rounded once at the end);
true: the calls that a program makes of this package.
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
IGNORE = -100
BLOCK = 256  # elements that share a scale where the moments are held in 8 bits


# ── cases ────────────────────────────────────────────────────────────────

def listed():
    return [
        # loss of the character transformer's batch: 64 x 256 tokens, 65 characters
        {"name": "xent-char", "op": "xent", "T": 16384, "D": 384, "V": 65, "dtype": "f32", "train": True, "reduction": "mean"},
        # loss of the byte-level transformer's batch: 32 x 512 tokens, 256 bytes
        {"name": "xent-byte", "op": "xent", "T": 16384, "D": 768, "V": 256, "dtype": "f32", "train": True, "reduction": "mean"},
        # the same width with a word-piece vocabulary of odd size, in the framework's own 32 bits
        {"name": "xent-words-f32", "op": "xent", "T": 4096, "D": 768, "V": 50001, "dtype": "f32", "train": True, "reduction": "mean"},
        # a wide model's large vocabulary in 16 bits
        {"name": "xent-large-bf16", "op": "xent", "T": 8192, "D": 2048, "V": 128000, "dtype": "bf16", "train": True, "reduction": "mean"},
        # scoring one short text: the losses of 33 tokens, no gradient
        {"name": "xent-score-f16", "op": "xent", "T": 33, "D": 1024, "V": 32003, "dtype": "f16", "train": False, "reduction": "none"},
        # one token on its way through a serving step
        {"name": "norm-token", "op": "norm", "T": 1, "D": 768, "dtype": "f32", "kind": "layer", "post": False, "gate": "none", "scale": 1.0, "train": False},
        # the byte-level transformer's batch between two of its blocks, forward and backward
        {"name": "norm-byte", "op": "norm", "T": 16384, "D": 768, "dtype": "f32", "kind": "layer", "post": False, "gate": "none", "scale": 1.0, "train": True},
        # a wide model with norms on both sides of the block, a gate per channel and a residual scale
        {"name": "norm-sandwich-bf16", "op": "norm", "T": 8191, "D": 4096, "dtype": "bf16", "kind": "rms", "post": True, "gate": "channel", "scale": 0.5, "train": True},
        # the two-layer perceptron: two padded value arrays and two biases, where the launch counts
        {"name": "adamw-mlp", "op": "adamw", "model": "mlp", "width": 512, "layers": 1, "dtype": "f32", "bits": 32},
        # all tensors of the byte-level transformer, sparse projections as padded value arrays
        {"name": "adamw-byte", "op": "adamw", "model": "sparse", "width": 768, "layers": 8, "dtype": "f32", "bits": 32},
        # a dense transformer of about 300 M weights in 16 bits with its moments in 8
        {"name": "adamw-dense-8bit", "op": "adamw", "model": "dense", "width": 1024, "layers": 24, "dtype": "bf16", "bits": 8},
        # the sparse transformer with its moments in 8 bits
        {"name": "adamw-byte-8bit", "op": "adamw", "model": "sparse", "width": 768, "layers": 8, "dtype": "f32", "bits": 8},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("xent", "norm", "adamw"))
    dtype = rng.choice(("f32", "bf16", "f16"))
    if op == "xent":
        T, D, V = _log(rng, 1, 16384), _log(rng, 32, 2048), _log(rng, 2, 128000)
        if rng.random() < 0.7:
            D = max(32, D // 64 * 64)
        T = max(1, min(T, 8192 * 2048 * 128000 // (D * V), (1 << 30) // V))
        train = rng.random() < 0.75
        return {"op": op, "T": T, "D": D, "V": V, "dtype": dtype, "train": train,
                "reduction": rng.choice(("mean", "sum")) if train else rng.choice(("mean", "none"))}
    if op == "norm":
        T, D = _log(rng, 1, 16384), _log(rng, 32, 8192)
        if rng.random() < 0.7:
            D = max(32, D // 32 * 32)
        T = max(1, min(T, 8191 * 4096 // D))
        return {"op": op, "T": T, "D": D, "dtype": dtype, "kind": rng.choice(("layer", "rms")), "post": rng.random() < 0.5,
                "gate": rng.choice(("none", "channel", "token")), "scale": rng.choice((1.0, 0.5, 0.7071)), "train": rng.random() < 0.75}
    return {"op": op, "model": rng.choice(("mlp", "sparse", "dense")), "width": _log(rng, 64, 1024), "layers": rng.randint(1, 16),
            "dtype": dtype, "bits": rng.choice((8, 32))}


# ── inputs ───────────────────────────────────────────────────────────────

def _sizes(c):
    """[(number of values, whether it is a padded value array)] of a model's weights."""
    w, n = c["width"], c["layers"]
    slots = lambda rows, cols, density: rows * max(1, math.ceil(cols * density * 1.2))  # noqa: E731  20 % padding a row
    if c["model"] == "mlp":
        return [(slots(w, 784, 0.1), True), (w, False), (slots(10, w, 0.1), True), (10, False)] * n
    if c["model"] == "sparse":  # attention projections 70 % sparse, feed-forward 90 %
        block = [(w, False)] * 4 + [(slots(3 * w, w, 0.3), True), (slots(w, w, 0.3), True), (slots(4 * w, w, 0.1), True), (slots(w, 4 * w, 0.1), True)]
        return block * n + [(256 * w, False), (512 * w, False), (w, False), (w, False), (256 * w, False)]
    block = [(w, False)] * 2 + [(3 * w * w, False), (w * w, False), (4 * w * w, False), (4 * w * w, False)]
    return block * n + [(32003 * w, False), (w, False)]


def _layout(c):
    """(offset, length, sparse) of each tensor in one flat buffer, each on a block's border, and the buffer's length."""
    at, got = 0, []
    for n, sparse in _sizes(c):
        got.append((at, n, sparse))
        at += -(-n // BLOCK) * BLOCK
    return got, at


def prepare(case, seed):
    c, dev = case, torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed) * 1000003 + 17)
    dt = _TYPES[c["dtype"]]
    randn = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    if c["op"] == "xent":
        T, D, V = c["T"], c["D"], c["V"]
        x, w = randn(T, D).to(dt), (randn(V, D) * (2.0 / math.sqrt(D))).to(dt)  # logits of deviation 2
        t = torch.randint(0, V, (T,), generator=g, device=dev)
        t[torch.rand(T, generator=g, device=dev) < 0.05] = IGNORE  # padding of the batch
        t[0] = V // 2
        return {"case": c, "x": x.requires_grad_(c["train"]), "w": w.requires_grad_(c["train"]), "t": t}
    if c["op"] == "norm":
        T, D, tr = c["T"], c["D"], c["train"]
        s = {"case": c, "y": randn(T, D).to(dt), "r": (2 * randn(T, D) + 0.3).to(dt), "w": (1 + 0.1 * randn(D)).to(dt),
             "b": (0.1 * randn(D)).to(dt) if c["kind"] == "layer" else None, "gate": None, "pw": None, "pb": None}
        if c["gate"] != "none":
            s["gate"] = (randn(D) if c["gate"] == "channel" else randn(T, D)).to(dt)
        if c["post"]:
            s["pw"] = (1 + 0.1 * randn(D)).to(dt)
            s["pb"] = (0.1 * randn(D)).to(dt) if c["kind"] == "layer" else None
        if tr:
            for k in ("y", "r", "w", "b", "gate", "pw", "pb"):
                if s[k] is not None:
                    s[k].requires_grad_(True)
            s["dr"], s["dh"] = randn(T, D).to(dt), randn(T, D).to(dt)
        return s
    layout, n = _layout(c)
    cut = lambda flat: [flat[o:o + k] for o, k, _ in layout]  # noqa: E731
    p = (0.02 * randn(n)).to(dt)
    gr = (1e-3 * randn(n)).to(dt)
    cols = (torch.arange(n, device=dev) % 6).sub_(1).to(torch.int32)  # one slot in six is padding: -1
    m, v = 3e-4 * randn(n), (1e-3 * randn(n)).square()
    pad = torch.zeros(n, dtype=torch.bool, device=dev)
    for o, k, sparse in layout:
        if sparse:
            pad[o:o + k] = cols[o:o + k] < 0
    pad |= ~_covered(layout, n, dev)
    p[pad], gr[pad], m[pad], v[pad] = 0, 0, 0, 0
    s = {"case": c, "p": p, "g": cut(gr), "params": cut(p), "live": [cols[o:o + k] if sparse else None for o, k, sparse in layout],
         "step": 10, "seed": int(seed) & 0x7FFFFFFF, "m": m, "v": v, "scales": None}
    if c["bits"] == 8:  # element = 8-bit value x its block's scale; the second moment as its square root
        mb, ub = m.view(-1, BLOCK), v.sqrt().view(-1, BLOCK)
        sm, su = mb.abs().amax(1).clamp_min(2.0 ** -100) / 448, ub.amax(1).clamp_min(2.0 ** -100) / 448
        s["m"] = (mb / sm[:, None]).clamp(-448, 448).to(torch.float8_e4m3fn).view(-1)
        s["v"] = (ub / su[:, None]).clamp(0, 448).to(torch.float8_e4m3fn).view(-1)
        s["sm"], s["su"] = sm, su
        s["scales"] = [(sm[o // BLOCK:o // BLOCK - (-k // BLOCK)], su[o // BLOCK:o // BLOCK - (-k // BLOCK)]) for o, k, _ in layout]
    s["ms"], s["vs"] = cut(s["m"]), cut(s["v"])
    return s


def _covered(layout, n, dev):
    edge = torch.zeros(n + 1, dtype=torch.int32, device=dev)
    edge[torch.tensor([o for o, _, _ in layout], device=dev)] += 1
    edge[torch.tensor([o + k for o, k, _ in layout], device=dev)] -= 1
    return edge.cumsum(0)[:n] > 0


LR, BETAS, EPS, DECAY = 3e-4, (0.9, 0.999), 1e-8, 0.01


# ── one pass ─────────────────────────────────────────────────────────────

def run(s):
    return {"xent": _xent, "norm": _norm, "adamw": _adamw}[s["case"]["op"]](s)


def _xent(s):
    c = s["case"]
    if own:
        import sparsecore_b200 as sl

        loss = sl.linear_cross_entropy(s["x"], s["w"], s["t"], ignore_index=IGNORE, reduction=c["reduction"])
        if not c["train"]:
            return {"loss": loss}
        dx, dw = torch.autograd.grad(loss, (s["x"], s["w"]))
        return {"loss": loss.detach(), "dx": dx, "dw": dw}
    x, w, t = s["x"].detach().float(), s["w"].detach().float(), s["t"]
    live = t != IGNORE
    at = torch.where(live, t, torch.zeros_like(t))[:, None]
    z = x @ w.t()
    z = z - z.amax(1, keepdim=True)
    target = z.gather(1, at)[:, 0]
    e = z.exp_()
    total = e.sum(1, keepdim=True)
    each = torch.where(live, total[:, 0].log() - target, torch.zeros_like(target))
    count = live.sum()
    loss = each if c["reduction"] == "none" else each.double().sum().float() if c["reduction"] == "sum" else (each.double().sum() / count).float()
    if not c["train"]:
        return {"loss": loss}
    d = e.div_(total)
    d.scatter_add_(1, at, torch.full_like(target, -1.0)[:, None])
    d.mul_((live / count if c["reduction"] == "mean" else live).to(torch.float32)[:, None])
    return {"loss": loss, "dx": (d @ w).to(s["x"].dtype), "dw": (d.t() @ x).to(s["w"].dtype)}


def _plain_norm(v, w, b, kind):
    """The norm of each row, its normalised values and the rows' 1 / deviation."""
    v = v - v.mean(1, keepdim=True) if kind == "layer" else v
    rstd = (v.square().mean(1, keepdim=True) + 1e-5).rsqrt()
    n = v * rstd
    return n * w if b is None else n * w + b, n, rstd


def _plain_norm_back(d, n, rstd, w, kind):
    """Gradient of the norm's input from that of its output."""
    dn = d * w
    back = dn - n * (dn * n).mean(1, keepdim=True)
    if kind == "layer":
        back = back - dn.mean(1, keepdim=True)
    return back * rstd


def _norm(s):
    c = s["case"]
    if own:
        import sparsecore_b200 as sl

        out, h = sl.residual_norm(s["y"], s["r"], s["w"], s["b"], kind=c["kind"], eps=1e-5, gate=s["gate"], scale=c["scale"],
                                  post_weight=s["pw"], post_bias=s["pb"])
        if not c["train"]:
            return {"out": out, "h": h}
        names = [k for k in ("y", "r", "w", "b", "gate", "pw", "pb") if s[k] is not None]
        grads = torch.autograd.grad((out, h), [s[k] for k in names], (s["dr"], s["dh"]))
        return {"out": out.detach(), "h": h.detach(), **{"d" + k: v for k, v in zip(names, grads)}}
    kind, dt = c["kind"], s["y"].dtype
    f = lambda t: None if t is None else t.detach().float()  # noqa: E731
    y, r, w, b, gate, pw, pb = (f(s[k]) for k in ("y", "r", "w", "b", "gate", "pw", "pb"))
    u, pn, prstd = (y, None, None) if pw is None else _plain_norm(y, pw, pb, kind)
    gu = u if gate is None else u * gate
    out = (r + c["scale"] * gu).to(dt)  # held in the stream's type: what the norm reads is what the next block's residual is
    h, n, rstd = _plain_norm(out.float(), w, b, kind)
    got = {"out": out, "h": h.to(dt)}
    if not c["train"]:
        return got
    dh, do = f(s["dh"]), f(s["dr"])
    got["dw"] = (dh * n).sum(0).to(dt)
    if b is not None:
        got["db"] = dh.sum(0).to(dt)
    d = do + _plain_norm_back(dh, n, rstd, w, kind)
    got["dr"] = d.to(dt)
    du = c["scale"] * d
    if gate is not None:
        dg = du * u
        got["dgate"] = (dg.sum(0) if gate.dim() == 1 else dg).to(dt)
        du = du * gate
    if pw is not None:
        got["dpw"] = (du * pn).sum(0).to(dt)
        if pb is not None:
            got["dpb"] = du.sum(0).to(dt)
        du = _plain_norm_back(du, pn, prstd, pw, kind)
    got["dy"] = du.to(dt)
    return got


def _mix(v):
    """32 mixed bits of each whole number (held in 64 bits): the dither of the 8-bit moments."""
    v = (v ^ (v >> 16)) * 0x5B2C9E6D & 0xFFFFFFFF
    v = (v ^ (v >> 13)) * 0x3F4A7C15 & 0xFFFFFFFF
    return v ^ (v >> 16)


def _mix_int(v):
    v = (v ^ (v >> 16)) * 0x5B2C9E6D & 0xFFFFFFFF
    v = (v ^ (v >> 13)) * 0x3F4A7C15 & 0xFFFFFFFF
    return v ^ (v >> 16)


def _dither(n, seed, step, which, dev):
    """Two fractions below 1, of 16 bits each, for each element of tensor number `which`."""
    key = _mix_int((seed + 0x9E3779B1 * step + 0x85EBCA77 * which) & 0xFFFFFFFF)
    bits = _mix((torch.arange(n, device=dev) * 0x9E3779B1 + key) & 0xFFFFFFFF)
    return bits & 0xFFFF, bits >> 16


def _to_8bit(v, bits, floor):
    """(8-bit values, scales) of `v`, [blocks, 256], rounded up or down by 16 dither bits; `floor`: what is not zero stays so."""
    top = v.abs().amax(1, keepdim=True).clamp_min(2.0 ** -100)
    x = (v.abs() * (448.0 / top)).clamp_max(448.0)
    small = torch.where(x < 2.0 ** -6, 2.0 ** -6, 0.0)  # 8-bit subnormals: evenly spaced, like the binade above
    raw = (x + small).float().view(torch.int32) + (bits.to(torch.int32) << 4)
    q = (raw & ~0xFFFFF).view(torch.float32) - small.float()
    if floor:
        q = torch.where(v > 0, q.clamp_min(2.0 ** -9), q)
    q = torch.where(v < 0, -q, q)
    return q.to(torch.float8_e4m3fn), (top * (1.0 / 448.0))[:, 0]


def _blocks(t):
    return torch.nn.functional.pad(t, (0, -t.numel() % BLOCK)).view(-1, BLOCK)


def _adamw_one(p, g, m, v, live, scale, step, seed, which):
    gf = g.float()
    if scale is not None:
        mf = (_blocks(m.float()) * scale[0][:, None]).view(-1)[:p.numel()]
        vf = (_blocks(v.float()) * scale[1][:, None]).view(-1)[:p.numel()].square()
    else:
        mf, vf = m, v
    b1, b2 = BETAS
    m1 = mf + (gf - mf) * (1 - b1)
    v1 = vf * b2 + gf * gf * (1 - b2)
    step_size, root = LR / (1 - b1 ** step), math.sqrt(1 - b2 ** step)
    pf = p.float() * (1 - LR * DECAY)
    p1 = pf - step_size * (m1 / (v1.sqrt() / root + EPS))
    if live is not None:
        pad = live < 0
        p1, m1, v1 = torch.where(pad, p.float(), p1), torch.where(pad, mf, m1), torch.where(pad, vf, v1)
    p.copy_(p1)
    if scale is None:
        m.copy_(m1)
        v.copy_(v1)
        return
    rm, ru = _dither(p.numel(), seed, step, which, p.device)
    for_m, for_u = _to_8bit(_blocks(m1), _blocks(rm), False), _to_8bit(_blocks(v1.sqrt()), _blocks(ru), True)
    m.copy_(for_m[0].view(-1)[:p.numel()])
    v.copy_(for_u[0].view(-1)[:p.numel()])
    scale[0].copy_(for_m[1])
    scale[1].copy_(for_u[1])


def _adamw(s):
    if own:
        import sparsecore_b200 as sl

        if "plan" not in s:  # what a program keeps from step to step: its tensors' table
            s["plan"] = sl.AdamWPlan(s["params"], s["ms"], s["vs"], live=s["live"], scales=s["scales"])
        s["plan"].step(s["g"], step=s["step"], lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY, seed=s["seed"])
    else:
        scales = s["scales"] or [None] * len(s["params"])
        [_adamw_one(p, g, m, v, live, sc, s["step"], s["seed"], i) for i, (p, g, m, v, live, sc) in
         enumerate(zip(s["params"], s["g"], s["ms"], s["vs"], s["live"], scales))]
    got = {"p": s["p"], "m": s["m"], "v": s["v"]}
    if s["scales"] is not None:
        got.update(sm=s["sm"], su=s["su"])
    return got


# ── what a pass cannot do without ────────────────────────────────────────

def work(case):
    c = case
    e = 4 if c["dtype"] == "f32" else 2
    if c["op"] == "xent":
        T, D, V = c["T"], c["D"], c["V"]
        once = e * (T * D + V * D)
        if not c["train"]:
            return {"bytes": once + 8 * T + (4 * T if c["reduction"] == "none" else 4), "flops": 2 * T * D * V}
        return {"bytes": 2 * once + 8 * T + 4, "flops": 6 * T * D * V}
    if c["op"] == "norm":
        n, D = c["T"] * c["D"], c["D"]
        gate = {"none": 0, "channel": D, "token": n}[c["gate"]]
        vectors = (1 + (c["kind"] == "layer")) * (2 if c["post"] else 1) * D + gate
        moved, flops = 4 * n + vectors, 10 * n
        if c["train"]:  # the outputs' gradients in, the inputs' gradients out
            moved, flops = moved + 4 * n + vectors, 40 * n
        return {"bytes": e * moved, "flops": flops}
    layout, _ = _layout(c)
    total = 0
    for _, n, sparse in layout:
        live = n - n // 6 if sparse else n
        total += 4 * n * sparse + live * (3 * e + (16 if c["bits"] == 32 else 4)) + (0 if c["bits"] == 32 else 16 * -(-n // BLOCK))
    return {"bytes": total, "flops": 16 * sum(n for _, n, _ in layout)}


# ── the definitions in 64 bits ───────────────────────────────────────────

def exact(case, seed):
    s = prepare(case, seed)
    return {"xent": _exact_xent, "norm": _exact_norm, "adamw": _exact_adamw}[case["op"]](s)


def _exact_xent(s):
    c = s["case"]
    x, w, t = s["x"].detach().double(), s["w"].detach().double(), s["t"]
    T, keep = x.shape[0], t != IGNORE
    count = float(keep.sum())
    loss = torch.zeros(T, dtype=torch.float64, device=x.device)
    dx, dw = torch.zeros_like(x), torch.zeros_like(w)
    rows = max(1, (1 << 28) // w.shape[0])
    for a in range(0, T, rows):
        xa, ka = x[a:a + rows], keep[a:a + rows]
        ta = t[a:a + rows].clamp_min(0)
        z = torch.mm(xa, w.t())
        lse = torch.logsumexp(z, 1)
        i = torch.arange(xa.shape[0], device=x.device)
        loss[a:a + rows] = (lse - z[i, ta]) * ka
        if c["train"]:
            d = torch.exp(z - lse[:, None])
            d[i, ta] -= 1
            d *= ka[:, None] / (count if c["reduction"] == "mean" else 1.0)
            dx[a:a + rows] = torch.mm(d, w)
            dw += torch.mm(d.t(), xa)
    out = loss if c["reduction"] == "none" else loss.sum() / (count if c["reduction"] == "mean" else 1.0)
    return {"loss": out, "dx": dx, "dw": dw} if c["train"] else {"loss": out}


def _exact_norm(s):
    """By differentiating the definition; the residual is held in its own type between its add and its norm."""
    c = s["case"]
    names = [k for k in ("y", "r", "w", "b", "gate", "pw", "pb") if s[k] is not None]
    a = {k: s[k].detach().double().requires_grad_(c["train"]) for k in names}

    def norm(v, w, b):
        mean = v.mean(-1, keepdim=True) if c["kind"] == "layer" else 0.0
        var = ((v - mean) ** 2).mean(-1, keepdim=True)
        n = (v - mean) / torch.sqrt(var + 1e-5) * w
        return n if b is None else n + b

    u = norm(a["y"], a["pw"], a.get("pb")) if c["post"] else a["y"]
    out = a["r"] + c["scale"] * (u * a["gate"] if "gate" in a else u)
    dt = s["y"].dtype
    held = out + (out.detach().float().to(dt).double() - out.detach()) if dt != torch.float32 else out
    h = norm(held, a["w"], a.get("b"))
    got = {"out": out.detach(), "h": h.detach()}
    if c["train"]:
        grads = torch.autograd.grad((out, h), [a[k] for k in names], (s["dr"].double(), s["dh"].double()))
        got.update({"d" + k: v for k, v in zip(names, grads)})
    return got


def _exact_adamw(s):
    c, step = s["case"], s["step"]
    b1, b2 = BETAS
    eight = c["bits"] == 8
    grid = torch.arange(0x7F, dtype=torch.uint8, device=s["p"].device).view(torch.float8_e4m3fn).double()  # 0 ... 448
    got = {"p": s["p"].double(), "m": None if eight else s["m"].double(), "v": None if eight else s["v"].double()}
    if eight:
        got.update(m=s["m"].double(), v=s["v"].double(), sm=s["sm"].double(), su=s["su"].double())

    def held(val, frac, floor):
        """Each value as the 8-bit neighbour below or above: above where its distance from the lower and the dither reach 1."""
        n = val.numel()
        blocks = torch.cat([val, val.new_zeros(-n % BLOCK)]).view(-1, BLOCK)
        top = torch.clamp(blocks.abs().max(1).values, min=2.0 ** -100)
        x = torch.clamp((blocks.abs() / top[:, None] * 448).view(-1)[:n], max=448.0)
        i = torch.searchsorted(grid, x, right=True) - 1
        lo, hi = grid[i], grid[torch.clamp(i + 1, max=grid.numel() - 1)]
        part = torch.where(hi > lo, (x - lo) / torch.clamp(hi - lo, min=2.0 ** -9), torch.zeros_like(x))
        q = torch.where(part + frac >= 1, hi, lo)
        if floor:
            q = torch.where((val > 0) & (q == 0), torch.full_like(q, 2.0 ** -9), q)
        return torch.sign(val) * q, top / 448

    for i, (o, n, sparse) in enumerate(_layout(c)[0]):
        p, g = s["p"][o:o + n].double(), s["g"][i].double()
        m, v = s["m"][o:o + n].double(), s["v"][o:o + n].double()
        if eight:
            at = torch.arange(n, device=p.device) // BLOCK
            m, v = m * s["scales"][i][0].double()[at], (v * s["scales"][i][1].double()[at]) ** 2
        live = s["live"][i] >= 0 if sparse else torch.ones(n, dtype=torch.bool, device=p.device)
        m1 = torch.where(live, b1 * m + (1 - b1) * g, m)
        v1 = torch.where(live, b2 * v + (1 - b2) * g ** 2, v)
        m_hat, v_hat = m1 / (1 - b1 ** step), v1 / (1 - b2 ** step)
        got["p"][o:o + n] = torch.where(live, p - LR * DECAY * p - LR * m_hat / (torch.sqrt(v_hat) + EPS), p)
        if eight:
            rm, ru = _dither(n, s["seed"], step, i, p.device)
            k = slice(o // BLOCK, o // BLOCK - (-n // BLOCK))
            got["m"][o:o + n], got["sm"][k] = held(m1, rm.double() / 65536, False)
            got["v"][o:o + n], got["su"][k] = held(torch.sqrt(v1), ru.double() / 65536, True)
        else:
            got["m"][o:o + n], got["v"][o:o + n] = m1, v1
    return got
