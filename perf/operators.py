"""The operators of a temporal classification head -- softmax cross entropy over a large set of prototypes straight from
the features, dropout without a stored mask, a gated linear recurrence over time -- as cases that can be measured.

`own = False` computes each operator in its plain form (elementary torch operations in 32 bits); `own = True` calls the
framework.  Outputs of both are laid out alike.
"""
import math

import numpy as np
import torch

own = False

_DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}
_IGNORE = -100


# ------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # evaluation of a few sampled cells against a small prototype set: latency of one call
        {"name": "ce_loss_bf16_few", "op": "linear_ce", "dtype": "bf16", "rows": 37, "classes": 1003, "dim": 128, "train": False},
        # nearest-prototype scoring of a handful of descriptors against a large codebook: bound by reading the codebook
        {"name": "ce_loss_f32_codebook", "op": "linear_ce", "dtype": "f32", "rows": 16, "classes": 65536, "dim": 512, "train": False},
        # one frame's stride-4 map (128 x 153 cells) of the 128-channel distillation head against 4096 prototypes, fp32 training
        {"name": "ce_train_f32_frame", "op": "linear_ce", "dtype": "f32", "rows": 19584, "classes": 4096, "dim": 128, "train": True},
        # odd sizes everywhere, fp16
        {"name": "ce_train_f16_odd", "op": "linear_ce", "dtype": "f16", "rows": 1531, "classes": 10007, "dim": 200, "train": True},
        # sampled cells of a batch, the encoder's 256 channels, 65536 prototypes
        {"name": "ce_train_bf16_prototypes", "op": "linear_ce", "dtype": "bf16", "rows": 8192, "classes": 65536, "dim": 256, "train": True},
        # wide token features against the largest prototype set
        {"name": "ce_train_bf16_wide", "op": "linear_ce", "dtype": "bf16", "rows": 4096, "classes": 131072, "dim": 1024, "train": True},
        # dropout on the 256-channel stride-4 map of a batch of 8 frames, forward and backward
        {"name": "dropout_f32_map", "op": "dropout", "dtype": "f32", "numel": 8 * 128 * 153 * 256, "p": 0.1, "residual": False},
        # dropout into a residual sum, 16-bit features of 8 x 4096 tokens
        {"name": "dropout_bf16_residual", "op": "dropout", "dtype": "bf16", "numel": 8 * 4096 * 1024, "p": 0.2, "residual": True},
        # a small odd activation: latency
        {"name": "dropout_f16_small", "op": "dropout", "dtype": "f16", "numel": 1003 * 257, "p": 0.5, "residual": False},
        # serving: one new frame's features for 64 streams
        {"name": "gated_step_bf16", "op": "gated", "dtype": "bf16", "batch": 64, "steps": 1, "channels": 512, "ragged": False, "train": False},
        # ragged batch of odd-sized sequences
        {"name": "gated_train_f32_ragged", "op": "gated", "dtype": "f32", "batch": 3, "steps": 4099, "channels": 97, "ragged": True, "train": True},
        # a few long token sequences, wide features
        {"name": "gated_train_bf16_long", "op": "gated", "dtype": "bf16", "batch": 4, "steps": 16384, "channels": 1024, "ragged": False, "train": True},
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["linear_ce", "linear_ce", "dropout", "gated"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op == "linear_ce":
        while True:
            n, v, d = _log_uniform(rng, 1, 20000), _log_uniform(rng, 2, 131072), _log_uniform(rng, 8, 1024)
            if n * v <= 8192 * 65536 and n * v * d <= 4096 * 131072 * (1024 if dtype != "f32" else 256):
                break
        return {"op": op, "dtype": dtype, "rows": n, "classes": v, "dim": d, "train": rng.random() < 0.7}
    if op == "dropout":
        return {"op": op, "dtype": dtype, "numel": _log_uniform(rng, 1, 8 * 128 * 153 * 256), "p": round(rng.uniform(0.02, 0.8), 3),
                "residual": rng.random() < 0.5}
    while True:
        b, t, c = _log_uniform(rng, 1, 20000), _log_uniform(rng, 1, 16384), _log_uniform(rng, 1, 1024)
        if b * t * c <= 4 * 16384 * 1024:
            break
    return {"op": op, "dtype": dtype, "batch": b, "steps": t, "channels": c, "ragged": rng.random() < 0.5, "train": rng.random() < 0.7}


def work(case):
    s = _SIZE[case["dtype"]]
    if case["op"] == "linear_ce":
        n, v, d = case["rows"], case["classes"], case["dim"]
        once = (n + v) * d * s
        if case["train"]:
            return {"bytes": 2 * once + 12 * n + 4, "flops": 6 * n * v * d}
        return {"bytes": once + 12 * n + 4, "flops": 2 * n * v * d}
    if case["op"] == "dropout":
        return {"bytes": case["numel"] * s * (5 if case["residual"] else 4), "flops": case["numel"] * (3 if case["residual"] else 2)}
    n, bc = case["batch"] * case["steps"] * case["channels"], case["batch"] * case["channels"]
    if case["train"]:                          # gate, x, dh in; h, dgate, dx out; the states and their gradients
        return {"bytes": 6 * n * s + 4 * bc * 4, "flops": 14 * n}
    return {"bytes": 3 * n * s + 2 * bc * 4, "flops": 6 * n}


# ------------------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed * 7919 + 17)
    dt = _DT[case["dtype"]]

    def rand(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    st = {"case": dict(case)}
    if case["op"] == "linear_ce":
        n, v, d = case["rows"], case["classes"], case["dim"]
        w = rand(v, d)
        w = w / w.norm(dim=1, keepdim=True)
        labels = torch.randint(0, v, (n,), generator=g, device=dev)
        x = w[labels] + rand(n, d) * (1.5 / math.sqrt(d))      # descriptors scatter about their prototype
        x = x / x.norm(dim=1, keepdim=True)
        skip = torch.rand(n, generator=g, device=dev) < 0.1    # unlabelled cells
        labels = torch.where(skip, torch.full_like(labels, _IGNORE), labels)
        st.update(x=x.to(dt), w=w.to(dt), labels=labels, temperature=0.1)
        if case["train"]:
            st["x"].requires_grad_(True)
            st["w"].requires_grad_(True)
    elif case["op"] == "dropout":
        n = case["numel"]
        st.update(x=rand(n).to(dt).requires_grad_(True), gy=rand(n).to(dt), seed=(1000003 * seed + 12345) % 2 ** 63, offset=(seed % 999983 << 33) + 5,
                  res=rand(n).to(dt).requires_grad_(True) if case["residual"] else None)
    else:
        b, t, c = case["batch"], case["steps"], case["channels"]
        st.update(gate=(rand(b, t, c) * 1.5 + 2.0).to(dt), x=rand(b, t, c).to(dt), h0=rand(b, c), lengths=None)
        if case["ragged"]:
            st["lengths"] = torch.randint(0, t + 1, (b,), generator=g, device=dev)
        if case["train"]:
            for k in ("gate", "x", "h0"):
                st[k].requires_grad_(True)
            st.update(gh=rand(b, t, c).to(dt), gh_last=rand(b, c))
    return st


# -------------------------------------------------------------------------------------------------------------- run
def run(state):
    op = state["case"]["op"]
    if own:
        return {"linear_ce": _own_linear_ce, "dropout": _own_dropout, "gated": _own_gated}[op](state)
    with torch.no_grad():
        return {"linear_ce": _plain_linear_ce, "dropout": _plain_dropout, "gated": _plain_gated}[op](state)


def _own_linear_ce(st):
    from creste_public_amd import loss_ops
    loss, nll = loss_ops.linear_cross_entropy(st["x"], st["w"], st["labels"], ignore_index=_IGNORE, temperature=st["temperature"])
    if not st["case"]["train"]:
        return loss, nll
    gx, gw = torch.autograd.grad(loss, (st["x"], st["w"]))
    return loss.detach(), nll, gx, gw


def _own_dropout(st):
    from creste_public_amd import train_ops
    y = train_ops.dropout(st["x"], st["case"]["p"], st["seed"], st["offset"], residual=st["res"])
    leaves = (st["x"],) if st["res"] is None else (st["x"], st["res"])
    return (y.detach(),) + torch.autograd.grad(y, leaves, st["gy"])


def _own_gated(st):
    from creste_public_amd import train_ops
    h, last = train_ops.gated_recurrence(st["gate"], st["x"], st["h0"], st["lengths"])
    if not st["case"]["train"]:
        return h, last
    return (h.detach(), last.detach()) + torch.autograd.grad((h, last), (st["gate"], st["x"], st["h0"]), (st["gh"], st["gh_last"]))


# ------------------------------------------------------------------------------------------------------ plain forms
def _plain_linear_ce(st):
    x, w, labels, tau = st["x"].float(), st["w"].float(), st["labels"], st["temperature"]
    z = (x @ w.t()) / tau
    m = z.max(dim=1, keepdim=True).values
    lse = m + torch.exp(z - m).sum(dim=1, keepdim=True).log()
    valid = labels != _IGNORE
    idx = torch.where(valid, labels, torch.zeros_like(labels))[:, None]
    nll = torch.where(valid, (lse - z.gather(1, idx))[:, 0], torch.zeros_like(lse[:, 0]))
    count = valid.sum().clamp(min=1)
    loss = nll.sum() / count
    if not st["case"]["train"]:
        return loss, nll
    z -= lse
    z.exp_()
    z.scatter_add_(1, idx, torch.full_like(lse, -1.0))
    z *= valid[:, None] / (count * tau)
    return loss, nll, (z @ w).to(st["x"].dtype), (z.t() @ x).to(st["w"].dtype)


_M32 = 0xFFFFFFFF


def _plain_words(n, seed, offset, device):
    """n words of Philox4x32-10 (Salmon et al., SC 2011): counter (i div 4, offset), key seed, 64 bits each."""
    i = torch.arange((n + 3) // 4, device=device)
    c0, c1 = i & _M32, i >> 32
    c2, c3 = torch.full_like(i, offset & _M32), torch.full_like(i, (offset >> 32) & _M32)
    k0, k1 = seed & _M32, (seed >> 32) & _M32
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57          # products modulo 2^64
        c0, c1, c2, c3 = ((p1 >> 32) & _M32) ^ c1 ^ k0, p1 & _M32, ((p0 >> 32) & _M32) ^ c3 ^ k1, p0 & _M32
        k0, k1 = (k0 + 0x9E3779B9) & _M32, (k1 + 0xBB67AE85) & _M32
    return torch.stack((c0, c1, c2, c3), dim=1).reshape(-1)[:n]


def _plain_dropout(st):
    p, dt = st["case"]["p"], st["x"].dtype
    keep = _plain_words(st["x"].numel(), st["seed"], st["offset"], st["x"].device) >= round(p * 2 ** 32)
    scale = 1.0 / (1.0 - p)
    zero = torch.zeros((), device=st["x"].device)
    y = torch.where(keep, st["x"].float() * scale, zero)
    gx = torch.where(keep, st["gy"].float() * scale, zero).to(dt)
    if st["res"] is None:
        return y.to(dt), gx
    return (y + st["res"].float()).to(dt), gx, st["gy"]


def _scan(a, b):
    """all b_t <- a_t b_{t-1} + b_t along dim 1 by doubling."""
    t, d = a.shape[1], 1
    while d < t:
        nb, na = b.clone(), a.clone()
        nb[:, d:] += a[:, d:] * b[:, :-d]
        na[:, d:] *= a[:, :-d]
        a, b, d = na, nb, 2 * d
    return b


def _plain_gated(st):
    g, x, h0, dt = st["gate"].float(), st["x"].float(), st["h0"], st["x"].dtype
    steps = g.shape[1]
    live = torch.ones(g.shape[:2], dtype=torch.bool, device=g.device)
    if st["lengths"] is not None:
        live = torch.arange(steps, device=g.device)[None] < st["lengths"][:, None]
    live = live[:, :, None]
    f = torch.where(live, 1.0 / (1.0 + torch.exp(-g)), torch.ones((), device=g.device))
    u = torch.where(live, 1.0 / (1.0 + torch.exp(g)), torch.zeros((), device=g.device))
    b = u * x
    b[:, 0] += f[:, 0] * h0
    h = _scan(f, b)
    last = h[:, -1].clone()
    out = torch.where(live, h, torch.zeros((), device=g.device)).to(dt)
    if not st["case"]["train"]:
        return out, last
    d = torch.where(live, st["gh"].float(), torch.zeros((), device=g.device))
    d[:, -1] += st["gh_last"]
    nxt = torch.cat((f[:, 1:], torch.ones_like(f[:, :1])), dim=1)
    d = _scan(nxt.flip(1), d.flip(1)).flip(1)
    prev = torch.cat((h0[:, None], h[:, :-1]), dim=1)
    return out, last, (d * (prev - x) * f * u).to(dt), (d * u).to(dt), f[:, 0] * d[:, 0]


# ------------------------------------------------------------------------------------------------ definitions, 64 bit
def exact(case, seed):
    with torch.no_grad():
        st = prepare(case, seed)
        return {"linear_ce": _exact_linear_ce, "dropout": _exact_dropout, "gated": _exact_gated}[case["op"]](st)


def _exact_linear_ce(st):
    x, w, y, tau = st["x"].detach().double(), st["w"].detach().double(), st["labels"], st["temperature"]
    n = x.shape[0]
    used = (y != _IGNORE).double()
    count = max(1.0, float(used.sum()))
    nll, gx, gw = torch.zeros(n, dtype=torch.double, device=x.device), torch.zeros_like(x), torch.zeros_like(w)
    step = max(1, (1 << 27) // w.shape[0])                 # rows whose 64-bit logits fit 1 GiB
    for i in range(0, n, step):
        z = torch.mm(x[i:i + step], w.t().contiguous()).div_(tau)
        lse = torch.logsumexp(z, dim=1)
        for_row = torch.arange(z.shape[0], device=x.device)
        col = y[i:i + step].clamp(min=0)
        nll[i:i + step] = (lse - z[for_row, col]) * used[i:i + step]
        if st["case"]["train"]:
            p = z.sub_(lse[:, None]).exp_()
            p[for_row, col] -= 1.0
            p.mul_((used[i:i + step] / (count * tau))[:, None])
            gx[i:i + step] = torch.mm(p, w)
            gw.add_(torch.mm(p.t().contiguous(), x[i:i + step]))
    loss = nll.sum() / count
    return (loss, nll, gx, gw) if st["case"]["train"] else (loss, nll)


def _exact_dropout(st):
    n, p = st["case"]["numel"], st["case"]["p"]
    blocks = -(-n // 4)
    ctr = np.zeros((4, blocks), dtype=np.uint64)
    ctr[0] = np.arange(blocks, dtype=np.uint64) & np.uint64(_M32)
    ctr[1] = np.arange(blocks, dtype=np.uint64) >> np.uint64(32)
    ctr[2], ctr[3] = st["offset"] % 2 ** 32, st["offset"] // 2 ** 32
    key = [st["seed"] % 2 ** 32, st["seed"] // 2 ** 32]
    lo, sh = np.uint64(_M32), np.uint64(32)
    for r in range(10):
        a, b = ctr[0] * np.uint64(0xD2511F53), ctr[2] * np.uint64(0xCD9E8D57)
        k = [np.uint64((key[0] + r * 0x9E3779B9) % 2 ** 32), np.uint64((key[1] + r * 0xBB67AE85) % 2 ** 32)]
        ctr = np.stack([(b >> sh) ^ ctr[1] ^ k[0], b & lo, (a >> sh) ^ ctr[3] ^ k[1], a & lo])
    words = ctr.T.reshape(-1)[:n]
    factor = torch.from_numpy((words >= np.uint64(round(p * 2 ** 32))).astype(np.float64) / (1.0 - p)).to(st["x"].device)
    y, gx = st["x"].detach().double() * factor, st["gy"].double() * factor
    if st["res"] is None:
        return y, gx
    return y + st["res"].detach().double(), gx, st["gy"].double()


def _exact_gated(st):
    g, x, h = st["gate"].detach().double(), st["x"].detach().double(), st["h0"].detach().double()
    steps = g.shape[1]
    lengths = st["lengths"] if st["lengths"] is not None else torch.full((g.shape[0],), steps, device=g.device)
    f, u = torch.sigmoid(g), torch.sigmoid(-g)
    out, before = torch.zeros_like(x), torch.empty_like(x)
    for t in range(steps):
        on = (t < lengths)[:, None]
        before[:, t] = h
        h = torch.where(on, torch.addcmul(u[:, t] * x[:, t], f[:, t], h), h)
        out[:, t] = h * on
    if not st["case"]["train"]:
        return out, h
    delta = st["gh_last"].double()
    gg, gx, gh = torch.zeros_like(x), torch.zeros_like(x), st["gh"].double()
    for t in reversed(range(steps)):
        on = (t < lengths)[:, None]
        d = (delta + gh[:, t]) * on
        gx[:, t] = d * u[:, t]
        gg[:, t] = d * (before[:, t] - x[:, t]) * f[:, t] * u[:, t]
        delta = torch.where(on, d * f[:, t], delta)
    return out, h, gg, gx, delta
