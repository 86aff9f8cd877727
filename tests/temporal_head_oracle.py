"""64-bit definitions of the temporal head's operators, with running error bounds, for the tests.

A kernel works with fp32 sums of `n` terms (each rounding is off by at most u = 2^-24 of the running value, so a sum is off by n u
times the sum of magnitudes) and rounds its outputs once to the type (half a step: torch.finfo(t).eps / 2)."""
import numpy as np
import torch

U32 = 2.0 ** -24
M32 = 0xFFFFFFFF


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def philox_words(blocks, offset, seed):
    """[n] uint64 counter blocks -> [n, 4] words of Philox4x32-10, counter (block, offset), key seed"""
    sh, lo = np.uint64(32), np.uint64(M32)
    c = [blocks & lo, blocks >> sh, np.full_like(blocks, offset & M32), np.full_like(blocks, offset >> 32 & M32)]
    k0, k1 = seed & M32, seed >> 32 & M32
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> sh) ^ c[1] ^ np.uint64(k0), b & lo, (a >> sh) ^ c[3] ^ np.uint64(k1), a & lo]
        k0, k1 = (k0 + 0x9E3779B9) & M32, (k1 + 0xBB67AE85) & M32
    return np.stack(c, axis=1)


def keep_mask(first, n, p, seed, offset):
    """which of the elements first .. first + n - 1 are kept"""
    b0, b1 = first // 4, -(-(first + n) // 4)
    w = philox_words(np.arange(b0, b1, dtype=np.uint64), offset % 2 ** 64, seed % 2 ** 64).reshape(-1)
    return torch.from_numpy(w[first - 4 * b0:first - 4 * b0 + n] >= np.uint64(min(round(p * 2 ** 32), 2 ** 32)))


def linear_ce(x, w, labels, ignore, tau, mean, gl=1.0):
    """-> dict of 64-bit results and elementwise error bounds (e_*) for features of x's type"""
    dt = x.dtype
    x, w = x.double().cpu(), w.double().cpu()
    labels = labels.cpu()
    N, D = x.shape
    V = w.shape[0]
    z = x @ w.t() / tau
    lse = torch.logsumexp(z, 1)
    on = labels != ignore
    col = labels.clamp(0, V - 1)[:, None]
    nll = torch.where(on, lse - z.gather(1, col)[:, 0], torch.zeros_like(lse))
    count = max(1, int(on.sum()))
    s = gl / tau / (count if mean else 1)
    p = torch.exp(z - lse[:, None])
    hot = torch.zeros_like(z).scatter_(1, col, 1.0)
    G = (p - hot) * on[:, None]
    mag = (p + hot) * on[:, None]
    # a logit: products of fp32 features are off by 2^-21 (two pieces of 11 bits each side), the fp32 sum of D terms by D u; a few
    # roundings of the scale, the exponent's argument and the maximum on top
    prod = 2.0 ** -21 if dt == torch.float32 else 0.0
    big = float((x.abs() @ w.abs().t()).max()) / tau
    e_z = big * (prod + (D + 8) * U32)
    e_lse = e_z + 512 * U32 + 4 * U32 * float(lse.abs().max())    # the sum of exponentials: <= 512 serial roundings (tiles joined in 16 runs)
    e_nll = (e_z + e_lse + 4 * U32 * big) * torch.ones(N, dtype=torch.double)
    # G: relative error of exp (argument error) and one rounding to the operand type; fp16 pieces also have an absolute floor
    e_p = 2 * (e_z + e_lse)
    u_g = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -21}[dt]
    floor = 0.0 if dt == torch.bfloat16 else 2.0 ** -25 / 16384
    u_out = half_step(dt)
    gx, gw = s * (G @ w), s * (G.t() @ x)
    live = on[:, None].double()
    e_gx = abs(s) * ((u_g + prod + e_p + (V + 64) * U32) * (mag @ w.abs()) + floor * live * w.abs().sum(0)) + u_out * gx.abs()
    e_gw = abs(s) * ((u_g + prod + e_p + (N + 64) * U32) * (mag.t() @ x.abs()) + floor * (live * x.abs()).sum(0)) + u_out * gw.abs()
    tiny = 2.0 ** -24 if dt == torch.float16 else 0.0              # fp16 outputs below the normal range: one subnormal step
    loss = nll.sum() / (count if mean else 1)
    return {"loss": loss, "nll": nll, "gx": gx, "gw": gw, "e_nll": e_nll, "e_gx": 1.01 * e_gx + tiny, "e_gw": 1.01 * e_gw + tiny,
            "e_loss": (e_nll * on).sum() / (count if mean else 1) + 2 * U32 * loss.abs()}


def gated(gate, x, h0, lengths, gh=None, gh_last=None):
    """-> dict of 64-bit results and elementwise bounds.  Every step is off by at most c u of the magnitudes it adds (the gate's
    exponential by (2 + 1.5 |g|) u relative, its reciprocal and products by a few u, a chunk's pair repeats the products), and an
    error is carried on by the later gates."""
    dt = x.dtype
    g, x = gate.double().cpu(), x.double().cpu()
    B, T, Cc = g.shape
    f, u = torch.sigmoid(g), torch.sigmoid(-g)
    L = lengths.cpu().clamp(0, T) if lengths is not None else torch.full((B,), T)
    live = (torch.arange(T)[None] < L[:, None])[:, :, None]
    f, u = torch.where(live, f, torch.ones_like(f)), torch.where(live, u, torch.zeros_like(u))
    xs = torch.where(live, x, torch.zeros_like(x))                # (what is behind the end may be anything)
    gmax = float(torch.where(live, g, torch.zeros_like(g)).abs().max()) if T else 0.0
    cu = (24 + 4 * gmax) * U32
    h = h0.double().cpu().clone() if h0 is not None else torch.zeros(B, Cc, dtype=torch.double)
    e = torch.zeros_like(h)
    hs, es, prev, eprev = [], [], [], []
    for t in range(T):
        prev.append(h)
        eprev.append(e)
        e = f[:, t] * e + cu * live[:, t] * (f[:, t] * h.abs() + u[:, t] * xs[:, t].abs())
        h = f[:, t] * h + u[:, t] * xs[:, t]
        hs.append(h)
        es.append(e)
    out = {"h": torch.stack(hs, 1) * live if T else g, "last": h, "e_last": e + 2 * U32 * h.abs()}
    half = half_step(dt)
    out["e_h"] = torch.stack(es, 1) * live + half * out["h"].abs() if T else g
    if gh is None:
        return out
    d0 = torch.where(live, gh.double().cpu(), torch.zeros_like(x))
    c = gh_last.double().cpu().clone() if gh_last is not None else torch.zeros_like(h)
    e = torch.zeros_like(c)
    gg, gx, egg, egx = [torch.zeros_like(x) for _ in range(4)]
    for t in reversed(range(T)):
        d, ed = d0[:, t] + c, e + cu * live[:, t] * (d0[:, t].abs() + c.abs())
        diff = (prev[t] - xs[:, t]) * live[:, t]
        gx[:, t] = d * u[:, t]
        egx[:, t] = ed * u[:, t] + cu * gx[:, t].abs()
        fu = f[:, t] * u[:, t]
        gg[:, t] = d * diff * fu
        egg[:, t] = fu * (ed * diff.abs() + d.abs() * (eprev[t] + U32 * (prev[t].abs() + xs[:, t].abs()))) + cu * gg[:, t].abs()
        c, e = f[:, t] * d, f[:, t] * ed + cu * live[:, t] * (f[:, t] * d).abs()
    tiny = 2.0 ** -24 if dt == torch.float16 else 0.0
    out.update(gg=gg, gx=gx, gh0=c, e_gg=egg + half * gg.abs() + tiny, e_gx=egx + half * gx.abs() + tiny, e_gh0=e + 2 * U32 * c.abs())
    out["e_h"] = out["e_h"] + tiny
    return out


def within(got, want, bound, what):
    """|got - want| <= bound everywhere (a tiny absolute allowance for fp32 underflow)"""
    got = got.detach().double().cpu()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    over = (got - want).abs() - (bound + 1e-37)
    assert float(over.max() if over.numel() else -1) <= 0, \
        f"{what}: off by {float((got - want).abs().max()):.3e}, worst excess {float(over.max()):.3e}, bound there {float((bound + 0 * got).flatten()[over.argmax()]):.3e}"
