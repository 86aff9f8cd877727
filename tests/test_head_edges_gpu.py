"""GPU: the operators of the temporal classification head where magnitudes, layouts and sizes are uneven, against 64-bit
definitions."""
import pytest
import torch

from creste_public_amd import _lib, loss_ops, ops, train_ops  # noqa: F401
from tests import temporal_head_oracle as O
from tests.temporal_head_oracle import within

pytestmark = pytest.mark.gpu
E = _lib.HipLibraryError
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def gen(seed):
    return torch.Generator().manual_seed(seed)


# --------------------------------------------------------------------------------------- cross entropy, fp32 rows of uneven magnitude
def _rowwise(x, w, labels, tau):
    """64-bit results (reduction: sum) and bounds that hold row by row.  A factor x_ik is off by 2^-22 of its row's largest magnitude X_i,
    w_jk by 2^-22 of W_j, a product of both remainders is left out (2^-22), and the fp32 sum of D terms is off by D 2^-24 of the magnitudes
    it adds: e_ij = (2^-21 + (D + 8) 2^-24) sum |x||w| + 2^-22 (X_i sum |w_j| + W_j sum |x_i|), over tau.  The logits' errors move a
    log-sum-exp to logsumexp(z + e) at most, and a probability to exp(z + e - (lse - e_lse)).  G is off by 2^-21 of its magnitude and
    2^-39, sums over n by n 2^-24."""
    x, w = x.double(), w.double()
    N, D = x.shape
    V = w.shape[0]
    u = O.U32
    z = x @ w.t() / tau
    xm, wm = x.abs().amax(1, keepdim=True), w.abs().amax(1, keepdim=True)
    e = ((2.0 ** -21 + (D + 8) * u) * (x.abs() @ w.abs().t()) + 2.0 ** -22 * (xm * w.abs().sum(1)[None] + wm.t() * x.abs().sum(1, keepdim=True))) / tau
    lse = torch.logsumexp(z, 1)
    on = labels != -100
    col = labels.clamp(min=0)[:, None]
    e_lse = torch.maximum(torch.logsumexp(z + e, 1) - lse, lse - torch.logsumexp(z - e, 1)) + (600 + 4 * lse.abs()) * u
    nll = torch.where(on, lse - z.gather(1, col)[:, 0], torch.zeros_like(lse))
    e_nll = e_lse + e.gather(1, col)[:, 0] + 8 * u * z.abs().gather(1, col)[:, 0]
    p = torch.exp(z - lse[:, None])
    hot = torch.zeros_like(z).scatter_(1, col, 1.0)
    live = on[:, None].double()
    G = (p - hot) * live
    # (a probability is 1 at most; the argument's own roundings: 4 u of its magnitude)
    up = torch.exp((z + e - (lse - e_lse)[:, None] + 4 * u * (z.abs() + lse.abs()[:, None])).clamp(max=0.0))
    dn = torch.exp(z - e - (lse + e_lse)[:, None] - 4 * u * (z.abs() + lse.abs()[:, None]))
    e_G = live * (torch.maximum(up - p, p - dn) + 2.0 ** -21 * (p + hot) + 2.0 ** -39)
    mag = live * (p + hot)
    gx, gw = G @ w / tau, G.t() @ x / tau
    wq, xq = w.abs() + 2.0 ** -22 * wm, x.abs() + 2.0 ** -22 * xm
    e_gx = (e_G @ wq + mag @ (2.0 ** -22 * wm.expand_as(w)) + (V + 64) * u * (mag @ w.abs())) / tau + 2 * u * gx.abs()
    e_gw = (e_G.t() @ xq + mag.t() @ (2.0 ** -22 * xm.expand_as(x)) + (N + 64) * u * (mag.t() @ x.abs())) / tau + 2 * u * gw.abs()
    return {k: v.cpu() for k, v in dict(nll=nll, e_nll=e_nll, gx=gx, e_gx=1.01 * e_gx, gw=gw, e_gw=1.01 * e_gw).items()}


def _unit(n, d, seed):
    t = torch.randn(n, d, generator=gen(seed))
    return t / t.norm(dim=1, keepdim=True)


def _uneven(N, V, D, seed=0):
    """features scattered about their prototypes, some rows not counted"""
    w, labels = _unit(V, D, seed), torch.randint(0, V, (N,), generator=gen(seed + 1))
    x = w[labels] + torch.randn(N, D, generator=gen(seed + 2)) * (1.5 / D ** 0.5)
    x = x / x.norm(dim=1, keepdim=True)
    labels[3::7] = -100
    return x.cuda(), w.cuda(), labels.cuda()


def _uneven_check(x, w, labels, tau=0.1):
    x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    loss, nll = loss_ops.linear_cross_entropy(x, w, labels, temperature=tau, reduction="sum")
    gx, gw = torch.autograd.grad(loss, (x, w))
    r = _rowwise(x.detach().cpu(), w.detach().cpu(), labels.cpu(), tau) if nll.numel() * w.shape[0] < 1 << 24 else \
        _rowwise(x.detach(), w.detach(), labels, tau)
    within(nll, r["nll"], r["e_nll"], "nll")
    within(gx, r["gx"], r["e_gx"], "dx")
    within(gw, r["gw"], r["e_gw"], "dw")


SIZES = [(16, 1000, 128), (64, 1000, 128), (300, 257, 40), (90, 700, 300), (513, 300, 65)]


@pytest.mark.parametrize("N,V,D", SIZES)
@pytest.mark.parametrize("big", [1e4, 1e7, 1e9, 1e12])
def test_linear_ce_f32_one_large_row(N, V, D, big):
    x, w, labels = _uneven(N, V, D)
    x[5] *= big
    _uneven_check(x, w, labels)


@pytest.mark.parametrize("N,V,D", SIZES)
@pytest.mark.parametrize("big", [1e4, 1e7, 1e9, 1e12])
def test_linear_ce_f32_one_large_class(N, V, D, big):
    x, w, labels = _uneven(N, V, D)
    w[V // 2] *= big
    _uneven_check(x, w, labels)


@pytest.mark.parametrize("N,V,D", SIZES)
def test_linear_ce_f32_rows_over_many_magnitudes(N, V, D):
    x, w, labels = _uneven(N, V, D)
    _uneven_check(x * 10.0 ** torch.linspace(-8, 0, N, device="cuda")[:, None], w, labels)
    _uneven_check(x, w * 10.0 ** torch.linspace(0, -8, V, device="cuda")[:, None], labels)
    x[1], w[2] = 0.0, 0.0                                             # rows of zeros beside ordinary ones
    _uneven_check(x, w, labels)


@pytest.mark.parametrize("N,V,D", SIZES)
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_linear_ce_f32_one_row_that_is_not_finite(N, V, D, bad):
    """its own loss is NaN, every other row's is right"""
    x, w, labels = _uneven(N, V, D)
    r = _rowwise(x.cpu(), w.cpu(), labels.cpu(), 0.1)
    x[5, D // 2] = bad
    loss, nll = loss_ops.linear_cross_entropy(x, w, labels, temperature=0.1)
    assert not torch.isfinite(loss) and not torch.isfinite(nll[5])
    keep = torch.arange(N) != 5
    within(nll.cpu()[keep], r["nll"][keep], r["e_nll"][keep], "nll")


@pytest.mark.parametrize("N,V,D", [(16, 33, 24), (70, 33, 24), (70, 65, 128), (70, 5, 300), (70, 300, 257)])
@pytest.mark.parametrize("sx,sw", [(1e-20, 1e-20), (1e-30, 1e-15), (1e18, 1e-38), (1e-38, 1e18)])
def test_linear_ce_f32_both_operands_tiny(N, V, D, sx, sw):
    """products that vanish beside 1: the loss of every row is log V; and magnitudes at the two ends of the type's range"""
    x, w, labels = _uneven(N, V, D)
    _uneven_check(x * sx, w * sw, labels)


@pytest.mark.parametrize("big", [1.0, 1e9])
def test_linear_ce_f32_uneven_rows_in_pieces_of_the_classes(big):
    """more G than one piece holds (2048 x 80000 x 4 bytes > 512 MiB); 64-bit results on the GPU"""
    x, w, labels = _uneven(2048, 80000, 136)
    x[5] *= big
    w[70000] *= big
    _uneven_check(x, w, labels)


@pytest.mark.parametrize("D", [100, 300])
def test_linear_ce_f32_even_and_uneven_rows_in_one_graph(D):
    """which way the products are formed is decided on the device, call by call: a captured step replayed with either kind of features;
    the forward's copies kept for the backward or made anew give the same bits"""
    N, V = 200, 500
    x, w, labels = _uneven(N, V, D)
    one, far = torch.ones((), device="cuda"), torch.ones(N, 1, device="cuda")
    far[7] = 1e10
    kinds = [x * far, x.clone(), x * far.flip(0)]

    def step(keep):
        loss, nll, saved = ops.linear_ce(x, w, labels, temperature=0.1, keep=keep)
        return (loss, nll, *ops.linear_ce_bwd(x, w, saved, one, temperature=0.1))
    want = []
    for k in kinds:
        x.copy_(k)
        want.append([t.clone() for t in step(True)])
        assert all(torch.equal(a, b) for a, b in zip(want[-1], step(False)))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(True)
    for rep in range(2):
        for k, ref in zip(kinds, want):
            x.copy_(k)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(ref, out))
            step(True)


# ------------------------------------------------------------------------------ cross entropy, 16 bit: rows surer than 2^-24
def _margin_bounds(x, w, labels, tau):
    """64-bit nll and how far it may be off: 16-bit products are exact, a fp32 sum of D terms is off by (D + 8) 2^-24 of their magnitudes,
    a difference of two logits by both and four roundings, and nll = log(1 + sum over the other classes of exp(-margin)) is as sure,
    relatively, as the margins (and 64 roundings)"""
    x, w = x.double(), w.double()
    col = labels[:, None]
    z = x @ w.t() / tau
    e = (x.shape[1] + 8) * O.U32 * (x.abs() @ w.abs().t()) / tau
    d = z - z.gather(1, col)
    e = e + e.gather(1, col) + 4 * O.U32 * (z.abs() + z.abs().gather(1, col))
    other = torch.ones_like(z).scatter_(1, col, 0.0)
    nll, up = torch.log1p((torch.exp(d) * other).sum(1)), torch.log1p((torch.exp(d + e) * other).sum(1))
    return nll, (up - nll) + 64 * O.U32 * nll


@pytest.mark.parametrize("dt", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("N,V,D", [(24, 1500, 64), (300, 1025, 64), (300, 5000, 256), (70, 70000, 128), (300, 1025, 320), (70, 9000, 512)])
def test_linear_ce_16_bit_confident_rows(N, V, D, dt):
    """logits of 10 to 500, the label's far in front: the loss is never negative and keeps its digits"""
    w = _unit(V, D, V).to(dt).cuda()
    labels = torch.randint(0, V, (N,), generator=gen(N)).cuda()
    x = (w[labels].float() * torch.logspace(-0.7, 1.0, N, device="cuda")[:, None]).to(dt)
    loss, nll = loss_ops.linear_cross_entropy(x, w, labels, temperature=0.02, reduction="sum")
    want, bound = _margin_bounds(x.cpu(), w.cpu(), labels.cpu(), 0.02)
    assert float(nll.min()) >= 0.0 and float(want.min()) < 2.0 ** -30
    within(nll, want, bound, "nll")


@pytest.mark.parametrize("dt", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("tau", [0.02, 1e-5, 1e-15])
@pytest.mark.parametrize("N,V,D", [(24, 700, 64), (300, 257, 64), (300, 3000, 128), (300, 3000, 256), (300, 1025, 320)])
def test_linear_ce_gradients_of_sure_rows(N, V, D, dt, tau):
    """logits of 10 to 500 at tau 0.02, to 10^16 at the smallest: the softmax gradient of a row is the other classes' probabilities and, at
    the label, minus their sum; each is as sure, relatively, as the margins e (and its rounding for the matrix cores: u_g, not below
    2^-39 of 1 for the fp16 pieces), so that a row that is sure beyond doubt gets no gradient"""
    w = _unit(V, D, V).to(dt).cuda()
    labels = torch.randint(0, V, (N,), generator=gen(N)).cuda()
    x = (w[labels].float() * torch.logspace(-0.7, 1.0, N, device="cuda")[:, None]).to(dt)
    a, b = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    loss, nll = loss_ops.linear_cross_entropy(a, b, labels, temperature=tau, reduction="sum")
    gx, gw = torch.autograd.grad(loss, (a, b))
    xd, wd, lab = x.double().cpu(), w.double().cpu(), labels.cpu()
    z = xd @ wd.t() / tau
    prod = 2.0 ** -20 if dt == F32 else 0.0
    e = (prod + (D + 8) * O.U32) * (xd.abs() @ wd.abs().t()) / tau
    d, e = z - z.gather(1, lab[:, None]), e + e.gather(1, lab[:, None])
    hot = torch.zeros_like(z).scatter_(1, lab[:, None], 1.0)
    e = e + 4 * O.U32 * (z.abs() + z.abs().gather(1, lab[:, None]))

    def others(t):                                                    # probabilities of the other classes for margins t
        q = torch.exp(t.clamp(max=700)) * (1 - hot)
        return q / (1 + q.sum(1, keepdim=True))
    q = others(d)
    top = (torch.exp((d + e).clamp(max=700)) * (1 - hot)).clamp(max=1.0)          # (a probability is at most its ratio to the label's, and 1)
    e_q = (top - q).clamp(min=0) + (q - (torch.exp(d - e) * (1 - hot)) / (1 + (torch.exp((d + e).clamp(max=700)) * (1 - hot)).sum(1, keepdim=True))).clamp(min=0)
    G, mag = q - hot * q.sum(1, keepdim=True), q + hot * q.sum(1, keepdim=True)
    u_g = {BF16: 2.0 ** -8, F16: 2.0 ** -11, F32: 2.0 ** -20}[dt]
    floor = 2.0 ** -126 if dt == BF16 else 2.0 ** -39                  # (bf16: a probability below fp32's normal range may be taken as 0)
    e_G = e_q + hot * e_q.sum(1, keepdim=True).clamp(max=1.0) + (u_g + (max(N, V) + 64) * O.U32) * mag + floor
    half = O.half_step(dt)
    tiny = 2.0 ** -24 if dt == F16 else 0.0
    for got, want, bound, name in ((gx, G @ wd / tau, e_G @ wd.abs() / tau, "dx"), (gw, G.t() @ xd / tau, e_G.t() @ xd.abs() / tau, "dw")):
        if dt == F16 and float(want.abs().max() + bound.max()) > 6e4:
            continue                                                  # (beyond the type)
        within(got, want, 1.01 * bound + half * want.abs() + tiny, name)


@pytest.mark.parametrize("xo,wo", [(0, 0), (1, 0), (0, 1), (1, 1)])
@pytest.mark.parametrize("N,V,D", [(32, 500, 64), (7, 500, 128), (20, 300, 320), (32, 300, 40)])
def test_linear_ce_f32_few_rows_in_place_or_copied(N, V, D, xo, wo):
    """up to 32 rows stay fp32 in both directions; rows off their 16 bytes are copied; kept copies or new ones: the same bits"""
    x, w, labels = _uneven(N, V, D)

    def at(t, off):
        buf = torch.zeros(t.numel() + 4, device="cuda")
        buf[off:off + t.numel()] = t.reshape(-1)
        return buf[off:off + t.numel()].view(t.shape)
    one, got = torch.ones((), device="cuda"), []
    for keep in (False, True):
        loss, nll, saved = ops.linear_ce(at(x, xo), at(w, wo), labels, temperature=0.1, keep=keep)
        got.append((loss, nll, *ops.linear_ce_bwd(at(x, xo), at(w, wo), saved, one, temperature=0.1)))
    assert all(torch.equal(u, v) for u, v in zip(*got))
    _uneven_check(at(x, xo), at(w, wo), labels)
    _uneven_check(at(x * 1e6, xo), at(w, wo), labels)                 # logits of 10^7


# ------------------------------------------------------------------------------------------------------------ very many rows
def test_linear_ce_more_than_2_29_rows():
    """four words a row for the backward pass 2^31 words; rows at both ends and around 2^29, all others ignored"""
    N, V, D = (1 << 29) + 1000, 5, 8
    w = _unit(V, D, 1).to(BF16).cuda()
    at = torch.tensor([0, 1, 65, (1 << 28) + 7, (1 << 29) - 1, 1 << 29, (1 << 29) + 63, N - 1], device="cuda")
    lab = torch.full((N,), -100, device="cuda")
    lab[at] = torch.arange(8, device="cuda") % V
    x = torch.zeros(N, D, dtype=BF16, device="cuda")
    x[at] = torch.randn(8, D, generator=gen(2)).to(BF16).cuda()
    loss, nll, saved = ops.linear_ce(x, w, lab, reduction="sum")
    r = O.linear_ce(x[at], w, lab[at], -100, 1.0, False)
    within(nll[at], r["nll"], r["e_nll"], "nll")
    assert int(torch.count_nonzero(nll)) == 8 and abs(float(loss) - float(r["loss"])) <= float(r["e_loss"])
    del lab
    gx, gw = ops.linear_ce_bwd(x, w, saved, torch.ones((), device="cuda"), reduction="sum")
    within(gx[at], r["gx"], r["e_gx"], "dx")
    within(gw, r["gw"], r["e_gw"], "dw")
    gx[at] = 0
    assert not gx[:1 << 20].any() and not gx[-(1 << 20):].any() and not gx[(1 << 29) - 4096:(1 << 29) + 1000].any()


# ------------------------------------------------------------------------------------------------------------- layouts
def test_views_that_record_a_negation():
    """.imag of a conjugate (also as a cotangent) is a view that keeps the memory and records the sign"""
    def neg(t):
        v = torch._neg_view(-t)
        assert v.is_neg() and v.is_contiguous() and torch.equal(v, t)
        return v
    x, res = torch.randn(2, 37, device="cuda").unbind(0)
    gate, xs, gh = torch.randn(3, 2, 70, 6, device="cuda").unbind(0)
    h0 = torch.randn(2, 6, device="cuda")
    f, w, lab = torch.randn(40, 64, device="cuda"), torch.randn(9, 64, device="cuda"), torch.arange(40, device="cuda") % 9

    def all_of(t):
        y = ops.dropout(t(x), 0.3, 1, residual=t(res))
        h, last, st = ops.gated_recurrence(t(gate), t(xs), t(h0), save=True)
        back = ops.gated_recurrence_bwd(t(gate), t(xs), None, st, t(gh), t(last))
        loss, nll, saved = ops.linear_ce(t(f), t(w), lab)
        out = [y, h, last, *back, loss, nll, *ops.linear_ce_bwd(t(f), t(w), saved, t(loss))]
        leaves = [u.clone().requires_grad_(True) for u in (x, gate, xs, h0, f, w)]
        h, last = train_ops.gated_recurrence(*leaves[1:4])
        loss, _ = loss_ops.linear_cross_entropy(leaves[4], leaves[5], lab)
        return out + list(torch.autograd.grad((train_ops.dropout(leaves[0], 0.3, 1), h, last, loss), leaves, (t(x), t(gh), t(h0), t(loss.detach()))))
    want, got = all_of(lambda t: t), all_of(neg)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("shape", [(0, 5, 4), (2, 70, 0), (2, 0, 4)])
def test_recurrence_halves_of_empty_batches(shape):
    """what the forward saves of an empty batch is what the backward asks for"""
    x = torch.zeros(shape, device="cuda")
    h, last, starts = ops.gated_recurrence(x, x, save=True)
    gg, gx, gh0 = ops.gated_recurrence_bwd(x, x, None, starts, h, last)
    assert gg.shape == gx.shape == h.shape == x.shape and gh0.shape == last.shape == (shape[0], shape[2])


@pytest.mark.parametrize("dt", [F32, BF16], ids=["f32", "bf16"])
def test_linear_ce_overlapping_windows(dt):
    """features that are windows of one signal, a row a few elements behind the one before"""
    for D, step in ((64, 8), (37, 3), (320, 64)):
        sig = torch.randn(3000, generator=gen(D)).to(dt).cuda()
        x, w = sig.unfold(0, D, step)[:40], sig[:1500].unfold(0, D, 2 * step)[:9]
        assert 0 < x.stride(0) < D
        lab = torch.arange(40, device="cuda") % 9
        want, got = [], []
        for a, b, out in ((x.contiguous(), w.contiguous(), want), (x, w, got)):
            loss, nll, saved = ops.linear_ce(a, b, lab)
            out += [loss, nll, *ops.linear_ce_bwd(a, b, saved, loss)]
            a, b = a.detach().requires_grad_(True), b.detach().requires_grad_(True)
            loss, nll = loss_ops.linear_cross_entropy(a, b, lab)
            out += [loss, nll, *torch.autograd.grad(loss, (a, b))]
        assert all(torch.equal(u, v) for u, v in zip(want, got))
