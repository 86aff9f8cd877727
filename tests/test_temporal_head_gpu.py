"""GPU: the operators of the temporal classification head (csrc/linear_ce.hip, dropout.hip, recurrence.hip) against their 64-bit
definitions, elementwise within derived bounds (temporal_head_oracle.py)."""
import contextlib

import pytest
import torch

from creste_public_amd import _lib, loss_ops, ops, train_ops
from tests import temporal_head_oracle as O
from tests.temporal_head_oracle import within

pytestmark = pytest.mark.gpu
E = _lib.HipLibraryError
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
ALL = [F32, BF16, F16]
IDS = ["f32", "bf16", "f16"]


def gen(seed):
    return torch.Generator().manual_seed(seed)


# ------------------------------------------------------------------------------------------------------------ dropout
def _dropout_ok(y, x, res, p, seed, offset, first=0):
    keep = O.keep_mask(first, x.numel(), p, seed, offset).reshape(x.shape)
    xd = x.double().cpu()
    scale = 1.0 / (1.0 - p) if p < 1 else 0.0
    want = torch.where(keep, xd * scale, torch.zeros_like(xd))
    mag = want.abs()
    if res is not None:
        want = want + res.double().cpu()
        mag = mag + want.abs()
    half = O.half_step(x.dtype)
    within(y, want, half * want.abs() + 3 * O.U32 * mag + (2.0 ** -25 if x.dtype == F16 else 0), "dropout")


@pytest.mark.parametrize("dt", ALL, ids=IDS)
@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 7, 8, 9, 15, 17, 63, 1000, 4099, 262147])
def test_dropout_forward_backward(dt, n):
    for k, (p, res) in enumerate([(0.1, False), (0.5, True)]):
        g = gen(n + k)
        x, r, gy = (torch.randn(n, generator=g).to(dt).cuda() for _ in range(3))
        x.requires_grad_(True)
        r.requires_grad_(True)
        seed, off = 0x9E3779B97F4A7C15 + n, (7 << 40) + k
        y = train_ops.dropout(x, p, seed, off, residual=r if res else None)
        assert y.dtype == dt and y.shape == x.shape
        _dropout_ok(y, x.detach(), r.detach() if res else None, p, seed, off)
        grads = torch.autograd.grad(y, (x, r) if res else (x,), gy)
        _dropout_ok(grads[0], gy, None, p, seed, off)
        if res:
            assert torch.equal(grads[1], gy)


@pytest.mark.parametrize("dt", ALL, ids=IDS)
def test_dropout_limits_and_masked_values(dt):
    x = torch.randn(1003, generator=gen(1)).to(dt).cuda()
    assert torch.equal(ops.dropout(x, 0.0, 3), x)
    assert torch.equal(ops.dropout(x, 1.0, 3), torch.zeros_like(x))
    assert torch.equal(ops.dropout(x, 1.0, 3, residual=x), x)
    assert torch.equal(ops.dropout(x, 1.0 - 2.0 ** -60, 3, residual=x), x)          # rounds to p = 1
    keep = O.keep_mask(0, 1003, 0.5, 3, 0)
    bad = torch.where(keep.cuda(), x, torch.full_like(x, float("nan")))
    bad[~keep.cuda()] = torch.where(torch.arange(int((~keep).sum()), device="cuda") % 2 == 0, float("inf"), float("nan")).to(dt)
    y = ops.dropout(bad, 0.5, 3)
    assert torch.isfinite(y).all() and torch.equal(y == 0, (~keep).cuda() | (x == 0))
    assert ops.dropout(x[:0], 0.5, 3).numel() == 0
    assert ops.dropout(x[:1].reshape(()), 0.0, 3).shape == ()


@pytest.mark.parametrize("dt", ALL, ids=IDS)
def test_dropout_strides_and_alignment(dt):
    """the draw goes by the element's index in x's shape, not by where it lies"""
    base = torch.randn(5, 33, 18, generator=gen(2)).to(dt).cuda()
    want = ops.dropout(base, 0.3, 11, 5)
    for v in (base.transpose(1, 2).contiguous().transpose(1, 2), base.permute(2, 0, 1).contiguous().permute(1, 2, 0)):
        assert not v.is_contiguous() and torch.equal(ops.dropout(v, 0.3, 11, 5), want)
        assert torch.equal(ops.dropout(base, 0.3, 11, 5, residual=v), ops.dropout(base, 0.3, 11, 5, residual=base))
    flat = torch.randn(4001, generator=gen(3)).to(dt).cuda()
    for o in (1, 2, 3, 5):                                                    # pointers that are not aligned to a vector
        assert torch.equal(ops.dropout(flat[o:], 0.3, 11), ops.dropout(flat[o:].clone(), 0.3, 11))
        assert torch.equal(ops.dropout(flat[o:], 0.3, 11, residual=flat[:-o]),
                           ops.dropout(flat[o:].clone(), 0.3, 11, residual=flat[:-o].clone()))


def test_dropout_draws_are_independent_and_fair():
    n = 1 << 20
    x = torch.ones(n, device="cuda")
    a, b, c = ops.dropout(x, 0.25, 5, 0) != 0, ops.dropout(x, 0.25, 5, 1) != 0, ops.dropout(x, 0.25, 6, 0) != 0
    for m in (a, b, c):
        assert abs(float(m.float().mean()) - 0.75) < 6 * (0.75 * 0.25 / n) ** 0.5        # six standard deviations
    for u, v in ((a, b), (a, c), (a[:-1], a[1:])):
        assert abs(float((u & v).float().mean()) - 0.5625) < 6 * (0.5625 * 0.4375 / n) ** 0.5
    t = torch.tensor([5, 1], device="cuda")
    assert torch.equal(ops.dropout(x, 0.25, t) != 0, b)                          # (seed, offset) on the device
    assert torch.equal(ops.dropout(x, 0.25, t, 2) != 0, ops.dropout(x, 0.25, 5, 3) != 0)


def test_dropout_seed_tensor_written_before_the_backward_is_an_error():
    x = torch.randn(64, device="cuda", requires_grad=True)
    t = torch.tensor([5, 1], device="cuda")
    y = train_ops.dropout(x, 0.25, t)
    t[1] += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_dropout_beyond_32_bits():
    n = (1 << 32) + 4096 + 5
    x = torch.ones(n, dtype=BF16, device="cuda")
    y = ops.dropout(x, 0.5, 77, 3)
    first = (1 << 32) - 2048 + 1
    _dropout_ok(y[first:], x[first:], None, 0.5, 77, 3, first)
    _dropout_ok(y[:4096], x[:4096], None, 0.5, 77, 3)


def test_dropout_refusals():
    x = torch.zeros(4, 4, device="cuda")
    for bad in (lambda: ops.dropout(x, -0.1, 1), lambda: ops.dropout(x, 1.5, 1), lambda: ops.dropout(x, float("nan"), 1),
                lambda: ops.dropout(x.double(), 0.1, 1), lambda: ops.dropout(x, 0.1, 1, residual=x[:2]),
                lambda: ops.dropout(x, 0.1, 1, residual=x.half()), lambda: ops.dropout(x, 0.1, torch.zeros(3, dtype=torch.long, device="cuda")),
                lambda: ops.dropout(x, 0.1, torch.zeros(2, dtype=torch.long)), lambda: ops.dropout(x, 0.1, 1 << 64)):
        with pytest.raises(E):
            bad()


# --------------------------------------------------------------------------------------------------- gated recurrence
def _rec_inputs(B, T, Cc, dt, seed=0, scale=1.5, shift=2.0):
    g = gen(seed + B + 31 * T + 7 * Cc)
    gate = (torch.randn(B, T, Cc, generator=g) * scale + shift).to(dt).cuda()
    x, gh = torch.randn(B, T, Cc, generator=g).to(dt).cuda(), torch.randn(B, T, Cc, generator=g).to(dt).cuda()
    h0, gl = torch.randn(B, Cc, generator=g).cuda(), torch.randn(B, Cc, generator=g).cuda()
    return gate, x, gh, h0, gl


def _rec_check(gate, x, h0, lengths, gh, gl):
    gate, x = gate.detach().requires_grad_(True), x.detach().requires_grad_(True)
    h0_ = h0.detach().requires_grad_(True) if h0 is not None else None
    h, last = train_ops.gated_recurrence(gate, x, h0_, lengths)
    assert h.dtype == x.dtype and last.dtype == F32 and h.is_contiguous()
    outs, cots = ((h, last), (gh, gl)) if gl is not None else ((h,), (gh,))
    grads = torch.autograd.grad(outs, (gate, x) + ((h0_,) if h0 is not None else ()), cots)
    ref = O.gated(gate.detach(), x.detach(), h0, lengths, gh, gl)
    within(h, ref["h"], ref["e_h"], "h")
    within(last, ref["last"], ref["e_last"], "h_last")
    within(grads[0], ref["gg"], ref["e_gg"], "dgate")
    within(grads[1], ref["gx"], ref["e_gx"], "dx")
    if h0 is not None:
        within(grads[2], ref["gh0"], ref["e_gh0"], "dh0")
    with torch.no_grad():                                           # the form without a backward gives the same
        h2, last2 = train_ops.gated_recurrence(gate, x, h0, lengths)
    assert torch.equal(h2, h) and torch.equal(last2, last)
    return h, last


@pytest.mark.parametrize("dt", ALL, ids=IDS)
@pytest.mark.parametrize("B,T,Cc", [(1, 1, 1), (64, 1, 33), (3, 2, 5), (2, 7, 130), (2, 8, 2), (1, 9, 64), (3, 63, 6), (2, 64, 128), (2, 65, 129),
                                    (1, 127, 3), (4, 128, 32), (1, 700, 2), (2, 1025, 97), (1, 4099, 1), (700, 20, 48), (3, 130, 260)])
def test_recurrence(B, T, Cc, dt):
    gate, x, gh, h0, gl = _rec_inputs(B, T, Cc, dt)
    _rec_check(gate, x, h0, None, gh, gl)


@pytest.mark.parametrize("dt", ALL, ids=IDS)
def test_recurrence_one_pass_over_many_columns(dt):
    """columns enough for one segment, several chunks of time walked by one workgroup"""
    gate, x, gh, h0, gl = _rec_inputs(140, 150, 512, dt)
    _rec_check(gate, x, h0, None, gh, gl)


@pytest.mark.parametrize("dt", ALL, ids=IDS)
def test_recurrence_lengths(dt):
    """ragged batch incl. empty, full and over-long; whatever lies behind an end -- NaN, infinities, the lowest value -- is not used"""
    B, T, Cc = 9, 200, 37
    gate, x, gh, h0, gl = _rec_inputs(B, T, Cc, dt)
    lengths = torch.tensor([0, 1, 63, 64, 65, 128, 199, 200, 1 << 40], device="cuda")
    _rec_check(gate, x, h0, lengths, gh, gl)
    h, last = _rec_check(gate, x, None, lengths, gh, None)
    poison = torch.arange(T, device="cuda")[None, :, None] >= lengths[:, None, None]
    for bad in (float("nan"), float("inf"), torch.finfo(dt).min):
        h2, last2, st = ops.gated_recurrence(torch.where(poison, bad, gate), torch.where(poison, bad, x), None, lengths, save=True)
        assert torch.equal(h2, h) and torch.equal(last2, last)
        clean = ops.gated_recurrence_bwd(gate, x, lengths, st, gh)
        dirty = ops.gated_recurrence_bwd(torch.where(poison, bad, gate), torch.where(poison, bad, x), lengths, st, torch.where(poison, bad, gh))
        assert all(torch.equal(a, b) for a, b in zip(clean, dirty))
    neg = ops.gated_recurrence(gate, x, h0, torch.full((B,), -3, device="cuda"))
    assert not neg[0].any() and torch.equal(neg[1], h0)


@pytest.mark.parametrize("dt", ALL, ids=IDS)
def test_recurrence_extreme_gates(dt):
    """gates at which sigmoid saturates: the state is held, or replaced"""
    gate, x, gh, h0, gl = _rec_inputs(2, 150, 10, dt, scale=0.0, shift=0.0)
    big = 60.0
    pat = torch.tensor([big, -big, 0.0, 20.0, -20.0], device="cuda").repeat(2).to(dt)
    _rec_check(gate + pat, x, h0, None, gh, gl)
    for v in (float("inf"), torch.finfo(dt).max):
        h, last = ops.gated_recurrence(torch.full_like(gate, v), x, h0)
        assert torch.equal(last, h0)
        h, last = ops.gated_recurrence(torch.full_like(gate, -v), x, h0)
        assert torch.equal(h, x) and torch.equal(last, x[:, -1].float())


@pytest.mark.parametrize("dt", ALL, ids=IDS)
def test_recurrence_strides(dt):
    B, T, Cc = 3, 70, 34
    gate, x, gh, h0, gl = _rec_inputs(B, T, Cc, dt)
    ref = ops.gated_recurrence(gate, x, h0, save=True)
    refb = ops.gated_recurrence_bwd(gate, x, None, ref[2], gh, gl)
    wide = torch.zeros(B, T, 3 * Cc + 1, dtype=dt, device="cuda")
    wide[..., 1:Cc + 1], wide[..., Cc + 1:2 * Cc + 1], wide[..., 2 * Cc + 1:] = gate, x, gh
    forms = [tuple(t.transpose(0, 1).contiguous().transpose(0, 1) for t in (gate, x, gh)),          # time-major
             (wide[..., 1:Cc + 1], wide[..., Cc + 1:2 * Cc + 1], wide[..., 2 * Cc + 1:]),            # slices of one buffer, odd start
             tuple(t.permute(2, 0, 1).contiguous().permute(1, 2, 0) for t in (gate, x, gh))]           # channels first
    for g_, x_, d_ in forms:
        assert not g_.is_contiguous()
        out = ops.gated_recurrence(g_, x_, h0, save=True)
        assert all(torch.equal(a, b) for a, b in zip(ref, out))
        assert all(torch.equal(a, b) for a, b in zip(refb, ops.gated_recurrence_bwd(g_, x_, None, out[2], d_, gl)))
    one = ops.gated_recurrence(gate[:1].expand(B, T, Cc), x, h0)
    assert torch.equal(one[0][0], ref[0][0])
    lead = gate.requires_grad_(True)                                  # a cotangent with zero strides, and none at all for h
    train_ops.gated_recurrence(lead, x, h0)[0].sum().backward()
    a = lead.grad.clone()
    want = ops.gated_recurrence_bwd(gate, x, None, ref[2], torch.ones_like(x))[0]
    assert torch.equal(a, want)
    lead.grad = None
    train_ops.gated_recurrence(lead, x, h0)[1].sum().backward()
    assert torch.equal(lead.grad, ops.gated_recurrence_bwd(gate, x, None, ref[2], torch.zeros_like(x), torch.ones_like(gl))[0])


@pytest.mark.parametrize("dt", ALL, ids=IDS)
def test_recurrence_step_by_step_equals_the_sequence(dt):
    """serving: one step at a time, the state handed on"""
    gate, x, _, h0, _ = _rec_inputs(4, 9, 40, dt)
    h, last = ops.gated_recurrence(gate, x, h0)
    ref = O.gated(gate, x, h0, None)
    s = h0
    for t in range(9):
        ht, s = ops.gated_recurrence(gate[:, t:t + 1], x[:, t:t + 1], s)
        within(ht[:, 0], ref["h"][:, t], ref["e_h"][:, t], f"step {t}")
    within(s, ref["last"], ref["e_last"], "state")


def test_recurrence_gradient_against_differences():
    """central differences of a linear functional of the outputs, step 2^-6: the third derivatives of sigmoid and of the linear scan
    are below 1 per unit step here, so the difference is off by < 2^-12 relative to the gradient's scale, the fp32 outputs' noise
    (2^-22 of a functional of norm ~ 1) by 2^-16: 2e-3 of the directional derivative's scale holds both"""
    gate, x, gh, h0, gl = _rec_inputs(2, 90, 6, F32)
    _, _, st = ops.gated_recurrence(gate, x, h0, save=True)
    gg, gx, gh0 = (t.double() for t in ops.gated_recurrence_bwd(gate, x, None, st, gh, gl))

    def f(a, b, c):
        h, last = ops.gated_recurrence(a, b, c)
        return float((h.double() * gh.double()).sum() + (last.double() * gl.double()).sum())
    eps = 2.0 ** -6
    for i, (t, g) in enumerate(((gate, gg), (x, gx), (h0, gh0))):
        d = torch.randn(t.shape, generator=gen(50 + i)).cuda()
        d /= d.norm()
        args = [gate, x, h0]
        up, dn = list(args), list(args)
        up[i], dn[i] = t + eps * d, t - eps * d
        num, ana = (f(*up) - f(*dn)) / (2 * eps), float((g * d.double()).sum())
        assert abs(num - ana) < 2e-3 * float(g.norm()) + 1e-4, (i, num, ana)


def test_recurrence_beyond_32_bits():
    B, T, Cc = 3, 1 << 16, 11008                                    # 2.2e9 elements: 64-bit offsets in every operand
    gate = torch.full((B, T, Cc), 1.0, dtype=BF16, device="cuda")
    x = torch.zeros((B, T, Cc), dtype=BF16, device="cuda")
    x[-1, -200:, -64:] = torch.randn(200, 64, generator=gen(9)).to(BF16).cuda()
    h, last = ops.gated_recurrence(gate, x)
    ref = O.gated(gate[-1:, -200:, -64:], x[-1:, -200:, -64:], None, None)
    within(h[-1:, -200:, -64:], ref["h"], ref["e_h"], "h")
    within(last[-1:, -64:], ref["last"], ref["e_last"], "h_last")
    assert not h[:-1].any()


def test_recurrence_refusals_and_empty():
    x = torch.zeros(2, 3, 4, device="cuda")
    for bad in (lambda: ops.gated_recurrence(x[0], x[0]), lambda: ops.gated_recurrence(x, x[:, :2]), lambda: ops.gated_recurrence(x, x.half()),
                lambda: ops.gated_recurrence(x.double(), x.double()), lambda: ops.gated_recurrence(x, x, x[:, 0].half()),
                lambda: ops.gated_recurrence(x, x, x[:, 0, :3]), lambda: ops.gated_recurrence(x, x, None, torch.tensor([1, 2])),
                lambda: ops.gated_recurrence(x, x, None, torch.tensor([1, 2], dtype=torch.int32, device="cuda")),
                lambda: ops.gated_recurrence(x, x, None, torch.tensor([1], device="cuda"))):
        with pytest.raises(E):
            bad()
    h0 = torch.randn(2, 4, device="cuda", requires_grad=True)
    e = torch.zeros(2, 0, 4, device="cuda", requires_grad=True)
    h, last = train_ops.gated_recurrence(e, e, h0)
    assert h.shape == (2, 0, 4) and torch.equal(last, h0)
    last.sum().backward()
    assert torch.equal(h0.grad, torch.ones_like(h0))
    assert ops.gated_recurrence(x[:0], x[:0])[1].shape == (0, 4)


# ------------------------------------------------------------------------------------------------ linear cross entropy
def _ce_inputs(N, V, D, dt, seed=0, ignore=0.1, normed=True):
    g = gen(seed + N + 3 * V + 7 * D)
    w = torch.randn(V, D, generator=g)
    labels = torch.randint(0, V, (N,), generator=g)
    x = torch.randn(N, D, generator=g)
    if normed:
        w = w / w.norm(dim=1, keepdim=True)
        x = w[labels] + x * (1.5 / D ** 0.5)
        x = x / x.norm(dim=1, keepdim=True)
    labels[torch.rand(N, generator=g) < ignore] = -100
    return x.to(dt).cuda(), w.to(dt).cuda(), labels.cuda()


def _ce_check(x, w, labels, tau=0.1, ignore=-100, reduction="mean", gl=1.0):
    x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    loss, nll = loss_ops.linear_cross_entropy(x, w, labels, ignore, tau, reduction)
    gx, gw = torch.autograd.grad(loss * gl, (x, w))
    r = O.linear_ce(x.detach(), w.detach(), labels, ignore, tau, reduction == "mean", gl)
    assert loss.dtype == nll.dtype == F32 and gx.dtype == x.dtype
    within(nll, r["nll"], r["e_nll"], "nll")
    within(loss, r["loss"], r["e_loss"], "loss")
    within(gx, r["gx"], r["e_gx"], "dx")
    within(gw, r["gw"], r["e_gw"], "dw")
    return loss, nll, gx, gw


@pytest.mark.parametrize("dt", ALL, ids=IDS)
@pytest.mark.parametrize("N,V,D", [(1, 1, 1), (1, 2, 8), (2, 3, 7), (5, 257, 64), (31, 255, 65), (32, 256, 128), (33, 1003, 24), (64, 64, 63), (257, 513, 130),
                                   (300, 1000, 256), (700, 129, 33), (1531, 700, 200), (100, 5000, 320), (16, 20000, 64),
                                   (70, 5377, 37), (70, 1345, 100), (70, 1345, 250), (70, 1281, 260), (40, 4097, 64)])
def test_linear_ce(N, V, D, dt):
    _ce_check(*_ce_inputs(N, V, D, dt))


@pytest.mark.parametrize("dt", ALL, ids=IDS)
def test_linear_ce_options(dt):
    x, w, labels = _ce_inputs(200, 300, 96, dt)
    _ce_check(x, w, labels, reduction="sum", gl=0.25)
    _ce_check(x, w, labels, tau=1.0, gl=-3.0)
    labels[labels == -100] = 7
    labels[::5] = 299
    _ce_check(x, w, labels, ignore=299)                               # a class as the ignored label
    x3 = x.reshape(10, 20, 96)                                        # leading dimensions
    loss, nll = loss_ops.linear_cross_entropy(x3, w, labels.reshape(10, 20), temperature=0.1)
    l2, n2 = loss_ops.linear_cross_entropy(x, w, labels, temperature=0.1)
    assert torch.equal(loss, l2) and torch.equal(nll.reshape(-1), n2)


@pytest.mark.parametrize("dt", ALL, ids=IDS)
def test_linear_ce_nothing_counts(dt):
    x, w, labels = _ce_inputs(70, 300, 64, dt)
    loss, nll, gx, gw = _ce_check(x, w, torch.full_like(labels, -100))
    assert float(loss) == 0 and not nll.any() and not gx.any() and not gw.any()
    x = x[:0].requires_grad_(True)
    w = w.requires_grad_(True)
    loss, nll = loss_ops.linear_cross_entropy(x, w, labels[:0])
    assert float(loss) == 0 and nll.shape == (0,)
    gx, gw = torch.autograd.grad(loss, (x, w))
    assert gx.shape == (0, 64) and not gw.any()


@pytest.mark.parametrize("N,V,D", [(5, 300, 64), (70, 300, 64), (70, 300, 37), (130, 2000, 128), (90, 300, 320)])
@pytest.mark.parametrize("keep", [False, True])
@pytest.mark.parametrize("dt", ALL, ids=IDS)
def test_linear_ce_ignored_rows_may_hold_anything(dt, N, V, D, keep):
    """padding: infinities, NaN and huge values in rows that do not count, the last one among them -- the same bits as with zeros there"""
    x, w, labels = _ce_inputs(N, V, D, dt)
    labels[::3] = -100
    labels[-1] = -100
    off = labels == -100
    one, got = torch.ones((), device="cuda"), []
    for bad in (False, True):
        xb = torch.where(off[:, None], torch.zeros_like(x), x)
        if bad:
            junk = torch.tensor([float("nan"), float("inf"), float("-inf"), torch.finfo(dt).max], device="cuda", dtype=dt)
            xb = torch.where(off[:, None], junk[torch.arange(N, device="cuda") % 4][:, None].expand(N, D), x).contiguous()
        loss, nll, saved = ops.linear_ce(xb, w, labels, temperature=0.1, keep=keep)
        got.append((loss, nll, *ops.linear_ce_bwd(xb, w, saved, one, temperature=0.1)))
    assert all(bool(t.isfinite().all()) for t in got[1])
    assert all(torch.equal(u, v) for u, v in zip(*got))
    assert not got[1][2][off].any()


def test_linear_ce_label_without_a_class_is_loud():
    x, w, labels = _ce_inputs(70, 300, 64, F32, ignore=0)
    for bad in (300, -1, 1 << 40, -(1 << 40)):
        lab = labels.clone()
        lab[13] = bad
        a, b = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        loss, nll = loss_ops.linear_cross_entropy(a, b, lab)
        assert torch.isnan(loss) and torch.isnan(nll[13]) and int(torch.isnan(nll).sum()) == 1
        gx, gw = torch.autograd.grad(loss, (a, b))
        assert torch.isnan(gx[13]).all() and torch.isnan(gw).any()


@pytest.mark.parametrize("dt", ALL, ids=IDS)
def test_linear_ce_large_logits(dt):
    """unnormalised features: logits of several hundred, confident and hopeless rows"""
    x, w, labels = _ce_inputs(130, 500, 128, dt, normed=False)
    _ce_check(x, w * 4, labels, tau=1.0)
    _ce_check(x * 0, w, labels)                                       # all classes alike (and a zero operand scale)


def test_linear_ce_uneven_scales_f32():
    x, w, labels = _ce_inputs(90, 300, 64, F32)
    _ce_check(x * 1e-6, w * 1e6, labels)
    _ce_check(x * 1e8, w * 1e-9, labels)


@pytest.mark.parametrize("dt", ALL, ids=IDS)
def test_linear_ce_strides(dt):
    x, w, labels = _ce_inputs(90, 300, 128, dt)
    ref = [t.clone() for t in _ce_check(x, w, labels)]
    wide = torch.zeros(90, 300, dtype=dt, device="cuda")
    wide[:, 5:133] = x
    wb = torch.zeros(300, 137, dtype=dt, device="cuda")
    wb[:, 9:] = w
    big = torch.zeros(300, 264, dtype=dt, device="cuda")
    big[:, 8:136] = w
    for xv, wv in ((wide[:, 5:133], wb[:, 9:]), (x.t().contiguous().t(), w.t().contiguous().t()), (x, big[:, 8:136])):
        got = _ce_check(xv, wv, labels)
        assert all(torch.equal(a, b) for a, b in zip(ref, got))
    _ce_check(x[:1].expand(90, 128), w, labels)


@pytest.mark.parametrize("dt", ALL, ids=IDS)
def test_linear_ce_kept_copies(dt):
    """the copies of the operands kept by the forward or made anew by the backward (large operands, tensors laid out anew): the same bits"""
    x, w, labels = _ce_inputs(90, 300, 100, dt)
    one = torch.ones((), device="cuda")
    a, b = ops.linear_ce(x, w, labels, temperature=0.1, keep=True), ops.linear_ce(x, w, labels, temperature=0.1)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and a[2].numel() > b[2].numel()        # (x [90,100]: padded)
    ga, gb = (ops.linear_ce_bwd(x, w, t[2], one, temperature=0.1) for t in (a, b))
    assert all(torch.equal(u, v) for u, v in zip(ga, gb))
    for bad in (a[2][:100], b[2].half()):
        with pytest.raises(E):
            ops.linear_ce_bwd(x, w, bad, one, temperature=0.1)


def test_linear_ce_saved_tensors_come_back_laid_out_anew():
    """16-bit features of 64: the weight off its 16 bytes is copied by the forward, and read in place after its way over the host"""
    buf = torch.randn(90 * 64 + 1, device="cuda", dtype=F16)
    x, labels = torch.randn(90, 64, device="cuda", dtype=F16), torch.randint(0, 90, (90,), device="cuda")
    grads = []
    for hooks in (False, True):
        wl = buf[1:].view(90, 64).detach().requires_grad_(True)
        xl = x.clone().requires_grad_(True)
        with torch.autograd.graph.save_on_cpu() if hooks else contextlib.nullcontext():
            loss, _ = loss_ops.linear_cross_entropy(xl, wl, labels, temperature=4.0)
        grads.append(torch.autograd.grad(loss, (xl, wl)))
    assert all(torch.equal(u, v) for u, v in zip(*grads))


def test_linear_ce_one_sided_gradients():
    x, w, labels = _ce_inputs(90, 300, 64, BF16)
    xa, wa = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    gx, gw = torch.autograd.grad(loss_ops.linear_cross_entropy(xa, wa, labels)[0], (xa, wa))
    assert torch.equal(gx, torch.autograd.grad(loss_ops.linear_cross_entropy(xa, w, labels)[0], xa)[0])
    assert torch.equal(gw, torch.autograd.grad(loss_ops.linear_cross_entropy(x, wa, labels)[0], wa)[0])
    assert not loss_ops.linear_cross_entropy(x, w, labels)[0].requires_grad


def test_linear_ce_is_deterministic():
    for dt in ALL:
        x, w, labels = _ce_inputs(700, 3000, 192, dt)
        a = [t.clone() for t in _ce_check(x, w, labels)]
        for _ in range(3):
            xa, wa = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
            loss, nll = loss_ops.linear_cross_entropy(xa, wa, labels, temperature=0.1)
            assert all(torch.equal(u, v) for u, v in zip(a, (loss, nll) + torch.autograd.grad(loss, (xa, wa))))


@pytest.mark.parametrize("D", [64, 264])
def test_linear_ce_pieces(D, dt=BF16):
    """more G than one piece holds: streamed past, or (D > 256) dx added up over pieces and dw written piece by piece.  64-bit results on
    the GPU"""
    N, V = 6000, 70000
    x, w, labels = _ce_inputs(N, V, D, dt)
    lib = _lib.load()
    assert 2 * N * V > 512 << 20 and lib.creste_linear_ce_workspace_bytes(N, V, D, _lib.DT_BF16, 1) < 2 * N * V
    xa, wa = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    loss, nll = loss_ops.linear_cross_entropy(xa, wa, labels, temperature=0.1)
    gx, gw = torch.autograd.grad(loss, (xa, wa))
    xd, wd = x.double(), w.double()
    on = labels != -100
    s = 1.0 / (0.1 * float(on.sum()))
    gw_ref, bw, gx_ref, bx = torch.zeros_like(wd), torch.zeros_like(wd), torch.zeros_like(xd), torch.zeros_like(xd)
    for i in range(0, N, 1000):
        z = xd[i:i + 1000] @ wd.t().contiguous() / 0.1
        p = torch.exp(z - torch.logsumexp(z, 1, keepdim=True))
        hot = torch.zeros_like(p).scatter_(1, labels[i:i + 1000].clamp(min=0)[:, None], 1.0)
        m = on[i:i + 1000, None]
        gx_ref[i:i + 1000], bx[i:i + 1000] = s * ((p - hot) * m) @ wd, s * ((p + hot) * m) @ wd.abs()
        gw_ref += s * ((p - hot) * m).t().contiguous() @ xd[i:i + 1000]
        bw += s * ((p + hot) * m).t().contiguous() @ xd[i:i + 1000].abs()
    e_p = 2 * (2 * (D + 8) * O.U32 * 10 * 1.5 + 600 * O.U32)          # |x| . |w| <= 1 for unit rows (1.5: rounding to bf16 and the label row)
    within(gx, gx_ref.cpu(), ((2.0 ** -8 + e_p + (V + 64) * O.U32) * bx + 2.0 ** -8 * gx_ref.abs()).cpu() * 1.01, "dx")
    within(gw, gw_ref.cpu(), ((2.0 ** -8 + e_p + (N + 64) * O.U32) * bw + 2.0 ** -8 * gw_ref.abs()).cpu() * 1.01, "dw")


def test_linear_ce_beyond_32_bits():
    """the class matrix passes 2^31 elements"""
    V, D = 2200000, 1024
    w = torch.zeros(V, D, dtype=BF16, device="cuda")
    rows = torch.tensor([0, 1, V - 2, V - 1], device="cuda")
    w[rows] = torch.randn(4, D, generator=gen(4)).to(BF16).cuda()
    x = w[rows].clone() / 64
    xa, wa = x.requires_grad_(True), w.requires_grad_(True)
    loss, nll = loss_ops.linear_cross_entropy(xa, wa, rows, reduction="sum")
    z = x.detach().double() @ w[rows].detach().double().t()
    lse = torch.log(torch.exp(z).sum(1) + (V - 4))                    # the other classes' logits are 0
    bound = torch.full((4,), float(z.abs().max()) * 2 * (D + 16) * O.U32 + 600 * O.U32, dtype=torch.double)
    within(nll, (lse - z.diag()).cpu(), bound, "nll")
    gx, gw = torch.autograd.grad(loss, (xa, wa))
    p = torch.exp(z - lse[:, None]) - torch.eye(4, device="cuda", dtype=torch.double)
    want = p.t() @ x.detach().double()
    tol = (2.0 ** -7 * (p.abs().t() @ x.detach().double().abs())).cpu()
    within(gw[rows], want.cpu(), tol, "dw")
    within(gx, (p @ w[rows].detach().double()).cpu(), (2.0 ** -7 * p.abs() @ w[rows].detach().double().abs()).cpu(), "dx")


def test_linear_ce_streamed_beyond_32_bits():
    """the same for up to 256 feature columns, on either side of the products"""
    V, D, N = 9000000, 256, 70
    w = torch.zeros(V, D, dtype=BF16, device="cuda")
    rows = torch.tensor([0, 1, V - 2, V - 1], device="cuda")
    w[rows] = torch.randn(4, D, generator=gen(4)).to(BF16).cuda()
    lab = rows[torch.arange(N, device="cuda") % 4]
    xa = (w[lab] / 32).requires_grad_(True)
    wa = w.requires_grad_(True)
    loss, nll = loss_ops.linear_cross_entropy(xa, wa, lab, reduction="sum")
    xd, wd = xa.detach().double(), w[rows].detach().double()
    z = xd @ wd.t()
    lse = torch.log(torch.exp(z).sum(1) + (V - 4))
    bound = torch.full((N,), float(z.abs().max()) * 2 * (D + 16) * O.U32 + 600 * O.U32, dtype=torch.double)
    within(nll, (lse - z.gather(1, (torch.arange(N, device="cuda") % 4)[:, None])[:, 0]).cpu(), bound, "nll")
    gx, gw = torch.autograd.grad(loss, (xa, wa))
    p = torch.exp(z - lse[:, None]) - torch.nn.functional.one_hot(torch.arange(N, device="cuda") % 4, 4)
    within(gw[rows], (p.t() @ xd).cpu(), (2.0 ** -7 * (p.abs().t() @ xd.abs())).cpu(), "dw")
    within(gx, (p @ wd).cpu(), (2.0 ** -7 * (p.abs() @ wd.abs())).cpu(), "dx")
    del wa, w, gw
    N, V = 9000000, 70                                                # the rows are the long side
    x = torch.zeros(N, D, dtype=BF16, device="cuda")
    w = torch.randn(V, D, generator=gen(5)).to(BF16).cuda()
    at = torch.tensor([0, 1, N - 2, N - 1], device="cuda")
    lab = torch.full((N,), -100, device="cuda")
    lab[at] = torch.tensor([3, 69, 0, 68], device="cuda")
    x[at] = torch.randn(4, D, generator=gen(6)).to(BF16).cuda() / 8
    xa, wa = x.requires_grad_(True), w.requires_grad_(True)
    loss, nll = loss_ops.linear_cross_entropy(xa, wa, lab, reduction="sum")
    gx, gw = torch.autograd.grad(loss, (xa, wa))
    r = O.linear_ce(x[at].detach(), w.detach(), lab[at], -100, 1.0, False)
    within(nll[at], r["nll"], r["e_nll"], "nll")
    within(gx[at], r["gx"], r["e_gx"], "dx")
    within(gw, r["gw"], r["e_gw"], "dw")
    assert not gx[2:-2].any() and not nll[2:-2].any()


@pytest.mark.parametrize("V", [2, 3, 40])
def test_linear_ce_confident_rows_f32(V):
    """the loss of a confident row is about exp(-margin): relative to it, only the margin's absolute error (twice a logit's) and a few
    roundings count, not the rounding of 1 + exp(-margin).  The same for its gradient, nll (w_other - w_label) in norm"""
    N, D = 300, 48
    g = gen(V)
    w = torch.randn(V, D, generator=g)
    w = (w / w.norm(dim=1, keepdim=True)).cuda()
    lab = torch.randint(0, V, (N,), generator=g).cuda()
    x = w[lab] + 0.05 * torch.randn(N, D, generator=g).cuda()
    for tau in (0.1, 0.05):
        r = O.linear_ce(x, w, lab, -100, tau, False)
        xa, wa = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        loss, nll = loss_ops.linear_cross_entropy(xa, wa, lab, temperature=tau, reduction="sum")
        gx, gw = torch.autograd.grad(loss, (xa, wa))
        big = float((x.double().abs() @ w.double().abs().t()).max()) / tau
        rel = 2 * big * (2.0 ** -21 + (D + 8) * O.U32) + 64 * O.U32
        assert float(r["nll"].min()) < 1e-2
        within(nll, r["nll"], rel * r["nll"], "nll")
        z = x.double().cpu() @ w.double().cpu().t() / tau
        p = torch.softmax(z, 1)
        hot = torch.nn.functional.one_hot(lab.cpu(), V).double()
        other = (p * (1 - hot)).sum(1, keepdim=True)
        mag = (p * (1 - hot) + other * hot) / tau                     # |G|
        bound = (rel + 2.0 ** -20 + (V + 64) * O.U32) * (mag @ w.double().cpu().abs()) + O.U32 * r["gx"].abs()
        within(gx, r["gx"], 1.01 * bound + 2.0 ** -39 / tau * w.double().cpu().abs().sum(0), "dx")


def test_linear_ce_gradient_against_differences():
    """central differences with step 2^-5 along unit directions: log-sum-exp's third derivative is below |w|^3 / tau^3 = 1 here and
    the step small, so 2^-10 / 6 of truncation; fp32 losses around 5 (2^-22 each) over 2^-4: 2^-16.  2e-3 absolute holds both"""
    x, w, labels = _ce_inputs(40, 90, 24, F32)
    xa, wa = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    grads = torch.autograd.grad(loss_ops.linear_cross_entropy(xa, wa, labels, temperature=1.0, reduction="sum")[0], (xa, wa))
    eps = 2.0 ** -5
    for i in range(2):
        d = torch.randn(grads[i].shape, generator=gen(60 + i)).cuda()
        d /= d.norm()
        up, dn = [x, w], [x, w]
        up[i], dn[i] = up[i] + eps * d, dn[i] - eps * d
        f = [float(loss_ops.linear_cross_entropy(*a, labels, reduction="sum")[1].double().sum()) for a in (up, dn)]
        assert abs((f[0] - f[1]) / (2 * eps) - float((grads[i] * d).sum())) < 2e-3


def test_linear_ce_refusals():
    x, w, labels = _ce_inputs(6, 5, 8, F32)
    f = loss_ops.linear_cross_entropy
    for bad in (lambda: f(x, w[:, :7], labels), lambda: f(x, w.half(), labels), lambda: f(x.double(), w.double(), labels),
                lambda: f(x, w, labels[:5]), lambda: f(x, w, labels.int()), lambda: f(x, w, labels.cpu()), lambda: f(x, w[0], labels),
                lambda: f(x, w, labels, reduction="none"), lambda: f(x, w, labels, temperature=0.0),
                lambda: f(x, w, labels, temperature=float("nan")), lambda: f(x, w[:0], labels), lambda: f(x[:, :0], w[:, :0], labels)):
        with pytest.raises(E):
            bad()


# ------------------------------------------------------------------------------------------------------------ together
def _head_reference(gate, x, h0, lengths, w, labels, p, seed, tau):
    """the head in 64 bits with torch autograd"""
    ins = [t.detach().double().cpu().requires_grad_(True) for t in (gate, x, h0, w)]
    g, x, h0, w = ins
    B, T, Cc = g.shape
    live = torch.arange(T)[None] < lengths.cpu()[:, None]
    h, hs = h0, []
    for t in range(T):
        n = torch.sigmoid(g[:, t]) * h + torch.sigmoid(-g[:, t]) * x[:, t]
        h = torch.where(live[:, t, None], n, h)
        hs.append(torch.where(live[:, t, None], n, torch.zeros_like(n)))
    y = torch.stack(hs, 1) * O.keep_mask(0, B * T * Cc, p, seed, 0).reshape(B, T, Cc) / (1 - p) + x
    loss = torch.nn.functional.cross_entropy(y.reshape(-1, Cc) @ w.t() / tau, labels.cpu().reshape(-1), ignore_index=-100)
    return loss, torch.autograd.grad(loss, ins)


@pytest.mark.parametrize("dt", ALL, ids=IDS)
def test_head_forward_and_backward(dt):
    """features of frames -> recurrence -> dropout into a residual sum -> prototypes, one training step's gradients.  Rounded
    intermediates (h, y and their cotangents: 5 roundings in a row to the type, G one) are each half a step; relative to a gradient's
    norm 8 half steps hold them, fp32 (products 2^-21, sums of some hundred terms) 2^-15"""
    B, T, Cc, V = 5, 70, 64, 400
    gate, x, _, h0, _ = _rec_inputs(B, T, Cc, dt)
    _, w, _ = _ce_inputs(4, V, Cc, dt)
    lengths = torch.tensor([70, 0, 33, 64, 69], device="cuda")
    labels = torch.randint(0, V, (B, T), generator=gen(8)).cuda()
    labels[torch.arange(T, device="cuda")[None] >= lengths[:, None]] = -100
    leaves = [t.detach().requires_grad_(True) for t in (gate, x, h0, w)]

    def step():
        h, _ = train_ops.gated_recurrence(leaves[0], leaves[1], leaves[2], lengths)
        y = train_ops.dropout(h, 0.2, 1234, residual=leaves[1])
        loss, _ = loss_ops.linear_cross_entropy(y, leaves[3], labels, temperature=0.5)
        return (loss.detach(),) + torch.autograd.grad(loss, leaves)
    got = step()
    loss, grads = _head_reference(gate, x, h0, lengths, w, labels, 0.2, 1234, 0.5)
    tol = 2.0 ** -15 if dt == F32 else 8 * O.half_step(dt)
    assert abs(float(got[0]) - float(loss)) < tol * float(loss)
    for a, b, name in zip(got[1:], grads, ("gate", "x", "h0", "w")):
        assert float((a.double().cpu() - b).norm()) < tol * float(b.norm()), name
    side = torch.cuda.Stream()                                        # another stream than the leaves' own
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


def test_two_calls_at_once():
    """the same operators on two streams at the same time (the recurrence's workgroups wait for each other within a call only)"""
    jobs = []
    for k in range(2):
        gate, x, gh, h0, gl = _rec_inputs(4, 3000 + 500 * k, 256, BF16, seed=k)
        xs, w, lab = _ce_inputs(3000, 2000, 128, BF16, seed=k)
        jobs.append((gate, x, gh, h0, gl, xs, w, lab))

    def work(j):
        gate, x, gh, h0, gl, xs, w, lab = j
        h, last, st = ops.gated_recurrence(gate, x, h0, save=True)
        back = ops.gated_recurrence_bwd(gate, x, None, st, gh, gl)
        loss, nll, saved = ops.linear_ce(xs, w, lab, temperature=0.1)
        return (h, last) + back + (loss, nll) + ops.linear_ce_bwd(xs, w, saved, torch.ones_like(loss), temperature=0.1)
    want = [[t.clone() for t in work(j)] for j in jobs]
    streams = [torch.cuda.Stream() for _ in jobs]
    torch.cuda.synchronize()
    outs = [[], []]
    for rep in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(work(jobs[i]))
    torch.cuda.synchronize()
    for w_, got in zip(want, outs):
        for o in got:
            assert all(torch.equal(a, b) for a, b in zip(w_, o))


def test_dropout_twice_differentiable():
    x = torch.randn(300, generator=gen(3)).cuda().requires_grad_(True)
    y = train_ops.dropout(x, 0.3, 9)
    g, = torch.autograd.grad((y ** 3).sum(), x, create_graph=True)
    gg, = torch.autograd.grad(g.sum(), x)
    k = O.keep_mask(0, 300, 0.3, 9, 0).cuda() / 0.7
    want = 6 * x.detach().double() * k ** 3
    within(gg, want.cpu(), (16 * O.U32 * want.abs()).cpu(), "second derivative")
    gate, xx, gh, h0, gl = _rec_inputs(1, 3, 2, F32)
    h, _ = train_ops.gated_recurrence(gate.requires_grad_(True), xx, h0)
    g, = torch.autograd.grad(h.sum(), gate, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable|does not require grad"):
        torch.autograd.grad(g.sum(), gate)


def test_autograd_is_refused_inside_a_capture():
    x = torch.randn(2, 3, 64, device="cuda", requires_grad=True)
    w, lab = torch.randn(5, 64, device="cuda"), torch.zeros(2, 3, dtype=torch.long, device="cuda")
    calls = (lambda t: train_ops.dropout(t, 0.5, 1), lambda t: train_ops.gated_recurrence(t, t), lambda t: loss_ops.linear_cross_entropy(t, w, lab))
    for f in calls:
        f(x.detach())
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        for f in calls:
            with pytest.raises(E, match="under stream capture"):
                f(x)
            f(x.detach())
    g.replay()
    torch.cuda.synchronize()


@pytest.mark.parametrize("dt", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("keep", [False, True])
def test_head_in_two_captured_graphs(keep, dt):
    """forward and backward entry points captured; two graphs with workspaces of their own, replayed in turn with eager work between,
    new inputs and a new draw each time"""
    B, T, Cc, V = 3, 200, 64, 600
    gate, x, _, h0, _ = _rec_inputs(B, T, Cc, dt)
    _, w, _ = _ce_inputs(4, V, Cc, dt)
    labels = torch.randint(0, V, (B * T,), generator=gen(8)).cuda()
    one = torch.ones((), device="cuda")

    def step(rng):
        h, last, st = ops.gated_recurrence(gate, x, h0, save=True)
        y = ops.dropout(h, 0.2, rng)
        loss, nll, saved = ops.linear_ce(y.reshape(-1, Cc), w, labels, temperature=0.5, keep=keep)
        gy, gw = ops.linear_ce_bwd(y.reshape(-1, Cc), w, saved, one, temperature=0.5)
        gg, gx, gh0 = ops.gated_recurrence_bwd(gate, x, None, st, ops.dropout(gy, 0.2, rng).reshape(B, T, Cc), last)
        return loss, nll, gw, gg, gx, gh0
    rngs = [torch.tensor([5, i], device="cuda") for i in range(2)]
    graphs, outs = [], []
    for r in rngs:
        step(r)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(r))
        graphs.append(g)
    for rep in range(4):
        x.copy_(torch.randn(B, T, Cc, generator=gen(100 + rep)).to(dt))
        for r in rngs:
            r[1] += 2
        want = [[t.clone() for t in step(r)] for r in rngs]
        torch.cuda.synchronize()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for a, b in zip(want, outs):
            assert all(torch.equal(u, v) for u, v in zip(a, b))
        assert not torch.equal(outs[0][0], outs[1][0])
