"""CPU: sizes that the operators of the temporal classification head refuse before anything is launched, and what their host side decides."""
import ctypes as C

import pytest
import torch
from torch.autograd import forward_ad

from creste_public_amd import _lib, loss_ops, ops, train_ops

P = C.c_void_p(4096)                       # never dereferenced


def _refused(rc, text):
    assert rc == -1 and text in _lib.load().creste_last_error(), (rc, _lib.load().creste_last_error())


def test_launches_of_more_threads_than_the_device_takes_are_refused():
    """a launch holds less than 2^32 threads a dimension; more is an error of the arguments, not of the launch"""
    lib = _lib.load()
    for B, T, Cc in ((1 << 12, 1, 1 << 21), (1 << 12, 1, (1 << 20) + 1), (1 << 8, 1 << 20, 1 << 14)):
        need = lib.creste_gated_recurrence_workspace_bytes(B, T, Cc)
        assert need >= 0
        rc = lib.creste_gated_recurrence_forward(P, T * Cc, Cc, P, T * Cc, Cc, None, None, B, T, Cc, 1, P, P, None, P, 1 << 62, None)
        _refused(rc, b"too many columns")
    N = V = 1 << 20
    rc = lib.creste_linear_ce_forward(P, 512, P, 512, P, N, V, 512, 1, -100, 1.0, 1, P, P, P, P, None, P, 1 << 62, None)
    _refused(rc, b"too many tiles")


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("call", [
    lambda d, p: train_ops.dropout(d, 0.5, 1), lambda d, p: train_ops.dropout(p, 0.5, 1, residual=d),
    lambda d, p: train_ops.gated_recurrence(d, p), lambda d, p: train_ops.gated_recurrence(p, d),
    lambda d, p: train_ops.gated_recurrence(p, p, d[:, 0]),
    lambda d, p: loss_ops.linear_cross_entropy(d, p[0], torch.zeros(2, 3, dtype=torch.long)),
    lambda d, p: loss_ops.linear_cross_entropy(p, d[0], torch.zeros(2, 3, dtype=torch.long))])
def test_forward_mode_derivatives_are_refused(call, grad):
    """a tangent that were dropped would read as a derivative of 0; also where nothing is recorded for a backward"""
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        d = forward_ad.make_dual(torch.randn(2, 3, 4), torch.ones(2, 3, 4))
        with pytest.raises(NotImplementedError):
            call(d, torch.randn(2, 3, 4))
    with pytest.raises(NotImplementedError):
        torch.func.jvp(lambda t: call(t, torch.randn(2, 3, 4)), (torch.randn(2, 3, 4),), (torch.ones(2, 3, 4),))


def test_a_level_without_tangents_is_no_obstacle():
    with forward_ad.dual_level():
        assert train_ops.recorded(torch.randn(3)) is False and train_ops.recorded(torch.randn(3, requires_grad=True), None) is True


def test_tensors_in_the_place_of_numbers_are_refused():
    """they would be read back to the host, and their gradient would be None without a word"""
    x, w, lab = torch.randn(3, 4), torch.randn(5, 4), torch.zeros(3, dtype=torch.long)
    for t in (torch.tensor(0.1), torch.tensor(0.1, requires_grad=True), torch.nn.Parameter(torch.ones(()))):
        for call in (lambda: loss_ops.linear_cross_entropy(x, w, lab, temperature=t), lambda: ops.linear_ce(x, w, lab, -100, t),
                     lambda: ops.linear_ce_bwd(x, w, x, x, temperature=t), lambda: train_ops.dropout(x, t, 1), lambda: ops.dropout(x, t, 1)):
            with pytest.raises(_lib.HipLibraryError, match="a number expected"):
                call()


@pytest.mark.parametrize("N,V,D,dt", [(156672, 131072, 256, 1), (1 << 20, 1 << 20, 64, 1), (19584, 4096, 128, 0), (100000, 50000, 200, 2),
                                      (33, 1 << 20, 64, 1), (1, 7, 3, 0), (32, 1 << 20, 128, 0)])
def test_streamed_forward_keeps_one_statistic_per_split(N, V, D, dt):
    """up to 256 feature columns (fp32: 128) the forward leaves one (maximum, rest) per row and split, and no more splits than fill eight
    rounds of 256 workgroups of 512 rows; few rows: one per 256 classes"""
    es, most = (4, 128) if dt == 0 else (2, 256)
    assert D <= most
    packs = (N + V) * (64 if D <= 64 else 128 if D <= 128 else 256) * es
    stats = 8 * (2048 * 512 + N) if N > 32 else 8 * N * max(-(-V // 256), 256)
    assert 0 < _lib.load().creste_linear_ce_workspace_bytes(N, V, D, dt, 0) <= packs + stats + 5 * N + 16384


def test_temperatures_whose_scale_overflows_are_refused():
    """logits are taken in units of log2(e) / temperature: 1 / temperature may be finite where that is not"""
    lib = _lib.load()
    for tau in (1 / 3.0e38, 1 / 2.4e38):
        rc = lib.creste_linear_ce_forward(P, 16, P, 16, P, 4, 8, 16, 0, -100, tau, 1, P, P, P, P, None, P, 1000, None)
        _refused(rc, b"temperature")
    rc = lib.creste_linear_ce_forward(P, 16, P, 16, P, 4, 8, 16, 0, -100, 1 / 2.3e38, 1, P, P, P, P, None, P, 1000, None)
    _refused(rc, b"workspace")
