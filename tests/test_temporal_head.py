"""CPU: what the operators of the temporal classification head refuse, the C ABI's own argument checks, and the oracle's random
words against the published vectors of the generator."""
import ctypes as C

import numpy as np
import pytest
import torch

from creste_public_amd import _lib, loss_ops, ops, train_ops
from tests.temporal_head_oracle import philox_words

E = _lib.HipLibraryError


def test_philox_known_answers():
    """the 10-round vectors published with the generator (Salmon et al., SC 2011, known-answer tests)"""
    def block(ctr, key):
        i = ctr[0] | ctr[1] << 32
        return [int(w) for w in philox_words(np.array([i], dtype=np.uint64), ctr[2] | ctr[3] << 32, key[0] | key[1] << 32)[0]]
    assert block((0, 0, 0, 0), (0, 0)) == [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]
    f = 0xffffffff
    assert block((f, f, f, f), (f, f)) == [0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd]
    assert block((0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344), (0xa4093822, 0x299f31d0)) == \
        [0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1]


@pytest.mark.parametrize("call", [
    lambda x: ops.dropout(x, 0.1, 1),
    lambda x: train_ops.dropout(x, 0.1, 1),
    lambda x: ops.gated_recurrence(x, x),
    lambda x: train_ops.gated_recurrence(x, x),
    lambda x: ops.linear_ce(x[0], x[0], torch.zeros(x.shape[1], dtype=torch.long)),
    lambda x: loss_ops.linear_cross_entropy(x, x[0], torch.zeros(x.shape[:2], dtype=torch.long))])
def test_cpu_tensors_are_refused(call):
    with pytest.raises(E, match="CUDA/HIP tensor"):
        call(torch.zeros(2, 3, 4))


def test_shapes_are_checked_before_the_library_is_asked():
    x = torch.zeros(2, 3, 4)
    with pytest.raises(E, match="labels must have the shape"):
        loss_ops.linear_cross_entropy(x, x[0], torch.zeros(6, dtype=torch.long))
    with pytest.raises(E, match=r"x \[\.\.\.,D\]"):
        loss_ops.linear_cross_entropy(torch.zeros(()), x[0], torch.zeros(1))
    with pytest.raises(E, match="does not fit 64 bits"):
        ops._int64(1 << 64, "seed")
    assert ops._int64((1 << 64) - 1, "seed") == -1 and ops._int64(-5, "seed") == -5


def test_entry_points_report_bad_arguments():
    """host-side checks only: every call returns before anything is launched"""
    lib = _lib.load()
    p = C.c_void_p(4096)                   # never dereferenced

    def err(rc, text):
        assert rc == -1 and text in lib.creste_last_error(), lib.creste_last_error()

    def fwd(x=p, N=4, V=8, D=16, dt=0, tau=1.0, ldx=16, ldw=16, work=p, nb=1 << 40):
        return lib.creste_linear_ce_forward(x, ldx, p, ldw, p, N, V, D, dt, -100, tau, 1, p, p, p, p, None, work, nb, None)
    err(fwd(x=None), b"null pointer")
    err(fwd(dt=3), b"dtype")
    err(fwd(N=0), b"N 0")
    err(fwd(V=1 << 30), b"V 1073741824")
    err(fwd(D=65537), b"D 65537")
    err(fwd(ldx=15), b"row strides")
    err(fwd(ldw=-16), b"row strides")
    err(fwd(tau=0.0), b"temperature")
    err(fwd(tau=float("nan")), b"temperature")
    err(fwd(tau=float("inf")), b"temperature")
    err(fwd(tau=1e-40), b"temperature")
    err(fwd(nb=1000), b"workspace")
    err(fwd(work=None), b"workspace")
    err(lib.creste_linear_ce_backward(p, 16, p, 16, p, 4, 8, 16, 0, 1.0, 1, p, p, None, None, None, p, 1 << 40, None), b"inputs")
    odd = C.c_void_p(4104)
    err(fwd(work=odd), b"16-byte")
    err(lib.creste_linear_ce_backward(p, 16, p, 16, p, 4, 8, 16, 0, 1.0, 1, p, p, None, odd, None, p, 1 << 40, None), b"16-byte")
    for bad in ((0, 8, 16, 0), (4, 0, 16, 0), (4, 8, 0, 0), (4, 8, 16, 5), (1 << 31, 8, 16, 0)):
        assert lib.creste_linear_ce_workspace_bytes(*bad, 1) == -1

    err(lib.creste_dropout(p, None, p, 0, 0, 0.1, 1, 0, None, None), b"bad args")
    err(lib.creste_dropout(p, None, p, 8, 0, -0.1, 1, 0, None, None), b"outside [0, 1]")
    err(lib.creste_dropout(p, None, p, 8, 0, float("nan"), 1, 0, None, None), b"outside [0, 1]")
    err(lib.creste_dropout(p, None, p, 8, 7, 0.1, 1, 0, None, None), b"dtype")

    def rec(gate=p, B=2, T=3, Cc=4, dt=0, nb=1 << 40):
        return lib.creste_gated_recurrence_forward(gate, 12, 4, p, 12, 4, None, None, B, T, Cc, dt, p, p, None, p, nb, None)
    err(rec(gate=None), b"null pointer")
    err(rec(T=0), b"T 0")
    err(rec(B=1 << 31), b"B 2147483648")
    err(rec(T=300, nb=3), b"workspace")
    assert lib.creste_gated_recurrence_workspace_bytes(2, 3, 4) == 0          # a single chunk of steps needs none
    err(rec(dt=9), b"dtype")
    err(lib.creste_gated_recurrence_backward(p, 12, 4, p, 12, 4, p, 12, 4, None, None, None, 2, 3, 4, 0, p, p, None, p, 1 << 40, None),
        b"null pointer")
    assert lib.creste_gated_recurrence_workspace_bytes(0, 3, 4) == -1


def test_which_operands_are_copied():
    """the backward reads a copy of x; of w only where it is not 16-bit rows of 64, 128, 256 or more multiples of 64 elements on 16 bytes"""
    f = _lib.load().creste_linear_ce_packs_bytes
    at = C.c_void_p(4096)
    alone = f(at, 128, at, 128, 100, 50, 128, 1)
    assert 100 * 128 * 2 <= alone < 100 * 128 * 2 + 8192
    assert f(at, 136, at, 4096, 100, 50, 128, 1) == alone                          # wider rows
    assert f(C.c_void_p(4098), 128, at, 128, 100, 50, 128, 1) == alone
    for both in (f(at, 100, at, 128, 100, 50, 100, 1), f(at, 128, C.c_void_p(4098), 128, 100, 50, 128, 1),
                 f(at, 128, at, 129, 100, 50, 128, 1), f(at, 128, at, 128, 100, 50, 128, 0) - 150 * 128 * 2):
        assert alone + 50 * 128 * 2 <= both < alone + 50 * 128 * 2 + 8192          # padded to 128; fp32: two pieces
    assert f(at, 128, at, 128, 30, 50, 128, 0) == 0                                # few rows: read in place by the forward
    assert f(at, 128, at, 128, 0, 50, 128, 0) == -1


@pytest.mark.parametrize("N,V,D,dt", [(1, 1, 1, 0), (19584, 4096, 128, 0), (4096, 131072, 1024, 1), (1 << 20, 1 << 20, 64, 1),
                                      ((1 << 30) - 1, 3, 8, 2)])
def test_gradient_workspace_is_bounded(N, V, D, dt):
    """no N x V buffer: the piece of G stays at 512 MiB (one 256-class tile at least) whatever N and V are"""
    lib = _lib.load()
    es, P = (4, 2) if dt == 0 else (2, 1)
    Dp = -(-D // 64) * 64
    packs = (N + V) * Dp * 2 * P
    train = lib.creste_linear_ce_workspace_bytes(N, V, D, dt, 1)
    tile = -(-N // 64) * 64 * 256 * 2 * P
    partials = 4 * max(N, 1) * (-(-D // 4) * 4) * 256 if N * D < 1 << 26 else 4 * N * (-(-D // 4) * 4)
    assert 0 < train <= packs + max(512 << 20, tile) + partials + (1 << 30)
    fwd = lib.creste_linear_ce_workspace_bytes(N, V, D, dt, 0)
    assert fwd <= packs + 8 * N * (-(-V // 256)) + 5 * N + 16384      # one (max, sum) pair per row and 256 classes
