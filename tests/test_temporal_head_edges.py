"""CPU: sizes that the operators of the temporal classification head refuse before anything is launched, and what their host side decides."""
import ctypes as C

from creste_public_amd import _lib

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
