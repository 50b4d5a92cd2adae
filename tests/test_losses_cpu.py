"""Refusals of the losses' C entry points that need no GPU, beside those of test_optim_cpu.py."""
import ctypes

import pytest


@pytest.fixture(scope="module")
def lib():
    from nvfp4_sm120_b200 import build, _lib
    build.build()
    return _lib


class Rows(ctypes.Structure):
    _fields_ = [("logits", ctypes.c_void_p), ("is_f32", ctypes.c_int)] + \
               [(n, ctypes.c_int64) for n in ("batch", "seq", "vocab", "stride_b", "stride_t")] + \
               [("labels", ctypes.c_void_p), ("ignore", ctypes.c_int64)]


def test_preference_checks_its_arguments_for_both_references(lib):
    buf = ctypes.create_string_buffer(1 << 16)
    p = (ctypes.addressof(buf) + 255) & ~255                   # host memory: only argument checks run
    rows = dict(logits=p, is_f32=1, batch=2, seq=3, vocab=5, stride_b=15, stride_t=5, labels=p, ignore=-100)

    def call(name, ref=p, stat=p, ws=1 << 20, **kw):
        return getattr(lib.lib(), name)(ctypes.byref(Rows(**{**rows, **kw})), ref, 0.1, 0.0, p, stat, p, p, p, p, ws, None)

    for name in ("nvfp4_preference_fwd", "nvfp4_preference_fwd_ref64"):
        assert call(name, batch=3) == -2 and call(name, ws=16) == -7 and call(name, ref=None) == -1
        assert call(name, ref=p + 2) == -3 and call(name, stat=p + 4) == -3 and call(name, logits=p + 2) == -3
    assert call("nvfp4_preference_fwd_ref64", ref=p + 4) == -3


def test_row_statistics_are_pairs(lib):
    """Two fp32 words a row, on an 8-byte boundary."""
    buf = ctypes.create_string_buffer(1 << 16)
    p = (ctypes.addressof(buf) + 255) & ~255
    r = Rows(p, 1, 2, 3, 5, 15, 5, p, -100)
    L = lib.lib()
    assert L.nvfp4_logprob_fwd(ctypes.byref(r), p, p + 4, None) == -3
    assert L.nvfp4_logprob_bwd(ctypes.byref(r), p + 4, p, 1, None, 0, p, 15, 5, None) == -3
    assert L.nvfp4_policy_fwd(ctypes.byref(r), p, p, 3, None, 0.2, 0.2, 0.0, p, p + 4, p, p, p, p, None, 0, 0, p, 1 << 20, None) == -3
