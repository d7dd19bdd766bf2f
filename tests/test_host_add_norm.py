"""`mxa_add_rms_norm_q8_k` and `HipFusedOps.add_rms_norm` without a GPU: what they refuse, with nothing launched."""

import ctypes

import pytest
import torch

from matricxon_amd.fused_ops import HipFusedOps, _broadcasts
from matricxon_amd.gemm import HipGemm


def test_argument_errors_return_status_without_launching() -> None:
    from matricxon_amd import _lib

    lib = _lib.load()
    vp = ctypes.c_void_p
    a = vp(0x10000)  # a well-aligned stand-in: nothing is dereferenced on these paths

    def call(x=a, ldx=512, r=a, ldr=512, post=None, gate=None, ldg=0, gstep=0, w=a, m=2, k=512, bf16=1, rbf16=1,
             hidden=a, out=a, ws=None, ws_bytes=0):
        return lib.mxa_add_rms_norm_q8_k(x, ldx, r, ldr, post, 1e-5, gate, ldg, gstep, 1.0, w, 1e-5, m, k, bf16, rbf16,
                                         hidden, out, ws, ws_bytes, None)

    for bad in (dict(x=None), dict(r=None), dict(w=None), dict(hidden=None), dict(out=None), dict(m=0), dict(k=0),
                dict(k=32769), dict(ldx=-1), dict(ldr=-1), dict(ldg=-1), dict(gstep=2), dict(bf16=0, rbf16=1),
                dict(x=vp(0x10001)), dict(bf16=0, rbf16=0, x=vp(0x10002)), dict(rbf16=0, r=vp(0x10002)),
                dict(gate=vp(0x10001)), dict(post=vp(0x10001)), dict(ws=vp(0x10008), ws_bytes=1 << 20),
                dict(ws=a, ws_bytes=1 << 20, k=300)):
        assert call(**bad) == -1, bad
    assert call(ws=a, ws_bytes=100) == -2


def test_host_tensors_are_left_to_the_caller() -> None:
    x, w = torch.zeros(2, 512), torch.zeros(512)
    assert HipFusedOps().add_rms_norm(x, x, w, 1e-5) is None
    with pytest.raises(ValueError, match="HIP device"):
        HipGemm.get().add_rms_norm_q8k(x, x, w, 1e-5)


def test_broadcasts() -> None:
    to = torch.Size((3, 5, 8))
    for shape in ((), (1,), (8,), (5, 1), (5, 8), (1, 8), (3, 1, 1), (3, 5, 8), (3, 1, 8)):
        assert _broadcasts(torch.Size(shape), to), shape
        torch.zeros(shape).expand(to)
    for shape in ((5,), (3, 8), (2, 5, 8), (1, 3, 5, 8), (3, 5, 2)):
        assert not _broadcasts(torch.Size(shape), to), shape
        with pytest.raises(RuntimeError):
            torch.zeros(shape).expand(to) if shape != (1, 3, 5, 8) else torch.zeros(shape).expand(*to)


def test_more_rows_than_a_grid_holds_are_refused() -> None:
    from matricxon_amd import _lib

    a = ctypes.c_void_p(0x10000)
    for m in ((1 << 24) + 1, 2 ** 31 - 1):
        assert _lib.load().mxa_add_rms_norm_q8_k(a, 1, a, 1, None, 1e-5, None, 0, 0, 1.0, a, 1e-5, m, 1, 1, 1, a, a, None,
                                                 0, None) == -1


def test_more_values_than_a_grid_holds_are_refused() -> None:
    """Rows of up to 1024 threads each, of counts that alone are within the limit; inputs of one row cost no memory."""
    from matricxon_amd import _lib

    a = ctypes.c_void_p(0x10000)
    for m, k in ((1 << 24, 4096), (1 << 23, 8192), (1 << 22, 16384), (1 << 22, 32768), ((1 << 20) + 1, 32768),
                 (1 << 24, 2049)):
        for bf16 in (0, 1):
            assert _lib.load().mxa_add_rms_norm_q8_k(a, 0, a, 0, None, 1e-5, None, 0, 0, 1.0, a, 1e-5, m, k, bf16, bf16, a,
                                                     a, None, 0, None) == -1, (m, k)


def test_every_grid_that_is_taken_is_below_2_to_the_32() -> None:
    """The launch's threads at the most rows that each length may have: whole waves of eight values a lane, in one, two
    or four vectors."""
    total, rows = 1 << 35, 1 << 24
    assert HipGemm.NORM_MAX_TOTAL == total and HipGemm.MAX_TOKENS == rows
    for k in range(1, HipGemm.NORM_MAX_VALUES + 1):
        vectors = (k + 7) // 8
        for per_thread in (1, 2, 4):
            threads = ((vectors + per_thread - 1) // per_thread + 63) // 64 * 64
            many = min(rows, total // k)
            if threads > 1024 or (per_thread == 1 and vectors >= 128):  # two at least where there are many rows
                continue
            assert (many + 3) * threads < 1 << 32, (k, per_thread)
