"""`mxa_norm_rope` and `mxa_kv4_*` without a GPU: sizes, and what is refused before anything is launched."""

import ctypes

import pytest
import torch

VP = ctypes.c_void_p
A, ODD, ST = VP(0x10000), VP(0x10001), (ctypes.c_longlong * 3)(0, 1024, 64)


@pytest.fixture(scope="module")
def lib():
    from matricxon_amd import _lib

    return _lib.load()


def test_page_bytes(lib) -> None:
    assert lib.mxa_kv4_page_bytes(8, 64, 128) == 8 * 2 * 5120  # 5 bits a value of keys and of values
    assert lib.mxa_kv4_page_bytes(1, 32, 8) == 1280 and lib.mxa_kv4_page_bytes(3, 96, 40) == 3 * 3 * 2560
    for bad in ((0, 64, 128), (4097, 64, 128), (8, 0, 128), (8, 48, 128), (8, 1 << 17, 128), (8, 64, 0), (8, 64, 12),
                (8, 64, 264), (-1, 64, 128), (8, -32, 128)):
        assert lib.mxa_kv4_page_bytes(*bad) == 0, bad


def test_norm_rope_refuses_without_launching(lib) -> None:
    def call(q=A, qs=ST, hq=4, qw=A, k=A, ks=ST, hk=2, kw=A, pos=A, pos64=1, turns=A, n=3, seq=3, dim=64, rot=64, bf16=1,
             q_out=A, k_out=A):
        return lib.mxa_norm_rope(q, qs, hq, qw, k, ks, hk, kw, 1e-6, pos, pos64, 0, 1, turns, n, seq, dim, rot, 0, 1.0,
                                 bf16, q_out, k_out, None)

    for bad in (dict(q=None), dict(qs=None), dict(hq=0), dict(hq=65537), dict(hk=-1), dict(hk=65537), dict(k=None),
                dict(ks=None), dict(k_out=None), dict(q_out=None), dict(pos=None), dict(turns=None), dict(n=0),
                dict(n=(1 << 24) + 1), dict(seq=0), dict(dim=0), dict(dim=63, rot=62), dict(dim=1026, rot=64), dict(rot=0),
                dict(rot=66), dict(rot=63), dict(q=ODD), dict(bf16=0, q=VP(0x10002)), dict(k=ODD), dict(q_out=ODD),
                dict(k_out=ODD), dict(qw=ODD), dict(kw=ODD), dict(pos=VP(0x10004)), dict(pos64=0, pos=VP(0x10002)),
                dict(turns=VP(0x10004))):
        assert call(**bad) == -1, bad


PLACES = dict(pages=A, n_pages=4, heads=2, page=32, dim=64, table=A, width=2, lengths=A, starts=None, n_seq=3)
BAD_PLACES = (dict(pages=None), dict(pages=VP(0x10008)), dict(n_pages=0), dict(heads=0), dict(heads=4097), dict(page=16),
              dict(page=40), dict(page=1 << 17), dict(dim=0), dict(dim=60), dict(dim=264), dict(table=None),
              dict(table=VP(0x10002)), dict(width=0), dict(width=(1 << 25) + 1), dict(lengths=None),
              dict(lengths=VP(0x10002)), dict(starts=VP(0x10002)), dict(n_seq=0), dict(n_seq=65536), dict(n=0), dict(n=4),
              dict(n=3 << 23))


def places(p):
    return (p["pages"], p["n_pages"], p["heads"], p["page"], p["dim"], p["table"], 2, p["width"], p["lengths"], p["starts"],
            p["n_seq"])


def test_append_refuses_without_launching(lib) -> None:
    def call(q=A, qs=ST, hq=4, qw=A, k=A, ks=ST, kw=A, v=A, vs=ST, pos=None, pos64=0, turns=A, n=3, seq=3, rot=64, bf16=1,
             q_out=A, **where):
        return lib.mxa_kv4_append(q, qs, hq, qw, k, ks, kw, v, vs, 1e-6, pos, pos64, 0, 1, turns, n, seq, rot, 0, 1.0, bf16,
                                  *places({**PLACES, **where}), q_out, None)

    for bad in (*BAD_PLACES, dict(q=None), dict(qs=None), dict(q_out=None), dict(hq=-1), dict(hq=3), dict(hq=65538),
                dict(k=None), dict(ks=None), dict(v=None), dict(vs=None), dict(q=ODD), dict(k=ODD), dict(v=ODD),
                dict(q_out=ODD), dict(qw=ODD), dict(kw=ODD), dict(bf16=0, k=VP(0x10002)), dict(seq=0), dict(rot=-2),
                dict(rot=66), dict(rot=31), dict(turns=None), dict(turns=VP(0x10004)), dict(pos=VP(0x10002)),
                dict(pos=VP(0x10004), pos64=1)):
        assert call(**bad) == -1, bad


def test_read_refuses_without_launching(lib) -> None:
    def call(n=3, bf16=1, k_out=A, v_out=A, **where):
        return lib.mxa_kv4_read(*places({**PLACES, **where}), n, bf16, k_out, v_out, None)

    for bad in (*BAD_PLACES, dict(k_out=None), dict(v_out=None), dict(k_out=ODD), dict(v_out=ODD),
                dict(bf16=0, v_out=VP(0x10002))):
        assert call(**bad) == -1, bad


def test_attend_refuses_without_launching(lib) -> None:
    def call(q=A, qs=ST, hq=4, n=3, seq=3, most=64, window=0, out=A, ws=A, ws_bytes=1 << 40, **where):
        return lib.mxa_kv4_attend(q, qs, hq, n, seq, *places({**PLACES, **where}), most, window, 0.1, out, ws, ws_bytes,
                                  None)

    for bad in (*BAD_PLACES, dict(q=None), dict(qs=None), dict(out=None), dict(q=ODD), dict(out=ODD), dict(hq=0), dict(hq=3),
                dict(hq=65538), dict(seq=0), dict(most=0), dict(window=-1), dict(n=1 << 24, hq=18, n_seq=1, seq=1 << 24)):
        assert call(**bad) == -1, bad
    long = dict(width=1 << 12, most=1 << 17)  # shared out over workgroups, which needs a workspace
    need = lib.mxa_kv4_attend_workspace_bytes(3, 3, 0, 4, 2, 64, 1 << 17, 0)
    assert need > 0
    assert call(ws=None, **long) == -2 and call(ws_bytes=need - 1, **long) == -2 and call(ws=VP(0x10008), **long) == -1


def test_workspace_bytes(lib) -> None:
    for bad in ((0, 3, 0, 4, 2, 64, 64, 0), (3, 0, 0, 4, 2, 64, 64, 0), (3, 4, 0, 4, 2, 64, 64, 0), (3, 3, 0, 4, 0, 64, 64, 0),
                (3, 3, 0, 1, 2, 64, 64, 0), (3, 3, 0, 5, 2, 64, 64, 0), (3, 3, 0, 4, 2, 0, 64, 0), (3, 3, 0, 4, 2, 264, 64, 0),
                (3, 3, 0, 4, 2, 64, 0, 0), (3, 3, 0, 4, 2, 64, 64, -1)):
        assert lib.mxa_kv4_attend_workspace_bytes(*bad) == 0, bad
    assert lib.mxa_kv4_attend_workspace_bytes(3, 3, 0, 4, 2, 64, 64, 0) == 0  # a workgroup takes all of 64 places
    # a window bounds what is shared out, whatever its size
    for n in (1, 174):
        want = lib.mxa_kv4_attend_workspace_bytes(7, 7 * n, 0, 10, 2, 64, 640, 0)
        for window in (1 << 30, (1 << 31) - 175, (1 << 31) - 1):
            assert lib.mxa_kv4_attend_workspace_bytes(7, 7 * n, 0, 10, 2, 64, 640, window) == want > 0
    assert lib.mxa_kv4_attend_workspace_bytes(1, 1, 0, 4, 2, 64, 1 << 20, 64) == 0


@pytest.mark.parametrize("max_length", [64, 640, 768, 20000, 1 << 30])
@pytest.mark.parametrize("shape", [(7, 174, 1, 10, 2, 64), (1, 512, 0, 32, 8, 128), (3, 3, 0, 4, 2, 256), (4, 515, 1, 40, 8, 64)])
def test_windows_past_every_length_change_no_workspace(lib, shape, max_length) -> None:
    """What a launch needs is computed with the window cut to the most places there are; the query's numbers are the same."""
    want = lib.mxa_kv4_attend_workspace_bytes(*shape, max_length, 0)
    for window in (1 << 30, (1 << 31) - 512, (1 << 31) - 175, (1 << 31) - 1):
        assert lib.mxa_kv4_attend_workspace_bytes(*shape, max_length, window) == want


def test_workspace_stays_small(lib) -> None:
    """Many sequences, rows that differ, long tables: the parts share 256 MiB, and are as many as the rows need."""
    for shape in ((64, 575, 1, 32, 8, 128), (64, 64, 0, 32, 8, 128), (1000, 1000, 0, 64, 8, 256), (65535, 65535, 1, 32, 8, 128),
                  (4, 8000, 1, 32, 8, 128)):
        for most in (4096, 1 << 20, 1 << 30):
            assert lib.mxa_kv4_attend_workspace_bytes(*shape, most, 0) <= 2 * (1 << 28), (shape, most)


def test_a_cache_lies_on_a_device() -> None:
    from matricxon_amd.attention import HipPagedCache

    with pytest.raises(ValueError, match="HIP device"):
        HipPagedCache(2, 32, 2, 64, device="cpu")
    with pytest.raises(ValueError, match="HIP device"):
        HipPagedCache(2, 32, 2, 64, pages=torch.zeros(2, 2, 1, 2560, dtype=torch.uint8))
    with pytest.raises(ValueError, match="page_size"):
        HipPagedCache(2, 48, 2, 64)
