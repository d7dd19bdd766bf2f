"""How kernels' work is laid out over workgroups, on the CPU: the host code that decides it, built alone."""

import ctypes
import shutil
import subprocess

import pytest

from tests.conftest import REPO

CSRC = REPO / "matricxon_amd" / "csrc"
SOURCE = """
#include "mxa_attend_plan.hpp"
#include "mxa_heads_grid.hpp"
extern "C" void heads(int cache, int size, int interleaved, int qh, int kh, int n, int dim, int rot, int* out) {
  const mxa::HeadGrid g = mxa::heads_grid(cache, size, interleaved, qh, kh, n, dim, rot);
  out[0] = g.fast, out[1] = g.L, out[2] = g.TP, out[3] = g.HQ, out[4] = g.HK, out[5] = g.split;
}
extern "C" void plan(int n_seq, int n, int ragged, int kv_heads, int group, int most, int window, int dim, long long* out) {
  const mxa::Plan p = mxa::plan_of(n_seq, n, ragged != 0, kv_heads, group, most, window, dim);
  out[0] = p.few ? p.splits[0] : 0, out[1] = p.chunk[0], out[2] = p.many ? p.splits[1] : 0, out[3] = p.per[0];
  out[4] = p.floats[0], out[5] = p.slots, out[6] = (long long)mxa::parts_bytes(p), out[7] = (long long)mxa::part_bytes(p, 0);
}
"""


@pytest.fixture(scope="module")
def grids(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("no g++")
    at = tmp_path_factory.mktemp("grids")
    (at / "grids.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", "-I", str(CSRC), "-o",
                    str(at / "grids.so"), str(at / "grids.cpp")], check=True)
    return ctypes.CDLL(str(at / "grids.so"))


HEADS = [(1, 1), (7, 3), (32, 8), (64, 8), (8, 64), (1, 65), (33, 65), (24, 0), (100, 0), (40000, 0), (65536, 3),
         (3, 65536), (65536, 65536)]
WIDTHS = [(128, 128), (64, 32), (80, 50), (2, 2), (256, 256), (256, 64), (192, 190), (1024, 1024), (1024, 8)]


@pytest.mark.parametrize("dim, rot", WIDTHS)
@pytest.mark.parametrize("size", [2, 4])
@pytest.mark.parametrize("interleaved", [0, 1])
def test_every_workgroup_of_head_norms_has_a_head(grids, dim, rot, size, interleaved) -> None:
    """Each head lies in one y, and no y begins behind the last head of both: a workgroup asks for its first rows before it
    counts them, and would read behind k."""
    out = (ctypes.c_int * 6)()
    for n in (1, 5, 512, 513, 9001):
        for qh, kh in [*HEADS, *((q, k) for q in range(1, 80, 3) for k in (0, 1, 2, 5, 8, 9))]:
            grids.heads(0, size, interleaved, qh, kh, n, dim, rot, out)
            _, lanes, _, hq, hk, split = out
            assert 1 <= split <= 4096 and 1 <= lanes <= 64
            assert split * hq >= qh and split * hk >= kh
            assert (split - 1) * hq < qh or (split - 1) * hk < kh, (qh, kh, n)


@pytest.mark.parametrize("dim, rot", [(8, 0), (40, 10), (64, 64), (128, 128), (256, 64), (256, 256)])
@pytest.mark.parametrize("size", [2, 4])
def test_every_workgroup_of_an_append_has_a_key_head(grids, dim, rot, size) -> None:
    """Its LDS within 64 KB, and the query heads of its key heads beside them."""
    out = (ctypes.c_int * 6)()
    for n in (1, 256, 257, 2499, 2500, 4096, 1 << 24):
        for kh in (1, 2, 3, 5, 8, 17, 100, 4096):
            for group in (0, 1, 3, 4, 16):
                grids.heads(1, size, 0, kh * group, kh, n, dim, rot, out)
                _, _, tokens, hq, hk, split = out
                assert hq == hk * group and split * hk >= kh > (split - 1) * hk
                assert tokens * (16 + 4 * (hk * -(-dim // 32) * 32 + rot)) <= 65536


def plan(grids, n_seq, n, ragged, kv_heads, group, most, window=0, dim=128):
    out = (ctypes.c_longlong * 8)()
    grids.plan(n_seq, n, ragged, kv_heads, group, most, window, dim, out)
    return list(out)


@pytest.mark.parametrize("most", [4096, 131072, 1 << 20])
@pytest.mark.parametrize("replies", [1, 3, 15])
def test_replies_keep_their_shares_beside_a_chunk(grids, replies, most) -> None:
    """However long the chunk: a reply's places go in shares of 128 blocks at most, or as many as the room for parts allows, of
    which a chunk's rows take none of this kind."""
    tiles = (replies + 1) * 8 * 8  # of 16 rows, of sequences of up to 128 rows
    for chunk in (40, 512, 2048, 4096, 8192, 60000, 1 << 20):
        splits, blocks, _, _, _, _, total, _ = plan(grids, replies + 1, replies + chunk, 1, 8, 4, most)
        assert splits * blocks >= most // 32 and total <= 1 << 28
        assert blocks <= 128 or splits > (32 << 20) // (tiles * 2080) * 0.95, (chunk, splits, blocks)


def test_parts_of_both_kinds_fit_together(grids) -> None:
    """256 MiB a call, whichever kinds of rows it may have."""
    for n_seq in (1, 2, 4, 33, 64, 300, 1000, 65535):
        for more in (0, 1, 31, 515, 4000, 70000):
            for heads, group, dim in ((8, 4, 128), (1, 1, 8), (8, 8, 256), (4096, 1, 64), (2, 20, 96)):
                for most in (64, 4096, 131072, 1 << 30):
                    n = n_seq + more
                    if n * heads * group > 1 << 28:
                        continue
                    few, _, many, per, floats, slots, total, _ = plan(grids, n_seq, n, 1, heads, group, most, 0, dim)
                    assert total <= 1 << 28 and few >= 1
                    # room for every tile that the call may have, by either way of counting them
                    part = heads * (512 * -(-dim // 32) + 32)
                    assert floats == part * (per * n_seq if per else slots)
                    assert per == 0 or per >= min(8, -(-n * group // 16))
