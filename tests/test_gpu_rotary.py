"""Rotary positions (`HipRotary`, `mxa_rope`) against the formula with 80-bit angles.

Tolerances, e = 2^-24 a float32 half step: the angle's fraction of a turn is exact to 2^-52 |p| f / 2 pi turns
(float64, product and table) and is rounded to float32 once, at most pi e radians; sincospif is within 4 e, the factor
on the values and the two products with their sum add 3 e of |a| + |b|. So a turned value is within
(pi + 7) e m (|a| + |b|) < 11 e m (|a| + |b|), the float64 term, and half a step of its type."""

import math

import numpy as np
import pytest
import torch

from matricxon_amd import synthetic as S
from matricxon_amd.device_packed import DevicePackedLinear
from matricxon_amd.fused_ops import project_shared
from matricxon_amd.rotary import HipRotary
from oracle import dequant as D

pytestmark = pytest.mark.gpu

E32 = 2.0 ** -24
F32, BF16 = torch.float32, torch.bfloat16


def check(rot, x, got, positions, scale=None):
    """got against x turned by positions (T,) or (B, T), x (..., T, heads, dim)."""
    assert got.shape == x.shape and got.dtype == x.dtype and got.is_contiguous()
    d, m = rot.rotary_dim, rot.scale if scale is None else scale
    p = positions.cpu().numpy().astype(np.longdouble)[..., None]
    f = rot.frequencies.numpy().astype(np.longdouble)
    angle = p * f
    cos, sin = (fn(angle).astype(np.float64)[..., None, :] for fn in (np.cos, np.sin))
    v, y = x.double().cpu().numpy(), got.double().cpu().numpy()
    first, second = (slice(0, d, 2), slice(1, d, 2)) if rot.interleaved else (slice(0, d // 2), slice(d // 2, d))
    a, b = v[..., first], v[..., second]
    step = torch.finfo(x.dtype).eps / 2
    size = m * (np.abs(a) + np.abs(b))
    far = (np.abs(angle) * 2.0 ** -52).astype(np.float64)[..., None, :]
    for at, want in ((first, m * (a * cos - b * sin)), (second, m * (a * sin + b * cos))):
        assert (np.abs(y[..., at] - want) <= (11 * E32 + far) * size + step * np.abs(want) + 1e-44).all()
    assert np.array_equal(y[..., d:], v[..., d:])


def rand(g, *shape, dt=F32):
    return torch.randn(*shape, device="cuda", generator=g).to(dt)


# head width, rotary part: whole vectors, halves that are not, pairs alone, one pair of many, wide heads
DIMS = [(128, 128), (64, 32), (80, 32), (96, 96), (2, 2), (6, 4), (20, 20), (66, 2), (256, 64), (192, 190), (1024, 1024)]


@pytest.mark.parametrize("dt", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rot_dim", DIMS)
@pytest.mark.parametrize("t", [1, 5])
def test_formula(gpu, dt, interleaved, dim, rot_dim, t) -> None:
    g = torch.Generator(device="cuda").manual_seed(dim + t)
    rot = HipRotary(dim, rotary_dim=rot_dim, interleaved=interleaved)
    for hq, hk in ((1, 1), (7, 3), (32, 8)):
        q, k = rand(g, t, hq, dim, dt=dt), rand(g, t, hk, dim, dt=dt)
        pos = torch.randint(0, 5000, (t,), device="cuda", generator=g)
        q2, k2 = rot(q, k, pos)
        check(rot, q, q2, pos)
        check(rot, k, k2, pos)
        alone, none = rot(q, None, pos.int())
        assert torch.equal(alone, q2) and none is None


SCALINGS = [None, {"type": "linear", "factor": 4.0}, {"type": "ntk", "factor": 8.0},
            {"type": "yarn", "factor": 16.0, "original_context": 4096},
            {"type": "yarn", "factor": 4.0, "original_context": 8192, "attention_factor": 1.3, "beta_fast": 16.0},
            {"type": "llama3", "factor": 8.0, "original_context": 8192}]


@pytest.mark.parametrize("scaling", SCALINGS, ids=lambda s: "none" if s is None else s["type"])
@pytest.mark.parametrize("start", [0, 1 << 20, (1 << 31) - 40, 1 << 40, -70])
def test_far_positions(gpu, scaling, start) -> None:
    """Positions whose angle in float32 would say nothing, past 32 bits, and negative ones."""
    t, dim = 33, 128
    g = torch.Generator(device="cuda").manual_seed(1)
    rot = HipRotary(dim, base=500000.0, scaling=scaling)
    q, k = rand(g, t, 4, dim), rand(g, t, 2, dim)
    pos = start + torch.arange(t, device="cuda")
    q2, k2 = rot(q, k, pos)
    check(rot, q, q2, pos)
    check(rot, k, k2, pos)


@pytest.mark.parametrize("t", [1, 3, 512, 513, 1023, 1024, 1027, 2051, 9001])
@pytest.mark.parametrize("dt", [F32, BF16], ids=["f32", "bf16"])
def test_columns_of_a_fused_projection(gpu, t, dt) -> None:
    """q and k as columns of one q | k | v buffer; token counts on both sides of the kernel's token tiles."""
    hq, hk, dim = 8, 2, 64
    g = torch.Generator(device="cuda").manual_seed(t)
    qkv = rand(g, t, (hq + 2 * hk) * dim + 3, dt=dt)
    kept = qkv.clone()
    q = qkv[:, 1 : 1 + hq * dim].unflatten(1, (hq, dim))  # a start that is not 16-byte aligned
    k = qkv[:, hq * dim : (hq + hk) * dim].unflatten(1, (hk, dim))
    pos = torch.arange(t, device="cuda").flip(0)
    rot = HipRotary(dim)
    q2, k2 = rot(q, k, pos)
    check(rot, q, q2, pos)
    check(rot, k, k2, pos)
    assert torch.equal(qkv, kept)


@pytest.mark.parametrize("positions_of", ["each", "shared", "one-row", "expanded"])
def test_batches(gpu, positions_of) -> None:
    """(B, T, heads, dim), also as the transpose of (B, heads, T, dim), and positions of every form."""
    b, t, h, dim = 3, 7, 5, 48
    g = torch.Generator(device="cuda").manual_seed(2)
    x = rand(g, b, h, t, dim).transpose(1, 2)
    k = rand(g, b, 2 * t, 2, dim)[:, ::2]
    pos = {"each": torch.randint(0, 900, (b, t), device="cuda", generator=g),
           "shared": torch.randint(0, 900, (t,), device="cuda", generator=g),
           "one-row": torch.randint(0, 900, (1, t), device="cuda", generator=g, dtype=torch.int32),
           "expanded": torch.randint(0, 900, (b, 1), device="cuda", generator=g).expand(b, t)}[positions_of]
    rot = HipRotary(dim, rotary_dim=32, interleaved=True)
    q2, k2 = rot(x, k, pos)
    check(rot, x, q2, pos)
    check(rot, k, k2, pos)


def test_freq_factors(gpu) -> None:
    g = torch.Generator(device="cuda").manual_seed(3)
    ff = 1 + 7 * torch.rand(32)
    rot, plain = HipRotary(64, freq_factors=ff), HipRotary(64)
    assert torch.allclose(rot.frequencies * ff.double(), plain.frequencies, rtol=1e-14, atol=0)
    q, pos = rand(g, 9, 3, 64), torch.arange(9, device="cuda") * 1000
    check(rot, q, rot(q, None, pos)[0], pos)


def test_shift_moves_cached_keys(gpu) -> None:
    """Keys turned for their places and then on by a shift are, to rounding, those of the new places: two turns, each
    within the bound of one, on values of the same size."""
    g = torch.Generator(device="cuda").manual_seed(4)
    rot = HipRotary(64, scaling={"type": "yarn", "factor": 4.0, "original_context": 2048})
    k, pos = rand(g, 50, 4, 64), 500 + torch.arange(50, device="cuda")
    turned = rot(k, None, pos)[0]
    delta = torch.full((50,), -480, device="cuda")
    moved = rot.shift(turned, delta)
    check(rot, turned, moved, delta, scale=1.0)
    want = rot(k, None, pos + delta)[0]
    size = rot.scale * 2 * (k.abs()[..., :32] + k.abs()[..., 32:]).repeat(1, 1, 2)
    assert ((moved - want).abs() <= 3 * 14 * E32 * size).all()


def test_infinities_and_nan_stay_in_their_pair(gpu) -> None:
    g = torch.Generator(device="cuda").manual_seed(5)
    q = rand(g, 2, 2, 64)
    q[1, 0, 3] = float("nan")
    q[0, 1, 40] = float("inf")
    got = HipRotary(64)(q, None, torch.arange(1, 3, device="cuda"))[0]
    bad = ~got.isfinite()
    assert bad[1, 0, 3] and bad[1, 0, 35] and bad[0, 1, 8] and bad[0, 1, 40] and bad.sum() == 4


def test_after_the_shared_projections(gpu) -> None:
    """q | k | v of a packed layer, then the heads' rotary positions, in bfloat16, against the same steps apart."""
    k_in, hq, hk, dim = 512, 4, 2, 64
    owner = torch.nn.Module()
    for i, (name, n) in enumerate((("q", hq * dim), ("k", hk * dim), ("v", hk * dim))):
        owner.add_module(name, DevicePackedLinear(torch.from_numpy(S.packed_weight(D.Q4_K, n, k_in, seed=i)).cuda(),
                                                  k_in, D.Q4_K))
    rot = HipRotary(dim)
    for t in (1, 16):
        x = torch.from_numpy(S.activations(t, k_in, seed=t)).cuda().bfloat16()
        q, k, _ = project_shared(owner, ("q", "k", "v"), x)
        q, k = q.unflatten(-1, (hq, dim)), k.unflatten(-1, (hk, dim))
        pos = 100 + torch.arange(t, device="cuda")
        q2, k2 = rot(q, k, pos)
        check(rot, q, q2, pos)
        check(rot, k, k2, pos)


def test_captured_and_replayed(gpu) -> None:
    g = torch.Generator(device="cuda").manual_seed(6)
    q, k, pos = rand(g, 4, 8, 128, dt=BF16), rand(g, 4, 2, 128, dt=BF16), torch.arange(4, device="cuda")
    rot = HipRotary(128)
    rot(q, k, pos)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = rot(q, k, pos)
    for i in range(4):
        q.copy_(rand(g, 4, 8, 128, dt=BF16))
        pos += 1000 * i
        want = rot(q, k, pos)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_on_another_stream(gpu) -> None:
    g = torch.Generator(device="cuda").manual_seed(7)
    q, pos, rot = rand(g, 64, 16, 128), torch.arange(64, device="cuda"), HipRotary(128)
    want = rot(q, None, pos)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = rot(q, None, pos)[0]
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_refusals(gpu) -> None:
    rot = HipRotary(64)
    q, k, pos = (torch.zeros(3, 4, 64, device="cuda"), torch.zeros(3, 2, 64, device="cuda"),
                 torch.zeros(3, dtype=torch.int64, device="cuda"))
    for a, b, p in ((q.half(), None, pos), (q[0], None, pos), (q[..., :62], None, pos), (q, k.bfloat16(), pos),
                    (q, k[:2], pos), (q, k.cpu(), pos), (q, k[..., :32], pos), (q, k, pos.float()), (q, k, pos.cpu()),
                    (q, k, pos[:2]), (q, k, pos[None]), (q, k, pos[0]), (q[:, :0], None, pos),
                    (q[None], k[None], pos[None].expand(2, 3)), (q.cpu(), None, pos)):
        with pytest.raises(ValueError):
            rot(a, b, p)
    q2, k2 = rot(q[:0], k[:0], pos[:0])  # no tokens
    assert q2.shape == (0, 4, 64) and k2.shape == (0, 2, 64)
    assert math.isclose(HipRotary(64, scaling=SCALINGS[3]).scale, 0.1 * math.log(16) + 1)


def test_more_heads_than_workgroups_side_by_side(gpu) -> None:
    g = torch.Generator(device="cuda").manual_seed(8)
    rot = HipRotary(1022)
    q, k, pos = rand(g, 2, 5000, 1022), rand(g, 2, 3, 1022), torch.tensor([7, 100000], device="cuda")
    q2, k2 = rot(q, k, pos)
    check(rot, q, q2, pos)
    check(rot, k, k2, pos)


def test_the_most_tokens(gpu) -> None:
    n = 1 << 24
    g = torch.Generator(device="cuda").manual_seed(9)
    rot, q, pos = HipRotary(2), rand(g, n, 1, 2, dt=BF16), torch.arange(n, dtype=torch.int32, device="cuda")
    got = rot(q, None, pos)[0]
    for part in (slice(0, 500), slice(n // 2 - 7, n // 2 + 900), slice(n - 500, n)):
        check(rot, q[part], got[part], pos[part])
    assert got.isfinite().all()
    more = torch.zeros(1, 1, 2, device="cuda").expand(n + 1, 1, 2)
    with pytest.raises(ValueError, match="tokens"):
        rot(more, None, torch.zeros(1, dtype=torch.int32, device="cuda").expand(n + 1))


# whole vectors, vectors of four, two and one value, whole heads and parts of them
WIDE = [(128, 128), (64, 64), (80, 32), (80, 20), (96, 24), (48, 44), (66, 2), (256, 64), (512, 512)]


@pytest.mark.parametrize("dt", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rot_dim", WIDE)
@pytest.mark.parametrize("t", [513, 1027, 2051])
def test_many_tokens(gpu, dt, interleaved, dim, rot_dim, t) -> None:
    """Token counts of every share of a workgroup, outputs of less than 4 MB and of more, in pieces of every width."""
    g = torch.Generator(device="cuda").manual_seed(dim + t)
    rot = HipRotary(dim, rotary_dim=rot_dim, interleaved=interleaved)
    q, k = rand(g, t, 5, dim, dt=dt), rand(g, t, 2, dim, dt=dt)
    pos = torch.randint(0, 100000, (t,), device="cuda", generator=g)
    q2, k2 = rot(q, k, pos)
    check(rot, q, q2, pos)
    check(rot, k, k2, pos)


@pytest.mark.parametrize("dt", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rot_dim", [(64, 64), (80, 32), (96, 24)])
@pytest.mark.parametrize("b,t", [(3, 401), (7, 333), (1031, 3), (2, 600)])
def test_workgroups_across_sequences(gpu, dt, interleaved, dim, rot_dim, b, t) -> None:
    """More than 512 tokens in sequences of odd lengths, a workgroup's tokens in two or more of them, with positions of
    their own."""
    g = torch.Generator(device="cuda").manual_seed(b * t)
    rot = HipRotary(dim, rotary_dim=rot_dim, interleaved=interleaved)
    q, k = rand(g, b, 9, t, dim, dt=dt).transpose(1, 2), rand(g, b, t + 1, 3, dim, dt=dt)[:, 1:]
    pos = torch.randint(0, 100000, (b, t), device="cuda", generator=g)
    for p in (pos, pos[:1].int(), pos[0]):
        q2, k2 = rot(q, k, p)
        check(rot, q, q2, p.expand(b, t))
        check(rot, k, k2, p.expand(b, t))


def test_the_library_face(gpu) -> None:
    """`HipGemm.rope` on a table of the caller's: `HipRotary`'s bits, and its refusals."""
    g = torch.Generator(device="cuda").manual_seed(10)
    rot = HipRotary(64, rotary_dim=32, interleaved=True, scaling=SCALINGS[3])
    q, k, pos = rand(g, 9, 4, 64), rand(g, 9, 2, 64), torch.arange(9, device="cuda")
    turns = (rot.frequencies / (2 * math.pi)).cuda()
    for a, b in zip(gpu.rope(q, k, pos, turns, 32, True, rot.scale), rot(q, k, pos)):
        assert torch.equal(a, b)
    for bad in (turns.float(), turns[:15], turns.cpu(), torch.zeros(32, dtype=torch.float64, device="cuda")[::2]):
        with pytest.raises(ValueError, match="turns"):
            gpu.rope(q, k, pos, bad, 32, True, 1.0)
    with pytest.raises(ValueError, match="HIP device"):
        gpu.rope(q.cpu(), None, pos, turns, 32, True, 1.0)
    wide = torch.zeros(33, dtype=torch.float64, device="cuda")
    with pytest.raises(ValueError, match="head_dim"):
        gpu.rope(q, k, pos, wide, 66, True, 1.0)
    for rotary_dim in (0, 3):  # no pair, and half a pair
        with pytest.raises(ValueError, match="rotary_dim"):
            gpu.rope(q, k, pos, turns[: rotary_dim // 2], rotary_dim, True, 1.0)


@pytest.mark.parametrize("dt", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("t,hq,hk,dim", [(300, 60, 60, 128), (1, 9000, 9000, 128), (511, 40, 3, 256)])
def test_few_tokens_of_many_heads(gpu, dt, interleaved, t, hq, hk, dim) -> None:
    """Outputs of more than 4 MB whose heads are split over workgroups."""
    g = torch.Generator(device="cuda").manual_seed(t)
    rot = HipRotary(dim, interleaved=interleaved)
    q, k = rand(g, t, hq, dim, dt=dt), rand(g, t, hk, dim, dt=dt)
    pos = torch.randint(0, 100000, (t,), device="cuda", generator=g)
    q2, k2 = rot(q, k, pos)
    check(rot, q, q2, pos)
    check(rot, k, k2, pos)
