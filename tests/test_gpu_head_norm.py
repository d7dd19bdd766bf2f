"""Head norms with rotary positions in one pass (`HipRotary` with weights, `mxa_norm_rope`) against 64-bit arithmetic.

Tolerances, e = 2^-24 a float32 half step: a head's squares are added up in chains of at most 2 * 8 or 16 values and six
steps across lanes (22 e, and one for each square), the mean, the addition of eps, the root and the reciprocal are
within 6 e, of which the root halves all before it: the factor is within (23 + 6) e, the two products add 2 e, so a normed
value is within 31 e of itself. The rotation adds 11 e of |a| + |b| (test_gpu_rotary.py), which the pair's own errors
meet: (31 + 11) e m (|a| + |b|), the float64 term of the angle, and half a step of the output's type."""

import math

import numpy as np
import pytest
import torch

from matricxon_amd.rotary import HipRotary

pytestmark = pytest.mark.gpu

E32 = 2.0 ** -24
F32, BF16 = torch.float32, torch.bfloat16


def check(rot, x, got, positions, weight, eps=1e-6):
    """got against x (..., T, heads, dim) normed by weight (or None) and turned by positions (T,) or (B, T)."""
    assert got.shape == x.shape and got.dtype == x.dtype and got.is_contiguous()
    d, m = rot.rotary_dim, rot.scale
    v, y = x.double().cpu().numpy(), got.double().cpu().numpy()
    if weight is not None:
        v = v / np.sqrt((v * v).mean(-1, keepdims=True) + eps) * weight.double().cpu().numpy()
    angle = positions.cpu().numpy().astype(np.longdouble)[..., None] * rot.frequencies.numpy().astype(np.longdouble)
    cos, sin = (fn(angle).astype(np.float64)[..., None, :] for fn in (np.cos, np.sin))
    first, second = (slice(0, d, 2), slice(1, d, 2)) if rot.interleaved else (slice(0, d // 2), slice(d // 2, d))
    a, b = v[..., first], v[..., second]
    step = torch.finfo(x.dtype).eps / 2
    size = m * (np.abs(a) + np.abs(b))
    far = (np.abs(angle) * 2.0 ** -52).astype(np.float64)[..., None, :]
    for at, want in ((first, m * (a * cos - b * sin)), (second, m * (a * sin + b * cos))):
        assert (np.abs(y[..., at] - want) <= (42 * E32 + far) * size + step * np.abs(want) + 1e-38).all()
    rest = v[..., d:]
    assert (np.abs(y[..., d:] - rest) <= (31 * E32 + step) * np.abs(rest) + 1e-38).all()


def rand(g, *shape, dt=F32):
    return torch.randn(*shape, device="cuda", generator=g).to(dt)


# head width, rotary part: whole vectors, halves that are not, pairs alone, one pair of many, wide heads
DIMS = [(128, 128), (64, 32), (80, 32), (80, 50), (96, 96), (2, 2), (6, 4), (20, 20), (66, 2), (256, 64), (192, 190),
        (1024, 1024)]


@pytest.mark.parametrize("dt", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rot_dim", DIMS)
@pytest.mark.parametrize("t", [1, 5])
def test_formula(gpu, dt, interleaved, dim, rot_dim, t) -> None:
    g = torch.Generator(device="cuda").manual_seed(dim + t)
    rot = HipRotary(dim, rotary_dim=rot_dim, interleaved=interleaved)
    for hq, hk in ((1, 1), (7, 3), (32, 8)):
        q, k = 3 * rand(g, t, hq, dim, dt=dt), 0.01 * rand(g, t, hk, dim, dt=dt)
        qw, kw = (1 + 0.3 * rand(g, dim)).to(dt), (1 + 0.3 * rand(g, dim)).to(dt)
        pos = torch.randint(0, 5000, (t,), device="cuda", generator=g)
        q2, k2 = rot(q, k, pos, q_weight=qw, k_weight=kw)
        check(rot, q, q2, pos, qw)
        check(rot, k, k2, pos, kw)
        alone, none = rot(q, None, pos.int(), q_weight=qw)
        assert torch.equal(alone, q2) and none is None


@pytest.mark.parametrize("t", [1, 3, 512, 513, 1023, 1025, 2051, 4099, 9001])
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
    rot = HipRotary(dim, scaling={"type": "yarn", "factor": 16.0, "original_context": 4096})
    qw = (1 + 0.3 * rand(g, 2 * dim)).to(dt)[::2]  # a weight that is not contiguous
    q2, k2 = rot(q, k, pos, q_weight=qw, k_weight=qw.flip(0), eps=1e-5)
    check(rot, q, q2, pos, qw, 1e-5)
    check(rot, k, k2, pos, qw.flip(0), 1e-5)
    assert torch.equal(qkv, kept)


@pytest.mark.parametrize("which", ["q", "k"])
def test_one_side_normed(gpu, which) -> None:
    """The side without a weight is what HipRotary gives without norms, bit for bit."""
    g = torch.Generator(device="cuda").manual_seed(2)
    rot = HipRotary(128)
    q, k, pos = rand(g, 9, 8, 128, dt=BF16), rand(g, 9, 2, 128, dt=BF16), torch.arange(9, device="cuda")
    w = (1 + 0.3 * rand(g, 128)).to(BF16)
    q2, k2 = rot(q, k, pos, **{which + "_weight": w})
    plain_q, plain_k = rot(q, k, pos)
    check(rot, q, q2, pos, w if which == "q" else None)
    check(rot, k, k2, pos, w if which == "k" else None)
    assert torch.equal(k2, plain_k) if which == "q" else torch.equal(q2, plain_q)


@pytest.mark.parametrize("positions_of", ["each", "shared", "expanded"])
def test_batches(gpu, positions_of) -> None:
    """(B, T, heads, dim) as the transpose of (B, heads, T, dim), and positions of every form."""
    b, t, dim = 3, 7, 64
    g = torch.Generator(device="cuda").manual_seed(4)
    q, k = rand(g, b, 6, t, dim).transpose(1, 2), rand(g, b, 2, t, dim).transpose(1, 2)
    w = 1 + 0.3 * rand(g, dim)
    pos = {"each": torch.randint(-50, 5000, (b, t), device="cuda", generator=g),
           "shared": torch.arange(t, device="cuda"),
           "expanded": torch.arange(t, device="cuda")[None].expand(b, t)}[positions_of]
    rot = HipRotary(dim, interleaved=True)
    q2, k2 = rot(q, k, pos, q_weight=w, k_weight=w)
    full = pos if pos.dim() == 2 else pos[None].expand(b, t)
    check(rot, q, q2, full, w)
    check(rot, k, k2, full, w)


def test_rows_of_zeros_and_large_values(gpu) -> None:
    """A head of zeros stays zeros; squares that pass float32's range give what float32 gives, and touch no other row."""
    rot = HipRotary(64)
    q = torch.zeros(4, 2, 64, device="cuda")
    q[1], q[2, 0], q[3, 1, 5] = 1.0, 1e30, math.nan
    pos, w = torch.arange(4, device="cuda"), torch.ones(64, device="cuda")
    got, _ = rot(q, None, pos, q_weight=w)
    assert (got[0] == 0).all() and (got[2] == 0).all()  # 1 / sqrt(inf) is 0
    check(rot, q[1:2], got[1:2].contiguous(), pos[1:2], w)
    assert got[3, 1].isnan().all() and (got[3, 0] == 0).all()


def test_streams_and_graphs(gpu) -> None:
    g = torch.Generator(device="cuda").manual_seed(5)
    rot = HipRotary(128)
    q, k = rand(g, 5, 8, 128, dt=BF16), rand(g, 5, 2, 128, dt=BF16)
    w, pos = (1 + 0.3 * rand(g, 128)).to(BF16), torch.arange(5, device="cuda")
    want = rot(q, k, pos, q_weight=w, k_weight=w)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = rot(q, k, pos, q_weight=w, k_weight=w)
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = rot(q, k, pos, q_weight=w, k_weight=w)
    for _ in range(3):
        pos += 100
        q.mul_(0.5)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, rot(q, k, pos, q_weight=w, k_weight=w)))


def test_refusals(gpu) -> None:
    rot = HipRotary(64)
    q, k, pos = torch.zeros(3, 4, 64, device="cuda"), torch.zeros(3, 2, 64, device="cuda"), torch.arange(3, device="cuda")
    w = torch.ones(64, device="cuda")
    for bad, match in ((dict(q_weight=w[:32]), "q_weight"), (dict(q_weight=w.bfloat16()), "q_weight"),
                       (dict(k_weight=w.cpu()), "k_weight"), (dict(k_weight=w[None]), "k_weight")):
        with pytest.raises(ValueError, match=match):
            rot(q, k, pos, **bad)
    with pytest.raises(ValueError, match="needs k"):
        rot(q, None, pos, k_weight=w)
    empty, _ = rot(q[:0], None, pos[:0], q_weight=w)
    assert empty.shape == (0, 4, 64)


@pytest.mark.parametrize("t", [1, 2, 512])
@pytest.mark.parametrize("hq, hk, dim, dt, interleaved",
                         [(64, 8, 128, F32, True), (64, 8, 256, BF16, True), (64, 8, 256, F32, False), (32, 8, 256, F32, True),
                          (8, 64, 128, F32, True), (33, 65, 64, BF16, False)])
def test_heads_that_share_out_unevenly(gpu, hq, hk, dim, dt, interleaved, t) -> None:
    """Heads of q and k whose shares are rounded up (test_host_grids.py), k the last of its buffer."""
    g = torch.Generator(device="cuda").manual_seed(hq + t)
    rot = HipRotary(dim, interleaved=interleaved)
    q, k = rand(g, t, hq, dim, dt=dt), rand(g, t, hk, dim, dt=dt)
    qw, kw = (1 + 0.3 * rand(g, dim)).to(dt), (1 + 0.3 * rand(g, dim)).to(dt)
    pos = torch.randint(0, 5000, (t,), device="cuda", generator=g)
    q2, k2 = rot(q, k, pos, q_weight=qw, k_weight=kw)
    check(rot, q, q2, pos, qw)
    check(rot, k, k2, pos, kw)


def test_more_heads_than_shares(gpu) -> None:
    """q alone, of as many heads as are shared out over 4096 workgroups a token by ten."""
    g = torch.Generator(device="cuda").manual_seed(6)
    rot = HipRotary(256, interleaved=True)
    q, w, pos = rand(g, 1, 40000, 256, dt=BF16), (1 + 0.3 * rand(g, 256)).to(BF16), torch.tensor([77], device="cuda")
    check(rot, q, rot(q, None, pos, q_weight=w)[0], pos, w)
