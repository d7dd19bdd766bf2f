"""The residual stream between two blocks (`HipFusedOps.add_rms_norm`) against its formula in 64 bits.

Tolerances, e = 2^-24 a float32 half step: a mean of squares is a sum of non-negative terms over at most 32 in a
thread, 6 levels of a wave and 16 waves, so its relative error is under 54 e, half of that after the square root; with
the division, the root's own rounding and the products that follow, a normed value is within 40 e of its own size.
hidden adds r + s g u with one rounding, so it is within 40 e (|r| + |s g u|) and, stored, half a step of its type.
normed is checked against the norm of the hidden that the call returned: 40 e and half a step of its type."""

import pytest
import torch

from matricxon_amd import synthetic as S
from matricxon_amd.device_packed import DevicePackedLinear
from matricxon_amd.fused_ops import HANDOFF, HipFusedOps, project_shared
from matricxon_amd.gemm import q8k_views
from oracle import dequant as D

pytestmark = pytest.mark.gpu

E32 = 2.0 ** -24
F32, BF16 = torch.float32, torch.bfloat16
EPS = 1e-5


@pytest.fixture
def ops(gpu):
    HipFusedOps.configure(True)
    yield HipFusedOps.active()
    HipFusedOps.configure(False)


def half_step(dt):
    return torch.finfo(dt).eps / 2


def rms64(v, w, eps):
    return v / torch.sqrt((v * v).mean(-1, keepdim=True) + eps) * w.double()


def rand(g, *shape, dt=F32, scale=1.0):
    return (scale * torch.randn(*shape, device="cuda", generator=g)).to(dt)


def check(res, x, r, w, eps, post=None, post_eps=None, gate=None, scale=1.0):
    assert res is not None
    hidden, normed = res
    assert hidden.dtype == r.dtype and normed.dtype == x.dtype
    assert hidden.shape == normed.shape == x.shape and hidden.is_contiguous() and normed.is_contiguous()
    u = x.double()
    if post is not None:
        u = rms64(u, post, eps if post_eps is None else post_eps)
    if gate is not None:
        u = u * gate.double()
    u = scale * u
    want = r.double() + u
    bound = 40 * E32 * (r.double().abs() + u.abs()) + half_step(r.dtype) * want.abs() + 1e-44
    assert ((hidden.double() - want).abs() <= bound).all()
    want = rms64(hidden.double(), w, eps)
    bound = (40 * E32 + half_step(x.dtype)) * want.abs() + 1e-44
    assert ((normed.double() - want).abs() <= bound).all()
    return hidden, normed


def assert_blocks(gpu, ws, normed):
    k = normed.shape[-1]
    out = normed.reshape(-1, k)
    for got, want in zip(q8k_views(ws, out.shape[0], k), gpu.quantize_q8_k(out)):
        assert torch.equal(got, want)


DTYPES = [(F32, F32), (BF16, BF16), (BF16, F32)]
# one value to the longest row; whole blocks, whole vectors and neither; one wave, several and four vectors a thread
SHAPES = [(1, 1), (3, 7), (2, 8), (5, 64), (1, 256), (9, 512), (4, 513), (6, 1155), (1, 4096), (3, 4096), (2, 8191),
          (2, 8192), (2, 8200), (1, 16384), (2, 20000), (1, 32768), (517, 256), (600, 1024), (515, 1280), (520, 2051)]


@pytest.mark.parametrize("dtypes", DTYPES, ids=["f32", "bf16", "bf16-f32"])
@pytest.mark.parametrize("m,k", SHAPES)
@pytest.mark.parametrize("post", [False, True])
def test_formula(gpu, ops, m, k, dtypes, post) -> None:
    dt, rt = dtypes
    g = torch.Generator(device="cuda").manual_seed(m * 31 + k)
    x, r = rand(g, m, k, dt=dt, scale=1.5), rand(g, m, k, dt=rt, scale=4)
    w, wp = 1 + rand(g, k, dt=dt, scale=0.2), 1 + rand(g, k, dt=dt, scale=0.2)
    if m > 2:
        x[1], r[1] = 0, 0  # an empty row: h = 0, n = 0
    _, normed = check(ops.add_rms_norm(r, x, w, EPS, post_weight=wp if post else None), x, r, w, EPS,
                      wp if post else None)
    ws = HANDOFF.claim(normed)
    if k % 256 == 0:
        assert_blocks(gpu, ws, normed)
    else:
        assert ws is None


@pytest.mark.parametrize("dtypes", DTYPES, ids=["f32", "bf16", "bf16-f32"])
@pytest.mark.parametrize("k", [1, 300, 2048])
@pytest.mark.parametrize("gate_of", ["one", "scalar", "channel", "row", "token", "full", "strided"])
def test_gates_and_scale(gpu, ops, dtypes, k, gate_of) -> None:
    dt, rt = dtypes
    m = 6
    g = torch.Generator(device="cuda").manual_seed(k)
    x, r, w, wp = rand(g, m, k, dt=dt), rand(g, m, k, dt=rt), 1 + rand(g, k, dt=dt, scale=0.2), 1 + rand(g, k, dt=dt)
    gate = {"one": lambda: rand(g, 1, dt=dt), "scalar": lambda: rand(g, 1, dt=dt).reshape(()),
            "channel": lambda: rand(g, k, dt=dt), "row": lambda: rand(g, 1, k, dt=dt),
            "token": lambda: rand(g, m, 1, dt=dt), "full": lambda: rand(g, m, k, dt=dt),
            "strided": lambda: rand(g, m, 2 * k, dt=dt)[:, ::2]}[gate_of]()
    res = ops.add_rms_norm(r, x, w, 1e-6, post_weight=wp, post_eps=1e-3, gate=gate, scale=-0.22)
    check(res, x, r, w, 1e-6, wp, 1e-3, gate, -0.22)


def test_broadcast_over_a_batch(gpu, ops) -> None:
    """(B, S, K) with a gate for each sequence, and outputs of that shape."""
    b, s, k = 3, 5, 512
    g = torch.Generator(device="cuda").manual_seed(0)
    x, r, w = rand(g, b, s, k, dt=BF16), rand(g, b, s, k), 1 + rand(g, k, dt=BF16, scale=0.1)
    for gate in (rand(g, b, 1, k, dt=BF16), rand(g, s, 1, dt=BF16), rand(g, b, 1, 1, dt=BF16)):
        check(ops.add_rms_norm(r, x, w, EPS, gate=gate), x, r, w, EPS, gate=gate)
    one = rand(g, k, dt=BF16)
    check(ops.add_rms_norm(one.clone(), one, w, EPS), one, one, w, EPS)  # no leading dimension


def test_strided_rows(gpu, ops) -> None:
    """Columns of wider buffers, rows of odd strides and starts, one row for all, and columns that are not adjacent."""
    m, k = 7, 1024
    g = torch.Generator(device="cuda").manual_seed(1)
    w = 1 + rand(g, k, dt=BF16, scale=0.1)
    wide, narrow = rand(g, m, 3 * k + 5, dt=BF16), rand(g, m, k + 3)
    for x, r in ((wide[:, k + 1 : 2 * k + 1], narrow[:, 3:]), (wide[:1, 7 : k + 7].expand(m, k), narrow[:, :k]),
                 (rand(g, k, m, dt=BF16).t(), rand(g, m, 2 * k, dt=BF16)[:, 1::2])):
        _, normed = check(ops.add_rms_norm(r, x, w, EPS), x, r, w, EPS)
        assert_blocks(gpu, HANDOFF.claim(normed), normed)


def test_infinities_and_nan_stay_in_their_row(gpu, ops) -> None:
    m, k = 4, 768
    g = torch.Generator(device="cuda").manual_seed(2)
    x, r, w = rand(g, m, k), rand(g, m, k), 1 + rand(g, k, scale=0.1)
    x[1, 5], x[2, 700] = float("nan"), float("inf")
    hidden, normed = ops.add_rms_norm(r, x, w, EPS)
    for row in (0, 3):
        h, n = ops.add_rms_norm(r[row], x[row], w, EPS)
        assert torch.equal(hidden[row], h) and torch.equal(normed[row], n)
    assert normed[1].isnan().all() and hidden[1].isnan().sum() == 1
    assert hidden[2, 700] == float("inf") and normed[2, 700].isnan() and (normed[2].nan_to_num(0) == 0).all()


def test_without_blocks(gpu, ops) -> None:
    """q8k=False: the same values, and nothing handed on."""
    g = torch.Generator(device="cuda").manual_seed(3)
    x, r, w = rand(g, 3, 512), rand(g, 3, 512), rand(g, 512)
    want = ops.add_rms_norm(r, x, w, EPS)
    HANDOFF.clear()
    got = ops.add_rms_norm(r, x, w, EPS, q8k=False)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and HANDOFF.claim(got[1]) is None


def test_inputs_are_left_as_they_were(gpu, ops) -> None:
    g = torch.Generator(device="cuda").manual_seed(4)
    x, r, w = rand(g, 5, 300), rand(g, 5, 300), rand(g, 300)
    kept = [t.clone() for t in (x, r, w)]
    first = ops.add_rms_norm(r, x, w, EPS, gate=w, post_weight=w)
    again = ops.add_rms_norm(r, x, w, EPS, gate=w, post_weight=w)
    assert all(torch.equal(a, b) for a, b in zip((x, r, w), kept))
    assert all(torch.equal(a, b) for a, b in zip(first, again))


@pytest.mark.parametrize("m", [1, 16])
def test_hands_on_to_the_projections(gpu, ops, m) -> None:
    """The stream between blocks as a layer runs it: the projections after it run on its blocks, bit for bit as they
    run on the values."""
    k = 1024
    owner = torch.nn.Module()
    for i, n in enumerate((256, 512)):
        packed = torch.from_numpy(S.packed_weight(D.Q4_K, n, k, seed=i)).cuda()
        setattr(owner, f"p{i}", DevicePackedLinear(packed, k, D.Q4_K))
    g = torch.Generator(device="cuda").manual_seed(m)
    x, r, w = rand(g, m, k, dt=BF16), rand(g, m, k, dt=BF16, scale=3), 1 + rand(g, k, dt=BF16, scale=0.1)
    hidden, normed = ops.add_rms_norm(r, x, w, EPS, post_weight=w, scale=0.5)
    assert HANDOFF.claim(normed) is not None
    got = project_shared(owner, ("p0", "p1"), normed)
    HANDOFF.clear()
    for a, b in zip(got, project_shared(owner, ("p0", "p1"), normed)):
        assert torch.equal(a, b)


def test_captured_and_replayed(gpu, ops) -> None:
    """A captured call on inputs that change between replays, with eager calls of its own kind between them."""
    m, k = 4, 2048
    g = torch.Generator(device="cuda").manual_seed(5)
    x, r, w = rand(g, m, k, dt=BF16), rand(g, m, k), 1 + rand(g, k, dt=BF16, scale=0.1)
    ops.add_rms_norm(r, x, w, EPS, post_weight=w)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        hidden, normed = ops.add_rms_norm(r, x, w, EPS, post_weight=w)
    for _ in range(4):
        x.copy_(rand(g, m, k, dt=BF16))
        r.copy_(rand(g, m, k))
        want = ops.add_rms_norm(r, x, w, EPS, post_weight=w)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(hidden, want[0]) and torch.equal(normed, want[1])


def test_on_another_stream(gpu, ops) -> None:
    g = torch.Generator(device="cuda").manual_seed(6)
    x, r, w = rand(g, 64, 4096, dt=BF16), rand(g, 64, 4096), rand(g, 4096, dt=BF16)
    want = ops.add_rms_norm(r, x, w, EPS)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.add_rms_norm(r, x, w, EPS)
        assert HANDOFF.claim(got[1]) is not None
    assert HANDOFF.claim(got[1]) is None  # not on this stream
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_refusals(gpu, ops) -> None:
    x = torch.zeros(2, 512, device="cuda")
    w = torch.zeros(512, device="cuda")
    refused = [
        (x, x.cpu(), w, {}), (x.cpu(), x, w, {}), (x.half(), x.half(), w.half(), {}), (x.bfloat16(), x, w, {}),
        (x, x.bfloat16(), w, {}), (x[:1], x, w, {}), (x, x, w[:1], {}), (x, x, w[None], {}),
        (x, x, w, {"post_weight": w[:5]}), (x, x, w, {"post_weight": w.bfloat16()}), (x, x, w, {"gate": w[:5]}),
        (x, x, w, {"gate": torch.zeros(3, 2, 512, device="cuda")}), (x, x, w, {"gate": w.cpu()}),
        (x[:0], x[:0], w, {}), (x[:, :0], x[:, :0], w[:0], {}),
    ]
    for r, y, weight, more in refused:
        assert ops.add_rms_norm(r, y, weight, EPS, **more) is None
    long = torch.zeros(1, 32769, device="cuda")
    assert ops.add_rms_norm(long, long, long[0], EPS) is None
    with pytest.raises(ValueError, match="NORM_MAX|32768"):
        gpu.add_rms_norm_q8k(long, long, long[0], EPS)
    with pytest.raises(ValueError, match="weight must be"):
        gpu.add_rms_norm_q8k(x, x, w[:1], EPS)
    with pytest.raises(ValueError, match="gate must be"):
        gpu.add_rms_norm_q8k(x, x, w, EPS, gate=w.bfloat16())
    hidden, out, _ = gpu.add_rms_norm_q8k(x[:0], x[:0], w, EPS)  # no rows: nothing to launch
    assert hidden.shape == out.shape == (0, 512)


def test_the_most_rows(gpu, ops) -> None:
    m = 1 << 24
    g = torch.Generator(device="cuda").manual_seed(7)
    x, r, w = rand(g, m, 1, dt=BF16), rand(g, m, 1, dt=BF16), 1 + rand(g, 1, dt=BF16)
    check(ops.add_rms_norm(r, x, w, EPS), x, r, w, EPS)
    more = torch.zeros(1, 1, device="cuda").expand(m + 1, 1)
    assert ops.add_rms_norm(more, more, more[0], EPS) is None
    with pytest.raises(ValueError, match="rows"):
        gpu.add_rms_norm_q8k(more, more, more[0], EPS)


def test_in_inference_mode(gpu, ops) -> None:
    """Tensors without a version hand no blocks on: the projections behind quantize the values they are given."""
    k = 512
    owner = torch.nn.Module()
    owner.p = DevicePackedLinear(torch.from_numpy(S.packed_weight(D.Q4_K, 256, k, seed=3)).cuda(), k, D.Q4_K)
    g = torch.Generator(device="cuda").manual_seed(8)
    x, r, w = rand(g, 4, k, dt=BF16), rand(g, 4, k, dt=BF16), 1 + rand(g, k, dt=BF16, scale=0.1)
    want = ops.add_rms_norm(r, x, w, EPS)
    y = project_shared(owner, ("p",), want[1])[0]
    with torch.inference_mode():
        got = ops.add_rms_norm(r, x, w, EPS)
        assert HANDOFF.claim(got[1]) is None
        assert torch.equal(project_shared(owner, ("p",), got[1])[0], y)
        got[1].mul_(2)
        twice = project_shared(owner, ("p",), got[1])[0]
    assert torch.equal(got[0], want[0]) and torch.equal(twice, project_shared(owner, ("p",), 2 * want[1])[0])


def test_more_values_than_a_grid_holds(gpu, ops) -> None:
    """Rows whose count alone is within the limit, their threads together not: refused before anything is allocated."""
    one = torch.zeros(1, 32768, dtype=BF16, device="cuda")
    for m, k in ((1 << 24, 4096), (1 << 23, 8192), ((1 << 20) + 1, 32768)):
        x, w = one[:, :k].expand(m, k), one[0, :k]
        assert ops.add_rms_norm(x, x, w, EPS) is None
        with pytest.raises(ValueError, match="values"):
            gpu.add_rms_norm_q8k(x, x, w, EPS)


# outputs of 1 MB in many rows and of 5 to 180 MB in few and many: stored past the caches or not, one, two and four
# vectors a thread, whole and not
@pytest.mark.parametrize("dtypes", DTYPES, ids=["f32", "bf16", "bf16-f32"])
@pytest.mark.parametrize("m,k", [(1030, 256), (300, 8192), (400, 3079), (100, 32768), (65, 32765), (5000, 513),
                                 (5003, 4096), (2500, 4099), (600, 20000), (12000, 4096), (90000, 500)])
def test_every_size_of_outputs(gpu, ops, m, k, dtypes) -> None:
    dt, rt = dtypes
    g = torch.Generator(device="cuda").manual_seed(m + k)
    x, r = rand(g, m, k, dt=dt, scale=1.5), rand(g, m, k, dt=rt, scale=4)
    w, wp = 1 + rand(g, k, dt=dt, scale=0.2), 1 + rand(g, k, dt=dt, scale=0.2)
    _, normed = check(ops.add_rms_norm(r, x, w, EPS, post_weight=wp), x, r, w, EPS, wp)
    if k % 256 == 0:
        assert_blocks(gpu, HANDOFF.claim(normed), normed)
