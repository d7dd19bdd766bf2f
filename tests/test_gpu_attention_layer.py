"""The attention half of a decoder layer as a model runs it, on the framework's packed projections: the stream joined and
normed, q | k | v from the norm's blocks, heads normed and turned and cached, attention over the cache, its projection, the
stream again. Each step against its formula on what the step before it returned, with the tolerances of the operators' own
tests, or bit for bit against the same step by itself; then captured and replayed along the sequences."""

import pytest
import torch

from matricxon_amd import synthetic as S
from matricxon_amd.attention import HipPagedCache
from matricxon_amd.device_packed import DevicePackedLinear
from matricxon_amd.fused_ops import HANDOFF, HipFusedOps, project_shared
from matricxon_amd.rotary import HipRotary
from oracle import dequant as D
from tests import test_gpu_add_norm as norms
from tests.test_gpu_paged_cache import check_attention, held, i32, same, starts_of

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
EMBD, HQ, HK, DIM, PAGE, EPS = 1024, 8, 2, 128, 64, 1e-6


@pytest.fixture
def ops(gpu):
    HipFusedOps.configure(True)
    yield HipFusedOps.active()
    HipFusedOps.configure(False)


def near(got, x):
    """Held values lie within half a step of x, or, at a group's ends, within the rounding of its minimum and of 15 scales
    to float16 (2^-11 each); x itself is known to some float32 steps (the order of its squares' sum differs)."""
    x, got = x.double().unflatten(-1, (-1, 32)), got.double().unflatten(-1, (-1, 32))
    lo, size = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True) - x.amin(-1, keepdim=True)
    assert ((got - x).abs() <= 1.01 * (size / 30 + (lo.abs() + size) * 2.0 ** -11) + 2.0 ** -24).all()


class Layer(torch.nn.Module):
    def __init__(self, ops, n_seq, seed):
        super().__init__()
        self.ops = ops
        for i, (name, n, k, t) in enumerate((("q", HQ * DIM, EMBD, D.Q4_K), ("k", HK * DIM, EMBD, D.Q4_K),
                                             ("v", HK * DIM, EMBD, D.Q6_K), ("o", EMBD, HQ * DIM, D.Q4_K))):
            packed = torch.from_numpy(S.packed_weight(t, n, k, seed=seed + i)).cuda()
            self.add_module(name, DevicePackedLinear(packed, k, t, None, BF16))
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.w1, self.w2 = ((1 + norms.rand(g, EMBD, scale=0.1)).to(BF16) for _ in range(2))
        self.qw, self.kw = ((1 + norms.rand(g, DIM, scale=0.1)).to(BF16) for _ in range(2))
        self.rot = HipRotary(DIM, base=500000.0)
        self.cache = HipPagedCache(n_seq * 8, PAGE, HK, DIM)

    def step(self, stream, x, *where):
        a = {"stream": stream, "x": x}
        a["hidden1"], a["normed1"] = self.ops.add_rms_norm(stream, x, self.w1, EPS)
        q, k, v = project_shared(self, ("q", "k", "v"), a["normed1"])
        a["q"], a["k"], a["v"] = (y.unflatten(-1, (-1, DIM)) for y in (q, k, v))
        a["q2"] = self.cache.append(a["q"], a["k"], a["v"], *where, rotary=self.rot, q_weight=self.qw, k_weight=self.kw, eps=EPS)
        a["attn"] = self.cache.attend(a["q2"], *where)
        a["o_out"] = self.o(a["attn"].flatten(-2))
        a["hidden2"], a["normed2"] = self.ops.add_rms_norm(a["hidden1"], a["o_out"], self.w2, EPS)
        return a

    def check(self, a, table, lengths, counts):
        t = sum(counts)
        norms.check((a["hidden1"], a["normed1"]), a["x"], a["stream"], self.w1, EPS)
        HANDOFF.clear()
        for name in ("q", "k", "v"):
            alone = getattr(self, name)(a["normed1"])
            assert torch.equal(a[name].reshape(alone.shape), alone), name
        where = (table, i32(lengths), starts_of(counts))
        places = torch.cat([torch.arange(n - c, n, device="cuda") for n, c in zip(lengths, counts)])
        q, k = (a[name][:t] for name in ("q", "k"))
        q2, k2 = self.rot(q, k, places, q_weight=self.qw, k_weight=self.kw, eps=EPS)
        assert same(a["q2"][:t], q2) and (a["q2"][t:] == 0).all()
        k2, v2 = self.cache.read(t, *where, dtype=F32)
        assert same(v2, held(a["v"][:t]))
        _, turned = self.rot(q.float(), k.float(), places, q_weight=self.qw.float(), k_weight=self.kw.float(), eps=EPS)
        near(k2, turned)
        check_attention(self.cache, a["q2"][:t], a["attn"][:t].contiguous(), table, lengths, counts)
        assert (a["attn"][t:] == 0).all()
        assert torch.equal(a["o_out"], self.o(a["attn"].flatten(-2)))
        norms.check((a["hidden2"], a["normed2"]), a["o_out"], a["hidden1"], self.w2, EPS)


def test_prompts_replies_and_a_graph(gpu, ops) -> None:
    layers = [Layer(ops, 3, seed) for seed in (500, 600)]
    g = torch.Generator(device="cuda").manual_seed(1)
    table = torch.randperm(24, device="cuda", generator=g).view(3, 8).int()
    lengths = [0, 0, 0]
    for counts, rows in (([70, 1, 33], 104), ([100, 0, 1], 105), ([1, 1, 1], 3)):  # one row of no sequence
        lengths = [n + c for n, c in zip(lengths, counts)]
        where = (table, i32(lengths), starts_of(counts))
        s, y = norms.rand(g, rows, EMBD, dt=BF16, scale=2.0), norms.rand(g, rows, EMBD, dt=BF16)
        for layer in layers:
            a = layer.step(s, y, *where)
            layer.check(a, table, lengths, counts)
            s, y = a["hidden2"], a["normed2"]
    counts = [1, 1, 1]
    length, starts = i32(lengths), starts_of(counts)
    s, y = norms.rand(g, 3, EMBD, dt=BF16, scale=2.0), norms.rand(g, 3, EMBD, dt=BF16)

    def both():
        a = layers[0].step(s, y, table, length, starts)
        return a, layers[1].step(a["hidden2"], a["normed2"], table, length, starts)

    both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    for _ in range(5):
        lengths = [n + 1 for n in lengths]
        length += 1
        s.copy_(norms.rand(g, 3, EMBD, dt=BF16, scale=2.0))
        graph.replay()
        got = [{k: v.clone() for k, v in a.items()} for a in out]
        for layer, a in zip(layers, got):
            layer.check(a, table, lengths, counts)
        for a, b in zip(got, both()):
            assert all(same(a[k], b[k]) for k in a)
