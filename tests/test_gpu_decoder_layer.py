"""`add_rms_norm`, `HipRotary` and `forward_logits` run together as a decoder of expert layers runs them, on the
framework's packed projections: the stream joined and normed, q | k | v from the norm's blocks, rotary positions, keys
and values into a cache, attention (torch, float32), its projection, the stream again, the router (torch) and the
experts. Each step against its formula on what the step before it returned, with the tolerances of the operators' own
tests, or bit for bit against the same step by itself; then the whole layer captured and replayed along a sequence."""

import pytest
import torch
import torch.nn.functional as F

from matricxon_amd import synthetic as S
from matricxon_amd.device_packed import DevicePackedLinear
from matricxon_amd.fused_ops import HANDOFF, HipFusedOps, project_shared
from matricxon_amd.rotary import HipRotary
from oracle import dequant as D
from tests import test_gpu_add_norm as norms
from tests import test_gpu_rotary as rotary
from tests.test_gpu_moe import build_experts, reference_forward
from tests.test_gpu_moe_layer import check_routing

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
EMBD, FFN, HQ, HK, DIM, EXPERTS, TOP_K, ROOM = 1024, 512, 8, 2, 128, 8, 2, 64
EPS = 1e-6


@pytest.fixture
def ops(gpu):
    HipFusedOps.configure(True)
    yield HipFusedOps.active()
    HipFusedOps.configure(False)


class Layer(torch.nn.Module):
    """One decoder layer; `step` returns the values between its steps by name."""

    def __init__(self, ops, dtype, seed):
        super().__init__()
        self.ops, self.dtype = ops, dtype
        for i, (name, n, k, t) in enumerate((("q", HQ * DIM, EMBD, D.Q4_K), ("k", HK * DIM, EMBD, D.Q4_K),
                                             ("v", HK * DIM, EMBD, D.Q6_K), ("o", EMBD, HQ * DIM, D.Q4_K))):
            packed = torch.from_numpy(S.packed_weight(t, n, k, seed=seed + i)).cuda()
            self.add_module(name, DevicePackedLinear(packed, k, t, None, dtype))
        self.experts, self.per_expert = build_experts((D.Q4_K, D.Q4_K, D.Q6_K), EXPERTS, EMBD, FFN, dtype, seed)
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.w1, self.w2, self.post = ((1 + norms.rand(g, EMBD, scale=0.1)).to(dtype) for _ in range(3))
        self.router = norms.rand(g, EXPERTS, EMBD, scale=EMBD ** -0.5)
        self.rot = HipRotary(DIM, base=500000.0)
        self.keys = torch.zeros(ROOM, HK, DIM, dtype=dtype, device="cuda")
        self.values = torch.zeros_like(self.keys)

    def attention(self, q, positions):
        heads = HQ // HK
        k, v = (c.float().repeat_interleave(heads, 1).transpose(0, 1).contiguous() for c in (self.keys, self.values))
        kt = k.transpose(1, 2).contiguous()
        s = torch.matmul(q.float().transpose(0, 1).contiguous(), kt) * DIM ** -0.5
        later = torch.arange(ROOM, device="cuda")[None, :] > positions[:, None]
        s = s.masked_fill(later[None], float("-inf"))
        return torch.matmul(s.softmax(-1), v).transpose(0, 1).reshape(len(q), HQ * DIM).to(self.dtype)

    def step(self, stream, x, positions, real):
        a = {"stream": stream, "x": x}
        a["hidden1"], a["normed1"] = self.ops.add_rms_norm(stream, x, self.w1, EPS)
        q, k, a["v"] = project_shared(self, ("q", "k", "v"), a["normed1"])
        a["q"], a["k"] = q.unflatten(-1, (HQ, DIM)), k.unflatten(-1, (HK, DIM))
        a["q2"], a["k2"] = self.rot(a["q"], a["k"], positions)
        self.keys.index_copy_(0, positions, a["k2"])
        self.values.index_copy_(0, positions, a["v"].unflatten(-1, (HK, DIM)))
        a["attn"] = self.attention(a["q2"], positions)
        a["o_out"] = self.o(a["attn"])
        a["hidden2"], a["normed2"] = self.ops.add_rms_norm(a["hidden1"], a["o_out"], self.w2, EPS,
                                                           post_weight=self.post, scale=0.5)
        logits = F.linear(a["normed2"].float(), self.router)
        a["logits"] = logits.masked_fill(~real[:, None], float("-inf"))  # padding goes to no expert
        a["out"], a["ids"], a["wts"] = self.experts.forward_logits(a["normed2"], a["logits"], TOP_K)
        return a

    def check(self, a, positions):
        norms.check((a["hidden1"], a["normed1"]), a["x"], a["stream"], self.w1, EPS)
        HANDOFF.clear()
        for name in ("q", "k", "v"):
            alone = getattr(self, name)(a["normed1"])
            assert torch.equal(a[name].reshape(alone.shape), alone), name
        rotary.check(self.rot, a["q"], a["q2"], positions)
        rotary.check(self.rot, a["k"], a["k2"], positions)
        norms.check((a["hidden2"], a["normed2"]), a["o_out"], a["hidden1"], self.w2, EPS, post=self.post, scale=0.5)
        check_routing(a["logits"], TOP_K, True, 1.0, a["ids"], a["wts"])
        want, live = torch.zeros_like(a["out"]), (a["ids"] >= 0).all(1)
        want[live] = reference_forward(a["normed2"][live], a["wts"][live], a["ids"][live].long(), self.per_expert,
                                       F.silu)
        assert torch.equal(a["out"], want)


def inputs(t, dtype, stream, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    real = torch.ones(t, dtype=torch.bool, device="cuda")
    if t > 2:
        real[t - 1] = False
    return norms.rand(g, t, EMBD, dt=stream, scale=2.0), norms.rand(g, t, EMBD, dt=dtype), real


@pytest.mark.parametrize("dtype,stream", [(F32, F32), (BF16, BF16), (BF16, F32)], ids=["f32", "bf16", "bf16-f32"])
@pytest.mark.parametrize("t", [1, 5, 40])
def test_layers_in_a_row(gpu, ops, t, dtype, stream) -> None:
    layers = [Layer(ops, dtype, seed) for seed in (300, 400)]
    hidden, x, real = inputs(t, dtype, stream, t)
    for start in (0, 40 if t < 24 else 20):  # a prompt, then more behind it
        positions = start + torch.arange(t, device="cuda")
        s, y = hidden, x
        for layer in layers:
            a = layer.step(s, y, positions, real)
            layer.check(a, positions)
            s, y = a["hidden2"], a["out"]


@pytest.mark.parametrize("t", [1, 5])
def test_a_captured_layer_along_a_sequence(gpu, ops, t) -> None:
    """The replayed layer writes its keys and values at positions read on the device; every replay gives the eager
    call's bits, which come from a cache of its own."""
    captured, eager = Layer(ops, BF16, 500), Layer(ops, BF16, 500)
    stream, x, real = inputs(t, BF16, F32, 9)
    positions = torch.arange(t, device="cuda")
    captured.step(stream, x, positions, real)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = captured.step(stream, x, positions, real)
    for i in range(5):
        new_stream, new_x, _ = inputs(t, BF16, F32, 20 + i)
        stream.copy_(new_stream)
        x.copy_(new_x)
        positions.copy_(i * t + torch.arange(t, device="cuda"))
        want = eager.step(stream, x, positions, real)
        graph.replay()
        torch.cuda.synchronize()
        for name, value in want.items():
            assert torch.equal(got[name], value), (i, name)
        assert torch.equal(captured.keys, eager.keys) and torch.equal(captured.values, eager.values)
