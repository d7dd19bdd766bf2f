"""A mixture-of-experts layer from the router's logits (`HipPackedMoEExperts.forward_logits`, `mxa_moe_layer`,
`mxa_moe_topk`).

* The routing against 64-bit arithmetic: the ids exactly. e = 2^-24: a weight is exp(l - max), whose argument is rounded
  once (|l - max| e) and which expf gives within 4 e, over a sum of up to 256 of them in 4 + 6 additions, times the scale:
  within (30 + 2 |l - max| + 2 max |l - max|) e of itself.
* The layer against the reference's loop over per-expert modules on the same ids and weights, bit for bit.
* The layer in float32 against its formula in 64 bits, the bound carried along from the kernel's roundings (below)."""

import numpy as np
import pytest
import torch
import torch.nn.functional as F

from matricxon_amd import synthetic as S
from matricxon_amd.gemm import q8k_bytes, q8k_views
from matricxon_amd.moe import HipPackedMoEExperts
from oracle import dequant as D
from tests.test_gpu_moe import build_experts, expert_weights, reference_forward

pytestmark = pytest.mark.gpu

E32 = 2.0 ** -24
F32, BF16 = torch.float32, torch.bfloat16
INF = float("inf")


def router(t, e, seed, dt=F32, spread=1.5):
    g = torch.Generator().manual_seed(seed)
    return (spread * torch.randn(t, e, generator=g)).to(dt).cuda()


def check_routing(logits, top_k, norm, scale, ids, wts):
    assert ids.dtype == torch.int32 and wts.dtype == F32 and ids.shape == wts.shape == (logits.shape[0], top_k)
    l64 = logits.double().cpu().numpy()
    ids, wts = ids.cpu().numpy(), wts.double().cpu().numpy()
    for row, (i, w) in enumerate(zip(ids, wts)):
        l = l64[row]
        best = sorted((e for e in range(len(l)) if l[e] > -INF), key=lambda e: (-l[e], e))
        chosen = best[:top_k]
        assert i.tolist() == chosen + [-1] * (top_k - len(chosen)), row
        assert (w[len(chosen):] == 0).all()
        if not chosen:
            continue
        d = l[chosen] - l[best[0]]
        total = np.exp(d).sum() if norm else np.exp(l[best] - l[best[0]]).sum()
        want = np.exp(d) / total * scale
        far = np.abs(l[best] - l[best[0]]).max()
        assert (np.abs(w[: len(chosen)] - want) <= (30 + 2 * np.abs(d) + 2 * far) * E32 * np.abs(want) + 1e-44).all(), row


@pytest.mark.parametrize("dt", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("t,e,k", [(1, 1, 1), (1, 8, 2), (5, 64, 8), (3, 256, 16), (9, 63, 5), (2, 3, 3), (1, 65, 1),
                                   (1000, 40, 8), (6, 130, 6)])
@pytest.mark.parametrize("norm", [False, True])
def test_topk(gpu, dt, t, e, k, norm) -> None:
    logits = router(t, e, t + e, dt)  # bfloat16 logits: many ties
    check_routing(logits, k, norm, 2.5, *gpu.moe_topk(logits, k, norm, 2.5))
    wide = router(t, e + 3, 1, dt)[:, 1 : e + 1]  # rows that are not adjacent
    check_routing(wide, k, norm, 1.0, *gpu.moe_topk(wide, k, norm))


def test_topk_masks_ties_and_extremes(gpu) -> None:
    logits = router(8, 12, 3)
    logits[0] = -INF
    logits[1, 1:] = -INF
    logits[2, ::2] = -INF
    logits[3] = 0.0
    logits[3, ::2] = -0.0  # the same value
    logits[4] = torch.finfo(F32).min  # a mask of the type's lowest value is a number like any other
    logits[5, :6] = torch.finfo(F32).min
    logits[6] = 1e38
    logits[7] = torch.linspace(-80, 80, 12)
    for norm in (False, True):
        check_routing(logits, 6, norm, 1.0, *gpu.moe_topk(logits, 6, norm))
    logits = torch.tensor([[1.0, float("nan"), 2.0, -INF], [1.0, 0.0, 2.0, -INF]], device="cuda")
    ids, wts = gpu.moe_topk(logits, 3)
    assert ids.tolist() == [[1, 2, 0], [2, 0, 1]]
    assert wts[0].isnan().all() and wts[1].isfinite().all()


# (gate and up, down, experts, n_embd, ffn_len, top_k): each type in each place; rows of 1 to 64 blocks, among them
# counts that do not divide a wave; rows that start between 16-byte words; output widths that leave the last rows of a
# wave and of a workgroup partial; experts of one row set
LAYERS = [
    (D.Q4_K, D.Q6_K, 8, 1024, 512, 2), (D.Q6_K, D.Q4_K, 6, 512, 1024, 3), (D.Q8_0, D.Q8_0, 40, 1536, 512, 8),
    (D.Q4_K, D.Q4_K, 64, 2048, 1024, 8), (D.Q6_K, D.Q8_0, 5, 768, 1280, 1), (D.Q8_0, D.Q6_K, 4, 256, 256, 4),
    (D.Q6_K, D.Q6_K, 3, 2816, 2304, 2), (D.Q4_K, D.Q6_K, 2, 4096, 14336, 2), (D.Q8_0, D.Q4_K, 3, 5120, 768, 2),
    (D.Q6_K, D.Q6_K, 16, 256, 256, 16), (D.Q4_K, D.Q8_0, 2, 16384, 256, 1), (D.Q4_K, D.Q6_K, 2, 256, 16384, 2),
    (D.Q8_0, D.Q8_0, 2, 8448, 8448, 1), (D.Q6_K, D.Q4_K, 129, 512, 256, 7),
]


def logits_for(t, e, k, seed, dt=F32):
    """Routings in which experts have no token, one, and (from five tokens on) more than four."""
    logits = router(t, e, seed, dt)
    if t >= 5:
        logits[:, 0] += 9  # one expert for all
    if t >= 3:
        logits[1, : e // 2] = -INF
        logits[t - 1] = -INF
    return logits


@pytest.mark.parametrize("case", range(len(LAYERS)))
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_layer_is_the_reference_loop(gpu, case, dtype) -> None:
    gt, dt, e, embd, ffn, k = LAYERS[case]
    mod, per_expert = build_experts((gt, gt, dt), e, embd, ffn, dtype, seed=900 + case)
    for t in (1, 2, 4, 8):
        if t * k > 64:
            continue
        assert gpu._lib.mxa_moe_layer_workspace_bytes(gt, dt, e, k, t, embd, ffn, int(dtype == BF16)) > 0
        x = torch.from_numpy(S.activations(t, embd, seed=case + t)).cuda().to(dtype)
        logits = logits_for(t, e, k, case, BF16 if t == 4 else F32)
        norm, scale = t != 2, 2.5 if t == 8 else 1.0
        out, ids, wts = mod.forward_logits(x, logits, k, norm, scale)
        check_routing(logits, k, norm, scale, ids, wts)
        live = (ids >= 0).all(1)
        want = torch.zeros_like(out)
        want[live] = reference_forward(x[live], wts[live], ids[live].long(), per_expert, F.silu)
        for row in ((ids >= 0).any(1) & ~live).nonzero().flatten().tolist():  # fewer experts than slots
            n = int((ids[row] >= 0).sum())
            want[row] = reference_forward(x[row][None], wts[row, :n][None], ids[row, :n].long()[None], per_expert, F.silu)
        assert out.dtype == dtype and out.shape == x.shape
        assert torch.equal(out, want), f"{t} tokens: max |diff| {(out.float() - want.float()).abs().max().item()}"


@pytest.mark.parametrize("t", [1, 5])
@pytest.mark.parametrize("gt,dt", [(D.Q6_K, D.Q8_0), (D.Q8_0, D.Q6_K)])
def test_layer_formula_in_64_bits(gpu, gt, dt, t) -> None:
    """A float32 layer of blocks whose values are one product. With e = 2^-24 and A = sum |w| |x| of a row of nb blocks,
    a float32 dot of exact integer blocks is within (nb + 4) e A. silu has a slope of at most 1.1 and is itself within
    6 e; so each activation's error is known, and with it whether its Q8_K code may be the neighbouring one (its
    unrounded code lies within its error of a half): those, and only those, are allowed one step."""
    e, embd, ffn, k = 6, 512, 768, 3
    w = {n: expert_weights(ty, e, a, b, seed) for n, ty, a, b, seed in
         (("gate", gt, ffn, embd, 1), ("up", gt, ffn, embd, 50), ("down", dt, embd, ffn, 90))}
    mod = HipPackedMoEExperts(*(torch.from_numpy(w[n]).cuda() for n in ("gate", "up", "down")), gt, gt, dt, embd, ffn,
                              F.silu, F32)
    x = S.activations(t, embd, seed=7)
    logits = router(t, e, 2)
    out, ids, wts = mod.forward_logits(torch.from_numpy(x).cuda(), logits, k)
    check_routing(logits, k, True, 1.0, ids, wts)
    value = lambda n, i, ty, rows: D.dequantize(ty, w[n][i]).astype(np.float64).reshape(rows, -1)  # noqa: E731
    step = lambda v: np.repeat(v, 256)  # noqa: E731
    l64, ids = logits.double().cpu().numpy(), ids.cpu().numpy()
    for row in range(t):
        top = np.abs(x[row].reshape(-1, 256)).max(1).astype(np.float32)
        q = np.rint(x[row] * step(np.float32(127) / top)).astype(np.float64)
        xq = q * step((top / np.float32(127)).astype(np.float64))
        p = np.exp(l64[row, ids[row]] - l64[row].max())
        want, bound = np.zeros(embd), np.zeros(embd)
        for expert, weight in zip(ids[row], p / p.sum()):
            (g, dg), (u, du) = ((m @ xq, (embd // 256 + 4) * E32 * (np.abs(m) @ np.abs(xq)))
                                for m in (value(n, expert, gt, ffn) for n in ("gate", "up")))
            s = g / (1 + np.exp(-g))
            ds = 1.1 * dg + 6 * E32 * np.abs(s)
            a = s * u
            da = np.abs(s) * du + np.abs(u) * ds + ds * du + E32 * np.abs(a)
            top = step(np.abs(a.reshape(-1, 256)).max(1))
            dtop = step(da.reshape(-1, 256).max(1))
            code = np.abs(a) * 127 / top
            dcode = 127 * da / top + code * dtop / top + 3 * E32 * code
            either = np.abs(code - np.floor(code) - 0.5) <= dcode
            aq = np.sign(a) * np.rint(code) * top / 127
            daq = np.where(either, top / 127, 0) + np.rint(code) * (dtop / 127 + 2 * E32 * top / 127)
            m = value("down", expert, dt, embd)
            y = m @ aq
            dy = np.abs(m) @ daq + (ffn // 256 + 4) * E32 * (np.abs(m) @ np.abs(aq))
            far = np.abs(l64[row] - l64[row].max()).max()
            want += weight * y
            bound += weight * dy + (30 + 4 * far + k + 2) * E32 * weight * np.abs(y)
        got = out[row].double().cpu().numpy()
        assert (np.abs(got - want) <= bound).all()
        assert np.median(bound) < 0.01 * np.sqrt(np.mean(want ** 2))  # and the bound says something


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_padding_is_left_out(gpu, dtype) -> None:
    """Tokens without an expert hold anything and get zeros, alone or among others, few or many."""
    mod, _ = build_experts((D.Q4_K, D.Q4_K, D.Q6_K), 8, 512, 512, dtype, seed=5)
    for t in (1, 3, 8, 20):
        x = torch.from_numpy(S.activations(t, 512, seed=t)).cuda().to(dtype)
        logits = router(t, 8, t)
        want = mod.forward_logits(x, logits, 2)[0]
        logits[::2] = -INF
        x[::2] = float("nan")
        out, ids, wts = mod.forward_logits(x, logits, 2)
        assert (out[::2] == 0).all() and (ids[::2] == -1).all() and (wts[::2] == 0).all()
        assert torch.equal(out[1::2], want[1::2])
        logits[:] = -INF
        assert (mod.forward_logits(x, logits, 2)[0] == 0).all()


def test_infinities_and_nan_stay_in_their_token(gpu) -> None:
    mod, _ = build_experts((D.Q4_K, D.Q4_K, D.Q6_K), 4, 512, 512, BF16, seed=6)
    x = torch.from_numpy(S.activations(4, 512, seed=1)).cuda().bfloat16()
    logits = router(4, 4, 1)
    want = mod.forward_logits(x, logits, 2)[0]
    x[1], logits[2, 0] = INF, float("nan")
    out = mod.forward_logits(x, logits, 2)[0]
    assert torch.equal(out[[0, 3]], want[[0, 3]]) and out[2].isnan().all()


def test_any_number_of_tokens_gives_the_same_rows(gpu) -> None:
    """Each token's row is the same alone, among eight (two launches) and among twenty (grouped)."""
    mod, _ = build_experts((D.Q4_K, D.Q4_K, D.Q6_K), 16, 1024, 512, BF16, seed=8)
    x = torch.from_numpy(S.activations(20, 1024, seed=2)).cuda().bfloat16()
    logits = router(20, 16, 4)
    out, ids, wts = mod.forward_logits(x, logits, 4)
    assert torch.equal(mod(x, wts, ids.long()), out)
    for part in [slice(i, i + 1) for i in range(20)] + [slice(0, 8), slice(8, 16), slice(3, 12)]:
        for a, b in zip(mod.forward_logits(x[part], logits[part], 4), (out, ids, wts)):
            assert torch.equal(a, b[part])


@pytest.mark.parametrize("why", ["types", "activation", "iq4_xs", "rows", "pairs"])
def test_layers_the_two_launches_do_not_take(gpu, why) -> None:
    """Mixed gate and up types, another activation, IQ4_XS, rows of more than 64 blocks, more than 64 pairs: the grouped
    launches."""
    gt, ut, act, embd, e, k, t = D.Q4_K, D.Q4_K, F.silu, 512, 4, 2, 3
    if why == "types":
        ut = D.Q6_K
    elif why == "activation":
        act = F.gelu
    elif why == "iq4_xs":
        gt = ut = D.IQ4_XS
    elif why == "rows":
        embd = 65 * 256
    else:
        e, k, t = 12, 12, 6
    mod, _ = build_experts((gt, ut, D.Q6_K), e, embd, 256, BF16, seed=9)
    mod.activation = act
    mod = HipPackedMoEExperts(mod.gate_packed, mod.up_packed, mod.down_packed, gt, ut, D.Q6_K, embd, 256, act, BF16)
    x = torch.from_numpy(S.activations(t, embd, seed=3)).cuda().bfloat16()
    logits = router(t, e, 6)
    assert mod._few_tokens(x, logits, k, True, 1.0) is None
    out, ids, wts = mod.forward_logits(x, logits, k)
    check_routing(logits, k, True, 1.0, ids, wts)
    assert torch.equal(out, mod(x, wts, ids.long()))


def torch_q8k(x):
    """The Q8_K workspace of x (rows, k) from torch operations, `127.0 / amax` as torch evaluates it."""
    v = x.float().view(len(x), -1, 256)
    top = v.abs().amax(-1, keepdim=True)
    q = torch.round(v * (127.0 / top)).clamp(-127, 127).to(torch.int8)
    ws = torch.zeros(q8k_bytes(*x.shape), dtype=torch.uint8, device="cuda")
    for view, part in zip(q8k_views(ws, *x.shape), (q.view(x.shape), (top / torch.full_like(top, 127.0)).squeeze(-1),
                                                    q.view(len(x), -1, 16, 16).sum(-1, dtype=torch.int16))):
        view.copy_(part)
    return ws


@pytest.mark.parametrize("t", [1, 8, 11])
def test_reciprocal_code_scales(gpu, t) -> None:
    """Blocks whose codes torch computes, through the projections of each expert, bit for bit."""
    gt, dt, e, embd, ffn, k = D.Q4_K, D.Q6_K, 4, 2048, 768, 2
    mod, per_expert = build_experts((gt, gt, dt), e, embd, ffn, BF16, seed=14)
    x = torch.from_numpy(S.activations(t, embd, seed=5)).cuda().bfloat16()
    x[0, :256] *= 3.90625 / x[0, :256].abs().max()  # a block whose codes differ
    logits = router(t, e, 8)
    out, ids, wts = mod.forward_logits(x, logits, k, q8k_scale="reciprocal")

    def through(linear, v):
        y = torch.empty(len(v), linear.out_features, dtype=BF16, device="cuda")
        return gpu.matmul_q8k(linear.ggml_type, linear.packed, torch_q8k(v), None, y, len(v), linear.out_features,
                              linear.in_features)

    want = torch.zeros(t, embd, device="cuda")
    for row in range(t):
        for slot in sorted(range(k), key=lambda j: int(ids[row, j])):
            gate, up, down = per_expert[int(ids[row, slot])]
            act = F.silu(through(gate, x[row][None])) * through(up, x[row][None])
            want[row] += through(down, act)[0].float() * wts[row, slot]
    assert torch.equal(out, want.to(BF16))
    assert not torch.equal(out, mod.forward_logits(x, logits, k)[0])
    with pytest.raises(ValueError, match="q8k_scale"):
        mod.forward_logits(x, logits, k, q8k_scale="other")
    mixed, _ = build_experts((D.Q4_K, D.Q6_K, D.Q6_K), 2, 256, 256, BF16, seed=15)
    with pytest.raises(ValueError, match="reciprocal"):
        mixed.forward_logits(x[:, :256], logits[:, :2], 1, q8k_scale="reciprocal")


def test_inputs_of_any_layout(gpu) -> None:
    """x of another float type, of wider rows, of a start that is not 16-byte aligned; transposed logits."""
    mod, _ = build_experts((D.Q4_K, D.Q4_K, D.Q4_K), 8, 512, 256, BF16, seed=10)
    x = torch.from_numpy(S.activations(3, 512, seed=4)).cuda().bfloat16()
    logits = router(3, 8, 7)
    want, ids, wts = mod.forward_logits(x, logits, 2)
    wide = torch.zeros(3, 600, dtype=BF16, device="cuda")
    wide[:, 1:513] = x
    flat = torch.zeros(3 * 512 + 1, dtype=BF16, device="cuda")
    flat[1:] = x.flatten()
    for y in (wide[:, 1:513], flat[1:].view(3, 512)):
        assert torch.equal(mod.forward_logits(y, logits.t().contiguous().t(), 2)[0], want)
    for dt in (F32, torch.float16):
        out = mod.forward_logits(x.to(dt), logits, 2)[0]
        assert out.dtype == dt and torch.equal(out, mod(x.to(dt), wts, ids.long()))
    none = mod.forward_logits(x[:0], logits[:0], 2)
    assert none[0].shape == (0, 512) and none[1].shape == none[2].shape == (0, 2)


def test_captured_and_replayed(gpu) -> None:
    """Two captured layers, one after the other, each replayed on new inputs with eager calls between."""
    mod, _ = build_experts((D.Q4_K, D.Q4_K, D.Q6_K), 16, 1024, 768, BF16, seed=11)
    state = []
    for t in (1, 6):
        x, logits = torch.zeros(t, 1024, dtype=BF16, device="cuda"), torch.zeros(t, 16, device="cuda")
        mod.forward_logits(x, logits, 4)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = mod.forward_logits(x, logits, 4)
        state.append((x, logits, graph, res))
    for i in range(4):
        for x, logits, graph, res in state:
            x.copy_(torch.from_numpy(S.activations(len(x), 1024, seed=i)))
            logits.copy_(router(len(x), 16, i))
        wants = [mod.forward_logits(x, logits, 4) for x, logits, _, _ in state]
        for _, _, graph, _ in state:
            graph.replay()
        torch.cuda.synchronize()
        for (_, _, _, res), want in zip(state, wants):
            assert all(torch.equal(a, b) for a, b in zip(res, want))


def test_two_streams_at_once(gpu) -> None:
    mod, _ = build_experts((D.Q4_K, D.Q4_K, D.Q6_K), 16, 1024, 768, BF16, seed=12)
    cases = [(torch.from_numpy(S.activations(t, 1024, seed=t)).cuda().bfloat16(), router(t, 16, t)) for t in (3, 7)]
    wants = [mod.forward_logits(x, logits, 4) for x, logits in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        for i, ((x, logits), s) in enumerate(zip(cases, streams)):
            with torch.cuda.stream(s):
                got[i].append(mod.forward_logits(x, logits, 4))
    torch.cuda.synchronize()
    for results, want in zip(got, wants):
        for res in results:
            assert all(torch.equal(a, b) for a, b in zip(res, want))


def test_refusals(gpu) -> None:
    mod, _ = build_experts((D.Q4_K, D.Q4_K, D.Q4_K), 4, 256, 256, BF16, seed=13)
    x, logits = torch.zeros(2, 256, dtype=BF16, device="cuda"), torch.zeros(2, 4, device="cuda")
    for a, b, k in ((x[:, :128], logits, 2), (x[0], logits, 2), (x.cpu(), logits, 2), (x, logits.cpu(), 2),
                    (x, logits[:1], 2), (x, logits[:, :3], 2), (x, logits.half(), 2), (x, logits[0], 2),
                    (x, logits, 0), (x, logits, 5)):
        with pytest.raises(ValueError):
            mod.forward_logits(a, b, k)
    for b, k in ((logits.cpu(), 2), (logits[0], 1), (logits.half(), 2), (logits, 5), (logits, 0),
                 (torch.zeros(1, 257, device="cuda"), 2), (torch.zeros(1, 40, device="cuda"), 17)):
        with pytest.raises(ValueError):
            gpu.moe_topk(b, k)


def test_an_activation_set_later(gpu) -> None:
    mod, _ = build_experts((D.Q4_K, D.Q4_K, D.Q6_K), 4, 512, 256, BF16, seed=16)
    x = torch.from_numpy(S.activations(3, 512, seed=6)).cuda().bfloat16()
    logits = router(3, 4, 9)
    silu = mod.forward_logits(x, logits, 2)[0]
    mod.activation = F.gelu
    out, ids, wts = mod.forward_logits(x, logits, 2)
    assert torch.equal(out, mod(x, wts, ids.long())) and not torch.equal(out, silu)
    mod.activation = torch.nn.SiLU()
    assert torch.equal(mod.forward_logits(x, logits, 2)[0], silu)


def test_the_most_tokens(gpu) -> None:
    n = 1 << 24
    ids, wts = gpu.moe_topk(torch.zeros(n, 1, dtype=BF16, device="cuda"), 1, True, 0.5)
    assert (ids == 0).all() and (wts == 0.5).all()
    with pytest.raises(ValueError, match="tokens"):
        gpu.moe_topk(torch.zeros(1, 2, device="cuda").expand(n + 1, 2), 1)
    for bad in (torch.zeros((), device="cuda"), torch.zeros(4, device="cuda")):
        with pytest.raises(ValueError, match="router logits"):
            gpu.moe_topk(bad, 1)


def test_many_tokens_half_of_them_padding(gpu) -> None:
    """More tokens than one routing launch takes; a row of padding costs the others nothing."""
    mod, _ = build_experts((D.Q8_0, D.Q8_0, D.Q8_0), 8, 256, 256, BF16, seed=17)
    t = 32768 + 40
    x = torch.from_numpy(S.activations(64, 256, seed=7)).cuda().bfloat16().repeat(t // 64 + 1, 1)[:t]
    logits = router(64, 8, 10).repeat(t // 64 + 1, 1)[:t]
    want, wids, _ = mod.forward_logits(x[:64], logits[:64], 2)
    logits[1::2] = -INF
    out, ids, _ = mod.forward_logits(x, logits, 2)
    even = torch.arange(0, t, 2, device="cuda")
    assert torch.equal(out[even], want[even % 64]) and torch.equal(ids[even], wids[even % 64])
    assert (out[1::2] == 0).all() and (ids[1::2] == -1).all()


@pytest.mark.parametrize("t,e,k", [(1, 1, 1), (1, 8, 2), (7, 256, 16), (63, 3, 3), (300, 64, 8), (5000, 16, 4)])
@pytest.mark.parametrize("share", [0.0, 0.3, 1.0])
@pytest.mark.parametrize("dt", [torch.int32, torch.int64], ids=["int32", "int64"])
def test_masked_routing(gpu, t, e, k, share, dt) -> None:
    """Pairs in expert order, those without an expert behind them in their own order."""
    g = torch.Generator().manual_seed(t + k)
    ids = torch.randint(0, e, (t, k), generator=g)
    ids[torch.rand(t, k, generator=g) < share] = -1
    offsets, pair_tok, rows, ids32 = gpu.moe_route(ids.to(dt).cuda(), e, masked=True)
    key = torch.where(ids < 0, e, ids).flatten()
    order = torch.argsort(key, stable=True)
    place = torch.empty_like(order)
    place[order] = torch.arange(t * k)
    assert torch.equal(offsets.cpu().long(), torch.tensor([int((key < i).sum()) for i in range(e + 1)]))
    assert torch.equal(pair_tok.cpu().long(), order // k) and torch.equal(rows.cpu().long(), place.view(t, k))
    assert torch.equal(ids32.cpu().long(), ids)


@pytest.mark.parametrize("e,k,t", [(1, 1, 1), (1, 1, 3), (1, 1, 8), (2, 2, 8), (256, 16, 4), (200, 9, 7), (64, 16, 1)])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_one_expert_to_the_most(gpu, e, k, t, dtype) -> None:
    """Every token's pairs in one item after another, and every pair an item of its own."""
    mod, _ = build_experts((D.Q8_0, D.Q8_0, D.Q4_K), e, 256, 512, dtype, seed=18)
    x = torch.from_numpy(S.activations(t, 256, seed=8)).cuda().to(dtype)
    logits = router(t, e, 11)
    out, ids, wts = mod.forward_logits(x, logits, k)
    assert mod._layer_bytes[t, k] > 0
    check_routing(logits, k, True, 1.0, ids, wts)
    assert torch.equal(out, mod._grouped(x, wts, ids))


@pytest.mark.parametrize("gt,dt,e,embd,ffn,k,t", [
    (D.Q4_K, D.Q6_K, 8, 512, 768, 4, 8), (D.Q8_0, D.Q8_0, 8, 512, 512, 4, 8), (D.Q8_0, D.Q8_0, 4, 1024, 256, 2, 1),
    (D.Q6_K, D.Q8_0, 16, 512, 512, 3, 7), (D.Q6_K, D.Q4_K, 3, 256, 14336, 2, 4), (D.Q8_0, D.Q6_K, 5, 256, 512, 2, 21),
    (D.Q4_K, D.Q4_K, 12, 256, 512, 9, 9)])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_reciprocal_code_scales_of_every_form(gpu, gt, dt, e, embd, ffn, k, t, dtype) -> None:
    """More than 16 pairs (down by items, summed by the combine), rows of down that leave the sum too few waves, more
    tokens than a call takes, 8-bit experts and float32 layers, whose activations are read and rounded by other code: the
    layer's own silu(gate) * up, through each expert's projections on blocks that torch computes."""
    mod, per_expert = build_experts((gt, gt, dt), e, embd, ffn, dtype, seed=19)
    x = torch.from_numpy(S.activations(t, embd, seed=9)).cuda().to(dtype)
    x[:, :256] *= 3.90625 / x[:, :256].abs().amax(1, keepdim=True)  # blocks whose codes differ
    logits = router(t, e, 12)
    out, ids, wts = mod.forward_logits(x, logits, k, q8k_scale="reciprocal")
    check_routing(logits, k, True, 1.0, ids, wts)

    def through(linear, v, out_dtype):
        y = torch.empty(len(v), linear.out_features, dtype=out_dtype, device="cuda")
        return gpu.matmul_q8k(linear.ggml_type, linear.packed, torch_q8k(v), None, y, len(v), linear.out_features,
                              linear.in_features)

    want = torch.zeros(t, embd, device="cuda")
    for row in range(t):
        for slot in sorted(range(k), key=lambda j: int(ids[row, j])):
            gate, up, down = per_expert[int(ids[row, slot])]
            g, u = (through(m, x[row][None], dtype) for m in (gate, up))
            act = F.silu(g) * u if dtype == BF16 else gpu.silu_mul_q8k(g, u)[0]
            want[row] += through(down, act, dtype)[0].float() * wts[row, slot]
    assert torch.equal(out, want.to(dtype))


@pytest.mark.parametrize("k", range(1, 17))
@pytest.mark.parametrize("masked", [False, True])
def test_combine_of_every_count_of_slots(gpu, k, masked) -> None:
    """1 to 16 slots a token and, masked, any number of them without an expert, whose rows and weights hold NaN: the sum
    in ascending id, one product and one addition at a time."""
    t, n = 40, 260
    g = torch.Generator(device="cuda").manual_seed(k)
    ids = torch.stack([torch.randperm(40, device="cuda", generator=g)[:k] for _ in range(t)]).int()
    wts, down = torch.rand(t, k, device="cuda", generator=g), torch.randn(t * k, n, device="cuda", generator=g)
    rows = torch.randperm(t * k, device="cuda", generator=g).int().view(t, k)
    if masked:
        off = torch.arange(k, device="cuda") >= torch.arange(t, device="cuda")[:, None] % (k + 1)
        off = off.gather(1, torch.rand(t, k, device="cuda", generator=g).argsort(1))
        ids[off], wts[off] = -1, float("nan")
        down[rows[off].long()] = float("nan")
    want = torch.zeros(t, n, device="cuda")
    order = torch.where(ids < 0, 1000, ids).argsort(1)
    for j in range(k):
        slot = order[:, j : j + 1]
        live = ids.gather(1, slot) >= 0
        term = down[rows.gather(1, slot).flatten().long()].bfloat16().float() * wts.gather(1, slot)
        want = torch.where(live, want + term, want)
    assert torch.equal(gpu.moe_combine(down, ids, wts, rows, round_bf16=True, masked=masked), want)
