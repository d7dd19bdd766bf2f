"""The operators around a decoder layer's packed projections, as measurable cases, each with a plain form.

* `norm`: the residual stream between two blocks. With block output x, stream r, gate g and residual scale s,
      u = x, or x * rsqrt(mean(x^2) + eps) * w_post   (a norm after the block)
      h = r + s * g * u                               (the new stream, in the stream's type)
      n = h * rsqrt(mean(h^2) + eps) * w              (the norm before the next block, in the block's type)
  `HipFusedOps.add_rms_norm`.
* `rotary`: rotary positions of q and k. Pair i of a head turns by the angle p * f_i at position p, the pair being
  elements (i, i + d/2) or (2i, 2i + 1) of the rotary part d of the head; f_i = base^(-2i/d), scaled for long contexts.
  `HipRotary`.
* `moe`: a mixture-of-experts layer from the router's logits for a few tokens: the top_k experts of each token, their
  weights, silu(gate) * up of each, down, and the weighted sum. The experts are packed GGUF blocks, which meet Q8_K
  activations (int8 of 256 values with one scale), and a bfloat16 layer holds gate, up, silu(gate), their product and
  each expert's output in bfloat16: these roundings are the layer's definition. A logit of -inf masks an expert; a
  slot without an expert has id -1 and weight 0.
  `HipPackedMoEExperts.forward_logits`.

Sizes are those of the benchmark's layers and expert sets (4096 wide with 32 + 8 heads of 128; 8 experts top 2 of
4096 x 14336, 64 top 8 of 2048 x 1024, 40 top 8 of 1536 x 512) and of ranges around them, from one token to a
prefill chunk of 4096 (a few tokens, up to eight, for `moe`).
"""

import math

import numpy as np
import torch

own = False

Q8_0, Q4_K, Q6_K = 8, 12, 14
GEOMETRY = {Q8_0: (32, 34), Q4_K: (256, 144), Q6_K: (256, 210)}  # (values, bytes) of a block
W_STD = 0.02
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ------------------------------------------------------------------------------------ the cases
def norm(name, m, k, x="bf16", stream="bf16", post=False, gate="none", scale=1.0):
    return {"name": name, "op": "norm", "m": m, "k": k, "x": x, "stream": stream, "post": post, "gate": gate,
            "scale": scale}


def rotary(name, t, q_heads, kv_heads, dim, rot, x="bf16", interleaved=False, scaling="none", factor=1.0,
           context=8192, far=0, decode=False):
    return {"name": name, "op": "rotary", "t": t, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "rot": rot,
            "x": x, "interleaved": interleaved, "scaling": scaling, "factor": factor, "context": context, "far": far,
            "decode": decode}


def moe(name, t, experts, top_k, embd, ffn, type_=Q4_K, down=Q6_K, logits="f32", norm_topk=True, scale=1.0,
        masked=False):
    return {"name": name, "op": "moe", "t": t, "experts": experts, "top_k": top_k, "embd": embd, "ffn": ffn,
            "type": type_, "down": down, "logits": logits, "norm_topk": norm_topk, "scale": scale, "masked": masked}


def listed():
    return [
        # one token of a decode step between attention and FFN: latency alone
        norm("norm_decode", 1, 4096),
        # sixteen replies of a model with norms on both sides of a block, a learned gate for each channel, a residual
        # scale, and its stream held in float32
        norm("norm_replies_sandwich", 16, 5120, stream="f32", post=True, gate="channel", scale=0.22),
        # a prompt of odd length and odd width in float32, with a gate for each token
        norm("norm_odd_f32", 333, 1155, x="f32", stream="f32", gate="token", scale=0.5),
        # a prefill chunk between two blocks, normed on both sides
        norm("norm_prefill", 4096, 4096, post=True),
        # one token's heads
        rotary("rotary_decode", 1, 32, 8, 128, 128, decode=True),
        # sixteen replies, each at its own place, interleaved pairs over part of a float32 head
        rotary("rotary_replies_partial", 16, 32, 32, 80, 32, x="f32", interleaved=True, decode=True),
        # a prompt of odd length near the end of a long context, scaled by wavelength
        rotary("rotary_far_yarn", 777, 40, 8, 128, 128, scaling="yarn", factor=32.0, context=32768, far=1 << 20),
        # a prefill chunk
        rotary("rotary_prefill", 4096, 32, 8, 128, 128, scaling="llama3", factor=8.0),
        # one token through few large experts
        moe("moe_large_1", 1, 8, 2, 4096, 14336),
        # one token through many small experts
        moe("moe_small_1", 1, 64, 8, 2048, 1024, norm_topk=False),
        # four replies, one of them padding, some experts masked; small 8-bit experts
        moe("moe_masked_4", 4, 40, 8, 1536, 512, type_=Q8_0, down=Q8_0, logits="bf16", masked=True),
        # eight replies through few large experts: the most weight that a few tokens touch
        moe("moe_large_8", 8, 8, 2, 4096, 14336, scale=2.5),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["norm", "rotary", "moe"])
    if op == "norm":
        x = rng.choice(["bf16", "bf16", "f32"])
        k = rng.choice([256 * _log(rng, 1, 32), 8 * _log(rng, 8, 1024), _log(rng, 64, 8192)])
        c = norm("", _log(rng, 1, 4096 * 4096 // k if k > 4096 else 4096), k, x,
                 "f32" if x == "f32" else rng.choice(["bf16", "f32"]), rng.random() < 0.5,
                 rng.choice(["none", "scalar", "channel", "token", "full"]), rng.choice([1.0, 0.22, 0.5, 1.4]))
    elif op == "rotary":
        dim = rng.choice([32, 64, 80, 96, 128, 128, 192, 256])
        kv = rng.choice([1, 2, 4, 8])
        context = rng.choice([4096, 8192, 32768])
        c = rotary("", _log(rng, 1, 4096), kv * rng.choice([1, 2, 4, 5]), kv, dim,
                   rng.choice([dim, dim, dim // 2, 2 * rng.randint(2, dim // 2)]), rng.choice(["bf16", "bf16", "f32"]),
                   rng.random() < 0.4, rng.choice(["none", "linear", "ntk", "yarn", "llama3"]),
                   rng.choice([2.0, 8.0, 32.0]), context, rng.choice([0, context, 1 << 20]), rng.random() < 0.3)
    else:
        experts, top_k, embd, ffn = rng.choice([(8, 2, 4096, 14336), (64, 8, 2048, 1024), (40, 8, 1536, 512),
                                                (16, 4, 2048, 1536), (32, 3, 2560, 768), (128, 6, 1024, 512),
                                                (5, 1, 4096, 4096)])
        type_ = rng.choice([Q4_K, Q4_K, Q6_K, Q8_0])
        c = moe("", _log(rng, 1, 8), experts, top_k, embd, ffn, type_, rng.choice([type_, Q6_K]),
                rng.choice(["f32", "bf16"]), rng.random() < 0.6, rng.choice([1.0, 2.5]), rng.random() < 0.3)
        c["type"] = Q4_K if embd * ffn > 1 << 25 else c["type"]  # no more weight than the largest listed case has
    del c["name"]
    return c


# --------------------------------------------------------------------------------------- inputs
def _bytes(g, shape):
    return torch.randint(0, 256, shape, dtype=torch.uint8, device="cuda", generator=g)


def _half(v):
    return v.to(torch.float16).view(torch.uint8).reshape(*v.shape, 2)


def packed(g, type_, n, k):
    """(n, row_bytes) packed rows of random quants whose values have a standard deviation of about W_STD."""
    size, nbytes = GEOMETRY[type_]
    nb = n * (k // size)
    out = _bytes(g, (nb, nbytes))
    s = W_STD * torch.exp(0.4 * torch.randn(nb, device="cuda", generator=g))  # block scales, a factor of about 2 apart
    if type_ == Q8_0:  # d, 32 signed bytes
        out[:, 0:2] = _half(s / 73)
        out[:, 2:] = torch.where(out[:, 2:] == 128, 129, out[:, 2:])
    elif type_ == Q4_K:  # d, dmin, 8 six-bit scales and mins, 128 bytes of nibbles
        sc = torch.randint(24, 64, (nb, 8), dtype=torch.uint8, device="cuda", generator=g)
        mn = (sc.int() + torch.randint(-6, 7, (nb, 8), device="cuda", generator=g)).clamp(0, 63).to(torch.uint8)
        d = s / (45 * 4.6)
        out[:, 0:2], out[:, 2:4] = _half(d), _half(7.5 * d)
        out[:, 4:8] = (sc[:, :4] & 63) | ((sc[:, 4:] >> 4) << 6)
        out[:, 8:12] = (mn[:, :4] & 63) | ((mn[:, 4:] >> 4) << 6)
        out[:, 12:16] = (sc[:, 4:] & 15) | ((mn[:, 4:] & 15) << 4)
    else:  # Q6_K: low nibbles, high bits, 16 signed scales, d
        out[:, 208:210] = _half(s / (74 * 18.5))
    return out.reshape(n, (k // size) * nbytes)


def _prepare_norm(case, g):
    m, k, xt, rt = case["m"], case["k"], TYPES[case["x"]], TYPES[case["stream"]]
    rand = lambda *shape: torch.randn(*shape, device="cuda", generator=g)  # noqa: E731
    weight = lambda: (1 + 0.2 * rand(k)).to(xt)  # noqa: E731
    shape = {"none": None, "scalar": (1,), "channel": (k,), "token": (m, 1), "full": (m, k)}[case["gate"]]
    # a stream grows with depth and has channels far above the rest
    r = 4 * rand(m, k) * torch.exp(0.8 * rand(k))
    return {"x": (1.5 * rand(m, k)).to(xt), "r": r.to(rt), "w": weight(), "post": weight() if case["post"] else None,
            "gate": None if shape is None else (0.6 + 0.3 * rand(*shape)).to(xt)}


def _positions(case, g):
    t, far = case["t"], case["far"]
    if case["decode"]:  # replies of different lengths
        return torch.randint(0, max(far, case["context"]), (t,), device="cuda", generator=g)
    return torch.arange(t, device="cuda") + int(torch.randint(0, far // 2 + 1, (1,), device="cuda", generator=g)) + far // 2


def _prepare_rotary(case, g):
    # q and k as a fused q | k | v projection leaves them: columns of one buffer
    t, hq, hk, d = case["t"], case["q_heads"], case["kv_heads"], case["dim"]
    qkv = torch.randn(t, (hq + 2 * hk) * d, device="cuda", generator=g).to(TYPES[case["x"]])
    q, k, _ = torch.split(qkv, [hq * d, hk * d, hk * d], dim=-1)
    return {"q": q.view(t, hq, d), "k": k.view(t, hk, d), "positions": _positions(case, g)}


def _prepare_moe(case, g):
    t, e, embd, ffn = case["t"], case["experts"], case["embd"], case["ffn"]
    logits = 1.5 * torch.randn(t, e, device="cuda", generator=g)
    if case["masked"]:  # a quarter of the experts is off, and the last token is padding
        logits[torch.rand(t, e, device="cuda", generator=g) < 0.25] = -math.inf
        logits[-1] = -math.inf
    s = {"x": torch.randn(t, embd, device="cuda", generator=g).to(torch.bfloat16),
         "logits": logits.to(TYPES[case["logits"]])}
    for name, type_, n, k in (("gate", case["type"], ffn, embd), ("up", case["type"], ffn, embd),
                              ("down", case["down"], embd, ffn)):
        s[name] = packed(g, type_, e * n, k).view(e, n, -1)
    return s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    make = {"norm": _prepare_norm, "rotary": _prepare_rotary, "moe": _prepare_moe}[case["op"]]
    return {"case": case, **make(case, g)}


# --------------------------------------------------------------------------------- plain forms
EPS = 1e-5
BASE = 10000.0


def _rms(x, w):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w


def _plain_norm(s):
    case = s["case"]
    u = s["x"].float()
    if s["post"] is not None:
        u = _rms(u, s["post"].float())
    if s["gate"] is not None:
        u = u * s["gate"].float()
    h = (s["r"].float() + case["scale"] * u).to(s["r"].dtype)
    return h, _rms(h.float(), s["w"].float()).to(s["x"].dtype)


def _frequencies(case, device):
    """The angle per position of each pair, in 64 bits, and the factor on the rotated values."""
    d, factor, context = case["rot"], case["factor"], case["context"]
    i = torch.arange(d // 2, dtype=torch.float64, device=device)
    base = BASE * factor ** (d / (d - 2)) if case["scaling"] == "ntk" else BASE
    f = base ** (-2 * i / d)
    if case["scaling"] == "linear":
        return f / factor, 1.0
    if case["scaling"] == "yarn":  # short wavelengths as they are, long ones stretched, a ramp between
        at = lambda turns: d * math.log(context / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        low, high = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), d - 1)
        ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
        return f / factor * ramp + f * (1 - ramp), 0.1 * math.log(factor) + 1
    if case["scaling"] == "llama3":  # the same by the turns that a context holds: 4 and more kept, 1 and fewer stretched
        s = ((context * f / (2 * math.pi) - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        return (1 - s) * f / factor + s * f, 1.0
    return f, 1.0


def _plain_rotary(s):
    case = s["case"]
    f, m = _frequencies(case, s["q"].device)
    angle = (s["positions"].double()[:, None] * f)[:, None, :]
    cos, sin = (m * torch.cos(angle)).float(), (m * torch.sin(angle)).float()
    d = case["rot"]

    def turn(x):
        v = x.float()
        if case["interleaved"]:
            a, b = v[..., 0:d:2], v[..., 1:d:2]
            r = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
        else:
            a, b = v[..., : d // 2], v[..., d // 2 : d]
            r = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
        return torch.cat((r, v[..., d:]), -1).to(x.dtype)

    return turn(s["q"]), turn(s["k"])


def _f16(b):
    return b.contiguous().view(torch.float16).float()


def _values(b, type_):
    """Packed bytes (..., row_bytes) as float32 values (..., k)."""
    lead = b.shape[:-1]
    b = b.reshape(-1, GEOMETRY[type_][1])
    if type_ == Q8_0:
        v = _f16(b[:, 0:2]) * b[:, 2:].contiguous().view(torch.int8).float()
    elif type_ == Q4_K:
        d, dmin, s = _f16(b[:, 0:2]), _f16(b[:, 2:4]), b[:, 4:16]
        sc = torch.cat((s[:, 0:4] & 63, (s[:, 8:12] & 15) | ((s[:, 0:4] >> 6) << 4)), 1).float() * d
        mn = torch.cat((s[:, 4:8] & 63, (s[:, 8:12] >> 4) | ((s[:, 4:8] >> 6) << 4)), 1).float() * dmin
        q = b[:, 16:].reshape(-1, 4, 1, 32)
        q = torch.cat((q & 15, q >> 4), 2).reshape(-1, 8, 32)
        v = q.float() * sc[:, :, None] - mn[:, :, None]
    else:
        ql, qh = b[:, :128].reshape(-1, 2, 1, 2, 32), b[:, 128:192].reshape(-1, 2, 1, 32)
        low = torch.cat((ql & 15, ql >> 4), 2).reshape(-1, 2, 4, 32)
        high = torch.cat((qh & 3, (qh >> 2) & 3, (qh >> 4) & 3, qh >> 6), 2)
        q = (low | (high << 4)).float() - 32
        sc = b[:, 192:208].contiguous().view(torch.int8).float() * _f16(b[:, 208:210])
        v = q.reshape(-1, 16, 16) * sc[:, :, None]
    return v.reshape(*lead, -1)


def _q8k(x):
    """The values that x (..., k) has as Q8_K blocks: int8 of 256 values with one float32 scale."""
    v = x.float().reshape(*x.shape[:-1], -1, 256)
    top = v.abs().amax(-1, keepdim=True)
    q = torch.where(top > 0, torch.round(v * (127.0 / top)).clamp(-127, 127), 0.0)
    return (q * (top / 127.0)).reshape(x.shape)


def _route(case, logits):
    """ids (-1 where a token has no expert left) and float32 weights, the top experts first, ties to the lowest id."""
    v, ids = torch.sort(logits.float(), dim=-1, descending=True, stable=True)
    p = torch.exp(v - torch.where(v[:, :1] == -math.inf, 0.0, v[:, :1]))
    k = case["top_k"]
    total = (p[:, :k] if case["norm_topk"] else p).sum(-1, keepdim=True)
    live = v[:, :k] > -math.inf
    w = torch.where(live, p[:, :k] / torch.where(total > 0, total, 1.0) * case["scale"], 0.0)
    return torch.where(live, ids[:, :k], -1).int(), w


def _plain_moe(s):
    case = s["case"]
    ids, w = _route(case, s["logits"])
    t, k = ids.shape
    e = ids.clamp(min=0).reshape(-1).long()
    xs = _q8k(s["x"]).repeat_interleave(k, 0).unsqueeze(-1)
    gate, up = (torch.bmm(_values(s[n][e], case["type"]), xs).squeeze(-1).bfloat16().float() for n in ("gate", "up"))
    silu = (gate / (1 + torch.exp(-gate))).bfloat16().float()
    act = _q8k((silu * up).bfloat16()).unsqueeze(-1)
    down = torch.bmm(_values(s["down"][e], case["down"]), act).squeeze(-1).bfloat16().float()
    down = torch.where(ids.reshape(-1, 1) < 0, 0.0, down * w.reshape(-1, 1))
    return down.view(t, k, -1).sum(1).to(s["x"].dtype), ids, w


# ----------------------------------------------------------------------- the framework's calls
def _own_norm(s):
    from matricxon_amd.fused_ops import HipFusedOps

    ops = HipFusedOps.active()
    if ops is None:
        HipFusedOps.configure(True)
        ops = HipFusedOps.active()
    return ops.add_rms_norm(s["r"], s["x"], s["w"], EPS, post_weight=s["post"], gate=s["gate"],
                            scale=s["case"]["scale"])


def _own_rotary(s):
    rot = s.get("plan")
    if rot is None:
        from matricxon_amd.rotary import HipRotary

        case = s["case"]
        scaling = None if case["scaling"] == "none" else {"type": case["scaling"], "factor": case["factor"],
                                                          "original_context": case["context"]}
        rot = s["plan"] = HipRotary(case["dim"], rotary_dim=case["rot"], base=BASE, interleaved=case["interleaved"],
                                    scaling=scaling, device=s["q"].device)
    return rot(s["q"], s["k"], s["positions"])


def _own_moe(s):
    case, layer = s["case"], s.get("plan")
    if layer is None:
        from matricxon_amd.moe import HipPackedMoEExperts

        layer = s["plan"] = HipPackedMoEExperts(s["gate"], s["up"], s["down"], case["type"], case["type"], case["down"],
                                                case["embd"], case["ffn"], torch.nn.functional.silu, torch.bfloat16)
    # the codes' scales as the plain form's torch operations round them
    return layer.forward_logits(s["x"], s["logits"], case["top_k"], norm_topk=case["norm_topk"], scale=case["scale"],
                                q8k_scale="reciprocal")


def run(state):
    op = state["case"]["op"]
    if own:
        return {"norm": _own_norm, "rotary": _own_rotary, "moe": _own_moe}[op](state)
    return {"norm": _plain_norm, "rotary": _plain_rotary, "moe": _plain_moe}[op](state)


# ------------------------------------------------------------------------------------ the work
def work(case):
    if case["op"] == "norm":
        m, k = case["m"], case["k"]
        size = lambda t: 2 if t == "bf16" else 4  # noqa: E731
        gate = {"none": 0, "scalar": 1, "channel": k, "token": m, "full": m * k}[case["gate"]]
        weights = (2 if case["post"] else 1) * k + gate
        return {"bytes": (2 * m * k + weights) * size(case["x"]) + 2 * m * k * size(case["stream"]),
                "flops": (12 if case["post"] else 8) * m * k}
    if case["op"] == "rotary":
        n = case["t"] * (case["q_heads"] + case["kv_heads"])
        return {"bytes": 2 * n * case["dim"] * (2 if case["x"] == "bf16" else 4) + 8 * case["t"],
                "flops": 3 * n * case["rot"]}
    t, e, k, embd, ffn = (case[n] for n in ("t", "experts", "top_k", "embd", "ffn"))
    row = lambda type_, n: n // GEOMETRY[type_][0] * GEOMETRY[type_][1]  # noqa: E731
    touched = e * (1 - (1 - k / e) ** t)  # experts that some token goes to, on average
    expert = 2 * ffn * row(case["type"], embd) + embd * row(case["down"], ffn)
    return {"bytes": touched * expert + t * (4 * embd + 4 * e + 8 * k), "flops": 2.0 * t * k * 3 * embd * ffn}


# ----------------------------------------------------------------------- from the definition, in 64 bits
def _exact_norm(case, s):
    x, r, w = (s[n].double().cpu().numpy() for n in ("x", "r", "w"))
    if s["post"] is not None:
        x = x / np.sqrt(np.mean(x * x, axis=1, keepdims=True) + EPS) * s["post"].double().cpu().numpy()
    if s["gate"] is not None:
        x = x * s["gate"].double().cpu().numpy()
    h = r + case["scale"] * x
    # the next block's norm reads the stream as it is held
    held = torch.from_numpy(h).to(s["r"].dtype).double().numpy()
    return h, held / np.sqrt(np.mean(held * held, axis=1, keepdims=True) + EPS) * w


def _exact_frequency(case, i):
    """The angle per position of pair i."""
    d, factor, context = case["rot"], case["factor"], case["context"]
    if case["scaling"] == "ntk":
        return (BASE * factor ** (d / (d - 2))) ** (-2 * i / d)
    f = BASE ** (-2 * i / d)
    if case["scaling"] == "yarn":
        place = [d * math.log(context / (2 * math.pi * turns)) / math.log(BASE) / 2 for turns in (32, 1)]
        low, high = max(math.floor(place[0]), 0), min(math.ceil(place[1]), d - 1)
        kept = 1 - min(max((i - low) / max(high - low, 0.001), 0.0), 1.0)
    elif case["scaling"] == "llama3":
        kept = min(max((context * f / (2 * math.pi) - 1) / 3, 0.0), 1.0)
    else:
        kept = 0.0 if case["scaling"] == "linear" else 1.0
    return kept * f + (1 - kept) * f / factor


def _exact_rotary(case, s):
    d = case["rot"]
    m = 1 + math.log(case["factor"]) / 10 if case["scaling"] == "yarn" else 1.0
    f = np.array([_exact_frequency(case, i) for i in range(d // 2)], dtype=np.longdouble)
    angle = s["positions"].cpu().numpy().astype(np.longdouble)[:, None] * f[None, :]
    turn = (m * np.exp(1j * angle.astype(np.clongdouble))).astype(np.complex128)[:, None, :]
    out = []
    for x in (s["q"], s["k"]):
        v = x.double().cpu().numpy()
        first, second = (slice(0, d, 2), slice(1, d, 2)) if case["interleaved"] else (slice(0, d // 2), slice(d // 2, d))
        z = (v[..., first] + 1j * v[..., second]) * turn
        y = v.copy()
        y[..., first], y[..., second] = z.real, z.imag
        out.append(y)
    return tuple(out)


def _exact_weight(rows, type_):
    """(n, k) values of packed rows (n, row_bytes), in 64 bits, unpacked value by value of a block."""
    size, nbytes = GEOMETRY[type_]
    b = rows.reshape(-1, nbytes).to(torch.int16)
    half = lambda at: rows.reshape(-1, nbytes)[:, at : at + 2].contiguous().view(torch.float16).double()  # noqa: E731
    signed = lambda v: torch.where(v > 127, v - 256, v).double()  # noqa: E731
    out = torch.empty(b.shape[0], size, dtype=torch.float64, device=rows.device)
    for j in range(size // 32):
        if type_ == Q8_0:
            out[:] = half(0) * signed(b[:, 2:])
        elif type_ == Q4_K:
            if j < 4:
                sc, mn = b[:, 4 + j] % 64, b[:, 8 + j] % 64
            else:
                sc, mn = b[:, 8 + j] % 16 + b[:, j] // 64 * 16, b[:, 8 + j] // 16 + b[:, 4 + j] // 64 * 16
            q = b[:, 16 + 32 * (j // 2) : 48 + 32 * (j // 2)] // (16 if j % 2 else 1) % 16
            out[:, 32 * j : 32 * j + 32] = half(0) * sc[:, None].double() * q.double() - half(2) * mn[:, None].double()
        else:
            h, g = divmod(j, 4)
            q = b[:, 64 * h + 32 * (g % 2) :][:, :32] // (16 if g > 1 else 1) % 16 + b[:, 128 + 32 * h :][:, :32] // 4**g % 4 * 16
            sc = signed(b[:, 192 + 2 * j : 194 + 2 * j]).repeat_interleave(16, 1)
            out[:, 32 * j : 32 * j + 32] = half(208) * sc * (q.double() - 32)
    return out.view(rows.shape[0], -1)


def _exact_q8k(v):
    """A vector through Q8_K blocks: the scales 127 / top and top / 127 are float32 by the block's definition."""
    b = v.float().view(-1, 256)
    top = b.abs().max(dim=1, keepdim=True).values
    q = torch.where(top == 0, torch.zeros_like(b), torch.round(b * (127.0 / top)))
    return (q.double() * (top / 127.0).double()).view(-1)


def _exact_moe(case, s):
    logits = s["logits"].double().cpu().numpy()
    t, k = case["t"], case["top_k"]
    ids, weights = np.full((t, k), -1, dtype=np.int32), np.zeros((t, k))
    out = torch.zeros(t, case["embd"], dtype=torch.float64, device=s["x"].device)
    held = lambda v: v.to(torch.bfloat16).double()  # noqa: E731
    for i in range(t):
        best = sorted((e for e in range(case["experts"]) if logits[i, e] > -math.inf), key=lambda e: (-logits[i, e], e))
        chosen = best[:k]
        total = sum(math.exp(logits[i, e] - logits[i, best[0]]) for e in (chosen if case["norm_topk"] else best))
        x = _exact_q8k(s["x"][i])
        for j, e in enumerate(chosen):
            ids[i, j], weights[i, j] = e, math.exp(logits[i, e] - logits[i, best[0]]) / total * case["scale"]
            gate, up = (held(_exact_weight(s[n][e], case["type"]) @ x) for n in ("gate", "up"))
            act = held(held(gate / (1 + torch.exp(-gate))) * up)
            out[i] += weights[i, j] * held(_exact_weight(s["down"][e], case["down"]) @ _exact_q8k(act))
    return out, ids, weights


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "rotary": _exact_rotary, "moe": _exact_moe}[case["op"]](case, s)
