"""The attention half of a decoder layer on a paged cache of 4-bit keys and values, as measurable cases, each with a plain
form.

* `heads`: RMS norms of the heads of q and k and their rotary positions, in one pass:
      y = turn(x * rsqrt(mean(x^2) + eps) * w, p)
  over each head's values x, pair i of its rotary part turning by the angle p * f_i. `HipRotary` with head weights.
* `append`: the same for q and k, and k and v written to a paged cache in 4 bits. 32 neighbouring values of a token's head
  share a scale and a minimum, both float16:
      m = f16(min x), s = f16((max x - min x) / 15), code = clamp(round((x - m) / s), 0, 15), held value = s * code + m
  Token i of the n that a sequence gets goes to place length - n + i, and that is its position. `HipPagedCache.append`;
  the cached tokens come back as the values that they are held as, `HipPagedCache.read`.
* `attend`: causal attention of the last n tokens of each sequence over its cached keys and values, query heads in groups
  of one key head each, within a window or not: one token (a decode step), some, a prefill chunk, sequences of each in one
  call. `HipPagedCache.attend`.
* `step`: `append` and then `attend`, as a decode step does both.

A page holds `page` tokens of every key head in blocks of 32 tokens. A block of a head of D values (in W = D / 32 groups,
rounded up) is 40 * 32 * W bytes: codes of keys, scales of keys, codes of values, scales of values.
* Key codes: (token, octet c of 4, group, 4 bytes); byte y holds values 32 group + 8 c + 2 y (low bits) and the next.
* Key scales: (token, group) of (s, m).
* Value codes, a byte for a token's values 32 group + 2 i (low) and the next: (pair of groups, g of 4, i of 16, group of the
  pair, half h, z of 4), the token being 16 h + 4 g + z; a last odd group has the same order without a pair.
* Value scales: (group, quad of 4 tokens) of s of tokens 0, 2, 1, 3, then their m.
Entry j of a sequence's row of the page table is the page of its places from j * page on.

Sizes are those of the benchmark's layer (32 + 8 heads of 128) and of ranges around them.
"""

import math

import numpy as np
import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
EPS = 1e-6
BASE = 500000.0
HELD = 65000.0  # what lies beyond is held as this


# ------------------------------------------------------------------------------------ the cases
def heads(name, t, q_heads, kv_heads, dim, rot, x="bf16", interleaved=False, scaling="none", far=0, decode=False):
    return {"name": name, "op": "heads", "t": t, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "rot": rot, "x": x,
            "interleaved": interleaved, "scaling": scaling, "far": far, "decode": decode}


def paged(name, op, b, n, q_heads, kv_heads, dim, length, page=64, x="bf16", counts="each", lengths="full", window=0, rot=0,
          interleaved=False, norms=True):
    """b sequences of up to `length` tokens, the last n of each in this call ("each"), or b * n of all of them in parts of
    any size ("ragged"), or n of the first and one of each other ("mixed")."""
    return {"name": name, "op": op, "b": b, "n": n, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "length": length,
            "page": page, "x": x, "counts": counts, "lengths": lengths, "window": window, "rot": rot or dim,
            "interleaved": interleaved, "norms": norms}


def listed():
    return [
        # one token's heads: latency alone
        heads("heads_decode", 1, 32, 8, 128, 128, decode=True),
        # a prompt of odd length in float32, interleaved pairs over half of an 80 wide head
        heads("heads_odd_f32", 333, 12, 4, 80, 40, x="f32", interleaved=True),
        # a prefill chunk of a model with head norms and a long context
        heads("heads_prefill", 4096, 32, 8, 128, 128, scaling="llama3"),
        # sixteen replies, each at its own place: a token of each into its page
        paged("append_replies", "append", 16, 1, 32, 8, 128, 8192, lengths="spread"),
        # five prompts of any length in float32, three heads' worth of groups, half of a head turning, no norms
        paged("append_ragged_f32", "append", 5, 151, 8, 4, 96, 1500, page=32, x="f32", counts="ragged", lengths="spread",
              rot=48, norms=False),
        # a prefill chunk behind an odd number of cached tokens
        paged("append_prefill", "append", 1, 4096, 32, 8, 128, 5111),
        # one reply of a short conversation
        paged("attend_reply", "attend", 1, 1, 32, 8, 128, 1000),
        # one reply at the end of a long document: few heads, a long axis
        paged("attend_long", "attend", 1, 1, 32, 8, 128, 131072, page=256),
        # the scheduler's full batch, replies of every length
        paged("attend_batch", "attend", 64, 1, 32, 8, 128, 16384, lengths="spread"),
        # a prompt's chunk beside three replies, within a window, narrow heads in groups of five
        paged("attend_mixed_window", "attend", 4, 512, 40, 8, 64, 3000, page=32, counts="mixed", lengths="spread", window=1024),
        # a prefill chunk of a long prompt
        paged("attend_prefill", "attend", 1, 2048, 32, 8, 128, 8192),
        # a decode step of sixteen replies: the token's keys and values appended, then attention
        paged("step_replies", "step", 16, 1, 32, 8, 128, 4096, lengths="spread"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["heads", "append", "attend", "attend", "step"])
    dim = rng.choice([32, 64, 80, 96, 128, 128, 192, 256])
    kv = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 4, 4, 5, 8, 16])
    rot = rng.choice([dim, dim, dim // 2, 2 * rng.randint(2, dim // 2)])
    x = rng.choice(["bf16", "bf16", "f32"]) if op in ("heads", "append") else "bf16"
    wide = kv * dim / 1024  # 1: the listed cases' width
    if op == "heads":
        c = heads("", _log(rng, 1, min(4096, int(4096 * 40 / (kv * (group + 1)) * 128 / dim))), kv * group, kv, dim, rot, x,
                  rng.random() < 0.4, rng.choice(["none", "llama3"]), rng.choice([0, 1 << 20]), rng.random() < 0.3)
    else:
        page = rng.choice([32, 64, 64, 128, 256])
        counts = rng.choice(["each", "each", "ragged", "mixed"])
        lengths = rng.choice(["full", "spread"])
        if op == "append":
            b = _log(rng, 1, 32)
            n = _log(rng, 1, max(1, int(2048 / b / max(wide * (group + 2) / 6, 0.25))))
            length = n * (b if counts == "ragged" else 1) + _log(rng, 1, 8192)
        elif op == "step" or rng.random() < 0.5:  # a decode step: few tokens of many replies
            b, counts = _log(rng, 1, 64), "each"
            n = 1 if op == "step" else rng.choice([1, 1, 1, 2, 4])
            length = max(n, _log(rng, 1, min(131072, int(400000 / b / max(wide, 0.25)))))
        else:  # a chunk
            b = _log(rng, 1, 4)
            n = _log(rng, 2, max(2, int(1024 / b)))
            most = int(8192 / max(wide * group / 4, 0.5))
            length = n * (b if counts == "ragged" else 1) + _log(rng, 1, max(1, most - n * b))
        c = paged("", op, b, n, kv * group, kv, dim, length, page, x, counts, lengths,
                  rng.choice([0, 0, 0, _log(rng, 1, 2048)]) if op != "append" else 0, rot, rng.random() < 0.3, rng.random() < 0.7)
    del c["name"]
    return c


# --------------------------------------------------------------------------------------- inputs
def _groups(dim):
    return (dim + 31) // 32


def _columns(g, t, hq, hk, dim, x):
    """q, k and v as a fused q | k | v projection leaves them: columns of one buffer."""
    qkv = torch.randn(t, (hq + 2 * hk) * dim, device="cuda", generator=g)
    # some channels of keys are far above the rest
    qkv[:, hq * dim : (hq + hk) * dim] *= torch.exp(0.5 * torch.randn(hk * dim, device="cuda", generator=g))
    q, k, v = torch.split(qkv.to(TYPES[x]), [hq * dim, hk * dim, hk * dim], dim=-1)
    return q.view(t, hq, dim), k.view(t, hk, dim), v.view(t, hk, dim)


def _weights(case, g):
    one = lambda: (1 + 0.2 * torch.randn(case["dim"], device="cuda", generator=g)).to(TYPES[case["x"]])  # noqa: E731
    return (one(), one()) if case.get("norms", True) else (None, None)


def _prepare_heads(case, g):
    t, far = case["t"], case["far"]
    q, k, _ = _columns(g, t, case["q_heads"], case["kv_heads"], case["dim"], case["x"])
    if case["decode"]:  # replies of different lengths
        positions = torch.randint(0, max(far, 8192), (t,), device="cuda", generator=g)
    else:
        positions = torch.arange(t, device="cuda") + far // 2
    qw, kw = _weights(case, g)
    return {"q": q, "k": k, "positions": positions, "qw": qw, "kw": kw}


def _counts(case, host):
    """How many tokens of each sequence are in the call."""
    b, n = case["b"], case["n"]
    if case["counts"] == "mixed":
        return [n] + [1] * (b - 1)
    if case["counts"] == "ragged":
        cuts = sorted(torch.randint(0, b * n + 1, (b - 1,), generator=host).tolist())
        return [v - u for u, v in zip([0] + cuts, cuts + [b * n])]
    return [n] * b


def _random_pages(case, g, n_pages):
    """Pages of cached tokens: scales and minima of keys and values of about unit size, every code."""
    w = _groups(case["dim"])
    blocks = n_pages * case["kv_heads"] * (case["page"] // 32)
    raw = torch.randint(0, 256, (blocks, 1280 * w), dtype=torch.uint8, device="cuda", generator=g)
    for at, key in ((512 * w, True), (1152 * w, False)):
        s = 0.2 * torch.exp(0.3 * torch.randn(blocks, 32 * w, device="cuda", generator=g))
        m = s * (0.5 * torch.randn(blocks, 32 * w, device="cuda", generator=g) - 7.5)
        pair = torch.stack((s, m), -1) if key else torch.stack((s.view(blocks, -1, 4), m.view(blocks, -1, 4)), -2)
        raw[:, at : at + 128 * w] = pair.to(torch.float16).reshape(blocks, -1).view(torch.uint8)
    return raw.view(n_pages, case["kv_heads"], case["page"] // 32, 1280 * w)


def _prepare_paged(case, g, seed):
    host = torch.Generator().manual_seed(seed)
    b, most, page = case["b"], case["length"], case["page"]
    counts = _counts(case, host)
    lengths = [most] * b
    if case["lengths"] == "spread":
        lengths = [max(c, int(torch.randint(most // 8, most + 1, (1,), generator=host))) for c in counts]
        lengths[-1] = max(counts[-1], most)
    width = -(-most // page)
    n_pages = b * width
    # pages in the order that a pool gives them out after some use, and nothing in the table behind a sequence's end
    table = torch.randperm(n_pages, device="cuda", generator=g).view(b, width).int()
    held = torch.tensor([-(-v // page) for v in lengths], device="cuda")
    table = torch.where(torch.arange(width, device="cuda") < held[:, None], table, -1).int()
    t = sum(counts)
    q, k, v = _columns(g, t, case["q_heads"], case["kv_heads"], case["dim"], case["x"])
    qw, kw = _weights(case, g)
    if case["op"] == "append":
        pages = torch.zeros(n_pages, case["kv_heads"], page // 32, 1280 * _groups(case["dim"]), dtype=torch.uint8, device="cuda")
    else:
        pages = _random_pages(case, g, n_pages)
        if case["op"] == "attend":  # as norms and training leave them: a few keys stand out
            q = (1.6 * q.float()).to(q.dtype)
    starts = None
    if case["counts"] != "each":
        starts = torch.tensor([0] + list(np.cumsum(counts)), dtype=torch.int32, device="cuda")
    return {"q": q, "k": k, "v": v, "qw": qw, "kw": kw, "pages": pages, "table": table, "counts": counts, "starts": starts,
            "lengths": torch.tensor(lengths, dtype=torch.int32, device="cuda")}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return {"case": case, **(_prepare_heads(case, g) if case["op"] == "heads" else _prepare_paged(case, g, seed))}


# --------------------------------------------------------------------------------- plain forms
def _frequencies(case, device):
    """The angle per position of each pair, in 64 bits."""
    d = case["rot"]
    f = BASE ** (-2 * torch.arange(d // 2, dtype=torch.float64, device=device) / d)
    if case.get("scaling") == "llama3":  # by the turns that a context holds: 4 and more kept, 1 and fewer stretched
        s = ((8192 * f / (2 * math.pi) - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        return (1 - s) * f / 8.0 + s * f
    return f


def _plain_head(case, x, w, positions):
    """Norm and rotation of x (T, heads, dim), in float32."""
    x = x.float()
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
    angle = (positions.double()[:, None] * _frequencies(case, x.device))[:, None, :]
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    d = case["rot"]
    if case["interleaved"]:
        a, b = x[..., 0:d:2], x[..., 1:d:2]
        r = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    else:
        a, b = x[..., : d // 2], x[..., d // 2 : d]
        r = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    return torch.cat((r, x[..., d:]), -1)


def _plain_held(x):
    """The values that x (..., dim) is held as in 4 bits."""
    d = x.shape[-1]
    full, rest = d // 32 * 32, d % 32
    out = []
    for part, size in ((x[..., :full], 32), (x[..., full:], rest)):
        if part.shape[-1]:
            v = part.clamp(-HELD, HELD).unflatten(-1, (-1, size))
            low, high = v.amin(-1, keepdim=True), v.amax(-1, keepdim=True)
            m, s = low.half().float(), ((high - low) / 15).half().float()
            c = torch.where(s > 0, torch.round((v - m) / torch.where(s > 0, s, 1.0)).clamp(0, 15), 0.0)
            out.append((c * s + m).flatten(-2))
    return torch.cat(out, -1)


def _plain_places(s):
    """The sequence and the place of each of the call's tokens."""
    counts = torch.tensor(s["counts"], device="cuda")
    seq = torch.repeat_interleave(torch.arange(len(s["counts"]), device="cuda"), counts, output_size=sum(s["counts"]))
    first = torch.cumsum(counts, 0) - counts
    return seq, s["lengths"].long()[seq] - counts[seq] + torch.arange(seq.numel(), device="cuda") - first[seq]


def _plain_pages(case, s):
    """Keys and values (b, kv_heads, places, dim) of the sequences' pages, in float32."""
    w, dim, pages = _groups(case["dim"]), case["dim"], s["pages"]
    raw = pages[s["table"].clamp(min=0).long()]  # (b, table entries, heads, blocks, bytes)
    raw = raw.permute(0, 2, 1, 3, 4).flatten(2, 3)  # (b, heads, blocks, bytes)
    lead = raw.shape[:3]
    split = [512 * w, 128 * w, 512 * w, 128 * w]
    kc, ks, vc, vs = (p.contiguous() for p in torch.split(raw, split, dim=-1))
    nibbles = lambda c: torch.stack((c & 15, c >> 4), -1).float()  # noqa: E731
    scale = ks.view(torch.float16).float().view(*lead, 32, w, 1, 2)
    codes = nibbles(kc.view(*lead, 32, 4, w, 4)).transpose(-4, -3).reshape(*lead, 32, w, 32)
    keys = (codes * scale[..., 0] + scale[..., 1]).reshape(*lead[:2], -1, 32 * w)[..., :dim]
    pairs, one = w // 2, w % 2
    parts = []
    for c, each in ((vc[..., : pairs * 1024].reshape(*lead, pairs, 4, 16, 2, 2, 4), 2),
                    (vc[..., pairs * 1024 :].reshape(*lead, one, 4, 16, 1, 2, 4), 1)):
        # (pair, g, i, group, h, z, value of the byte) -> (h, g, z, pair, group, i, value)
        v = nibbles(c).permute(0, 1, 2, 7, 4, 8, 3, 6, 5, 9)
        parts.append(v.reshape(*lead, 32, each * c.shape[3], 32))
    codes = torch.cat(parts, -2)
    scale = vs.view(torch.float16).float().view(*lead, w, 8, 2, 2, 2)  # (group, quad, s or m, token % 2, token / 2 % 2)
    scale = scale.permute(0, 1, 2, 4, 7, 6, 3, 5).reshape(*lead, 32, w, 1, 2)
    values = (codes * scale[..., 0] + scale[..., 1]).reshape(*lead[:2], -1, 32 * w)[..., :dim]
    return keys, values


def _plain_attention(case, s, q, keys, values):
    """q (T, heads, dim) over keys and values (b, kv_heads, places, dim)."""
    counts, kv, dim = s["counts"], case["kv_heads"], case["dim"]
    b, n, group = case["b"], max(s["counts"]), case["q_heads"] // case["kv_heads"]
    seq, place = _plain_places(s)
    row = place - s["lengths"].long()[seq] + torch.tensor(counts, device="cuda")[seq]  # the token's number in its sequence
    padded = torch.zeros(b, n, case["q_heads"], dim, device="cuda")
    padded[seq, row] = q.float()
    at = torch.full((b, n), -1, device="cuda")
    at[seq, row] = place
    padded = padded.view(b, n, kv, group, dim).permute(0, 2, 3, 1, 4).reshape(b, kv, group * n, dim)
    scores = torch.matmul(padded, keys.transpose(-1, -2)).view(b, kv, group, n, -1) / math.sqrt(dim)
    places = torch.arange(keys.shape[2], device="cuda")
    seen = places <= at[..., None]
    if case["window"]:
        seen &= places > at[..., None] - case["window"]
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul((p / torch.where(total > 0, total, 1.0)).view(b, kv, group * n, -1), values)
    out = out.view(b, kv, group, n, dim).permute(0, 3, 1, 2, 4).reshape(b, n, case["q_heads"], dim)
    return out[seq, row].to(s["q"].dtype)


def _plain(s):
    case, op = s["case"], s["case"]["op"]
    if op == "heads":
        return tuple(_plain_head(case, s[n], s[n + "w"], s["positions"]).to(s[n].dtype) for n in ("q", "k"))
    if op == "attend":
        return _plain_attention(case, s, s["q"], *_plain_pages(case, s))
    seq, place = _plain_places(s)
    q = _plain_head(case, s["q"], s["qw"], place).to(s["q"].dtype)
    k, v = _plain_held(_plain_head(case, s["k"], s["kw"], place)), _plain_held(s["v"].float())
    if op == "append":
        return q, k.bfloat16(), v.bfloat16()
    keys, values = _plain_pages(case, s)
    keys[seq, :, place], values[seq, :, place] = k, v
    return _plain_attention(case, s, q, keys, values)


# ----------------------------------------------------------------------- the framework's calls
def _plan(s):
    from matricxon_amd.rotary import HipRotary

    case, device = s["case"], s["q"].device
    scaling = {"type": "llama3", "factor": 8.0, "original_context": 8192} if case.get("scaling") == "llama3" else None
    rot = HipRotary(case["dim"], rotary_dim=case["rot"], base=BASE, interleaved=case["interleaved"], scaling=scaling,
                    device=device)
    if case["op"] == "heads":
        return rot, None
    from matricxon_amd.attention import HipPagedCache

    return rot, HipPagedCache(s["pages"].shape[0], case["page"], case["kv_heads"], case["dim"], pages=s["pages"])


def _own(s):
    case, op = s["case"], s["case"]["op"]
    rot, cache = s["plan"] if "plan" in s else s.setdefault("plan", _plan(s))
    if op == "heads":
        return rot(s["q"], s["k"], s["positions"], q_weight=s["qw"], k_weight=s["kw"], eps=EPS)
    where = (s["table"], s["lengths"], s["starts"])
    q = s["q"]
    if op != "attend":
        q = cache.append(q, s["k"], s["v"], *where, rotary=rot, q_weight=s["qw"], k_weight=s["kw"], eps=EPS)
    if op == "append":
        return (q, *cache.read(q.shape[0], *where))
    return cache.attend(q, *where, window=case["window"])


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------------------------ the work
def work(case):
    size = 2 if case["x"] == "bf16" else 4
    hq, hk, dim = case["q_heads"], case["kv_heads"], case["dim"]
    if case["op"] == "heads":
        n = case["t"] * (hq + hk) * dim
        return {"bytes": 2 * n * size + 8 * case["t"], "flops": 7 * n}
    b, n = case["b"], case["n"]
    t = n + b - 1 if case["counts"] == "mixed" else b * n
    held = 40 * _groups(dim)  # bytes of a token's key and value of a head
    w = {"bytes": 0, "flops": 0}
    if case["op"] != "attend":  # the step's q stays in hand between its halves
        w["bytes"] += t * ((hq + 2 * hk) * dim * size + hk * held)
        w["flops"] += t * (7 * (hq + hk) * dim + 6 * 2 * hk * dim)
        if case["op"] == "append":
            w["bytes"] += t * (hq * dim * size + hk * (held + 4 * dim))
            return w
    most, window = case["length"], case["window"]
    spread = [most] if case["lengths"] == "full" else [most * (1 / 8 + 7 / 8 * (i + 0.5) / 16) for i in range(16)]
    parts = [(n, 1.0), (1, b - 1.0)] if case["counts"] == "mixed" else [(n, float(b))]
    for count, many in parts:
        for length in spread:
            length = max(length, count)
            far = min(length, window + count - 1) if window else length
            pairs = count * min(window, length) if window and length - count >= window else count * (length - (count - 1) / 2)
            w["bytes"] += many / len(spread) * far * hk * held
            w["flops"] += many / len(spread) * 4 * pairs * hq * dim
    w["bytes"] += t * hq * dim * 2 * (1 if case["op"] == "step" else 2)
    return w


# ----------------------------------------------------------------------- from the definition, in 64 bits
def _exact_head(case, x, w, positions):
    d = case["rot"]
    x = x.double().cpu().numpy()
    if w is not None:
        x = x / np.sqrt(np.mean(x * x, axis=-1, keepdims=True) + EPS) * w.double().cpu().numpy()
    f = np.array([BASE ** (-2 * i / d) for i in range(d // 2)], dtype=np.longdouble)
    if case.get("scaling") == "llama3":
        kept = np.clip((8192 * f / (2 * np.pi) - 1) / 3, 0, 1)
        f = kept * f + (1 - kept) * f / 8
    angle = np.asarray(positions).astype(np.longdouble)[:, None] * f[None, :]
    turn = np.exp(1j * angle.astype(np.clongdouble)).astype(np.complex128)[:, None, :]
    first, second = (slice(0, d, 2), slice(1, d, 2)) if case["interleaved"] else (slice(0, d // 2), slice(d // 2, d))
    z = (x[..., first] + 1j * x[..., second]) * turn
    y = x.copy()
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _exact_held(x):
    """Group by group: the scale and the minimum are float16 by the format's definition."""
    y = np.empty_like(x)
    for at in range(0, x.shape[-1], 32):
        v = np.clip(x[..., at : at + 32], -HELD, HELD)
        low, high = v.min(-1, keepdims=True), v.max(-1, keepdims=True)
        m = low.astype(np.float16).astype(np.float64)
        s = ((high - low) / 15).astype(np.float16).astype(np.float64)
        safe = np.where(s > 0, s, 1.0)
        y[..., at : at + 32] = np.where(s > 0, np.clip(np.rint((v - m) / safe), 0, 15), 0) * s + m
    return y


def _exact_places(s):
    out = []
    for b, (count, length) in enumerate(zip(s["counts"], s["lengths"].tolist())):
        out += [(b, length - count + i) for i in range(count)]
    return out


def _exact_cached(case, s, b, length):
    """Keys and values (places, kv_heads, dim) of one sequence in float64, each looked up by the address of its code."""
    dim, page, w = case["dim"], case["page"], _groups(case["dim"])
    place, d = torch.arange(length, device="cuda")[:, None], torch.arange(dim, device="cuda")[None, :]
    token, g = place % 32, d // 32
    block = s["table"][b].long()[place // page] * case["kv_heads"] * (page // 32) + place % page // 32
    heads_ = torch.arange(case["kv_heads"], device="cuda")[:, None, None] * (page // 32)
    base = (block + heads_) * (1280 * w)
    raw = s["pages"].view(-1)
    halves = raw.view(torch.float16)
    held = lambda code, shift, s_at, m_at: (  # noqa: E731
        ((raw[base + code].long() >> shift) & 15).double() * halves[(base + s_at) // 2].double() + halves[(base + m_at) // 2].double())
    shift = d % 2 * 4
    key_scale = 512 * w + (token * w + g) * 4
    keys = held(token * 16 * w + d % 32 // 8 * 4 * w + g * 4 + d % 8 // 2, shift, key_scale, key_scale + 2)
    h, quad, z, i = token // 16, token // 4 % 4, token % 4, d % 32 // 2
    paired = g // 2 * 1024 + (quad * 16 + i) * 16 + g % 2 * 8 + h * 4 + z
    last = w // 2 * 1024 + (quad * 16 + i) * 8 + h * 4 + z
    code = 640 * w + torch.where(g < w // 2 * 2, paired, last)
    slot = 1152 * w + (g * 8 + token // 4) * 16 + (z % 2 * 2 + z // 2) * 2
    values = held(code, shift, slot, slot + 8)
    return keys, values  # (kv_heads, places, dim)


def _exact_attention(case, s, q, new=None):
    q = torch.as_tensor(q, dtype=torch.float64, device="cuda")
    group, out, at = case["q_heads"] // case["kv_heads"], torch.zeros_like(q), 0
    for b, (count, length) in enumerate(zip(s["counts"], s["lengths"].tolist())):
        if count == 0:
            continue
        keys, values = _exact_cached(case, s, b, length)
        if new is not None:
            for mine, theirs in ((keys, new[0]), (values, new[1])):
                mine[:, length - count :] = torch.as_tensor(theirs[at : at + count], device="cuda").transpose(0, 1)
        place = torch.arange(length - count, length, device="cuda")[:, None]
        hidden = torch.arange(length, device="cuda") > place
        if case["window"]:
            hidden |= torch.arange(length, device="cuda") <= place - case["window"]
        for h in range(case["q_heads"]):
            score = q[at : at + count, h] @ keys[h // group].T / math.sqrt(case["dim"])
            out[at : at + count, h] = torch.softmax(score.masked_fill(hidden, -math.inf), -1) @ values[h // group]
        at += count
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "heads":
        return tuple(_exact_head(case, s[n], s[n + "w"], s["positions"].cpu().numpy()) for n in ("q", "k"))
    if case["op"] == "attend":
        return _exact_attention(case, s, s["q"].double())
    place = np.array([p for _, p in _exact_places(s)])
    q = _exact_head(case, s["q"], s["qw"], place)
    k, v = _exact_held(_exact_head(case, s["k"], s["kw"], place)), _exact_held(s["v"].double().cpu().numpy())
    if case["op"] == "append":
        return q, k, v
    held = torch.from_numpy(q).to(s["q"].dtype)  # attention reads the turned q as it is held
    return _exact_attention(case, s, held.double(), (k, v))
