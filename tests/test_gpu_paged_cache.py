"""`HipPagedCache`: what is appended and read back, and attention over it, against 64-bit arithmetic.

Appending. The held values follow from the float32 values by exact steps (two roundings to float16, one division, one
rounding to a code), so that rows that are neither normed nor turned are held to the same bits as a restatement of the
format in float32; keys that are normed and turned are held as what `HipRotary` gives for them in float32 is held
(test_gpu_head_norm.py holds that to the formula).

Attention, with h = 2^-11 half a step of float16 and e = 2^-24 one of float32, against the held values in 64 bits:
* a key is widened with one rounding, so a score is off by scale * sum |q k| (h + (dim + 2) e); q itself is exact in
  float16 but for values below 2^-24 of the row's largest, half a step of which is 2^-35 of that: scale * top * sum |k|
  2^-35; float16's subnormal keys add 2^-25 * scale * sum |q|.
* exp of a score that is off by d is off by e^d - 1; the scaled difference to the maximum (at most some 200 where p counts)
  and the exponential add 200 e + 2 e; p is rounded to float16 (h, or 2^-25 of 2^8 where it is subnormal), a value's
  widening is one rounding (h, and 2^-25), the sums in float32 add (places + 32) e.
* the output is rounded to bfloat16: 2^-8 of itself.
With E the largest of a row's score errors the output is within (e^(2 E) - 1 + 2.1 h + (places + 300) e) sum p |v| / sum p
+ 2^-33 sum |v| / sum p' + 2^-25 + 2^-8 |o|, p' = p / max p."""

import math

import pytest
import torch

from matricxon_amd.attention import HipPagedCache
from matricxon_amd.rotary import HipRotary

pytestmark = pytest.mark.gpu

F32, BF16, F64 = torch.float32, torch.bfloat16, torch.float64
H16, E32 = 2.0 ** -11, 2.0 ** -24


def rand(g, *shape, dt=F32):
    return torch.randn(*shape, device="cuda", generator=g).to(dt)


def same(a, b):
    return bool((a == b).all()) and a.shape == b.shape and a.dtype == b.dtype


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def held(x):
    """The format in float32: what x (..., dim) is held as. Quotients are formed in float64 and rounded, which gives
    float32's own (torch multiplies by 1 / 15 where it divides a float32 tensor by 15)."""
    out = []
    for at in range(0, x.shape[-1], 32):
        v = x[..., at : at + 32].float()
        v = torch.where(v.isnan(), 0.0, v).clamp(-65000.0, 65000.0)
        low, high = v.amin(-1, keepdim=True), v.amax(-1, keepdim=True)
        m, s = low.half().float(), ((high - low).double() / 15).float().half().float()
        code = ((v - m).double() / torch.where(s > 0, s, 1.0).double()).float()
        c = torch.where(s > 0, torch.round(code).clamp(0, 15), 0.0)
        out.append((c.double() * s.double() + m.double()).float())
    return torch.cat(out, -1)


def a_table(g, b, width, spare=0):
    """Pages in any order, and how many there are."""
    n = b * width + spare
    return torch.randperm(n, device="cuda", generator=g)[: b * width].view(b, width).int(), n


def rows_of(counts, lengths):
    """(sequence, place) of each row."""
    return [(b, n - c + i) for b, (c, n) in enumerate(zip(counts, lengths)) for i in range(c)]


def starts_of(counts):
    out = [0]
    for c in counts:
        out.append(out[-1] + c)
    return i32(out)


# ------------------------------------------------------------------------------- appending, reading
@pytest.mark.parametrize("dim", [8, 32, 40, 64, 96, 128, 160, 200, 256])
@pytest.mark.parametrize("dt", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("counts,lengths", [([1], [1]), ([1, 1, 1], [7, 32, 33]), ([5, 0, 70, 3], [5, 9, 99, 67]),
                                            ([600], [633])], ids=["one", "replies", "ragged", "chunk"])
def test_held_values(gpu, dim, dt, counts, lengths) -> None:
    g = torch.Generator(device="cuda").manual_seed(dim)
    page, heads, b, t = 64, 3, len(counts), sum(counts)
    table, n = a_table(g, b, -(-max(lengths) // page), 2)
    cache = HipPagedCache(n, page, heads, dim)
    cache.pages.random_(0, 256, generator=g)  # as another sequence left them
    before = cache.pages.clone()
    k, v = 3 * rand(g, t, heads, dim, dt=dt), (rand(g, t, heads, dim) + 5).to(dt)
    assert cache.append(None, k, v, table, i32(lengths), starts_of(counts)) is None
    for out in (F32, BF16):
        k2, v2 = cache.read(t, table, i32(lengths), starts_of(counts), dtype=out)
        assert same(k2, held(k).to(out)) and same(v2, held(v).to(out))
    # earlier tokens of the same blocks are what they were, and so are pages of no token
    others = [x - c for x, c in zip(lengths, counts)]
    if sum(others) > 0:
        where = sum(others), table, i32(others), starts_of(others)
        was = HipPagedCache(n, page, heads, dim, pages=before).read(*where, dtype=F32)
        assert all(same(a.nan_to_num(), c.nan_to_num()) for a, c in zip(cache.read(*where, dtype=F32), was))
    changed = (cache.pages != before).flatten(1).any(1).nonzero().flatten().tolist()
    written = {int(table[s, p // page]) for s, p in rows_of(counts, lengths)}
    assert set(changed) <= written


@pytest.mark.parametrize("n", [1, 4, 37])
def test_appending_in_parts_gives_the_same_pages(gpu, n) -> None:
    """Token by token, some at a time and all at once: the same bytes."""
    g = torch.Generator(device="cuda").manual_seed(n)
    total, heads, dim = 111, 2, 96
    table = i32([[3, 0, 2, 1]])
    rot = HipRotary(dim)
    q, k, v = rand(g, total, 4, dim, dt=BF16), rand(g, total, heads, dim, dt=BF16), rand(g, total, heads, dim, dt=BF16)
    w = (1 + 0.2 * rand(g, dim)).to(BF16)
    whole, parts = HipPagedCache(4, 32, heads, dim), HipPagedCache(4, 32, heads, dim)
    want = whole.append(q, k, v, table, i32([total]), rotary=rot, q_weight=w, k_weight=w)
    got = [parts.append(q[i : i + n], k[i : i + n], v[i : i + n], table, i32([min(i + n, total)]), rotary=rot, q_weight=w,
                        k_weight=w) for i in range(0, total, n)]
    assert same(torch.cat(got), want) and same(whole.pages, parts.pages)


@pytest.mark.parametrize("dim,rot_dim,interleaved", [(128, 128, False), (128, 128, True), (128, 64, False), (96, 96, False),
                                                     (80, 50, False), (64, 36, True), (256, 256, False), (40, 10, True)])
@pytest.mark.parametrize("norms", [False, True])
def test_normed_and_turned(gpu, dim, rot_dim, interleaved, norms) -> None:
    """q as HipRotary gives it, keys held as its float32 result is; positions are the places, or given."""
    g = torch.Generator(device="cuda").manual_seed(dim)
    counts, lengths, hq, hk = [9, 1, 4], [9, 50, 64], 4, 2
    t, table = sum(counts), a_table(g, 3, 2)[0]
    rot = HipRotary(dim, rotary_dim=rot_dim, interleaved=interleaved)
    q, k, v = rand(g, t, hq, dim), 2 * rand(g, t, hk, dim), rand(g, t, hk, dim)
    weights = {"q_weight": 1 + 0.3 * rand(g, dim), "k_weight": 1 + 0.3 * rand(g, dim)} if norms else {}
    places = torch.tensor([p for _, p in rows_of(counts, lengths)], device="cuda")
    for given in (None, places + 12345, (places - 20).int()):
        cache = HipPagedCache(6, 32, hk, dim)
        q2 = cache.append(q, k, v, table, i32(lengths), starts_of(counts), rotary=rot, positions=given, eps=1e-5, **weights)
        want_q, want_k = rot(q, k, places if given is None else given, eps=1e-5, **weights)
        k2, v2 = cache.read(t, table, i32(lengths), starts_of(counts), dtype=F32)
        assert same(q2, want_q)
        assert same(k2, held(want_k)) and same(v2, held(v))


def test_head_norms_without_rotation(gpu) -> None:
    g = torch.Generator(device="cuda").manual_seed(3)
    q, k = rand(g, 5, 4, 64), rand(g, 5, 2, 64)
    w = 1 + 0.3 * rand(g, 64)
    cache = HipPagedCache(1, 32, 2, 64)
    q2 = cache.append(q, k, k, i32([[0]]), i32([5]), q_weight=w, k_weight=w)
    rot = HipRotary(64, interleaved=True)  # at position 0 nothing turns, and squares are added up in the same order
    want = rot(q, k, torch.zeros(5, dtype=torch.int32, device="cuda"), q_weight=w, k_weight=w)
    assert same(q2, want[0]) and same(cache.read(5, i32([[0]]), i32([5]), dtype=F32)[0], held(want[1]))


def test_batched_inputs_and_strides(gpu) -> None:
    """(B, T, heads, dim) as columns of a q | k | v buffer that starts off a 16-byte boundary."""
    g = torch.Generator(device="cuda").manual_seed(4)
    b, n, hq, hk, dim = 2, 3, 4, 2, 64
    qkv = rand(g, b, n, (hq + 2 * hk) * dim + 2, dt=BF16)
    q, k, v = (x.unflatten(-1, (-1, dim)) for x in torch.split(qkv[..., 1:-1], [hq * dim, hk * dim, hk * dim], dim=-1))
    table, lengths = i32([[1, 2], [3, 0]]), i32([3, 35])
    rot = HipRotary(dim)
    one, two = HipPagedCache(4, 32, hk, dim), HipPagedCache(4, 32, hk, dim)
    q2 = one.append(q, k, v, table, lengths, rotary=rot)
    q3 = two.append(*(x.flatten(0, 1).contiguous() for x in (q, k, v)), table, lengths, rotary=rot)
    assert q2.shape == q.shape and same(q2.flatten(0, 1), q3) and same(one.pages, two.pages)
    wide = torch.stack((torch.zeros_like(table), table), -1).flatten(1)[:, 1:]  # rows of a wider table
    assert wide.stride(1) == 1
    three = HipPagedCache(4, 32, hk, dim)
    three.append(q, k, v, torch.cat((table, table), 1)[:, :2], lengths, rotary=rot)
    assert same(one.pages, three.pages)


def test_values_that_have_no_code(gpu) -> None:
    """Constant groups, zeros, NaN, infinities and what passes float16: held finite, and within its own group."""
    x = torch.zeros(6, 1, 64, device="cuda")
    x[0] = 3.25
    x[1, 0, 3] = math.nan
    x[2, 0, 40:] = math.inf
    x[3, 0, :32], x[3, 0, 5] = -1e30, 7e4
    x[4] = torch.linspace(-1, 1, 64, device="cuda")
    x[5, 0, 0] = 1e-30
    cache = HipPagedCache(1, 32, 1, 64)
    cache.append(None, x, x.flip(0), i32([[0]]), i32([6]))
    k, v = cache.read(6, i32([[0]]), i32([6]), dtype=F32)
    assert same(k, held(x)) and same(v, held(x.flip(0)))
    assert k.isfinite().all() and (k[0] == 3.25).all() and (k[1] == 0).all() and (k[2, 0, :32] == 0).all()


def test_places_without_a_page(gpu) -> None:
    """A page number that is none, places behind the table, places before 0: nothing is written, zeros are read."""
    g = torch.Generator(device="cuda").manual_seed(6)
    table, lengths, counts = i32([[1, -1, 0], [2, 99, 3], [1 << 30, 4, -5]]), [70, 100, 2], [70, 40, 5]
    t = sum(counts)
    cache = HipPagedCache(5, 32, 2, 64)
    q, k, v = rand(g, t, 2, 64), rand(g, t, 2, 64), rand(g, t, 2, 64)
    q2 = cache.append(q, k, v, table, i32(lengths), starts_of(counts), rotary=HipRotary(64))
    assert q2.isfinite().all()
    k2, v2 = cache.read(t, table, i32(lengths), starts_of(counts), dtype=F32)
    for row, (b, p) in enumerate(rows_of(counts, lengths)):
        cached = p >= 0 and p // 32 < 3 and 0 <= int(table[b, p // 32]) < 5
        want = torch.zeros(2, 64, device="cuda")
        assert same(v2[row], held(v[row]) if cached else want), (b, p)
    # of page 4 nothing was written
    assert (cache.pages[4] == 0).all()


def test_rows_of_no_sequence(gpu) -> None:
    g = torch.Generator(device="cuda").manual_seed(7)
    q, k = rand(g, 12, 2, 64, dt=BF16), rand(g, 12, 2, 64, dt=BF16)
    table, lengths, starts = i32([[0], [1]]), i32([3, 4]), i32([2, 5, 9])  # rows 0, 1, 9, 10 and 11 are of none
    cache = HipPagedCache(2, 32, 2, 64)
    q2 = cache.append(q, k, k, table, lengths, starts, rotary=HipRotary(64))
    k2, _ = cache.read(12, table, lengths, starts)
    out = torch.full_like(q, 7.0)
    cache.attend(q2, table, lengths, starts, out=out)
    fresh = cache.attend(q2, table, lengths, starts)
    none = [0, 1, 9, 10, 11]
    assert (q2[none] == 0).all() and (k2[none] == 0).all() and (out[none] == 7).all() and (fresh[none] == 0).all()
    assert same(out[2:9], fresh[2:9]) and (q2[2:9] != 0).any(-1).all()


# ------------------------------------------------------------------------------------- attention
def check_attention(cache, q, got, table, lengths, counts, scale=None, window=0, rows=None):
    """got against the held values; counts, lengths: lists; rows: the first row of each sequence (adjacent unless given)."""
    dim, hq = q.shape[-1], q.shape[-2]
    group, at = hq // cache.kv_heads, 0
    scale = dim ** -0.5 if scale is None else scale
    assert got.shape == q.shape and got.dtype == BF16 and got.is_contiguous()
    q, got = q.reshape(-1, hq, dim).double(), got.reshape(-1, hq, dim).double()
    for b, (count, length) in enumerate(zip(counts, lengths)):
        if count == 0:
            continue
        here = slice(at, at + count) if rows is None else slice(rows[b], rows[b] + count)
        at += count
        x, y = q[here], got[here]
        if length <= 0:
            assert (y == 0).all()
            continue
        k, v = (z.double().repeat_interleave(group, 1).transpose(0, 1)
                for z in cache.read(length, table[b : b + 1], i32([length]), dtype=F32))  # (heads, places, dim)
        x = x.transpose(0, 1)
        place = torch.arange(length - count, length, device="cuda")[:, None]
        col = torch.arange(length, device="cuda")
        seen = col <= place
        if window:
            seen &= col > place - window
        page = table[b].long()[col // cache.page_size]
        seen = seen & (page >= 0) & (page < cache.n_pages)
        s = x @ k.transpose(1, 2) * scale
        err = abs(scale) * (x.abs() @ k.abs().transpose(1, 2) * (H16 + (dim + 2) * E32)
                            + x.abs().amax(-1, keepdim=True) * k.abs().sum(-1)[:, None] * 2.0 ** -35
                            + x.abs().sum(-1, keepdim=True) * 2.0 ** -25)
        s = s.masked_fill(~seen, -math.inf)
        top = s.amax(-1, keepdim=True)
        p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
        total = p.sum(-1, keepdim=True)
        some = total > 0
        want = torch.where(some, p @ v / torch.where(some, total, 1.0), 0.0)
        size = torch.where(some, p @ v.abs() / torch.where(some, total, 1.0), 0.0)
        spread = torch.where(some, seen.double() @ v.abs() / torch.where(some, total, 1.0), 0.0)
        e = torch.where(seen, err, 0.0).amax(-1, keepdim=True)
        bound = ((torch.exp(2 * e) - 1 + 2.1 * H16 + (length + 300) * E32) * size + 2.0 ** -33 * spread + 2.0 ** -25
                 + 2.0 ** -8 * want.abs())
        off = (y.transpose(0, 1) - want).abs()
        assert (off <= bound).all(), (b, float((off - bound).max()), float((off / bound).max()))


def filled(g, b, lengths, heads, dim, page, spare=1, width=None, scale=1.0):
    """A cache with tokens of every sequence, other bytes where no token is."""
    width = width or max(1, -(-max(lengths) // page))
    table, n = a_table(g, b, width, spare)
    cache = HipPagedCache(n, page, heads, dim)
    cache.pages.fill_(0xFF)  # NaN scales where nothing is written
    lengths = [max(x, 0) for x in lengths]
    t = sum(lengths)
    if t:
        cache.append(None, scale * rand(g, t, heads, dim), rand(g, t, heads, dim) + 0.5, table, i32(lengths), starts_of(lengths))
    return cache, table


@pytest.mark.parametrize("dim", [8, 32, 40, 64, 96, 128, 160, 200, 224, 256])
@pytest.mark.parametrize("group", [1, 3, 4, 16, 20])
@pytest.mark.parametrize("n", [1, 3, 40])
def test_attention(gpu, dim, group, n) -> None:
    g = torch.Generator(device="cuda").manual_seed(dim + group + n)
    heads, lengths = 2, [n, max(n, 31), max(n, 32), 33 + n, 200]
    cache, table = filled(g, 5, lengths, heads, dim, 32)
    q = rand(g, 5 * n, heads * group, dim, dt=BF16)
    got = cache.attend(q, table, i32(lengths))
    check_attention(cache, q, got, table, lengths, [n] * 5)


@pytest.mark.parametrize("window", [0, 1, 5, 32, 100, 1 << 31])
@pytest.mark.parametrize("page", [32, 96, 256])
def test_ragged_windows(gpu, window, page) -> None:
    """Sequences of no token, of one, of chunks; lengths of 0; pages that end inside a tile."""
    window = min(window, (1 << 31) - 1)
    g = torch.Generator(device="cuda").manual_seed(window % 1000 + page)
    counts, lengths = [1, 0, 130, 7, 1, 33, 2], [1, 50, 130, 301, 640, 97, 33]
    cache, table = filled(g, 7, lengths, 2, 64, page)
    q = rand(g, sum(counts), 10, 64, dt=BF16)
    got = cache.attend(q, table, i32(lengths), starts_of(counts), window=window)
    check_attention(cache, q, got, table, lengths, counts, window=window)


@pytest.mark.parametrize("length", [1, 100, 3000, 20000])
@pytest.mark.parametrize("max_length", [None, 64, 5000])
def test_long_axis_is_split(gpu, length, max_length) -> None:
    """One reply, its places shared out over many workgroups, also where it is longer than was said."""
    g = torch.Generator(device="cuda").manual_seed(length)
    lengths = [length, max(1, length // 3)]
    cache, table = filled(g, 2, lengths, 2, 128, 128)
    for n in (1, 2):
        if n > min(lengths):
            continue
        q = 2 * rand(g, 2 * n, 8, 128, dt=BF16)
        got = cache.attend(q, table, i32(lengths), max_length=max_length)
        check_attention(cache, q, got, table, lengths, [n, n])


def test_steep_and_flat_scores(gpu) -> None:
    """Scores of some hundreds, all alike, of large and small rows of one tile, a negative scale, and 0."""
    g = torch.Generator(device="cuda").manual_seed(8)
    lengths = [700]
    cache, table = filled(g, 1, lengths, 1, 64, 64, scale=4.0)
    q = rand(g, 1, 16, 64) * torch.logspace(-6, 1.3, 16, device="cuda")[:, None]
    q[0, 3] = 0
    for scale in (None, -0.25, 0.0, 1.0):
        got = cache.attend(q.bfloat16(), table, i32(lengths), scale=scale)
        check_attention(cache, q.bfloat16(), got, table, lengths, [1], scale=scale)
    big = (q * 1e30).bfloat16()  # beyond float16, brought into it by a power of two
    got = cache.attend(big, table, i32(lengths), scale=1e-30)
    check_attention(cache, big, got, table, lengths, [1], scale=1e-30)


def test_rows_that_attend_to_nothing(gpu) -> None:
    """Lengths of 0, below 0, shorter than the call's rows, pages that are none."""
    g = torch.Generator(device="cuda").manual_seed(9)
    cache, table = filled(g, 5, [64, 64, 64, 64, 64], 2, 64, 32)
    table[3], table[4, 0] = -1, cache.n_pages
    lengths, counts = [0, -7, 2, 64, 64], [3] * 5
    q = rand(g, 15, 4, 64, dt=BF16)
    got = cache.attend(q, table, i32(lengths))
    assert (got[:7] == 0).all() and (got[9:12] == 0).all() and got.isfinite().all()
    check_attention(cache, q[9:], got[9:], table[3:], lengths[3:], counts[3:])
    check_attention(cache, q[7:9], got[7:9].contiguous(), table[2:3], [2], [2])


def test_not_a_number_stays_in_its_row(gpu) -> None:
    g = torch.Generator(device="cuda").manual_seed(10)
    cache, table = filled(g, 1, [90], 1, 64, 32)
    q = rand(g, 4, 4, 64, dt=BF16)
    clean = cache.attend(q, table, i32([90]))
    q[1, 2, 7], q[3, 0, 0] = math.nan, math.inf
    got = cache.attend(q, table, i32([90]))
    assert got[1, 2].isnan().all()
    others = torch.ones(4, 4, dtype=torch.bool, device="cuda")
    others[1, 2] = others[3, 0] = False
    assert same(got[others], clean[others])


def test_a_tokens_bad_values_touch_only_who_attends_to_them(gpu) -> None:
    """Not-a-numbers in later tokens of a chunk, and in bytes behind the end, do not reach earlier rows."""
    g = torch.Generator(device="cuda").manual_seed(11)
    q, k, v = rand(g, 40, 2, 64, dt=BF16), rand(g, 40, 2, 64, dt=BF16), rand(g, 40, 2, 64, dt=BF16)
    table, out = i32([[0, 1]]), []
    for bad in (False, True):
        if bad:
            k[33:], v[33:] = math.nan, math.inf
        cache = HipPagedCache(2, 32, 2, 64)
        cache.pages.fill_(0xFF)
        cache.append(None, k, v, table, i32([40]))
        out.append(cache.attend(q, table, i32([40])))
    assert same(out[0][:33], out[1][:33]) and out[1].isfinite().all()


def test_one_token_as_in_a_chunk_and_in_any_company(gpu) -> None:
    """A row's result lies within rounding of itself alone, in a chunk, and among other sequences."""
    g = torch.Generator(device="cuda").manual_seed(12)
    lengths = [300, 700, 50]
    cache, table = filled(g, 3, lengths, 2, 128, 64)
    q = rand(g, 300, 8, 128, dt=BF16)
    chunk = cache.attend(q, table[:1], i32([300]))
    check_attention(cache, q, chunk, table[:1], [300], [300])
    alone = cache.attend(q[-1:], table[:1], i32([300]))
    check_attention(cache, q[-1:], alone, table[:1], [300], [1])
    both = cache.attend(torch.stack((q[-1], q[0], q[1])), table, i32(lengths))
    assert same(both[:1], alone) or (both[:1].float() - alone.float()).abs().max() < 0.02


def test_batched_queries_and_strides(gpu) -> None:
    g = torch.Generator(device="cuda").manual_seed(13)
    lengths = [100, 77]
    cache, table = filled(g, 2, lengths, 2, 64, 32)
    buf = rand(g, 2, 6, 5 * 64 * 2 + 1, dt=BF16)
    q = buf[..., 1 : 1 + 4 * 64].unflatten(-1, (4, 64))
    got = cache.attend(q, table, i32(lengths))
    assert got.shape == q.shape
    assert same(got.flatten(0, 1), cache.attend(q.flatten(0, 1).contiguous(), table, i32(lengths)))
    every = cache.attend(buf[..., : 4 * 128].unflatten(-1, (4, 64, 2))[..., 0], table, i32(lengths))  # a copy is made
    assert every.shape == q.shape
    check_attention(cache, q, got, table, lengths, [6, 6])


def test_streams_and_graphs(gpu) -> None:
    """On another stream, and captured: the replays move on with lengths, tables and inputs."""
    g = torch.Generator(device="cuda").manual_seed(14)
    b, hq, hk, dim = 3, 8, 2, 64
    table = torch.arange(b * 8, device="cuda").view(b, 8).int()
    cache = HipPagedCache(b * 8, 64, hk, dim)
    rot = HipRotary(dim)
    lengths = i32([100, 1, 300])
    q, k, v = (rand(g, b, h, dim, dt=BF16) for h in (hq, hk, hk))
    t = 401
    cache.append(None, rand(g, t, hk, dim, dt=BF16), rand(g, t, hk, dim, dt=BF16), table, lengths, starts_of([100, 1, 300]))

    def step():
        q2 = cache.append(q, k, v, table, lengths, rotary=rot)
        return cache.attend(q2, table, lengths)

    want = step()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = step()
    stream.synchronize()
    assert same(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    other = torch.cuda.CUDAGraph()
    with torch.cuda.graph(other):
        out2 = step()
    for i in range(4):
        lengths += 1
        q.copy_(rand(g, b, hq, dim, dt=BF16))
        graph.replay()
        kept = out.clone()
        other.replay()
        want = step()
        torch.cuda.synchronize()
        assert same(kept, want) and same(out2, want), i
    check_attention(cache, cache.append(q, k, v, table, lengths, rotary=rot), want, table, lengths.tolist(), [1] * b)


def test_prompt_and_replies_as_a_model_runs_them(gpu) -> None:
    """Prompts in ragged chunks, then replies, against float32 attention over the values before they were held: the
    cache's own error is within what 4 bits allow, and every step is within rounding of the held values."""
    g = torch.Generator(device="cuda").manual_seed(15)
    hq, hk, dim, page = 8, 2, 64, 32
    rot = HipRotary(dim, base=500000.0)
    prompts, steps = [70, 33, 129], 5
    table, n = a_table(g, 3, 6)
    cache = HipPagedCache(n, page, hk, dim)
    qw, kw = (1 + 0.2 * rand(g, dim)).to(BF16), (1 + 0.2 * rand(g, dim)).to(BF16)
    lengths = [0, 0, 0]
    for counts in ([64, 33, 64], [6, 0, 65], *[[1, 1, 1]] * steps):
        lengths = [a + c for a, c in zip(lengths, counts)]
        t = sum(counts)
        qkv = rand(g, t, (hq + 2 * hk) * dim, dt=BF16)
        q, k, v = (x.unflatten(-1, (-1, dim)) for x in torch.split(qkv, [hq * dim, hk * dim, hk * dim], dim=-1))
        where = (table, i32(lengths), starts_of(counts))
        q2 = cache.append(q, k, v, *where, rotary=rot, q_weight=qw, k_weight=kw)
        got = cache.attend(q2, *where)
        check_attention(cache, q2, got, table, lengths, counts)
    assert lengths == [p + steps for p in prompts]


def test_offsets_past_32_bits(gpu) -> None:
    """A pool of more than 4 GiB: its last pages are written, read and attended to."""
    heads, dim, page = 8, 256, 1024
    each = page // 32 * heads * 10240
    n = (1 << 32) // each + 5
    g = torch.Generator(device="cuda").manual_seed(16)
    cache = HipPagedCache(n, page, heads, dim)
    table, lengths = i32([[n - 1, 0], [1, n - 2]]), [1100, 1500]
    t = sum(lengths)
    k, v = rand(g, t, heads, dim, dt=BF16), rand(g, t, heads, dim, dt=BF16)
    cache.append(None, k, v, table, i32(lengths), starts_of(lengths))
    k2, v2 = cache.read(t, table, i32(lengths), starts_of(lengths), dtype=F32)
    assert same(k2, held(k)) and same(v2, held(v))
    q = rand(g, 2, heads, dim, dt=BF16)
    check_attention(cache, q, cache.attend(q, table, i32(lengths)), table, lengths, [1, 1])


def test_many_sequences_and_rows(gpu) -> None:
    g = torch.Generator(device="cuda").manual_seed(17)
    b = 1000
    lengths = torch.randint(1, 64, (b,), generator=torch.Generator().manual_seed(1)).tolist()
    cache, table = filled(g, b, lengths, 1, 32, 32, width=2)
    q = rand(g, b, 2, 32, dt=BF16)
    got = cache.attend(q, table, i32(lengths))
    for at in (0, 499, 999):
        check_attention(cache, q[at : at + 1], got[at : at + 1], table[at : at + 1], lengths[at : at + 1], [1])
    starts = torch.arange(b + 1, device="cuda").int()
    assert same(cache.attend(q, table, i32(lengths), starts), got)


def test_refusals(gpu) -> None:
    for bad in (dict(n_pages=0), dict(page_size=48), dict(page_size=0), dict(page_size=1 << 17), dict(kv_heads=0),
                dict(head_dim=20), dict(head_dim=264), dict(head_dim=0), dict(device="cpu")):
        with pytest.raises(ValueError):
            HipPagedCache(**{**dict(n_pages=2, page_size=32, kv_heads=2, head_dim=64), **bad})
    cache = HipPagedCache(4, 32, 2, 64)
    for pages in (cache.pages[:2], cache.pages.view(torch.int8), cache.pages.cpu(), cache.pages.transpose(0, 1)):
        with pytest.raises(ValueError, match="pages"):
            HipPagedCache(4, 32, 2, 64, pages=pages)
    q, k = torch.zeros(4, 4, 64, device="cuda", dtype=BF16), torch.zeros(4, 2, 64, device="cuda", dtype=BF16)
    table, lengths, w = i32([[0, 1], [2, 3]]), i32([2, 2]), torch.ones(64, device="cuda", dtype=BF16)

    def append(q=q, k=k, v=k, table=table, lengths=lengths, query_starts=None, **more):
        return cache.append(q, k, v, table, lengths, query_starts, **more)

    def attend(q=q, table=table, lengths=lengths, query_starts=None, **more):
        return cache.attend(q, table, lengths, query_starts, **more)

    for call in (append, attend):
        for bad, match in ((dict(table=table.long()), "table"), (dict(table=table[0]), "table"),
                           (dict(table=table.cpu()), "table"), (dict(table=table.T), "table"),
                           (dict(table=table[:, :0]), "table"), (dict(lengths=lengths[:1]), "lengths"),
                           (dict(lengths=lengths.long()), "lengths"), (dict(query_starts=i32([0, 4])), "query_starts"),
                           (dict(query_starts=i32([0, 2, 4]).long()), "query_starts"),
                           (dict(q=q[:, :3]), "heads"), (dict(q=q[..., :32]), "q must"), (dict(q=q.cpu()), "q must"),
                           (dict(table=table[:0], lengths=lengths[:0]), "sequences|rows")):
            with pytest.raises(ValueError, match=match):
                call(**bad)
    three = torch.zeros(3, 4, 64, device="cuda", dtype=BF16)
    with pytest.raises(ValueError, match="same number"):
        attend(q=three)
    with pytest.raises(ValueError, match="query_starts"):
        attend(q=q[None], query_starts=i32([0, 2, 4]))
    with pytest.raises(ValueError, match="sequences"):
        attend(q=q[None])
    for bad, match in ((dict(q=q.float()), "bfloat16"), (dict(window=-1), "window"), (dict(out=q[:2]), "out"),
                       (dict(out=q.float()), "out"), (dict(out=torch.empty(4, 64, 4, device="cuda", dtype=BF16).mT), "out")):
        with pytest.raises(ValueError, match=match):
            attend(**bad)
    for bad, match in ((dict(k=k[:, :1]), "k must"), (dict(v=k.float()), "v must"), (dict(v=k[:2]), "v must"),
                       (dict(q=q[:2]), "q must"), (dict(q=q.float()), "q must"), (dict(k=k.half()), "k must"),
                       (dict(rotary=HipRotary(32)), "rotary"), (dict(positions=torch.zeros(3, device="cuda").int()), "positions"),
                       (dict(positions=torch.zeros(4, device="cuda")), "positions"), (dict(q_weight=w.float()), "q_weight"),
                       (dict(k_weight=w[:3]), "k_weight"), (dict(q=None, q_weight=w), "needs q")):
        with pytest.raises(ValueError, match=match):
            append(**bad)
    for n, more in ((3, {}), (-1, {}), (4, dict(dtype=torch.float16))):
        with pytest.raises(ValueError):
            cache.read(n, table, lengths, **more)
    # nothing to do is no error
    assert attend(q=q[:0]).shape == (0, 4, 64) and append(q=q[:0], k=k[:0], v=k[:0]).shape == (0, 4, 64)
    assert cache.read(0, table, lengths)[0].shape == (0, 2, 64)
    assert attend(q=q[:0], table=table[:0], lengths=lengths[:0]).numel() == 0


# ---- many rows of a key head: tiles of 128 and 256 rows, whose places may be shared out
@pytest.mark.parametrize("dim", [8, 32, 64, 96, 128, 160, 200, 256])
@pytest.mark.parametrize("group, n", [(1, 65), (1, 129), (4, 33), (5, 70), (16, 40)])
@pytest.mark.parametrize("length", [0, 2500])
def test_many_rows(gpu, dim, group, n, length) -> None:
    """At the beginning of a sequence and behind some thousand places; ends inside a block, a page and a tile."""
    g = torch.Generator(device="cuda").manual_seed(dim + group + n + length)
    lengths = [n + length, n, n + length // 2 + 7]
    cache, table = filled(g, 3, lengths, 2, dim, 96)
    q = rand(g, 3 * n, 2 * group, dim, dt=BF16)
    check_attention(cache, q, cache.attend(q, table, i32(lengths)), table, lengths, [n] * 3)


@pytest.mark.parametrize("window", [1, 31, 64, 700])
@pytest.mark.parametrize("dim, n", [(64, 40), (128, 300), (192, 70)])
def test_many_rows_in_a_window(gpu, dim, n, window) -> None:
    g = torch.Generator(device="cuda").manual_seed(window + n)
    lengths = [1500, n]
    cache, table = filled(g, 2, lengths, 1, dim, 64)
    q = rand(g, 2 * n, 4, dim, dt=BF16)
    for most in (None, 100):
        got = cache.attend(q, table, i32(lengths), window=window, max_length=most)
        check_attention(cache, q, got, table, lengths, [n, n], window=window)


@pytest.mark.parametrize("n", [40, 300])
def test_many_rows_with_steep_scores(gpu, n) -> None:
    """As test_steep_and_flat_scores; places whose scores rise, fall, and are alike."""
    g = torch.Generator(device="cuda").manual_seed(n)
    lengths = [700]
    cache, table = filled(g, 1, lengths, 1, 64, 64, scale=4.0)
    q = rand(g, n, 4, 64) * torch.logspace(-6, 1.3, 4 * n, device="cuda").view(n, 4, 1)
    q[3] = 0
    for scale in (None, -0.25, 0.0, 1.0):
        got = cache.attend(q.bfloat16(), table, i32(lengths), scale=scale)
        check_attention(cache, q.bfloat16(), got, table, lengths, [n], scale=scale)
    big = (q * 1e30).bfloat16()
    check_attention(cache, big, cache.attend(big, table, i32(lengths), scale=1e-30), table, lengths, [n], scale=1e-30)
    ramp = torch.linspace(-20, 20, 700, device="cuda")[:, None, None] + 0.1 * rand(g, 700, 1, 64)
    for sign in (1, -1):
        cache.append(None, (sign * ramp).contiguous(), rand(g, 700, 1, 64), table, i32(lengths))
        q = rand(g, n, 4, 64, dt=BF16).abs()
        check_attention(cache, q, cache.attend(q, table, i32(lengths)), table, lengths, [n])


def test_many_rows_that_attend_to_nothing(gpu) -> None:
    """Lengths of 0, below 0 and shorter than the rows; pages that are none before, in and behind what is attended to."""
    g = torch.Generator(device="cuda").manual_seed(21)
    cache, table = filled(g, 5, [512] * 5, 2, 64, 32)
    table[3, :4], table[3, 9], table[4] = -1, cache.n_pages, -5
    lengths, n = [0, -7, 30, 512, 512], 70
    q = rand(g, 5 * n, 4, 64, dt=BF16)
    for window in (0, 40):
        got = cache.attend(q, table, i32(lengths), window=window)
        assert (got[: 2 * n + 40] == 0).all() and (got[4 * n :] == 0).all() and got.isfinite().all()
        check_attention(cache, q[3 * n : 4 * n], got[3 * n : 4 * n], table[3:4], [512], [n], window=window)
        check_attention(cache, q[2 * n + 40 : 3 * n], got[2 * n + 40 : 3 * n], table[2:3], [30], [30], window=window)


@pytest.mark.parametrize("n", [70, 300])
def test_many_rows_and_not_a_number(gpu, n) -> None:
    """In q it stays in its row; in later tokens, and in what lies behind the end, it reaches nobody before."""
    g = torch.Generator(device="cuda").manual_seed(n)
    cache, table = filled(g, 1, [900], 1, 64, 32)
    q = rand(g, n, 4, 64, dt=BF16)
    clean = cache.attend(q, table, i32([900]))
    dirty = q.clone()
    dirty[1, 2, 7], dirty[n - 1, 0, 0] = math.nan, math.inf
    got = cache.attend(dirty, table, i32([900]))
    others = torch.ones(n, 4, dtype=torch.bool, device="cuda")
    others[1, 2] = others[n - 1, 0] = False
    assert got[1, 2].isnan().all()
    check_attention(cache, q, torch.where(others[..., None], got, clean), table, [900], [n])
    k, v = rand(g, n, 1, 64, dt=BF16), rand(g, n, 1, 64, dt=BF16)
    cache.append(None, k, v, table, i32([900]))
    clean = cache.attend(q, table, i32([900]))
    k[n // 2 :], v[n // 2 :] = math.nan, math.inf
    cache.append(None, k, v, table, i32([900]))
    got = cache.attend(q, table, i32([900]))
    assert same(got[: n // 2], clean[: n // 2]) and got.isfinite().all()


def test_many_rows_captured(gpu) -> None:
    """Chunks and replies in one captured call, which moves on with lengths and starts; two graphs in turn."""
    g = torch.Generator(device="cuda").manual_seed(23)
    lengths, counts = [900, 640, 33], [100, 1, 33]
    cache, table = filled(g, 3, [1000, 700, 300], 2, 128, 64)
    q, out = rand(g, 160, 8, 128, dt=BF16), torch.full((160, 8, 128), 7.0, dtype=BF16, device="cuda")
    length, starts = i32(lengths), starts_of(counts)
    graphs = []
    for _ in range(2):
        cache.attend(q, table, length, starts, out=out)
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            cache.attend(q, table, length, starts, out=out)
    for i in range(4):
        lengths = [lengths[0] + 20, lengths[1] + 11, lengths[2] + 60]
        counts = [counts[0] - 20, 1 + 25 * i, counts[2] + 3]
        length.copy_(i32(lengths))
        starts.copy_(starts_of(counts))
        q.copy_(rand(g, 160, 8, 128, dt=BF16))
        out.fill_(7.0)
        graphs[i % 2].replay()
        got = out.clone()
        t = sum(counts)
        assert (got[t:] == 7.0).all()  # rows of no sequence: as they were
        check_attention(cache, q[:t], got[:t], table, lengths, counts)
        out.fill_(7.0)
        assert same(cache.attend(q, table, length, starts, out=out), got)


@pytest.mark.parametrize("b", [3, 70, 300])
def test_many_ragged_sequences(gpu, b) -> None:
    """Replies, short chunks, sequences without rows and rows in front of the first, long places among short ones."""
    g = torch.Generator(device="cuda").manual_seed(b)
    counts = [(1, 0, 1, 5, 1, 40)[i % 6] for i in range(b)]
    counts[b // 2] = 150
    lengths = [c + (0, 700, 31)[i % 3] for i, c in enumerate(counts)]
    lengths[1], lengths[b // 2] = 3000, 400
    cache, table = filled(g, b, lengths, 2, 64, 32, width=3008 // 32)
    t = sum(counts)
    q, out = rand(g, t + 5, 8, 64, dt=BF16), torch.full((t + 5, 8, 64), 3.0, dtype=BF16, device="cuda")
    cache.attend(q, table, i32(lengths), starts_of(counts) + 3, out=out)
    assert (out[:3] == 3.0).all() and (out[t + 3 :] == 3.0).all()
    check_attention(cache, q[3 : t + 3], out[3 : t + 3], table, lengths, counts)


@pytest.mark.parametrize("n", [1, 130])
def test_as_many_heads_as_there_may_be(gpu, n) -> None:
    g = torch.Generator(device="cuda").manual_seed(31)
    heads, lengths = 4096, [n + 40]
    cache, table = filled(g, 1, lengths, heads, 8, 32)
    q, k, v = (rand(g, n, heads, 8, dt=BF16) for _ in range(3))
    q2 = cache.append(q, k, v, table, i32(lengths))
    k2, v2 = cache.read(n, table, i32(lengths), dtype=F32)
    assert same(q2, q) and same(k2, held(k)) and same(v2, held(v))
    check_attention(cache, q, cache.attend(q, table, i32(lengths)), table, lengths, [n])


@pytest.mark.parametrize("starts", [[6, 0, 3], [6, 6, 0], [9, 2, -1], [-3, 6, 2]])
def test_starts_that_descend_touch_nothing_else(gpu, starts) -> None:
    """What the rows then get means nothing, but it lies in the rows, and an ascending call behind it is right."""
    g = torch.Generator(device="cuda").manual_seed(32)
    heads, group, dim, lengths = 2, 32, 32, [90, 80]
    cache, table = filled(g, 2, lengths, heads, dim, 32)
    pages = cache.pages.clone()
    q = rand(g, 6, heads * group, dim, dt=BF16)
    for most in (96, None):
        around = torch.full((8, heads * group, dim), 7.0, dtype=BF16, device="cuda")
        cache.attend(q, table, i32(lengths), i32(starts), max_length=most, out=around[1:7])
        assert (around[0] == 7).all() and (around[7] == 7).all()
        assert cache.append(q, q[:, :heads], q[:, :heads], i32([[-1] * 3] * 2), i32(lengths), i32(starts)).isfinite().all()
        assert same(cache.pages, pages)
        got = cache.attend(q, table, i32(lengths), starts_of([2, 4]), max_length=most)
        check_attention(cache, q, got, table, lengths, [2, 4])


@pytest.mark.parametrize("n", [1, 70, 300])
@pytest.mark.parametrize("dim", [64, 200])
def test_a_scale_that_is_no_number(gpu, n, dim) -> None:
    """Few rows and many: not-a-number in every row that attends to something, zeros in the others."""
    g = torch.Generator(device="cuda").manual_seed(n)
    lengths = [2000, 0, n // 2]
    cache, table = filled(g, 3, lengths, 2, dim, 32)
    q = rand(g, 3 * n, 8, dim, dt=BF16)
    for window in (0, 20):
        got = cache.attend(q, table, i32(lengths), scale=math.nan, window=window)
        some = torch.zeros(3 * n, dtype=torch.bool, device="cuda")
        some[:n] = some[3 * n - n // 2 :] = True
        assert got[some].isnan().all() and (got[~some] == 0).all()


@pytest.mark.parametrize("chunk", [130, 700, 2100])
def test_long_replies_beside_a_chunk(gpu, chunk) -> None:
    """Replies whose places are shared out, between and behind sequences of many rows, and one of few rows of its own."""
    g = torch.Generator(device="cuda").manual_seed(chunk)
    counts, lengths = [1, chunk, 0, 1, 20, 2], [20000, chunk + 300, 40, 5, 9000, 13000]
    cache, table = filled(g, 6, lengths, 2, 64, 64)
    q = rand(g, sum(counts), 8, 64, dt=BF16)
    for most in (None, 3000):
        got = cache.attend(q, table, i32(lengths), starts_of(counts), max_length=most)
        check_attention(cache, q, got, table, lengths, counts)


# ---- what a copy, a wider table and 4 bits do to the values
def test_queries_whose_values_are_not_adjacent(gpu) -> None:
    """attend makes a copy of such a q: the bits of the call with a contiguous one, of three and of four dimensions."""
    g = torch.Generator(device="cuda").manual_seed(33)
    lengths = [100, 77]
    cache, table = filled(g, 2, lengths, 2, 64, 32)
    every = rand(g, 2, 6, 4, 64, 2, dt=BF16)[..., 1]
    turned = rand(g, 2, 6, 64, 4, dt=BF16).transpose(2, 3)
    for q in (every, turned):
        assert q.stride(-1) != 1
        want = cache.attend(q.contiguous(), table, i32(lengths))
        got = cache.attend(q, table, i32(lengths))
        assert same(got, want) and got.is_contiguous()
        assert same(cache.attend(q.flatten(0, 1), table, i32(lengths), starts_of([6, 6])), want.flatten(0, 1))
        check_attention(cache, q, got, table, lengths, [6, 6])


def test_keys_and_values_that_are_not_adjacent(gpu) -> None:
    g = torch.Generator(device="cuda").manual_seed(34)
    q, k, v = rand(g, 9, 4, 64, 2), rand(g, 9, 64, 2).transpose(1, 2), rand(g, 9, 2, 128)[..., ::2]
    q, w, rot = q[..., 0], 1 + 0.2 * rand(g, 128), HipRotary(64)
    caches = [HipPagedCache(1, 32, 2, 64) for _ in range(2)]
    out = [c.append(*x, i32([[0]]), i32([9]), rotary=rot, q_weight=y, k_weight=y)
           for c, x, y in ((caches[0], (q, k, v), w[::2]),
                           (caches[1], (q.contiguous(), k.contiguous(), v.contiguous()), w[::2].contiguous()))]
    assert same(*out) and same(caches[0].pages, caches[1].pages) and bool((caches[0].pages != 0).any())
    assert same(caches[0].read(9, i32([[0]]), i32([9]), dtype=F32)[1], held(v))


def test_a_table_that_is_part_of_a_wider_one(gpu) -> None:
    """Columns from the middle of rows whose other entries name other pages."""
    g = torch.Generator(device="cuda").manual_seed(35)
    wide = i32([[5, 0, 2, 4, 4], [5, 1, 3, 4, 5]])
    table, lengths, counts = wide[:, 1:3], [64, 50], [64, 50]
    assert table.stride(0) > table.shape[1]
    caches = [HipPagedCache(6, 32, 2, 64) for _ in range(2)]
    k, v, q = rand(g, 114, 2, 64), rand(g, 114, 2, 64), rand(g, 114, 4, 64, dt=BF16)
    for cache, t in zip(caches, (table, table.contiguous())):
        cache.append(None, k, v, t, i32(lengths), starts_of(counts))
    assert same(caches[0].pages, caches[1].pages)
    assert (caches[0].pages[4:] == 0).all() and (caches[0].pages[:4] != 0).any()
    read = caches[0].read(114, table, i32(lengths), starts_of(counts), dtype=F32)
    assert same(read[0], held(k)) and same(read[1], held(v))
    for n in (1, 50):
        x = q[: 2 * n]
        got = caches[0].attend(x, table, i32(lengths))
        assert same(got, caches[1].attend(x, table.contiguous(), i32(lengths)))
        check_attention(caches[0], x, got, table, lengths, [n, n])


def test_against_values_that_were_never_held(gpu) -> None:
    """Prompts and replies as test_prompt_and_replies_as_a_model_runs_them has them, against attention in 64 bits over the
    float32 keys and values that were given to the cache.

    A held value is within half a step of its group, s / 2 with s = f16((max - min) / 15), and what the roundings of s and of
    the minimum leave at the group's ends: 15 |s - (max - min) / 15| and |m - min|, half a step of float16 each (2^-11 of
    themselves, 2^-25 where subnormal): |dx| <= (max - min) (1/30 + 2^-10) + 2^-11 |min| + 2^-20. With E_t = scale sum |q dk_t|
    and E the largest of them a probability is off by e^(2 E) - 1 of itself, so that the output is within
    (e^(2 E) - 1) sum p |v| + e^(2 E) sum p |dv| of attention over what was given, and the kernel's own error besides, for which
    check_attention's bound on each step is taken with 0.03 of the largest |v|: 2^-8 for the output and e^(2 e) - 1 + 2.1 h for
    e = scale sum |q k| (h + 66 2^-24) up to 5e-3."""
    g = torch.Generator(device="cuda").manual_seed(36)
    hq, hk, dim, page = 8, 2, 64, 32
    rot = HipRotary(dim, base=500000.0)
    table, n = a_table(g, 3, 6)
    cache = HipPagedCache(n, page, hk, dim)
    qw, kw = (1 + 0.2 * rand(g, dim)).to(BF16), (1 + 0.2 * rand(g, dim)).to(BF16)
    lengths, given = [0, 0, 0], [([], []) for _ in range(3)]
    for counts in ([64, 33, 64], [6, 0, 65], [1, 1, 1], [1, 1, 1]):
        lengths = [a + c for a, c in zip(lengths, counts)]
        t = sum(counts)
        qkv = rand(g, t, (hq + 2 * hk) * dim, dt=BF16)
        q, k, v = (x.unflatten(-1, (-1, dim)) for x in torch.split(qkv, [hq * dim, hk * dim, hk * dim], dim=-1))
        where = (table, i32(lengths), starts_of(counts))
        q2 = cache.append(q, k, v, *where, rotary=rot, q_weight=qw, k_weight=kw)
        got = cache.attend(q2, *where)
        places = torch.tensor([p for _, p in rows_of(counts, lengths)], device="cuda")
        turned = rot(k.float(), None, places, q_weight=kw.float())[0]
        at = 0
        for b, c in enumerate(counts):
            if c == 0:
                continue
            given[b][0].append(turned[at : at + c]), given[b][1].append(v[at : at + c].float())
            x, y = (z[at : at + c].double().transpose(0, 1) for z in (q2, got))
            at += c
            keys, values = (torch.cat(z) for z in given[b])
            off = []
            for z, kept in zip((keys, values), cache.read(lengths[b], table[b : b + 1], i32([lengths[b]]), dtype=F32)):
                low, high = (f(z.unflatten(-1, (-1, 32)), -1, keepdim=True).expand(-1, -1, -1, 32).flatten(2)
                             for f in (torch.amin, torch.amax))
                off.append((kept.double() - z.double()).abs())
                assert (off[-1] <= (high - low) * (1 / 30 + 2.0 ** -10) + low.abs() * H16 + 2.0 ** -20).all()
            keys, values, dk, dv = (z.double().repeat_interleave(hq // hk, 1).transpose(0, 1) for z in (keys, values, *off))
            place = torch.arange(lengths[b] - c, lengths[b], device="cuda")[:, None]
            seen = torch.arange(lengths[b], device="cuda") <= place
            scores = (x @ keys.transpose(1, 2) * dim ** -0.5).masked_fill(~seen, -math.inf)
            p = torch.softmax(scores, -1)
            e = torch.where(seen, x.abs() @ dk.transpose(1, 2) * dim ** -0.5, 0.0).amax(-1, keepdim=True)
            own = torch.where(seen, x.abs() @ keys.abs().transpose(1, 2) * dim ** -0.5, 0.0).amax()
            assert float(own) * (H16 + 66 * E32) < 5e-3
            bound = (torch.exp(2 * e) - 1) * (p @ values.abs()) + torch.exp(2 * e) * (p @ dv) + 0.03 * values.abs().amax()
            assert ((y - p @ values).abs() <= bound).all()


def test_more_tiles_than_a_grid_takes_one_by_one(gpu) -> None:
    """With query_starts, so many sequences that the grid is one of every sequence's most; one of them a chunk."""
    g = torch.Generator(device="cuda").manual_seed(37)
    b = 60000
    lengths = torch.randint(1, 60, (b,), generator=torch.Generator().manual_seed(1)).tolist()
    lengths[b // 2], lengths[b - 2] = 60, 33
    cache, table = filled(g, b, lengths, 1, 8, 32, width=2)
    q = rand(g, b, 4, 8, dt=BF16)
    want = cache.attend(q, table, i32(lengths))
    assert same(cache.attend(q, table, i32(lengths), torch.arange(b + 1, device="cuda").int()), want)
    counts = [1] * b
    counts[5], counts[b // 2], counts[b - 2] = 0, 50, 3
    q = rand(g, sum(counts), 4, 8, dt=BF16)
    got = cache.attend(q, table, i32(lengths), starts_of(counts))
    for s in (0, 5, 6, b // 2 - 1, b // 2, b // 2 + 1, b - 2, b - 1):
        first = sum(counts[:s])
        rows = slice(first, first + counts[s])
        check_attention(cache, q[rows], got[rows], table[s : s + 1], [lengths[s]], [counts[s]])
