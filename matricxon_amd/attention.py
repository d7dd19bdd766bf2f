"""Attention over a paged cache of 4-bit keys and values: what a decoder layer does between its q | k | v projections
(`matricxon_amd.fused_ops.project_shared`) and o.

    cache = HipPagedCache(n_pages, page_size, kv_heads, head_dim)
    q = cache.append(q, k, v, table, lengths, rotary=rot, q_weight=qw, k_weight=kw)
    out = cache.attend(q, table, lengths)

32 neighbouring values of a token's head share a float16 scale and minimum and are held as 4-bit codes: 5 bits a value, a
third of bfloat16's. Which tokens a call is about is said by three int32 tensors on the cache's device, so that a captured
call moves on with them:

* `table` (B, width): the page of places j * page_size .. of sequence b is `table[b, j]`. A number outside
  [0, n_pages) is no page: what would lie there is neither written nor attended to, and reads as zeros.
* `lengths` (B,): tokens of each sequence, those of this call among them.
* `query_starts` (B + 1,), ascending, or None: rows [query_starts[b], query_starts[b + 1]) of q, k and v are the last
  tokens of sequence b; rows behind the last sequence belong to none. None: the same number of rows for each. (Of starts
  that descend the results mean nothing; no memory outside the tensors is touched.)

q, k and v are (T, heads, head_dim), or (B, T, heads, head_dim) without `query_starts`, of any strides with adjacent
values in a head, as the columns of a q | k | v buffer. The reference keeps its cache in tensors of the layer's dtype
(app/runtime/batch_cache.py) and attends over it in torch operations, on the CPU in app/native/src/mx_attention.c.
"""

import math

import torch

from matricxon_amd.gemm import (_FLOATS, _INTS, HipGemm, _elsewhere, _head_strides, _head_weight, _require_device_tensor,
                                _stream)
from matricxon_amd.rotary import HipRotary

_BF16 = torch.bfloat16


class HipPagedCache:
    """`n_pages` pages of `page_size` tokens (a multiple of 32) of `kv_heads` heads of `head_dim` values (a multiple of 8
    up to 256), zeros at first, or `pages` as another cache of this shape holds them."""

    BLOCK = 32  # tokens
    MAX_PAGE = 65536
    MAX_PLACES = 1 << 30  # width of a table times page_size
    MAX_SEQUENCES = 65535
    MAX_ROWS = 1 << 28  # tokens times heads of attend's q

    def __init__(self, n_pages: int, page_size: int, kv_heads: int, head_dim: int, *,
                 device: torch.device | str = "cuda", pages: torch.Tensor | None = None) -> None:
        self.n_pages, self.page_size = int(n_pages), int(page_size)
        self.kv_heads, self.head_dim = int(kv_heads), int(head_dim)
        self._gemm = HipGemm.get()
        self._lib = self._gemm._lib
        page_bytes = self._lib.mxa_kv4_page_bytes(self.kv_heads, self.page_size, self.head_dim)
        if page_bytes == 0 or not 1 <= self.n_pages < 1 << 31:
            raise ValueError(f"a cache needs pages, a page_size that is a multiple of {self.BLOCK} up to {self.MAX_PAGE}, "
                             f"1..4096 heads and a head_dim that is a multiple of 8 up to 256, got {n_pages} pages of "
                             f"{page_size} tokens, {kv_heads} heads of {head_dim}")
        blocks = self.page_size // self.BLOCK
        shape = (self.n_pages, self.kv_heads, blocks, page_bytes // (self.kv_heads * blocks))
        if pages is None:
            device = torch.device(device)
            if device.type != "cuda":
                raise ValueError(f"a cache lies on a HIP device, got {device}")
            pages = torch.zeros(shape, dtype=torch.uint8, device=device)
        else:
            _require_device_tensor("pages", pages)
            if pages.dtype != torch.uint8 or pages.shape != shape or not pages.is_contiguous() or pages.data_ptr() % 16:
                raise ValueError(f"pages must be contiguous uint8 {shape} on a 16-byte boundary, got {pages.dtype} "
                                 f"{tuple(pages.shape)}")
        self.pages, self.device = pages, pages.device

    # -- checks ---------------------------------------------------------------------------------
    def _where(self, table: torch.Tensor, lengths: torch.Tensor, query_starts: torch.Tensor | None, n_tokens: int,
               batch: int | None) -> tuple:
        """The library's arguments for the pages and sequences of n_tokens rows (batch: of a 4-dimensional input)."""
        dev, ts = self.device, table.shape
        if table.dtype is not torch.int32 or table.device != dev or len(ts) != 2 or ts[1] < 1 or \
                (table.stride(1) != 1 and ts[1] > 1) or ts[1] * self.page_size > self.MAX_PLACES:
            raise ValueError(f"table must be int32 (B, pages) on {dev}, its rows' values adjacent, up to "
                             f"{self.MAX_PLACES} places, got {table.dtype} {tuple(ts)} on {table.device}")
        n_seq = ts[0]
        if lengths.dtype is not torch.int32 or lengths.device != dev or lengths.shape != (n_seq,) or \
                not lengths.is_contiguous():
            raise ValueError(f"lengths must be contiguous int32 ({n_seq},) on {dev}, got {lengths.dtype} "
                             f"{tuple(lengths.shape)} on {lengths.device}")
        if not 1 <= n_seq <= self.MAX_SEQUENCES and n_tokens > 0:
            raise ValueError(f"table must have 1..{self.MAX_SEQUENCES} rows, got {n_seq}")
        starts = 0
        if query_starts is not None:
            if query_starts.dtype is not torch.int32 or query_starts.device != dev or \
                    query_starts.shape != (n_seq + 1,) or not query_starts.is_contiguous() or batch is not None:
                raise ValueError(f"query_starts must be contiguous int32 ({n_seq + 1},) on {dev}, with rows (T, heads, "
                                 f"head_dim), got {query_starts.dtype} {tuple(query_starts.shape)} on "
                                 f"{query_starts.device}")
            starts = query_starts.data_ptr()
        elif n_tokens % n_seq if n_seq else n_tokens:
            raise ValueError(f"{n_tokens} rows are not the same number for each of {n_seq} sequences")
        elif batch is not None and batch != n_seq:
            raise ValueError(f"table must have a row for each of {batch} sequences, got {n_seq}")
        if n_tokens > self._gemm.MAX_TOKENS:
            raise ValueError(f"up to {self._gemm.MAX_TOKENS} rows, got {n_tokens}")
        return (self.pages.data_ptr(), self.n_pages, self.kv_heads, self.page_size, self.head_dim, table.data_ptr(),
                table.stride(0), ts[1], lengths.data_ptr(), starts, n_seq)

    def _rows(self, name: str, x: torch.Tensor, heads: int | None, like: torch.Tensor | None = None) -> tuple[int, int]:
        """(rows, rows of a batch entry) of q, k or v."""
        s = x.shape
        if x.dtype not in _FLOATS or x.device != self.device or len(s) not in (3, 4) or s[-1] != self.head_dim or \
                (heads is not None and s[-2] != heads):
            raise ValueError(f"{name} must be float32 or bfloat16 (T, {heads or 'heads'}, {self.head_dim}) or (B, T, "
                             f"{heads or 'heads'}, {self.head_dim}) on {self.device}, got {x.dtype} {tuple(s)} on {x.device}")
        if like is not None and (x.dtype is not like.dtype or len(s) != like.dim() or s[:-2] != like.shape[:-2]):
            raise ValueError(f"{name} must have k's dtype and rows, {like.dtype} {tuple(like.shape)}, got {x.dtype} "
                             f"{tuple(s)}")
        return (s[0], max(s[0], 1)) if len(s) == 3 else (s[0] * s[1], max(s[1], 1))

    def _query_heads(self, q: torch.Tensor) -> int:
        heads = q.shape[-2]
        if heads < 1 or heads % self.kv_heads or heads > self._gemm.ROPE_MAX_HEADS:
            raise ValueError(f"q must have a multiple of {self.kv_heads} heads, got {heads}")
        return heads

    # -- calls ----------------------------------------------------------------------------------
    def append(self, q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor,
               lengths: torch.Tensor, query_starts: torch.Tensor | None = None, *, rotary: HipRotary | None = None,
               positions: torch.Tensor | None = None, q_weight: torch.Tensor | None = None,
               k_weight: torch.Tensor | None = None, eps: float = 1e-6) -> torch.Tensor | None:
        """Writes the rows of k and v to the cache, in one launch with what comes before it: the heads of q and k normed
        by `q_weight` and `k_weight` where given and turned by `rotary` for the tokens' places, or for `positions`
        (int32 or int64, of the rows' shape or (T,)). Returns the new q (contiguous, in its dtype), None for None.
        float32 or bfloat16. Two sequences of a call must not write to the same page."""
        n, seq = self._rows("k", k, self.kv_heads)
        self._rows("v", v, self.kv_heads, k)
        dev, dt, nd, dim = self.device, k.dtype, k.dim(), self.head_dim
        heads = 0
        if q is not None:
            self._rows("q", q, None, k)
            heads = self._query_heads(q)
        elif q_weight is not None:
            raise ValueError("q_weight needs q")
        where = self._where(table, lengths, query_starts, n, k.shape[0] if nd == 4 else None)
        qw, kw = _head_weight("q_weight", q_weight, dim, dt, dev), _head_weight("k_weight", k_weight, dim, dt, dev)
        rot, turns, inter, scale = 0, 0, False, 1.0
        if rotary is not None:
            if rotary.head_dim != dim:
                raise ValueError(f"rotary must be for heads of {dim} values, got {rotary.head_dim}")
            rot, turns, inter, scale = rotary.rotary_dim, rotary._table(dev).data_ptr(), rotary.interleaved, rotary.scale
        pos, pos64, pos_batch, pos_tok = 0, False, 0, 0
        if positions is not None:
            ps = positions.shape
            if positions.dtype not in _INTS or positions.device != dev or ps not in (k.shape[:-2], k.shape[nd - 3 : nd - 2]):
                raise ValueError(f"positions must be int32 or int64 {tuple(k.shape[:-2])} on {dev}, got {positions.dtype} "
                                 f"{tuple(ps)} on {positions.device}")
            pos, pos64, pos_tok = positions.data_ptr(), positions.dtype is torch.int64, positions.stride(-1)
            pos_batch = positions.stride(0) if len(ps) == 2 else 0
        if _elsewhere(dev):
            with torch.cuda.device(dev):
                return self.append(q, k, v, table, lengths, query_starts, rotary=rotary, positions=positions,
                                   q_weight=q_weight, k_weight=k_weight, eps=eps)
        q_ptr, q_strides, out, out_ptr = 0, None, None, 0
        if q is not None:
            q, q_strides = _head_strides(q, nd)
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
            q_ptr, out_ptr = q.data_ptr(), out.data_ptr()
        if n == 0:
            return out
        k, k_strides = _head_strides(k, nd)
        v, v_strides = _head_strides(v, nd)
        status = self._lib.mxa_kv4_append(
            q_ptr, q_strides, heads, 0 if qw is None else qw.data_ptr(), k.data_ptr(), k_strides,
            0 if kw is None else kw.data_ptr(), v.data_ptr(), v_strides, float(eps), pos, pos64, pos_batch, pos_tok, turns,
            n, seq, rot, inter, scale, dt is _BF16, *where, out_ptr, _stream(dev))
        if status != 0:
            self._gemm._check(status, "mxa_kv4_append", 0)
        return out

    def attend(self, q: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor,
               query_starts: torch.Tensor | None = None, *, scale: float | None = None, window: int = 0,
               max_length: int | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
        """Causal attention of the rows of q (bfloat16; a multiple of kv_heads heads, neighbouring ones sharing a key
        head) over their sequences' cached places up to their own, the last `window` of them if that is positive:
        softmax(scale * q . k) v, `scale` 1 / sqrt(head_dim) unless given. Returns a contiguous bfloat16 tensor of q's
        shape, or `out`. A row that attends to nothing is zeros; rows of no sequence are zeros, in `out` as they were.

        One token, a few, a chunk, or any mixture. `max_length` (the table's places unless given) bounds the lengths for
        sharing out the work: a captured call should give what the lengths will grow to. A token's result does not
        depend on what other sequences are in the call, but by rounding on how many rows and places share the work."""
        n, seq = self._rows("q", q, None)
        nd, dev = q.dim(), self.device
        if q.dtype is not _BF16:
            raise ValueError(f"q must be bfloat16, got {q.dtype}")
        heads = self._query_heads(q)
        if n * heads > self.MAX_ROWS:
            raise ValueError(f"q must have up to {self.MAX_ROWS} tokens times heads, got {tuple(q.shape)}")
        where = self._where(table, lengths, query_starts, n, q.shape[0] if nd == 4 else None)
        places = table.shape[1] * self.page_size
        most = places if max_length is None else min(max(int(max_length), 1), places)
        window = int(window)
        if not 0 <= window < 1 << 31:
            raise ValueError(f"window must not be negative, got {window}")
        if out is not None and (out.dtype is not _BF16 or out.shape != q.shape or out.device != dev
                                or not out.is_contiguous()):
            raise ValueError(f"out must be contiguous bfloat16 {tuple(q.shape)} on {dev}, got {out.dtype} "
                             f"{tuple(out.shape)} on {out.device}")
        if _elsewhere(dev):
            with torch.cuda.device(dev):
                return self.attend(q, table, lengths, query_starts, scale=scale, window=window, max_length=max_length,
                                   out=out)
        q, q_strides = _head_strides(q, nd)
        if out is None:
            make = torch.empty_like if query_starts is None else torch.zeros_like
            out = make(q, memory_format=torch.contiguous_format)
        if n == 0:
            return out
        lib = self._lib
        size = lib.mxa_kv4_attend_workspace_bytes(where[-1], n, query_starts is not None, heads, self.kv_heads,
                                                  self.head_dim, most, window)
        ws = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
        status = lib.mxa_kv4_attend(
            q.data_ptr(), q_strides, heads, n, seq, *where, most, window,
            1.0 / math.sqrt(self.head_dim) if scale is None else float(scale), out.data_ptr(),
            0 if ws is None else ws.data_ptr(), size, _stream(dev))
        if status != 0:
            self._gemm._check(status, "mxa_kv4_attend", 0)
        return out

    def read(self, n_tokens: int, table: torch.Tensor, lengths: torch.Tensor, query_starts: torch.Tensor | None = None,
             *, dtype: torch.dtype = _BF16) -> tuple[torch.Tensor, torch.Tensor]:
        """The keys and values that the last tokens of the sequences are held as, (n_tokens, kv_heads, head_dim) each:
        n_tokens / B of each sequence, or rows as `query_starts` has them. Zeros for what is not cached."""
        if dtype not in _FLOATS:
            raise ValueError(f"dtype must be float32 or bfloat16, got {dtype}")
        n, dev = int(n_tokens), self.device
        if n < 0:
            raise ValueError(f"n_tokens must not be negative, got {n_tokens}")
        where = self._where(table, lengths, query_starts, n, None)
        if _elsewhere(dev):
            with torch.cuda.device(dev):
                return self.read(n, table, lengths, query_starts, dtype=dtype)
        k = torch.empty((n, self.kv_heads, self.head_dim), dtype=dtype, device=dev)
        v = torch.empty_like(k)
        if n:
            status = self._lib.mxa_kv4_read(*where, n, dtype is _BF16, k.data_ptr(), v.data_ptr(), _stream(dev))
            if status != 0:
                self._gemm._check(status, "mxa_kv4_read", 0)
        return k, v
