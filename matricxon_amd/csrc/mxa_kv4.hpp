// The paged cache of 4-bit keys and values: how its bytes lie, shared by the kernels that write, read and attend over it.
//
// 32 neighbouring values of a token's head (a group) share a float16 scale s and minimum m, a value being s * code + m.
// A page holds its tokens for every key head in blocks of 32 tokens; a block of W groups is 1280 W bytes:
//
//   0       key codes     [token 32][octet 4][group W][4 bytes], a byte two neighbouring values, the first in its low bits
//   512 W   key scales    [token 32][group W](s, m)
//   640 W   value codes   a byte two neighbouring values of a token, in words of four neighbouring tokens (below)
//   1152 W  value scales  [group W][quad of tokens 8](s0 s2 s1 s3 m0 m2 m1 m3)
//
// The order is that of the matrix instructions' operands, so that a lane's codes are adjacent and are widened in its
// registers: of 16 keys lane l holds octet l / 16 of each group of token l % 16; of 32 tokens' values lane l holds values
// 2 (l % 16) and 2 (l % 16) + 1 of each group for tokens 4 (l / 16) .. + 3 and 16 + 4 (l / 16) .. + 3. A pair in a byte is
// two dimensions of one token, never two tokens: a token is appended without reading its neighbours' bytes.
#pragma once

#include "mxa_device.hpp"
#include "mxa_kv4_shape.hpp"

namespace mxa {

constexpr float kKvHeld = 65000.0f;    // values beyond are held as this: s * 15 + m then stays a finite float16

__host__ __device__ constexpr int kv_block_bytes(int w) { return 1280 * w; }
__host__ __device__ constexpr int kv_key_scales(int w) { return 512 * w; }
__host__ __device__ constexpr int kv_value_codes(int w) { return 640 * w; }
__host__ __device__ constexpr int kv_value_scales(int w) { return 1152 * w; }

// Byte offset in the value codes of the word of tokens 16 half + 4 quad .. + 3 and value pair i of a group.
__device__ __forceinline__ int kv_value_word(int w, int group, int quad, int i, int half) {
  const int lane = quad * 16 + i, pair = group >> 1;
  if (group < (w & ~1)) return pair * 1024 + lane * 16 + (group & 1) * 8 + half * 4;
  return pair * 1024 + lane * 8 + half * 4;
}

// Where a sequence's tokens lie.
struct KvPages {
  uint8_t* pages;
  const int32_t* table;    // n_seq rows of `width` page numbers, `stride` apart
  const int32_t* lengths;  // tokens of each sequence, the call's own among them
  const int32_t* starts;   // n_seq + 1 rows at which the sequences' tokens begin, or nullptr: `each` of every sequence
  long long stride;
  int n_pages, heads, page, width, n_seq, each;
};

// The rows [first, first + count) of the call that are sequence b's; never outside [0, n_tokens).
__host__ __device__ inline void kv_rows_of(const KvPages& p, int b, int n_tokens, int& first, int& count) {
  if (p.starts == nullptr) {
    first = b * p.each;
    count = p.each;
    return;
  }
  const int begin = p.starts[b], end = p.starts[b + 1] < n_tokens ? p.starts[b + 1] : n_tokens;
  first = begin < 0 ? 0 : begin > n_tokens ? n_tokens : begin;
  count = end > first ? end - first : 0;
}

// The block (of one head at 0) of a place, or -1 where the table has no page for it.
__host__ __device__ inline long long kv_block(const KvPages& p, int b, int place) {
  if (place < 0) return -1;
  const int entry = place / p.page;
  if (entry >= p.width) return -1;
  const int page = p.table[(long long)b * p.stride + entry];
  if (page < 0 || page >= p.n_pages) return -1;
  return (long long)page * p.heads * (p.page / kKvBlock) + (place - entry * p.page) / kKvBlock;
}

// A sequence's length, held to where sums with it do not overflow (no more than 2^30 places can be cached).
__host__ __device__ inline int kv_length(const KvPages& p, int b) {
  const int n = p.lengths[b], most = (1 << 30) + (1 << 25);
  return n < -most ? -most : n > most ? most : n;
}

// Sequence and place of row t of the call; sequence -1: of none.
__host__ __device__ inline int kv_place(const KvPages& p, int t, int n_tokens, int& place) {
  int b = -1;
  place = 0;
  if (p.starts == nullptr) {
    b = t / p.each;
    place = kv_length(p, b) - p.each + (t - b * p.each);
    return b;
  }
  int lo = 0, hi = p.n_seq;  // the last b with starts[b] <= t
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (p.starts[mid] <= t)
      lo = mid + 1;
    else
      hi = mid;
  }
  b = lo - 1;
  if (b < 0) return -1;
  const int end = p.starts[b + 1] < n_tokens ? p.starts[b + 1] : n_tokens;
  if (t >= end) return -1;
  place = kv_length(p, b) - end + t;
  return b;
}

struct Spot {      // of one token of a workgroup
  long long at;    // byte offset of its block of the first head in the pages, or -1: it has none
  int place, seq;  // seq -1: a row of no sequence
};
__device__ __forceinline__ Spot kv_spot(const KvPages& p, int t, int n_tokens, int W) {
  Spot s;
  s.seq = kv_place(p, t, n_tokens, s.place);
  const long long block = s.seq < 0 ? -1 : kv_block(p, s.seq, s.place);
  s.at = block < 0 ? -1 : block * kv_block_bytes(W);
  return s;
}

// V adjacent values, and their rounding.
template <class T, int V>
struct Vec {
  typedef T type __attribute__((ext_vector_type(V), aligned(sizeof(T))));
};

template <class T, int V>
__device__ __forceinline__ typename Vec<T, V>::type narrow_all(const float (&v)[V]) {
  typename Vec<T, V>::type r;
#pragma unroll
  for (int i = 0; i < V; i += 2) {
    if constexpr (sizeof(T) == 2) {
      typedef float f2 __attribute__((ext_vector_type(2)));
      typedef __bf16 b2 __attribute__((ext_vector_type(2)));
      const uint32_t w = __builtin_bit_cast(uint32_t, __builtin_convertvector((f2){v[i], v[i + 1]}, b2));
      r[i] = (uint16_t)w, r[i + 1] = (uint16_t)(w >> 16);
    } else {
      r[i] = v[i], r[i + 1] = v[i + 1];
    }
  }
  return r;
}

// Heads normed and turned, with a cache or without (mxa_heads.hip); cached values read back (mxa_kv4.hip).
int launch_heads(const void* q, const long long* q_strides, int q_heads, const void* q_weight, const void* k,
                 const long long* k_strides, int k_heads, const void* k_weight, float eps, const void* pos, bool pos64,
                 long long pos_batch, long long pos_tok, const double* turns, int n_tokens, int seq, int dim, int rot,
                 bool interleaved, float mscale, bool bf16, void* q_out, void* k_out, hipStream_t stream);
int launch_kv4_append(const void* q, const long long* q_strides, int q_heads, const void* q_weight, const void* k,
                      const long long* k_strides, const void* k_weight, const void* v, const long long* v_strides,
                      float eps, const void* pos, bool pos64, long long pos_batch, long long pos_tok,
                      const double* turns, int n_tokens, int seq, int dim, int rot, bool interleaved, float mscale,
                      bool bf16, const KvPages& kv, void* q_out, hipStream_t stream);
int launch_kv4_read(const KvPages& kv, int n_tokens, int dim, bool bf16, void* k_out, void* v_out, hipStream_t stream);

}  // namespace mxa
