// What the attention kernels over the 4-bit cache share: their arguments, which rows a workgroup has, operands from codes.
#pragma once

#include "mxa_attend_plan.hpp"
#include "mxa_kv4.hpp"

namespace mxa {

constexpr float kLog2e = 1.4426950408889634f;
// exp(s - max) is held times 2^8, so that a probability keeps its bits in float16 down to 2^-22 of the largest.
constexpr float kProbShift = 8.0f;
// A row's reference is its maximum so far, or up to this (log2) below: its sums are rescaled only where a score passes it
// by more. A probability then is at most 2^15, within float16.
constexpr float kSlack = 7.0f;
constexpr float kProbMost = 32768.0f;
constexpr float kLowest = -3e38f;  // the reference of a row that has seen no place

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

typedef uint16_t u16x8 __attribute__((ext_vector_type(8), aligned(2)));

__device__ __forceinline__ float exp2_(float v) { return __builtin_amdgcn_exp2f(v); }

// A split's part of a pair's rows, unnormalised.
struct AttendPart {
  float* o;   // 16 rows of 32 W values
  float* ml;  // 16 references of log2 p, 16 sums
};

struct AttendArgs {
  const uint16_t* q;
  uint16_t* out;  // contiguous (n_tokens, heads, dim)
  float* part;
  long long q_batch, q_tok, q_head;  // strides in elements
  KvPages kv;
  int n_tokens, seq, dim, heads, group, window;  // token t is step t % seq of q's batch entry t / seq
  int least_rows, most_rows;  // sequences of fewer or more rows a key head are left out
  int pairs, splits, chunk;  // of the grid: pairs and splits of a sequence, blocks of a split at least (0: each tile in
                             // `splits` even parts)
  int compact;               // the grid has the tiles of the call, not as many for each sequence
  int per;                   // tiles that the parts have room for of each sequence; 0: as they lie in the call
  float scale;

  __device__ __forceinline__ const uint16_t* q_row(int t, int h) const {
    const int b = seq >= n_tokens ? 0 : t / seq;
    return q + (long long)b * q_batch + (long long)(t - b * seq) * q_tok + (long long)h * q_head;
  }
  __device__ __forceinline__ uint16_t* out_row(int t, int h) const { return out + ((long long)t * heads + h) * dim; }
  // Of tile rt of sequence b, whose rows begin at `first`. As they lie in the call: as each sequence has one tile of 16 rows
  // more than its rows' share of the call's at most, the tiles of those before it are first * group / 16 + b and fewer.
  __device__ __forceinline__ AttendPart part_of(int b, int first, int rt, int h, int split, int w) const {
    const long long tile = per > 0 ? (long long)b * per + rt : (long long)first * group / 16 + b + rt;
    float* const p = part + ((tile * kv.heads + h) * splits + split) * (16 * 32 * w + 32);
    return AttendPart{p, p + 16 * 32 * w};
  }
};

// What the call has of a sequence. Its rows of one key head (token i and query head of the group: row i * group + head)
// go in tiles of 16; a (key head, tile) is a pair, and a pair has `blocks` blocks of places, one at least.
struct Sequence {
  int first, count;    // rows of the call
  int rows, tiles;     // of one key head; 0: none, or another kernel's
  int length, place0;  // its tokens, the place of its first row
  int first_block, blocks;
  int chunk, splits;  // blocks of a split, splits that have any
  // The same in scalar registers, where b is one for all lanes.
  __device__ __forceinline__ Sequence uniform() const {
    Sequence s = *this;
    s.first = __builtin_amdgcn_readfirstlane(first), s.count = __builtin_amdgcn_readfirstlane(count);
    s.rows = __builtin_amdgcn_readfirstlane(rows), s.tiles = __builtin_amdgcn_readfirstlane(tiles);
    s.length = __builtin_amdgcn_readfirstlane(length), s.place0 = __builtin_amdgcn_readfirstlane(place0);
    s.first_block = __builtin_amdgcn_readfirstlane(first_block), s.blocks = __builtin_amdgcn_readfirstlane(blocks);
    s.chunk = __builtin_amdgcn_readfirstlane(chunk), s.splits = __builtin_amdgcn_readfirstlane(splits);
    return s;
  }
  __host__ __device__ inline Sequence(const AttendArgs& a, int b) {
    kv_rows_of(a.kv, b, a.n_tokens, first, count);
    const long long all = (long long)count * a.group;
    rows = all >= a.least_rows && all <= a.most_rows ? (int)all : 0;
    tiles = (rows + 15) / 16;
    const int known = kv_length(a.kv, b);
    place0 = known - count;
    length = known < 0 ? 0 : known < a.kv.width * a.kv.page ? known : a.kv.width * a.kv.page;
    int lo = a.window > 0 ? (place0 + 1 > 0 ? place0 + 1 : 0) - a.window : 0;
    lo = lo < 0 ? 0 : lo > length ? length : lo;
    first_block = lo / kKvBlock;
    blocks = (length + kKvBlock - 1) / kKvBlock - first_block;
    if (blocks < 1) blocks = 1;
    const int least = (blocks + a.splits - 1) / a.splits;  // more where a length passes what the host was told
    chunk = a.chunk > least ? a.chunk : least;
    splits = a.chunk > 0 ? (blocks + chunk - 1) / chunk : a.splits;
  }
};

// The sequence and the tile (of `rows` rows a key head, the last first: those attend to most) that tile `flat` of the call
// is; false behind the last. Lanes look at 64 sequences at a time.
__device__ __forceinline__ bool find_tile(const AttendArgs& a, int flat, int rows, int& b, int& tile) {
  const int lane = threadIdx.x & 63;
  for (int base = 0; base < a.kv.n_seq; base += 64) {
    int tiles = 0;
    if (base + lane < a.kv.n_seq) tiles = (Sequence(a, base + lane).rows + rows - 1) / rows;
    int run = tiles;
#pragma unroll
    for (int i = 1; i < 64; i *= 2) {
      const int other = __shfl_up(run, i);
      if (lane >= i) run += other;
    }
    const unsigned long long past = __ballot(run > flat);
    if (past != 0) {
      const int at = __builtin_ctzll(past);
      b = base + at;
      tile = __builtin_amdgcn_readlane(run, at) - 1 - flat;
      return true;
    }
    flat -= __builtin_amdgcn_readlane(run, 63);
  }
  return false;
}

// The power of two that a row of q is divided by: its largest value then lies in [2^10, 2^11).
__device__ __forceinline__ int row_exponent(float top) {
  int e = 0;
  if (top > 0.0f && top < INFINITY) frexpf(top, &e), e -= 11;
  return e;
}

// Eight neighbouring values times 2^e in the order in which a word of codes is widened: 0 4 1 5 2 6 3 7.
__device__ __forceinline__ half8 key_order(const float (&v)[8], int e) {
  half8 h;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    h[2 * j] = (_Float16)ldexpf(v[j], e);
    h[2 * j + 1] = (_Float16)ldexpf(v[4 + j], e);
  }
  return h;
}

// The float16 pairs of a word's codes, nibbles 0 and 4, 1 and 5, 2 and 6, 3 and 7: 1024 + c is 0x6400 | c, and 64 + c is
// 0x5400 | c << 4.
struct CodeBits {
  uint32_t low, high, k1024, k64;
  __device__ __forceinline__ CodeBits() : low(0x000F000Fu), high(0x00F000F0u), k1024(0x64006400u), k64(0x54005400u) {
    // in registers, masks scalar and the others not: an and and an or then are one instruction, which takes no constant
    // and one scalar register
    asm("" : "+s"(low), "+s"(high), "+v"(k1024), "+v"(k64));
  }
};
__device__ __forceinline__ void codes8(const CodeBits& b, uint32_t w, half2v (&c)[4]) {
  const half2v k1024{(_Float16)-1024.0f, (_Float16)-1024.0f}, k64{(_Float16)-64.0f, (_Float16)-64.0f};
  const uint32_t x = w >> 8;
  c[0] = __builtin_bit_cast(half2v, (w & b.low) | b.k1024) + k1024;
  c[1] = __builtin_bit_cast(half2v, (w & b.high) | b.k64) + k64;
  c[2] = __builtin_bit_cast(half2v, (x & b.low) | b.k1024) + k1024;
  c[3] = __builtin_bit_cast(half2v, (x & b.high) | b.k64) + k64;
}

// A word as two float16. (By value: a bit cast of a vector's element itself reads element 0.)
__device__ __forceinline__ half2v half2_of(uint32_t w) { return __builtin_bit_cast(half2v, w); }

// s * c + m, rounded once.
__device__ __forceinline__ half2v fma2(half2v c, half2v s, half2v m) { return __builtin_elementwise_fma(c, s, m); }

// Eight keys' or one key's eight values from a word of codes and (s, m).
__device__ __forceinline__ half8 widen8(const CodeBits& b, uint32_t w, uint32_t sm) {
  half2v c[4];
  codes8(b, w, c);
  const half2v p = half2_of(sm), s{p[0], p[0]}, m{p[1], p[1]};
  half8 h;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const half2v v = fma2(c[j], s, m);
    h[2 * j] = v[0], h[2 * j + 1] = v[1];
  }
  return h;
}

typedef _Float16 half4v __attribute__((ext_vector_type(4)));

// Two neighbouring values of four tokens, in the order 0 2 1 3, from a word and its scales: v0 the even value.
template <class H4>
__device__ __forceinline__ void value4(const CodeBits& bits, uint32_t w, u32x4 sm, H4& v0, H4& v1) {
  half2v c[4];
  codes8(bits, w, c);
  const half2v s02 = half2_of(sm[0]), s13 = half2_of(sm[1]), m02 = half2_of(sm[2]), m13 = half2_of(sm[3]);
  const half2v a = fma2(c[0], s02, m02), d = fma2(c[1], s02, m02), b = fma2(c[2], s13, m13), e = fma2(c[3], s13, m13);
  v0[0] = a[0], v0[1] = a[1], v0[2] = b[0], v0[3] = b[1];
  v1[0] = d[0], v1[1] = d[1], v1[2] = e[0], v1[3] = e[1];
}

// Two neighbouring values of eight tokens (four and four, words w and their scales) as operands: v0 the even value.
__device__ __forceinline__ void value_operands(const CodeBits& bits, const uint32_t (&w)[2], u32x4 sa, u32x4 sb, half8& v0,
                                               half8& v1) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    half4v a, b;
    value4(bits, w[i], i ? sb : sa, a, b);
#pragma unroll
    for (int j = 0; j < 4; ++j) v0[4 * i + j] = a[j], v1[4 * i + j] = b[j];
  }
}

// The probabilities of the lane's eight tokens in value_operands' order: 0 2 1 3 of each four.
__device__ __forceinline__ half8 prob_order(const float (&p)[8]) {
  half8 h;
#pragma unroll
  for (int i = 0; i < 8; i += 4) {
    h[i] = (_Float16)p[i], h[i + 1] = (_Float16)p[i + 2];
    h[i + 2] = (_Float16)p[i + 1], h[i + 3] = (_Float16)p[i + 3];
  }
  return h;
}

// A lane's part of a block as it is loaded: its codes, and W of the block's 64 W words of scales.
template <int W>
struct BlockPart {
  uint32_t kc[2][W], vc[W][2], sc[W];
  __device__ __forceinline__ void load(const uint8_t* blk, int lane) {
    const int n = lane & 15, g = lane >> 4;
    const uint32_t* const from = (const uint32_t*)(blk + (lane < 32 ? kv_key_scales(W) : kv_value_scales(W)));
#pragma unroll
    for (int j = 0; j < W; ++j) sc[j] = from[(lane & 31) * W + j];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int w = 0; w < W; ++w) kc[i][w] = *(const uint32_t*)(blk + (i * 16 + n) * 16 * W + g * 4 * W + w * 4);
#pragma unroll
    for (int w = 0; w < W; ++w)
#pragma unroll
      for (int i = 0; i < 2; ++i) vc[w][i] = *(const uint32_t*)(blk + kv_value_codes(W) + kv_value_word(W, w, g, n, i));
  }
  // The scales into the wave's 64 W words of LDS: keys' (token, group), then values'.
  __device__ __forceinline__ void share(uint32_t* lds, int lane) const {
#pragma unroll
    for (int j = 0; j < W; ++j) lds[lane * W + j] = sc[j];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
};

// Scales of places behind the sequence's end (`have` tokens of the block are its own) become 0: what a page holds there,
// another sequence's or none, may be no number, and 0 times that is none either.
template <int W>
__device__ __forceinline__ void clear_tail(uint32_t* sc, int lane, int have) {
  for (int i = lane; i < 32 * W; i += 64) {
    if (i / W >= have) sc[i] = 0;
    const int quad = i / 4 % 8, k = i % 2;  // word k of s (or m) has tokens k and k + 2 of the quad
    uint32_t v = sc[32 * W + i];
    if (quad * 4 + k >= have) v &= 0xFFFF0000u;
    if (quad * 4 + k + 2 >= have) v &= 0x0000FFFFu;
    sc[32 * W + i] = v;
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
}

size_t attend_workspace(int n_seq, int n_tokens, bool ragged, int kv_heads, int group, int max_length, int window, int dim);
// The form for many rows, of 256 (heads of up to 128 values) or 128 rows of a key head a workgroup.
void launch_attend_tile(const AttendArgs& a, int rows, long long tiles, hipStream_t stream);
constexpr int kAttendUnsupported = -1, kAttendWorkspace = -2;
int launch_attend(AttendArgs a, int max_length, void* workspace, size_t workspace_bytes, hipStream_t stream);

}  // namespace mxa
