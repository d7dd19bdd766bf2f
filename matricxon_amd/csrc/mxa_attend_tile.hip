// Causal attention over the 4-bit cache for many rows (mxa_attend.hip has the mathematics and the form for few rows): a
// workgroup takes 32 rows a wave of one key head, and widens each tile of 64 places once for all of them, into LDS in the
// order of the matrix instructions' operands:
//
//   scores^T = K q^T    32 keys by 32 rows, 16 of a head's values an instruction
//   o^T     += V^T p^T  32 of a head's values by 32 rows, 16 places an instruction; p as the scores come out
//
// The codes of the next tile are requested before a tile is computed, and widened into the other half of LDS behind it.
#include "mxa_attend.hpp"
#include "mxa_kernels.hpp"

#pragma clang fp contract(off)

namespace mxa {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));

constexpr int kTilePlaces = 2 * kKvBlock;

template <int W>
struct TileShape {
  static constexpr int waves = W <= 4 ? 8 : 4;  // two to a SIMD where their registers allow
  static constexpr int threads = 64 * waves, rows = 32 * waves;
  static constexpr int key_waves = waves / 2;   // widen keys; the others widen values
  static constexpr int octets = 8 / waves * 1;  // of a token's four, that a lane of a key wave has: 1 or 2
  static constexpr int pairs = (W + 1) / 2;     // pairs of groups
  static constexpr int items = (2 * pairs + waves / 2 - 1) / (waves / 2);  // (block, pair) that a value wave has at most
  static constexpr int frags = 4 * W;           // operands of 1 KB: keys' of a tile, and as many of values
};

// A thread's codes and scales of the next tile, as loaded.
template <int W>
struct Staged {
  using S = TileShape<W>;
  union {
    struct {
      uint32_t codes[S::octets][W], scales[W];
    } key;
    struct {
      uint32_t codes[S::items][4];
      u32x4 scales[S::items][4];
    } value;
  };
};

template <int W>
__global__ __launch_bounds__(TileShape<W>::threads, W <= 4 ? 2 : 1) void attend_tile_kernel(AttendArgs a) {
  using S = TileShape<W>;
  extern __shared__ __align__(16) unsigned char smem[];
  half8* const lds = (half8*)smem;  // [half of LDS][keys' operands, values' operands][lane]
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 31, g = lane >> 5;
  const int h = blockIdx.x % a.kv.heads, split = blockIdx.y;
  int b, tile;
  if (!find_tile(a, blockIdx.x / a.kv.heads, S::rows, b, tile)) return;
  const Sequence seq(a, b);
  if (split >= seq.splits) return;
  const int row0 = tile * S::rows, row = row0 + wave * 32 + n;
  const bool live = row < seq.rows;
  const int place = seq.place0 + (live ? row / a.group : 0);
  const int limit = live ? min(place + 1, seq.length) : 0, low = a.window > 0 ? max(place + 1, 0) - a.window : 0;
  // blocks that some row of the workgroup attends to
  const int last = min(row0 + S::rows, seq.rows) - 1;
  const int hi = min(max(seq.place0 + last / a.group + 1, 0), seq.length);
  const int lo = a.window > 0 ? max(max(seq.place0 + row0 / a.group + 1, 0) - a.window, 0) : 0;
  const int begin = max(seq.first_block + split * seq.chunk, lo / kKvBlock);
  const int end = min(min(seq.first_block + min((split + 1) * seq.chunk, seq.blocks), (hi + kKvBlock - 1) / kKvBlock),
                      a.kv.width * (a.kv.page / kKvBlock));
  const CodeBits bits;

  // q, by a power of two
  half8 q[2 * W];
  float back;
  {
    const uint16_t* const src = a.q_row(seq.first + (live ? row / a.group : 0), h * a.group + (live ? row % a.group : 0));
    u16x8 raw[2 * W];
    float top = 0.0f;
#pragma unroll
    for (int k = 0; k < 2 * W; ++k) {
      raw[k] = u16x8{};
      if (live && 16 * k + 8 * g < a.dim) raw[k] = *(const u16x8*)(src + 16 * k + 8 * g);
#pragma unroll
      for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(bf16_to_float(raw[k][j])));
    }
    top = fmaxf(top, __shfl_xor(top, 32));
    const int e = row_exponent(top);
#pragma unroll
    for (int k = 0; k < 2 * W; ++k) {
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = bf16_to_float(raw[k][j]);
      q[k] = key_order(v, -e);
    }
    if (a.scale < 0.0f)  // its sign goes to q: the largest product is the largest score
#pragma unroll
      for (int k = 0; k < 2 * W; ++k) q[k] = -q[k];
    back = fmaxf(ldexpf(fabsf(a.scale) * kLog2e, e), 1e-37f);  // not 0, with which a place left out would be no number
  }
  f32x16 o[W];
#pragma unroll
  for (int i = 0; i < W; ++i)
#pragma unroll
    for (int j = 0; j < 16; ++j) o[i][j] = 0.0f;
  float m = kLowest, l = 0.0f;
  const int wave_last = min(row0 + wave * 32 + 31, seq.rows - 1);
  const int inside_lo = a.window > 0 ? max(seq.place0 + wave_last / a.group + 1, 0) - a.window : 0;
  const int inside_hi = min(seq.place0 + (row0 + wave * 32) / a.group + 1, seq.length);

  // Lane i knows where the i-th of 64 blocks lies; every wave looks up the same.
  const int blocks_of_page = a.kv.page / kKvBlock;
  long long where = -1;
  int looked = begin - 64;  // the block that lane 0 has
  const auto block_at = [&](int u) -> long long {  // -1: no page, or behind the last
    if (u >= end) return -1;
    if (u >= looked + 64) {
      looked = u;
      const long long block = u + lane < end ? kv_block(a.kv, b, (u + lane) * kKvBlock) : -1;
      where = block < 0 ? -1 : (block + (long long)h * blocks_of_page) * kv_block_bytes(W);
    }
    const uint32_t w0 = __builtin_amdgcn_readlane((int)(uint32_t)where, u - looked);
    const uint32_t w1 = __builtin_amdgcn_readlane((int)(where >> 32), u - looked);
    return (long long)((uint64_t)w1 << 32 | w0);
  };
  int next0 = 0, next1 = 0;  // places of the requested tile's blocks that are the sequence's
  Staged<W> st;
  const bool key_wave = wave < S::key_waves;
  // key wave w: block w / (waves / 4) of the tile; with 8 waves two to a block, an octet a lane, else two octets a lane
  const int key_block = (wave * 4 / S::waves) & 1, key_octet = S::waves == 8 ? (wave & 1) * 2 + g : 2 * g;
  const auto request = [&](int u) {
    const long long w0 = block_at(u), w1 = block_at(u + 1);
    // no page: any block, none of whose places count
    const uint8_t *const at0 = a.kv.pages + max(w0, 0LL), *const at1 = a.kv.pages + max(w1, 0LL);
    next0 = w0 < 0 ? 0 : min(seq.length - u * kKvBlock, kKvBlock);
    next1 = w1 < 0 ? 0 : min(seq.length - (u + 1) * kKvBlock, kKvBlock);
    if (key_wave) {
      const uint8_t* const blk = key_block ? at1 : at0;
#pragma unroll
      for (int c = 0; c < S::octets; ++c)
#pragma unroll
        for (int w = 0; w < W; ++w)
          st.key.codes[c][w] = *(const uint32_t*)(blk + n * 16 * W + (key_octet + c) * 4 * W + w * 4);
#pragma unroll
      for (int w = 0; w < W; ++w) st.key.scales[w] = *(const uint32_t*)(blk + kv_key_scales(W) + (n * W + w) * 4);
    } else {
#pragma unroll
      for (int t = 0; t < S::items; ++t) {
        const int item = (wave - S::key_waves) + t * (S::waves - S::key_waves);
        if (item >= 2 * S::pairs) break;
        const uint8_t* const blk = item & 1 ? at1 : at0;
        const int pair = item >> 1, i = lane & 15, quad = lane >> 4;
        const bool two = 2 * pair + 1 < W;
#pragma unroll
        for (int k = 0; k < 4; ++k) {  // (group of the pair, half)
          if (k >= 2 && !two) break;
          const int group = 2 * pair + (k >> 1);
          st.value.codes[t][k] = *(const uint32_t*)(blk + kv_value_codes(W) + kv_value_word(W, group, quad, i, k & 1));
          st.value.scales[t][k] = *(const u32x4*)(blk + kv_value_scales(W) + (group * 8 + (k & 1) * 4 + quad) * 16);
        }
      }
    }
  };
  const auto widen = [&](half8* to) {
    if (key_wave) {
#pragma unroll
      for (int c = 0; c < S::octets; ++c)
#pragma unroll
        for (int w = 0; w < W; ++w) {
          const int octet = key_octet + c;
          to[(key_block * 2 * W + 2 * w + (octet >> 1)) * 64 + (octet & 1) * 32 + n] =
              widen8(bits, st.key.codes[c][w], st.key.scales[w]);
        }
    } else {
      half4* const vt = (half4*)(to + S::frags * 64);
#pragma unroll
      for (int t = 0; t < S::items; ++t) {
        const int item = (wave - S::key_waves) + t * (S::waves - S::key_waves);
        if (item >= 2 * S::pairs) break;
        const int blk = item & 1, pair = item >> 1, i = lane & 15, quad = lane >> 4;
        const bool two = 2 * pair + 1 < W;
        const int have = blk ? next1 : next0;
        if (have < kKvBlock) {  // behind the sequence's end, or no page: whatever is there, 0
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int first = (k & 1) * 16 + quad * 4;
            const uint32_t keep02 = (first < have ? 0xFFFFu : 0u) | (first + 2 < have ? 0xFFFF0000u : 0u);
            const uint32_t keep13 = (first + 1 < have ? 0xFFFFu : 0u) | (first + 3 < have ? 0xFFFF0000u : 0u);
            u32x4& sm = st.value.scales[t][k];
            sm[0] &= keep02, sm[1] &= keep13, sm[2] &= keep02, sm[3] &= keep13;
          }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (k >= 2 && !two) break;
          half4 v0, v1;
          value4(bits, st.value.codes[t][k], st.value.scales[t][k], v0, v1);
          half4* const p = vt + ((((blk * 2 + (k & 1)) * W + 2 * pair + (k >> 1)) * 64 + (quad & 1) * 32 + 2 * i) * 2 + (quad >> 1));
          p[0] = v0;
          p[2] = v1;
        }
      }
    }
  };

  int turn = 0;  // the half of LDS that holds the present tile
  int have0 = 0, have1 = 0;
  if (begin < end) {
    request(begin);
    widen(lds);
    have0 = next0, have1 = next1;
  }
  __syncthreads();
  for (int u = begin; u < end; u += 2) {
    const half8* const kt = lds + turn * 2 * S::frags * 64;
    const half8* const vt = kt + S::frags * 64;
    const bool more = u + 2 < end;
    if (more) request(u + 2);
    f32x16 s[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 16; ++j) s[i][j] = 0.0f;
#pragma unroll
    for (int k = 0; k < 2 * W; ++k)
#pragma unroll
      for (int i = 0; i < 2; ++i)
        s[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kt[(i * 2 * W + k) * 64 + lane], q[k], s[i], 0, 0, 0);
    const int first = u * kKvBlock;
    const bool inside = have0 == kKvBlock && have1 == kKvBlock && first >= inside_lo && first + kTilePlaces <= inside_hi;
    if (!inside) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const int t = j / 4 * 8 + g * 4 + j % 4, at = first + i * kKvBlock + t;
          if (t >= (i ? have1 : have0) || at >= limit || at < low) s[i][j] = -INFINITY;
        }
    }
    // p against the row's reference so far: a sum within float16's range says that every p is. A row's first places, whose
    // reference is the lowest of all, sum to +inf.
    half8 p[4];
    float sum = 0.0f;
    const auto probabilities = [&]() {
      const float ref = kProbShift - m;
      sum = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float e[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          e[j] = exp2_(fmaf(s[i >> 1][(i & 1) * 8 + j], back, ref));
          sum += e[j];
        }
        p[i] = prob_order(e);
      }
    };
    probabilities();
    if (__any(!(sum <= kProbMost))) {
      float top = s[0][0];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) top = fmaxf(top, s[i][j]);
      top = fmaxf(top, __shfl_xor(top, 32));
      const float m2 = fmaxf(m, top * back), alpha = exp2_(m - m2);
      m = m2;
      l *= alpha;
#pragma unroll
      for (int i = 0; i < W; ++i) o[i] *= alpha;
      probabilities();
    }
    l += sum;
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int i = 0; i < W; ++i)
        o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vt[(k * W + i) * 64 + lane], p[k], o[i], 0, 0, 0);
    if (more) {
      turn ^= 1;
      widen(lds + turn * 2 * S::frags * 64);
      have0 = next0, have1 = next1;
    }
    __syncthreads();
  }
  l += __shfl_xor(l, 32);
  if (!live) return;
  if (seq.splits == 1) {
    const float norm = l > 0.0f || l != l ? 1.0f / l : 0.0f;
    uint16_t* const dst = a.out_row(seq.first + row / a.group, h * a.group + row % a.group);
#pragma unroll
    for (int i = 0; i < W; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int d = 32 * i + 8 * j + 4 * g;
        if (d < a.dim) {
          typedef uint16_t u16x4 __attribute__((ext_vector_type(4), aligned(2)));
          u16x4 v;
#pragma unroll
          for (int k = 0; k < 4; ++k) v[k] = bf16_rne(o[i][4 * j + k] * norm);
          *(u16x4*)(dst + d) = v;
        }
      }
  } else {
    const AttendPart part = a.part_of(b, row / 16 * a.kv.heads + h, split, W);
    if (g == 0) {
      part.ml[row % 16] = m;
      part.ml[16 + row % 16] = l;
    }
#pragma unroll
    for (int i = 0; i < W; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        f32x4 v;
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = o[i][4 * j + k];
        *(f32x4*)(part.o + (row % 16) * 32 * W + 32 * i + 8 * j + 4 * g) = v;
      }
  }
}

template <int W>
void launch_w(const AttendArgs& a, long long tiles, hipStream_t stream) {
  using S = TileShape<W>;
  constexpr size_t lds = 4 * (size_t)S::frags * 1024;
  static const hipError_t once =
      hipFuncSetAttribute((const void*)attend_tile_kernel<W>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
  (void)once;
  hipLaunchKernelGGL(attend_tile_kernel<W>, dim3((unsigned)(tiles * a.kv.heads), a.splits), dim3(S::threads), lds,
                     stream, a);
}

}  // namespace

int attend_tile_rows(int dim) { return kv_groups(dim) <= 4 ? TileShape<4>::rows : TileShape<8>::rows; }

void launch_attend_tile(const AttendArgs& a, long long tiles, hipStream_t stream) {
  switch (kv_groups(a.dim)) {
#define MXA_CASE(W) \
  case W: launch_w<W>(a, tiles, stream); break;
    MXA_CASE(1) MXA_CASE(2) MXA_CASE(3) MXA_CASE(4) MXA_CASE(5) MXA_CASE(6) MXA_CASE(7) MXA_CASE(8)
#undef MXA_CASE
  }
}

}  // namespace mxa
