// Causal attention over the 4-bit cache for many rows (mxa_attend.hip has the mathematics and the form for few rows): a
// workgroup takes 32 rows a wave of one key head, and widens each tile of 64 (or 32) places once for all of them, into LDS
// in the order of the matrix instructions' operands:
//
//   scores^T = K q^T    32 keys by 32 rows, 16 of a head's values an instruction
//   o^T     += V^T p^T  32 of a head's values by 32 rows, 16 places an instruction; p as the scores come out
//
// A tile's packed bytes are copied into a ring of LDS slots by copies that no wave waits for until they are widened, some
// tiles later.
//
// Matrix instructions bound it from below: 2048 tokens of 32 heads of 128 behind 6144 places take 297 us, 810 TFLOP/s, of
// which they alone would take some 200. A place is widened once for 256 rows (128 rows: 350 us, beside 290); two waves of a
// SIMD a step apart took 347 us to 306, and four slots of copies on their way that to 290, measured in one session on a
// card a little faster.
#include "mxa_attend.hpp"
#include "mxa_kernels.hpp"

#pragma clang fp contract(off)

namespace mxa {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kAhead = 6;  // operands read from LDS ahead of the instruction that takes them

// A barrier that waits for LDS alone: copies stay on their way.
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// W groups a head, NW waves.
template <int W, int NW>
struct TileShape {
  static constexpr int threads = 64 * NW, rows = 32 * NW;
  static constexpr int blocks = NW / 4;                 // of a tile
  static constexpr int value_waves = NW / 2;            // widen values; those before them keys
  static constexpr int pairs = (W + 1) / 2;             // pairs of groups
  static constexpr int items = (blocks * pairs + value_waves - 1) / value_waves;  // (block, pair) of a value wave at most
  static constexpr int frags = 2 * W * blocks;          // operands of 1 KB: a tile's keys, and as many of its values
  static constexpr int raw = blocks * 1280 * W;         // bytes of a tile in the cache
  static constexpr int copies = (320 * W + 1023) / 1024;  // of a wave, a tile: a quarter of a block
  static constexpr int ring = 4;                        // tiles in LDS as they are in the cache
  static constexpr size_t lds = 4 * (size_t)frags * 1024 + (size_t)ring * raw;
};

// A thread's share of a tile, as it is in the cache.
template <int W, int NW>
struct Packed {
  using S = TileShape<W, NW>;
  union {
    struct {
      uint32_t codes[W], scales[W];
    } key;
    struct {
      uint32_t codes[S::items][4];
      u32x4 scales[S::items][4];
    } value;
  };
};

template <int W, int NW>
__global__ __launch_bounds__(64 * NW, W <= 4 ? 2 : 1) void attend_tile_kernel(AttendArgs a) {
  using S = TileShape<W, NW>;
  constexpr int B = S::blocks;
  extern __shared__ __align__(16) unsigned char smem[];
  half8* const lds = (half8*)smem;  // [half of LDS][keys' operands, values' operands][lane]
  unsigned char* const raw = smem + 4 * S::frags * 1024;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 31, g = lane >> 5;
  const int h = blockIdx.x % a.kv.heads, split = blockIdx.y;
  int b, tile;
  if (!find_tile(a, blockIdx.x / a.kv.heads, S::rows, b, tile)) return;
  b = __builtin_amdgcn_readfirstlane(b), tile = __builtin_amdgcn_readfirstlane(tile);
  const Sequence seq = Sequence(a, b).uniform();
  const int row0 = tile * S::rows, row = row0 + wave * 32 + n;
  const bool live = row < seq.rows;
  const int place = seq.place0 + (live ? row / a.group : 0);
  const int limit = live ? min(place + 1, seq.length) : 0, low = a.window > 0 ? max(place + 1, 0) - a.window : 0;
  // blocks that some row of the workgroup attends to
  const int last = min(row0 + S::rows, seq.rows) - 1;
  const int hi = min(max(seq.place0 + last / a.group + 1, 0), seq.length);
  const int lo = a.window > 0 ? max(max(seq.place0 + row0 / a.group + 1, 0) - a.window, 0) : 0;
  const int first_block = lo / kKvBlock, blocks = max((hi + kKvBlock - 1) / kKvBlock - first_block, 0);
  const int part_blocks = ((blocks + a.splits - 1) / a.splits + B - 1) / B * B;
  const int begin = first_block + min(split * part_blocks, blocks), end = first_block + min((split + 1) * part_blocks, blocks);
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
    if (!(a.scale >= 0.0f)) {  // its sign goes to q: the largest product is the largest score; so does what is no number
      const _Float16 by = a.scale < 0.0f ? -1.0f : a.scale;
#pragma unroll
      for (int k = 0; k < 2 * W; ++k) q[k] *= by;
    }
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
  int looked = begin - 64;  // the block that lane 0 has (a multiple of 2 from begin: a tile's blocks are in one look)
  const auto look_up = [&](int u) {
    looked = u;
    const long long block = u + lane < end ? kv_block(a.kv, b, (u + lane) * kKvBlock) : -1;
    where = block < 0 ? -1 : (block + (long long)h * blocks_of_page) * kv_block_bytes(W);
  };
  // Tile t (blocks begin + B t ..) into slot t % ring: every wave copies a quarter of a block, also of tiles behind the
  // last, whose bytes are the pool's first, so that the copies on their way are always as many.
  uint32_t there = 0;  // bit b of pair t of the last tiles requested: block b has a page
  int asked = begin, slot = 0;  // the first block of the next tile, and its slot
  const auto request = [&]() {
    uint32_t lo[B], hi[B];
    there <<= 2;
#pragma unroll
    for (int i = 0; i < B; ++i) {
      lo[i] = __builtin_amdgcn_readlane((int)(uint32_t)where, (asked + i - looked) & 63);
      hi[i] = __builtin_amdgcn_readlane((int)(where >> 32), (asked + i - looked) & 63);
      there |= (hi[i] >> 31 ^ 1) << i;
    }
    const bool second = B > 1 && wave >= 4;
    uint32_t l = second ? lo[B - 1] : lo[0], u = second ? hi[B - 1] : hi[0];
    if (u >> 31) l = u = 0;
    const uint8_t* const from = a.kv.pages + ((uint64_t)u << 32 | l) + (wave & 3) * 320 * W;
    const uint32_t to = lds_addr(raw) + slot * S::raw + wave * 320 * W;
#pragma unroll
    for (int c = 0; c < S::copies; ++c)
      if (1024 * c + lane * 16 < 320 * W) copy16_to_lds_s(from, 1024 * c + lane * 16, to + 1024 * c);
    asked += B;
    slot = slot + 1 == S::ring ? 0 : slot + 1;
  };
  const auto prepare = [&]() {  // for the next request
    if (asked >= looked + 64) look_up(asked);
  };
  // The places of block u, of the tile `back` requests before the last, that are the sequence's.
  const auto places = [&](int u, int block, int back) {
    return there >> (2 * back + block) & 1 ? max(min(seq.length - u * kKvBlock, kKvBlock), 0) : 0;
  };
  const bool key_wave = wave < NW - S::value_waves;
  const int key_block = B > 1 ? wave >> 1 & 1 : 0, key_octet = (wave & 1) * 2 + g;
  Packed<W, NW> packed;
  const auto unpack = [&](int from) {  // a thread's share of the tile in slot `from`
    const unsigned char* const tile_raw = raw + from * S::raw;
    if (key_wave) {
      const unsigned char* const blk = tile_raw + key_block * 1280 * W;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        packed.key.codes[w] = *(const uint32_t*)(blk + n * 16 * W + key_octet * 4 * W + w * 4);
        packed.key.scales[w] = *(const uint32_t*)(blk + kv_key_scales(W) + (n * W + w) * 4);
      }
    } else {
#pragma unroll
      for (int j = 0; j < S::items; ++j) {
        const int item = wave - (NW - S::value_waves) + j * S::value_waves;
        if (item >= B * S::pairs) break;
        const int pair = item / B, i = lane & 15, quad = lane >> 4;
        const unsigned char* const blk = tile_raw + item % B * 1280 * W;
#pragma unroll
        for (int k = 0; k < 4; ++k) {  // (group of the pair, half)
          if (k >= 2 && 2 * pair + 1 >= W) break;
          const int group = 2 * pair + (k >> 1);
          packed.value.codes[j][k] = *(const uint32_t*)(blk + kv_value_codes(W) + kv_value_word(W, group, quad, i, k & 1));
          packed.value.scales[j][k] = *(const u32x4*)(blk + kv_value_scales(W) + (group * 8 + (k & 1) * 4 + quad) * 16);
        }
      }
    }
  };
  const auto widen = [&](int u, int back, half8* to) {  // it, of first block u, into the operands
    if (key_wave) {
#pragma unroll
      for (int w = 0; w < W; ++w)
        to[(key_block * 2 * W + 2 * w + (key_octet >> 1)) * 64 + (key_octet & 1) * 32 + n] =
            widen8(bits, packed.key.codes[w], packed.key.scales[w]);
    } else {
      half4v* const vt = (half4v*)(to + S::frags * 64);
#pragma unroll
      for (int j = 0; j < S::items; ++j) {
        const int item = wave - (NW - S::value_waves) + j * S::value_waves;
        if (item >= B * S::pairs) break;
        const int blk = item % B, pair = item / B, i = lane & 15, quad = lane >> 4;
        const int have = places(u + blk, blk, back);
        if (have < kKvBlock) {  // behind the sequence's end, or no page: whatever is there, 0
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int first = (k & 1) * 16 + quad * 4;
            const uint32_t keep02 = (first < have ? 0xFFFFu : 0u) | (first + 2 < have ? 0xFFFF0000u : 0u);
            const uint32_t keep13 = (first + 1 < have ? 0xFFFFu : 0u) | (first + 3 < have ? 0xFFFF0000u : 0u);
            u32x4& sm = packed.value.scales[j][k];
            sm[0] &= keep02, sm[1] &= keep13, sm[2] &= keep02, sm[3] &= keep13;
          }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (k >= 2 && 2 * pair + 1 >= W) break;
          half4v v0, v1;
          value4(bits, packed.value.codes[j][k], packed.value.scales[j][k], v0, v1);
          half4v* const p =
              vt + ((((blk * 2 + (k & 1)) * W + 2 * pair + (k >> 1)) * 64 + (quad & 1) * 32 + 2 * i) * 2 + (quad >> 1));
          p[0] = v0;
          p[2] = v1;
        }
      }
    }
  };

  const int tiles = begin < end ? (end - begin + B - 1) / B : 0;
  half8 p[2 * B];
#pragma unroll
  for (int i = 0; i < 2 * B; ++i) p[i] = half8{};
  const auto add_values = [&](const half8* vt) {
#pragma unroll
    for (int k = 0; k < 2 * B; ++k)
#pragma unroll
      for (int i = 0; i < W; ++i)
        o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vt[(k * W + i) * 64 + lane], p[k], o[i], 0, 0, 0);
  };
  // A tile is two steps, with a barrier behind each: the matrix instructions of the last tile's values and of this one's
  // scores, then the exponentials and the widening of the next tile. Where two waves share a SIMD, the value waves are a
  // step behind the key waves, so that one has the matrix unit while the other has the vector unit. (Values of tile t + 1
  // are written where those of t - 1 were, which both have read by then; keys of t + 1 while the value waves read those of
  // t.) A tile is requested ring - 1 tiles before it is computed, in the first step, when both have unpacked the slot's last.
  // A wave's copies of tile t + 1 have landed by the barrier before the key waves unpack it: ring - 2 later tiles are on
  // their way then, of the value waves' one less.
  const bool behind = NW == 8 && !key_wave;
  if (tiles > 0) {
    for (int i = 0; i < S::ring - 1; ++i) {
      prepare();
      request();
    }
    prepare();
    for (int i = threadIdx.x; i < S::frags * 64; i += S::threads) lds[3 * S::frags * 64 + i] = half8{};
    wait_vmcnt((S::ring - 2) * S::copies);
    lds_barrier();
    unpack(0);
    widen(begin, S::ring - 2, lds);
    if (behind) wait_vmcnt((S::ring - 3) * S::copies);
    lds_barrier();
    if (behind) lds_barrier();
    int turn = 0;  // the half of LDS that holds the present tile
    for (int t = 0; t < tiles; ++t) {
      const int u = begin + B * t;
      const half8* const kt = lds + turn * 2 * S::frags * 64;
      request();
      add_values(lds + ((turn ^ 1) * 2 + 1) * S::frags * 64);  // of the first tile: zeros
      f32x16 s[B];
#pragma unroll
      for (int i = 0; i < B; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) s[i][j] = 0.0f;
#pragma unroll
      for (int k = 0; k < 2 * W; ++k)
#pragma unroll
        for (int i = 0; i < B; ++i)
          s[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kt[(i * 2 * W + k) * 64 + lane], q[k], s[i], 0, 0, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);
#pragma unroll
      for (int i = 0; i < 4 * W * B - kAhead; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x008, kAhead, 0);
      if (!behind) wait_vmcnt((S::ring - 2) * S::copies);
      lds_barrier();
      const int next = t + 1 & S::ring - 1;
      if (t + 1 < tiles) unpack(next);

      const int first = u * kKvBlock;
      const int have0 = places(u, 0, S::ring - 1), have1 = B > 1 ? places(u + 1, 1, S::ring - 1) : 0;
      const bool inside = have0 == kKvBlock && (B == 1 || have1 == kKvBlock) && first >= inside_lo &&
                          first + B * kKvBlock <= inside_hi;
      if (!inside) {
#pragma unroll
        for (int i = 0; i < B; ++i)
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const int at = j / 4 * 8 + g * 4 + j % 4, place_ = first + i * kKvBlock + at;
            if (at >= (i ? have1 : have0) || place_ >= limit || place_ < low) s[i][j] = -INFINITY;
          }
      }
      // p against the row's reference so far: a sum within float16's range says that every p is. A row's first places,
      // whose reference is the lowest of all, sum to +inf.
      float sum = 0.0f;
      const auto probabilities = [&]() {
        const float ref = kProbShift - m;
        sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 2 * B; ++i) {
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
        for (int i = 0; i < B; ++i)
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
      if (t + 1 < tiles) {
        turn ^= 1;
        widen(u + B, S::ring - 2, lds + turn * 2 * S::frags * 64);
      }
      prepare();
      if (behind) wait_vmcnt((S::ring - 3) * S::copies);
      lds_barrier();
    }
    add_values(lds + (turn * 2 + 1) * S::frags * 64);
    if (NW == 8 && key_wave) lds_barrier();
    wait_vmcnt(0);  // no copy outlives the workgroup's LDS
  }
  l += __shfl_xor(l, 32);
  if (!live) return;
  if (a.splits == 1) {
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
    const AttendPart part = a.part_of(b, seq.first, row / 16, h, split, W);
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

template <int W, int NW>
void launch_w(const AttendArgs& a, long long tiles, hipStream_t stream) {
  using S = TileShape<W, NW>;
  allow_lds((const void*)attend_tile_kernel<W, NW>, (int)S::lds);
  hipLaunchKernelGGL((attend_tile_kernel<W, NW>), dim3((unsigned)(tiles * a.kv.heads), a.splits), dim3(S::threads), S::lds,
                     stream, a);
}

}  // namespace

void launch_attend_tile(const AttendArgs& a, int rows, long long tiles, hipStream_t stream) {
  const bool wide = rows == TileShape<1, 8>::rows;
  switch (kv_groups(a.dim)) {
#define MXA_CASE(W) \
  case W: wide ? launch_w<W, 8>(a, tiles, stream) : launch_w<W, 4>(a, tiles, stream); break;
    MXA_CASE(1) MXA_CASE(2) MXA_CASE(3) MXA_CASE(4)
#undef MXA_CASE
#define MXA_CASE(W) \
  case W: launch_w<W, 4>(a, tiles, stream); break;
    MXA_CASE(5) MXA_CASE(6) MXA_CASE(7) MXA_CASE(8)
#undef MXA_CASE
  }
}

}  // namespace mxa
