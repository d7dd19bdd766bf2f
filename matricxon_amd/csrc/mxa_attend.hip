// Causal attention of the last tokens of each sequence over its cached keys and values (mxa_kv4.hpp has their layout):
//
//   o = sum_t p_t v_t / sum_t p_t,   p_t = exp(scale q . k_t),   over the places t up to the query's, or the last `window`
//
// in one pass with the running maximum and sum of each row. A row is one query head of one token; the rows of the query
// heads that share a key head, and of neighbouring tokens, go through the matrix instructions together, 16 at a time:
//
//   scores^T = K q^T     32 keys by 16 rows, a lane's scores all of one row
//   o^T     += V^T p^T   the lane's own p, rounded to float16, is the second operand as it stands: the layout of the value
//                        codes has the tokens in the order in which the scores come out
//
// so nothing but the row's maximum crosses lanes. Codes are widened in registers, code to float16 exactly (an or of its
// bits into a float16's, less that float16), then s * code + m rounded once; q is brought by a power of two into float16's
// range, exactly but for values below 2^-24 of its largest. Scores, maxima, sums and outputs are float32.
#include "mxa_attend.hpp"
#include "mxa_kernels.hpp"

#pragma clang fp contract(off)

namespace mxa {
namespace {

constexpr int kAttendThreads = 256, kAttendWaves = kAttendThreads / 64;

// W groups of 32 values a head. Workgroup (split, key head and row tile, sequence): `chunk` blocks of 32 tokens, which its
// waves take in turn and join in LDS; more than one split: unnormalised outputs, maxima and sums into `part`.
template <int W>
__global__ __launch_bounds__(kAttendThreads) void attend_kernel(AttendArgs a) {
  __shared__ __align__(16) uint32_t scales[kAttendWaves][64 * W];
  __shared__ float o_join[kAttendWaves][16][32 * W + 4];
  __shared__ float m_join[kAttendWaves][16], l_join[kAttendWaves][16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, g = lane >> 4;
  const int split = blockIdx.x, h = blockIdx.y % a.kv.heads, rt = blockIdx.y / a.kv.heads, b = blockIdx.z;
  RowTile tile;
  if (!tile.find(a, b, rt)) return;
  if (split > 0 && split >= tile.used) return;
  const int begin = tile.first_block + split * tile.chunk, end = min(begin + tile.chunk, tile.end_block);

  const int row = rt * 16 + n;  // the lane's row
  const bool live = row < tile.rows;
  const int place = tile.place0 + (live ? row / a.group : 0);
  const int limit = live ? min(place + 1, tile.length) : 0, low = a.window > 0 ? max(place + 1, 0) - a.window : 0;

  // q, by a power of two
  half8 q[W];
  float back = 0.0f;  // scale * log2(e) and what q was divided by
  {
    float qf[W][8];
    float top = 0.0f;
    const uint16_t* const src = a.q_row(tile.first + (live ? row / a.group : 0), h * a.group + (live ? row % a.group : 0));
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const bool here = live && 32 * w + 8 * g < a.dim;
      u16x8 v{};
      if (here) v = *(const u16x8*)(src + 32 * w + 8 * g);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        qf[w][j] = here ? bf16_to_float(v[j]) : 0.0f;
        top = fmaxf(top, fabsf(qf[w][j]));
      }
    }
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(top, __shfl_xor(top, 32));
    const int e = row_exponent(top);
#pragma unroll
    for (int w = 0; w < W; ++w) q[w] = key_order(qf[w], -e);
    back = ldexpf(a.scale * kLog2e, e);
  }

  f32x4 o[2 * W];
#pragma unroll
  for (int i = 0; i < 2 * W; ++i) o[i] = f32x4{0, 0, 0, 0};
  float m = -INFINITY, l = 0.0f;
  uint32_t* const sc = scales[wave];
  const int blocks = a.kv.page / kKvBlock;

  for (int u = begin + wave; u < end; u += kAttendWaves) {
    const long long block = kv_block(a.kv, b, u * kKvBlock);
    if (block < 0) continue;
    const uint8_t* const blk = a.kv.pages + (block + (long long)h * blocks) * kv_block_bytes(W);
    uint32_t kc[2][W], vc[W][2];
    load_block<W>(blk, lane, kc, vc, sc);
    if ((u + 1) * kKvBlock > tile.length) clear_tail<W>(sc, lane, tile.length - u * kKvBlock);
    float s[8];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      f32x4 acc = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int w = 0; w < W; ++w)
        acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(widen8(kc[i][w], sc[(i * 16 + n) * W + w]), q[w], acc, 0, 0, 0);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int t = u * kKvBlock + i * 16 + g * 4 + j;
        s[i * 4 + j] = t < limit && t >= low ? acc[j] * back : -INFINITY;
      }
    }
    float top = s[0];
#pragma unroll
    for (int j = 1; j < 8; ++j) top = fmaxf(top, s[j]);
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(top, __shfl_xor(top, 32));
    const float m2 = fmaxf(m, top), ref = m2 == -INFINITY ? 0.0f : m2;
    const float alpha = exp2_(m - ref);
    m = m2;
    float p[8], sum = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      p[j] = exp2_(s[j] - ref + kProbShift);
      sum += p[j];
    }
    l = l * alpha + sum;
    const half8 ph = prob_order(p);
#pragma unroll
    for (int w = 0; w < W; ++w) {
      half8 v0, v1;
      value_operands(vc[w], *(const u32x4*)(sc + 32 * W + (w * 8 + g) * 4), *(const u32x4*)(sc + 32 * W + (w * 8 + 4 + g) * 4),
                     v0, v1);
      o[2 * w] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, ph, o[2 * w] * alpha, 0, 0, 0);
      o[2 * w + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, ph, o[2 * w + 1] * alpha, 0, 0, 0);
    }
  }
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);

  // the waves' parts
#pragma unroll
  for (int w = 0; w < W; ++w)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      o_join[wave][n][32 * w + 8 * g + 2 * j] = o[2 * w][j];
      o_join[wave][n][32 * w + 8 * g + 2 * j + 1] = o[2 * w + 1][j];
    }
  if (g == 0) {
    m_join[wave][n] = m;
    l_join[wave][n] = l;
  }
  __syncthreads();
  const int rows = min(16, tile.rows - rt * 16);
  const int r = threadIdx.x >> 4, piece = threadIdx.x & 15;  // sixteen threads a row
  if (r >= rows) return;
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < kAttendWaves; ++i) top = fmaxf(top, m_join[i][r]);
  const float ref = top == -INFINITY ? 0.0f : top;
  float f[kAttendWaves], total = 0.0f;
#pragma unroll
  for (int i = 0; i < kAttendWaves; ++i) {
    f[i] = exp2_(m_join[i][r] - ref);
    total += f[i] * l_join[i][r];
  }
  const bool alone = tile.used <= 1;
  const float norm = alone ? (total > 0.0f || total != total ? 1.0f / total : 0.0f) : 1.0f;
  const AttendPart part = a.part_of(b, h, rt, split, W);
  uint16_t* const dst = a.out_row(tile.first + (rt * 16 + r) / a.group, h * a.group + (rt * 16 + r) % a.group);
  if (!alone && piece == 0) {
    part.ml[r] = top;
    part.ml[16 + r] = total;
  }
  for (int d = piece; d < a.dim; d += 16) {
    float v = 0.0f;
#pragma unroll
    for (int i = 0; i < kAttendWaves; ++i) v += f[i] * o_join[i][r][d];
    if (alone)
      dst[d] = bf16_rne(v * norm);
    else
      part.o[r * 32 * W + d] = v;
  }
}

// The splits' parts joined; rows of one split are written already.
__global__ __launch_bounds__(kAttendThreads) void attend_join_kernel(AttendArgs a, int W) {
  __shared__ float f[16][kAttendMaxSplits];
  __shared__ float norm[16];
  const int h = blockIdx.y % a.kv.heads, rt = blockIdx.y / a.kv.heads, b = blockIdx.z;
  RowTile tile;
  if (!tile.find(a, b, rt)) return;
  const int used = tile.used;
  if (used <= 1) return;
  const int rows = min(16, tile.rows - rt * 16);
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  for (int r = wave; r < rows; r += kAttendWaves) {
    float top = -INFINITY;
    for (int s = lane; s < used; s += 64) top = fmaxf(top, a.part_of(b, h, rt, s, W).ml[r]);
    for (int i = 1; i < 64; i *= 2) top = fmaxf(top, __shfl_xor(top, i));
    const float ref = top == -INFINITY ? 0.0f : top;
    float total = 0.0f;
    for (int s = lane; s < used; s += 64) {
      const AttendPart p = a.part_of(b, h, rt, s, W);
      const float e = exp2_(p.ml[r] - ref);
      f[r][s] = e;
      total += e * p.ml[16 + r];
    }
    for (int i = 1; i < 64; i *= 2) total += __shfl_xor(total, i);
    if (lane == 0) norm[r] = total > 0.0f || total != total ? 1.0f / total : 0.0f;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < rows * a.dim; i += kAttendThreads) {
    const int r = i / a.dim, d = i - r * a.dim;
    float v = 0.0f;
    for (int s = 0; s < used; ++s) v += f[r][s] * a.part_of(b, h, rt, s, W).o[r * 32 * W + d];
    a.out_row(tile.first + (rt * 16 + r) / a.group, h * a.group + (rt * 16 + r) % a.group)[d] = bf16_rne(v * norm[r]);
  }
}

// Row tiles, splits and blocks a split for up to `most` rows a key head and max_length tokens.
struct Plan {
  int tiles, splits, chunk;
};
Plan plan_of(int n_seq, int kv_heads, int group, int most, int max_length, int window) {
  Plan p;
  p.tiles = (int)(((long long)most * group + 15) / 16);
  const int reach = window > 0 ? (int)min((long long)max_length, (long long)window + most) : max_length;
  const int blocks = reach / kKvBlock + 2;
  const long long groups = (long long)n_seq * kv_heads * p.tiles;
  const long long want = max(1LL, min((long long)kAttendMaxSplits, 1024 / groups));
  p.chunk = max(kAttendWaves, (int)((blocks + want - 1) / want));
  p.splits = min(kAttendMaxSplits, (blocks + p.chunk - 1) / p.chunk);
  return p;
}

}  // namespace

size_t attend_workspace(int n_seq, int kv_heads, int group, int most, int max_length, int window, int dim) {
  const Plan p = plan_of(n_seq, kv_heads, group, most, max_length, window);
  if (p.splits <= 1) return 0;
  return (size_t)n_seq * kv_heads * p.tiles * p.splits * part_floats(kv_groups(dim)) * sizeof(float);
}

int launch_attend(AttendArgs a, int most, int max_length, void* workspace, hipStream_t stream) {
  const Plan p = plan_of(a.kv.n_seq, a.kv.heads, a.group, most, max_length, a.window);
  if ((long long)a.kv.heads * p.tiles > 65535 || a.kv.n_seq > 65535) return -1;
  a.tiles = p.tiles, a.splits = p.splits, a.chunk = p.chunk, a.part = (float*)workspace;
  const dim3 grid(p.splits, a.kv.heads * p.tiles, a.kv.n_seq);
  switch (kv_groups(a.dim)) {
#define MXA_CASE(W) \
  case W: hipLaunchKernelGGL(attend_kernel<W>, grid, dim3(kAttendThreads), 0, stream, a); break;
    MXA_CASE(1) MXA_CASE(2) MXA_CASE(3) MXA_CASE(4) MXA_CASE(5) MXA_CASE(6) MXA_CASE(7) MXA_CASE(8)
#undef MXA_CASE
    default: return -1;
  }
  if (p.splits > 1)
    hipLaunchKernelGGL(attend_join_kernel, dim3(1, a.kv.heads * p.tiles, a.kv.n_seq), dim3(kAttendThreads), 0, stream, a,
                       kv_groups(a.dim));
  return 0;
}

}  // namespace mxa
