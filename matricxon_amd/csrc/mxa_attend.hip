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
// so nothing but the row's maximum crosses lanes. HBM bounds it: 64 replies at 16384 places each, 8 key heads of 128 values,
// read 1.34 GB in 257 us (5.2 TB/s), one at 131072 168 MB in 42 us with its join. Codes are widened in registers, code to
// float16 exactly (an or of its bits into a float16's, less that float16), then s * code + m rounded once; q is brought by a
// power of two into float16's range, exactly but for values below 2^-24 of its largest. Scores, maxima, sums and outputs are
// float32.
#include "mxa_attend.hpp"
#include "mxa_kernels.hpp"

#pragma clang fp contract(off)

namespace mxa {
namespace {

constexpr int kAttendThreads = 256, kAttendWaves = kAttendThreads / 64;

// The sequence, tile and key head of workgroup (y, z): y a pair of sequence z, or, `compact`, y the head and z the tile of the
// call as its parts are laid out (part_of). 64 replies as sequences of a ragged call have 80 tiles so, not 64 times as many as
// one sequence could have: 16384 places at most 247 us, and 148 so. Lanes look for the last sequence that does not
// begin behind tile z. (Starts that descend may find one that does; its tile would be before its first, and is none.)
__device__ __forceinline__ bool tile_of(const AttendArgs& a, int y, int z, int& b, int& rt, int& h) {
  if (!a.compact) {
    b = z, rt = y / a.kv.heads, h = y - rt * a.kv.heads;
    return true;
  }
  const auto begin = [&](int i) {
    int first, count;
    kv_rows_of(a.kv, i, a.n_tokens, first, count);
    return (int)((long long)first * a.group / 16) + i;
  };
  int lo = 0, hi = a.kv.n_seq;  // as many as lo are known to begin by then, no more than hi do
  while (lo < hi) {
    const int step = (hi - lo + 63) / 64, at = lo + (int)(threadIdx.x & 63) * step;
    const int some = __popcll(__ballot(at < hi && begin(at) <= z));
    if (some == 0) break;
    lo += (some - 1) * step + 1;
    hi = min(hi, lo + step - 1);
  }
  if (lo == 0) return false;
  b = lo - 1, rt = z - begin(b), h = y;
  return rt >= 0;
}

// W groups of 32 values a head. Workgroup (split, pair, sequence) takes a split's blocks of a pair, which its waves take in
// turn; their parts are joined in LDS, and the parts of a pair of several splits go to the workspace. No LDS holds the
// codes: a lane's are adjacent and go to its registers, the next blocks' while the present one is computed, as many as leave
// room for three workgroups a CU (two of heads above 128 values).
template <int W>
__global__ __launch_bounds__(kAttendThreads, W <= 4 ? 3 : 2) void attend_kernel(AttendArgs a) {
  constexpr int AHEAD = W <= 3 ? 3 : 2;  // blocks of a wave in registers, all but one of them on their way
  __shared__ __align__(16) uint32_t scales[kAttendWaves][64 * W];
  __shared__ float o_join[kAttendWaves][16][32 * W + 4];
  __shared__ float m_join[kAttendWaves][16], l_join[kAttendWaves][16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, g = lane >> 4;
  const int split = blockIdx.x;
  int b, rt, h;
  if (!tile_of(a, blockIdx.y, blockIdx.z, b, rt, h)) return;
  b = __builtin_amdgcn_readfirstlane(b), rt = __builtin_amdgcn_readfirstlane(rt);
  const Sequence seq = Sequence(a, b).uniform();
  if (rt >= seq.tiles || split >= seq.splits) return;
  const int begin = split * seq.chunk, end = min(begin + seq.chunk, seq.blocks);
  const int blocks_of_page = a.kv.page / kKvBlock;
  const CodeBits bits;
  uint32_t* const sc = scales[wave];

  const int row = rt * 16 + n;  // the lane's row
  const bool live = row < seq.rows;
  const int place = seq.place0 + (live ? row / a.group : 0);
  const int limit = live ? min(place + 1, seq.length) : 0, low = a.window > 0 ? max(place + 1, 0) - a.window : 0;

  // The wave's blocks are begin + wave, + 4, ..; lane i finds where the i-th of 64 of them lies, so that no block's
  // address waits for the page table.
  long long where = -1;
  int looked = 64;
  BlockPart<W> part[AHEAD];
  bool has[AHEAD];
  const auto request = [&](BlockPart<W>& p, bool& there, int u) {
    if (looked == 64) {
      looked = 0;
      const int mine = u + lane * kAttendWaves;
      const long long block = mine < end ? kv_block(a.kv, b, (seq.first_block + mine) * kKvBlock) : -1;
      where = block < 0 ? -1 : (block + (long long)h * blocks_of_page) * kv_block_bytes(W);
    }
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)where, looked);
    const uint32_t hi = __builtin_amdgcn_readlane((int)(where >> 32), looked);
    ++looked;
    there = (int)hi >= 0;
    if (there) p.load(a.kv.pages + ((uint64_t)hi << 32 | lo), lane);
  };
  int u = begin + wave;
#pragma unroll
  for (int i = 0; i < AHEAD; ++i)
    if (u + i * kAttendWaves < end) request(part[i], has[i], u + i * kAttendWaves);

  // q, by a power of two
  half8 q[W];
  float back = 0.0f;  // scale * log2(e) and what q was divided by
  {
    float qf[W][8];
    float top = 0.0f;
    const uint16_t* const src = a.q_row(seq.first + (live ? row / a.group : 0), h * a.group + (live ? row % a.group : 0));
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
  float m = -INFINITY, l = 0.0f;  // the row's reference (its maximum, or up to kSlack below) and the lane's sum
  // places that every row of the tile attends to, but for rows that there are not
  const int last_row = min(rt * 16 + 15, seq.rows - 1);
  const int inside_lo = a.window > 0 ? max(seq.place0 + last_row / a.group + 1, 0) - a.window : 0;
  const int inside_hi = min(seq.place0 + rt * 16 / a.group + 1, seq.length);

  const auto compute = [&](const BlockPart<W>& p_, int u) {
    const int first = (seq.first_block + u) * kKvBlock;
    p_.share(sc, lane);
    const bool inside = first >= inside_lo && first + kKvBlock <= inside_hi;
    if (first + kKvBlock > seq.length) clear_tail<W>(sc, lane, seq.length - first);
    float s[8];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      f32x4 acc = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int w = 0; w < W; ++w)
        acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(widen8(bits, p_.kc[i][w], sc[(i * 16 + n) * W + w]), q[w], acc, 0, 0, 0);
#pragma unroll
      for (int j = 0; j < 4; ++j) s[i * 4 + j] = acc[j] * back;
    }
    if (!inside) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int t = first + j / 4 * 16 + g * 4 + j % 4;
        if (t >= limit || t < low) s[j] = -INFINITY;
      }
    }
    float top = fmaxf(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])), fmaxf(fmaxf(s[4], s[5]), fmaxf(s[6], s[7])));
    if (__any(top > m + kSlack)) {  // the row's first places among them: its reference is -inf
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      const float m2 = fmaxf(m, top);
      const float alpha = m2 == -INFINITY ? 1.0f : exp2_(m - m2);
      m = m2;
      l *= alpha;
#pragma unroll
      for (int i = 0; i < 2 * W; ++i) o[i] *= alpha;
    }
    const float ref = (m == -INFINITY ? 0.0f : m) - kProbShift;
    float p[8], sum = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      p[j] = exp2_(s[j] - ref);
      sum += p[j];
    }
    l += sum;
    const half8 ph = prob_order(p);
#pragma unroll
    for (int w = 0; w < W; ++w) {
      half8 v0, v1;
      value_operands(bits, p_.vc[w], *(const u32x4*)(sc + 32 * W + (w * 8 + g) * 4),
                     *(const u32x4*)(sc + 32 * W + (w * 8 + 4 + g) * 4), v0, v1);
      o[2 * w] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, ph, o[2 * w], 0, 0, 0);
      o[2 * w + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, ph, o[2 * w + 1], 0, 0, 0);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  };
  while (u < end) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      if (u >= end) break;
      if (has[i]) compute(part[i], u);
      if (u + AHEAD * kAttendWaves < end) request(part[i], has[i], u + AHEAD * kAttendWaves);
      u += kAttendWaves;
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
  const int r = threadIdx.x >> 4, piece = threadIdx.x & 15;  // sixteen threads a row
  if (r < min(16, seq.rows - rt * 16)) {
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
    const bool whole = seq.splits == 1;
    const float norm = total > 0.0f || total != total ? 1.0f / total : 0.0f;
    const AttendPart to = a.part_of(b, seq.first, rt, h, split, W);
    uint16_t* const dst = a.out_row(seq.first + (rt * 16 + r) / a.group, h * a.group + (rt * 16 + r) % a.group);
    if (!whole && piece == 0) {
      to.ml[r] = top;
      to.ml[16 + r] = total;
    }
    for (int d = piece; d < a.dim; d += 16) {
      float v = 0.0f;
#pragma unroll
      for (int i = 0; i < kAttendWaves; ++i) v += f[i] * o_join[i][r][d];
      if (whole)
        dst[d] = bf16_rne(v * norm);
      else
        to.o[r * 32 * W + d] = v;
    }
  }
}

// The parts of each pair of several splits, joined: a workgroup takes a row of a pair, its threads parts and vectors of
// four values.
__global__ __launch_bounds__(kAttendThreads) void attend_join_kernel(AttendArgs a, int W) {
  __shared__ float f[kAttendMaxSplits];
  __shared__ f32x4 sums[kAttendThreads];
  __shared__ float wave_max[kAttendWaves], wave_sum[kAttendWaves];
  const int r = blockIdx.x, tid = threadIdx.x;
  int b, rt, h;
  if (!tile_of(a, blockIdx.y, blockIdx.z, b, rt, h)) return;
  const Sequence seq(a, b);
  const int parts = seq.splits;
  if (rt * 16 + r >= seq.rows || parts == 1) return;
  float top = -INFINITY, total = 0.0f;
  const auto part = [&](int i) { return a.part_of(b, seq.first, rt, h, i, W); };
  for (int i = tid; i < parts; i += kAttendThreads) top = fmaxf(top, part(i).ml[r]);
  for (int i = 1; i < 64; i *= 2) top = fmaxf(top, __shfl_xor(top, i));
  if ((tid & 63) == 0) wave_max[tid >> 6] = top;
  __syncthreads();
  for (int i = 0; i < kAttendWaves; ++i) top = fmaxf(top, wave_max[i]);
  const float ref = top == -INFINITY ? 0.0f : top;
  for (int i = tid; i < parts; i += kAttendThreads) {
    const AttendPart p = part(i);
    f[i] = exp2_(p.ml[r] - ref);
    total += f[i] * p.ml[16 + r];
  }
  for (int i = 1; i < 64; i *= 2) total += __shfl_xor(total, i);
  if ((tid & 63) == 0) wave_sum[tid >> 6] = total;
  __syncthreads();
  const int vectors = a.dim / 4, side = kAttendThreads / vectors, mine = tid / vectors, at = tid - mine * vectors;
  f32x4 v{0, 0, 0, 0};
  if (mine < side) {
#pragma unroll 4
    for (int i = mine; i < parts; i += side) v += f[i] * *(const f32x4*)(part(i).o + r * 32 * W + 4 * at);
  }
  sums[tid] = v;
  __syncthreads();
  if (tid >= vectors) return;
  total = 0.0f;
  for (int i = 0; i < kAttendWaves; ++i) total += wave_sum[i];
  for (int i = 1; i < side; ++i) v += sums[i * vectors + tid];
  const float norm = total > 0.0f || total != total ? 1.0f / total : 0.0f;
  uint16_t* const dst = a.out_row(seq.first + (rt * 16 + r) / a.group, h * a.group + (rt * 16 + r) % a.group);
#pragma unroll
  for (int j = 0; j < 4; ++j) dst[4 * tid + j] = bf16_rne(v[j] * norm);
}

// The same for few parts (16 and fewer): a workgroup takes the rows of a pair, its threads vectors of four values, whose
// parts are requested eight at a time. 64 replies of up to 6 parts: 5 us,
// 11 with sixteen threads a row and parts in turn, 17 with a workgroup a row; one reply of 96 parts takes 5 with that.
__global__ __launch_bounds__(kAttendThreads) void attend_join_rows_kernel(AttendArgs a, int W) {
  constexpr int U = 8;
  int b, rt, h;
  if (!tile_of(a, blockIdx.x, blockIdx.y, b, rt, h)) return;
  b = __builtin_amdgcn_readfirstlane(b), rt = __builtin_amdgcn_readfirstlane(rt);
  const Sequence seq = Sequence(a, b).uniform();
  const int parts = seq.splits, rows = min(16, seq.rows - rt * 16), vectors = a.dim / 4;
  if (parts == 1) return;
  const AttendPart first = a.part_of(b, seq.first, rt, h, 0, W);
  const size_t step = 16 * 32 * W + 32;
  for (int item = threadIdx.x; item < rows * vectors; item += kAttendThreads) {
    const int r = item / vectors, at = item - r * vectors;
    float top = -INFINITY, total = 0.0f;
    f32x4 v{0, 0, 0, 0};
    for (int base = 0; base < parts; base += U) {
      float m[U], l[U], most = top;
      f32x4 o[U];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const size_t from = step * min(base + i, parts - 1);  // behind the last, its own again, and left out
        m[i] = first.ml[from + r], l[i] = first.ml[from + 16 + r];
        o[i] = *(const f32x4*)(first.o + from + r * 32 * W + 4 * at);
        most = fmaxf(most, m[i]);
      }
      const float ref = most == -INFINITY ? 0.0f : most, alpha = exp2_(top - ref);
      total *= alpha, v *= alpha;
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const float f = base + i < parts ? exp2_(m[i] - ref) : 0.0f;
        total += f * l[i];
        v += f * o[i];
      }
      top = most;
    }
    const float norm = total > 0.0f || total != total ? 1.0f / total : 0.0f;
    uint16_t* const dst = a.out_row(seq.first + (rt * 16 + r) / a.group, h * a.group + (rt * 16 + r) % a.group) + 4 * at;
#pragma unroll
    for (int j = 0; j < 4; ++j) dst[j] = bf16_rne(v[j] * norm);
  }
}

template <int W>
void launch_few(const AttendArgs& a, int z, hipStream_t stream) {
  hipLaunchKernelGGL(attend_kernel<W>, dim3(a.splits, a.pairs, z), dim3(kAttendThreads), 0, stream, a);
}

}  // namespace

size_t attend_workspace(int n_seq, int n_tokens, bool ragged, int kv_heads, int group, int max_length, int window, int dim) {
  const Plan p = plan_of(n_seq, n_tokens, ragged, kv_heads, group, max_length, window, dim);
  return parts_bytes(p);
}

int launch_attend(AttendArgs a, int max_length, void* workspace, size_t workspace_bytes, hipStream_t stream) {
  const Plan p = plan_of(a.kv.n_seq, a.n_tokens, a.kv.starts != nullptr, a.kv.heads, a.group, max_length, a.window, a.dim);
  if (p.pairs[0] > 65535 || p.tiles * a.kv.heads >= 1 << 23) return kAttendUnsupported;  // past the limits of a grid
  const size_t need = parts_bytes(p);  // of the plan that is launched
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) return kAttendWorkspace;
  const int W = kv_groups(a.dim);
  for (int kind = 0; kind < 2; ++kind) {
    if (!(kind ? p.many : p.few)) continue;
    a.least_rows = kind ? kFewRows + 1 : 1, a.most_rows = kind ? 0x7fffffff : kFewRows;
    a.splits = p.splits[kind], a.chunk = p.chunk[kind];
    a.compact = a.kv.starts != nullptr && p.slots <= 65535 && p.slots * a.kv.heads < p.pairs[kind] * a.kv.n_seq;
    a.per = p.per[kind];
    a.pairs = a.compact ? a.kv.heads : (int)p.pairs[kind];
    const int z = a.compact ? (int)p.slots : a.kv.n_seq;
    a.part = (float*)((char*)workspace + (kind ? part_bytes(p, 0) : 0));
    if (kind == 1) {
      launch_attend_tile(a, p.rows, p.tiles, stream);
    } else {
      switch (W) {
#define MXA_CASE(W) \
  case W: launch_few<W>(a, z, stream); break;
        MXA_CASE(1) MXA_CASE(2) MXA_CASE(3) MXA_CASE(4) MXA_CASE(5) MXA_CASE(6) MXA_CASE(7) MXA_CASE(8)
#undef MXA_CASE
      }
    }
    if (a.splits > 1 && a.splits <= kFewParts)
      hipLaunchKernelGGL(attend_join_rows_kernel, dim3(a.pairs, z), dim3(kAttendThreads), 0, stream, a, W);
    else if (a.splits > 1)
      hipLaunchKernelGGL(attend_join_kernel, dim3(16, a.pairs, z), dim3(kAttendThreads), 0, stream, a, W);
  }
  return 0;
}

}  // namespace mxa
