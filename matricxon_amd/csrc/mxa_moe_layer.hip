// A mixture-of-experts layer of packed experts for a few tokens, from the router's logits, in two launches:
//
//   ids, w  = the top_k largest logits of a token and their softmax weights         (both launches need them)
//   act_p   = silu(gate_e x_t) * (up_e x_t)        for each pair p = (token t, expert e = ids[p])   first launch
//   y_t     = sum over the token's pairs, experts ascending, of w_p * (down_e act_p)                second launch
//
// with the steps of the grouped path (mxa_gemm_moe, mxa_silu_mul_q8_k, mxa_moe_combine): x and act as Q8_K blocks,
// gate, up, silu, their product and each down row rounded to bfloat16 in a bfloat16 layer, the sum in float32. The
// block arithmetic (mxa_lpb.hpp), the folds and the order of the sum are the same, so the bits are.
//
// Bound: the routed experts' packed bytes, read once each. A work item is one expert with up to MAXM of its pairs
// (experts of more are read again), and the workgroups (one a CU) are shared out evenly over the items, each taking
// a contiguous range of the expert's rows. Every workgroup routes for itself: a wave per token finds the top_k of up
// to 256 logits with one wave-wide maximum a slot, which costs less than a launch that does it once. No host sync,
// no sort, no gather.
//
// A workgroup's first W waves own rows: a wave copies the packed bytes of R = 64 / nb rows (gate's and up's) into
// its LDS stage (global_load_lds_dwordx4, coalesced, no registers), waits for its own copies only, computes a block
// per lane and folds a row per lane. The other waves turn the item's activations into Q8_K in LDS meanwhile; their
// loads are issued before the copies, behind which they would otherwise queue.
//
// The second launch's items share output rows: each writes its down rows, and the last workgroup to finish a range
// of rows (a counter per range, cleared by the first launch) adds them up.
#include "mxa_kernels.hpp"
#include "mxa_lpb.hpp"

#pragma clang fp contract(off)

namespace mxa {
namespace {

constexpr int kLayerLds = 160 * 1024;
constexpr int kLayerMaxPairs = 64;  // a lane per pair
constexpr int kActStride = QK + kActPad;

struct LayerArgs {
  const uint8_t* w0;  // gate, or down
  const uint8_t* w1;  // up
  long long stride;   // bytes of an expert's matrix
  long long row_bytes;
  const void* x;       // x (tokens, k), or act (pairs, k)
  int32_t* ids;
  float* wts;
  void* act;         // first launch: act (pairs, n); second: down rows (pairs, n) float32
  int32_t* counters;   // a finished-items count per range of rows
  const void* logits;
  uintptr_t out;       // second launch: YOut of (tokens, n)
  int n, k, nb, R, W;
  int n_experts, top_k, n_tokens;
  int logits_bf16, norm_topk, xbf16;
  int reciprocal;  // the activations' code scale: q8k_part16
  float scale;
};

// Maximum over the wave, in every lane.
__device__ __forceinline__ uint32_t wave_umax(uint32_t v) {
#define MXA_DPP_UMAX(ctrl) v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, ctrl, 0xF, 0xF, false))
  MXA_DPP_UMAX(0xB1);
  MXA_DPP_UMAX(0x4E);
  MXA_DPP_UMAX(0x141);
  MXA_DPP_UMAX(0x140);
#undef MXA_DPP_UMAX
  const auto at = [&](int l) { return (uint32_t)__builtin_amdgcn_readlane((int)v, l); };
  return max(max(at(0), at(16)), max(at(32), at(48)));
}

// The top_k experts of one token by a wave: lane i < top_k gets slot i's id and weight (id -1, weight 0 where no
// expert is left: a logit of -inf is no expert). Larger logits first, ties to the lowest id, NaN above all (its
// token's weights are NaN).
__device__ __forceinline__ void route_token(const void* logits, bool bf16, long long first, int n_experts, int top_k,
                                            bool norm_topk, float scale, int& id, float& wt) {
  const int lane = threadIdx.x & 63;
  float v[4];
  uint32_t key[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int e = 4 * lane + j;
    v[j] = -__builtin_inff();
    if (e < n_experts)
      v[j] = bf16 ? bf16_to_float(((const uint16_t*)logits)[first + e]) : ((const float*)logits)[first + e];
    const uint32_t u = __builtin_bit_cast(uint32_t, v[j] + 0.0f);  // -0 as +0
    key[j] = (u & 0x7FFFFFFFu) > 0x7F800000u ? 0xFFFFFFFFu : u == 0xFF800000u ? 0u : (u >> 31) ? ~u : u | 0x80000000u;
  }
  id = -1;
  float mine = -__builtin_inff(), top = 0.0f;
  for (int i = 0; i < top_k; ++i) {
    uint32_t best = key[0];
    int at = 0;
    float val = v[0];
#pragma unroll
    for (int j = 1; j < 4; ++j)
      if (key[j] > best) best = key[j], at = j, val = v[j];
    const uint32_t most = wave_umax(best);
    if (most == 0) break;  // uniform
    const int owner = __builtin_ctzll(__ballot(best == most));
    const int e = 4 * owner + __builtin_amdgcn_readlane(at, owner);
    const float l = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, val), owner));
    if (i == 0) top = l;
    if (lane == i) id = e, mine = l;
    if (lane == owner) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j == at) key[j] = 0;
    }
  }
  const float p = id >= 0 ? expf(mine - top) : 0.0f;
  float s = p;
  if (!norm_topk) {
    s = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (v[j] != -__builtin_inff()) s += expf(v[j] - top);
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o);
  wt = id >= 0 ? p / s * scale : 0.0f;
}

// The number of work items of the pairs whose experts the lanes hold (e < 0: none): MAXM pairs of one expert each, in
// lane order. `same`: the lanes of this lane's expert; `leaders`: the first lane of each item. Every lane calls it.
template <int MAXM>
__device__ __forceinline__ int count_items(int e, int bits, uint64_t& same, uint64_t& leaders) {
  const int lane = threadIdx.x & 63;
  uint64_t m = __ballot(e >= 0);
  for (int b = 0; b < bits; ++b) {
    const bool one = (e >> b) & 1;
    const uint64_t ones = __ballot(one);
    m &= one ? ones : ~ones;
  }
  same = m;
  const int rank = __popcll(m & ((1ull << lane) - 1ull));
  leaders = __ballot(e >= 0 && rank % MAXM == 0);
  return __popcll(leaders);
}

template <int TYPE>
constexpr int layer_stage_bytes(int blocks) {  // Q6_K rows start on any even byte
  return (blocks * Lpb<TYPE>::kBytes + (TYPE == T_Q6_K ? 15 : 0) + 1023) / 1024 * 1024;
}
template <int TYPE, int MAXM, bool GATEUP>
constexpr int layer_region_bytes(int blocks) {
  constexpr int kMats = GATEUP ? 2 : 1;
  return kMats * (layer_stage_bytes<TYPE>(blocks) + 64 * 4 * (MAXM + (Lpb<TYPE>::kHasD ? 1 : 0)));
}
// Activations of `rows` rows in LDS: q (272 bytes a block), bsums, d; and the routing.
constexpr int layer_row_act(int nb) { return nb * (kActStride + 32 + 4); }
constexpr int layer_act_bytes(int rows, int nb) { return (rows * layer_row_act(nb) + 15) / 16 * 16; }
constexpr int kLayerFixed = 2 * 4 * kLayerMaxPairs + 16;

template <int TYPE, int MAXM, bool GATEUP>
__global__ __launch_bounds__(MAXM == 1 ? 1024 : 512) void moe_layer_kernel(LayerArgs a) {
  using L = Lpb<TYPE>;
  constexpr int kMats = GATEUP ? 2 : 1;
  extern __shared__ __align__(16) uint8_t smem[];
  const int tid = threadIdx.x, lane = tid & 63, wg = blockIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), waves = blockDim.x >> 6;
  const int pairs = a.n_tokens * a.top_k, W = a.W, nb = a.nb;
  int* const sid = (int*)smem;  // the pairs' experts, then their weights or places
  float* const swt = (float*)(smem + 4 * kLayerMaxPairs);
  int* const flag = (int*)(smem + 8 * kLayerMaxPairs);
  uint8_t* const acts = smem + kLayerFixed;
  int8_t* const aq = (int8_t*)acts;  // row m, block b at (m nb + b) 272
  int16_t* const abs_ = (int16_t*)(acts + MAXM * nb * kActStride);
  float* const ad = (float*)(acts + MAXM * nb * (kActStride + 32));

  // the pairs' experts
  if constexpr (GATEUP) {
    for (int t = wave; t < a.n_tokens; t += waves) {
      int id;
      float wt;
      route_token(a.logits, a.logits_bf16 != 0, (long long)t * a.n_experts, a.n_experts, a.top_k, a.norm_topk != 0,
                  a.scale, id, wt);
      if (lane < a.top_k) {
        sid[t * a.top_k + lane] = id;
        if (wg == 0) a.ids[t * a.top_k + lane] = id, a.wts[t * a.top_k + lane] = wt;
      }
    }
    if (wg == 0)
      for (int i = tid; i < (int)gridDim.x; i += blockDim.x) a.counters[i] = 0;
    __syncthreads();
  } else {
    if (wave == 0 && lane < pairs) {
      sid[lane] = a.ids[lane];
      swt[lane] = a.wts[lane];
    }
    __syncthreads();
  }
  const int e_lane = lane < pairs ? sid[lane] : -1;
  uint64_t same, leaders;
  const int bits = a.n_experts > 1 ? 32 - __builtin_clz(a.n_experts - 1) : 0;
  const int items = count_items<MAXM>(e_lane, bits, same, leaders);
  const YOut out{a.out};
  if (items == 0) {  // no token has an expert
    if constexpr (!GATEUP)
      for (long long i = (long long)wg * blockDim.x + tid; i < (long long)a.n_tokens * a.n;
           i += (long long)gridDim.x * blockDim.x)
        out.put(i, 0.0f);
    return;
  }
  const int wpi = (int)gridDim.x / items, item = wg / wpi, part = wg - item * wpi;
  if (item >= items) return;
  // the item's leading pair (the item-th set bit of the leaders), its expert and pairs
  uint64_t rest = leaders;
  for (int i = 0; i < item; ++i) rest &= rest - 1;
  const int lead = __builtin_ctzll(rest);
  const int expert = __builtin_amdgcn_readlane(e_lane, lead);
  const uint64_t own = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)same, lead) |
                       (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(same >> 32), lead) << 32;
  const uint64_t mine = own & ~((1ull << lead) - 1ull);  // this item's pairs: up to MAXM from the leader on
  const int M = min(MAXM, __popcll(mine));
  const auto next = [](uint64_t& left) {  // its lowest bit's place, -1 past the last
    const int p = left != 0 ? __builtin_ctzll(left) : -1;
    left &= left - 1;
    return p;
  };
  uint64_t left = mine;
  const int p0 = next(left), p1 = next(left), p2 = next(left), p3 = next(left);
  static_assert(MAXM <= 4, "an item's pairs");
  const auto pair = [=](int m) __attribute__((always_inline)) { return m == 0 ? p0 : m == 1 ? p1 : m == 2 ? p2 : p3; };  // pair m < M

  const int R = a.R, sets = (a.n + R - 1) / R;
  const int lo = (int)((long long)part * sets / wpi), hi = (int)((long long)(part + 1) * sets / wpi);
  const int blocks = R * nb, stage = layer_stage_bytes<TYPE>(blocks);
  uint8_t* const region = acts + layer_act_bytes(MAXM, nb) + (size_t)wave * layer_region_bytes<TYPE, MAXM, GATEUP>(blocks);
  float* const Vbuf = (float*)(region + kMats * stage);  // [matrix][row m][64]
  float* const Dbuf = Vbuf + kMats * MAXM * 64;          // [matrix][64]
  const bool rows_wave = wave < W;
  const uintptr_t base0 = (uintptr_t)a.w0 + (uintptr_t)((long long)expert * a.stride);
  const uintptr_t base1 = (uintptr_t)a.w1 + (uintptr_t)((long long)expert * a.stride);
  const uint32_t lane16 = 16u * (uint32_t)lane;

  // the packed bytes of set s's rows into the stage, from the 16-byte word that holds the first
  const auto issue = [&](int s) {
    const int n0 = s * R, nrows = min(R, a.n - n0);
#pragma unroll
    for (int t = 0; t < kMats; ++t) {
      const uintptr_t src = (t == 0 ? base0 : base1) + (uintptr_t)n0 * (uintptr_t)a.row_bytes;
      const uint32_t bytes = (uint32_t)nrows * (uint32_t)a.row_bytes + (uint32_t)(src & 15);
      const void* from = (const void*)(src & ~(uintptr_t)15);
      const uint32_t to = lds_addr(region) + (uint32_t)(t * stage);
      for (uint32_t c = 0; c < bytes; c += 1024)
        if (c + lane16 < bytes) copy16_to_lds_s_nt(from, c + lane16, to + c);
    }
  };

  // the item's activation rows to Q8_K, by the waves that own no rows: 16 lanes a block, four blocks a wave at a
  // time, the first eight a wave requested before the weights
  const int stagers = waves - W, total = M * nb, p16 = lane & 15;
  const auto source = [&](int g) __attribute__((always_inline)) {  // block g's 16 values of this lane
    const int m = g / nb, b = g - m * nb;
    int row = MAXM == 1 ? lead : pair(m);
    if constexpr (GATEUP) row /= a.top_k;
    return (long long)row * a.k + b * QK + 16 * p16;
  };
  const auto fetch = [&](int g, uint4 (&raw)[4]) __attribute__((always_inline)) {
    if (g >= total) return;
    const uint4* src = (const uint4*)((const uint8_t*)a.x + source(g) * (a.xbf16 ? 2 : 4));
    raw[0] = src[0], raw[1] = src[1];
    if (!a.xbf16) raw[2] = src[2], raw[3] = src[3];
  };
  const auto quantize = [&](int g, const uint4 (&raw)[4]) __attribute__((always_inline)) {
    if (g >= total) return;  // uniform over the block's 16 lanes
    float v[16];
    const uint32_t r[16] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w, raw[1].x, raw[1].y, raw[1].z, raw[1].w,
                            raw[2].x, raw[2].y, raw[2].z, raw[2].w, raw[3].x, raw[3].y, raw[3].z, raw[3].w};
    if (a.xbf16) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[2 * i] = bf16_to_float(r[i]), v[2 * i + 1] = bf16_to_float(r[i] >> 16);
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = __builtin_bit_cast(float, r[i]);
    }
    q8k_part16(v, p16, aq + (size_t)g * kActStride, abs_ + 16 * g, ad + g, a.reciprocal != 0);
  };
  int s = lo + wave;
  if (rows_wave) {
    __syncthreads();  // the activations are requested
    if (s < hi) issue(s);
  } else {
    const int step = 4 * stagers;
    int g = 4 * (wave - W) + (lane >> 4);
    uint4 first[4] = {}, second[4] = {};
    fetch(g, first);
    fetch(g + step, second);
    __syncthreads();
    for (;;) {
      quantize(g, first);
      quantize(g + step, second);
      g += 2 * step;
      if (__ballot(g < total) == 0) break;
      fetch(g, first);
      fetch(g + step, second);
    }
  }
  __syncthreads();  // the activations are in LDS

  if (rows_wave) {
    const int b = lane % nb;
    ActBlock ab[MAXM];
#pragma unroll
    for (int m = 0; m < MAXM; ++m) {
      const int g = m * nb + b;
      ab[m] = ActBlock{aq + (size_t)g * kActStride, abs_ + 16 * g, 0.0f, nullptr};
    }
    for (; s < hi; s += W) {
      const int n0 = s * R, nrows = min(R, a.n - n0);
      const int jl = min(lane, nrows * nb - 1);  // lanes past the rows redo the last block
      wait_vmcnt(0);
#pragma unroll 1  // one copy of the block arithmetic
      for (int t = 0; t < kMats; ++t) {
        // bases are 16-byte aligned; only Q6_K rows can start between 16-byte words
        const int delta = TYPE == T_Q6_K ? (int)(((uintptr_t)n0 * (uintptr_t)a.row_bytes) & 15) : 0;
        float V[MAXM], D;
        L::template compute<MAXM, ActBlock>(region + t * stage, delta + jl * L::kBytes, ab, M, V, D);
#pragma unroll
        for (int m = 0; m < MAXM; ++m)
          if (m < M) Vbuf[(t * MAXM + m) * 64 + lane] = V[m];
        if (L::kHasD) Dbuf[t * 64 + lane] = D;
      }
      __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): the stage has been read
      wave_sync();
      if (s + W < hi) issue(s + W);
      for (int f = lane; f < R * M; f += 64) {  // row f % R of activation row f / R
        const int fr = f % R, fm = f / R;
        if (fr >= nrows) continue;
        const float* xd = ad + fm * nb;
        float acc[2] = {0.0f, 0.0f};
        for (int i = 0; i < nb; ++i)
#pragma unroll
          for (int t = 0; t < kMats; ++t)
            acc[t] = L::fold(acc[t], xd[i], Vbuf[(t * MAXM + fm) * 64 + fr * nb + i],
                             L::kHasD ? Dbuf[t * 64 + fr * nb + i] : 0.0f);
        const int p = MAXM == 1 ? lead : pair(fm);
        const long long at = (long long)p * a.n + n0 + fr;
        if constexpr (GATEUP) {
          if (a.xbf16) {
            const float g = bf16_to_float(bf16_rne(acc[0])), u = bf16_to_float(bf16_rne(acc[1]));
            const float si = bf16_to_float(bf16_rne(g / (1.0f + expf(-g))));
            ((uint16_t*)a.act)[at] = bf16_rne(si * u);
          } else {
            ((float*)a.act)[at] = acc[0] / (1.0f + expf(-acc[0])) * acc[1];
          }
        } else {
          ((float*)a.act)[at] = acc[0];
        }
      }
      wave_sync();  // the block values are read before the next set's are written
    }
  }
  if constexpr (!GATEUP) {
    // the range's last item adds the items' rows up
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this wave's rows are written
    __syncthreads();
    if (tid == 0) {
      __threadfence();
      *flag = atomicAdd(a.counters + part, 1);
    }
    __syncthreads();
    if (*flag != items - 1) return;
    __threadfence();
    // a token's slots in ascending expert, those without one last (and not read)
    int* const place = (int*)acts;
    __syncthreads();
    if (wave == 0 && lane < pairs) {
      const int t = lane / a.top_k, e = sid[lane];
      int rank = 0, live = 0;
      for (int i = t * a.top_k; i < (t + 1) * a.top_k; ++i) {
        const int o = sid[i];
        rank += o >= 0 && (e < 0 || o < e || (o == e && i < lane));
        live += o >= 0;
      }
      if (e >= 0) place[t * a.top_k + rank] = lane;
      if (lane == t * a.top_k) place[kLayerMaxPairs + t] = live;
    }
    __syncthreads();
    const int r0 = lo * R, nr = min(a.n, hi * R) - r0;
    const float* down = (const float*)a.act;
    for (int i = tid; i < nr * a.n_tokens; i += blockDim.x) {
      const int t = i / nr, r = r0 + i - t * nr, live = place[kLayerMaxPairs + t];
      float acc = 0.0f;
      for (int j = 0; j < live; ++j) {
        const int p = place[t * a.top_k + j];
        float v = down[(long long)p * a.n + r];
        if (a.xbf16) v = bf16_to_float(bf16_rne(v));
        acc = acc + v * swt[p];
      }
      out.put((long long)t * a.n + r, acc);
    }
  }
}

// The routing alone: a wave per token.
__global__ __launch_bounds__(256) void moe_topk_kernel(const void* __restrict__ logits, int bf16, int n_tokens,
                                                       int n_experts, int top_k, int norm_topk, float scale,
                                                       int32_t* __restrict__ ids, float* __restrict__ wts) {
  const int lane = threadIdx.x & 63, t = (int)blockIdx.x * 4 + ((int)threadIdx.x >> 6);
  if (t >= n_tokens) return;
  int id;
  float wt;
  route_token(logits, bf16 != 0, (long long)t * n_experts, n_experts, top_k, norm_topk != 0, scale, id, wt);
  if (lane < top_k) ids[(long long)t * top_k + lane] = id, wts[(long long)t * top_k + lane] = wt;
}

// Rows per wave, row waves and LDS for a matrix of rows of nb blocks; false when not one wave's rows fit.
template <int TYPE, int MAXM, bool GATEUP>
bool layer_shape(int nb, int& R, int& W, int& lds) {
  constexpr int kWaves = MAXM == 1 ? 16 : 8, kStagers = MAXM == 1 ? 4 : 2;
  R = 64 / nb;
  const int region = layer_region_bytes<TYPE, MAXM, GATEUP>(R * nb);
  const int act = kLayerFixed + layer_act_bytes(MAXM, nb);
  W = min(kWaves - kStagers, (kLayerLds - act) / region);
  lds = act + W * region;
  return W >= 1;
}

template <int TYPE, int MAXM, bool GATEUP>
int launch_layer(LayerArgs a, int grid, hipStream_t stream) {
  int lds;
  if (!layer_shape<TYPE, MAXM, GATEUP>(a.nb, a.R, a.W, lds)) return -1;
  auto kern = moe_layer_kernel<TYPE, MAXM, GATEUP>;
  allow_lds((const void*)kern, kLayerLds);
  hipLaunchKernelGGL(kern, dim3(grid), dim3(MAXM == 1 ? 1024 : 512), lds, stream, a);
  return 0;
}

template <bool GATEUP>
bool layer_fits(int type, int nb, bool one) {
  int R, W, lds;
  switch (type) {
    case T_Q4_K: return one ? layer_shape<T_Q4_K, 1, GATEUP>(nb, R, W, lds) : layer_shape<T_Q4_K, 4, GATEUP>(nb, R, W, lds);
    case T_Q6_K: return one ? layer_shape<T_Q6_K, 1, GATEUP>(nb, R, W, lds) : layer_shape<T_Q6_K, 4, GATEUP>(nb, R, W, lds);
    case T_Q8_0: return one ? layer_shape<T_Q8_0, 1, GATEUP>(nb, R, W, lds) : layer_shape<T_Q8_0, 4, GATEUP>(nb, R, W, lds);
    default: return false;
  }
}

template <bool GATEUP>
int launch_layer_type(int type, bool one, const LayerArgs& a, int grid, hipStream_t stream) {
  switch (type) {
    case T_Q4_K: return one ? launch_layer<T_Q4_K, 1, GATEUP>(a, grid, stream) : launch_layer<T_Q4_K, 4, GATEUP>(a, grid, stream);
    case T_Q6_K: return one ? launch_layer<T_Q6_K, 1, GATEUP>(a, grid, stream) : launch_layer<T_Q6_K, 4, GATEUP>(a, grid, stream);
    case T_Q8_0: return one ? launch_layer<T_Q8_0, 1, GATEUP>(a, grid, stream) : launch_layer<T_Q8_0, 4, GATEUP>(a, grid, stream);
    default: return -1;
  }
}

}  // namespace

bool moe_layer_supported(int gate_type, int down_type, int n_experts, int top_k, int n_tokens, int n_embd, int ffn) {
  if (n_tokens < 1 || n_tokens > kMoeLayerMaxTokens || top_k < 1 || top_k > min(n_experts, kMoeMaxTopK) ||
      n_experts > kMoeRouteMaxExperts || n_tokens * top_k > kLayerMaxPairs || n_embd % QK != 0 || ffn % QK != 0 ||
      n_embd < QK || ffn < QK || n_embd > 64 * QK || ffn > 64 * QK)
    return false;
  const bool one = n_tokens == 1;
  return layer_fits<true>(gate_type, n_embd / QK, one) && layer_fits<false>(down_type, ffn / QK, one);
}

size_t moe_layer_workspace(int n_tokens, int top_k, int n_embd, int ffn, bool bf16) {
  const size_t pairs = (size_t)n_tokens * top_k;
  return align256(pairs * ffn * (bf16 ? 2 : 4)) + align256(pairs * n_embd * 4) + align256((size_t)cu_count() * 4);
}

int launch_moe_layer(int gate_type, int down_type, const uint8_t* gate, const uint8_t* up, long long gate_stride,
                     long long gate_row, const uint8_t* down, long long down_stride, long long down_row, int n_experts,
                     const void* x, bool bf16, const void* logits, bool logits_bf16, int top_k, bool norm_topk,
                     float scale, int n_tokens, int n_embd, int ffn, bool reciprocal, int32_t* ids, float* wts,
                     YOut out, void* ws, hipStream_t stream) {
  const int grid = cu_count();
  if (!moe_layer_supported(gate_type, down_type, n_experts, top_k, n_tokens, n_embd, ffn) || grid < n_tokens * top_k)
    return -1;
  const size_t pairs = (size_t)n_tokens * top_k;
  uint8_t* const act = (uint8_t*)ws;
  uint8_t* const rows = act + align256(pairs * ffn * (bf16 ? 2 : 4));
  int32_t* const counters = (int32_t*)(rows + align256(pairs * n_embd * 4));
  LayerArgs a{gate, up, gate_stride, gate_row, x, ids, wts, act, counters, logits, 0, ffn, n_embd, n_embd / QK, 0, 0,
              n_experts, top_k, n_tokens, logits_bf16 ? 1 : 0, norm_topk ? 1 : 0, bf16 ? 1 : 0, reciprocal ? 1 : 0, scale};
  if (launch_layer_type<true>(gate_type, n_tokens == 1, a, grid, stream) != 0) return -1;
  a.w0 = down, a.w1 = nullptr, a.stride = down_stride, a.row_bytes = down_row, a.x = act, a.act = rows, a.out = out.v;
  a.n = n_embd, a.k = ffn, a.nb = ffn / QK;
  return launch_layer_type<false>(down_type, n_tokens == 1, a, grid, stream);
}

int launch_moe_topk(const void* logits, bool bf16, int n_tokens, int n_experts, int top_k, bool norm_topk, float scale,
                    int32_t* ids, float* wts, hipStream_t stream) {
  if (n_tokens < 1 || n_experts < 1 || n_experts > kMoeRouteMaxExperts || top_k < 1 || top_k > min(n_experts, 64)) return -1;
  hipLaunchKernelGGL(moe_topk_kernel, dim3((n_tokens + 3) / 4), dim3(256), 0, stream, logits, bf16 ? 1 : 0, n_tokens,
                     n_experts, top_k, norm_topk ? 1 : 0, scale, ids, wts);
  return 0;
}

}  // namespace mxa
