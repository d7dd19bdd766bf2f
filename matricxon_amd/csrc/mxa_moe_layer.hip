// A mixture-of-experts layer of packed experts for a few tokens, from the router's logits, in two launches:
//
//   ids, w  = the top_k largest logits of a token and their softmax weights
//   act_p   = silu(gate_e x_t) * (up_e x_t)    for each pair p = (token t, expert e = ids[p])     first launch
//   down_p  = down_e act_p                                                                       second launch
//   y_t     = sum over the token's pairs, experts ascending, of w_p * down_p   second, or for many pairs mxa_moe.hip's
//
// with the steps of the grouped path (mxa_gemm_moe, mxa_silu_mul_q8_k, mxa_moe_combine): x and act as Q8_K blocks,
// gate, up, silu, their product and each down row rounded to bfloat16 in a bfloat16 layer, the sum in float32. The
// block arithmetic (mxa_lpb.hpp), the folds and the order of the sum are the same, so the bits are.
//
// Bound: the routed experts' packed bytes, read once each. A work item is one expert with up to MAXM of its pairs
// (experts of more are read again), and the workgroups (one a CU) are shared out over the items, each taking a
// contiguous range of the expert's rows. Every workgroup routes for itself: a wave per token finds the top_k of up to
// 256 logits, which costs less than a launch that does it once. No host sync, no sort, no gather.
//
// A workgroup's first W waves own rows: a wave copies the packed bytes of R = 64 / nb rows (gate's and up's) into
// its LDS stages (global_load_lds_dwordx4, coalesced, no registers), waits for its own copies only, computes a block
// per lane and folds a row per lane; a stage is requested again as soon as its blocks are computed. The other waves
// turn the item's activations into Q8_K in LDS meanwhile; their loads are issued before the copies, behind which
// they would otherwise queue (with one token x's before the routing).
//
// What bounds it, MI355X, kernel alone with weights that no cache holds: 8 experts top 2 of 4096 x 14336 (Q4_K, Q6_K
// down), one token, gate and up 28 us for 132 MB (4.7 TB/s; a read of as many bytes 21), of which 3 us before the
// first copy and 3 after the last; down 26 us for 96 MB (3.7 TB/s): 3 us before the first copy, 9 before the two
// activation rows are blocks, then the LDS holds 10 rows of 56 blocks, which wait and compute in turn. Eight tokens: 95
// and 86 us, 5.0 and 4.0 TB/s: each further pair of an expert takes LDS from the rows and adds to the part of a wave's
// turn in which its stage is not in flight. 64 experts top 8 of 2048 x 1024, one token: 12 and 9 us for 19 and 14 MB,
// latency (logits, routing, activations, weights) and, not timed apart, the arithmetic of few waves: rows a wave are
// taken by what LDS holds (layer_rows), eight in the first launch, so that a workgroup's share is four sets for its
// eight waves with rows, each of which computes gate, then up, then folds; of the second, half the lanes hold a block.
//
// The sum needs every pair's rows in one place. Up to 16 pairs the second launch's workgroups take rows, each through
// all items, and add up in LDS. For more they take items, and the combine is a launch of its own (3 to 4 us): adding up
// by the last workgroup to finish a range of rows was slower, the fences that such a hand-over needs between XCDs cost
// the weights' stream more (down 62.8 against then 29.3 + 4.4 us, one token of 8 experts top 2, 4096 x 14336).
#include "mxa_kernels.hpp"
#include "mxa_lpb.hpp"

#pragma clang fp contract(off)

namespace mxa {
namespace {

constexpr int kLayerLds = 160 * 1024;
constexpr int kLayerWaves = 16, kLayerStagers = 4;  // waves of a workgroup; of them without rows, at least
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
  const void* logits;
  int n, k, nb, R, W;
  int n_experts, top_k, n_tokens;
  int logits_bf16, norm_topk, xbf16;
  int reciprocal;  // the activations' code scale: q8k_part16
  float scale;
};

// Reductions over the wave, in every lane: DPP within rows of 16, then the four rows.
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
__device__ __forceinline__ float lane_value(float v, int l) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), l));
}
__device__ __forceinline__ float wave_sum(float v) {
  v = quad_sum(v);
  v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x141, 0xF, 0xF, false));
  v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x140, 0xF, 0xF, false));
  return (lane_value(v, 0) + lane_value(v, 16)) + (lane_value(v, 32) + lane_value(v, 48));
}

// The top_k experts of one token by a wave: put(slot, id, weight) is called for every slot by one lane (id -1, weight
// 0 where no expert is left: a logit of -inf is no expert). Larger logits first, ties to the lowest id, NaN above all
// (its token's weights are NaN). A lane holds logits lane + 64 j.
//
// Up to 64 logits: each lane counts the logits that go before its own, broadcast one by one, which no step waits for
// (64 logits, 8 slots: 0.5 us; a maximum over the wave per slot 1.5). More: a maximum per slot.
template <class Put>
__device__ __forceinline__ void route_token(const void* logits, bool bf16, long long first, int n_experts, int top_k,
                                            bool norm_topk, float scale, bool weights, Put put) {
  const int lane = threadIdx.x & 63;
  float v[4];
  uint32_t key[4];  // ordered as the logits, 0 for no expert
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int e = lane + 64 * j;
    v[j] = -__builtin_inff();
    if (e < n_experts)
      v[j] = bf16 ? bf16_to_float(((const uint16_t*)logits)[first + e]) : ((const float*)logits)[first + e];
    const uint32_t u = __builtin_bit_cast(uint32_t, v[j] + 0.0f);  // -0 as +0
    key[j] = (u & 0x7FFFFFFFu) > 0x7F800000u ? 0xFFFFFFFFu : u == 0xFF800000u ? 0u : (u >> 31) ? ~u : u | 0x80000000u;
  }
  int slot = top_k, id = lane, live;  // this lane's slot (top_k or more: none) and its expert
  float mine = v[0], top;
  if (n_experts <= 64) {
    live = __popcll(__ballot(key[0] != 0));
    int before = 0;
#pragma unroll
    for (int l = 0; l < 64; ++l)  // lanes past the experts hold key 0
      before += (uint32_t)__builtin_amdgcn_readlane((int)key[0], l) > key[0] - (l < lane ? 1u : 0u);
    if (key[0] != 0) slot = before;  // o >= key where an equal lower id goes before, o > key else; key 0 has no slot
    top = live > 0 ? lane_value(v[0], __builtin_ctzll(__ballot(slot == 0))) : 0.0f;
  } else {
    top = 0.0f;
    for (live = 0; live < top_k; ++live) {
      uint32_t best = key[0];
      int at = 0;
      float val = v[0];
#pragma unroll
      for (int j = 1; j < 4; ++j)
        if (key[j] > best) best = key[j], at = j, val = v[j];
      const uint32_t most = wave_umax(best);
      if (most == 0) break;  // uniform
      // the lowest id of that logit: the lowest j, then the lowest lane
      int j = 0;
      uint64_t with = __ballot(key[0] == most);
#pragma unroll
      for (int i = 1; i < 4; ++i)
        if (with == 0) with = __ballot(key[i] == most), j = i;
      const int owner = __builtin_ctzll(with);
      const float l = lane_value(val, owner);  // its best: no lower j of its own has that logit
      if (live == 0) top = l;
      if (lane == live) slot = live, id = owner + 64 * j, mine = l;
      if (lane == owner) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (i == j) key[i] = 0;
      }
    }
  }
  if (lane >= live && lane < top_k) put(lane, -1, 0.0f);
  float wt = 0.0f;
  if (weights) {
    const float p = slot < top_k ? expf(mine - top) : 0.0f;
    float s = p;
    if (!norm_topk) {
      s = 0.0f;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (v[j] != -__builtin_inff()) s += expf(v[j] - top);
    }
    wt = p / wave_sum(s) * scale;
  }
  if (slot < top_k) put(slot, id, wt);
}

// A barrier for what the waves wrote to LDS: loads in flight stay in flight.
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
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

// The expert and the pairs of the item that lane `lead` leads: the lanes of `mine`, the first M of them.
struct LayerItem {
  int expert, M, p0, p1, p2, p3;
  __device__ __forceinline__ int pair(int m) const {  // m < M
    return p0 + (m > 0 ? p1 - p0 : 0) + (m > 1 ? p2 - p1 : 0) + (m > 2 ? p3 - p2 : 0);
  }
};
template <int MAXM>
__device__ __forceinline__ LayerItem layer_item(int lead, int e_lane, uint64_t same) {
  static_assert(MAXM <= 4, "an item's pairs");
  const uint64_t own = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)same, lead) |
                       (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(same >> 32), lead) << 32;
  uint64_t left = own & ~((1ull << lead) - 1ull);
  const auto next = [&]() __attribute__((always_inline)) {  // the next pair, -1 past the last
    const int p = left != 0 ? __builtin_ctzll(left) : -1;
    left &= left - 1;
    return p;
  };
  LayerItem it;
  it.expert = __builtin_amdgcn_readlane(e_lane, lead);
  it.M = min(MAXM, __popcll(left));
  it.p0 = next(), it.p1 = next(), it.p2 = next(), it.p3 = next();
  return it;
}

// Activations to Q8_K by the waves that own no rows, 16 lanes a block. A buffer holds a lane's 16 values of a float32
// block, or of two bfloat16 blocks; block(i) gives the lane's i-th block: whether there is one, the value of x that the
// lane's part starts at, and where its codes, sums and scale go.
struct ActPart {
  bool on;
  long long at;
  int8_t* q;
  int16_t* bs;
  float* d;
};
template <int BUFS, class Block>
__device__ __forceinline__ void fetch_acts(const LayerArgs& a, int i0, Block block, uint4 (&raw)[BUFS][4]) {
#pragma unroll
  for (int j = 0; j < BUFS; ++j) {
    const ActPart p = block(i0 + (a.xbf16 ? 2 * j : j));
    if (p.on) {
      const uint4* src = (const uint4*)((const uint8_t*)a.x + p.at * (a.xbf16 ? 2 : 4));
      raw[j][0] = src[0], raw[j][1] = src[1];
      if (!a.xbf16) raw[j][2] = src[2], raw[j][3] = src[3];
    }
    if (a.xbf16) {
      const ActPart p2 = block(i0 + 2 * j + 1);
      if (p2.on) {
        const uint4* src = (const uint4*)((const uint8_t*)a.x + p2.at * 2);
        raw[j][2] = src[0], raw[j][3] = src[1];
      }
    }
  }
}
__device__ __forceinline__ void widen_bf16x16(uint4 lo, uint4 hi, float (&v)[16]) {
  const uint32_t r[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) v[2 * i] = bf16_to_float(r[i]), v[2 * i + 1] = bf16_to_float(r[i] >> 16);
}
template <int BUFS, class Block>
__device__ __forceinline__ void quantize_acts(const LayerArgs& a, int i0, Block block, const uint4 (&raw)[BUFS][4]) {
  const int p16 = threadIdx.x & 15;
#pragma unroll
  for (int j = 0; j < BUFS; ++j) {
    const ActPart p = block(i0 + (a.xbf16 ? 2 * j : j));
    if (p.on) {  // uniform over the block's 16 lanes
      float v[16];
      if (a.xbf16) {
        widen_bf16x16(raw[j][0], raw[j][1], v);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v[4 * i] = __builtin_bit_cast(float, raw[j][i].x), v[4 * i + 1] = __builtin_bit_cast(float, raw[j][i].y);
          v[4 * i + 2] = __builtin_bit_cast(float, raw[j][i].z), v[4 * i + 3] = __builtin_bit_cast(float, raw[j][i].w);
        }
      }
      q8k_part16(v, p16, p.q, p.bs, p.d, a.reciprocal != 0);
    }
    if (a.xbf16) {
      const ActPart p2 = block(i0 + 2 * j + 1);
      if (p2.on) {
        float v[16];
        widen_bf16x16(raw[j][2], raw[j][3], v);
        q8k_part16(v, p16, p2.q, p2.bs, p2.d, a.reciprocal != 0);
      }
    }
  }
}
// Buffers of a wave: what it requests before the weights (what is left comes behind them).
constexpr int kLayerBufs = 2;

// `bytes` packed bytes at src, with those before them in src's 16-byte word, to LDS address `to`; the copies it took.
__device__ __forceinline__ int copy_rows(uintptr_t src, uint32_t bytes, uint32_t to) {
  const uint32_t lane16 = 16u * (threadIdx.x & 63), end = bytes + (uint32_t)(src & 15);
  const void* from = (const void*)(src & ~(uintptr_t)15);
  for (uint32_t c = 0; c < end; c += 1024)
    if (c + lane16 < end) copy16_to_lds_s_nt(from, c + lane16, to + c);
  return (int)((end + 1023) / 1024);
}

// Rows of block values and of scales in LDS start on 16 bytes: their stride in floats.
__host__ __device__ constexpr int layer_fold_row(int nb) { return (nb + 3) / 4 * 4; }

// The fold of one row's nb block values in order, of MATS matrices at once (their values v `vstep`, their scales d
// `dstep` apart); xd the activation row's scales. Four blocks a read: few lanes fold, and an instruction costs what it
// costs a whole wave (56 blocks one at a time, their places clamped to the row's end, took 3 us).
template <int TYPE, int MATS>
__device__ __forceinline__ void fold_row(int nb, const float* xd, const float* v, int vstep, const float* d, int dstep,
                                         float (&acc)[MATS]) {
  using L = Lpb<TYPE>;
  constexpr int kQuads = 2;  // read before the first is folded
#pragma unroll
  for (int t = 0; t < MATS; ++t) acc[t] = 0.0f;
  for (int i = 0; i < nb; i += 4 * kQuads) {
    float4 xx[kQuads], vv[MATS][kQuads], dd[MATS][kQuads];
#pragma unroll
    for (int q = 0; q < kQuads; ++q) {
      const int c = i + 4 * q;
      if (c >= nb) break;
      xx[q] = *(const float4*)(xd + c);
#pragma unroll
      for (int t = 0; t < MATS; ++t) {
        vv[t][q] = *(const float4*)(v + t * vstep + c);
        if (L::kHasD) dd[t][q] = *(const float4*)(d + t * dstep + c);
      }
    }
#pragma unroll
    for (int q = 0; q < kQuads; ++q) {
      const int c = i + 4 * q;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (c + j >= nb) break;
#pragma unroll
        for (int t = 0; t < MATS; ++t) {
          const auto at = [&](const float4& f) { return j == 0 ? f.x : j == 1 ? f.y : j == 2 ? f.z : f.w; };
          acc[t] = L::fold(acc[t], at(xx[q]), at(vv[t][q]), L::kHasD ? at(dd[t][q]) : 0.0f);
        }
      }
    }
  }
}

template <int TYPE>
__host__ __device__ constexpr int layer_stage_bytes(int blocks) {  // Q6_K rows start on any even byte
  return (blocks * Lpb<TYPE>::kBytes + (TYPE == T_Q6_K ? 15 : 0) + 1023) / 1024 * 1024;
}
// A wave's LDS for R rows and M activation rows: its stages and block values.
template <int TYPE, bool GATEUP>
__host__ __device__ constexpr int layer_region_bytes(int M, int R, int nb) {
  constexpr int kMats = GATEUP ? 2 : 1;
  return kMats * (layer_stage_bytes<TYPE>(R * nb) + R * layer_fold_row(nb) * 4 * (M + (Lpb<TYPE>::kHasD ? 1 : 0)));
}
// Activations of `rows` rows in LDS: q (272 bytes a block), bsums, d; and the routing.
__host__ __device__ constexpr int layer_row_act(int nb) { return nb * (kActStride + 32) + 4 * layer_fold_row(nb); }
__host__ __device__ constexpr int layer_act_bytes(int rows, int nb) {
  return (rows * layer_row_act(nb) + 15) / 16 * 16;
}
constexpr int kLayerFixed = 4 * kLayerMaxPairs;
// Waves with rows of an item of M pairs, 0 or less where not one's fit. Fewer pairs leave LDS to more of them (with
// as many waves for any item, eight tokens of 8 experts top 2, 4096 x 14336, took 99 and 100 us, not 95 and 86).
template <int TYPE, bool GATEUP>
__host__ __device__ constexpr int layer_waves(int M, int R, int nb) {
  const int w = (kLayerLds - kLayerFixed - layer_act_bytes(M, nb)) / layer_region_bytes<TYPE, GATEUP>(M, R, nb);
  return w < kLayerWaves - kLayerStagers ? w : kLayerWaves - kLayerStagers;
}

template <int TYPE, int MAXM, bool GATEUP>
__global__ __launch_bounds__(64 * kLayerWaves) void moe_layer_kernel(LayerArgs a) {
  using L = Lpb<TYPE>;
  constexpr int kMats = GATEUP ? 2 : 1;
  constexpr bool kReg = MAXM == 1 && TYPE != T_Q6_K;  // Q6_K's arithmetic leaves no registers
  extern __shared__ __align__(16) uint8_t smem[];
  const int tid = threadIdx.x, lane = tid & 63, wg = blockIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), waves = blockDim.x >> 6;
  const int pairs = a.n_tokens * a.top_k, nb = a.nb, R = a.R;
  int* const sid = (int*)smem;  // the pairs' experts
  uint8_t* const acts = smem + kLayerFixed;
  int8_t* const aq = (int8_t*)acts;  // row m, block b at (m nb + b) 272

  constexpr int kBufs = kLayerBufs;
  uint4 raw[kBufs][4] = {};
  const int p16 = lane & 15;
  constexpr bool kOneToken = GATEUP && MAXM == 1;  // its row is known before its experts are
  if constexpr (kOneToken) {
    const int W = layer_waves<TYPE, GATEUP>(1, R, nb);
    const auto token_block = [&](int i) __attribute__((always_inline)) {
      const int g = 4 * (wave - W) + (lane >> 4) + 4 * (waves - W) * i;
      return ActPart{g < nb, (long long)g * QK + 16 * p16, nullptr, nullptr, nullptr};
    };
    if (wave >= W) fetch_acts(a, 0, token_block, raw);
  }

  // the pairs' experts
  int e_lane = -1;
  if constexpr (GATEUP) {
    for (int t = wave; t < a.n_tokens; t += waves) {
      route_token(a.logits, a.logits_bf16 != 0, (long long)t * a.n_experts, a.n_experts, a.top_k, a.norm_topk != 0,
                  a.scale, wg == 0, [&](int slot, int id, float wt) {
                    sid[t * a.top_k + slot] = id;
                    if (wg == 0) a.ids[t * a.top_k + slot] = id, a.wts[t * a.top_k + slot] = wt;
                  });
    }
    lds_barrier();
    if (lane < pairs) e_lane = sid[lane];
  } else {
    if (lane < pairs) e_lane = a.ids[lane];
  }
  uint64_t same, leaders;
  const int bits = a.n_experts > 1 ? 32 - __builtin_clz(a.n_experts - 1) : 0;
  const int items = count_items<MAXM>(e_lane, bits, same, leaders);
  if (items == 0) return;  // no token has an expert
  // The item of this workgroup, its leading pair, and the workgroup's place among the item's. The workgroups are
  // shared out by the items' costs, a set of rows taking about a third longer for each further pair (with equal shares
  // of 8 tokens of 8 experts top 2, 4096 x 14336, an item of one pair was done after 58 us, one of four after 117).
  int lead, part, wpi;
  if constexpr (MAXM == 1) {
    wpi = (int)gridDim.x / items;
    const int item = wg / wpi;
    part = wg - item * wpi;
    if (item >= items) return;
    uint64_t rest = leaders;
    for (int i = 0; i < item; ++i) rest &= rest - 1;
    lead = __builtin_ctzll(rest);
  } else {
    const bool leads = (leaders >> lane) & 1;
    const int cost = leads ? 2 + min(MAXM, __popcll(same & ~((1ull << lane) - 1ull))) : 0;
    int upto = cost;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int x = __shfl_up(upto, off, 64);
      if (lane >= off) upto += x;
    }
    const int all = __builtin_amdgcn_readlane(upto, 63), grid = (int)gridDim.x;
    const int from = (upto - cost) * grid / all, to = upto * grid / all;  // at least two each: launch_moe_layer
    lead = __builtin_ctzll(__ballot(leads && wg >= from && wg < to));
    wpi = __builtin_amdgcn_readlane(to - from, lead);
    part = wg - __builtin_amdgcn_readlane(from, lead);
  }
  const LayerItem it = layer_item<MAXM>(lead, e_lane, same);
  const int M = it.M, W = layer_waves<TYPE, GATEUP>(M, R, nb);
  const bool rows_wave = wave < W;
  int16_t* const abs_ = (int16_t*)(acts + M * nb * kActStride);
  float* const ad = (float*)(acts + M * nb * (kActStride + 32));

  const int sets = (a.n + R - 1) / R;
  const int lo = part * sets / wpi, hi = (part + 1) * sets / wpi;  // below 2^8 * 2^14
  const int blocks = R * nb, stage = layer_stage_bytes<TYPE>(blocks);
  uint8_t* const region = acts + layer_act_bytes(M, nb) + (size_t)wave * layer_region_bytes<TYPE, GATEUP>(M, R, nb);
  const int fold = layer_fold_row(nb), fold_set = R * fold;
  float* const Vbuf = (float*)(region + kMats * stage);  // [matrix][activation row][row][fold]
  float* const Dbuf = Vbuf + kMats * M * fold_set;       // [matrix][row][fold]
  const uintptr_t base0 = (uintptr_t)a.w0 + (uintptr_t)((long long)it.expert * a.stride);
  const uintptr_t base1 = (uintptr_t)a.w1 + (uintptr_t)((long long)it.expert * a.stride);
  // The packed bytes of set s's rows of matrix t into its stage, and the copies that takes (none past the last set).
  const auto issue = [&](int s, int t) __attribute__((always_inline)) {
    if (s >= hi) return 0;
    const int n0 = s * R;
    return copy_rows((t == 0 ? base0 : base1) + (uintptr_t)n0 * (uintptr_t)a.row_bytes,
                     (uint32_t)min(R, a.n - n0) * (uint32_t)a.row_bytes, lds_addr(region) + (uint32_t)(t * stage));
  };

  const int total = M * nb, step = 4 * (waves - W), g0 = 4 * (wave - W) + (lane >> 4);
  const auto item_block = [&](int i) __attribute__((always_inline)) {  // of the item's rows
    const int g = g0 + step * i, m = MAXM == 1 ? 0 : g / nb, p = MAXM == 1 ? lead : it.pair(m);
    return ActPart{g < total, (long long)(GATEUP ? p / a.top_k : p) * a.k + (g - m * nb) * QK + 16 * p16,
                   aq + (size_t)g * kActStride, abs_ + 16 * g, ad + m * fold + g - m * nb};
  };
  int s = lo + wave, behind = 0;  // copies issued behind those of the stage that is waited for next
  if (rows_wave) {
    __builtin_amdgcn_s_barrier();  // the activations are requested
    // no load of this wave's is in flight: said here, or the compiler, which sees the other waves' loads into the
    // same registers, waits for every copy before it issues the next
    wait_vmcnt(0);
    issue(s, 0);
    if constexpr (GATEUP) behind = issue(s, 1);
  } else {
    if (!kOneToken) fetch_acts(a, 0, item_block, raw);
    __builtin_amdgcn_sched_barrier(0);  // not sunk below the barrier
    __builtin_amdgcn_s_barrier();
    const int per = a.xbf16 ? 2 * kBufs : kBufs;
    for (int i = 0;;) {
      quantize_acts(a, i, item_block, raw);
      i += per;
      if (__ballot(g0 + step * i < total) == 0) break;
      fetch_acts(a, i, item_block, raw);
    }
  }
  lds_barrier();  // the activations are in LDS

  if (rows_wave) {
    const int b = lane % nb, to = lane / nb * fold + b;  // the lane's block, and its place in the folds
    ActBlock ab[MAXM];
#pragma unroll
    for (int m = 0; m < MAXM; ++m) {
      const int g = m * nb + b;
      ab[m] = ActBlock{aq + (size_t)g * kActStride, abs_ + 16 * g, 0.0f, nullptr};
    }
    for (; s < hi; s += W) {
      const int n0 = s * R, nrows = min(R, a.n - n0);
      const int jl = min(lane, nrows * nb - 1);  // lanes past the rows redo the last block
      ActRegs areg;  // the lane's activation block, for both matrices (again for every set: held across them it spills)
      if constexpr (kReg) {
#pragma unroll
        for (int i = 0; i < 16; ++i) areg.q[i] = ab[0].q16(16 * i);
        areg.bs[0] = ab[0].bs8(0);
        areg.bs[1] = ab[0].bs8(1);
      }
#pragma unroll 1  // one copy of the block arithmetic
      for (int t = 0; t < kMats; ++t) {
        // Copies land in order: a stage is computed while the other one's are in flight. (A store of the last set's
        // fold behind them makes this wait for one copy more than it has to.)
        wait_vmcnt(behind);
        // bases are 16-byte aligned; only Q6_K rows can start between 16-byte words
        const int delta = TYPE == T_Q6_K ? (int)(((uintptr_t)n0 * (uintptr_t)a.row_bytes) & 15) : 0;
        float V[MAXM], D;
        if constexpr (kReg)
          L::template compute<1, ActRegs>(region + t * stage, delta + jl * L::kBytes, &areg, 1, V, D);
        else
          L::template compute<MAXM, ActBlock>(region + t * stage, delta + jl * L::kBytes, ab, M, V, D);
        uint32_t v_at = (uint32_t)(t * M * fold_set + to);
        if constexpr (MAXM > 1) asm volatile("" : "+v"(v_at));  // counted up, not MAXM kept across the sets: they spill
#pragma unroll
        for (int m = 0; m < MAXM; ++m, v_at += (uint32_t)fold_set)
          if (m < M && lane < blocks) Vbuf[v_at] = V[m];
        if (L::kHasD && lane < blocks) Dbuf[t * fold_set + to] = D;
        __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): the stage has been read
        wave_sync();
        const int n = issue(s + W, t);
        if constexpr (GATEUP) behind = n;
      }
      for (int f = lane; f < R * M; f += 64) {  // row f % R of activation row f / R
        const int fr = f % R, fm = f / R;
        if (fr >= nrows) continue;
        float acc[kMats];
        fold_row<TYPE, kMats>(nb, ad + fm * fold, Vbuf + fm * fold_set + fr * fold, M * fold_set, Dbuf + fr * fold,
                              fold_set, acc);
        const int p = MAXM == 1 ? lead : it.pair(fm);
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
}

// Bytes of the second launch's LDS besides its waves' regions when it adds the pairs up itself: the pairs' weights and
// places, each token's pairs, the activations of all pairs, and their down values of the workgroup's `rows` rows.
constexpr int kSumFixed = (2 * kLayerMaxPairs + kMoeLayerMaxTokens) * 4;
constexpr int layer_sum_bytes(int pairs, int nb, int rows) {
  return kSumFixed + layer_act_bytes(pairs, nb) + (pairs * rows * 4 + 15) / 16 * 16;
}

// The second launch where all pairs' activations fit LDS: a workgroup takes a range of `rows` output rows through every
// item (a wave an item's R rows at a time, as above), keeps the down values in LDS and adds them up.
template <int TYPE, int MAXM>
__global__ __launch_bounds__(64 * kLayerWaves) void moe_down_sum_kernel(LayerArgs a, YOut out, int rows) {
  using L = Lpb<TYPE>;
  constexpr bool kReg = MAXM == 1 && TYPE != T_Q6_K;
  extern __shared__ __align__(16) uint8_t smem[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), waves = blockDim.x >> 6;
  const int pairs = a.n_tokens * a.top_k, W = a.W, nb = a.nb, R = a.R;
  float* const swt = (float*)smem;
  int* const place = (int*)smem + kLayerMaxPairs;  // a token's pairs, experts ascending
  int* const live = place + kLayerMaxPairs;        // how many they are
  uint8_t* const acts = smem + kSumFixed;
  int8_t* const aq = (int8_t*)acts;  // pair p, block b at (p nb + b) 272
  int16_t* const abs_ = (int16_t*)(acts + pairs * nb * kActStride);
  float* const ad = (float*)(acts + pairs * nb * (kActStride + 32));
  float* const down = (float*)(acts + layer_act_bytes(pairs, nb));  // (pairs, rows)
  const int r0 = (int)blockIdx.x * rows, nr = min(rows, a.n - r0), fold = layer_fold_row(nb);
  if (nr <= 0) return;

  int e_lane = -1;
  float w_lane = 0.0f;
  if (lane < pairs) e_lane = a.ids[lane], w_lane = a.wts[lane];
  // Every pair's row is requested before the pairs' experts are known, also a row of no expert, which nothing has
  // written and nothing reads.
  constexpr int kBufs = kLayerBufs;
  const int step = 4 * (waves - W), p16 = lane & 15, g0 = 4 * (wave - W) + (lane >> 4), total = pairs * nb;
  uint4 raw[kBufs][4] = {};
  const auto block = [&](int i) __attribute__((always_inline)) {
    const int g = g0 + step * i, p = g / nb;
    return ActPart{g < total, (long long)p * a.k + (g - p * nb) * QK + 16 * p16, aq + (size_t)g * kActStride,
                   abs_ + 16 * g, ad + p * fold + g - p * nb};
  };
  if (wave >= W) fetch_acts(a, 0, block, raw);
  __builtin_amdgcn_sched_barrier(0);  // not sunk below the barrier
  __builtin_amdgcn_s_barrier();       // the activations are requested
  uint64_t same, leaders;
  const int bits = a.n_experts > 1 ? 32 - __builtin_clz(a.n_experts - 1) : 0;
  const int items = count_items<MAXM>(e_lane, bits, same, leaders);
  const int sets = (nr + R - 1) / R, tasks = items * sets;
  const int blocks = R * nb, stage = layer_stage_bytes<TYPE>(blocks);
  uint8_t* const region =
      acts + layer_sum_bytes(pairs, nb, rows) - kSumFixed + (size_t)wave * layer_region_bytes<TYPE, false>(MAXM, R, nb);
  const int fold_set = R * fold;
  float* const Vbuf = (float*)(region + stage);  // [activation row][row][fold]
  float* const Dbuf = Vbuf + MAXM * fold_set;
  const auto lead_of = [&](int task) __attribute__((always_inline)) {
    uint64_t rest = leaders;
    for (int i = task / sets; i > 0; --i) rest &= rest - 1;
    return (int)__builtin_ctzll(rest);
  };
  const auto issue = [&](int task) __attribute__((always_inline)) {
    if (task >= tasks) return;
    const int n0 = r0 + task % sets * R, expert = __builtin_amdgcn_readlane(e_lane, lead_of(task));
    copy_rows((uintptr_t)a.w0 + (uintptr_t)((long long)expert * a.stride) + (uintptr_t)n0 * (uintptr_t)a.row_bytes,
              (uint32_t)min(R, r0 + nr - n0) * (uint32_t)a.row_bytes, lds_addr(region));
  };

  int task = wave;
  if (wave < W) {
    wait_vmcnt(0);  // as in moe_layer_kernel
    issue(task);
  } else {
    if (wave == W) {  // the sum's order
      const int t = lane / a.top_k;
      int rank = 0, n = 0;
      for (int i = 0; i < pairs; ++i) {
        const int o = __builtin_amdgcn_readlane(e_lane, i);
        const bool counts = i / a.top_k == t && o >= 0;
        rank += counts && (o < e_lane || (o == e_lane && i < lane));
        n += counts;
      }
      if (lane < pairs) {
        if (e_lane >= 0) place[t * a.top_k + rank] = lane;
        live[t] = n;
        swt[lane] = w_lane;
      }
    }
    const int per = a.xbf16 ? 2 * kBufs : kBufs;
    for (int i = 0;;) {
      quantize_acts(a, i, block, raw);
      i += per;
      if (__ballot(g0 + step * i < total) == 0) break;
      fetch_acts(a, i, block, raw);
    }
  }
  lds_barrier();  // the activations are in LDS

  if (wave < W) {
    const int b = lane % nb, to = lane / nb * fold + b;
    for (; task < tasks; task += W) {
      const int n0 = task % sets * R, nrows = min(R, nr - n0);  // rows of the workgroup's
      const LayerItem it = layer_item<MAXM>(lead_of(task), e_lane, same);
      const int M = it.M, jl = min(lane, nrows * nb - 1);
      ActBlock ab[MAXM];
#pragma unroll
      for (int m = 0; m < MAXM; ++m) {
        const int g = it.pair(m < M ? m : 0) * nb + b;
        ab[m] = ActBlock{aq + (size_t)g * kActStride, abs_ + 16 * g, 0.0f, nullptr};
      }
      ActRegs areg;
      if constexpr (kReg) {
#pragma unroll
        for (int i = 0; i < 16; ++i) areg.q[i] = ab[0].q16(16 * i);
        areg.bs[0] = ab[0].bs8(0);
        areg.bs[1] = ab[0].bs8(1);
      }
      wait_vmcnt(0);
      const int delta = TYPE == T_Q6_K ? (int)(((uintptr_t)(r0 + n0) * (uintptr_t)a.row_bytes) & 15) : 0;
      float V[MAXM], D;
      if constexpr (kReg)
        L::template compute<1, ActRegs>(region, delta + jl * L::kBytes, &areg, 1, V, D);
      else
        L::template compute<MAXM, ActBlock>(region, delta + jl * L::kBytes, ab, M, V, D);
#pragma unroll
      for (int m = 0; m < MAXM; ++m)
        if (m < M && lane < blocks) Vbuf[m * fold_set + to] = V[m];
      if (L::kHasD && lane < blocks) Dbuf[to] = D;
      __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): the stage has been read
      wave_sync();
      issue(task + W);
      for (int f = lane; f < R * M; f += 64) {
        const int fr = f % R, fm = f / R;
        if (fr >= nrows) continue;
        const int p = it.pair(fm);
        float acc[1];
        fold_row<TYPE, 1>(nb, ad + p * fold, Vbuf + fm * fold_set + fr * fold, 0, Dbuf + fr * fold, 0, acc);
        down[p * rows + n0 + fr] = acc[0];
      }
      wave_sync();  // the block values are read before the next set's are written
    }
  }
  lds_barrier();  // the down values are in LDS
  for (int i = tid; i < nr * a.n_tokens; i += blockDim.x) {
    const int t = i / nr, r = i - t * nr, n = live[t];
    float acc = 0.0f;
    for (int j = 0; j < n; ++j) {
      const int p = place[t * a.top_k + j];
      float v = down[p * rows + r];
      if (a.xbf16) v = bf16_to_float(bf16_rne(v));
      acc = acc + v * swt[p];
    }
    out.put((long long)t * a.n + r0 + r, acc);
  }
}

// The routing alone: a wave per token.
__global__ __launch_bounds__(256) void moe_topk_kernel(const void* __restrict__ logits, int bf16, int n_tokens,
                                                       int n_experts, int top_k, int norm_topk, float scale,
                                                       int32_t* __restrict__ ids, float* __restrict__ wts) {
  const int t = (int)blockIdx.x * 4 + ((int)threadIdx.x >> 6);
  if (t >= n_tokens) return;
  route_token(logits, bf16 != 0, (long long)t * n_experts, n_experts, top_k, norm_topk != 0, scale, true,
              [&](int slot, int id, float wt) {
                ids[(long long)t * top_k + slot] = id;
                wts[(long long)t * top_k + slot] = wt;
              });
}

// Rows per wave for a matrix of rows of nb blocks, the most rows that the LDS holds at once (of 6 blocks of Q8_0, gate
// and up, seven waves of 6 rows, not four of 10); 0 where not one wave's rows fit. Whatever a workgroup's share of
// rows is: small experts leave waves without any (above).
template <int TYPE, int MAXM, bool GATEUP>
int layer_rows(int nb) {
  int R = 0, most = 0;
  for (int r = 64 / nb; r >= 1; --r) {
    const int held = r * layer_waves<TYPE, GATEUP>(MAXM, r, nb);
    if (held > most) R = r, most = held;
  }
  return R;
}

// The shape of the second launch that adds up: `rows` output rows a workgroup, at least kSumWaves waves of them, and up
// to kSumPairs pairs, all of whose activations a workgroup quantizes. The second launch adding up, and by items with
// the combine's launch: one token of 8 experts top 2 (4096 x 14336) 26 us and 25.7 + 4.4, of 64 top 8 (2048 x 1024)
// 9.0 and 9.0 + 3.5, of 5 top 1 (4096 x 4096) 7.6 and 8.2 + 2.5; 12 pairs (16 top 4, 2048 x 1536) 11.2 and 10.4 + 3.8;
// 16 pairs (128 top 8, 2048 x 768) 11.3 and 9.3 + 3.8; 24 pairs (40 top 8, 1536 x 512) 13.3 and 7.4 + 3.5, (32 top 3,
// 2560 x 768) 18.7 and 12.8 + 3.9; 32 and 64 pairs of 64 top 8 24.0 and 15.6 + 3.8, 40.4 and 21.1 + 3.9. With six waves
// (two tokens of 8 top 2, 4096 x 14336) 45.5 and 35.8 + 4.5.
constexpr int kSumWaves = 8, kSumPairs = 16;
template <int TYPE, int MAXM>
bool layer_sum_shape(int nb, int pairs, int rows, int& R, int& W, int& lds) {
  R = min(64 / nb, rows);
  const int region = layer_region_bytes<TYPE, false>(MAXM, R, nb);
  const int fixed = layer_sum_bytes(pairs, nb, rows);
  W = min(kLayerWaves - kLayerStagers, (kLayerLds - fixed) / region);
  if (pairs > kSumPairs || fixed >= kLayerLds || W < kSumWaves) return false;
  W = min(W, pairs * ((rows + R - 1) / R));  // the others quantize
  lds = fixed + W * region;
  return true;
}

// Pairs of an item: one for one token, four for more. With two, experts of three and four pairs are read twice: eight
// tokens of 8 experts top 2 (4096 x 14336) 234 us, with four 187; where experts rarely have more than two, two save
// registers only (eight tokens of 32 top 3, 2560 x 768, 41 and 44; of 64 top 8, 2048 x 1024, 56 and 54).
inline int layer_pairs(bool one) { return one ? 1 : 4; }

// f.template operator()<TYPE, MAXM>() of a type and a number of pairs; -1 for another type.
template <class F>
int with_layer_kernel(int type, int pairs, F f) {
  switch (type) {
#define MXA_LAYER(t) \
  case t: return pairs == 1 ? f.template operator()<t, 1>() : f.template operator()<t, 4>();
    MXA_LAYER(T_Q4_K)
    MXA_LAYER(T_Q6_K)
    MXA_LAYER(T_Q8_0)
#undef MXA_LAYER
    default: return -1;
  }
}

// The first launch (GATEUP) or the second's item form; `dry`: whether it fits, no launch. -1 where it does not.
template <bool GATEUP>
struct LaunchLayer {
  LayerArgs a;
  int grid;
  hipStream_t stream;
  bool dry;
  template <int TYPE, int MAXM>
  int operator()() {
    a.R = layer_rows<TYPE, MAXM, GATEUP>(a.nb);
    if (a.R == 0) return -1;
    if (dry) return 0;
    auto kern = moe_layer_kernel<TYPE, MAXM, GATEUP>;
    allow_lds((const void*)kern, kLayerLds);
    hipLaunchKernelGGL(kern, dim3(grid), dim3(64 * kLayerWaves), kLayerLds, stream, a);
    return 0;
  }
};

struct LaunchSum {  // -1 for many pairs, and where its LDS leaves too few waves
  LayerArgs a;
  YOut out;
  int grid;
  hipStream_t stream;
  template <int TYPE, int MAXM>
  int operator()() {
    const int rows = (a.n + grid - 1) / grid;
    int lds;
    if (!layer_sum_shape<TYPE, MAXM>(a.nb, a.n_tokens * a.top_k, rows, a.R, a.W, lds)) return -1;
    auto kern = moe_down_sum_kernel<TYPE, MAXM>;
    allow_lds((const void*)kern, kLayerLds);
    hipLaunchKernelGGL(kern, dim3((a.n + rows - 1) / rows), dim3(64 * kLayerWaves), lds, stream, a, out, rows);
    return 0;
  }
};

}  // namespace

bool moe_layer_supported(int gate_type, int down_type, int n_experts, int top_k, int n_tokens, int n_embd, int ffn) {
  if (n_tokens < 1 || n_tokens > kMoeLayerMaxTokens || top_k < 1 || top_k > min(n_experts, kMoeMaxTopK) ||
      n_experts > kMoeRouteMaxExperts || n_tokens * top_k > kLayerMaxPairs || n_embd % QK != 0 || ffn % QK != 0 ||
      n_embd < QK || ffn < QK || n_embd > 64 * QK || ffn > 64 * QK)
    return false;
  const bool one = n_tokens == 1;
  LayerArgs a{};
  a.nb = n_embd / QK;
  if (with_layer_kernel(gate_type, layer_pairs(one), LaunchLayer<true>{a, 0, nullptr, true}) != 0) return false;
  a.nb = ffn / QK;
  return with_layer_kernel(down_type, layer_pairs(one), LaunchLayer<false>{a, 0, nullptr, true}) == 0;
}

size_t moe_layer_workspace(int n_tokens, int top_k, int n_embd, int ffn, bool bf16) {
  const size_t pairs = (size_t)n_tokens * top_k;
  return align256(pairs * ffn * (bf16 ? 2 : 4)) + align256(pairs * n_embd * 4);
}

int launch_moe_layer(int gate_type, int down_type, const uint8_t* gate, const uint8_t* up, long long gate_stride,
                     long long gate_row, const uint8_t* down, long long down_stride, long long down_row, int n_experts,
                     const void* x, bool bf16, const void* logits, bool logits_bf16, int top_k, bool norm_topk,
                     float scale, int n_tokens, int n_embd, int ffn, bool reciprocal, int32_t* ids, float* wts,
                     YOut out, void* ws, hipStream_t stream) {
  const int grid = cu_count();
  // a workgroup for every item, by their costs of 3 to 6
  if (!moe_layer_supported(gate_type, down_type, n_experts, top_k, n_tokens, n_embd, ffn) ||
      grid < 2 * n_tokens * top_k)
    return -1;
  const size_t pairs = (size_t)n_tokens * top_k;
  uint8_t* const act = (uint8_t*)ws;
  uint8_t* const rows = act + align256(pairs * ffn * (bf16 ? 2 : 4));
  LayerArgs a{gate, up, gate_stride, gate_row, x, ids, wts, act, logits, ffn, n_embd, n_embd / QK, 0, 0,
              n_experts, top_k, n_tokens, logits_bf16 ? 1 : 0, norm_topk ? 1 : 0, bf16 ? 1 : 0, reciprocal ? 1 : 0,
              scale};
  const bool one = n_tokens == 1;
  if (with_layer_kernel(gate_type, layer_pairs(one), LaunchLayer<true>{a, grid, stream, false}) != 0) return -1;
  a.w0 = down, a.w1 = nullptr, a.stride = down_stride, a.row_bytes = down_row, a.x = act, a.act = rows;
  a.n = n_embd, a.k = ffn, a.nb = ffn / QK;
  if (with_layer_kernel(down_type, layer_pairs(one), LaunchSum{a, out, grid, stream}) == 0) return 0;
  if (with_layer_kernel(down_type, layer_pairs(one), LaunchLayer<false>{a, grid, stream, false}) != 0) return -1;
  return launch_moe_combine((const float*)rows, nullptr, ids, wts, n_tokens, top_k, n_embd, bf16 ? 1 : 0, 1, out,
                            stream);
}

int launch_moe_topk(const void* logits, bool bf16, int n_tokens, int n_experts, int top_k, bool norm_topk, float scale,
                    int32_t* ids, float* wts, hipStream_t stream) {
  if (n_tokens < 1 || n_experts < 1 || n_experts > kMoeRouteMaxExperts || top_k < 1 || top_k > min(n_experts, 64))
    return -1;
  hipLaunchKernelGGL(moe_topk_kernel, dim3((n_tokens + 3) / 4), dim3(256), 0, stream, logits, bf16 ? 1 : 0, n_tokens,
                     n_experts, top_k, norm_topk ? 1 : 0, scale, ids, wts);
  return 0;
}

}  // namespace mxa
