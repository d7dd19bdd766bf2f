// The residual stream between two blocks in one pass: a block's output x (optionally normed), gated and
// scaled, is added to the stream r, and the new stream is normed for the next block, whose packed
// projections find its Q8_K blocks written:
//
//   u = x, or x * w_post / sqrt(mean(x^2) + eps_post)
//   h = r + scale * g * u                 rounded once, to the stream's type
//   n = h * w / sqrt(mean(h^2) + eps)     of h as it was stored, rounded once, to the block's type
//
// Every step is float32. The second mean is of the rounded h, so that n is the norm of the stream that
// the next block adds to. (The bfloat16 rms_norm kernel rounds twice, as the torch steps that it restates
// do; here there is no such sequence to restate, and one rounding is closer.)
//
// A row is read once: its values stay in registers, eight to a vector, through both sums. Vectors need no
// alignment beyond their elements' (a row of odd length starts anywhere), and the last one of a row may be
// short. Rows of up to 512 values take one wave each, four rows to a workgroup, with no barrier; longer
// rows a workgroup.
//
// Bound: memory from some 1000 rows on (4096 x 4096 bfloat16 with both norms 28.4 us a call among others for the 134 MB
// of x, r, h and n and the 19 MB of blocks: 5.4 TB/s, a large copy's rate), below that the latency of loads one behind
// another, and of the reductions (1 x 4096 3.8 us; 16 x 5120 with both norms and a gate 6.0). As compiled, a bfloat16
// vector is waited for before the next array's, or the thread's second, is requested (it is widened in the branch that
// loads it); post, gate and w are requested behind the reductions; and of a short last vector one value at a time.
#include "mxa_kernels.hpp"

#pragma clang fp contract(off)

namespace mxa {
namespace {

constexpr int kNormMaxThreads = 1024;

struct NormArgs {
  const void* x;
  const void* r;
  const void* post;  // nullptr: no norm after the block
  const void* gate;  // nullptr: none
  const void* w;
  void* h;
  void* n;
  long long ldx, ldr, ldg;  // row strides in elements
  int gstep;                // the gate's column stride: 1, or 0 for one value a row
  int rows, k;
  float eps, post_eps, scale;
};

typedef uint16_t h16x8 __attribute__((ext_vector_type(8), aligned(2)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

template <bool BF16>
__device__ __forceinline__ float load1(const void* p, long long i) {
  if constexpr (BF16)
    return bf16_to_float(((const uint16_t*)p)[i]);
  else
    return ((const float*)p)[i];
}

// Values i .. i + 7 of p, or the first `count` of them (the rest zero).
template <bool BF16>
__device__ __forceinline__ void load8(const void* p, long long i, int count, float (&v)[8]) {
  if (count == 8) {
    if constexpr (BF16) {
      const h16x8 t = *(const h16x8*)((const uint16_t*)p + i);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = bf16_to_float(t[e]);
    } else {
      const f32x4u a = *(const f32x4u*)((const float*)p + i), b = *(const f32x4u*)((const float*)p + i + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = a[e], v[4 + e] = b[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < count ? load1<BF16>(p, i + e) : 0.0f;
  }
}

// Stores v as p's type (ONCE: past the caches, for what is not read again soon) and leaves in v what was stored.
template <bool BF16, bool ONCE>
__device__ __forceinline__ void store8(void* p, long long i, int count, float (&v)[8]) {
  if constexpr (BF16) {
    h16x8 t;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      t[e] = bf16_rne(v[e]);
      v[e] = bf16_to_float(t[e]);
    }
    if (count == 8) {
      h16x8* to = (h16x8*)((uint16_t*)p + i);
      if constexpr (ONCE)
        __builtin_nontemporal_store(t, to);
      else
        *to = t;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < count) ((uint16_t*)p)[i + e] = t[e];
    }
  } else {
    if (count == 8) {
      const f32x4u t0{v[0], v[1], v[2], v[3]}, t1{v[4], v[5], v[6], v[7]};
      f32x4u* to = (f32x4u*)((float*)p + i);
      if constexpr (ONCE) {
        __builtin_nontemporal_store(t0, to);
        __builtin_nontemporal_store(t1, (f32x4u*)((float*)p + i + 4));
      } else {
        *to = t0;
        *(f32x4u*)((float*)p + i + 4) = t1;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < count) ((float*)p)[i + e] = v[e];
    }
  }
}

// Q8_K of two 256-value blocks held by a wave, eight values per lane (lanes 0..31 the first, 32..63 the
// second; either half may hold a block that is not stored): the steps of q8k_part16.
__device__ __forceinline__ void q8k_part8(const float (&v)[8], int lane, bool store, int8_t* qblk, int16_t* bsblk,
                                          float* dp) {
  float amax = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(v[i]));
  amax = max16(amax);
  const auto lane_max = [&](int l) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, amax), l));
  };
  const float m0 = fmaxf(lane_max(0), lane_max(16)), m1 = fmaxf(lane_max(32), lane_max(48));
  amax = lane < 32 ? m0 : m1;
  int qv[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) qv[i] = 0;
  if (amax != 0.0f) {
    const float iscale = 127.0f / amax;
#pragma unroll
    for (int i = 0; i < 8; ++i) qv[i] = (int)fminf(fmaxf(rintf(v[i] * iscale), -127.0f), 127.0f);
  }
  uint32_t packed[2];
  int bsum = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    packed[i] = (uint32_t)(qv[4 * i] & 0xFF) | ((uint32_t)(qv[4 * i + 1] & 0xFF) << 8) |
                ((uint32_t)(qv[4 * i + 2] & 0xFF) << 16) | ((uint32_t)(qv[4 * i + 3] & 0xFF) << 24);
    bsum += qv[4 * i] + qv[4 * i + 1] + qv[4 * i + 2] + qv[4 * i + 3];
  }
  bsum += quad_xor1(bsum);  // 16 values: two lanes
  if (!store) return;
  const int p = lane & 31;
  *(uint2*)(qblk + 8 * p) = uint2{packed[0], packed[1]};
  if ((p & 1) == 0) bsblk[p >> 1] = (int16_t)bsum;
  if (p == 0) *dp = amax / 127.0f;
}

// Thread t of a row's T holds vectors t + T j, j < P.
template <bool XB, bool RB, bool POST, int P, bool ONCE>
__global__ __launch_bounds__(kNormMaxThreads) void add_rms_norm_kernel(NormArgs a, int T, int8_t* __restrict__ q,
                                                                       float* __restrict__ d,
                                                                       int16_t* __restrict__ bsums) {
  __shared__ float part[2][kNormMaxThreads / 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const bool solo = T == 64;  // a wave per row
  const int row = solo ? (int)(blockIdx.x * (blockDim.x >> 6)) + wave : (int)blockIdx.x;
  if (solo && row >= a.rows) return;  // no barrier follows for such rows
  const int t = solo ? lane : (int)threadIdx.x, k = a.k;
  const auto row_sum = [&](float s, int which) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) s = s + __shfl_xor(s, o);
    if (solo) return s;
    if (lane == 0) part[which][wave] = s;
    __syncthreads();
    float sum = 0.0f;
    for (int i = 0; i < T / 64; ++i) sum = sum + part[which][i];
    return sum;
  };
  int count[P];
  float u[P][8], h[P][8] = {};
#pragma unroll
  for (int j = 0; j < P; ++j) {
    const int i = 8 * (t + T * j);
    count[j] = min(8, k - i);
    if (count[j] > 0) {
      load8<XB>(a.x, (long long)row * a.ldx + i, count[j], u[j]);
      load8<RB>(a.r, (long long)row * a.ldr + i, count[j], h[j]);
    }
  }
  if constexpr (POST) {
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < P; ++j)
      if (count[j] > 0)
#pragma unroll
        for (int e = 0; e < 8; ++e) s = fmaf(u[j][e], u[j][e], s);
    const float scale = 1.0f / sqrtf(row_sum(s, 0) / (float)k + a.post_eps);
#pragma unroll
    for (int j = 0; j < P; ++j) {
      if (count[j] <= 0) continue;
      float w[8];
      load8<XB>(a.post, 8 * (t + T * j), count[j], w);
#pragma unroll
      for (int e = 0; e < 8; ++e) u[j][e] = u[j][e] * scale * w[e];
    }
  }
  float s = 0.0f;
#pragma unroll
  for (int j = 0; j < P; ++j) {
    if (count[j] <= 0) continue;
    const int i = 8 * (t + T * j);
    if (a.gate != nullptr) {
      float g[8];
      if (a.gstep == 0) {
        g[0] = load1<XB>(a.gate, (long long)row * a.ldg);
#pragma unroll
        for (int e = 1; e < 8; ++e) g[e] = g[0];
      } else {
        load8<XB>(a.gate, (long long)row * a.ldg + i, count[j], g);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) u[j][e] = u[j][e] * g[e];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) h[j][e] = fmaf(a.scale, u[j][e], h[j][e]);
    store8<RB, ONCE>(a.h, (long long)row * k + i, count[j], h[j]);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < count[j]) s = fmaf(h[j][e], h[j][e], s);
  }
  const float scale = 1.0f / sqrtf(row_sum(s, 1) / (float)k + a.eps);
  const int nb = k / QK;
#pragma unroll
  for (int j = 0; j < P; ++j) {
    const int i = 8 * (t + T * j);
    if (count[j] > 0) {
      float w[8];
      load8<XB>(a.w, i, count[j], w);
#pragma unroll
      for (int e = 0; e < 8; ++e) h[j][e] = h[j][e] * scale * w[e];
      store8<XB, ONCE>(a.n, (long long)row * k + i, count[j], h[j]);
    }
    if (q != nullptr) {  // every lane of the wave: k is a multiple of 256, a half wave holds a block or nothing
      const size_t b = (size_t)row * nb + (i >> 8);
      q8k_part8(h[j], lane, count[j] > 0, q + b * QK, bsums + b * 16, d + b);
    }
  }
}

template <bool XB, bool RB, bool POST>
void launch_norm(const NormArgs& a, const ActBuffers* q, hipStream_t stream) {
  const int nv = (a.k + 7) / 8;
  // Few rows: as many threads a row as there are vectors. Many rows: two vectors a thread, half the waves and
  // reductions (4096 bfloat16 rows of 4096 with a norm on both sides, kernel alone: one vector a thread 37.1 us, two
  // 35.8, four 45.8).
  const bool many = a.rows > 512;
  // h and n past the caches from 8 MB of them together. Times past the caches against plain stores, of this kernel
  // alone and with the next add_rms_norm behind it, which reads h and n at once (every output in memory of its own, x
  // just written or not): below 8 MB within 8%, both; both bfloat16 12 to 48 MB 4 to 29% less alone and from 19% less
  // to 3% more together, 56 to 128 MB 3 to 15% less and -9 to +9%, above 0 to 10% and 1 to 8% less; one or both float32
  // 12 to 28 MB 11 to 17% and 1 to 19% less, 32 to 128 MB -15 to +4% and -3 to +13%, above -5 to +1% and -4 to +4%. (A
  // layer reads n at once or its blocks alone, h after the block. 1024 bfloat16 rows of 4096: 10.2 us plain and 8.5,
  // with the next 18.4 and 16.1.)
  const bool once = (long long)a.rows * a.k * ((RB ? 2 : 4) + (XB ? 2 : 4)) >= 8000000;
  const int fewest = (nv + kNormMaxThreads - 1) / kNormMaxThreads;
  const int want = many && nv >= 128 ? 2 : 1;
  const int p = max(fewest, want) <= 1 ? 1 : max(fewest, want) <= 2 ? 2 : 4;
  const int T = ((nv + p - 1) / p + 63) / 64 * 64;
  const int waves = T == 64 ? 4 : T / 64;
  const dim3 grid(T == 64 ? (a.rows + 3) / 4 : a.rows), block(64 * waves);
  int8_t* qq = q != nullptr ? q->q : nullptr;
  float* qd = q != nullptr ? q->d : nullptr;
  int16_t* qb = q != nullptr ? q->bsums : nullptr;
  auto kern = once ? (p == 1 ? add_rms_norm_kernel<XB, RB, POST, 1, true>
                      : p == 2 ? add_rms_norm_kernel<XB, RB, POST, 2, true>
                               : add_rms_norm_kernel<XB, RB, POST, 4, true>)
                   : (p == 1 ? add_rms_norm_kernel<XB, RB, POST, 1, false>
                      : p == 2 ? add_rms_norm_kernel<XB, RB, POST, 2, false>
                               : add_rms_norm_kernel<XB, RB, POST, 4, false>);
  hipLaunchKernelGGL(kern, grid, block, 0, stream, a, T, qq, qd, qb);
}

}  // namespace

int launch_add_rms_norm(const void* x, long long ldx, const void* r, long long ldr, const void* post,
                        float post_eps, const void* gate, long long ldg, int gstep, float scale, const void* w,
                        float eps, bool xbf16, bool rbf16, int rows, int k, void* h, void* n,
                        const ActBuffers* q, hipStream_t stream) {
  if (k > kNormMaxValues || (rbf16 && !xbf16)) return -1;
  const NormArgs a{x, r, post, gate, w, h, n, ldx, ldr, ldg, gstep, rows, k, eps, post_eps, scale};
  if (post != nullptr) {
    if (!xbf16) launch_norm<false, false, true>(a, q, stream);
    else if (rbf16) launch_norm<true, true, true>(a, q, stream);
    else launch_norm<true, false, true>(a, q, stream);
  } else {
    if (!xbf16) launch_norm<false, false, false>(a, q, stream);
    else if (rbf16) launch_norm<true, true, false>(a, q, stream);
    else launch_norm<true, false, false>(a, q, stream);
  }
  return 0;
}

}  // namespace mxa
