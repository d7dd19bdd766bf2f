// Rotary positions of q and k, one launch: pair i of a head's rotary part (d = rot values) turns by p * f_i at
// position p,
//
//   (a, b) -> m (a cos - b sin, a sin + b cos),
//
// the pair being elements (i, i + d / 2), or (2 i, 2 i + 1) when interleaved; the values behind the rotary part
// are copied.
//
// Angles. In float32 the product p * f_i of a far position is off by p * 2^-24 radians (0.06 at a million), so the
// table holds the turns per position f_i / (2 pi) in float64 and the angle is the fraction of p * turns, taken
// there: off by less than 2^-33 turns up to p = 2^20. The sine and cosine of that fraction are float32. Both are
// computed once for a (token, pair) and read from LDS by every head.
//
// A thread keeps one place of the heads (a vector of V pairs, or of V / 2 pairs interleaved) and walks over the
// (token, head) rows of its workgroup, a batch of rows loaded before the first is computed, the first batch before the
// angles. As compiled, a row's loads wait for those of the row before it in the batch (its address is formed behind a
// branch, in registers that those loads write), the table's load for the position's, and the outputs are flat stores
// (their pointer is q's or k's), behind which the reads of the next row's cosines wait.
//
// Bound: memory from some thousand tokens on (4096 tokens of 32 + 8 bfloat16 heads of 128: 15.6 us for 84 MB, 5.4 TB/s,
// a large copy's rate), below that latency, of the loads above one behind another and of sine and cosine (one token
// 3.1 us; 777 tokens of 40 + 8 heads 6.5, whose 19 MB take 3.7 at a copy's rate).
#include "mxa_kernels.hpp"

#pragma clang fp contract(off)

namespace mxa {
namespace {

constexpr int kRopeThreads = 256, kRopeBatch = 4;

struct RopeSide {  // q or k
  const void* x;
  void* out;
  long long batch, tok, head;  // strides in elements
  int heads;
};
struct RopeArgs {
  RopeSide q, k;
  const void* pos;
  long long pos_batch, pos_tok;
  const double* turns;
  int pos64, n_tokens, seq, dim, rot;  // token t is step t % seq of sequence t / seq
  float mscale;
};

template <class T, int V>
struct Vec {
  typedef T type __attribute__((ext_vector_type(V), aligned(sizeof(T))));
};
template <class T>
struct Vec<T, 1> {
  typedef T type;
};

template <class T>
__device__ __forceinline__ float widen(T v) {
  if constexpr (sizeof(T) == 2)
    return bf16_to_float(v);
  else
    return v;
}
template <class T>
__device__ __forceinline__ T narrow(float v) {
  if constexpr (sizeof(T) == 2)
    return bf16_rne(v);
  else
    return v;
}

// T the element type; V values of a vector (an even number for interleaved pairs); ONCE: stored past the caches.
template <class T, bool INTER, int V, bool ONCE>
__global__ __launch_bounds__(kRopeThreads) void rope_kernel(RopeArgs a, int TP, int C, int CR, int HP) {
  extern __shared__ __align__(16) float trig[];  // cos of (token, pair), then sin
  union Piece {
    typename Vec<T, V>::type v;
    T e[V];
  };
  const int half = a.rot / 2, tid = threadIdx.x;
  const int tok0 = (int)blockIdx.x * TP, nt = min(TP, a.n_tokens - tok0);
  const int H = a.q.heads + a.k.heads, rows = nt * H;
  float* const cs = trig;
  float* const sn = trig + TP * half;
  const int width = min(C, kRopeThreads), r0 = tid / width, step = HP * (int)gridDim.y;
  const int first = r0 < HP ? (int)blockIdx.y * HP + r0 : rows;  // threads past the last whole row of places idle

  const bool one = a.seq >= a.n_tokens;  // one sequence: no division for a token's
  // the source and the destination of row r (token r / H, head r % H)
  const auto place = [&](int r, const T*& src, T*& dst) {
    const int t = tok0 + r / H, hh = r % H;
    const bool isq = hh < a.q.heads;
    const RopeSide& s = isq ? a.q : a.k;
    const int h = isq ? hh : hh - a.q.heads;
    const int b = one ? 0 : t / a.seq;
    src = (const T*)s.x + (long long)b * s.batch + (long long)(t - b * a.seq) * s.tok + (long long)h * s.head;
    dst = (T*)s.out + ((long long)t * s.heads + h) * a.dim;
  };
  const auto load = [&](const T* src, int c, Piece& x, Piece& y) {
    if (c >= CR) {
      x.v = *(const typename Vec<T, V>::type*)(src + a.rot + (c - CR) * V);
    } else {
      x.v = *(const typename Vec<T, V>::type*)(src + c * V);
      if constexpr (!INTER) y.v = *(const typename Vec<T, V>::type*)(src + half + c * V);
    }
  };
  const auto put = [&](T* to, const Piece& p) __attribute__((always_inline)) {
    if constexpr (ONCE)
      __builtin_nontemporal_store(p.v, (typename Vec<T, V>::type*)to);
    else
      *(typename Vec<T, V>::type*)to = p.v;
  };
  const auto store = [&](T* dst, int t, int c, Piece& x, Piece& y) {
    if (c >= CR) {
      put(dst + a.rot + (c - CR) * V, x);
      return;
    }
    if constexpr (INTER) {
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        const float co = cs[t * half + c * (V / 2) + i], si = sn[t * half + c * (V / 2) + i];
        const float u = widen(x.e[2 * i]), v = widen(x.e[2 * i + 1]);
        x.e[2 * i] = narrow<T>(fmaf(u, co, -(v * si)));
        x.e[2 * i + 1] = narrow<T>(fmaf(u, si, v * co));
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float co = cs[t * half + c * V + i], si = sn[t * half + c * V + i];
        const float u = widen(x.e[i]), v = widen(y.e[i]);
        x.e[i] = narrow<T>(fmaf(u, co, -(v * si)));
        y.e[i] = narrow<T>(fmaf(u, si, v * co));
      }
      put(dst + half + c * V, y);
    }
    put(dst + c * V, x);
  };

  bool angles = false;
  for (int c = tid - r0 * width; c < C; c += kRopeThreads) {  // once unless a head has more than 256 places
    int r = first;
    do {
      const T* src[kRopeBatch];
      T* dst[kRopeBatch];
      Piece x[kRopeBatch], y[kRopeBatch];
#pragma unroll
      for (int j = 0; j < kRopeBatch; ++j)
        if (r + j * step < rows) {
          place(r + j * step, src[j], dst[j]);
          load(src[j], c, x[j], y[j]);
        }
      if (!angles) {  // uniform over the workgroup: every thread comes here once
        angles = true;
        for (int i = tid; i < nt * half; i += kRopeThreads) {
          const int t = tok0 + i / half, b = one ? 0 : t / a.seq;
          const long long at = b * a.pos_batch + (t - b * a.seq) * a.pos_tok;
          const double p = a.pos64 ? (double)((const long long*)a.pos)[at] : (double)((const int32_t*)a.pos)[at];
          const double turns = p * a.turns[i % half];
          float s, co;
          sincospif(2.0f * (float)(turns - rint(turns)), &s, &co);
          cs[i] = a.mscale * co;
          sn[i] = a.mscale * s;
        }
        __syncthreads();
      }
#pragma unroll
      for (int j = 0; j < kRopeBatch; ++j)
        if (r + j * step < rows) store(dst[j], (r + j * step) / H, c, x[j], y[j]);
      r += kRopeBatch * step;
    } while (r < rows);
  }
}

template <class T, bool INTER, int V>
void launch_rope_v(const RopeArgs& a, hipStream_t stream) {
  const int CR = INTER ? a.rot / V : a.rot / 2 / V;  // places of a head: rotary, then copied
  const int C = CR + (a.dim - a.rot) / V;
  const int HP = max(1, kRopeThreads / C);  // heads side by side in a workgroup
  const int H = a.q.heads + a.k.heads;
  // Up to 512 tokens the heads of one token over several workgroups, a row a thread (32 + 8 bfloat16 heads of 128,
  // kernel alone: 300 tokens 5.0 us, a workgroup a token 5.4; 700 tokens 7.0 and 6.3). More: a workgroup a token, or
  // as many tokens each as leave about a thousand workgroups, what the CUs hold at once (1500 tokens by one 11.2, by
  // two 10.2, by four 11.6; 4096 by two 19.6, by four 17.3, by eight 19.6).
  const bool many = a.n_tokens > 512;
  const int TP = many ? min(8, (a.n_tokens + 1023) / 1024) : 1;
  const int split = many ? 1 : min(4096, (H + HP - 1) / HP);  // a grid's threads have to stay below 2^32
  // The outputs past the caches from 4 MB of them on, where every head turns whole, in 16-byte vectors. Times past the
  // caches against plain stores, of this kernel alone and with a kernel behind it that reads what it wrote (every
  // output in memory of its own, q and k just written or not): below 4 MB within 5%, both; bfloat16 4 to 12 MB 1 to
  // 13% less alone and 0 to 13% less together, 16 to 48 MB 3 to 29% less and from 21% less to 8% more, 56 to 128 MB 2
  // to 15% less and -10 to +7%, above 0 to 8% less and from 9% less to 1% more; float32 in halves much the same,
  // interleaved from 20 MB on from 30% less to 1% more and -8 to +13%. Parts of a head, stored in pieces that are no
  // whole lines, and vectors of less than 16 bytes gain less than they lose: from 29% less to 26% more alone, up to
  // 38% more with the reader (bfloat16 32 of 80 values, 42 MB: 33.9 us plain and 35.1, with the reader 61.8 and 76.3;
  // 20 of 80 127 and 117, 241 and 259).
  auto kern = rope_kernel<T, INTER, V, false>;
  if constexpr (V * sizeof(T) == 16) {
    if (a.rot == a.dim && (long long)a.n_tokens * H * a.dim * (long long)sizeof(T) >= 4000000)
      kern = rope_kernel<T, INTER, V, true>;
  }
  hipLaunchKernelGGL(kern, dim3((a.n_tokens + TP - 1) / TP, split), dim3(kRopeThreads),
                     (size_t)TP * a.rot * sizeof(float), stream, a, TP, C, CR, HP);
}

template <class T, bool INTER>
void launch_rope_t(const RopeArgs& a, hipStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  if ((INTER ? a.rot : a.rot / 2) % V == 0 && (a.dim - a.rot) % V == 0)
    launch_rope_v<T, INTER, V>(a, stream);
  else
    launch_rope_v<T, INTER, INTER ? 2 : 1>(a, stream);
}

}  // namespace

int launch_rope(const void* q, const long long* q_strides, int q_heads, const void* k, const long long* k_strides,
                int k_heads, const void* pos, bool pos64, long long pos_batch, long long pos_tok,
                const double* turns, int n_tokens, int seq, int dim, int rot, bool interleaved, float mscale,
                bool bf16, void* q_out, void* k_out, hipStream_t stream) {
  const RopeArgs a{{q, q_out, q_strides[0], q_strides[1], q_strides[2], q_heads},
                   {k, k_out, k_heads ? k_strides[0] : 0, k_heads ? k_strides[1] : 0, k_heads ? k_strides[2] : 0,
                    k_heads},
                   pos, pos_batch, pos_tok, turns, pos64 ? 1 : 0, n_tokens, seq, dim, rot, mscale};
  if (bf16)
    interleaved ? launch_rope_t<uint16_t, true>(a, stream) : launch_rope_t<uint16_t, false>(a, stream);
  else
    interleaved ? launch_rope_t<float, true>(a, stream) : launch_rope_t<float, false>(a, stream);
  return 0;
}

}  // namespace mxa
