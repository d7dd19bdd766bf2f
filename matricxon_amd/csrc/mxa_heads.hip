// What stands between a layer's q | k | v projections and its attention, in one launch:
//
//   y = turn(x * w / sqrt(mean(x^2) + eps), p)       each head of q and of k; either step may be absent
//
// (mxa_rope.hip has the rotation without norms), and, with a cache, k so turned and v written to its pages in 4 bits:
// of 32 neighbouring values m = f16(min), s = f16((max - min) / 15), code = clamp(rint((x - m) / s), 0, 15).
//
// Every step is float32 (angles as in mxa_rope.hip: turns in float64, reduced there), q and an uncached k are rounded
// once, and the codes are taken of the float32 values against the rounded s and m, so that the held values are the
// nearest that these two allow.
//
// L lanes hold a head, each the vectors at i and i + rot / 2 whose values turn with each other, so that nothing but the
// sum of squares crosses lanes. Heads whose rotary part does not split into whole vectors take a wave each, a pair of
// values at a time.
#include "mxa_kernels.hpp"
#include "mxa_kv4.hpp"

#pragma clang fp contract(off)

namespace mxa {
namespace {

constexpr int kHeadThreads = 256, kHeadBatch = 4;

struct HeadSide {
  const void* x;
  void* out;
  const void* w;               // nullptr: no norm
  long long batch, tok, head;  // strides in elements
  int heads;
};
struct HeadArgs {
  HeadSide q, k, v;
  const void* pos;  // nullptr: a token's place in its sequence
  long long pos_batch, pos_tok;
  const double* turns;
  int pos64, n_tokens, seq, dim, rot;  // token t is step t % seq of sequence t / seq
  float mscale, eps;
  KvPages kv;
};

template <class T, int V>
struct Vec {
  typedef T type __attribute__((ext_vector_type(V), aligned(sizeof(T))));
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

template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xF, 0xF, false));
}
// The sum over L neighbouring lanes (a power of two), in all of them.
__device__ __forceinline__ float lanes_sum(float v, int L) {
  if (L > 1) v += dpp<0xB1>(v);
  if (L > 2) v += dpp<0x4E>(v);
  if (L > 4) v += dpp<0x141>(v);
  if (L > 8) v += dpp<0x140>(v);
  if (L > 16) v += __shfl_xor(v, 16);
  if (L > 32) v += __shfl_xor(v, 32);
  return v;
}
__device__ __forceinline__ float quad_min(float v) {
  v = fminf(v, dpp<0xB1>(v));
  return fminf(v, dpp<0x4E>(v));
}
__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, dpp<0xB1>(v));
  return fmaxf(v, dpp<0x4E>(v));
}

// The codes of eight values of a group that the four lanes of a quad hold between them (`here`: whether this lane has
// any), and the group's scale and minimum, which come back as bits of float16. A NaN is held as 0 and an infinity as
// the largest: a cached value is always finite.
__device__ __forceinline__ void quantize8(float (&x)[8], bool here, int (&code)[8], uint16_t& s_bits, uint16_t& m_bits) {
  float lo = INFINITY, hi = -INFINITY;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    x[j] = x[j] == x[j] ? fminf(fmaxf(x[j], -kKvHeld), kKvHeld) : 0.0f;
    if (here) {
      lo = fminf(lo, x[j]);
      hi = fmaxf(hi, x[j]);
    }
  }
  lo = quad_min(lo);
  hi = quad_max(hi);
  const _Float16 mh = (_Float16)lo, sh = (_Float16)((hi - lo) / 15.0f);
  const float m = (float)mh, s = (float)sh;
#pragma unroll
  for (int j = 0; j < 8; ++j) code[j] = here && s > 0.0f ? (int)fminf(fmaxf(rintf((x[j] - m) / s), 0.0f), 15.0f) : 0;
  s_bits = __builtin_bit_cast(uint16_t, sh);
  m_bits = __builtin_bit_cast(uint16_t, mh);
}

struct Spot {       // of one token of the workgroup
  long long block;  // of its first head, or -1: it is not cached
  int place, seq;   // seq -1: a row of no sequence
};

// T the element type; FAST: vectors of V values. A workgroup takes TP tokens and, from grid.y, HQ heads of q and HK of k.
template <class T, bool INTER, bool FAST, bool CACHE>
__global__ __launch_bounds__(kHeadThreads) void heads_kernel(HeadArgs a, int TP, int L, int HQ, int HK) {
  constexpr int V = FAST ? 16 / (int)sizeof(T) : 1;
  extern __shared__ __align__(16) unsigned char smem[];
  typedef typename Vec<T, FAST ? V : 2>::type Vv;
  union Piece {
    Vv v;
    T e[FAST ? V : 2];
  };
  const int half = a.rot / 2, tid = threadIdx.x;
  const int W = kv_groups(a.dim);
  Spot* const spots = (Spot*)smem;
  float* const cs = (float*)(smem + (CACHE ? TP * sizeof(Spot) : 0));  // cos of (token, pair), then sin
  float* const sn = cs + TP * half;
  float* const keys = sn + TP * half;  // CACHE: turned keys (token, head, 32 W)
  const int tok0 = (int)blockIdx.x * TP, nt = min(TP, a.n_tokens - tok0);
  const int q0 = (int)blockIdx.y * HQ, nq = max(0, min(HQ, a.q.heads - q0));
  const int k0 = (int)blockIdx.y * HK, nk = max(0, min(HK, a.k.heads - k0));
  const int H = nq + nk, rows = nt * H;
  const bool one = a.seq >= a.n_tokens;
  const auto from = [&](const HeadSide& s, int t, int h) {
    const int b = one ? 0 : t / a.seq;
    return (const T*)s.x + (long long)b * s.batch + (long long)(t - b * a.seq) * s.tok + (long long)h * s.head;
  };

  if constexpr (CACHE) {
    for (int t = tid; t < nt; t += kHeadThreads) {
      int place;
      const int b = kv_place(a.kv, tok0 + t, a.n_tokens, place);
      spots[t].place = place;
      spots[t].seq = b;
      spots[t].block = b < 0 ? -1 : kv_block(a.kv, b, place);
    }
    __syncthreads();
  }
  for (int i = tid; i < nt * half; i += kHeadThreads) {
    const int t = i / half, tt = tok0 + t, b = one ? 0 : tt / a.seq;
    double p;
    if (CACHE && a.pos == nullptr) {
      p = (double)spots[t].place;
    } else {
      const long long at = b * a.pos_batch + (tt - b * a.seq) * a.pos_tok;
      p = a.pos64 ? (double)((const long long*)a.pos)[at] : (double)((const int32_t*)a.pos)[at];
    }
    const double turns = p * a.turns[i - t * half];
    float s, co;
    sincospif(2.0f * (float)(turns - rint(turns)), &s, &co);
    cs[i] = a.mscale * co;
    sn[i] = a.mscale * s;
  }
  __syncthreads();

  const int per = kHeadThreads / L, c = tid % L;
  const int CR = FAST ? (INTER ? a.rot / V : half / V) : 0, C = FAST ? CR + (a.dim - a.rot) / V : 0;
  for (int base = 0; base < rows; base += per) {  // the same count for every thread: lanes exchange sums
    const int r = base + tid / L;
    const bool live = r < rows;
    const int t = live ? r / H : 0, hh = live ? r - t * H : 0;
    const bool isq = hh < nq;
    const HeadSide& s = isq ? a.q : a.k;
    const int h = isq ? q0 + hh : k0 + hh - nq;
    const T* const src = from(s, tok0 + t, h);
    T* const dst = (T*)s.out + ((long long)(tok0 + t) * s.heads + h) * a.dim;
    float* const key = CACHE && !isq ? keys + (t * HK + hh - nq) * 32 * W : nullptr;
    const T* const w = (const T*)s.w;
    const bool none = CACHE && spots[t].seq < 0;  // its q comes back as zeros
    if constexpr (FAST) {
      Piece x, y;
      float xf[V], yf[V];
      const bool mine = live && c < C, turned = c < CR;
      const int at = turned ? c * V : a.rot + (c - CR) * V;
      float ss = 0.0f;
#pragma unroll
      for (int i = 0; i < V; ++i) xf[i] = yf[i] = 0.0f;
      if (mine) {
        x.v = *(const Vv*)(src + at);
        if (!INTER && turned) y.v = *(const Vv*)(src + half + at);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          xf[i] = widen(x.e[i]);
          yf[i] = !INTER && turned ? widen(y.e[i]) : 0.0f;
          ss += xf[i] * xf[i] + yf[i] * yf[i];
        }
      }
      if (a.q.w != nullptr || a.k.w != nullptr) ss = lanes_sum(ss, L);
      if (mine) {
        if (w != nullptr) {
          const float rn = 1.0f / sqrtf(ss / (float)a.dim + a.eps);
          Piece wx, wy;
          wx.v = *(const Vv*)(w + at);
          if (!INTER && turned) wy.v = *(const Vv*)(w + half + at);
#pragma unroll
          for (int i = 0; i < V; ++i) {
            xf[i] = xf[i] * rn * widen(wx.e[i]);
            if (!INTER && turned) yf[i] = yf[i] * rn * widen(wy.e[i]);
          }
        }
        if (turned) {
          if constexpr (INTER) {
#pragma unroll
            for (int i = 0; i < V / 2; ++i) {
              const float co = cs[t * half + c * (V / 2) + i], si = sn[t * half + c * (V / 2) + i];
              const float u = xf[2 * i], v = xf[2 * i + 1];
              xf[2 * i] = fmaf(u, co, -(v * si));
              xf[2 * i + 1] = fmaf(u, si, v * co);
            }
          } else {
#pragma unroll
            for (int i = 0; i < V; ++i) {
              const float co = cs[t * half + c * V + i], si = sn[t * half + c * V + i];
              const float u = xf[i], v = yf[i];
              xf[i] = fmaf(u, co, -(v * si));
              yf[i] = fmaf(u, si, v * co);
            }
          }
        }
        if (key != nullptr) {
#pragma unroll
          for (int i = 0; i < V; ++i) {
            key[at + i] = xf[i];
            if (!INTER && turned) key[half + at + i] = yf[i];
          }
        } else {
#pragma unroll
          for (int i = 0; i < V; ++i) {
            x.e[i] = narrow<T>(none ? 0.0f : xf[i]);
            y.e[i] = narrow<T>(none ? 0.0f : yf[i]);
          }
          *(Vv*)(dst + at) = x.v;
          if (!INTER && turned) *(Vv*)(dst + half + at) = y.v;
        }
      }
    } else {
      float ss = 0.0f;
      if (live && w != nullptr)
        for (int i = c; i < a.dim; i += L) {
          const float v = widen(src[i]);
          ss += v * v;
        }
      if (a.q.w != nullptr || a.k.w != nullptr) ss = lanes_sum(ss, L);
      const float rn = w != nullptr ? 1.0f / sqrtf(ss / (float)a.dim + a.eps) : 1.0f;
      const auto get = [&](int i) {
        const float v = widen(src[i]);
        return w != nullptr ? v * rn * widen(w[i]) : v;
      };
      const auto put = [&](int i, float v) {
        if (key != nullptr)
          key[i] = v;
        else
          dst[i] = narrow<T>(none ? 0.0f : v);
      };
      if (live) {
        for (int i = c; i < half; i += L) {
          const int iu = INTER ? 2 * i : i, iv = INTER ? 2 * i + 1 : half + i;
          const float co = cs[t * half + i], si = sn[t * half + i], u = get(iu), v = get(iv);
          put(iu, fmaf(u, co, -(v * si)));
          put(iv, fmaf(u, si, v * co));
        }
        for (int i = a.rot + c; i < a.dim; i += L) put(i, get(i));
      }
    }
  }

  if constexpr (CACHE) {
    __syncthreads();
    const int O = 4 * W, blocks = a.kv.page / kKvBlock;
    const long long bytes = kv_block_bytes(W);
    for (int base = 0; base < nt * nk * O; base += kHeadThreads) {  // quads of lanes share a group: O is whole quads
      const int item = base + tid;
      const bool live = item < nt * nk * O;
      const int row = live ? item / O : 0, o = live ? item - row * O : 0, t = row / nk, h = row - t * nk;
      const bool here = live && o * 8 < a.dim;
      float x[8];
      int code[8];
      uint16_t sb, mb;
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = here ? keys[(t * HK + h) * 32 * W + o * 8 + j] : 0.0f;
      quantize8(x, here, code, sb, mb);
      if (!live || spots[t].block < 0) continue;
      uint32_t word = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) word |= (uint32_t)code[j] << (4 * j);
      uint8_t* const blk = a.kv.pages + (spots[t].block + (long long)(k0 + h) * blocks) * bytes;
      const int tok = spots[t].place % kKvBlock;
      *(uint32_t*)(blk + tok * 16 * W + (o % 4) * 4 * W + (o / 4) * 4) = word;
      if (o % 4 == 0) *(uint32_t*)(blk + kv_key_scales(W) + (tok * W + o / 4) * 4) = sb | (uint32_t)mb << 16;
    }
    const int quads = (nt + 3) / 4;
    for (int base = 0; base < quads * nk * O; base += kHeadThreads) {
      const int item = base + tid;
      const bool live = item < quads * nk * O;
      const int row = live ? item / O : 0, o = live ? item - row * O : 0, qd = row / nk, h = row - qd * nk;
      const bool here = live && o * 8 < a.dim;
      uint32_t words[4] = {0, 0, 0, 0};
      uint16_t sb[4], mb[4];
#pragma unroll
      for (int z = 0; z < 4; ++z) {
        const int t = qd * 4 + z;
        const bool has = here && t < nt;
        float x[8];
        int code[8];
        const T* const src = from(a.v, tok0 + min(t, nt - 1), k0 + h) + o * 8;
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = has ? widen(src[j]) : 0.0f;
        quantize8(x, has, code, sb[z], mb[z]);
#pragma unroll
        for (int j = 0; j < 4; ++j) words[j] |= (uint32_t)(code[2 * j] | code[2 * j + 1] << 4) << (8 * z);
      }
      if (!live) continue;
      const Spot first = spots[qd * 4];
      bool whole = qd * 4 + 3 < nt && first.block >= 0 && first.place % 4 == 0;
#pragma unroll
      for (int z = 1; z < 4; ++z)
        whole = whole && spots[min(qd * 4 + z, nt - 1)].block == first.block &&
                spots[min(qd * 4 + z, nt - 1)].place == first.place + z;
      const auto at = [&](long long block) { return a.kv.pages + (block + (long long)(k0 + h) * blocks) * bytes; };
      const int gg = o / 4;
      if (whole) {
        uint8_t* const blk = at(first.block);
        const int tok = first.place % kKvBlock;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          *(uint32_t*)(blk + kv_value_codes(W) + kv_value_word(W, gg, tok / 4 % 4, o % 4 * 4 + j, tok / 16)) = words[j];
        if (o % 4 == 0) {
          uint32_t* const to = (uint32_t*)(blk + kv_value_scales(W) + (gg * 8 + tok / 4) * 16);
          to[0] = sb[0] | (uint32_t)sb[2] << 16;
          to[1] = sb[1] | (uint32_t)sb[3] << 16;
          to[2] = mb[0] | (uint32_t)mb[2] << 16;
          to[3] = mb[1] | (uint32_t)mb[3] << 16;
        }
      } else {
#pragma unroll
        for (int z = 0; z < 4; ++z) {
          const int t = qd * 4 + z;
          if (t >= nt || spots[t].block < 0) continue;
          uint8_t* const blk = at(spots[t].block);
          const int tok = spots[t].place % kKvBlock;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            blk[kv_value_codes(W) + kv_value_word(W, gg, tok / 4 % 4, o % 4 * 4 + j, tok / 16) + tok % 4] =
                (uint8_t)(words[j] >> (8 * z));
          if (o % 4 == 0) {
            uint16_t* const to = (uint16_t*)(blk + kv_value_scales(W) + (gg * 8 + tok / 4) * 16) + (tok % 2 * 2 + tok / 2 % 2);
            to[0] = sb[z];
            to[4] = mb[z];
          }
        }
      }
    }
  }
}

template <class T, bool INTER, bool CACHE>
void launch_heads_t(const HeadArgs& a, hipStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  const int half = a.rot / 2;
  const int CR = INTER ? a.rot / V : half / V, C = CR + (a.dim - a.rot) / V;
  const bool fast = (INTER ? a.rot : half) % V == 0 && (a.dim - a.rot) % V == 0 && C <= 64;
  int L = 64;
  if (fast)
    for (L = 1; L < C;) L *= 2;
  const int per = kHeadThreads / L, W = kv_groups(a.dim);
  const int kh = a.k.heads, qh = a.q.heads, H = qh + kh;
  int TP, HQ, HK, split;
  if (CACHE) {
    TP = a.n_tokens > 512 ? 4 : 1;
    const int G = qh / kh;
    const int room = max(1, 8192 / (TP * 32 * W));  // keys that 32 KB hold
    HK = min(min(kh, room), max(1, 2 * per / (TP * (G + 1))));
    HQ = HK * G;
    split = (kh + HK - 1) / HK;
  } else {
    TP = a.n_tokens > 512 ? min(8, (a.n_tokens + 1023) / 1024) : 1;
    split = a.n_tokens > 512 ? 1 : min(4096, (H + per - 1) / per);
    HQ = (qh + split - 1) / split;
    HK = (kh + split - 1) / split;
  }
  const size_t lds = (CACHE ? TP * sizeof(Spot) + (size_t)TP * HK * 32 * W * 4 : 0) + (size_t)TP * a.rot * sizeof(float);
  const dim3 grid((a.n_tokens + TP - 1) / TP, split);
  if (fast)
    hipLaunchKernelGGL((heads_kernel<T, INTER, true, CACHE>), grid, dim3(kHeadThreads), lds, stream, a, TP, L, HQ, HK);
  else
    hipLaunchKernelGGL((heads_kernel<T, INTER, false, CACHE>), grid, dim3(kHeadThreads), lds, stream, a, TP, L, HQ, HK);
}

template <bool CACHE>
void launch_heads_c(const HeadArgs& a, bool bf16, bool interleaved, hipStream_t stream) {
  if (bf16)
    interleaved ? launch_heads_t<uint16_t, true, CACHE>(a, stream) : launch_heads_t<uint16_t, false, CACHE>(a, stream);
  else
    interleaved ? launch_heads_t<float, true, CACHE>(a, stream) : launch_heads_t<float, false, CACHE>(a, stream);
}

HeadSide side(const void* x, const long long* st, int heads, const void* w, void* out) {
  return HeadSide{x, out, w, heads ? st[0] : 0, heads ? st[1] : 0, heads ? st[2] : 0, heads};
}

}  // namespace

int launch_heads(const void* q, const long long* q_strides, int q_heads, const void* q_weight, const void* k,
                 const long long* k_strides, int k_heads, const void* k_weight, float eps, const void* pos, bool pos64,
                 long long pos_batch, long long pos_tok, const double* turns, int n_tokens, int seq, int dim, int rot,
                 bool interleaved, float mscale, bool bf16, void* q_out, void* k_out, hipStream_t stream) {
  HeadArgs a{};
  a.q = side(q, q_strides, q_heads, q_weight, q_out);
  a.k = side(k, k_strides, k_heads, k_weight, k_out);
  a.pos = pos, a.pos64 = pos64, a.pos_batch = pos_batch, a.pos_tok = pos_tok, a.turns = turns;
  a.n_tokens = n_tokens, a.seq = seq, a.dim = dim, a.rot = rot, a.mscale = mscale, a.eps = eps;
  launch_heads_c<false>(a, bf16, interleaved, stream);
  return 0;
}

int launch_kv4_append(const void* q, const long long* q_strides, int q_heads, const void* q_weight, const void* k,
                      const long long* k_strides, const void* k_weight, const void* v, const long long* v_strides,
                      float eps, const void* pos, bool pos64, long long pos_batch, long long pos_tok,
                      const double* turns, int n_tokens, int seq, int dim, int rot, bool interleaved, float mscale,
                      bool bf16, const KvPages& kv, void* q_out, hipStream_t stream) {
  HeadArgs a{};
  a.q = side(q, q_strides, q_heads, q_weight, q_out);
  a.k = side(k, k_strides, kv.heads, k_weight, nullptr);
  a.v = side(v, v_strides, kv.heads, nullptr, nullptr);
  a.pos = pos, a.pos64 = pos64, a.pos_batch = pos_batch, a.pos_tok = pos_tok, a.turns = turns;
  a.n_tokens = n_tokens, a.seq = seq, a.dim = dim, a.rot = rot, a.mscale = mscale, a.eps = eps;
  a.kv = kv;
  launch_heads_c<true>(a, bf16, interleaved && rot > 0, stream);
  return 0;
}

}  // namespace mxa
