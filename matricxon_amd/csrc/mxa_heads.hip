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
//
// Memory bounds the form without a cache (4096 tokens of 32 + 8 heads of 128, bfloat16: 84 MB in 16 us of a stream of calls,
// 5.2 TB/s), the vector units the one with a cache (a launch of 28 us, 3.1 TB/s; a division a code and 32-bit indexes took
// 34), and what waits for what both on few tokens (3.6 us and 6.8).
#include "mxa_heads_grid.hpp"
#include "mxa_kernels.hpp"
#include "mxa_kv4.hpp"

#pragma clang fp contract(off)

namespace mxa {
namespace {

constexpr int kHeadBatch = 3;  // rows of a lane that are requested together (2: 3 to 6% slower)

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
// any), two to a byte's value, and the group's scale and minimum, which come back as bits of float16. A NaN is held as 0
// and an infinity as the largest: a cached value is always finite.
//
// Quotients by s share its reciprocal, brought to the last bit by a Newton step; a product with it is put right by its
// residual, which is exact (Markstein's division).
__device__ __forceinline__ void quantize8(float (&x)[8], bool here, float (&bytes)[4], uint16_t& s_bits, uint16_t& m_bits) {
  float lo = INFINITY, hi = -INFINITY;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    x[j] = __builtin_amdgcn_fmed3f(x[j] == x[j] ? x[j] : 0.0f, -kKvHeld, kKvHeld);
    lo = fminf(lo, x[j]);
    hi = fmaxf(hi, x[j]);
  }
  lo = quad_min(here ? lo : INFINITY);
  hi = quad_max(here ? hi : -INFINITY);
  const _Float16 mh = (_Float16)lo, sh = (_Float16)((hi - lo) / 15.0f);
  const float m = (float)mh, s = (float)sh;
  float y = __builtin_amdgcn_rcpf(s);
  y = fmaf(fmaf(-s, y, 1.0f), y, y);
  if (!here || !(s > 0.0f)) y = 0.0f;
  float c[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float d = x[j] - m, q = d * y;
    c[j] = here ? __builtin_amdgcn_fmed3f(rintf(fmaf(fmaf(-q, s, d), y, q)), 0.0f, 15.0f) : 0.0f;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) bytes[j] = fmaf(c[2 * j + 1], 16.0f, c[2 * j]);
  s_bits = __builtin_bit_cast(uint16_t, sh);
  m_bits = __builtin_bit_cast(uint16_t, mh);
}

// Products for indexes below 2^23: one of 32 bits costs four of these.
__device__ __forceinline__ int mul24(int a, int b) { return __mul24(a, b); }
__device__ __forceinline__ long long mul64(int a, long long b) { return (long long)((uint64_t)(uint32_t)a * (uint64_t)b); }

// T the element type; FAST: vectors of V values. A workgroup takes TP tokens and, from grid.y, HQ heads of q and HK of k, one
// head at least (heads_grid).
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
  const auto from = [&](const HeadSide& s, int t, int h) {  // t: of the workgroup
    if (one) return (const T*)s.x + tok0 * s.tok + mul64(t, s.tok) + mul64(h, s.head);
    const int b = (tok0 + t) / a.seq;
    return (const T*)s.x + mul64(b, s.batch) + mul64(tok0 + t - b * a.seq, s.tok) + mul64(h, s.head);
  };

  const int per = kHeadThreads / L, c = tid % L;
  const int CR = FAST ? (INTER ? a.rot / V : half / V) : 0, C = FAST ? CR + (a.dim - a.rot) / V : 0;
  const bool turned = c < CR;
  const int at = turned ? c * V : a.rot + (c - CR) * V;  // the lane's vector in a head, and its partner's at half + at
  const bool paired = !INTER && turned;

  // A thread's rows, `per` apart: (token, head of the workgroup's), stepped on without a division each.
  struct Row {
    int t, hh, h;
    bool live, isq;
  };
  const int step_t = per / H, step_h = per - step_t * H;
  const auto row_at = [&](int t, int hh) {
    Row w;
    w.live = t < nt;
    w.t = w.live ? t : 0;
    w.hh = w.live ? hh : 0;
    w.isq = w.hh < nq;
    w.h = w.isq ? q0 + w.hh : k0 + w.hh - nq;
    return w;
  };
  const auto step = [&](int& t, int& hh) {
    t += step_t, hh += step_h;
    if (hh >= H) hh -= H, ++t;
  };
  int now_t = tid / L / H, now_h = tid / L - now_t * H;
  // The rows of a batch, and a quad's values, are requested before what depends on the page table and the positions.
  Piece x[kHeadBatch], y[kHeadBatch];
  const auto load_rows = [&] {
    int t = now_t, hh = now_h;
#pragma unroll
    for (int j = 0; j < kHeadBatch; ++j) {
      const Row w = row_at(t, hh);
      if (w.live && c < C) {
        const T* const src = from(w.isq ? a.q : a.k, w.t, w.h) + at;
        x[j].v = *(const Vv*)src;
        if (paired) y[j].v = *(const Vv*)(src + half);
      }
      step(t, hh);
    }
  };
  // The workgroup's four tokens' values of a head's group go to sixteen lanes: lane % 4 the octet, lane / 4 % 4 the token.
  const int vlanes = 16 * W * nk, over_w = 65536 / W + 1;  // x * over_w >> 16 is x / W, for x up to some thousands
  struct Place {
    bool live, here;
    int h, gg, t, o;
  };
  const auto value_of = [&](int item) {
    Place v;
    v.live = item < vlanes;
    const int in = v.live ? item : 0;
    v.h = mul24(in >> 4, over_w) >> 16;
    v.gg = (in >> 4) - mul24(v.h, W);
    v.t = in >> 2 & 3;
    v.o = 4 * v.gg + (in & 3);
    v.here = v.live && v.t < nt && v.o * 8 < a.dim;
    return v;
  };
  typedef typename Vec<T, 8>::type V8;
  V8 first_values{};
  Piece qw, qw2, kw, kw2;  // a lane's norm weights are the same for all of its rows
  if constexpr (FAST) {
    load_rows();
    if (c < C && a.q.w != nullptr) {
      qw.v = *(const Vv*)((const T*)a.q.w + at);
      if (paired) qw2.v = *(const Vv*)((const T*)a.q.w + half + at);
    }
    if (c < C && a.k.w != nullptr) {
      kw.v = *(const Vv*)((const T*)a.k.w + at);
      if (paired) kw2.v = *(const Vv*)((const T*)a.k.w + half + at);
    }
  }
  const double first_turn = tid < nt * half ? a.turns[tid % half] : 0.0;
  if constexpr (CACHE) {
    const Place v = value_of(tid);
    if (v.here) first_values = *(const V8*)(from(a.v, v.t, k0 + v.h) + v.o * 8);
    for (int t = tid; t < nt; t += kHeadThreads) spots[t] = kv_spot(a.kv, tok0 + t, a.n_tokens, W);
    __syncthreads();
  }
  for (int i = tid; i < nt * half; i += kHeadThreads) {
    const int t = i / half, tt = tok0 + t, b = one ? 0 : tt / a.seq;
    double p;
    if (CACHE && a.pos == nullptr) {
      p = (double)spots[t].place;
    } else {
      const long long from_ = b * a.pos_batch + (tt - b * a.seq) * a.pos_tok;
      p = a.pos64 ? (double)((const long long*)a.pos)[from_] : (double)((const int32_t*)a.pos)[from_];
    }
    const double turns = p * (i == tid ? first_turn : a.turns[i - t * half]);
    float s, co;
    sincospif(2.0f * (float)(turns - rint(turns)), &s, &co);
    cs[i] = a.mscale * co;
    sn[i] = a.mscale * s;
  }
  __syncthreads();

  const bool normed = a.q.w != nullptr || a.k.w != nullptr;
  for (int base = 0; base < rows; base += kHeadBatch * per) {  // the same count for every thread: lanes exchange sums
    if constexpr (FAST) {
      if (base > 0) load_rows();
    }
#pragma unroll
    for (int j = 0; j < kHeadBatch; ++j) {
      if (base + j * per >= rows) break;
      const Row r = row_at(now_t, now_h);
      step(now_t, now_h);
      const HeadSide& s = r.isq ? a.q : a.k;
      T* const dst = (T*)s.out + (long long)tok0 * s.heads * a.dim + mul24(mul24(r.t, s.heads) + r.h, a.dim);
      float* const key = CACHE && !r.isq ? keys + (r.t * HK + r.hh - nq) * 32 * W : nullptr;
      const T* const w = (const T*)s.w;
      const bool none = CACHE && spots[r.t].seq < 0;  // its q comes back as zeros
      if constexpr (FAST) {
        const bool mine = r.live && c < C;
        float xf[V], yf[V];
        float ss = 0.0f;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          xf[i] = mine ? widen(x[j].e[i]) : 0.0f;
          yf[i] = mine && paired ? widen(y[j].e[i]) : 0.0f;
          ss += xf[i] * xf[i] + yf[i] * yf[i];
        }
        if (normed) ss = lanes_sum(ss, L);
        if (mine) {
          if (w != nullptr) {
            const float rn = 1.0f / sqrtf(ss / (float)a.dim + a.eps);
            const Piece wx = r.isq ? qw : kw, wy = r.isq ? qw2 : kw2;
#pragma unroll
            for (int i = 0; i < V; ++i) {
              xf[i] = xf[i] * rn * widen(wx.e[i]);
              if (paired) yf[i] = yf[i] * rn * widen(wy.e[i]);
            }
          }
          if (turned) {
            const float* const co = cs + r.t * half + (INTER ? c * (V / 2) : c * V);
            const float* const si = sn + r.t * half + (INTER ? c * (V / 2) : c * V);
            if constexpr (INTER) {
#pragma unroll
              for (int i = 0; i < V / 2; ++i) {
                const float u = xf[2 * i], v = xf[2 * i + 1];
                xf[2 * i] = fmaf(u, co[i], -(v * si[i]));
                xf[2 * i + 1] = fmaf(u, si[i], v * co[i]);
              }
            } else {
#pragma unroll
              for (int i = 0; i < V; ++i) {
                const float u = xf[i], v = yf[i];
                xf[i] = fmaf(u, co[i], -(v * si[i]));
                yf[i] = fmaf(u, si[i], v * co[i]);
              }
            }
          }
          if (key != nullptr) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
              key[at + i] = xf[i];
              if (paired) key[half + at + i] = yf[i];
            }
          } else {
            *(Vv*)(dst + at) = none ? Vv{} : narrow_all<T, V>(xf);
            if (paired) *(Vv*)(dst + half + at) = none ? Vv{} : narrow_all<T, V>(yf);
          }
        }
      } else {
        const T* const src = from(s, r.t, r.h);
        float ss = 0.0f;
        if (r.live && w != nullptr)
          for (int i = c; i < a.dim; i += L) {
            const float v = widen(src[i]);
            ss += v * v;
          }
        if (normed) ss = lanes_sum(ss, L);
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
        if (r.live) {
          for (int i = c; i < half; i += L) {
            const int iu = INTER ? 2 * i : i, iv = INTER ? 2 * i + 1 : half + i;
            const float co = cs[r.t * half + i], si = sn[r.t * half + i], u = get(iu), v = get(iv);
            put(iu, fmaf(u, co, -(v * si)));
            put(iv, fmaf(u, si, v * co));
          }
          for (int i = a.rot + c; i < a.dim; i += L) put(i, get(i));
        }
      }
    }
  }

  if constexpr (CACHE) {
    const int O = 4 * W;
    const uint32_t head_bytes = (uint32_t)(a.kv.page / kKvBlock * kv_block_bytes(W));
    for (int base = 0; base < vlanes; base += kHeadThreads) {  // whole rows of sixteen lanes
      const Place p = value_of(base + tid);
      V8 v = first_values;
      if (base > 0 && p.here) v = *(const V8*)(from(a.v, p.t, k0 + p.h) + p.o * 8);
      float f[8];
      float codes[4];
      uint16_t sb, mb;
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = p.here ? widen(v[j]) : 0.0f;
      quantize8(f, p.here, codes, sb, mb);
      const int z = tid >> 2 & 3, t = min(p.t, nt - 1);
      const Spot spot = spots[t];
      const bool cached = p.live && p.t < nt && spot.at >= 0;
      uint8_t* const blk = a.kv.pages + spot.at + (uint64_t)(uint32_t)(k0 + p.h) * head_bytes;
      const int tok = spot.place & (kKvBlock - 1), oct = p.o & 3;
      // four neighbouring tokens of one block: whole words, of which lane z stores the z-th
      const Spot head = spots[0];
      const bool in_row = cached && spot.at == head.at && spot.place == head.place + z && head.place % 4 == 0;
      const bool whole = (__ballot(in_row) >> (tid & 48) & 0xFFFF) == 0xFFFF;
      uint32_t word = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (!whole && cached)
          blk[kv_value_codes(W) + kv_value_word(W, p.gg, tok >> 2 & 3, oct * 4 + j, tok >> 4) + (tok & 3)] = (uint8_t)codes[j];
        uint32_t w = __builtin_amdgcn_cvt_pk_u8_f32(codes[j], z, 0);
        w |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w, 0x128, 0xF, 0xF, false);  // row_ror:8, then 4: over z
        w |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w, 0x124, 0xF, 0xF, false);
        if (j == z) word = w;
      }
      if (whole)
        *(uint32_t*)(blk + kv_value_codes(W) + kv_value_word(W, p.gg, tok >> 2 & 3, oct * 4 + z, tok >> 4)) = word;
      if (cached && oct == 0) {
        uint16_t* const quad = (uint16_t*)(blk + kv_value_scales(W) + (p.gg * 8 + (tok >> 2)) * 16);
        uint16_t* const to = quad + ((tok & 1) * 2 + (tok >> 1 & 1));
        to[0] = sb;
        to[4] = mb;
      }
    }
    __syncthreads();
    for (int base = 0; base < nt * nk * O; base += kHeadThreads) {  // quads of lanes share a group: O is whole quads
      const int item = base + tid;
      const bool live = item < nt * nk * O;
      const int rw = live ? item >> 2 : 0, row = mul24(rw, over_w) >> 16, o = live ? item - mul24(row, O) : 0;
      const int t = (row >= nk) + (row >= 2 * nk) + (row >= 3 * nk), h = row - mul24(t, nk);
      const bool here = live && o * 8 < a.dim;
      float f[8];
      float codes[4];
      uint16_t sb, mb;
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = here ? keys[mul24(mul24(t, HK) + h, 32 * W) + o * 8 + j] : 0.0f;
      quantize8(f, here, codes, sb, mb);
      if (!live || spots[t].at < 0) continue;
      uint32_t word = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) word = __builtin_amdgcn_cvt_pk_u8_f32(codes[j], j, word);
      uint8_t* const blk = a.kv.pages + spots[t].at + (uint64_t)(uint32_t)(k0 + h) * head_bytes;
      const int tok = spots[t].place & (kKvBlock - 1);
      *(uint32_t*)(blk + tok * 16 * W + (o % 4) * 4 * W + (o / 4) * 4) = word;
      if (o % 4 == 0) *(uint32_t*)(blk + kv_key_scales(W) + (tok * W + o / 4) * 4) = sb | (uint32_t)mb << 16;
    }
  }
}

template <class T, bool INTER, bool CACHE>
void launch_heads_t(const HeadArgs& a, hipStream_t stream) {
  const HeadGrid g = heads_grid(CACHE, sizeof(T), INTER, a.q.heads, a.k.heads, a.n_tokens, a.dim, a.rot);
  const size_t keys = CACHE ? g.TP * sizeof(Spot) + (size_t)g.TP * g.HK * 32 * kv_groups(a.dim) * 4 : 0;
  const size_t lds = keys + (size_t)g.TP * a.rot * sizeof(float);
  const dim3 grid((a.n_tokens + g.TP - 1) / g.TP, g.split);
  if (g.fast)
    hipLaunchKernelGGL((heads_kernel<T, INTER, true, CACHE>), grid, dim3(kHeadThreads), lds, stream, a, g.TP, g.L, g.HQ, g.HK);
  else
    hipLaunchKernelGGL((heads_kernel<T, INTER, false, CACHE>), grid, dim3(kHeadThreads), lds, stream, a, g.TP, g.L, g.HQ, g.HK);
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
