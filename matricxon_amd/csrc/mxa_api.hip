// extern "C" entry points of libmatricxon_amd.so (declared in include/matricxon_amd.h):
// argument checks, workspace layout, kernel dispatch, status codes.
#include <stdio.h>
#include <string.h>

#include "../../include/matricxon_amd.h"
#include "mxa_attend.hpp"
#include "mxa_kernels.hpp"

namespace {

thread_local char g_last_error[256] = "";

}  // namespace

namespace mxa {
void set_last_error(const char* text) { snprintf(g_last_error, sizeof g_last_error, "%s", text); }
}  // namespace mxa

namespace {

int check_launch() {
  const hipError_t e = hipGetLastError();
  if (e == hipSuccess) return MXA_OK;
  snprintf(g_last_error, sizeof g_last_error, "%s", hipGetErrorString(e));
  return MXA_ERR_LAUNCH;
}

bool known_type(int t) {
  return t == MXA_TYPE_Q8_0 || t == MXA_TYPE_Q4_K || t == MXA_TYPE_Q6_K || t == MXA_TYPE_IQ4_XS;
}

int block_elems(int t) { return t == MXA_TYPE_Q8_0 ? 32 : 256; }

int block_bytes(int t) {
  switch (t) {
    case MXA_TYPE_Q8_0: return 34;
    case MXA_TYPE_Q4_K: return 144;
    case MXA_TYPE_Q6_K: return 210;
    case MXA_TYPE_IQ4_XS: return 136;
    default: return 0;
  }
}

bool aligned(const void* p, uintptr_t a);

bool kv4_supported(int kv_heads, int page_size, int head_dim) {
  return kv_heads >= 1 && kv_heads <= MXA_KV4_MAX_HEADS && page_size >= mxa::kKvBlock && page_size % mxa::kKvBlock == 0 &&
         page_size <= MXA_KV4_MAX_PAGE && head_dim >= 8 && head_dim % 8 == 0 && head_dim <= MXA_KV4_MAX_DIM;
}

// The arguments of a call on the 4-bit cache; false where they do not fit together.
bool kv4_pages(mxa::KvPages& kv, void* pages, int n_pages, int kv_heads, int page_size, int head_dim,
               const int32_t* table, long long table_stride, int table_width, const int32_t* lengths,
               const int32_t* query_starts, int n_seq, int n_tokens) {
  if (!kv4_supported(kv_heads, page_size, head_dim) || pages == nullptr || table == nullptr || lengths == nullptr ||
      n_pages < 1 || table_width < 1 || (long long)table_width * page_size > MXA_KV4_MAX_PLACES || n_seq < 1 ||
      n_seq > MXA_KV4_MAX_SEQ || n_tokens < 1 || n_tokens > MXA_MAX_TOKENS || !aligned(pages, 16) ||
      !aligned(table, 4) || !aligned(lengths, 4) || !aligned(query_starts, 4) ||
      (query_starts == nullptr && n_tokens % n_seq != 0))
    return false;
  kv = mxa::KvPages{(uint8_t*)pages, table, lengths, query_starts, table_stride, n_pages, kv_heads, page_size,
                    table_width, n_seq, n_tokens / n_seq};
  return true;
}

bool needs_q8k(int t) { return t != MXA_TYPE_IQ4_XS; }

// The kernels read packed blocks as dwords and activations / workspace as 16-byte vectors.
bool aligned(const void* p, uintptr_t a) { return ((uintptr_t)p & (a - 1)) == 0; }

// Up to fmax activation rows (the crossover, read once per call) the matmul kernel quantizes x
// itself (no workspace).
bool fused_quant(int n_tokens, int fmax) { return n_tokens <= fmax; }

mxa::Act make_act(const float* x, const mxa::ActBuffers* a, int k) {
  mxa::Act act;
  act.q = a ? a->q : nullptr;
  act.d = a ? a->d : nullptr;
  act.bsums = a ? a->bsums : nullptr;
  act.x = x;
  act.k = k;
  act.nb = k / mxa::QK;
  act.xsplit = nullptr;
  act.xbf16 = 0;
  return act;
}

// Workspace parts, each 256-byte aligned: the Q8_K activations (types other than IQ4_XS, more than
// fmax rows), then the bf16 split of x (IQ4_XS, kIq4MfmaMinRows rows or more).
size_t q8k_part(bool any_q8k, int n_tokens, int k, int fmax) {
  return any_q8k && !fused_quant(n_tokens, fmax) ? mxa::align256(mxa::act_bytes(n_tokens, k)) : 0;
}
size_t split_part(bool any_iq4, int n_tokens, int k) {
  return any_iq4 && n_tokens >= mxa::kIq4MfmaMinRows ? mxa::iq4_prefill_workspace(n_tokens, k) : 0;
}


// Workspace parts of a call on bfloat16 x, each 256-byte aligned: the Q8_K activations (any
// K-quant / Q8_0 weight: x is quantized into them whenever the floor-shaped decode kernel, which
// reads bfloat16 x itself, does not take the call), then x widened to float32 (any IQ4_XS weight,
// which multiplies float activations), then the IQ4_XS prefill split.
size_t widen_part(bool any_iq4, int n_tokens, int k) {
  return any_iq4 ? mxa::align256((size_t)n_tokens * k * 4) : 0;
}

int gemm_multi_core(int n, const int* types, const void* const* ws, const int* outs,
                    const void* x, bool xbf16, mxa::YOut y, int n_tokens, int in_features,
                    void* workspace, size_t workspace_bytes, hipStream_t s) {
  if (n < 1 || n > 4 || types == nullptr || ws == nullptr || outs == nullptr)
    return MXA_ERR_UNSUPPORTED;
  if (x == nullptr || (y.v & ~(uintptr_t)1) == 0 || n_tokens <= 0 || !aligned(x, 16) ||
      !aligned(workspace, 16))
    return MXA_ERR_UNSUPPORTED;
  bool any_q8k = false, any_iq4 = false;
  long long total = 0;
  for (int i = 0; i < n; ++i) {
    if (!mxa_supports(types[i], in_features) || ws[i] == nullptr || outs[i] <= 0 ||
        !aligned(ws[i], 4))
      return MXA_ERR_UNSUPPORTED;
    any_q8k |= needs_q8k(types[i]);
    any_iq4 |= !needs_q8k(types[i]);
    total += outs[i];
  }
  const int fmax = mxa::fused_max_rows();
  const size_t q8k_bytes = xbf16 ? (any_q8k ? mxa::align256(mxa::act_bytes(n_tokens, in_features)) : 0)
                                 : q8k_part(any_q8k, n_tokens, in_features, fmax);
  const size_t widen_bytes = xbf16 ? widen_part(any_iq4, n_tokens, in_features) : 0;
  const size_t split_bytes = split_part(any_iq4, n_tokens, in_features);
  const size_t need = q8k_bytes + widen_bytes + split_bytes;
  mxa::DecodeSeg seg[4];
  long long c0 = 0;
  for (int i = 0; i < n; ++i) {
    seg[i] = mxa::DecodeSeg{types[i], (const uint8_t*)ws[i],
                            (long long)mxa_row_bytes(types[i], in_features), y.at(c0), outs[i]};
    c0 += outs[i];
  }
  if (xbf16 && !any_iq4 && n_tokens <= fmax) {
    // the floor-shaped decode kernel reads bfloat16 x and quantizes it itself (one launch, no
    // workspace); a launcher that declines has launched nothing
    mxa::Act a = make_act((const float*)x, nullptr, in_features);
    a.xbf16 = 1;
    const int st = n == 1 ? mxa::launch_gemv_wave_m(types[0], seg[0].w, seg[0].row_bytes, a, y,
                                                    total, n_tokens, outs[0], s)
                 : n_tokens == 1 ? mxa::launch_gemv_wave_multi(seg, n, a, s)
                                 : -1;
    if (st == 0) return check_launch();
  }
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) return MXA_ERR_WORKSPACE;
  const float* xf = xbf16 ? nullptr : (const float*)x;
  if (widen_bytes > 0) {
    float* wide = (float*)((uint8_t*)workspace + q8k_bytes);
    mxa::launch_widen_bf16((const uint16_t*)x, wide, (long long)n_tokens * in_features, s);
    xf = wide;
  }
  mxa::ActBuffers buf{};
  const mxa::ActBuffers* abuf = nullptr;
  if (q8k_bytes > 0) {
    buf = mxa::act_layout(workspace, n_tokens, in_features);
    abuf = &buf;
    if (xbf16)
      mxa::launch_quantize_q8k_bf16((const uint16_t*)x, buf, n_tokens, in_features, s);
    else
      mxa::launch_quantize_q8k(xf, buf, n_tokens, in_features, s);
  }
  const int qst = check_launch();
  if (qst != MXA_OK) return qst;
  mxa::Act act = make_act(xf, abuf, in_features);
  if (split_bytes > 0) act.xsplit = (uint8_t*)workspace + q8k_bytes + widen_bytes;
  if (n > 1 && !any_iq4 && n_tokens <= 16) {  // decode: one launch for all weights
    int st = -1;
    if (n_tokens <= fmax) {
      st = mxa::launch_decode_multi(seg, n, act, total, n_tokens, s);
    } else {
      st = mxa::launch_bwave_multi(seg, n, act, total, n_tokens, s);
      if (st != 0) st = mxa::launch_bres_multi(seg, n, act, total, n_tokens, s);
      if (st != 0) st = mxa::launch_bstream_multi(seg, n, act, total, n_tokens, s);
    }
    if (st == 0) return check_launch();
  }
  for (int i = 0; i < n; ++i) {
    if (mxa::launch_matmul(types[i], seg[i].w, seg[i].row_bytes, act, seg[i].y, total, n_tokens,
                           outs[i], s) != 0)
      return MXA_ERR_UNSUPPORTED;
    const int st = check_launch();
    if (st != MXA_OK) return st;
  }
  return MXA_OK;
}

int gemm_q8k_core(int ggml_type, const void* w, const float* x, mxa::YOut y, int n_tokens,
                  int out_features, int in_features, const void* workspace,
                  size_t workspace_bytes, hipStream_t s) {
  if (!mxa_supports(ggml_type, in_features) || w == nullptr || n_tokens <= 0 ||
      out_features <= 0 || !aligned(w, 4) || !aligned(x, 16) || !aligned(workspace, 16))
    return MXA_ERR_UNSUPPORTED;
  mxa::ActBuffers buf{};
  const mxa::ActBuffers* abuf = nullptr;
  if (needs_q8k(ggml_type)) {
    if (workspace == nullptr || workspace_bytes < mxa::act_bytes(n_tokens, in_features))
      return MXA_ERR_WORKSPACE;
    buf = mxa::act_layout((void*)workspace, n_tokens, in_features);
    abuf = &buf;
  } else if (x == nullptr) {
    return MXA_ERR_UNSUPPORTED;
  }
  const mxa::Act act = make_act(x, abuf, in_features);
  const long long rb = (long long)mxa_row_bytes(ggml_type, in_features);
  if (mxa::launch_matmul(ggml_type, (const uint8_t*)w, rb, act, y, out_features, n_tokens,
                         out_features, s) != 0)
    return MXA_ERR_UNSUPPORTED;
  return check_launch();
}

int gemm_multi_q8k_core(int n, const int* types, const void* const* ws, const int* outs,
                        mxa::YOut y, int n_tokens, int in_features, const void* workspace,
                        size_t workspace_bytes, hipStream_t s) {
  if (n < 1 || n > 4 || types == nullptr || ws == nullptr || outs == nullptr || n_tokens <= 0 ||
      !aligned(workspace, 16))
    return MXA_ERR_UNSUPPORTED;
  long long total = 0;
  for (int i = 0; i < n; ++i) {
    if (!mxa_supports(types[i], in_features) || !needs_q8k(types[i]) || ws[i] == nullptr ||
        outs[i] <= 0 || !aligned(ws[i], 4))
      return MXA_ERR_UNSUPPORTED;
    total += outs[i];
  }
  if (workspace == nullptr || workspace_bytes < mxa::act_bytes(n_tokens, in_features))
    return MXA_ERR_WORKSPACE;
  const mxa::ActBuffers buf = mxa::act_layout((void*)workspace, n_tokens, in_features);
  const mxa::Act act = make_act(nullptr, &buf, in_features);
  mxa::DecodeSeg seg[4];
  long long c0 = 0;
  for (int i = 0; i < n; ++i) {
    seg[i] = mxa::DecodeSeg{types[i], (const uint8_t*)ws[i],
                            (long long)mxa_row_bytes(types[i], in_features), y.at(c0), outs[i]};
    c0 += outs[i];
  }
  if (n > 1 && n_tokens <= 16) {  // one launch for the group
    const int fmax = mxa::fused_max_rows();
    int st = n_tokens <= fmax ? mxa::launch_decode_multi(seg, n, act, total, n_tokens, s)
                              : mxa::launch_bwave_multi(seg, n, act, total, n_tokens, s);
    if (st != 0 && n_tokens > fmax) st = mxa::launch_bres_multi(seg, n, act, total, n_tokens, s);
    if (st != 0 && n_tokens > fmax)
      st = mxa::launch_bstream_multi(seg, n, act, total, n_tokens, s);
    if (st == 0) return check_launch();
  }
  for (int i = 0; i < n; ++i) {
    if (mxa::launch_matmul(types[i], seg[i].w, seg[i].row_bytes, act, seg[i].y, total, n_tokens,
                           outs[i], s) != 0)
      return MXA_ERR_UNSUPPORTED;
    const int st = check_launch();
    if (st != MXA_OK) return st;
  }
  return MXA_OK;
}

}  // namespace

extern "C" {

const char* mxa_build_info(void) {
  return "matricxon_amd gfx950: bit-exact dequant (Q8_0/Q4_K/Q6_K/IQ4_XS); decode M<=3: "
         "LDS-DMA wave GEMV with in-kernel Q8_K quantization; M 4..16: int8 MFMA gather kernel, "
         "each wave streaming its own block columns; prefill: int8 MFMA tiles (Q4_K/Q6_K/Q8_0), "
         "bf16 split MFMA (IQ4_XS)";
}

int mxa_supports(int ggml_type, int in_features) {
  return known_type(ggml_type) && in_features > 0 && in_features % mxa::QK == 0;
}

int mxa_supports_dequant_rows(int ggml_type, int row_width) {
  return mxa_supports(ggml_type, row_width);
}

void mxa_set_fused_max_tokens(int n_tokens) { mxa::set_fused_max_rows(n_tokens); }

int mxa_fused_max_tokens(void) { return mxa::fused_max_rows(); }

size_t mxa_row_bytes(int ggml_type, int in_features) {
  if (!mxa_supports(ggml_type, in_features)) return 0;
  return (size_t)(in_features / block_elems(ggml_type)) * block_bytes(ggml_type);
}

size_t mxa_workspace_bytes(int ggml_type, int n_tokens, int in_features) {
  if (!mxa_supports(ggml_type, in_features) || n_tokens <= 0) return 0;
  if (needs_q8k(ggml_type))
    return q8k_part(true, n_tokens, in_features, mxa::fused_max_rows());
  return split_part(true, n_tokens, in_features);
}

size_t mxa_workspace_bytes_bf16(int ggml_type, int n_tokens, int in_features) {
  if (!mxa_supports(ggml_type, in_features) || n_tokens <= 0) return 0;
  if (needs_q8k(ggml_type)) return mxa::align256(mxa::act_bytes(n_tokens, in_features));
  return widen_part(true, n_tokens, in_features) + split_part(true, n_tokens, in_features);
}

int mxa_quantize_q8_k_bf16(const void* x, int n_tokens, int in_features, void* workspace,
                           size_t workspace_bytes, void* stream) {
  if (x == nullptr || n_tokens <= 0 || in_features <= 0 || in_features % mxa::QK != 0 ||
      !aligned(x, 16) || !aligned(workspace, 16))
    return MXA_ERR_UNSUPPORTED;
  if (workspace == nullptr || workspace_bytes < mxa::act_bytes(n_tokens, in_features))
    return MXA_ERR_WORKSPACE;
  const mxa::ActBuffers a = mxa::act_layout(workspace, n_tokens, in_features);
  mxa::launch_quantize_q8k_bf16((const uint16_t*)x, a, n_tokens, in_features, (hipStream_t)stream);
  return check_launch();
}

int mxa_quantize_q8_k(const float* x, int n_tokens, int in_features, void* workspace,
                      size_t workspace_bytes, void* stream) {
  if (x == nullptr || n_tokens <= 0 || in_features <= 0 || in_features % mxa::QK != 0 ||
      !aligned(x, 16) || !aligned(workspace, 16))
    return MXA_ERR_UNSUPPORTED;
  if (workspace == nullptr || workspace_bytes < mxa::act_bytes(n_tokens, in_features))
    return MXA_ERR_WORKSPACE;
  const mxa::ActBuffers a = mxa::act_layout(workspace, n_tokens, in_features);
  mxa::launch_quantize_q8k(x, a, n_tokens, in_features, (hipStream_t)stream);
  return check_launch();
}

int mxa_gemm(int ggml_type, const void* w, const float* x, float* y, int n_tokens,
             int out_features, int in_features, void* workspace, size_t workspace_bytes,
             void* stream) {
  const int outs[1] = {out_features};
  const int types[1] = {ggml_type};
  const void* ws[1] = {w};
  return gemm_multi_core(1, types, ws, outs, x, false, mxa::YOut::f32(y), n_tokens, in_features,
                         workspace, workspace_bytes, (hipStream_t)stream);
}

int mxa_gemm_bf16(int ggml_type, const void* w, const void* x, void* y, int n_tokens,
                  int out_features, int in_features, void* workspace, size_t workspace_bytes,
                  void* stream) {
  if (!aligned(y, 2)) return MXA_ERR_UNSUPPORTED;
  const int outs[1] = {out_features};
  const int types[1] = {ggml_type};
  const void* ws[1] = {w};
  return gemm_multi_core(1, types, ws, outs, x, true, mxa::YOut::bf16(y), n_tokens, in_features,
                         workspace, workspace_bytes, (hipStream_t)stream);
}

int mxa_gemv_f32(int ggml_type, const void* w, const float* x, float* y, int n_tokens,
                 int out_features, int in_features, void* stream) {
  if (!mxa_supports(ggml_type, in_features) || w == nullptr || x == nullptr || y == nullptr ||
      n_tokens <= 0 || out_features <= 0 || !aligned(w, 4) || !aligned(x, 16))
    return MXA_ERR_UNSUPPORTED;
  const long long rb = (long long)mxa_row_bytes(ggml_type, in_features);
  const mxa::YOut yo = mxa::YOut::f32(y);
  for (int m0 = 0; m0 < n_tokens; m0 += 4) {  // activation rows m0 .. m0 + 3
    const int rows = n_tokens - m0 < 4 ? n_tokens - m0 : 4;
    if (mxa::launch_gemv_f32(ggml_type, (const uint8_t*)w, rb, x + (size_t)m0 * in_features,
                             in_features, yo.at((long long)m0 * out_features), out_features, rows,
                             out_features, (hipStream_t)stream) != 0)
      return MXA_ERR_UNSUPPORTED;
  }
  return check_launch();
}

int mxa_gemm_q8k(int ggml_type, const void* w, const float* x, float* y, int n_tokens,
                 int out_features, int in_features, const void* workspace,
                 size_t workspace_bytes, void* stream) {
  if (y == nullptr) return MXA_ERR_UNSUPPORTED;
  return gemm_q8k_core(ggml_type, w, x, mxa::YOut::f32(y), n_tokens, out_features, in_features,
                       workspace, workspace_bytes, (hipStream_t)stream);
}

int mxa_gemm_q8k_bf16(int ggml_type, const void* w, void* y, int n_tokens, int out_features,
                      int in_features, const void* workspace, size_t workspace_bytes,
                      void* stream) {
  if (y == nullptr || !aligned(y, 2) || !needs_q8k(ggml_type)) return MXA_ERR_UNSUPPORTED;
  return gemm_q8k_core(ggml_type, w, nullptr, mxa::YOut::bf16(y), n_tokens, out_features,
                       in_features, workspace, workspace_bytes, (hipStream_t)stream);
}

namespace {

int gemm_moe_core(int ggml_type, const void* w, long long expert_stride, int n_experts,
                  const float* x, const int32_t* offsets, int n_rows, int max_rows_per_expert,
                  mxa::YOut y, int out_features, int in_features, void* workspace,
                  size_t workspace_bytes, void* stream) {
  if (!mxa_supports(ggml_type, in_features) || w == nullptr || offsets == nullptr ||
      (y.v & ~(uintptr_t)1) == 0 || n_experts < 1 || n_rows < 1 || out_features < 1 ||
      max_rows_per_expert < 1 || !aligned(w, 4) || !aligned(x, 16) || !aligned(workspace, 16))
    return MXA_ERR_UNSUPPORTED;
  // every expert's weight starts as aligned as mxa_gemm asks of its w
  const long long rb = (long long)mxa_row_bytes(ggml_type, in_features);
  if (expert_stride < (long long)out_features * rb || expert_stride % 4 != 0)
    return MXA_ERR_UNSUPPORTED;
  if (!needs_q8k(ggml_type)) {  // IQ4_XS: float activations, no workspace
    if (x == nullptr) return MXA_ERR_UNSUPPORTED;
    const mxa::Act act = make_act(x, nullptr, in_features);
    if (mxa::launch_moe_lpb(ggml_type, (const uint8_t*)w, rb, expert_stride, n_experts, act,
                            offsets, n_rows, min(max_rows_per_expert, n_rows), y,
                            out_features, out_features, (hipStream_t)stream) != 0)
      return MXA_ERR_UNSUPPORTED;
    return check_launch();
  }
  if (workspace == nullptr || workspace_bytes < mxa::act_bytes(n_rows, in_features))
    return MXA_ERR_WORKSPACE;
  const mxa::ActBuffers buf = mxa::act_layout(workspace, n_rows, in_features);
  const hipStream_t s = (hipStream_t)stream;
  if (x != nullptr) mxa::launch_quantize_q8k(x, buf, n_rows, in_features, s);
  const mxa::Act act = make_act(x, &buf, in_features);
  if (mxa::launch_moe_dec(ggml_type, (const uint8_t*)w, rb, expert_stride, n_experts, act,
                          offsets, n_rows, min(max_rows_per_expert, n_rows), y,
                          out_features, out_features, s) != 0)
    return MXA_ERR_UNSUPPORTED;
  return check_launch();
}

}  // namespace

int mxa_gemm_moe(int ggml_type, const void* w, long long expert_stride, int n_experts,
                 const float* x, const int32_t* offsets, int n_rows, int max_rows_per_expert,
                 float* y, int out_features, int in_features, void* workspace,
                 size_t workspace_bytes, void* stream) {
  if (y == nullptr) return MXA_ERR_UNSUPPORTED;
  return gemm_moe_core(ggml_type, w, expert_stride, n_experts, x, offsets, n_rows,
                       max_rows_per_expert, mxa::YOut::f32(y), out_features, in_features,
                       workspace, workspace_bytes, stream);
}

int mxa_gemm_moe_bf16(int ggml_type, const void* w, long long expert_stride, int n_experts,
                      const float* x, const int32_t* offsets, int n_rows, int max_rows_per_expert,
                      void* y, int out_features, int in_features, void* workspace,
                      size_t workspace_bytes, void* stream) {
  if (y == nullptr || !aligned(y, 2)) return MXA_ERR_UNSUPPORTED;
  return gemm_moe_core(ggml_type, w, expert_stride, n_experts, x, offsets, n_rows,
                       max_rows_per_expert, mxa::YOut::bf16(y), out_features, in_features,
                       workspace, workspace_bytes, stream);
}

int mxa_gemm_moe_pairs(int ggml_type, const void* w, long long expert_stride, int n_experts,
                       const int32_t* ids, int n_pairs, const float* x, int x_rows, float* y,
                       int out_features, int in_features, void* workspace, size_t workspace_bytes,
                       void* stream) {
  if (!mxa_supports(ggml_type, in_features) || !needs_q8k(ggml_type) || w == nullptr ||
      ids == nullptr || y == nullptr || n_experts < 1 || n_pairs < 1 || out_features < 1 ||
      (x_rows != 1 && x_rows != n_pairs) || !aligned(x, 16) || !aligned(workspace, 16))
    return MXA_ERR_UNSUPPORTED;
  const long long rb = (long long)mxa_row_bytes(ggml_type, in_features);
  if (expert_stride < (long long)out_features * rb) return MXA_ERR_UNSUPPORTED;
  const hipStream_t s = (hipStream_t)stream;
  const int x_step = x_rows == 1 ? 0 : 1;
  const mxa::YOut yo = mxa::YOut::f32(y);
  if (x != nullptr) {  // x quantized in the kernel where it can be
    const mxa::Act act = make_act(x, nullptr, in_features);
    if (mxa::launch_gemv_wave_pairs(ggml_type, (const uint8_t*)w, rb, expert_stride, ids,
                                    n_experts, n_pairs, x_step, act, yo, out_features, s) == 0)
      return check_launch();
  }
  if (workspace == nullptr || workspace_bytes < mxa::act_bytes(x_rows, in_features))
    return x == nullptr ? MXA_ERR_WORKSPACE : MXA_ERR_UNSUPPORTED;
  const mxa::ActBuffers buf = mxa::act_layout(workspace, x_rows, in_features);
  const mxa::Act act = make_act(nullptr, &buf, in_features);
  // x quantized into the workspace first (the workspace is the caller's scratch: on a shape the
  // kernel does not take, only it has been written)
  if (x != nullptr) mxa::launch_quantize_q8k(x, buf, x_rows, in_features, s);
  if (mxa::launch_gemv_wave_pairs(ggml_type, (const uint8_t*)w, rb, expert_stride, ids, n_experts,
                                  n_pairs, x_step, act, yo, out_features, s) != 0)
    return MXA_ERR_UNSUPPORTED;
  return check_launch();
}

int mxa_gemm_moe_pairs_bf16(int ggml_type, const void* w, long long expert_stride, int n_experts,
                            const int32_t* ids, int n_pairs, const void* x, int x_rows, void* y,
                            int out_features, int in_features, void* workspace,
                            size_t workspace_bytes, void* stream) {
  if (!mxa_supports(ggml_type, in_features) || !needs_q8k(ggml_type) || w == nullptr ||
      ids == nullptr || y == nullptr || n_experts < 1 || n_pairs < 1 || out_features < 1 ||
      (x_rows != 1 && x_rows != n_pairs) || !aligned(x, 16) || !aligned(y, 2) ||
      !aligned(workspace, 16))
    return MXA_ERR_UNSUPPORTED;
  const long long rb = (long long)mxa_row_bytes(ggml_type, in_features);
  if (expert_stride < (long long)out_features * rb) return MXA_ERR_UNSUPPORTED;
  const hipStream_t s = (hipStream_t)stream;
  const int x_step = x_rows == 1 ? 0 : 1;
  const mxa::YOut yo = mxa::YOut::bf16(y);
  if (x != nullptr) {  // bfloat16 x read and quantized in the kernel where it can be
    mxa::Act act = make_act((const float*)x, nullptr, in_features);
    act.xbf16 = 1;
    if (mxa::launch_gemv_wave_pairs(ggml_type, (const uint8_t*)w, rb, expert_stride, ids,
                                    n_experts, n_pairs, x_step, act, yo, out_features, s) == 0)
      return check_launch();
  }
  if (workspace == nullptr || workspace_bytes < mxa::act_bytes(x_rows, in_features))
    return x == nullptr ? MXA_ERR_WORKSPACE : MXA_ERR_UNSUPPORTED;
  const mxa::ActBuffers buf = mxa::act_layout(workspace, x_rows, in_features);
  const mxa::Act act = make_act(nullptr, &buf, in_features);
  if (x != nullptr) mxa::launch_quantize_q8k_bf16((const uint16_t*)x, buf, x_rows, in_features, s);
  if (mxa::launch_gemv_wave_pairs(ggml_type, (const uint8_t*)w, rb, expert_stride, ids, n_experts,
                                  n_pairs, x_step, act, yo, out_features, s) != 0)
    return MXA_ERR_UNSUPPORTED;
  return check_launch();
}

int mxa_moe_route(const void* ids, int ids_int64, int n_tokens, int top_k, int n_experts,
                  int32_t* offsets, int32_t* pair_tok, int32_t* rows, int32_t* ids32,
                  void* stream) {
  if (mxa::launch_moe_route(ids, ids_int64 != 0, n_tokens, top_k, n_experts, false, offsets, pair_tok,
                            rows, ids32, (hipStream_t)stream) != 0)
    return MXA_ERR_UNSUPPORTED;
  return check_launch();
}

int mxa_moe_route_masked(const void* ids, int ids_int64, int n_tokens, int top_k, int n_experts, int32_t* offsets,
                         int32_t* pair_tok, int32_t* rows, int32_t* ids32, void* stream) {
  if (mxa::launch_moe_route(ids, ids_int64 != 0, n_tokens, top_k, n_experts, true, offsets, pair_tok,
                            rows, ids32, (hipStream_t)stream) != 0)
    return MXA_ERR_UNSUPPORTED;
  return check_launch();
}

int mxa_moe_combine(const float* down, const int32_t* rows, const int32_t* ids,
                    const float* weights, int n_tokens, int top_k, int n_embd, int round_bf16,
                    float* out, void* stream) {
  if (down == nullptr || ids == nullptr || weights == nullptr || out == nullptr)
    return MXA_ERR_UNSUPPORTED;
  if (mxa::launch_moe_combine(down, rows, ids, weights, n_tokens, top_k, n_embd, round_bf16 != 0, 0,
                              mxa::YOut::f32(out), (hipStream_t)stream) != 0)
    return MXA_ERR_UNSUPPORTED;
  return check_launch();
}

int mxa_moe_combine_masked(const float* down, const int32_t* rows, const int32_t* ids, const float* weights,
                           int n_tokens, int top_k, int n_embd, int round_bf16, float* out, void* stream) {
  if (down == nullptr || ids == nullptr || weights == nullptr || out == nullptr)
    return MXA_ERR_UNSUPPORTED;
  if (mxa::launch_moe_combine(down, rows, ids, weights, n_tokens, top_k, n_embd, round_bf16 != 0, 1,
                              mxa::YOut::f32(out), (hipStream_t)stream) != 0)
    return MXA_ERR_UNSUPPORTED;
  return check_launch();
}

int mxa_moe_topk(const void* logits, int logits_bf16, int n_tokens, int n_experts, int top_k, int norm_topk,
                 float scale, int32_t* ids, float* weights, void* stream) {
  if (logits == nullptr || ids == nullptr || weights == nullptr || n_tokens > MXA_MAX_TOKENS ||
      !aligned(logits, logits_bf16 ? 2 : 4) || !aligned(ids, 4) || !aligned(weights, 4))
    return MXA_ERR_UNSUPPORTED;
  if (mxa::launch_moe_topk(logits, logits_bf16 != 0, n_tokens, n_experts, top_k, norm_topk != 0, scale, ids, weights,
                           (hipStream_t)stream) != 0)
    return MXA_ERR_UNSUPPORTED;
  return check_launch();
}

size_t mxa_moe_layer_workspace_bytes(int gate_type, int down_type, int n_experts, int top_k, int n_tokens, int n_embd,
                                     int ffn_len, int bf16) {
  if (!mxa::moe_layer_supported(gate_type, down_type, n_experts, top_k, n_tokens, n_embd, ffn_len)) return 0;
  return mxa::moe_layer_workspace(n_tokens, top_k, n_embd, ffn_len, bf16 != 0);
}

int mxa_moe_layer(int gate_type, int down_type, const void* gate, const void* up, long long gate_stride,
                  const void* down, long long down_stride, int n_experts, const void* x, int bf16, const void* logits,
                  int logits_bf16, int top_k, int norm_topk, float scale, int n_tokens, int n_embd, int ffn_len,
                  int reciprocal, int32_t* ids, float* weights, void* out, int out_bf16, void* workspace,
                  size_t workspace_bytes, void* stream) {
  const size_t need =
      mxa_moe_layer_workspace_bytes(gate_type, down_type, n_experts, top_k, n_tokens, n_embd, ffn_len, bf16);
  if (need == 0 || gate == nullptr || up == nullptr || down == nullptr || x == nullptr || logits == nullptr ||
      ids == nullptr || weights == nullptr || out == nullptr || !aligned(gate, 16) || !aligned(up, 16) ||
      !aligned(down, 16) || !aligned(x, 16) || !aligned(logits, logits_bf16 ? 2 : 4) || !aligned(ids, 4) ||
      !aligned(weights, 4) || !aligned(out, out_bf16 ? 2 : 4) || !aligned(workspace, 16))
    return MXA_ERR_UNSUPPORTED;
  const long long gate_row = (long long)mxa_row_bytes(gate_type, n_embd);
  const long long down_row = (long long)mxa_row_bytes(down_type, ffn_len);
  if (gate_stride < gate_row * ffn_len || down_stride < down_row * n_embd || gate_stride % 16 != 0 ||
      down_stride % 16 != 0)
    return MXA_ERR_UNSUPPORTED;
  if (workspace == nullptr || workspace_bytes < need) return MXA_ERR_WORKSPACE;
  if (mxa::launch_moe_layer(gate_type, down_type, (const uint8_t*)gate, (const uint8_t*)up, gate_stride, gate_row,
                            (const uint8_t*)down, down_stride, down_row, n_experts, x, bf16 != 0, logits,
                            logits_bf16 != 0, top_k, norm_topk != 0, scale, n_tokens, n_embd, ffn_len,
                            reciprocal != 0, ids, weights,
                            out_bf16 ? mxa::YOut::bf16(out) : mxa::YOut::f32((float*)out), workspace,
                            (hipStream_t)stream) != 0)
    return MXA_ERR_UNSUPPORTED;
  return check_launch();
}

int mxa_gemm_multi(int n, const int* types, const void* const* ws, const int* outs,
                   const float* x, float* y, int n_tokens, int in_features, void* workspace,
                   size_t workspace_bytes, void* stream) {
  return gemm_multi_core(n, types, ws, outs, x, false, mxa::YOut::f32(y), n_tokens, in_features,
                         workspace, workspace_bytes, (hipStream_t)stream);
}

int mxa_gemm_multi_bf16(int n, const int* types, const void* const* ws, const int* outs,
                        const void* x, void* y, int n_tokens, int in_features, void* workspace,
                        size_t workspace_bytes, void* stream) {
  if (!aligned(y, 2)) return MXA_ERR_UNSUPPORTED;
  return gemm_multi_core(n, types, ws, outs, x, true, mxa::YOut::bf16(y), n_tokens, in_features,
                         workspace, workspace_bytes, (hipStream_t)stream);
}

int mxa_gemm_multi_q8k(int n, const int* types, const void* const* ws, const int* outs, float* y,
                       int n_tokens, int in_features, const void* workspace,
                       size_t workspace_bytes, void* stream) {
  if (y == nullptr) return MXA_ERR_UNSUPPORTED;
  return gemm_multi_q8k_core(n, types, ws, outs, mxa::YOut::f32(y), n_tokens, in_features,
                             workspace, workspace_bytes, (hipStream_t)stream);
}

int mxa_gemm_multi_q8k_bf16(int n, const int* types, const void* const* ws, const int* outs,
                            void* y, int n_tokens, int in_features, const void* workspace,
                            size_t workspace_bytes, void* stream) {
  if (y == nullptr || !aligned(y, 2)) return MXA_ERR_UNSUPPORTED;
  return gemm_multi_q8k_core(n, types, ws, outs, mxa::YOut::bf16(y), n_tokens, in_features,
                             workspace, workspace_bytes, (hipStream_t)stream);
}

int mxa_rms_norm_q8_k(const float* x, const float* weight, float eps, int n_tokens, int dim,
                      float* out, void* workspace, size_t workspace_bytes, void* stream) {
  if (x == nullptr || weight == nullptr || n_tokens <= 0 || dim <= 0 || dim % mxa::QK != 0 ||
      !aligned(x, 16) || !aligned(weight, 4) || !aligned(out, 16) || !aligned(workspace, 16))
    return MXA_ERR_UNSUPPORTED;
  if (workspace == nullptr || workspace_bytes < mxa::act_bytes(n_tokens, dim)) return MXA_ERR_WORKSPACE;
  const mxa::ActBuffers a = mxa::act_layout(workspace, n_tokens, dim);
  mxa::launch_rms_norm_q8k(x, weight, eps, out, a, n_tokens, dim, (hipStream_t)stream);
  return check_launch();
}

int mxa_silu_mul_q8_k(const float* gate, const float* up, long long ld, int n_tokens, int dim,
                      float* out, void* workspace, size_t workspace_bytes, void* stream) {
  if (gate == nullptr || up == nullptr || n_tokens <= 0 || dim <= 0 || dim % mxa::QK != 0 ||
      ld < dim || !aligned(gate, 4) || !aligned(up, 4) || !aligned(out, 16) ||
      !aligned(workspace, 16))
    return MXA_ERR_UNSUPPORTED;
  if (workspace == nullptr || workspace_bytes < mxa::act_bytes(n_tokens, dim)) return MXA_ERR_WORKSPACE;
  const mxa::ActBuffers a = mxa::act_layout(workspace, n_tokens, dim);
  mxa::launch_silu_mul_q8k(gate, up, ld, out, a, n_tokens, dim, (hipStream_t)stream);
  return check_launch();
}

int mxa_rms_norm_q8_k_bf16(const void* x, const void* weight, float eps, int n_tokens, int dim,
                           void* out, void* workspace, size_t workspace_bytes, void* stream) {
  if (x == nullptr || weight == nullptr || n_tokens <= 0 || dim <= 0 || dim % mxa::QK != 0 ||
      !aligned(workspace, 16))
    return MXA_ERR_UNSUPPORTED;
  if (workspace == nullptr || workspace_bytes < mxa::act_bytes(n_tokens, dim)) return MXA_ERR_WORKSPACE;
  const mxa::ActBuffers a = mxa::act_layout(workspace, n_tokens, dim);
  if (mxa::launch_rms_norm_q8k_bf16((const uint16_t*)x, (const uint16_t*)weight, eps,
                                    (uint16_t*)out, a, n_tokens, dim, (hipStream_t)stream) != 0)
    return MXA_ERR_UNSUPPORTED;
  return check_launch();
}

int mxa_silu_mul_q8_k_bf16(const void* gate, const void* up, long long ld, int n_tokens, int dim,
                           void* out, void* workspace, size_t workspace_bytes, void* stream) {
  if (gate == nullptr || up == nullptr || n_tokens <= 0 || dim <= 0 || dim % mxa::QK != 0 ||
      ld < dim || !aligned(workspace, 16))
    return MXA_ERR_UNSUPPORTED;
  if (workspace == nullptr || workspace_bytes < mxa::act_bytes(n_tokens, dim)) return MXA_ERR_WORKSPACE;
  const mxa::ActBuffers a = mxa::act_layout(workspace, n_tokens, dim);
  if (mxa::launch_silu_mul_q8k_bf16((const uint16_t*)gate, (const uint16_t*)up, ld, (uint16_t*)out,
                                    a, n_tokens, dim, (hipStream_t)stream) != 0)
    return MXA_ERR_UNSUPPORTED;
  return check_launch();
}

int mxa_add_rms_norm_q8_k(const void* x, long long ldx, const void* residual, long long ldr,
                          const void* post_weight, float post_eps, const void* gate, long long ldg,
                          int gate_step, float scale, const void* weight, float eps, int n_tokens,
                          int dim, int bf16, int residual_bf16, void* hidden, void* out,
                          void* workspace, size_t workspace_bytes, void* stream) {
  const uintptr_t xa = bf16 ? 2 : 4, ra = residual_bf16 ? 2 : 4;
  if (x == nullptr || residual == nullptr || weight == nullptr || hidden == nullptr || out == nullptr ||
      n_tokens <= 0 || n_tokens > MXA_MAX_TOKENS || dim <= 0 || ldx < 0 || ldr < 0 || ldg < 0 ||
      (long long)n_tokens * dim > MXA_NORM_MAX_TOTAL ||
      (gate_step != 0 && gate_step != 1) ||
      (residual_bf16 && !bf16) || !aligned(x, xa) || !aligned(weight, xa) || !aligned(post_weight, xa) ||
      !aligned(gate, xa) || !aligned(out, xa) || !aligned(residual, ra) || !aligned(hidden, ra) ||
      !aligned(workspace, 16))
    return MXA_ERR_UNSUPPORTED;
  mxa::ActBuffers a{};
  if (workspace != nullptr) {
    if (dim % mxa::QK != 0) return MXA_ERR_UNSUPPORTED;
    if (workspace_bytes < mxa::act_bytes(n_tokens, dim)) return MXA_ERR_WORKSPACE;
    a = mxa::act_layout(workspace, n_tokens, dim);
  }
  if (mxa::launch_add_rms_norm(x, ldx, residual, ldr, post_weight, post_eps, gate, ldg, gate_step, scale,
                               weight, eps, bf16 != 0, residual_bf16 != 0, n_tokens, dim, hidden, out,
                               workspace != nullptr ? &a : nullptr, (hipStream_t)stream) != 0)
    return MXA_ERR_UNSUPPORTED;
  return check_launch();
}

int mxa_rope(const void* q, const long long* q_strides, int q_heads, const void* k, const long long* k_strides,
             int k_heads, const void* positions, int positions_int64, long long pos_batch, long long pos_token,
             const double* turns, int n_tokens, int seq_len, int head_dim, int rotary_dim, int interleaved,
             float scale, int bf16, void* q_out, void* k_out, void* stream) {
  const uintptr_t ea = bf16 ? 2 : 4;
  if (q == nullptr || q_strides == nullptr || q_out == nullptr || positions == nullptr || turns == nullptr ||
      q_heads < 1 || k_heads < 0 || q_heads > MXA_ROPE_MAX_HEADS || k_heads > MXA_ROPE_MAX_HEADS ||
      n_tokens < 1 || n_tokens > MXA_MAX_TOKENS || seq_len < 1 || head_dim < 2 || head_dim > MXA_ROPE_MAX_DIM ||
      head_dim % 2 != 0 ||
      rotary_dim < 2 || rotary_dim > head_dim || rotary_dim % 2 != 0 || !aligned(q, ea) || !aligned(q_out, ea) ||
      !aligned(positions, positions_int64 ? 8 : 4) || !aligned(turns, 8))
    return MXA_ERR_UNSUPPORTED;
  if (k_heads > 0 &&
      (k == nullptr || k_strides == nullptr || k_out == nullptr || !aligned(k, ea) || !aligned(k_out, ea)))
    return MXA_ERR_UNSUPPORTED;
  if (mxa::launch_rope(q, q_strides, q_heads, k, k_strides, k_heads, positions, positions_int64 != 0, pos_batch,
                       pos_token, turns, n_tokens, seq_len, head_dim, rotary_dim, interleaved != 0, scale,
                       bf16 != 0, q_out, k_out, (hipStream_t)stream) != 0)
    return MXA_ERR_UNSUPPORTED;
  return check_launch();
}

int mxa_norm_rope(const void* q, const long long* q_strides, int q_heads, const void* q_weight, const void* k,
                  const long long* k_strides, int k_heads, const void* k_weight, float eps, const void* positions,
                  int positions_int64, long long pos_batch, long long pos_token, const double* turns, int n_tokens,
                  int seq_len, int head_dim, int rotary_dim, int interleaved, float scale, int bf16, void* q_out,
                  void* k_out, void* stream) {
  const uintptr_t ea = bf16 ? 2 : 4;
  if (q == nullptr || q_strides == nullptr || q_out == nullptr || positions == nullptr || turns == nullptr ||
      q_heads < 1 || k_heads < 0 || q_heads > MXA_ROPE_MAX_HEADS || k_heads > MXA_ROPE_MAX_HEADS || n_tokens < 1 ||
      n_tokens > MXA_MAX_TOKENS || seq_len < 1 || head_dim < 2 || head_dim > MXA_ROPE_MAX_DIM || head_dim % 2 != 0 ||
      rotary_dim < 2 || rotary_dim > head_dim || rotary_dim % 2 != 0 || !aligned(q, ea) || !aligned(q_out, ea) ||
      !aligned(q_weight, ea) || !aligned(positions, positions_int64 ? 8 : 4) || !aligned(turns, 8))
    return MXA_ERR_UNSUPPORTED;
  if (k_heads > 0 && (k == nullptr || k_strides == nullptr || k_out == nullptr || !aligned(k, ea) ||
                      !aligned(k_out, ea) || !aligned(k_weight, ea)))
    return MXA_ERR_UNSUPPORTED;
  if (mxa::launch_heads(q, q_strides, q_heads, q_weight, k, k_strides, k_heads, k_weight, eps, positions,
                        positions_int64 != 0, pos_batch, pos_token, turns, n_tokens, seq_len, head_dim, rotary_dim,
                        interleaved != 0, scale, bf16 != 0, q_out, k_out, (hipStream_t)stream) != 0)
    return MXA_ERR_UNSUPPORTED;
  return check_launch();
}

size_t mxa_kv4_page_bytes(int kv_heads, int page_size, int head_dim) {
  if (!kv4_supported(kv_heads, page_size, head_dim)) return 0;
  return (size_t)kv_heads * (page_size / mxa::kKvBlock) * mxa::kv_block_bytes(mxa::kv_groups(head_dim));
}

int mxa_kv4_append(const void* q, const long long* q_strides, int q_heads, const void* q_weight, const void* k,
                   const long long* k_strides, const void* k_weight, const void* v, const long long* v_strides,
                   float eps, const void* positions, int positions_int64, long long pos_batch, long long pos_token,
                   const double* turns, int n_tokens, int seq_len, int rotary_dim, int interleaved, float scale,
                   int bf16, void* pages, int n_pages, int kv_heads, int page_size, int head_dim, const int32_t* table,
                   long long table_stride, int table_width, const int32_t* lengths, const int32_t* query_starts,
                   int n_seq, void* q_out, void* stream) {
  const uintptr_t ea = bf16 ? 2 : 4;
  mxa::KvPages kv;
  if (!kv4_pages(kv, pages, n_pages, kv_heads, page_size, head_dim, table, table_stride, table_width, lengths,
                 query_starts, n_seq, n_tokens))
    return MXA_ERR_UNSUPPORTED;
  if (k == nullptr || k_strides == nullptr || v == nullptr || v_strides == nullptr || !aligned(k, ea) ||
      !aligned(v, ea) || !aligned(k_weight, ea) || q_heads < 0 || q_heads > MXA_ROPE_MAX_HEADS ||
      q_heads % kv_heads != 0 || seq_len < 1 || rotary_dim < 0 || rotary_dim > head_dim || rotary_dim % 2 != 0 ||
      (rotary_dim > 0 && turns == nullptr) || !aligned(turns, 8) || !aligned(positions, positions_int64 ? 8 : 4))
    return MXA_ERR_UNSUPPORTED;
  if (q_heads > 0 && (q == nullptr || q_strides == nullptr || q_out == nullptr || !aligned(q, ea) ||
                      !aligned(q_out, ea) || !aligned(q_weight, ea)))
    return MXA_ERR_UNSUPPORTED;
  if (mxa::launch_kv4_append(q, q_strides, q_heads, q_weight, k, k_strides, k_weight, v, v_strides, eps, positions,
                             positions_int64 != 0, pos_batch, pos_token, turns, n_tokens, seq_len, head_dim, rotary_dim,
                             interleaved != 0, scale, bf16 != 0, kv, q_out, (hipStream_t)stream) != 0)
    return MXA_ERR_UNSUPPORTED;
  return check_launch();
}

int mxa_kv4_read(const void* pages, int n_pages, int kv_heads, int page_size, int head_dim, const int32_t* table,
                 long long table_stride, int table_width, const int32_t* lengths, const int32_t* query_starts,
                 int n_seq, int n_tokens, int bf16, void* k_out, void* v_out, void* stream) {
  const uintptr_t ea = bf16 ? 2 : 4;
  mxa::KvPages kv;
  if (!kv4_pages(kv, (void*)pages, n_pages, kv_heads, page_size, head_dim, table, table_stride, table_width, lengths,
                 query_starts, n_seq, n_tokens) ||
      k_out == nullptr || v_out == nullptr || !aligned(k_out, ea) || !aligned(v_out, ea))
    return MXA_ERR_UNSUPPORTED;
  if (mxa::launch_kv4_read(kv, n_tokens, head_dim, bf16 != 0, k_out, v_out, (hipStream_t)stream) != 0)
    return MXA_ERR_UNSUPPORTED;
  return check_launch();
}

size_t mxa_kv4_attend_workspace_bytes(int n_seq, int n_tokens, int ragged, int q_heads, int kv_heads, int head_dim,
                                      int max_length, int window) {
  if (n_seq < 1 || n_tokens < 1 || (!ragged && n_tokens % n_seq != 0) || kv_heads < 1 || q_heads < kv_heads || q_heads % kv_heads != 0 ||
      (long long)n_tokens * q_heads > MXA_KV4_MAX_ROWS || head_dim < 8 || head_dim > mxa::kKvMaxDim || max_length < 1 || window < 0)
    return 0;
  return mxa::attend_workspace(n_seq, n_tokens, ragged != 0, kv_heads, q_heads / kv_heads, max_length, window, head_dim);
}

int mxa_kv4_attend(const void* q, const long long* q_strides, int q_heads, int n_tokens, int seq_len,
                   const void* pages, int n_pages, int kv_heads, int page_size, int head_dim, const int32_t* table,
                   long long table_stride, int table_width, const int32_t* lengths, const int32_t* query_starts,
                   int n_seq, int max_length, int window, float scale, void* out, void* workspace,
                   size_t workspace_bytes, void* stream) {
  mxa::AttendArgs a{};
  if (!kv4_pages(a.kv, (void*)pages, n_pages, kv_heads, page_size, head_dim, table, table_stride, table_width, lengths,
                 query_starts, n_seq, n_tokens) ||
      q == nullptr || q_strides == nullptr || out == nullptr || !aligned(q, 2) || !aligned(out, 2) || q_heads < 1 ||
      q_heads > MXA_ROPE_MAX_HEADS || q_heads % kv_heads != 0 || (long long)n_tokens * q_heads > MXA_KV4_MAX_ROWS || seq_len < 1 ||
      max_length < 1 || window < 0)
    return MXA_ERR_UNSUPPORTED;
  if (!aligned(workspace, 16)) return MXA_ERR_UNSUPPORTED;
  a.q = (const uint16_t*)q;
  a.q_batch = q_strides[0], a.q_tok = q_strides[1], a.q_head = q_strides[2];
  a.out = (uint16_t*)out;
  a.n_tokens = n_tokens, a.seq = seq_len, a.dim = head_dim, a.heads = q_heads, a.group = q_heads / kv_heads;
  a.window = window < MXA_KV4_MAX_PLACES ? window : MXA_KV4_MAX_PLACES, a.scale = scale;
  const int status = mxa::launch_attend(a, max_length, workspace, workspace_bytes, (hipStream_t)stream);
  if (status != 0) return status == mxa::kAttendWorkspace ? MXA_ERR_WORKSPACE : MXA_ERR_UNSUPPORTED;
  return check_launch();
}

int mxa_dequantize(int ggml_type, const void* blocks, long long n_blocks, float* out,
                   void* stream) {
  if (!known_type(ggml_type) || blocks == nullptr || out == nullptr || n_blocks <= 0)
    return MXA_ERR_UNSUPPORTED;
  if (mxa::launch_dequant(ggml_type, (const uint8_t*)blocks, nullptr, nullptr, 0, 0, 1, n_blocks,
                          mxa::YOut::f32(out), (hipStream_t)stream) != 0)
    return MXA_ERR_UNSUPPORTED;
  return check_launch();
}

int mxa_dequant_rows(int ggml_type, const void* w, long long n_src_rows, const int32_t* rows,
                     int n_rows, int row_width, float* out, void* stream) {
  if (!mxa_supports(ggml_type, row_width) || w == nullptr || rows == nullptr || out == nullptr ||
      n_rows <= 0 || n_src_rows <= 0)
    return MXA_ERR_UNSUPPORTED;
  const int bpr = row_width / block_elems(ggml_type);
  const long long rb = (long long)mxa_row_bytes(ggml_type, row_width);
  if (mxa::launch_dequant(ggml_type, (const uint8_t*)w, rows, nullptr, n_src_rows, rb, bpr,
                          (long long)n_rows * bpr, mxa::YOut::f32(out), (hipStream_t)stream) != 0)
    return MXA_ERR_UNSUPPORTED;
  return check_launch();
}

int mxa_embed_rows(int ggml_type, const void* w, long long n_src_rows, const int64_t* ids, int n_ids,
                   int row_width, void* out, int out_bf16, void* stream) {
  if (!mxa_supports(ggml_type, row_width) || w == nullptr || ids == nullptr || out == nullptr ||
      n_ids <= 0 || n_src_rows <= 0 || !aligned(ids, 8) || !aligned(out, 16))
    return MXA_ERR_UNSUPPORTED;
  const int bpr = row_width / block_elems(ggml_type);
  const long long rb = (long long)mxa_row_bytes(ggml_type, row_width);
  if (mxa::launch_dequant(ggml_type, (const uint8_t*)w, nullptr, ids, n_src_rows, rb, bpr,
                          (long long)n_ids * bpr, out_bf16 ? mxa::YOut::bf16(out) : mxa::YOut::f32((float*)out),
                          (hipStream_t)stream) != 0)
    return MXA_ERR_UNSUPPORTED;
  return check_launch();
}

int mxa_gather_rows(const void* src, long long n_src_rows, long long row_bytes,
                    const int32_t* order, int n_rows, void* dst, void* stream) {
  if (src == nullptr || order == nullptr || dst == nullptr || n_src_rows <= 0 || row_bytes <= 0 ||
      n_rows <= 0 || !aligned(order, 4))
    return MXA_ERR_UNSUPPORTED;
  mxa::launch_gather_rows(src, n_src_rows, row_bytes, order, n_rows, dst, (hipStream_t)stream);
  return check_launch();
}

int mxa_stream_read(const void* src, long long bytes, void* sink, void* stream) {
  if (src == nullptr || sink == nullptr || bytes <= 0 || bytes % 16 != 0 || !aligned(src, 16) ||
      !aligned(sink, 4))
    return MXA_ERR_UNSUPPORTED;
  mxa::launch_stream_read(src, bytes, (uint32_t*)sink, (hipStream_t)stream);
  return check_launch();
}

const char* mxa_last_error(void) { return g_last_error; }

}  // extern "C"
