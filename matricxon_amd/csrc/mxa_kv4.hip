// Cached keys and values read back: the values that a sequence's last tokens are held as (mxa_kv4.hpp has the layout).
#include "mxa_kernels.hpp"
#include "mxa_kv4.hpp"

#pragma clang fp contract(off)

namespace mxa {
namespace {

constexpr int kReadThreads = 256;

// A thread takes eight values of a token's key and of its value: one word of the key's codes, a byte of four words of the
// value's. s * code + m is rounded once to float32 (its product is exact), then to the output's type.
template <bool BF16>
__global__ __launch_bounds__(kReadThreads) void kv4_read_kernel(KvPages kv, int n_tokens, int dim, void* k_out, void* v_out) {
  const int O = dim / 8, W = kv_groups(dim), blocks = kv.page / kKvBlock;
  const long long item = (long long)blockIdx.x * kReadThreads + threadIdx.x;
  if (item >= (long long)n_tokens * kv.heads * O) return;
  const int o = (int)(item % O);
  const long long row = item / O;
  const int h = (int)(row % kv.heads), t = (int)(row / kv.heads);
  int place;
  const int b = kv_place(kv, t, n_tokens, place);
  const long long block = b < 0 ? -1 : kv_block(kv, b, place);
  float k[8], v[8];
  if (block < 0) {
#pragma unroll
    for (int j = 0; j < 8; ++j) k[j] = v[j] = 0.0f;
  } else {
    const uint8_t* const blk = kv.pages + (block + (long long)h * blocks) * kv_block_bytes(W);
    const int tok = place % kv.page % kKvBlock, gg = o / 4;
    const uint32_t word = *(const uint32_t*)(blk + tok * 16 * W + (o % 4) * 4 * W + gg * 4);
    const uint32_t sm = *(const uint32_t*)(blk + kv_key_scales(W) + (tok * W + gg) * 4);
    const uint16_t* const vs =
        (const uint16_t*)(blk + kv_value_scales(W) + (gg * 8 + tok / 4) * 16) + (tok % 2 * 2 + tok / 2 % 2);
    const float ks = half_to_float(sm), km = half_to_float(sm >> 16), s = half_to_float(vs[0]), m = half_to_float(vs[4]);
#pragma unroll
    for (int j = 0; j < 8; ++j) k[j] = fmaf((float)(word >> (4 * j) & 15), ks, km);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int byte = blk[kv_value_codes(W) + kv_value_word(W, gg, tok / 4 % 4, o % 4 * 4 + j, tok / 16) + tok % 4];
      v[2 * j] = fmaf((float)(byte & 15), s, m);
      v[2 * j + 1] = fmaf((float)(byte >> 4), s, m);
    }
  }
  const long long at = row * dim + o * 8;
  if constexpr (BF16) {
    typedef uint16_t u16x8 __attribute__((ext_vector_type(8), aligned(2)));
    u16x8 kb, vb;
#pragma unroll
    for (int j = 0; j < 8; ++j) kb[j] = bf16_rne(k[j]), vb[j] = bf16_rne(v[j]);
    *(u16x8*)((uint16_t*)k_out + at) = kb;
    *(u16x8*)((uint16_t*)v_out + at) = vb;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) ((float*)k_out)[at + j] = k[j], ((float*)v_out)[at + j] = v[j];
  }
}

}  // namespace

int launch_kv4_read(const KvPages& kv, int n_tokens, int dim, bool bf16, void* k_out, void* v_out, hipStream_t stream) {
  const long long items = (long long)n_tokens * kv.heads * (dim / 8);
  const dim3 grid((unsigned)((items + kReadThreads - 1) / kReadThreads));
  if (bf16)
    hipLaunchKernelGGL(kv4_read_kernel<true>, grid, dim3(kReadThreads), 0, stream, kv, n_tokens, dim, k_out, v_out);
  else
    hipLaunchKernelGGL(kv4_read_kernel<false>, grid, dim3(kReadThreads), 0, stream, kv, n_tokens, dim, k_out, v_out);
  return 0;
}

}  // namespace mxa
