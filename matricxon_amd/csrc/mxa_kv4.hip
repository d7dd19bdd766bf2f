// Cached keys and values read back: the values that a sequence's last tokens are held as (mxa_kv4.hpp has the layout).
#include <algorithm>

#include "mxa_kernels.hpp"
#include "mxa_kv4.hpp"

#pragma clang fp contract(off)

namespace mxa {
namespace {

constexpr int kReadThreads = 256, kReadTokens = 4;

// A workgroup takes `tokens` tokens, a thread eight values of one's key and of its value: one word of the key's codes, a
// byte of four words of the value's. s * code + m is rounded once to float32 (its product is exact), then to the output's
// type. 4096 tokens of 8 heads of 128 take 8 us; one token a workgroup fills the CUs up to some thousand.
template <class T>
__global__ __launch_bounds__(kReadThreads) void kv4_read_kernel(KvPages kv, int n_tokens, int dim, int tokens, T* k_out,
                                                                T* v_out) {
  __shared__ Spot spots[kReadTokens];
  const int O = dim / 8, W = kv_groups(dim), tid = threadIdx.x;
  const int tok0 = (int)blockIdx.x * tokens, nt = min(tokens, n_tokens - tok0);
  if (tid < nt) spots[tid] = kv_spot(kv, tok0 + tid, n_tokens, W);
  __syncthreads();
  const uint32_t head_bytes = (uint32_t)(kv.page / kKvBlock * kv_block_bytes(W));
  const long long first = (long long)tok0 * kv.heads * dim;
  const int items = nt * kv.heads * O, stride = kReadThreads * (int)gridDim.y;  // heads * O: up to 2^17
  for (int item = (int)blockIdx.y * kReadThreads + tid; item < items; item += stride) {
    const int row = (int)((uint32_t)item / (uint32_t)O), o = item - row * O;
    const int t = (row >= kv.heads) + (row >= 2 * kv.heads) + (row >= 3 * kv.heads), h = row - t * kv.heads;
    const Spot spot = spots[t];
    float k[8]{}, v[8]{};
    if (spot.at >= 0) {
      const uint8_t* const blk = kv.pages + spot.at + (uint64_t)(uint32_t)h * head_bytes;
      const int tok = spot.place & (kKvBlock - 1), gg = o / 4;
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
    typedef typename Vec<T, 8>::type V8;
    *(V8*)(k_out + first + row * dim + o * 8) = narrow_all<T, 8>(k);
    *(V8*)(v_out + first + row * dim + o * 8) = narrow_all<T, 8>(v);
  }
}

}  // namespace

int launch_kv4_read(const KvPages& kv, int n_tokens, int dim, bool bf16, void* k_out, void* v_out, hipStream_t stream) {
  const int tokens = n_tokens > 1024 ? kReadTokens : 1, items = tokens * kv.heads * (dim / 8);
  const dim3 grid((n_tokens + tokens - 1) / tokens, std::min((items + kReadThreads - 1) / kReadThreads, 64));
  if (bf16)
    hipLaunchKernelGGL(kv4_read_kernel<uint16_t>, grid, dim3(kReadThreads), 0, stream, kv, n_tokens, dim, tokens,
                       (uint16_t*)k_out, (uint16_t*)v_out);
  else
    hipLaunchKernelGGL(kv4_read_kernel<float>, grid, dim3(kReadThreads), 0, stream, kv, n_tokens, dim, tokens,
                       (float*)k_out, (float*)v_out);
  return 0;
}

}  // namespace mxa
