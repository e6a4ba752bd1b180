// paged_attention.cu -- attention of one new token per request over a paged
// key-value cache (no counterpart in the reference, which lists attention as
// in progress, README.md:12; it stands beside the prefill form).
//
// For request r, query head h and the keys j of r:
//   s_j = scale q . k_j,  o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m).
// Bound: HBM, each key and value of the cache read once for the
// Hq / Hkv query heads that share it.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <cmath>

#include "runtime.cuh"

namespace rb {
namespace paged {

constexpr int kMaxRequests = 8192;

struct Args {
  const void *q, *kc, *vc;
  const int32_t *table, *lens;
  void* out;
  float* lse;
  int64_t q_t, q_h, o_t, o_h;
  int64_t kc_b, kc_t, kc_h, vc_b, vc_t, vc_h;
  int64_t ld_table, window;
  int32_t R, Hq, Hkv, D, num_blocks, bs, max_blocks;
  float scale2, k_scale, v_scale;  // scale2 = scale * log2(e)
};

template <typename T> __device__ __forceinline__ float up(T v);
template <> __device__ __forceinline__ float up(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float up(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float up(__nv_fp8_e4m3 v) { return float(v); }
template <typename T> __device__ __forceinline__ T down(float v);
template <> __device__ __forceinline__ __nv_bfloat16 down(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half down(float v) { return __float2half_rn(v); }

// One warp per (request, query head), one key at a time.
template <typename T, typename C>
__global__ void __launch_bounds__(128) k_paged_simple(const __grid_constant__ Args a) {
  const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (w >= (int64_t)a.R * a.Hq) return;
  const int r = (int)(w / a.Hq), h = (int)(w - (int64_t)r * a.Hq);
  const int hk = h / (a.Hq / a.Hkv);
  const int64_t room = (int64_t)a.max_blocks * a.bs;
  int64_t len = a.lens[r];
  if (len < 0 || len > room) {
    atomicExch(&g_device_error, 3);
    len = len < 0 ? 0 : room;
  }
  const T* q = (const T*)a.q + r * a.q_t + h * a.q_h;
  const int n = a.D / 32;
  float x[8], o[8] = {}, m = -INFINITY, l = 0;
  for (int i = 0; i < n; ++i) x[i] = up(q[lane + 32 * i]);
  for (int64_t j = a.window > 0 && len > a.window ? len - a.window : 0; j < len; ++j) {
    const int page = (int)(j / a.bs), off = (int)(j - (int64_t)page * a.bs);
    const int id = a.table[r * a.ld_table + page];
    if (id < 0 || id >= a.num_blocks) {
      atomicExch(&g_device_error, 3);
      continue;
    }
    const C* k = (const C*)a.kc + id * a.kc_b + off * a.kc_t + hk * a.kc_h;
    const C* v = (const C*)a.vc + id * a.vc_b + off * a.vc_t + hk * a.vc_h;
    float s = 0;
    for (int i = 0; i < n; ++i) s += x[i] * up(k[lane + 32 * i]);
    for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(~0u, s, d);
    s *= a.scale2 * a.k_scale;
    const float m1 = fmaxf(m, s), base = m1 == -INFINITY ? 0.0f : m1;
    const float c = exp2f(m - base), p = exp2f(s - base);
    l = l * c + p;
    m = m1;
    for (int i = 0; i < n; ++i) o[i] = o[i] * c + p * up(v[lane + 32 * i]);
  }
  T* out = (T*)a.out + r * a.o_t + h * a.o_h;
  const float inv = l == 0.0f ? 0.0f : a.v_scale / l;
  for (int i = 0; i < n; ++i) out[lane + 32 * i] = down<T>(o[i] * inv);
  if (a.lse && lane == 0)
    a.lse[(int64_t)r * a.Hq + h] = l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}

inline bool shape_ok(int64_t R, int64_t Hq, int64_t Hkv, int64_t D) {
  return R >= 0 && R <= kMaxRequests && Hkv >= 1 && Hq >= 1 && Hq <= 65536 && Hq % Hkv == 0 &&
         (D == 64 || D == 128 || D == 256);
}

}  // namespace paged
}  // namespace rb

extern "C" size_t remora_b200_paged_attention_workspace_bytes(int64_t R, int64_t Hq, int64_t Hkv,
                                                              int64_t D) {
  return rb::paged::shape_ok(R, Hq, Hkv, D) ? 16 : 0;
}

extern "C" int remora_b200_paged_attention(
    const void* q, const void* k_cache, const void* v_cache, const int32_t* block_table,
    const int32_t* lens, void* out, float* lse, int dtype, int cache_dtype, int64_t R, int64_t Hq,
    int64_t Hkv, int64_t D, int64_t q_t, int64_t q_h, int64_t out_t, int64_t out_h,
    int64_t num_blocks, int64_t block_size, int64_t kc_block, int64_t kc_token, int64_t kc_head,
    int64_t vc_block, int64_t vc_token, int64_t vc_head, int64_t ld_table, int64_t max_blocks,
    float scale, int64_t window, float k_scale, float v_scale, void* workspace,
    size_t workspace_bytes, void* stream) {
  using namespace rb;
  using namespace rb::paged;
  clear_error();
  RB_CHECK_ARG(dtype == REMORA_B200_BF16 || dtype == REMORA_B200_F16,
               "paged_attention: dtype must be BF16 or F16");
  RB_CHECK_ARG(cache_dtype == dtype || cache_dtype == REMORA_B200_E4M3,
               "paged_attention: cache_dtype must be dtype or E4M3");
  RB_CHECK_ARG(shape_ok(R, Hq, Hkv, D),
               "paged_attention: needs R in [0, %d], Hq a multiple of Hkv and head_dim 64, 128 or "
               "256 (got R %lld, Hq %lld, Hkv %lld, head_dim %lld)",
               kMaxRequests, (long long)R, (long long)Hq, (long long)Hkv, (long long)D);
  RB_CHECK_ARG(block_size >= 1 && num_blocks >= 1 && block_size <= 0x7fffffff &&
                   num_blocks <= 0x7fffffff / block_size,
               "paged_attention: num_blocks * block_size must be in [1, 2^31)");
  RB_CHECK_ARG(max_blocks >= 1 && max_blocks <= 0x7fffffff / block_size && ld_table >= max_blocks,
               "paged_attention: max_blocks * block_size must be in [1, 2^31) and ld_table at "
               "least max_blocks");
  RB_CHECK_ARG(std::isfinite(scale), "paged_attention: scale is not finite");
  RB_CHECK_ARG(window >= 0, "paged_attention: window must not be negative");
  RB_CHECK_ARG(std::isfinite(k_scale) && k_scale > 0 && std::isfinite(v_scale) && v_scale > 0,
               "paged_attention: the cache scales must be positive and finite");
  RB_CHECK_ARG(cache_dtype == REMORA_B200_E4M3 || (k_scale == 1.0f && v_scale == 1.0f),
               "paged_attention: the scales must be 1 unless the cache is E4M3");
  if (R == 0) return REMORA_B200_OK;
  RB_CHECK_ARG(q && k_cache && v_cache && block_table && lens && out,
               "paged_attention: null pointer");
  RB_CHECK_ARG(aligned16(q) && aligned16(k_cache) && aligned16(v_cache) && aligned16(out),
               "paged_attention: q, the caches and out must be 16-byte aligned");
  const int64_t ce = cache_dtype == REMORA_B200_E4M3 ? 16 : 8;
  RB_CHECK_ARG(q_t % 8 == 0 && q_h % 8 == 0 && out_t % 8 == 0 && out_h % 8 == 0 &&
                   kc_block % ce == 0 && kc_token % ce == 0 && kc_head % ce == 0 &&
                   vc_block % ce == 0 && vc_token % ce == 0 && vc_head % ce == 0,
               "paged_attention: strides must be multiples of 16 bytes");
  const size_t need = remora_b200_paged_attention_workspace_bytes(R, Hq, Hkv, D);
  RB_CHECK_ARG(workspace && workspace_bytes >= need && aligned16(workspace),
               "paged_attention: workspace of %zu bytes, 16-byte aligned, is needed", need);
  Args a{q, k_cache, v_cache, block_table, lens, out, lse, q_t, q_h, out_t, out_h, kc_block,
         kc_token, kc_head, vc_block, vc_token, vc_head, ld_table, window, (int32_t)R, (int32_t)Hq,
         (int32_t)Hkv, (int32_t)D, (int32_t)num_blocks, (int32_t)block_size, (int32_t)max_blocks,
         scale * 1.4426950408889634f, k_scale, v_scale};
  const int grid = (int)((R * Hq + 3) / 4);
  cudaStream_t st = as_stream(stream);
  const bool f8 = cache_dtype == REMORA_B200_E4M3;
  if (dtype == REMORA_B200_BF16) {
    if (f8) k_paged_simple<__nv_bfloat16, __nv_fp8_e4m3><<<grid, 128, 0, st>>>(a);
    else k_paged_simple<__nv_bfloat16, __nv_bfloat16><<<grid, 128, 0, st>>>(a);
  } else {
    if (f8) k_paged_simple<__half, __nv_fp8_e4m3><<<grid, 128, 0, st>>>(a);
    else k_paged_simple<__half, __half><<<grid, 128, 0, st>>>(a);
  }
  RB_LAUNCH_CHECK();
  return REMORA_B200_OK;
}
