// Attention of the newest tokens over a paged key-value cache.
#include <math_constants.h>

#include "paged.cuh"

namespace syn {

constexpr int PAGED_WARPS = 4;

template <typename T>
__device__ __forceinline__ float load16(const T* p);
template <>
__device__ __forceinline__ float load16(const __half* p) { return __half2float(*p); }
template <>
__device__ __forceinline__ float load16(const __nv_bfloat16* p) { return __bfloat162float(*p); }
template <>
__device__ __forceinline__ float load16(const __nv_fp8_e4m3* p) { return static_cast<float>(*p); }

// One block per new token and query head; its warps take the keys in turn and join at the end.
template <typename T, typename C, int D>
__global__ void __launch_bounds__(PAGED_WARPS * 32) paged_attn_kernel(syn_paged_attn_args p) {
  constexpr int N = D / 32;
  __shared__ float s_m[PAGED_WARPS], s_l[PAGED_WARPS], s_o[PAGED_WARPS][D];
  const int t = blockIdx.x, h = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int z = t, first_row = t, rows = 1;
  if (p.starts != nullptr) {
    int a = 0, b = p.requests;  // the last request that starts at or before the token and has rows
    while (b - a > 1) {
      const int m = (a + b) >> 1;
      (p.starts[m] <= t ? a : b) = m;
    }
    z = a;
    first_row = p.starts[z];
    rows = p.starts[z + 1] - first_row;
    if (t < first_row || t >= first_row + rows) return;
  }
  const int64_t room = static_cast<int64_t>(p.width) * p.page_size;
  int len = p.lens[z];
  if (len < 0) {
    if (threadIdx.x == 0) paged_record(p.status, SYN_DEV_BAD_INDEX, z, len);
    len = 0;
  }
  if (len > room) len = static_cast<int>(min(room + 1, static_cast<int64_t>(INT_MAX)));
  const int pos = len - rows + (t - first_row);
  const int hi = p.causal ? min(len, pos + 1) : len;
  const int lo = p.window > 0 ? max(0, pos - p.window + 1) : 0;
  const int kh = h / (p.Hq / p.Hkv);
  const float ks = p.k_scale ? p.k_scale[kh] : 1.f, vs = p.v_scale ? p.v_scale[kh] : 1.f;
  const float mult = p.sm_scale * CUDART_L2E_F * ks;
  float q[N], o[N] = {}, m = -CUDART_INF_F, l = 0.f;
  const T* qp = static_cast<const T*>(p.q) + t * p.q_strides[0] + h * p.q_strides[1];
  for (int i = 0; i < N; ++i) q[i] = load16(qp + i * 32 + lane);
  for (int j = lo + warp; j < hi; j += PAGED_WARPS) {
    const int page = j / p.page_size < p.width ? p.table[z * p.table_stride + j / p.page_size] : -1;
    const bool ok = static_cast<unsigned>(page) < static_cast<unsigned>(p.num_pages);
    if (!ok && lane == 0) paged_record(p.status, SYN_DEV_BAD_INDEX, z, page);
    const int64_t at = ok ? page * p.cache_strides[0] + j % p.page_size * p.cache_strides[1] + kh * p.cache_strides[2] : 0;
    float s = 0.f;
    for (int i = 0; i < N; ++i) s += q[i] * load16(static_cast<const C*>(p.k_cache) + at + i * 32 + lane);
    for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(~0u, s, d);
    s = ok ? s * mult : CUDART_NAN_F;
    const float top = fmaxf(m, s), base = top == -CUDART_INF_F ? 0.f : top;
    const float a = exp2f(m - base), w = exp2f(s - base);
    l = l * a + w;
    for (int i = 0; i < N; ++i) o[i] = o[i] * a + w * load16(static_cast<const C*>(p.v_cache) + at + i * 32 + lane);
    m = top;
  }
  if (lane == 0) s_m[warp] = m, s_l[warp] = l;
  for (int i = 0; i < N; ++i) s_o[warp][i * 32 + lane] = o[i];
  __syncthreads();
  float top = -CUDART_INF_F, total = 0.f;
  for (int w = 0; w < PAGED_WARPS; ++w) top = fmaxf(top, s_m[w]);
  const float base = top == -CUDART_INF_F ? 0.f : top;
  for (int w = 0; w < PAGED_WARPS; ++w) total += s_l[w] * exp2f(s_m[w] - base);
  T* op = static_cast<T*>(p.o) + t * p.o_strides[0] + h * p.o_strides[1];
  for (int d = threadIdx.x; d < D; d += PAGED_WARPS * 32) {
    float x = 0.f;
    for (int w = 0; w < PAGED_WARPS; ++w) x += s_o[w][d] * exp2f(s_m[w] - base);
    op[d] = static_cast<T>(total == 0.f ? 0.f : x / total * vs);
  }
  if (threadIdx.x == 0 && p.lse != nullptr) p.lse[static_cast<int64_t>(t) * p.Hq + h] = top + log2f(total);
}

template <typename T, typename C>
static int launch_paged(const syn_paged_attn_args& a, cudaStream_t stream) {
  const dim3 grid(a.tokens, a.Hq);
  if (a.D == 64) paged_attn_kernel<T, C, 64><<<grid, PAGED_WARPS * 32, 0, stream>>>(a);
  else if (a.D == 128) paged_attn_kernel<T, C, 128><<<grid, PAGED_WARPS * 32, 0, stream>>>(a);
  else paged_attn_kernel<T, C, 256><<<grid, PAGED_WARPS * 32, 0, stream>>>(a);
  SYN_CUDA_TRY(cudaGetLastError());
  return SYN_OK;
}

int preload_paged_attn_kernels() { return SYN_OK; }

}  // namespace syn

extern "C" int64_t syn_paged_attention_workspace(int num_sms) { return num_sms < 0 ? SYN_ERR_INVALID : 0; }

extern "C" int syn_paged_attention(const syn_paged_attn_args* a, void* stream) {
  using namespace syn;
  if (a == nullptr || a->tokens < 0 || a->requests <= 0 || a->Hq <= 0 || a->Hkv <= 0 || a->Hq % a->Hkv != 0 ||
      a->page_size <= 0 || a->num_pages <= 0 || a->width <= 0 || a->window < 0 || (a->window > 0 && !a->causal) ||
      a->num_sms < 0)
    return SYN_ERR_INVALID;
  if (a->starts == nullptr && a->tokens != a->requests) return SYN_ERR_INVALID;
  if (a->D != 64 && a->D != 128 && a->D != 256) return SYN_ERR_UNSUPPORTED;
  if (a->dtype != SYN_DTYPE_F16 && a->dtype != SYN_DTYPE_BF16) return SYN_ERR_UNSUPPORTED;
  if (a->cache_dtype != SYN_CACHE_SAME && a->cache_dtype != SYN_CACHE_E4M3) return SYN_ERR_UNSUPPORTED;
  if (static_cast<int64_t>(a->num_pages) * a->page_size > INT_MAX) return SYN_ERR_TOO_LARGE;
  if (a->tokens == 0) return SYN_OK;
  syn_paged_attn_args p = *a;
  const bool e4m3 = a->cache_dtype == SYN_CACHE_E4M3;
  if (a->q == nullptr || a->k_cache == nullptr || a->v_cache == nullptr || a->table == nullptr || a->lens == nullptr ||
      a->o == nullptr || a->table_stride < a->width)
    return SYN_ERR_INVALID;
  if (e4m3 ? (a->k_scale == nullptr || a->v_scale == nullptr) : (a->k_scale != nullptr || a->v_scale != nullptr))
    return SYN_ERR_INVALID;
  if (!paged_aligned(a->q) || !paged_aligned(a->k_cache) || !paged_aligned(a->v_cache) || !paged_aligned(a->o) ||
      !paged_aligned(a->workspace) || !paged_strides(p.q_strides, {a->tokens, a->Hq}, 2) ||
      !paged_strides(p.o_strides, {a->tokens, a->Hq}, 2) ||
      !paged_strides(p.cache_strides, {a->num_pages, a->page_size, a->Hkv}, e4m3 ? 1 : 2))
    return SYN_ERR_INVALID;
  PagedDevice device(a->device);
  SYN_CUDA_TRY(device.error());
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a->dtype == SYN_DTYPE_BF16) {
    return e4m3 ? launch_paged<__nv_bfloat16, __nv_fp8_e4m3>(p, s) : launch_paged<__nv_bfloat16, __nv_bfloat16>(p, s);
  }
  return e4m3 ? launch_paged<__half, __nv_fp8_e4m3>(p, s) : launch_paged<__half, __half>(p, s);
}
