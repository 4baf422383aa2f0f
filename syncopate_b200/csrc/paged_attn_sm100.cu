// Host side of the paged attention (see paged_attn_sm100.cuh).
#include "paged_attn_sm100.cuh"

#include <atomic>

namespace syn {

template <typename C>
constexpr int64_t paged_worker_bytes() {
  return PA_DESC * 4 + 2 * (C::ROWS * 2 + C::ROWS * C::D) * 4;
}

// Enough for every variant of head dimension D.
static int64_t paged_workspace(int sms, int D) {
  using T = __half;
  auto most = [](int64_t a, int64_t b, int64_t c) { return a > b ? (a > c ? a : c) : b > c ? b : c; };
  auto size = [](auto cfg) {
    using C = decltype(cfg);
    return C::BLOCKS * PA_WARPS * paged_worker_bytes<C>();
  };
  const int64_t bytes = D == 256   ? most(size(PagedCfg<T, false, 256, 1>()), size(PagedCfg<T, false, 256, 2>()), 0)
                        : D == 128 ? most(size(PagedCfg<T, false, 128, 1>()), size(PagedCfg<T, false, 128, 2>()), size(PagedCfg<T, false, 128, 4>()))
                                   : most(size(PagedCfg<T, false, 64, 1>()), size(PagedCfg<T, false, 64, 2>()), size(PagedCfg<T, false, 64, 4>()));
  return sms * bytes;
}

// Opts the kernel into its shared memory, once a device.
template <typename C>
static int configure_paged() {
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  SYN_CUDA_TRY(cudaGetDevice(&dev));
  const uint64_t bit = 1ull << (dev & 63);
  if (dev < 64 && (done.load(std::memory_order_relaxed) & bit)) return SYN_OK;
  SYN_CUDA_TRY(cudaFuncSetAttribute(paged_attn_kernel<C>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
  cudaFuncAttributes attr;
  SYN_CUDA_TRY(cudaFuncGetAttributes(&attr, paged_join_kernel<C>));
  done.fetch_or(bit, std::memory_order_relaxed);
  return SYN_OK;
}

template <typename C>
static int launch_paged(const syn_paged_attn_args& a, int sms, cudaStream_t stream) {
  // The variants for 8-bit caches have the blocks and units of those that paged_workspace counts.
  using Counted = PagedCfg<__half, false, C::D, C::RT>;
  static_assert(C::BLOCKS == Counted::BLOCKS && paged_worker_bytes<C>() == paged_worker_bytes<Counted>(), "workspace");
  int rc = configure_paged<C>();
  if (rc != SYN_OK) return rc;
  PagedAttnParams p;
  p.a = a;
  p.grid = sms * C::BLOCKS;
  const int warps = p.grid * PA_WARPS;
  // 700 keys of 8 heads: 12.8 us with two steps a worker at least, 13.6 with one (more parts to join), 14.3 with four.
  p.min_steps = 2;
  // Neighbouring heads side by side until 256 bytes are read in a row: 8-bit keys of 128 dimensions 248 us -> 218, of 64
  // dimensions 101 -> 72, 16-bit ones of 64 dimensions 123 -> 109.  Where a head's keys lie together (pages of [heads,
  // slots]) it would change nothing but the number of parts.
  p.tracks = 1;
  if (a.cache_strides[2] * (C::E4M3 ? 1 : 2) == C::ROWB)
    while (p.tracks * C::ROWB < 256 && a.Hkv % (2 * p.tracks) == 0) p.tracks *= 2;
  // mulhi(n, 2^(31 + b) / d rounded up) >> (b - 1) = n / d for 0 <= n < 2^31, 2^(b - 1) < d <= 2^b
  p.page_mul = 0, p.page_shift = 0;
  if (a.page_size > 1) {
    int b = 1;
    while ((1ll << b) < a.page_size) ++b;
    p.page_mul = static_cast<uint32_t>(((1ull << (31 + b)) + a.page_size - 1) / a.page_size);
    p.page_shift = b - 1;
  }
  p.desc = static_cast<int32_t*>(a.workspace);
  p.part_ml = reinterpret_cast<float*>(p.desc + warps * PA_DESC);
  p.part_o = p.part_ml + static_cast<int64_t>(2) * warps * C::ROWS * 2;
  paged_attn_kernel<C><<<p.grid, PA_THREADS, C::SMEM, stream>>>(p);
  SYN_CUDA_TRY(cudaGetLastError());
  // The join's blocks are brought in while the last shares are still at work and wait for them there.
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config = {};
  const PagedJoinGrid<C> join(warps);
  config.gridDim = dim3(join.few + join.many);
  config.blockDim = dim3(PA_JOIN_WARPS * 32);
  config.stream = stream;
  config.attrs = &attr;
  config.numAttrs = 1;
  SYN_CUDA_TRY(cudaLaunchKernelEx(&config, paged_join_kernel<C>, p));
  return SYN_OK;
}

template <typename T, bool E4M3>
static int launch_paged(const syn_paged_attn_args& a, int sms, cudaStream_t stream) {
  // Units hold the rows that requests bring a head on average, in eights (at most 32, 16 where D = 256, which
  // is what the output takes of the registers).  Larger units would read keys and values once for more rows, but pay
  // for rows that are not there: 16 rows a head in units of 32, 200 us against 117 in units of 16.  The host knows
  // the sizes of q and table alone, so rows behind the last request and requests without rows count too: 64 requests
  // with one token each in a q of 512 rows, 181 us against 117 (8-bit cache 228 against 97).  Who calls chooses those.
  const int64_t rows = static_cast<int64_t>(a.tokens) * (a.Hq / a.Hkv);
  const int rt = rows <= 8 * static_cast<int64_t>(a.requests) ? 1 : rows <= 16 * static_cast<int64_t>(a.requests) ? 2 : 4;
  if (a.D == 256) {
    return rt == 1 ? launch_paged<PagedCfg<T, E4M3, 256, 1>>(a, sms, stream) : launch_paged<PagedCfg<T, E4M3, 256, 2>>(a, sms, stream);
  }
  if (a.D == 128) {
    return rt == 1   ? launch_paged<PagedCfg<T, E4M3, 128, 1>>(a, sms, stream)
           : rt == 2 ? launch_paged<PagedCfg<T, E4M3, 128, 2>>(a, sms, stream)
                     : launch_paged<PagedCfg<T, E4M3, 128, 4>>(a, sms, stream);
  }
  return rt == 1   ? launch_paged<PagedCfg<T, E4M3, 64, 1>>(a, sms, stream)
         : rt == 2 ? launch_paged<PagedCfg<T, E4M3, 64, 2>>(a, sms, stream)
                   : launch_paged<PagedCfg<T, E4M3, 64, 4>>(a, sms, stream);
}

template <typename T, bool E4M3>
static int preload_paged() {
  int rc = configure_paged<PagedCfg<T, E4M3, 64, 1>>();
  if (rc == SYN_OK) rc = configure_paged<PagedCfg<T, E4M3, 64, 2>>();
  if (rc == SYN_OK) rc = configure_paged<PagedCfg<T, E4M3, 64, 4>>();
  if (rc == SYN_OK) rc = configure_paged<PagedCfg<T, E4M3, 128, 1>>();
  if (rc == SYN_OK) rc = configure_paged<PagedCfg<T, E4M3, 128, 2>>();
  if (rc == SYN_OK) rc = configure_paged<PagedCfg<T, E4M3, 128, 4>>();
  if (rc == SYN_OK) rc = configure_paged<PagedCfg<T, E4M3, 256, 1>>();
  if (rc == SYN_OK) rc = configure_paged<PagedCfg<T, E4M3, 256, 2>>();
  return rc;
}

int preload_paged_attn_kernels() {
  int rc = preload_paged<__half, false>();
  if (rc == SYN_OK) rc = preload_paged<__half, true>();
  if (rc == SYN_OK) rc = preload_paged<__nv_bfloat16, false>();
  if (rc == SYN_OK) rc = preload_paged<__nv_bfloat16, true>();
  return rc;
}

}  // namespace syn

extern "C" int64_t syn_paged_attention_workspace(int num_sms, int D) {
  if (num_sms <= 0) return SYN_ERR_INVALID;
  if (D != 64 && D != 128 && D != 256) return SYN_ERR_UNSUPPORTED;
  return syn::paged_workspace(num_sms, D);
}

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
  if (a->tokens > INT_MAX / 2 / (a->Hq / a->Hkv)) return SYN_ERR_TOO_LARGE;  // rows of a head
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
  // So that positions less the window stay numbers of 32 bits.
  if (p.window > INT_MAX - 64 - a->tokens) p.window = INT_MAX - 64 - a->tokens;
  // So that numbers of keys do: what lies behind counts as behind the table.
  if (p.width > (INT_MAX - 64) / a->page_size) p.width = (INT_MAX - 64) / a->page_size;
  int sms = 0;
  const int rc = device_sm_count(&sms);
  if (rc != SYN_OK) return rc;
  if (a->num_sms > 0 && a->num_sms < sms) sms = a->num_sms;
  if (a->workspace == nullptr || a->workspace_bytes < paged_workspace(sms, a->D)) return SYN_ERR_INVALID;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a->dtype == SYN_DTYPE_BF16) {
    return e4m3 ? launch_paged<__nv_bfloat16, true>(p, sms, s) : launch_paged<__nv_bfloat16, false>(p, sms, s);
  }
  return e4m3 ? launch_paged<__half, true>(p, sms, s) : launch_paged<__half, false>(p, sms, s);
}
