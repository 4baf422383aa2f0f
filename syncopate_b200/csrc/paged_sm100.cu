// Step plan and append of the paged key-value cache (see include/syncopate_b200.h for what they
// compute).
#include "paged.cuh"

namespace syn {

constexpr int PLAN_THREADS = 1024;

struct PlanSums {
  long long given, want, more;  // pages pushed, pages popped, tokens appended
};

__device__ __forceinline__ PlanSums operator+(PlanSums a, PlanSums b) {
  return {a.given + b.given, a.want + b.want, a.more + b.more};
}
__device__ __forceinline__ PlanSums shfl_up(PlanSums a, int d) {
  return {__shfl_up_sync(~0u, a.given, d), __shfl_up_sync(~0u, a.want, d), __shfl_up_sync(~0u, a.more, d)};
}

// One block: running sums over the requests give every request its place on the stack of free pages
// and its first token; then pages are pushed, popped and the tokens' slots written.
__global__ void __launch_bounds__(PLAN_THREADS) page_plan_kernel(syn_page_plan_args p) {
  extern __shared__ int32_t plan_smem[];
  int32_t* s_lens = plan_smem;                  // [requests]
  int32_t* s_given = s_lens + p.requests;       // pages pushed before the request; -1: the request goes on
  int32_t* s_want = s_given + p.requests;       // pages popped before it
  int32_t* s_start = s_want + p.requests;       // [requests + 1]
  __shared__ PlanSums warp_sums[32];
  __shared__ int s_bad;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) s_bad = INT_MAX;
  __syncthreads();

  const int per = (p.requests + PLAN_THREADS - 1) / PLAN_THREADS;
  const int z0 = min(tid * per, p.requests), z1 = min(z0 + per, p.requests);
  const long long room = static_cast<long long>(p.width) * p.page_size;
  auto sums_of = [&](int len, int add) {
    const int held = (static_cast<long long>(len) + p.page_size - 1) / p.page_size;
    PlanSums s = {0, 0, 0};
    if (add < 0) {
      s.given = held;
    } else {
      s.want = (static_cast<long long>(len) + add + p.page_size - 1) / p.page_size - held;
      s.more = add;
    }
    return s;
  };
  PlanSums mine = {0, 0, 0};
  for (int z = z0; z < z1; ++z) {
    const int len = p.lens[z], add = p.add[z];
    s_lens[z] = len;
    if (len < 0 || static_cast<long long>(len) + max(add, 0) > room) {
      atomicMin(&s_bad, z);
    } else {
      mine = mine + sums_of(len, add);
    }
  }
  PlanSums upto = mine;
  for (int d = 1; d < 32; d <<= 1) {
    const PlanSums o = shfl_up(upto, d);
    if (lane >= d) upto = upto + o;
  }
  if (lane == 31) warp_sums[warp] = upto;
  __syncthreads();
  if (warp == 0) {
    PlanSums w = warp_sums[lane];
    for (int d = 1; d < 32; d <<= 1) {
      const PlanSums o = shfl_up(w, d);
      if (lane >= d) w = w + o;
    }
    warp_sums[lane] = w;
  }
  __syncthreads();
  const PlanSums total = warp_sums[31];
  PlanSums at = upto;
  if (warp > 0) at = at + warp_sums[warp - 1];
  const int top0 = p.num_free[0];
  const long long top = top0 + total.given;

  const bool range = s_bad != INT_MAX || top0 < 0 || top0 > p.num_pages || top > p.num_pages || total.more > p.tokens;
  const bool refused = range || total.want > top;
  at.given -= mine.given, at.want -= mine.want, at.more -= mine.more;
  for (int z = z0; z < z1; ++z) {
    const int len = s_lens[z], add = p.add[z];
    if (!refused) {
      s_given[z] = add < 0 ? static_cast<int>(at.given) : -1;
      s_want[z] = static_cast<int>(at.want);
      s_start[z] = static_cast<int>(at.more);
      at = at + sums_of(len, add);
    } else {
      s_start[z] = 0;
    }
  }
  if (tid == 0) s_start[p.requests] = refused ? 0 : static_cast<int>(total.more);
  __syncthreads();  // after this nobody reads lens, add or num_free again: the outputs may be the inputs

  if (refused) {
    if (tid == 0) {
      if (range) {
        paged_record(p.status, SYN_DEV_BAD_INDEX, s_bad != INT_MAX ? s_bad : -1, s_bad != INT_MAX ? s_lens[s_bad] : top0);
      } else {
        paged_record(p.status, SYN_DEV_NO_PAGES, -1, static_cast<int>(min(total.want, static_cast<long long>(INT_MAX))));
      }
    }
  } else {
    for (int z = warp; z < p.requests; z += PLAN_THREADS / 32) {
      if (s_given[z] < 0) continue;
      const int held = (s_lens[z] + p.page_size - 1) / p.page_size;
      for (int j = lane; j < held; j += 32) p.free_pages[top0 + s_given[z] + j] = p.table[z * p.table_stride + j];
    }
    __syncthreads();
    for (int z = warp; z < p.requests; z += PLAN_THREADS / 32) {
      if (s_given[z] >= 0) continue;
      const int held = (s_lens[z] + p.page_size - 1) / p.page_size;
      const int want = (z + 1 < p.requests ? s_want[z + 1] : static_cast<int>(total.want)) - s_want[z];
      for (int j = lane; j < want; j += 32)
        p.table[z * p.table_stride + held + j] = p.free_pages[top - 1 - s_want[z] - j];
    }
    __syncthreads();
  }
  for (int t = tid; t < p.tokens; t += PLAN_THREADS) {
    int slot = -1, position = 0;
    if (t < s_start[p.requests]) {
      int a = 0, b = p.requests;  // the last request that starts at or before t
      while (b - a > 1) {
        const int m = (a + b) >> 1;
        (s_start[m] <= t ? a : b) = m;
      }
      position = s_lens[a] + t - s_start[a];
      const int page = p.table[a * p.table_stride + position / p.page_size];
      if (static_cast<unsigned>(page) < static_cast<unsigned>(p.num_pages)) {
        slot = page * p.page_size + position % p.page_size;
      } else {
        paged_record(p.status, SYN_DEV_BAD_INDEX, a, page);
      }
    }
    p.slots[t] = slot;
    if (p.positions != nullptr) p.positions[t] = position;
  }
  for (int z = tid; z < p.requests; z += PLAN_THREADS) {
    p.starts[z] = s_start[z];
    p.lens_out[z] = refused ? s_lens[z] : s_given[z] >= 0 ? 0 : s_lens[z] + s_start[z + 1] - s_start[z];
  }
  if (tid == 0) {
    p.starts[p.requests] = s_start[p.requests];
    p.num_free_out[0] = refused ? top0 : static_cast<int>(top - total.want);
  }
}

// ----------------------------------------------------------------------------- append
constexpr int APPEND_THREADS = 256;

__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }

// One thread moves 16 elements of one head.
template <typename T, bool E4M3>
__global__ void __launch_bounds__(APPEND_THREADS) paged_append_kernel(syn_paged_append_args p) {
  const int parts = p.D / 16;
  const long long items = static_cast<long long>(p.tokens) * 2 * p.Hkv * parts;
  const long long i = static_cast<long long>(blockIdx.x) * APPEND_THREADS + threadIdx.x;
  if (i >= items) return;
  const int part = static_cast<int>(i % parts);
  const int h = static_cast<int>(i / parts % p.Hkv);
  const int which = static_cast<int>(i / parts / p.Hkv % 2);
  const int t = static_cast<int>(i / parts / p.Hkv / 2);
  const int slot = p.slots[t];
  if (slot < 0) return;
  if (slot >= p.num_pages * p.page_size) {
    paged_record(p.status, SYN_DEV_BAD_INDEX, t, slot);
    return;
  }
  const int64_t* xs = which ? p.v_strides : p.k_strides;
  const T* x = static_cast<const T*>(which ? p.v : p.k) + t * xs[0] + h * xs[1] + part * 16;
  const int64_t at = slot / p.page_size * p.cache_strides[0] + slot % p.page_size * p.cache_strides[1] +
                     h * p.cache_strides[2] + part * 16;
  const uint4 a = reinterpret_cast<const uint4*>(x)[0], b = reinterpret_cast<const uint4*>(x)[1];
  if constexpr (E4M3) {
    const float scale = (which ? p.v_scale : p.k_scale)[h];
    uint4 packed;
    unsigned char* out = reinterpret_cast<unsigned char*>(&packed);
    const T* in = reinterpret_cast<const T*>(&a);
    const T* in2 = reinterpret_cast<const T*>(&b);
    for (int j = 0; j < 8; ++j) {
      out[j] = __nv_cvt_float_to_fp8(__fdiv_rn(to_float(in[j]), scale), __NV_SATFINITE, __NV_E4M3);
      out[8 + j] = __nv_cvt_float_to_fp8(__fdiv_rn(to_float(in2[j]), scale), __NV_SATFINITE, __NV_E4M3);
    }
    *reinterpret_cast<uint4*>(static_cast<unsigned char*>(which ? p.v_cache : p.k_cache) + at) = packed;
  } else {
    uint4* out = reinterpret_cast<uint4*>(static_cast<T*>(which ? p.v_cache : p.k_cache) + at);
    out[0] = a;
    out[1] = b;
  }
}

static int launch_append(const syn_paged_append_args& a, cudaStream_t stream) {
  const long long items = static_cast<long long>(a.tokens) * 2 * a.Hkv * (a.D / 16);
  const unsigned grid = static_cast<unsigned>((items + APPEND_THREADS - 1) / APPEND_THREADS);
  const bool bf16 = a.dtype == SYN_DTYPE_BF16;
  if (a.cache_dtype == SYN_CACHE_E4M3) {
    if (bf16) paged_append_kernel<__nv_bfloat16, true><<<grid, APPEND_THREADS, 0, stream>>>(a);
    else paged_append_kernel<__half, true><<<grid, APPEND_THREADS, 0, stream>>>(a);
  } else {  // a copy of 16-bit words
    paged_append_kernel<__half, false><<<grid, APPEND_THREADS, 0, stream>>>(a);
  }
  SYN_CUDA_TRY(cudaGetLastError());
  return SYN_OK;
}

constexpr int PLAN_SMEM_MAX = (4 * SYN_PAGE_PLAN_MAX_REQUESTS + 1) * 4;

int preload_paged_kernels() {
  cudaFuncAttributes attr;
  SYN_CUDA_TRY(cudaFuncSetAttribute(page_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, PLAN_SMEM_MAX));
  SYN_CUDA_TRY(cudaFuncGetAttributes(&attr, page_plan_kernel));
  SYN_CUDA_TRY(cudaFuncGetAttributes(&attr, paged_append_kernel<__half, false>));
  SYN_CUDA_TRY(cudaFuncGetAttributes(&attr, paged_append_kernel<__half, true>));
  SYN_CUDA_TRY(cudaFuncGetAttributes(&attr, paged_append_kernel<__nv_bfloat16, true>));
  return SYN_OK;
}

}  // namespace syn

extern "C" int syn_page_plan(const syn_page_plan_args* a, void* stream) {
  using namespace syn;
  if (a == nullptr || a->lens == nullptr || a->add == nullptr || a->table == nullptr || a->free_pages == nullptr ||
      a->num_free == nullptr || a->starts == nullptr || a->lens_out == nullptr || a->num_free_out == nullptr)
    return SYN_ERR_INVALID;
  if (a->requests <= 0 || a->width <= 0 || a->page_size <= 0 || a->num_pages <= 0 || a->tokens < 0) return SYN_ERR_INVALID;
  if (a->tokens > 0 && a->slots == nullptr) return SYN_ERR_INVALID;
  if (a->table_stride < a->width) return SYN_ERR_INVALID;
  if (a->requests > SYN_PAGE_PLAN_MAX_REQUESTS) return SYN_ERR_TOO_LARGE;
  if (static_cast<int64_t>(a->num_pages) * a->page_size > INT_MAX) return SYN_ERR_TOO_LARGE;
  PagedDevice device(a->device);
  SYN_CUDA_TRY(device.error());
  const int smem = (4 * a->requests + 1) * 4;
  if (smem > 48 * 1024)
    SYN_CUDA_TRY(cudaFuncSetAttribute(page_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, PLAN_SMEM_MAX));
  page_plan_kernel<<<1, PLAN_THREADS, smem, static_cast<cudaStream_t>(stream)>>>(*a);
  SYN_CUDA_TRY(cudaGetLastError());
  return SYN_OK;
}

extern "C" int syn_paged_append(const syn_paged_append_args* a, void* stream) {
  using namespace syn;
  if (a == nullptr || a->tokens < 0 || a->Hkv <= 0 || a->D <= 0 || a->page_size <= 0 || a->num_pages <= 0)
    return SYN_ERR_INVALID;
  if (a->dtype != SYN_DTYPE_F16 && a->dtype != SYN_DTYPE_BF16) return SYN_ERR_UNSUPPORTED;
  if (a->cache_dtype != SYN_CACHE_SAME && a->cache_dtype != SYN_CACHE_E4M3) return SYN_ERR_UNSUPPORTED;
  if (a->D % 16 != 0) return SYN_ERR_UNSUPPORTED;
  if (static_cast<int64_t>(a->num_pages) * a->page_size > INT_MAX) return SYN_ERR_TOO_LARGE;
  if (static_cast<int64_t>(a->tokens) * a->Hkv * (a->D / 16) > INT_MAX) return SYN_ERR_TOO_LARGE;
  if (a->tokens == 0) return SYN_OK;
  syn_paged_append_args p = *a;
  const bool e4m3 = a->cache_dtype == SYN_CACHE_E4M3;
  if (a->k == nullptr || a->v == nullptr || a->slots == nullptr || a->k_cache == nullptr || a->v_cache == nullptr)
    return SYN_ERR_INVALID;
  if (e4m3 && (a->k_scale == nullptr || a->v_scale == nullptr)) return SYN_ERR_INVALID;
  if (!paged_aligned(a->k) || !paged_aligned(a->v) || !paged_aligned(a->k_cache) || !paged_aligned(a->v_cache) ||
      !paged_strides(p.k_strides, {a->tokens, a->Hkv}, 2) || !paged_strides(p.v_strides, {a->tokens, a->Hkv}, 2) ||
      !paged_strides(p.cache_strides, {a->num_pages, a->page_size, a->Hkv}, e4m3 ? 1 : 2))
    return SYN_ERR_INVALID;
  PagedDevice device(a->device);
  SYN_CUDA_TRY(device.error());
  return launch_append(p, static_cast<cudaStream_t>(stream));
}
