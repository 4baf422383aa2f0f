// Step plan and append of the paged key-value cache (see include/syncopate_b200.h for what they
// compute).
#include "paged.cuh"

#include <cuda_fp8.h>
#include <math_constants.h>

#include <atomic>
#include <type_traits>

namespace syn {

// The plan is short work on a few tables: its time is that of its dependent steps.  A few requests and tokens take one
// small block (8 requests: 3.4 us, 4.6 as a cluster); more are dealt out to a cluster, whose blocks all run the
// same sums (1021 requests: 8.1 us, 14.1 in one block of 1024 threads; 82k tokens: 14.7 against 66).
constexpr int PLAN_THREADS = 1024;
constexpr int PLAN_CLUSTER = 8;
constexpr int PLAN_SMALL_THREADS = 256;
constexpr int PLAN_SMALL_REQUESTS = 256;
constexpr int PLAN_SMALL_TOKENS = 1024;

struct PlanSums {
  long long given, want, more;  // pages pushed, pages popped, tokens appended
};

__device__ __forceinline__ PlanSums operator+(PlanSums a, PlanSums b) {
  return {a.given + b.given, a.want + b.want, a.more + b.more};
}
__device__ __forceinline__ PlanSums shfl_up(PlanSums a, int d) {
  return {__shfl_up_sync(~0u, a.given, d), __shfl_up_sync(~0u, a.want, d), __shfl_up_sync(~0u, a.more, d)};
}

// Running sums over the requests give every request its place on the stack of free pages and its first token; then
// pages are pushed, popped and the tokens' slots written.  BLOCKS = blocks of the only cluster.
template <int BLOCKS>
__global__ void __launch_bounds__(PLAN_THREADS) page_plan_kernel(const __grid_constant__ syn_page_plan_args p) {
  extern __shared__ int32_t plan_smem[];
  int32_t* s_lens = plan_smem;                  // [requests]
  int32_t* s_given = s_lens + p.requests;       // pages pushed before the request; -1: the request goes on
  int32_t* s_want = s_given + p.requests;       // pages popped before it
  int32_t* s_start = s_want + p.requests;       // [requests + 1]
  __shared__ PlanSums warp_sums[32];
  __shared__ int s_bad;
  const int tid = threadIdx.x, threads = blockDim.x, lane = tid & 31, warp = tid >> 5, warps = threads >> 5;
  const int block = BLOCKS == 1 ? 0 : blockIdx.x;
  if (tid == 0) s_bad = INT_MAX;
  __syncthreads();

  const int per = (p.requests + threads - 1) / threads;
  const int z0 = min(tid * per, p.requests), z1 = min(z0 + per, p.requests);
  const long long room = static_cast<long long>(p.width) * p.page_size;
  const uint32_t page_size = p.page_size;
  auto pages_of = [&](uint32_t n) { return n / page_size + (n % page_size != 0); };
  auto sums_of = [&](int len, int add) {  // len + add is at most width * page_size, or the request is refused
    const int held = pages_of(len);
    PlanSums s = {0, 0, 0};
    if (add < 0) {
      s.given = held;
    } else {
      s.want = pages_of(static_cast<uint32_t>(len) + add) - held;
      s.more = add;
    }
    return s;
  };
  const int top0 = p.num_free[0];
  PlanSums mine = {0, 0, 0};
  for (int z = z0; z < z1; ++z) {
    const int len = p.lens[z], add = p.add[z];
    s_lens[z] = len;
    s_given[z] = add;
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
    PlanSums w = lane < warps ? warp_sums[lane] : PlanSums{0, 0, 0};
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
  const long long top = top0 + total.given;

  const bool range = s_bad != INT_MAX || top0 < 0 || top0 > p.num_pages || top > p.num_pages || total.more > p.tokens;
  const bool refused = range || total.want > top;
  at.given -= mine.given, at.want -= mine.want, at.more -= mine.more;
  for (int z = z0; z < z1; ++z) {
    const int len = s_lens[z], add = s_given[z];
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
  __syncthreads();

  const int first = block * warps + warp, skip = BLOCKS * warps;  // a warp takes a request
  if (!refused && total.given > 0) {
    for (int z = first; z < p.requests; z += skip) {
      if (s_given[z] < 0) continue;
      const int held = pages_of(s_lens[z]);
      const int32_t* from = p.table + z * p.table_stride;
      int32_t* to = p.free_pages + top0 + s_given[z];
      for (int j0 = 0; j0 < held; j0 += 128) {  // four loads on the way
        int page[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (j0 + i * 32 + lane < held) page[i] = from[j0 + i * 32 + lane];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (j0 + i * 32 + lane < held) to[j0 + i * 32 + lane] = page[i];
      }
    }
  }
  // Pages pushed are seen by all, and nobody reads lens, add or num_free again: the outputs may be the inputs.
  if constexpr (BLOCKS == 1) {
    __syncthreads();
  } else {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
  if (refused) {
    if (block == 0 && tid == 0) {
      if (range) {
        paged_record(p.status, SYN_DEV_BAD_INDEX, s_bad != INT_MAX ? s_bad : -1, s_bad != INT_MAX ? s_lens[s_bad] : top0);
      } else {
        paged_record(p.status, SYN_DEV_NO_PAGES, -1, static_cast<int>(min(total.want, static_cast<long long>(INT_MAX))));
      }
    }
  } else if (total.want > 0) {
    for (int z = first; z < p.requests; z += skip) {
      if (s_given[z] >= 0) continue;
      const int held = pages_of(s_lens[z]);
      const int want = (z + 1 < p.requests ? s_want[z + 1] : static_cast<int>(total.want)) - s_want[z];
      for (int j = lane; j < want; j += 32)
        p.table[z * p.table_stride + held + j] = __ldcg(p.free_pages + top - 1 - s_want[z] - j);
    }
  }
  const int tokens = s_start[p.requests];
  for (int t = block * threads + tid; t < p.tokens; t += BLOCKS * threads) {
    int slot = -1, position = 0;
    if (t < tokens) {
      int a = 0, b = p.requests;  // the last request that starts at or before t
      while (b - a > 1) {
        const int m = (a + b) >> 1;
        (s_start[m] <= t ? a : b) = m;
      }
      position = s_lens[a] + t - s_start[a];
      const int i = position / page_size, held = pages_of(s_lens[a]);
      // A page that the request had is in the table; a new one is read where it comes from, not where another warp puts it.
      const int page = i < held ? p.table[a * p.table_stride + i] : __ldcg(p.free_pages + top - 1 - s_want[a] - (i - held));
      if (static_cast<unsigned>(page) < static_cast<unsigned>(p.num_pages)) {
        slot = page * p.page_size + position % page_size;
      } else {
        paged_record(p.status, SYN_DEV_BAD_INDEX, a, page);
      }
    }
    p.slots[t] = slot;
    if (p.positions != nullptr) p.positions[t] = position;
  }
  if (block != 0) return;
  for (int z = tid; z < p.requests; z += threads) {
    p.starts[z] = s_start[z];
    p.lens_out[z] = refused ? s_lens[z] : s_given[z] >= 0 ? 0 : s_lens[z] + s_start[z + 1] - s_start[z];
  }
  if (tid == 0) {
    p.starts[p.requests] = tokens;
    p.num_free_out[0] = refused ? top0 : static_cast<int>(top - total.want);
  }
}

// ----------------------------------------------------------------------------- append
// Threads of a block: conversions do better in smaller ones (99 MB into e4m3: 26.3 us with 256, 24.3 with 128), the copy
// does not (264 MB: 41.5 and 41.9).  The products of a pair in one instruction: 22.8.
template <bool E4M3>
constexpr int APPEND_THREADS = E4M3 ? 128 : 256;

template <typename T>
__device__ __forceinline__ float2 pair_to_float(uint32_t x) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xFFFF0000u));
  else
    return __half22float2(*reinterpret_cast<const __half2*>(&x));
}
__device__ __forceinline__ uint32_t e4m3_pair(float x, float y) {
  return __nv_cvt_float2_to_fp8x2(make_float2(x, y), __NV_SATFINITE, __NV_E4M3);
}
// Two products at once.
__device__ __forceinline__ float2 mul2(float2 x, float y) {
  float2 z;
  asm("{\n.reg .b64 a, b, c;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %4};\nmul.rn.f32x2 c, a, b;\nmov.b64 {%0, %1}, c;\n}"
      : "=f"(z.x), "=f"(z.y)
      : "f"(x.x), "f"(x.y), "f"(y));
  return z;
}

// Eight quotients as e4m3.  x * r, r = 1 / scale rounded, is within 2^-22 of the 32-bit quotient (two roundings against
// one), and rounding to e4m3 keeps order: where both ends of x * r (1 -+ 2^-21) become the same number, so does the
// quotient.  Only where a border lies between them are the divisions needed.  `fast`: r is a normal number.
template <typename T>
__device__ __forceinline__ uint2 e4m3_quotients(const uint4& v, float scale, float r, bool fast) {
  constexpr float LOW = 1.f - 0x1p-21f, HIGH = 1.f + 0x1p-21f;
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  uint32_t q[4], differ = fast ? 0 : 1;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 x = mul2(pair_to_float<T>(w[j]), r), low = mul2(x, LOW), high = mul2(x, HIGH);
    q[j] = e4m3_pair(low.x, low.y);
    differ |= q[j] ^ e4m3_pair(high.x, high.y);
  }
  if (differ != 0) {
#pragma unroll 1
    for (int j = 0; j < 4; ++j) {
      const float2 x = pair_to_float<T>(j == 0 ? w[0] : j == 1 ? w[1] : j == 2 ? w[2] : w[3]);
      const uint32_t exact = e4m3_pair(__fdiv_rn(x.x, scale), __fdiv_rn(x.y, scale));
      if (j == 0) q[0] = exact;
      else if (j == 1) q[1] = exact;
      else if (j == 2) q[2] = exact;
      else q[3] = exact;
    }
  }
  return make_uint2(q[0] | q[1] << 16, q[2] | q[3] << 16);
}

// Eight elements of one head are an item.  A thread has one item of a token, whose place it works out once, and moves
// it for TOKENS tokens, all of which it has on the way before the first is stored.
template <typename T, bool E4M3, int TOKENS>
__global__ void __launch_bounds__(APPEND_THREADS<E4M3>) paged_append_kernel(const __grid_constant__ syn_paged_append_args p) {
  constexpr int THREADS = APPEND_THREADS<E4M3>;
  // Slots behind the last row, dealt out to the threads of the grid's first column.
  if (blockIdx.y == 0) {
    const int64_t skip = static_cast<int64_t>(gridDim.x) * THREADS;
    for (int64_t t = p.tokens + static_cast<int64_t>(blockIdx.x) * THREADS + threadIdx.x; t < p.num_slots; t += skip) {
      const int slot = __ldg(p.slots + t);
      if (slot >= 0) paged_record(p.status, SYN_DEV_BAD_INDEX, static_cast<int>(t), slot);
    }
  }
  const int parts = p.D / 8, items = 2 * p.Hkv * parts;
  const int at_once = items < THREADS ? THREADS / items : 1;  // tokens that a block moves side by side
  const int width = items < THREADS ? items : THREADS;
  const int side = threadIdx.x / width, item = blockIdx.y * THREADS + threadIdx.x % width;
  if (side >= at_once || item >= items) return;
  const int part = item % parts, h = item / parts % p.Hkv;
  const bool values = item >= p.Hkv * parts;
  const int64_t row = values ? p.v_strides[0] : p.k_strides[0];
  const T* x = static_cast<const T*>(values ? p.v : p.k) + h * (values ? p.v_strides[1] : p.k_strides[1]) + part * 8;
  const int64_t place = h * p.cache_strides[2] + part * 8;
  void* cache = values ? p.v_cache : p.k_cache;
  const int t0 = blockIdx.x * (at_once * TOKENS) + side;
  int slot[TOKENS];
  uint4 v[TOKENS];
#pragma unroll
  for (int i = 0; i < TOKENS; ++i) {
    const int t = t0 + i * at_once;
    slot[i] = t < p.tokens ? __ldg(p.slots + t) : -1;
  }
#pragma unroll
  for (int i = 0; i < TOKENS; ++i)
    if (slot[i] >= 0) v[i] = __ldg(reinterpret_cast<const uint4*>(x + (t0 + i * at_once) * row));
  float scale = 1.f, reciprocal = 1.f;
  bool fast = true;
  if constexpr (E4M3) {
    scale = (values ? p.v_scale : p.k_scale)[h];
    reciprocal = __frcp_rn(scale);
    fast = fabsf(reciprocal) >= 0x1p-126f && fabsf(reciprocal) < CUDART_INF_F;
  }
#pragma unroll
  for (int i = 0; i < TOKENS; ++i) {
    if (slot[i] < 0) continue;
    const uint32_t page = static_cast<uint32_t>(slot[i]) / static_cast<uint32_t>(p.page_size);
    if (page >= static_cast<uint32_t>(p.num_pages)) {
      paged_record(p.status, SYN_DEV_BAD_INDEX, t0 + i * at_once, slot[i]);
      continue;
    }
    const int64_t at = page * p.cache_strides[0] + (slot[i] - static_cast<int>(page) * p.page_size) * p.cache_strides[1] + place;
    if constexpr (E4M3) {
      *reinterpret_cast<uint2*>(static_cast<unsigned char*>(cache) + at) = e4m3_quotients<T>(v[i], scale, reciprocal, fast);
    } else {
      *reinterpret_cast<uint4*>(static_cast<T*>(cache) + at) = v[i];
    }
  }
}

template <typename T, bool E4M3>
static int launch_append(const syn_paged_append_args& a, cudaStream_t stream) {
  constexpr int THREADS = APPEND_THREADS<E4M3>;
  const int items = 2 * a.Hkv * (a.D / 8);
  const int at_once = items < THREADS ? THREADS / items : 1;
  const int columns = (items + THREADS - 1) / THREADS;
  // Four tokens a thread where that still makes a few blocks for every SM: 64 bytes on the way a thread carry the
  // stream; one where there are so few that latency counts.
  const int64_t rows = (a.tokens + at_once - 1) / at_once;
  const dim3 one(static_cast<unsigned>(rows), columns), four(static_cast<unsigned>((rows + 3) / 4), columns);
  if (columns > 65535) return SYN_ERR_TOO_LARGE;
  if (rows == 0) paged_append_kernel<T, E4M3, 1><<<1, THREADS, 0, stream>>>(a);
  else if (rows * columns >= 4096) paged_append_kernel<T, E4M3, 4><<<four, THREADS, 0, stream>>>(a);
  else paged_append_kernel<T, E4M3, 1><<<one, THREADS, 0, stream>>>(a);
  SYN_CUDA_TRY(cudaGetLastError());
  return SYN_OK;
}

template <typename T, bool E4M3>
static int preload_append() {
  cudaFuncAttributes attr;
  SYN_CUDA_TRY(cudaFuncGetAttributes(&attr, paged_append_kernel<T, E4M3, 1>));
  SYN_CUDA_TRY(cudaFuncGetAttributes(&attr, paged_append_kernel<T, E4M3, 4>));
  return SYN_OK;
}

constexpr int PLAN_SMEM_MAX = (4 * SYN_PAGE_PLAN_MAX_REQUESTS + 1) * 4;

template <int BLOCKS>
static int configure_plan() {
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  SYN_CUDA_TRY(cudaGetDevice(&dev));
  const uint64_t bit = 1ull << (dev & 63);
  if (dev < 64 && (done.load(std::memory_order_relaxed) & bit)) return SYN_OK;
  SYN_CUDA_TRY(cudaFuncSetAttribute(page_plan_kernel<BLOCKS>, cudaFuncAttributeMaxDynamicSharedMemorySize, PLAN_SMEM_MAX));
  done.fetch_or(bit, std::memory_order_relaxed);
  return SYN_OK;
}

template <int BLOCKS>
static int launch_plan(const syn_page_plan_args& a, int threads, cudaStream_t stream) {
  const int rc = configure_plan<BLOCKS>();
  if (rc != SYN_OK) return rc;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = BLOCKS, attr.val.clusterDim.y = 1, attr.val.clusterDim.z = 1;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(BLOCKS);
  config.blockDim = dim3(threads);
  config.dynamicSmemBytes = (4 * a.requests + 1) * 4;
  config.stream = stream;
  config.attrs = &attr;
  config.numAttrs = BLOCKS > 1 ? 1 : 0;
  SYN_CUDA_TRY(cudaLaunchKernelEx(&config, page_plan_kernel<BLOCKS>, a));
  return SYN_OK;
}

int preload_paged_kernels() {
  int rc = configure_plan<1>();
  if (rc == SYN_OK) rc = configure_plan<PLAN_CLUSTER>();
  if (rc == SYN_OK) rc = preload_append<__half, false>();
  if (rc == SYN_OK) rc = preload_append<__half, true>();
  if (rc == SYN_OK) rc = preload_append<__nv_bfloat16, true>();
  return rc;
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
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a->requests <= PLAN_SMALL_REQUESTS && a->tokens <= PLAN_SMALL_TOKENS) return launch_plan<1>(*a, PLAN_SMALL_THREADS, s);
  return launch_plan<PLAN_CLUSTER>(*a, PLAN_THREADS, s);
}

extern "C" int syn_paged_append(const syn_paged_append_args* a, void* stream) {
  using namespace syn;
  if (a == nullptr || a->tokens < 0 || a->num_slots < 0 || a->Hkv <= 0 || a->D <= 0 || a->page_size <= 0 || a->num_pages <= 0)
    return SYN_ERR_INVALID;
  if (a->dtype != SYN_DTYPE_F16 && a->dtype != SYN_DTYPE_BF16) return SYN_ERR_UNSUPPORTED;
  if (a->cache_dtype != SYN_CACHE_SAME && a->cache_dtype != SYN_CACHE_E4M3) return SYN_ERR_UNSUPPORTED;
  if (a->D % 16 != 0) return SYN_ERR_UNSUPPORTED;
  if (static_cast<int64_t>(a->num_pages) * a->page_size > INT_MAX) return SYN_ERR_TOO_LARGE;
  if (static_cast<int64_t>(a->Hkv) * a->D > INT_MAX / 2) return SYN_ERR_TOO_LARGE;
  syn_paged_append_args p = *a;
  if (a->status == nullptr) p.num_slots = 0;  // nobody to tell
  if (a->tokens == 0 && p.num_slots == 0) return SYN_OK;
  const bool e4m3 = a->cache_dtype == SYN_CACHE_E4M3;
  if ((a->tokens > 0 && (a->k == nullptr || a->v == nullptr)) || a->slots == nullptr || a->k_cache == nullptr || a->v_cache == nullptr)
    return SYN_ERR_INVALID;
  if (e4m3 && (a->k_scale == nullptr || a->v_scale == nullptr)) return SYN_ERR_INVALID;
  if (!paged_aligned(a->k) || !paged_aligned(a->v) || !paged_aligned(a->k_cache) || !paged_aligned(a->v_cache) ||
      !paged_strides(p.k_strides, {a->tokens, a->Hkv}, 2) || !paged_strides(p.v_strides, {a->tokens, a->Hkv}, 2) ||
      !paged_strides(p.cache_strides, {a->num_pages, a->page_size, a->Hkv}, e4m3 ? 1 : 2))
    return SYN_ERR_INVALID;
  PagedDevice device(a->device);
  SYN_CUDA_TRY(device.error());
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (!e4m3) return launch_append<__half, false>(p, s);  // a copy of 16-bit words
  return a->dtype == SYN_DTYPE_BF16 ? launch_append<__nv_bfloat16, true>(p, s) : launch_append<__half, true>(p, s);
}
