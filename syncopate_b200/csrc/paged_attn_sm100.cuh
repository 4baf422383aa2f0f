// Attention of the newest tokens over a paged key-value cache (decoding, drafted tokens).
//
// Mathematics.  Rows are (new token, query head) pairs.  Over its keys in any order a row keeps a reference m
// near the maximum of its scores s (times log2 e), the sum l of 2^(s - m) and the output o = sum 2^(s - m) v, rescaled
// by 2^(m - m') when the reference rises; parts of a row's keys are joined by the same rule.
//
// What bounds it.  Every key and value is read once and serves the group of query heads that share it:
// 4 * group * D operations for 2 * D stored numbers, about `group` operations a byte, against 250 at
// which the matrix units would become the bound.  So the work is a stream from HBM, the matrix products
// are small ones on mma.sync, whose fragments stay in registers; they are turned round (keys by rows,
// dimensions by rows) because rows then come in eights, as groups do, and not in sixteens.  The layout is chosen
// for loads in flight:
//   * Every warp streams keys of its own through a ring of its own in shared memory (cp.async of 16
//     bytes, a page lookup per key), so no barrier stands between loading and computing; the warps of a
//     block meet only when a unit of rows ends.
//   * The work (requests x key-value heads x row tiles x key tiles) is laid out in one line and cut into
//     equal shares for a grid that fills the GPU, whatever the lengths; loads run on across the borders of
//     units.  A unit that a border cuts leaves partial results, which a second small kernel joins in a fixed
//     order: results do not depend on timing, there are no atomics and no state between calls.
#pragma once
#include <math_constants.h>

#include <type_traits>

#include "paged.cuh"

namespace syn {

constexpr int PA_WARPS = 4;
constexpr int PA_THREADS = PA_WARPS * 32;
constexpr int PA_MAX_BLOCKS = 3;  // resident blocks an SM, over all variants
// The reference a row's weights are taken against (m) follows its maximum only when that has risen by more
// than this power of two: a vote without shuffles on most steps, and few rescales.  Weights stay below 2^8.
constexpr float PA_SLACK = 8.f;
constexpr int PA_DESC = 4;  // int32 words a block leaves for the join

struct PagedAttnParams {
  syn_paged_attn_args a;
  int32_t grid;       // blocks of the launch
  int32_t min_tiles;  // fewest key tiles worth a block
  uint32_t page_mul;  // key / page_size = mulhi(key, page_mul) >> page_shift (page_mul 0: pages of one key)
  int32_t page_shift;
  float* part_o;      // [2 * grid][rows of a unit][D]
  float* part_ml;     // [2 * grid][rows of a unit][2]
  int32_t* desc;      // [grid][PA_DESC]
};

template <typename T, bool E4M3_, int D_, int RT_>
struct PagedCfg {
  using type = T;
  static constexpr bool E4M3 = E4M3_;
  static constexpr int D = D_;
  static constexpr int RT = RT_;                     // 8-row tiles of a unit
  static constexpr int ROWS = 8 * RT;
  static constexpr int KEYS = E4M3 ? 32 : 16;        // keys of a warp's step
  static constexpr int TILE = KEYS * PA_WARPS;       // keys of a block's step
  static constexpr int ROWB = D * (E4M3 ? 1 : 2);    // bytes of a stored head
  static constexpr int CPR = ROWB / 16;              // 16-byte chunks of it
  static constexpr int HALFB = KEYS * ROWB;          // the keys of a step, or its values
  static constexpr int BLOCKS = D == 256 ? 3 - RT : RT <= 2 ? 3 : 2;  // resident on an SM
  static constexpr int SLOTS = (D == 256 ? 24 : RT <= 2 ? 16 : 20) * 1024 / HALFB;
  static constexpr int RING = SLOTS * HALFB;         // bytes a warp
  static constexpr bool QREG = RT * D <= 256;        // query fragments in registers, else in shared memory
  static constexpr int KSTEPS = D / 16;
  static constexpr int DT = D / 16;                  // 16-dimension tiles of the output
  static constexpr int DC = RT == 4 ? 16 : 32;  // output dimensions of a merge pass
  static constexpr int NT_PASS = DC / 8;
  static constexpr int PASSES = D / DC;
  static constexpr int MERGE_LD = DC + 4;
  static constexpr int SMEM_Q = QREG ? 0 : KSTEPS * RT * 256;
  static constexpr int SMEM_MERGE = PA_WARPS * ROWS * MERGE_LD * 4;
  static constexpr int SMEM_ML = PA_WARPS * ROWS * 2 * 4;
  static constexpr int SMEM = PA_WARPS * RING + SMEM_Q + SMEM_MERGE + SMEM_ML;
  static_assert(BLOCKS * (SMEM + 1280) <= 228 * 1024, "shared memory of an SM");
  static_assert(SLOTS >= 3, "a key half, a value half and one on its way");
};

// ----------------------------------------------------------------------------- instructions
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint4 lds16(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint2 lds8(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void sts16(uint32_t addr, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
template <bool BF16>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (BF16) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  } else {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Four e4m3 bytes as two pairs of halves (exact).
__device__ __forceinline__ void e4m3x4_to_h2x2(uint32_t x, uint32_t& lo, uint32_t& hi) {
  asm("{\n.reg .b16 l, h;\nmov.b32 {l, h}, %2;\ncvt.rn.f16x2.e4m3x2 %0, l;\ncvt.rn.f16x2.e4m3x2 %1, h;\n}"
      : "=r"(lo), "=r"(hi)
      : "r"(x));
}
// 8 x 8 matrix of 16-bit numbers, a row in four lanes, transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  if constexpr (BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
template <bool BF16>
__device__ __forceinline__ float2 unpack2(uint32_t x) {
  if constexpr (BF16) {
    return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xFFFF0000u));
  } else {
    return __half22float2(*reinterpret_cast<const __half2*>(&x));
  }
}

// ----------------------------------------------------------------------------- the line of work
struct PagedRequest {
  int s0, n;       // rows of q: first one, how many
  int len;         // keys (one more than the table has room for, where the length says more)
  int first;       // first key that any row sees
  int tiles, rt;   // key tiles of a unit; row tiles a head
};

template <typename C>
__device__ __forceinline__ PagedRequest paged_request(const syn_paged_attn_args& a, int z) {
  PagedRequest r;
  r.s0 = z, r.n = 1;
  if (a.starts != nullptr) {
    r.s0 = min(max(a.starts[z], 0), a.tokens);
    r.n = min(max(a.starts[z + 1], r.s0), a.tokens) - r.s0;
  }
  const long long room = static_cast<long long>(a.width) * a.page_size;
  int len = max(a.lens[z], 0);
  if (len > room) len = static_cast<int>(min(room + 1, static_cast<long long>(INT_MAX)));
  r.len = len;
  r.first = a.window > 0 ? max(0, min(len, len - r.n - a.window + 1)) : 0;
  r.tiles = max(1, (len - r.first + C::TILE - 1) / C::TILE);
  r.rt = (r.n * (a.Hq / a.Hkv) + C::ROWS - 1) / C::ROWS;
  return r;
}

__device__ __forceinline__ long long paged_border(long long total, int shares, int c) { return total * c / shares; }

// Position on the line: key tile `tile` of unit `sub` (head * row tiles + row tile) of request z.
template <typename C>
struct PagedCursor {
  int z, sub, tile;
  PagedRequest r;

  __device__ __forceinline__ void at(const syn_paged_attn_args& a, int z_, long long rest) {
    z = z_;
    r = paged_request<C>(a, z);
    sub = static_cast<int>(rest / r.tiles);
    tile = static_cast<int>(rest % r.tiles);
  }
  // To the first tile of the next unit; the caller knows that there is one.
  __device__ __forceinline__ void next_unit(const syn_paged_attn_args& a) {
    tile = 0;
    if (++sub < a.Hkv * r.rt) return;
    sub = 0;
    do {
      ++z;
      r = paged_request<C>(a, z);
    } while (r.rt == 0 && z + 1 < a.requests);
  }
};

// ----------------------------------------------------------------------------- fragments
// Calls f(dt, a) with the fragments of the transposed values (16 dimensions by the 16 keys of group `kk` of the
// step) for every 16-dimension tile of the output.  Row c (0 .. 7) of the tile's halves nt = 2 dt, 2 dt + 1 is
// dimension 8 nt + c of 16-bit values.  8-bit values are fetched 16 (D = 64: 8) dimensions of one key at a
// time and paired with the next key's, so there it is dimension 16 c + nt % 16 + 128 (nt / 16) (D = 64:
// 8 c + nt): a permutation that the epilogue undoes.
template <typename C, typename F>
__device__ __forceinline__ void each_v(uint32_t v, int lane, int kk, F f) {
  if constexpr (!C::E4M3) {
    const int row = (lane & 7) + (lane >> 4) * 8;
#pragma unroll
    for (int j = 0; j < C::DT; ++j) {
      uint32_t a[4];
      ldsm4t(v + row * C::ROWB + (((j * 2 + ((lane >> 3) & 1)) ^ (row & 7)) << 4), a);
      f(j, a);
    }
  } else {
    const int g = lane >> 2, t = lane & 3;
    const uint32_t row0 = v + (kk * 16 + 2 * t) * C::ROWB;
    auto words = [&](int dt, uint32_t x0, uint32_t x1, uint32_t x8, uint32_t x9) {
      const uint32_t lo01 = __byte_perm(x0, x1, 0x5140), hi01 = __byte_perm(x0, x1, 0x7362);
      const uint32_t lo89 = __byte_perm(x8, x9, 0x5140), hi89 = __byte_perm(x8, x9, 0x7362);
      uint32_t a[4];
      e4m3x4_to_h2x2(lo01, a[0], a[1]);
      e4m3x4_to_h2x2(lo89, a[2], a[3]);
      f(dt, a);
      e4m3x4_to_h2x2(hi01, a[0], a[1]);
      e4m3x4_to_h2x2(hi89, a[2], a[3]);
      f(dt + 1, a);
    };
    if constexpr (C::D == 64) {
      const uint32_t at = (((g >> 1) ^ t) << 4) + (g & 1) * 8;
      const uint2 x0 = lds8(row0 + at), x1 = lds8(row0 + C::ROWB + at);
      const uint2 x8 = lds8(row0 + 8 * C::ROWB + at), x9 = lds8(row0 + 9 * C::ROWB + at);
      words(0, x0.x, x1.x, x8.x, x9.x);
      words(2, x0.y, x1.y, x8.y, x9.y);
    } else {
#pragma unroll
      for (int half = 0; half < C::D / 128; ++half) {
        const uint32_t at = ((g + half * 8) ^ (t << 1)) << 4;
        const uint4 x0 = lds16(row0 + at), x1 = lds16(row0 + C::ROWB + at);
        const uint4 x8 = lds16(row0 + 8 * C::ROWB + at), x9 = lds16(row0 + 9 * C::ROWB + at);
        words(half * 8, x0.x, x1.x, x8.x, x9.x);
        words(half * 8 + 2, x0.y, x1.y, x8.y, x9.y);
        words(half * 8 + 4, x0.z, x1.z, x8.z, x9.z);
        words(half * 8 + 6, x0.w, x1.w, x8.w, x9.w);
      }
    }
  }
}

// Place of 16-byte chunk `chunk` of row `row` in a warp's ring (chosen so that the reads above and those of
// the keys below meet no bank twice; D = 64 in 8 bits reads its values two deep).
template <typename C, bool VALUES>
__device__ __forceinline__ uint32_t ring_at(int row, int chunk) {
  int c = chunk;
  if constexpr (!C::E4M3) c ^= row & 7;
  else if constexpr (VALUES) c ^= C::D == 64 ? (row >> 1) & 3 : ((row >> 1) & 3) << 1;
  else if constexpr (C::D != 64) c ^= (row & 1) << 2;
  return row * C::ROWB + (c << 4);
}

// Dimension of entry e (0 .. DC - 1) of merge pass `pass`; entries 2 i and 2 i + 1 are neighbours.
template <typename C>
__device__ __forceinline__ int merge_dim(int pass, int e) {
  if constexpr (!C::E4M3) return pass * C::DC + e;
  const int nt = pass * C::NT_PASS + e % C::NT_PASS, c = e / C::NT_PASS;
  if constexpr (C::D == 64) return 8 * c + nt;
  return (nt / 16) * 128 + 16 * c + nt % 16;
}
// Entry of row c of the pass's i-th 8-dimension tile.
template <typename C>
__device__ __forceinline__ int merge_entry(int i, int c) {
  return C::E4M3 ? c * C::NT_PASS + i : i * 8 + c;
}

template <typename C>
__global__ void __launch_bounds__(PA_THREADS, C::BLOCKS) paged_attn_kernel(const __grid_constant__ PagedAttnParams p) {
  using T = typename C::type;
  constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr bool MBF16 = BF16 && !C::E4M3;  // type of the matrix products: 8-bit values are halves there
  constexpr int RT = C::RT;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ long long s_sum[PA_WARPS];
  __shared__ long long s_rest;
  __shared__ int s_z;
  const syn_paged_attn_args& a = p.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
  const int group = a.Hq / a.Hkv;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // ---- this block's share of the line
  const int per = (a.requests + PA_THREADS - 1) / PA_THREADS;
  const int z0 = min(tid * per, a.requests), z1 = min(z0 + per, a.requests);
  long long mine = 0;
  for (int z = z0; z < z1; ++z) {
    const PagedRequest r = paged_request<C>(a, z);
    mine += static_cast<long long>(r.tiles) * a.Hkv * r.rt;
    if (blockIdx.x == 0) {
      if (a.lens[z] < 0) paged_record(a.status, SYN_DEV_BAD_INDEX, z, a.lens[z]);
      if (a.starts != nullptr && (a.starts[z] < 0 || a.starts[z + 1] < a.starts[z] || a.starts[z + 1] > a.tokens))
        paged_record(a.status, SYN_DEV_BAD_INDEX, z, a.starts[z + 1]);
    }
  }
  long long upto = mine;
  for (int d = 1; d < 32; d <<= 1) {
    const long long o = __shfl_up_sync(~0u, upto, d);
    if (lane >= d) upto += o;
  }
  if (lane == 31) s_sum[warp] = upto;
  __syncthreads();
  long long total = 0;
  for (int w = 0; w < PA_WARPS; ++w) {
    if (w < warp) upto += s_sum[w];
    total += s_sum[w];
  }
  const int shares = static_cast<int>(min(static_cast<long long>(p.grid), max(1LL, total / p.min_tiles)));
  const int block = blockIdx.x;
  const long long t0 = block < shares ? paged_border(total, shares, block) : total;
  const long long t1 = block < shares ? paged_border(total, shares, block + 1) : total;
  if (t0 >= t1) {
    if (tid == 0) *reinterpret_cast<int4*>(p.desc + block * PA_DESC) = make_int4(0, 0, 0, -1);
    return;
  }
  if (upto - mine <= t0 && t0 < upto) {
    long long rest = t0 - (upto - mine);
    int z = z0;
    for (; z < z1; ++z) {
      const PagedRequest r = paged_request<C>(a, z);
      const long long w = static_cast<long long>(r.tiles) * a.Hkv * r.rt;
      if (rest < w) break;
      rest -= w;
    }
    s_z = z;
    s_rest = rest;
  }
  __syncthreads();

  PagedCursor<C> cur;
  cur.at(a, s_z, s_rest);

  // ---- producer: halves of steps (keys, values, keys, ...) are asked for SLOTS - 1 halves ahead, across units
  const uint32_t ring = smem_u32(smem) + warp * C::RING;
  PagedCursor<C> ahead = cur;
  long long t_ahead = t0;
  int page = -2, inside = 0;  // page of key (lane % KEYS) of the next step (-2: no such key), slot in it
  int head_ahead = ahead.sub / ahead.r.rt;
  constexpr int EB = C::E4M3 ? 1 : 2, RPI = 32 / C::CPR == 0 ? 1 : 32 / C::CPR, LOADS = C::HALFB / 512;
  auto look_up = [&]() {
    page = -2;
    if (t_ahead < t1) {
      const int key = ahead.r.first + ahead.tile * C::TILE + warp * C::KEYS + (lane & (C::KEYS - 1));
      if (key < ahead.r.len) {
        const int i = p.page_mul ? __umulhi(key, p.page_mul) >> p.page_shift : key;
        inside = key - i * a.page_size;
        page = i < a.width ? __ldg(a.table + ahead.z * a.table_stride + i) : -1;
      }
    }
  };
  long long off = -2;     // byte offset of this lane's key in the caches (-2: no such key, -1: no such page)
  bool one_page = false;  // the step's keys lie behind one another in one page, all of them there
  auto issue = [&](uint32_t slot, bool values) {
    if (t_ahead < t1) {
      if (!values) {
        off = -2;
        if (page != -2) {
          if (static_cast<unsigned>(page) < static_cast<unsigned>(a.num_pages)) {
            off = (page * a.cache_strides[0] + inside * a.cache_strides[1] + head_ahead * a.cache_strides[2]) * EB;
          } else {
            off = -1;
            paged_record(a.status, SYN_DEV_BAD_INDEX, ahead.z, page);
          }
        }
        const int last = __shfl_sync(~0u, inside, C::KEYS - 1), from = __shfl_sync(~0u, inside, 0);
        one_page = __all_sync(~0u, off >= 0) && last == from + C::KEYS - 1;
        if (one_page)  // a lane's own place: row lane / CPR, chunk lane % CPR
          off = __shfl_sync(~0u, off, 0) + (lane / C::CPR) * a.cache_strides[1] * EB + lane % C::CPR * 16;
      }
      const char* base = static_cast<const char*>(values ? a.v_cache : a.k_cache);
      if (one_page) {
        const char* from = base + off;
        const int64_t skip = RPI * a.cache_strides[1] * EB;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
          const int row = (i * 32 + lane) / C::CPR, chunk = (i * 32 + lane) % C::CPR;
          cp_async16(slot + (values ? ring_at<C, true>(row, chunk) : ring_at<C, false>(row, chunk)), from);
          from += skip;
        }
      } else {
#pragma unroll 2
        for (int i = 0; i < LOADS; ++i) {
          const int row = (i * 32 + lane) / C::CPR, chunk = (i * 32 + lane) % C::CPR;
          const long long o = __shfl_sync(~0u, off, row);
          const uint32_t to = slot + (values ? ring_at<C, true>(row, chunk) : ring_at<C, false>(row, chunk));
          if (o == -1) sts16(to, ~0u, ~0u, ~0u, ~0u);  // no such page: NaN in every type
          else if (o == -2) sts16(to, 0, 0, 0, 0);     // keys behind the end come as zeros
          else cp_async16(to, base + o + chunk * 16);
        }
      }
      if (values) {
        ++t_ahead;
        if (++ahead.tile == ahead.r.tiles) {
          if (t_ahead < t1) ahead.next_unit(a);
          head_ahead = ahead.sub / ahead.r.rt;
        }
        look_up();
      }
    }
    cp_async_commit();
  };
  look_up();
#pragma unroll
  for (int s = 0; s < C::SLOTS - 1; ++s) issue(ring + s * C::HALFB, s & 1);
  // Slot of the half being read; the one read before it is the next to fill.
  int slot = 0;
  auto next_half = [&](bool values) {
    cp_async_wait<C::SLOTS - 2>();
    __syncwarp();
    const uint32_t at = ring + slot * C::HALFB;
    issue(ring + (slot == 0 ? C::SLOTS - 1 : slot - 1) * C::HALFB, (C::SLOTS & 1) ? values : !values);
    if (++slot == C::SLOTS) slot = 0;
    return at;
  };

  const uint32_t q_smem = smem_u32(smem) + PA_WARPS * C::RING;
  float* merge = reinterpret_cast<float*>(smem + PA_WARPS * C::RING + C::SMEM_Q);
  float* s_m = merge + C::SMEM_MERGE / 4;  // [warp][row]
  float* s_l = s_m + PA_WARPS * C::ROWS;
  long long t = t0;
  int parts = 0;       // of the unit that this block comes in in the middle of, from the block before on
  int tail_slot = -1;  // part of the unit that it begins and does not end
  const int z_first = cur.z, sub_first = cur.sub;
  bool first_segment = true;

  while (t < t1) {
    // ---- a unit: rows row0 .. row0 + rows of head kv_head of request z
    const PagedRequest r = cur.r;
    const int kv_head = cur.sub / r.rt, row0 = (cur.sub - kv_head * r.rt) * C::ROWS;
    const int rows = min(C::ROWS, r.n * group - row0);
    const int pos0 = r.len - r.n;
    const int tiles = static_cast<int>(min(static_cast<long long>(r.tiles - cur.tile), t1 - t));
    // This lane's rows: the scores' columns 8 i + 2 t4 + (0, 1) (statistics and output), and 8 i + g (queries).
    // Rows behind the last repeat it.
    int lo[2 * RT], hi[2 * RT];
    float mult[2 * RT];
#pragma unroll
    for (int x = 0; x < 2 * RT; ++x) {
      const int tok = (row0 + min((x >> 1) * 8 + 2 * t4 + (x & 1), rows - 1)) / group;
      hi[x] = a.causal ? min(r.len, pos0 + tok + 1) : r.len;
      lo[x] = a.window > 0 ? max(0, pos0 + tok - a.window + 1) : 0;
      mult[x] = a.sm_scale * CUDART_L2E_F;
      if constexpr (C::E4M3) mult[x] *= a.k_scale[kv_head];
    }
    const T* qrow[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      const int row = row0 + min(8 * i + g, rows - 1), tok = row / group, head = kv_head * group + row - tok * group;
      qrow[i] = static_cast<const T*>(a.q) + static_cast<int64_t>(r.s0 + tok) * a.q_strides[0] + head * a.q_strides[1];
    }
    const int tok_a = row0 / group, tok_b = (row0 + rows - 1) / group;
    const int all_lo = a.window > 0 ? max(0, pos0 + tok_b - a.window + 1) : 0;  // keys that every row sees
    const int all_hi = a.causal ? min(r.len, pos0 + tok_a + 1) : r.len;

    // ---- query fragments
    float up[RT];  // bf16 queries over 8-bit keys: a power of two brings each row into the range of halves
    if constexpr (C::E4M3 && BF16) {
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        uint32_t top = 0;  // largest magnitude as bits
#pragma unroll
        for (int c = 0; c < C::D / 32; ++c) {
          const uint4 x = __ldg(reinterpret_cast<const uint4*>(qrow[i]) + c * 4 + t4);
          const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) top = max(top, max(w[j] & 0x7FFFu, (w[j] >> 16) & 0x7FFFu));
        }
        top = max(top, __shfl_xor_sync(~0u, top, 1));
        top = max(top, __shfl_xor_sync(~0u, top, 2));
        const int e = static_cast<int>(top >> 7);  // biased exponent: the row becomes less than 2^15
        const int shift = e == 0xFF || top == 0 ? 0 : min(max(141 - e, -100), 100);
        up[i] = __uint_as_float(static_cast<uint32_t>(127 + shift) << 23);
        const float down = __uint_as_float(static_cast<uint32_t>(127 - shift) << 23);
#pragma unroll
        for (int c = 0; c < 2; ++c) mult[2 * i + c] *= __shfl_sync(~0u, down, (2 * t4 + c) * 4);
      }
    }
    auto q_frag = [&](int ks, int i, uint32_t (&f)[2]) {
      if constexpr (!C::E4M3) {
        f[0] = __ldg(reinterpret_cast<const uint32_t*>(qrow[i]) + ks * 8 + t4);
        f[1] = __ldg(reinterpret_cast<const uint32_t*>(qrow[i]) + ks * 8 + t4 + 4);
      } else {  // the order in which the 8-bit keys are fetched
        const uint2 v = __ldg(reinterpret_cast<const uint2*>(qrow[i]) + (t4 + ks / 4 * 4) * 4 + ks % 4);
        f[0] = v.x, f[1] = v.y;
        if constexpr (BF16) {
          const float2 x = unpack2<true>(v.x), y = unpack2<true>(v.y);
          f[0] = pack2<false>(x.x * up[i], x.y * up[i]);
          f[1] = pack2<false>(y.x * up[i], y.y * up[i]);
        }
      }
    };
    uint32_t qreg[C::QREG ? C::KSTEPS * RT : 1][2];
    if constexpr (C::QREG) {
#pragma unroll
      for (int ks = 0; ks < C::KSTEPS; ++ks)
#pragma unroll
        for (int i = 0; i < RT; ++i) q_frag(ks, i, qreg[ks * RT + i]);
    } else {
#pragma unroll
      for (int j = 0; j < C::KSTEPS / PA_WARPS; ++j) {
        const int ks = j * PA_WARPS + warp;
#pragma unroll
        for (int i = 0; i < RT; ++i) {
          uint32_t f[2];
          q_frag(ks, i, f);
          asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(q_smem + (ks * RT + i) * 256 + lane * 8), "r"(f[0]), "r"(f[1])
                       : "memory");
        }
      }
      __syncthreads();
    }
    auto q_at = [&](int ks, int i, uint32_t (&f)[2]) {
      if constexpr (C::QREG) {
        f[0] = qreg[ks * RT + i][0], f[1] = qreg[ks * RT + i][1];
      } else {
        const uint2 x = lds8(q_smem + (ks * RT + i) * 256 + lane * 8);
        f[0] = x.x, f[1] = x.y;
      }
    };

    float o[C::DT][RT][4], m[2 * RT], l[2 * RT];
#pragma unroll
    for (int x = 0; x < 2 * RT; ++x) m[x] = -CUDART_INF_F, l[x] = 0.f;
#pragma unroll
    for (int dt = 0; dt < C::DT; ++dt)
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) o[dt][i][c] = 0.f;

    for (int i = 0; i < tiles; ++i) {
      const uint32_t k_at = next_half(false);
      const int base = r.first + (cur.tile + i) * C::TILE + warp * C::KEYS;
      if (base >= r.len) {  // no key of this warp
        next_half(true);
        continue;
      }

      // ---- scores, transposed: 16 keys by 8 rows a product
      constexpr int SN = C::KEYS / 16;
      float s[SN][RT][4];
#pragma unroll
      for (int n = 0; n < SN; ++n)
#pragma unroll
        for (int j = 0; j < RT; ++j)
#pragma unroll
          for (int c = 0; c < 4; ++c) s[n][j][c] = 0.f;
      if constexpr (!C::E4M3) {
        const int row = lane & 15;
#pragma unroll
        for (int ks = 0; ks < C::KSTEPS; ++ks) {
          uint32_t k[4];
          ldsm4(k_at + row * C::ROWB + (((ks * 2 + (lane >> 4)) ^ (row & 7)) << 4), k);
#pragma unroll
          for (int j = 0; j < RT; ++j) {
            uint32_t f[2];
            q_at(ks, j, f);
            mma16816<MBF16>(s[0][j], k, f[0], f[1]);
          }
        }
      } else {
#pragma unroll
        for (int part = 0; part < C::D / 64; ++part) {
          uint32_t f[4][RT][2];
#pragma unroll
          for (int w = 0; w < 4; ++w)
#pragma unroll
            for (int j = 0; j < RT; ++j) q_at(part * 4 + w, j, f[w][j]);
#pragma unroll
          for (int n = 0; n < SN; ++n) {
            const uint4 x = lds16(k_at + ring_at<C, false>(n * 16 + g, t4 + part * 4));
            const uint4 y = lds16(k_at + ring_at<C, false>(n * 16 + 8 + g, t4 + part * 4));
            const uint32_t xw[4] = {x.x, x.y, x.z, x.w}, yw[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              uint32_t k[4];
              e4m3x4_to_h2x2(xw[w], k[0], k[2]);
              e4m3x4_to_h2x2(yw[w], k[1], k[3]);
#pragma unroll
              for (int j = 0; j < RT; ++j) mma16816<false>(s[n][j], k, f[w][j][0], f[w][j][1]);
            }
          }
        }
      }

      // ---- weights
      const bool whole = base >= all_lo && base + C::KEYS <= all_hi;  // every row sees every key
      bool rise = false;
#pragma unroll
      for (int x = 0; x < 2 * RT; ++x)
#pragma unroll
        for (int n = 0; n < SN; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float& v = s[n][x >> 1][2 * h + (x & 1)];
            v *= mult[x];
            const int key = base + n * 16 + h * 8 + g;
            if (!whole && (key < lo[x] || key >= hi[x])) v = -CUDART_INF_F;
            rise |= v > m[x] + PA_SLACK;
          }
      if (__any_sync(~0u, rise)) {
#pragma unroll
        for (int x = 0; x < 2 * RT; ++x) {
          float top = m[x];
#pragma unroll
          for (int n = 0; n < SN; ++n) top = fmaxf(top, fmaxf(s[n][x >> 1][x & 1], s[n][x >> 1][2 + (x & 1)]));
          top = fmaxf(top, __shfl_xor_sync(~0u, top, 4));
          top = fmaxf(top, __shfl_xor_sync(~0u, top, 8));
          top = fmaxf(top, __shfl_xor_sync(~0u, top, 16));
          const float alpha = ex2(m[x] - (top == -CUDART_INF_F ? 0.f : top));
          m[x] = top;
          l[x] *= alpha;
#pragma unroll
          for (int dt = 0; dt < C::DT; ++dt) {
            o[dt][x >> 1][x & 1] *= alpha;
            o[dt][x >> 1][2 + (x & 1)] *= alpha;
          }
        }
      }
#pragma unroll
      for (int x = 0; x < 2 * RT; ++x) {
        const float zero = m[x] == -CUDART_INF_F ? 0.f : m[x];
#pragma unroll
        for (int n = 0; n < SN; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float& v = s[n][x >> 1][2 * h + (x & 1)];
            v = ex2(v - zero);
            l[x] += v;
          }
      }
      const uint32_t v_at = next_half(true);

      // ---- values, transposed: 16 dimensions by 8 rows a product.  The weights enter as two 16-bit numbers, the
      // second one what the first left, so that their rounding does not add to that of the output.
#pragma unroll
      for (int kk = 0; kk < SN; ++kk) {
        uint32_t ph[RT][2], pl[RT][2];
#pragma unroll
        for (int j = 0; j < RT; ++j)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float x = s[kk][j][2 * h], y = s[kk][j][2 * h + 1];
            const uint32_t top = pack2<MBF16>(x, y);
            ph[j][h] = transpose8(top);
            const float2 b = unpack2<MBF16>(top);
            pl[j][h] = transpose8(pack2<MBF16>(x - b.x, y - b.y));
          }
        bool odd = false;  // values that are not finite, at keys that not every row sees
        if (!whole && r.n > 1) {
          constexpr uint32_t EXP = MBF16 ? 0x7F807F80u : 0x7C007C00u, ONE = MBF16 ? 0x00800080u : 0x04000400u;
          each_v<C>(v_at, lane, kk, [&](int, const uint32_t (&v)[4]) {
#pragma unroll
            for (int c = 0; c < 4; ++c) odd |= (((v[c] & EXP) + ONE) & 0x80008000u) != 0;
          });
          odd = __any_sync(~0u, odd);
        }
        if (!odd) {
          each_v<C>(v_at, lane, kk, [&](int dt, const uint32_t (&v)[4]) {
#pragma unroll
            for (int j = 0; j < RT; ++j) {
              mma16816<MBF16>(o[dt][j], v, ph[j][0], ph[j][1]);
              mma16816<MBF16>(o[dt][j], v, pl[j][0], pl[j][1]);
            }
          });
        } else {
          // Zero times infinity: such values may only enter the rows that see them, so one row at a time,
          // with what it does not see taken out.
#pragma unroll
          for (int x = 0; x < 2 * RT; ++x) {
            const int j = x >> 1;
#pragma unroll 1
            for (int q = 0; q < 4; ++q) {  // row 8 j + 2 q + (x & 1), a column of lanes t4 == q
              const int row_lo = __shfl_sync(~0u, lo[x], q), row_hi = __shfl_sync(~0u, hi[x], q);
              const int key = base + kk * 16 + t4 * 2;
              auto seen = [&](int k) {
                return (k >= row_lo && k < row_hi ? 0xFFFFu : 0u) | (k + 1 >= row_lo && k + 1 < row_hi ? 0xFFFF0000u : 0u);
              };
              const uint32_t mask0 = seen(key), mask1 = seen(key + 8);
              each_v<C>(v_at, lane, kk, [&](int dt, const uint32_t (&v)[4]) {
                const uint32_t u[4] = {v[0] & mask0, v[1] & mask0, v[2] & mask1, v[3] & mask1};
                float c[4] = {0.f, 0.f, 0.f, 0.f};
                mma16816<MBF16>(c, u, ph[j][0], ph[j][1]);
                mma16816<MBF16>(c, u, pl[j][0], pl[j][1]);
                if (t4 == q) {
                  o[dt][j][x & 1] += c[x & 1];
                  o[dt][j][2 + (x & 1)] += c[2 + (x & 1)];
                }
              });
            }
          }
        }
      }
    }

    // ---- the warps' parts of the unit are put together
#pragma unroll
    for (int x = 0; x < 2 * RT; ++x) {
      l[x] += __shfl_xor_sync(~0u, l[x], 4);
      l[x] += __shfl_xor_sync(~0u, l[x], 8);
      l[x] += __shfl_xor_sync(~0u, l[x], 16);
      const int row = (x >> 1) * 8 + 2 * t4 + (x & 1);
      if (g == 0) s_m[warp * C::ROWS + row] = m[x], s_l[warp * C::ROWS + row] = l[x];
    }
    __syncthreads();
#pragma unroll
    for (int x = 0; x < 2 * RT; ++x) {
      const int row = (x >> 1) * 8 + 2 * t4 + (x & 1);
      float top = -CUDART_INF_F;
#pragma unroll
      for (int w = 0; w < PA_WARPS; ++w) top = fmaxf(top, s_m[w * C::ROWS + row]);
      const float f = ex2(m[x] - (top == -CUDART_INF_F ? 0.f : top));
#pragma unroll
      for (int dt = 0; dt < C::DT; ++dt) {
        o[dt][x >> 1][x & 1] *= f;
        o[dt][x >> 1][2 + (x & 1)] *= f;
      }
    }
    constexpr int TPR = C::DC / 4;  // threads a row
    static_assert(C::ROWS * TPR <= PA_THREADS, "a thread for every four outputs of a pass");
    const bool writer = tid < C::ROWS * TPR;
    const int row = writer ? tid / TPR : 0, entry = (tid % TPR) * 4;
    float top = -CUDART_INF_F, sum = 0.f;
#pragma unroll
    for (int w = 0; w < PA_WARPS; ++w) top = fmaxf(top, s_m[w * C::ROWS + row]);
#pragma unroll
    for (int w = 0; w < PA_WARPS; ++w) sum += s_l[w * C::ROWS + row] * ex2(s_m[w * C::ROWS + row] - (top == -CUDART_INF_F ? 0.f : top));
    const bool from_start = cur.tile == 0, to_end = cur.tile + tiles == r.tiles, partial = !(from_start && to_end);
    const int part = 2 * block + (first_segment ? 0 : 1);
    const int unit_row = row0 + row, tok = unit_row / group, head = kv_head * group + unit_row - tok * group;
    float factor = 1.f;
    if (!partial) {
      factor = sum == 0.f ? 0.f : 1.f / sum;
      if constexpr (C::E4M3) factor *= a.v_scale[kv_head];
    }
    if (writer && row < rows && entry == 0) {
      if (partial) {
        p.part_ml[(part * C::ROWS + row) * 2] = top;
        p.part_ml[(part * C::ROWS + row) * 2 + 1] = sum;
      } else if (a.lse != nullptr) {
        a.lse[static_cast<int64_t>(r.s0 + tok) * a.Hq + head] = top + log2f(sum);
      }
    }
    T* out = static_cast<T*>(a.o) + static_cast<int64_t>(r.s0 + tok) * a.o_strides[0] + head * a.o_strides[1];
    float* out_part = p.part_o + (static_cast<int64_t>(part) * C::ROWS + row) * C::D;
#pragma unroll
    for (int pass = 0; pass < C::PASSES; ++pass) {
      if (pass > 0) __syncthreads();
#pragma unroll
      for (int x = 0; x < 2 * RT; ++x) {
        const int to_row = (x >> 1) * 8 + 2 * t4 + (x & 1);
        if (to_row < rows) {
          float* to = merge + (warp * C::ROWS + to_row) * C::MERGE_LD;
#pragma unroll
          for (int n = 0; n < C::NT_PASS; ++n) {
            const int nt = pass * C::NT_PASS + n;
            to[merge_entry<C>(n, g)] = o[nt >> 1][x >> 1][2 * (nt & 1) + (x & 1)];
          }
        }
      }
      __syncthreads();
      if (writer && row < rows) {
        float4 v = *reinterpret_cast<const float4*>(merge + row * C::MERGE_LD + entry);
#pragma unroll
        for (int w = 1; w < PA_WARPS; ++w) {
          const float4 u = *reinterpret_cast<const float4*>(merge + (w * C::ROWS + row) * C::MERGE_LD + entry);
          v.x += u.x, v.y += u.y, v.z += u.z, v.w += u.w;
        }
        const int d0 = merge_dim<C>(pass, entry), d1 = merge_dim<C>(pass, entry + 2);
        if (partial) {
          *reinterpret_cast<float2*>(out_part + d0) = make_float2(v.x, v.y);
          *reinterpret_cast<float2*>(out_part + d1) = make_float2(v.z, v.w);
        } else {
          *reinterpret_cast<uint32_t*>(out + d0) = pack2<BF16>(v.x * factor, v.y * factor);
          *reinterpret_cast<uint32_t*>(out + d1) = pack2<BF16>(v.z * factor, v.w * factor);
        }
      }
    }
    __syncthreads();

    // ---- what the join needs to know
    if (first_segment && !from_start) {  // the block that holds the unit's last tile
      const long long end = t + (r.tiles - cur.tile);
      int c = static_cast<int>(min((end * shares - 1) / total, static_cast<long long>(shares - 1)));
      while (c + 1 < shares && paged_border(total, shares, c + 1) < end) ++c;
      while (paged_border(total, shares, c) >= end) --c;
      parts = c - block + 2;
    }
    if (from_start && !to_end) tail_slot = part;
    first_segment = false;
    t += tiles;
    if (t < t1) cur.next_unit(a);
  }
  if (tid == 0) *reinterpret_cast<int4*>(p.desc + block * PA_DESC) = make_int4(parts, z_first, sub_first, tail_slot);
}

// Joins the parts of the units that borders between blocks cut.  The unit that block c comes in in the middle of
// is listed for joining if block c - 1 began it.  Every block reads all descriptions, and rows of listed
// units are dealt out: a unit of many parts (a long request has hundreds) takes a whole block a row, whose warps
// share the parts; one of few takes a warp a row.
constexpr int PA_JOIN_WARPS = 16;
constexpr int PA_JOIN_MAX = 1024;  // blocks of the attention kernel
constexpr int PA_JOIN_MANY = 16;   // parts from which on a row takes a block

template <typename C>
__device__ __forceinline__ void paged_join_store(const PagedAttnParams& p, const PagedRequest& r, int kv_head, int unit_row, int lane,
                                                 const float2 (&v)[C::D / 64], float top, float sum) {
  using T = typename C::type;
  constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
  const syn_paged_attn_args& a = p.a;
  const int group = a.Hq / a.Hkv;
  float factor = sum == 0.f ? 0.f : 1.f / sum;
  if constexpr (C::E4M3) factor *= a.v_scale[kv_head];
  const int tok = unit_row / group, head = kv_head * group + unit_row - tok * group;
  T* out = static_cast<T*>(a.o) + static_cast<int64_t>(r.s0 + tok) * a.o_strides[0] + head * a.o_strides[1];
#pragma unroll
  for (int j = 0; j < C::D / 64; ++j)
    *reinterpret_cast<uint32_t*>(out + j * 64 + lane * 2) = pack2<BF16>(v[j].x * factor, v[j].y * factor);
  if (lane == 0 && a.lse != nullptr) a.lse[static_cast<int64_t>(r.s0 + tok) * a.Hq + head] = top + log2f(sum);
}

template <typename C>
__global__ void __launch_bounds__(PA_JOIN_WARPS * 32) paged_join_kernel(const __grid_constant__ PagedAttnParams p) {
  constexpr int N = C::D / 64;  // pairs of columns a lane
  __shared__ float2 s_o[PA_JOIN_WARPS][C::D / 2];
  __shared__ float s_m[PA_JOIN_WARPS], s_l[PA_JOIN_WARPS];
  __shared__ int16_t s_list[2][PA_JOIN_MAX];
  __shared__ int s_found[2][PA_JOIN_WARPS];
  const syn_paged_attn_args& a = p.a;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int group = a.Hq / a.Hkv;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  int count[2] = {0, 0};
  for (int c0 = 1; c0 < p.grid; c0 += PA_JOIN_WARPS * 32) {  // in the order of the blocks: all have the same lists
    const int c = c0 + threadIdx.x;
    bool listed = false, many = false;
    if (c < p.grid) {
      const int parts = p.desc[c * PA_DESC];
      listed = parts > 0 && p.desc[(c - 1) * PA_DESC + 3] >= 0;
      many = parts >= PA_JOIN_MANY;
    }
    const unsigned mask[2] = {__ballot_sync(~0u, listed && many), __ballot_sync(~0u, listed && !many)};
    __syncthreads();
    if (lane < 2) s_found[lane][warp] = __popc(mask[lane]);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      int at = count[k];
      for (int w = 0; w < PA_JOIN_WARPS; ++w) {
        if (w < warp) at += s_found[k][w];
        count[k] += s_found[k][w];
      }
      if (listed && many == (k == 0)) s_list[k][at + __popc(mask[k] & ((1u << lane) - 1))] = static_cast<int16_t>(c);
    }
  }
  __syncthreads();
#pragma unroll 1
  for (int k = 0; k < 2; ++k) {
    const int wide = k == 0 ? PA_JOIN_WARPS : 1;  // warps a row
    const int share = k == 0 ? warp : 0;
    const int items = count[k] * C::ROWS;
    const int from = k == 0 ? blockIdx.x : blockIdx.x * PA_JOIN_WARPS + warp;
    const int skip = k == 0 ? gridDim.x : gridDim.x * PA_JOIN_WARPS;
    for (int item = from; item < items; item += skip) {
      const int c = s_list[k][item / C::ROWS], row = item % C::ROWS;
      const int4 d = *reinterpret_cast<const int4*>(p.desc + c * PA_DESC);
      const int before = p.desc[(c - 1) * PA_DESC + 3], parts = d.x;
      const PagedRequest r = paged_request<C>(a, d.y);
      const int kv_head = d.z / r.rt, row0 = (d.z - kv_head * r.rt) * C::ROWS;
      if (row >= r.n * group - row0) continue;
      auto slot = [&](int i) { return i == 0 ? before : 2 * (c - 1 + i); };
      float top = -CUDART_INF_F, sum = 0.f;
      float2 v[N];
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] = make_float2(0.f, 0.f);
      for (int i0 = share; i0 < parts; i0 += 32 * wide) {  // a part's statistics a lane, then one part after the other
        const int i = i0 + lane * wide;
        float2 ml = make_float2(-CUDART_INF_F, 0.f);
        if (i < parts) ml = *reinterpret_cast<const float2*>(p.part_ml + (static_cast<int64_t>(slot(i)) * C::ROWS + row) * 2);
        float now = fmaxf(top, ml.x);
        for (int d = 16; d > 0; d >>= 1) now = fmaxf(now, __shfl_xor_sync(~0u, now, d));
        const float zero = now == -CUDART_INF_F ? 0.f : now, alpha = ex2(top - zero);
        top = now;
        const float w = ex2(ml.x - zero);
        float more = ml.y * w;
        for (int d = 16; d > 0; d >>= 1) more += __shfl_xor_sync(~0u, more, d);
        sum = sum * alpha + more;
#pragma unroll
        for (int j = 0; j < N; ++j) v[j].x *= alpha, v[j].y *= alpha;
        const int count = min(32, (parts - i0 + wide - 1) / wide);
#pragma unroll 8
        for (int q = 0; q < count; ++q) {
          const float f = __shfl_sync(~0u, w, q);
          const float* at = p.part_o + (static_cast<int64_t>(slot(i0 + q * wide)) * C::ROWS + row) * C::D + lane * 2;
#pragma unroll
          for (int j = 0; j < N; ++j) {
            const float2 u = *reinterpret_cast<const float2*>(at + j * 64);
            v[j].x += u.x * f, v[j].y += u.y * f;
          }
        }
      }
      if (k == 0) {
        __syncthreads();
        if (lane == 0) s_m[warp] = top, s_l[warp] = sum;
#pragma unroll
        for (int j = 0; j < N; ++j) s_o[warp][j * 32 + lane] = v[j];
        __syncthreads();
        if (warp > 0) continue;
        for (int w = 1; w < PA_JOIN_WARPS; ++w) top = fmaxf(top, s_m[w]);
        const float zero = top == -CUDART_INF_F ? 0.f : top;
        sum = 0.f;
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = make_float2(0.f, 0.f);
        for (int w = 0; w < PA_JOIN_WARPS; ++w) {
          const float f = ex2(s_m[w] - zero);
          sum += s_l[w] * f;
#pragma unroll
          for (int j = 0; j < N; ++j) {
            const float2 u = s_o[w][j * 32 + lane];
            v[j].x += u.x * f, v[j].y += u.y * f;
          }
        }
      }
      paged_join_store<C>(p, r, kv_head, row0 + row, lane, v, top, sum);
    }
  }
}

}  // namespace syn
