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
//   * Every warp is a worker of its own: it streams its keys and values through a ring of its own in shared memory
//     (cp.async of 16 bytes, a page lookup a step), with no barrier between the warps of a block on the way.
//   * The work (requests x key-value heads x row tiles x steps of keys) is laid out in one line and cut into
//     equal shares for the warps of a grid that fills the GPU, whatever the lengths; loads run on across the
//     borders of units.  Where a head is less than 256 bytes and the heads of a token lie side by side, two or
//     four warps take neighbouring heads at the same keys (`tracks`): HBM answers 128 bytes here and there a
//     tenth slower than 256 side by side, 64 bytes a third.  A unit that a border cuts leaves partial results, which a second small kernel joins
//     in a fixed order (the warps of a block that work on one and the same unit join theirs first): results do
//     not depend on timing, there are no atomics and no state between calls.
#pragma once
#include <float.h>
#include <math_constants.h>

#include <type_traits>

#include "paged.cuh"

namespace syn {

constexpr int PA_WARPS = 4;
constexpr int PA_THREADS = PA_WARPS * 32;
// The reference a row's weights are taken against (m) follows its maximum only when that has risen by more
// than PA_SLACK powers of two: a vote without shuffles on most steps, and few rescales.  Weights stay below 2^8.
constexpr float PA_SLACK = 8.f;
// Halves hold all bits of numbers from 2^-14 to 2^16, so weights that may enter products of halves are taken against
// a reference that lies 2^11 below and follows sooner: they stay below 2^15, a row's largest is 2^11 or more, and from
// PA_SMALL on two halves hold 17 bits.  A step with smaller ones takes the products of PAIR_TF32.
constexpr float PA_SLACK_HALF = 4.f, PA_BIAS = 11.f, PA_SMALL = 0x1p-8f;
constexpr float PA_NONE = -1e30f;  // reference of a row without a key so far
constexpr int PA_DESC = 12;  // int32 words a worker leaves for the join (PagedJoin)

struct PagedAttnParams {
  syn_paged_attn_args a;
  int32_t grid;       // blocks of the launch
  int32_t min_steps;  // fewest steps worth a worker
  int32_t tracks;     // neighbouring heads that as many warps of a block take at the same keys (1, 2 or 4)
  uint32_t page_mul;  // key / page_size = mulhi(key, page_mul) >> page_shift (page_mul 0: pages of one key)
  int32_t page_shift;
  float* part_o;      // [2 * warps][fragments of the output: D / 16, 8-row tiles][lanes][4]
  float* part_ml;     // [2 * warps][rows of a unit][2]
  int32_t* desc;      // [warps][PA_DESC]
};

// A unit that borders cut, as left by the second worker on it.  Its parts in order: `n1` of single workers (the
// first in slot `slot1`, then slot 2 w of the workers that follow worker w1), `n2` of blocks (slot 2 wide b of
// block b2 and those that follow), `n3` of single workers (from w3 on); `wide` workers a block.  With tracks
// those are slots of a track.
struct alignas(16) PagedJoin {
  int n1, slot1, w1;
  int n2, b2, wide;
  int n3, w3;
  int s0, kv_head, row0, rows;
  __device__ __forceinline__ int parts() const { return n1 + n2 + n3; }
  __device__ __forceinline__ int slot(int i) const {
    int at;
    if (i < n1) at = i == 0 ? slot1 : 2 * (w1 + i);
    else if (i < n1 + n2) at = 2 * wide * (b2 + i - n1);
    else at = 2 * (w3 + i - n1 - n2);
    const int tracks = PA_WARPS / wide;
    return at * tracks + kv_head % tracks;
  }
};
static_assert(sizeof(PagedJoin) == PA_DESC * 4, "PagedJoin");

template <typename T, bool E4M3_, int D_, int RT_>
struct PagedCfg {
  using type = T;
  static constexpr bool E4M3 = E4M3_;
  static constexpr int D = D_;
  static constexpr int RT = RT_;                     // 8-row tiles of a unit
  static constexpr int ROWS = 8 * RT;
  static constexpr int KEYS = E4M3 ? 32 : 16;        // keys of a warp's step
  static constexpr int ROWB = D * (E4M3 ? 1 : 2);    // bytes of a stored head
  static constexpr int CPR = ROWB / 16;              // 16-byte chunks of it
  static constexpr int HALFB = KEYS * ROWB;          // the keys of a step, or its values
  // Blocks on an SM and halves in a ring: as many bytes on the way as shared memory holds, and the registers that the
  // output leaves.  8 rows: three blocks of four slots; with four of three too little is on the way (2500-token
  // requests 126 us against 115).  16 rows: two blocks where three leave too few registers (D = 128: 117 against
  // 136), three where they do not (D = 64: 79 against 102).
  static constexpr int BLOCKS = D == 256 ? 3 - RT : RT == 1 || (RT == 2 && D == 64) ? 3 : 2;
  static constexpr int SLOTS = D == 256 ? 3 : D == 128 ? (RT == 1 ? 4 : 5) : (RT <= 2 ? 8 : 10);
  static constexpr int RING = SLOTS * HALFB;         // bytes a warp
  static constexpr bool QREG = RT * D <= 256;        // query fragments in registers, else in shared memory
  static constexpr int KSTEPS = D / 16;
  static constexpr int DT = D / 16;                  // 16-dimension tiles of the output
  static constexpr int FRAGS = DT * RT;              // output fragments of a unit, four numbers a lane
  static constexpr int QB = QREG ? 0 : KSTEPS * RT * 256;
  static constexpr int SMEM = PA_WARPS * (RING + QB);
  static_assert(BLOCKS * (SMEM + 1280) <= 228 * 1024, "shared memory of an SM");
  static_assert(RING >= FRAGS * 512 + RT * 512, "the parts of a pooled block");
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
// TF32: numbers of 32 bits whose lower 13 are 0.
__device__ __forceinline__ void mma1688_tf32(float (&c)[4], const float (&a)[4], float b0, float b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(__float_as_uint(a[0])), "r"(__float_as_uint(a[1])), "r"(__float_as_uint(a[2])), "r"(__float_as_uint(a[3])),
        "r"(__float_as_uint(b0)), "r"(__float_as_uint(b1)));
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
  int pos0;        // position of the first row, by length and border as they are given: rows behind the table stay
                   // behind it, and rows that q does not have do not move those that it has
  int first;       // first key that any row sees
  int steps, rt;   // steps of a unit; row tiles a head
};

// First key that the window leaves to position `at`; the key that stands for those behind the table is left to every
// position behind it, which so becomes NaN.
__device__ __forceinline__ int paged_window_from(const syn_paged_attn_args& a, int len, int at) {
  return min(at - a.window + 1, len - 1);
}

template <typename C>
__device__ __forceinline__ PagedRequest paged_request(const syn_paged_attn_args& a, int z) {
  PagedRequest r;
  r.s0 = z, r.n = 1;
  int end = z + 1;  // behind the request's last row
  if (a.starts != nullptr) {
    r.s0 = min(max(a.starts[z], 0), a.tokens);
    end = max(a.starts[z + 1], r.s0);
    r.n = min(end, a.tokens) - r.s0;
  }
  // One key too many stands for all that the table has no room for (the host keeps the room below 2^31 - 64).
  const int room = a.width * a.page_size, len = max(a.lens[z], 0);
  r.len = min(len, room + 1);
  r.pos0 = max(len - (end - r.s0), -a.tokens);  // (a row at a position below 0 sees nothing)
  r.first = a.window > 0 ? max(0, paged_window_from(a, r.len, r.pos0)) : 0;
  r.steps = max(1, (r.len - r.first + C::KEYS - 1) / C::KEYS);
  r.rt = (r.n * (a.Hq / a.Hkv) + C::ROWS - 1) / C::ROWS;
  return r;
}

// The line cut into `shares` pieces: the first `more` of them have one step more than the others.
struct PagedCut {
  long long each;
  int shares, more;
  __device__ __forceinline__ PagedCut(long long total, int shares_) : shares(shares_) {
    each = total <= UINT_MAX ? static_cast<uint32_t>(total) / static_cast<uint32_t>(shares) : total / shares;
    more = static_cast<int>(total - each * shares);
  }
  __device__ __forceinline__ long long at(int c) const { return c * each + min(c, more); }  // where piece c begins
  __device__ __forceinline__ int piece(long long step) const {  // the piece that a step lies in
    const long long longer = more * (each + 1);
    return step < longer ? quotient(step, each + 1) : more + quotient(step - longer, each);
  }
  static __device__ __forceinline__ int quotient(long long n, long long d) {
    return static_cast<int>(n <= UINT_MAX ? static_cast<uint32_t>(n) / static_cast<uint32_t>(d) : n / d);
  }
};

// Position on the line: step `step` of unit `sub` (head * row tiles + row tile) of request z.
template <typename C>
struct PagedCursor {
  int z, sub, step;
  PagedRequest r;

  __device__ __forceinline__ void at(const syn_paged_attn_args& a, int z_, long long rest) {
    z = z_;
    r = paged_request<C>(a, z);
    sub = static_cast<int>(rest / r.steps);
    step = static_cast<int>(rest % r.steps);
  }
  // To the first step of the next unit; the caller knows that there is one.
  __device__ __forceinline__ void next_unit(const syn_paged_attn_args& a, int heads) {
    step = 0;
    if (++sub < heads * r.rt) return;
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
    const uint32_t at = v + ((lane & 7) + (lane >> 4) * 8) * C::ROWB + ((((lane >> 3) & 1) ^ (lane & 7)) << 4);
#pragma unroll
    for (int j = 0; j < C::DT; ++j) {
      uint32_t a[4];
      ldsm4t((at ^ (j % 4 * 32)) + j / 4 * 128, a);
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

// The weights of an 8-row tile at 16 keys, from the scores' fragment (keys by rows) to the values' products: each as two
// numbers of fewer bits, the second one what the first left, so that their rounding does not add to that of the output.
//   bf16 values: two bf16, 16 bits.
//   Halves, 8-bit values among them: two halves, 17 bits, where no weight of the step is smaller than those hold; else
//   two TF32, 20 bits of any weight.  Small weights count: where a key takes the weight and its values are small, the
//   output is made of the others.  All steps in TF32: 96 requests on an 8-bit cache 250 us against 222, drafts in fp16
//   88 against 82, 32 rows 470 against 376.  Scores that spread by tens of powers of two, nearly all steps in TF32: one
//   token a request 219 (8 bits) and 118 (fp16) against 217 and 116 for scores that do not, 32 rows 516 against 376.
enum PagedKind { PAIR_BF16, PAIR_F16, PAIR_TF32 };
template <PagedKind K>
struct PagedWeights {
  uint32_t hi[2], lo[2];
  __device__ __forceinline__ void set(const float (&w)[4]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t top = pack2<K == PAIR_BF16>(w[2 * h], w[2 * h + 1]);
      hi[h] = transpose8(top);
      const float2 b = unpack2<K == PAIR_BF16>(top);
      lo[h] = transpose8(pack2<K == PAIR_BF16>(w[2 * h] - b.x, w[2 * h + 1] - b.y));
    }
  }
};

template <>
struct PagedWeights<PAIR_TF32> {
  float hi[2][2], lo[2][2];  // [8 keys each][key 2 t4, 2 t4 + 1] of row g
  __device__ __forceinline__ void set(const float (&w)[4]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t x = __float_as_uint(w[2 * h]), y = __float_as_uint(w[2 * h + 1]);
      const uint32_t top = transpose8(__byte_perm(x, y, 0x7632)), low = transpose8(__byte_perm(x, y, 0x5410));
      const uint32_t z[2] = {__byte_perm(low, top, 0x5410), __byte_perm(low, top, 0x7632)};
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        hi[h][i] = __uint_as_float(z[i] & 0xFFFFE000u);
        lo[h][i] = __uint_as_float(__float_as_uint(__uint_as_float(z[i]) - hi[h][i]) & 0xFFFFE000u);
      }
    }
  }
};

// A fragment of the values (16 dimensions by 16 keys) and its product with weights.
template <PagedKind K>
struct PagedValues {
  const uint32_t (&v)[4];
  __device__ __forceinline__ explicit PagedValues(const uint32_t (&v_)[4]) : v(v_) {}
  __device__ __forceinline__ void times(float (&c)[4], const PagedWeights<K>& w) const {
    mma16816<K == PAIR_BF16>(c, v, w.hi[0], w.hi[1]);
    mma16816<K == PAIR_BF16>(c, v, w.lo[0], w.lo[1]);
  }
};

template <>
struct PagedValues<PAIR_TF32> {
  float v[2][4];  // of 8 keys each: the even keys of dimensions g and g + 8, the odd ones (an order that the weights share)
  __device__ __forceinline__ explicit PagedValues(const uint32_t (&u)[4]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float2 x = unpack2<false>(u[2 * h]), y = unpack2<false>(u[2 * h + 1]);
      v[h][0] = x.x, v[h][1] = y.x, v[h][2] = x.y, v[h][3] = y.y;
    }
  }
  __device__ __forceinline__ void times(float (&c)[4], const PagedWeights<PAIR_TF32>& w) const {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      mma1688_tf32(c, v[h], w.hi[h][0], w.hi[h][1]);
      mma1688_tf32(c, v[h], w.lo[h][0], w.lo[h][1]);
    }
  }
};

// Keys from .. to - 1 are seen from position `at` of a request.
__device__ __forceinline__ int paged_seen_from(const syn_paged_attn_args& a, int len, int at) {
  return a.window > 0 ? paged_window_from(a, len, at) : 0;
}
__device__ __forceinline__ int paged_seen_to(const syn_paged_attn_args& a, int len, int at) {
  return a.causal ? min(len, at + 1) : len;
}

// Values that are not finite, at keys that only some rows see.  Zero times infinity: they may only enter the rows that see
// them, so these groups of 16 keys (set in `groups`, the step's first key is `base`) are taken one row at a time, with what
// it does not see taken out.  A function of its own, whose operands go through memory: inlined, its registers cost the steps
// without such values (32 rows, 8-bit cache, all steps in TF32: 624 us against 468).
template <typename C>
struct alignas(16) PagedOdd {
  float o[C::DT][C::RT][4], w[C::KEYS / 16][C::RT][4];
  int pos[2 * C::RT];
};
template <typename C>
__device__ __noinline__ void paged_odd(PagedOdd<C>& x, uint32_t v_at, int base, uint32_t groups, const syn_paged_attn_args& a, int len) {
  constexpr bool MBF16 = std::is_same<typename C::type, __nv_bfloat16>::value && !C::E4M3;
  constexpr PagedKind K = MBF16 ? PAIR_BF16 : PAIR_TF32;
  const int lane = threadIdx.x & 31, t4 = lane & 3;
#pragma unroll 1
  for (int kk = 0; kk < C::KEYS / 16; ++kk) {
    if ((groups >> kk & 1) == 0) continue;
#pragma unroll 1
    for (int row = 0; row < C::ROWS; ++row) {  // column row % 2 of the lanes with t4 == row % 8 / 2
      const int j = row >> 3, at = __shfl_sync(~0u, x.pos[2 * j + (row & 1)], row >> 1 & 3);
      const int from = paged_seen_from(a, len, at), to = paged_seen_to(a, len, at), key = base + kk * 16 + t4 * 2;
      auto seen = [&](int k) { return (k >= from && k < to ? 0xFFFFu : 0u) | (k + 1 >= from && k + 1 < to ? 0xFFFF0000u : 0u); };
      const uint32_t mask0 = seen(key), mask1 = seen(key + 8);
      PagedWeights<K> w;
      w.set(x.w[kk][j]);
      each_v<C>(v_at, lane, kk, [&](int dt, const uint32_t (&v)[4]) {
        const uint32_t u[4] = {v[0] & mask0, v[1] & mask0, v[2] & mask1, v[3] & mask1};
        float c[4] = {0.f, 0.f, 0.f, 0.f};
        PagedValues<K>(u).times(c, w);
        if (t4 == (row >> 1 & 3)) {
          x.o[dt][j][row & 1] += row & 1 ? c[1] : c[0];
          x.o[dt][j][2 + (row & 1)] += row & 1 ? c[3] : c[2];
        }
      });
    }
  }
}

// Place of 16-byte chunk `chunk` of row `row` in a half of a warp's ring: chunks change places within 128 bytes
// so that the reads above and those of the keys below meet no bank twice (D = 64 in 8 bits reads its values two
// deep).  Halves are aligned to 128 bytes, so a change of chunk is an exclusive or with the address.  (Rows 16 bytes
// apart instead cost the copies into shared memory more than the plainer addresses gave: 585 against 549 us on
// 3.5 GB of 16-bit keys and values.)
template <typename C, bool VALUES>
__device__ __forceinline__ uint32_t ring_at(int row, int chunk) {
  int c = chunk;
  if constexpr (!C::E4M3) c ^= row & 7;
  else if constexpr (VALUES) c ^= C::D == 64 ? (row >> 1) & 3 : ((row >> 1) & 3) << 1;
  else if constexpr (C::D != 64) c ^= (row & 1) << 2;
  return row * C::ROWB + (c << 4);
}
// The same for the chunk that lane `lane` brings in its i-th turn, row i * (32 / CPR) + lane / CPR, given its place
// in turn 0: `own` = ring_at(lane / CPR, lane % CPR).
template <typename C, bool VALUES>
__device__ __forceinline__ uint32_t ring_turn(uint32_t own, int i) {
  constexpr int RPI = 32 / C::CPR;
  const int row = i * RPI;  // shares no bit with lane / CPR
  int flip = 0;
  if constexpr (!C::E4M3) flip = row & 7;
  else if constexpr (VALUES) flip = C::D == 64 ? (row >> 1) & 3 : ((row >> 1) & 3) << 1;
  else if constexpr (C::D != 64) flip = (row & 1) << 2;
  return (own ^ (flip << 4)) + row * C::ROWB;
}

__device__ __forceinline__ void paged_lse(const syn_paged_attn_args& a, int s0, int kv_head, int unit_row, float m, float l) {
  const int group = a.Hq / a.Hkv, tok = unit_row / group;
  if (a.lse != nullptr) a.lse[static_cast<int64_t>(s0 + tok) * a.Hq + kv_head * group + unit_row - tok * group] = m + log2f(l);
}

// Writes rows (8 rows of tile j, those below `rows`) of COUNT output fragments from fragment tile `dt` on, which hold
// dimensions by rows, times `factor` of the lane's two rows.
template <typename C, int COUNT>
__device__ __forceinline__ void store_frags(const syn_paged_attn_args& a, const float (&o)[COUNT][4], int dt, const float (&factor)[2],
                                            int s0, int kv_head, int unit_row, int rows, int lane) {
  using T = typename C::type;
  constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
  const int g = lane >> 2, t4 = lane & 3, group = a.Hq / a.Hkv;
  auto out_row = [&](int row) {
    const int tok = (unit_row + row) / group, head = kv_head * group + unit_row + row - tok * group;
    return static_cast<T*>(a.o) + static_cast<int64_t>(s0 + tok) * a.o_strides[0] + head * a.o_strides[1];
  };
  if constexpr (!C::E4M3) {  // turned back 8 x 8: lane (g, t4) then has dimensions 2 t4, 2 t4 + 1 of row g
    T* out = out_row(min(g, rows - 1)) + dt * 16 + 2 * t4;
#pragma unroll
    for (int i = 0; i < COUNT; ++i) {
      const uint32_t x = transpose8(pack2<BF16>(o[i][0] * factor[0], o[i][1] * factor[1]));
      const uint32_t y = transpose8(pack2<BF16>(o[i][2] * factor[0], o[i][3] * factor[1]));
      if (g < rows) {
        *reinterpret_cast<uint32_t*>(out + i * 16) = x;
        *reinterpret_cast<uint32_t*>(out + i * 16 + 8) = y;
      }
    }
  } else {  // the halves of a fragment are neighbours
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      if (2 * t4 + c < rows) {
        T* out = out_row(2 * t4 + c);
#pragma unroll
        for (int i = 0; i < COUNT; ++i) {
          const int nt = 2 * (dt + i), d = C::D == 64 ? 8 * g + nt : (nt / 16) * 128 + 16 * g + nt % 16;
          *reinterpret_cast<uint32_t*>(out + d) = pack2<BF16>(o[i][c] * factor[c], o[i][2 + c] * factor[c]);
        }
      }
    }
  }
}

// Rows of COUNT output fragments whose sums are complete: divided, stored, and their log-sum-exp with the first.
template <typename C, int COUNT>
__device__ __forceinline__ void paged_finish(const syn_paged_attn_args& a, const float (&o)[COUNT][4], const float (&m)[2],
                                             const float (&l)[2], int dt, int s0, int kv_head, int unit_row, int rows, int lane) {
  float factor[2];
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const int row = 2 * (lane & 3) + c;
    factor[c] = l[c] == 0.f ? 0.f : 1.f / l[c];
    if constexpr (C::E4M3) factor[c] *= a.v_scale[kv_head];
    if (dt == 0 && lane < 4 && row < rows) paged_lse(a, s0, kv_head, unit_row + row, m[c], l[c]);
  }
  store_frags<C, COUNT>(a, o, dt, factor, s0, kv_head, unit_row, rows, lane);
}

// Output fragments of parts of a unit's keys, joined one after the other.
template <int N>
struct PagedSum {
  float m[2], l[2], o[N][4];
  __device__ __forceinline__ void clear() {
    m[0] = m[1] = -CUDART_INF_F, l[0] = l[1] = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c) o[i][c] = 0.f;
  }
  __device__ __forceinline__ void add(const float4& ml, const float4 (&u)[N]) {
    const float um[2] = {ml.x, ml.z}, ul[2] = {ml.y, ml.w};
    float mine[2], other[2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const float top = fmaxf(m[c], um[c]), zero = top == -CUDART_INF_F ? 0.f : top;
      mine[c] = ex2(m[c] - zero), other[c] = ex2(um[c] - zero);
      m[c] = top;
      l[c] = l[c] * mine[c] + ul[c] * other[c];
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      o[i][0] = o[i][0] * mine[0] + u[i].x * other[0];
      o[i][1] = o[i][1] * mine[1] + u[i].y * other[1];
      o[i][2] = o[i][2] * mine[0] + u[i].z * other[0];
      o[i][3] = o[i][3] * mine[1] + u[i].w * other[1];
    }
  }
};

template <typename C>
__global__ void __launch_bounds__(PA_THREADS, C::BLOCKS) paged_attn_kernel(const __grid_constant__ PagedAttnParams p) {
  using T = typename C::type;
  constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr bool MBF16 = BF16 && !C::E4M3;  // type of the matrix products: 8-bit values are halves there
  constexpr float BIAS = MBF16 ? 0.f : PA_BIAS, RISE = MBF16 ? PA_SLACK : PA_SLACK_HALF + PA_BIAS;
  constexpr int RT = C::RT;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ long long s_sum[PA_WARPS], s_rest[PA_WARPS];
  __shared__ int s_z[PA_WARPS];
  const syn_paged_attn_args& a = p.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
  const int group = a.Hq / a.Hkv;
  // Workers are teams of `tracks` warps, a warp for a track: head sub / rt * tracks + track.  On the line a group of
  // `tracks` heads counts as one.
  const int heads = a.Hkv / p.tracks, wide = PA_WARPS / p.tracks, team = warp / p.tracks, track = warp % p.tracks;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // ---- this warp's share of the line
  const int per = (a.requests + PA_THREADS - 1) / PA_THREADS;
  const int z0 = min(tid * per, a.requests), z1 = min(z0 + per, a.requests);
  long long mine = 0;
  for (int z = z0; z < z1; ++z) {
    const PagedRequest r = paged_request<C>(a, z);
    mine += static_cast<long long>(r.steps) * heads * r.rt;
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
  const int shares = static_cast<int>(min(static_cast<long long>(p.grid) * wide, max(1LL, total / p.min_steps)));
  const PagedCut cut(total, shares);
#pragma unroll
  for (int w = 0; w < PA_WARPS; ++w) {
    const int share = blockIdx.x * wide + w;
    const long long from = w < wide && share < shares ? cut.at(share) : total;
    if (upto - mine <= from && from < upto) {
      long long rest = from - (upto - mine);
      int z = z0;
      for (; z < z1; ++z) {
        const PagedRequest r = paged_request<C>(a, z);
        const long long n = static_cast<long long>(r.steps) * heads * r.rt;
        if (rest < n) break;
        rest -= n;
      }
      s_z[w] = z;
      s_rest[w] = rest;
    }
  }
  __syncthreads();  // from here on the warps go their own ways
  // Every warp has a record: those without work one of nothing to join.
  int32_t* const record = p.desc + (blockIdx.x * PA_WARPS + warp) * PA_DESC;
  const int worker = blockIdx.x * wide + team;
  const bool works = worker < shares;
  const long long t0 = works ? cut.at(worker) : total;
  const long long t1 = works ? cut.at(worker + 1) : total;
  PagedJoin join;
  join.n1 = join.n2 = join.n3 = 0;
  auto nothing_to_join = [&]() {
    for (int i = 0; i < 2; ++i) reinterpret_cast<int4*>(record)[i] = make_int4(0, 0, 0, 0);  // the counts are in these
  };
  if (t0 >= t1) {
    if (lane == 0) nothing_to_join();
    return;
  }

  PagedCursor<C> cur;
  cur.at(a, s_z[team], s_rest[team]);
  const long long unit0 = t0 - cur.step, unit1 = unit0 + cur.r.steps;  // the first unit, on the line
  // A block all of whose shares lie in one unit joins its warps' parts itself.
  auto pooled = [&](int block) {
    return wide > 1 && cut.at(block * wide) >= unit0 &&
           cut.at(min((block + 1) * wide, shares)) <= unit1;
  };
  const bool pool = pooled(blockIdx.x);
  if (worker > 0 && cur.step > 0 && cut.at(worker - 1) <= unit0) {  // the second worker on the unit
    const int first = worker - 1, b_first = first / wide;
    const int last = cut.piece(unit1 - 1), b_last = last / wide;
    const bool pool_first = pooled(b_first), pool_last = pooled(b_last);
    join.slot1 = 2 * first + (cut.at(first) != unit0), join.w1 = first;
    join.wide = wide, join.w3 = b_last * wide;
    if (b_first == b_last) {
      join.n1 = pool_first ? 0 : last - first + 1;  // pooled: the block has the whole unit
      join.b2 = 0;
    } else {
      join.n1 = pool_first ? 0 : (b_first + 1) * wide - first;
      join.b2 = pool_first ? b_first : b_first + 1;
      join.n2 = (pool_last ? b_last + 1 : b_last) - join.b2;
      join.n3 = pool_last ? 0 : last - join.w3 + 1;
    }
    const int head = cur.sub / cur.r.rt;
    join.s0 = cur.r.s0, join.kv_head = head * p.tracks + track, join.row0 = (cur.sub - head * cur.r.rt) * C::ROWS;
    join.rows = min(C::ROWS, cur.r.n * group - join.row0);
  }
  if (lane == 0) {
    if (join.parts() > 0) *reinterpret_cast<PagedJoin*>(record) = join;
    else nothing_to_join();
  }

  // ---- producer: halves of steps (keys, values, keys, ...) are asked for SLOTS - 1 halves ahead, across units
  const uint32_t ring = smem_u32(smem) + warp * C::RING;
  PagedCursor<C> ahead = cur;
  int left = static_cast<int>(t1 - t0);  // steps that are yet to be asked for
  int page = -2, inside = 0;  // page of key (lane % KEYS) of the next step (-2: no such key), slot in it
  int head_ahead = ahead.sub / ahead.r.rt * p.tracks + track;
  constexpr int EB = C::E4M3 ? 1 : 2, RPI = 32 / C::CPR, LOADS = C::KEYS / RPI;
  auto look_up = [&]() {
    page = -2;
    if (left > 0) {
      const int key = ahead.r.first + ahead.step * C::KEYS + (lane & (C::KEYS - 1));
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
    if (left > 0) {
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
        const uint32_t own = slot + (values ? ring_at<C, true>(lane / C::CPR, lane % C::CPR) : ring_at<C, false>(lane / C::CPR, lane % C::CPR));
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
          cp_async16(values ? ring_turn<C, true>(own, i) : ring_turn<C, false>(own, i), from);
          from += skip;
        }
      } else {
#pragma unroll 2
        for (int i = 0; i < LOADS; ++i) {
          const int row = i * RPI + lane / C::CPR, chunk = lane % C::CPR;
          const long long o = __shfl_sync(~0u, off, row);
          const uint32_t to = slot + (values ? ring_at<C, true>(row, chunk) : ring_at<C, false>(row, chunk));
          if (o == -1) sts16(to, ~0u, ~0u, ~0u, ~0u);  // no such page: NaN in every type
          else if (o == -2) sts16(to, 0, 0, 0, 0);     // keys behind the end come as zeros
          else cp_async16(to, base + o + chunk * 16);
        }
      }
      if (values) {
        --left;
        if (++ahead.step == ahead.r.steps) {
          if (left > 0) ahead.next_unit(a, heads);
          head_ahead = ahead.sub / ahead.r.rt * p.tracks + track;
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
  auto ready = [&]() {
    cp_async_wait<C::SLOTS - 2>();
    __syncwarp();
    return ring + slot * C::HALFB;
  };
  auto refill = [&](bool values) {  // `values`: what the half being read holds
    issue(ring + (slot == 0 ? C::SLOTS - 1 : slot - 1) * C::HALFB, (C::SLOTS & 1) ? values : !values);
    if (++slot == C::SLOTS) slot = 0;
  };

  const uint32_t q_smem = smem_u32(smem) + PA_WARPS * C::RING + warp * C::QB;
  long long t = t0;
  bool first_segment = true;

  while (t < t1) {
    // ---- a unit: rows row0 .. row0 + rows of head kv_head of request z
    const PagedRequest r = cur.r;
    const int head_group = cur.sub / r.rt, kv_head = head_group * p.tracks + track, row0 = (cur.sub - head_group * r.rt) * C::ROWS;
    const int rows = min(C::ROWS, r.n * group - row0);
    const int pos0 = r.pos0;
    const bool one = r.n == 1;  // one new token: spares the divisions
    const bool newest = one && pos0 >= r.len - 1;  // its only row sees whatever is loaded (behind the end: zeros)
    const int steps = static_cast<int>(min(static_cast<long long>(r.steps - cur.step), t1 - t));
    // This lane's rows: the scores' columns 8 i + 2 t4 + (0, 1) (statistics and output), and 8 i + g (queries).
    // Rows behind the last repeat it.
    int pos[2 * RT];
#pragma unroll
    for (int x = 0; x < 2 * RT; ++x) {
      const int tok = one ? 0 : (row0 + min((x >> 1) * 8 + 2 * t4 + (x & 1), rows - 1)) / group;
      pos[x] = pos0 + tok;
    }
    auto lo = [&](int at) { return paged_seen_from(a, r.len, at); };
    auto hi = [&](int at) { return paged_seen_to(a, r.len, at); };
    // From product to power of two; a key that is not seen gets the product that stands for a power of -inf, so the
    // factor must not be 0: the least normal number then stands for it.
    auto nonzero = [](float x) { return fabsf(x) < FLT_MIN ? copysignf(FLT_MIN, x) : x; };
    const float scale = a.sm_scale * CUDART_L2E_F, key_scale = C::E4M3 ? a.k_scale[kv_head] : 1.f;
    const float mult = nonzero(scale * key_scale);
    const float unseen = mult > 0.f ? -CUDART_INF_F : CUDART_INF_F;
    const T* qrow[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      const int row = row0 + min(8 * i + g, rows - 1), tok = one ? 0 : row / group, head = kv_head * group + row - tok * group;
      qrow[i] = static_cast<const T*>(a.q) + static_cast<int64_t>(r.s0 + tok) * a.q_strides[0] + head * a.q_strides[1];
    }
    const int all_lo = lo(pos0 + (one ? 0 : (row0 + rows - 1) / group));  // keys that every row sees
    const int all_hi = hi(pos0 + (one ? 0 : row0 / group));

    // ---- query fragments
    // bf16 queries over 8-bit keys: a power of two brings each row into the range of halves.
    constexpr bool SHIFT = C::E4M3 && BF16;
    float up[RT], down[SHIFT ? 2 * RT : 1] = {};
    if constexpr (SHIFT) {
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
        const int shift = e == 0xFF || top == 0 ? 0 : min(141 - e, 100);  // from -113 on
        up[i] = __uint_as_float(static_cast<uint32_t>(127 + shift) << 23);
        const float back = nonzero(scale * __uint_as_float(static_cast<uint32_t>(127 - shift) << 23) * key_scale);
#pragma unroll
        for (int c = 0; c < 2; ++c) down[2 * i + c] = __shfl_sync(~0u, back, (2 * t4 + c) * 4);
      }
    }
    auto factor = [&](int x) { return SHIFT ? down[SHIFT ? x : 0] : mult; };
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
      __syncwarp();
#pragma unroll
      for (int ks = 0; ks < C::KSTEPS; ++ks)
#pragma unroll
        for (int i = 0; i < RT; ++i) {
          uint32_t f[2];
          q_frag(ks, i, f);
          asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(q_smem + (ks * RT + i) * 256 + lane * 8), "r"(f[0]), "r"(f[1])
                       : "memory");
        }
      __syncwarp();
    }
    auto q_at = [&](int ks, int i, uint32_t (&f)[2]) {
      if constexpr (C::QREG) {
        f[0] = qreg[ks * RT + i][0], f[1] = qreg[ks * RT + i][1];
      } else {
        const uint2 x = lds8(q_smem + (ks * RT + i) * 256 + lane * 8);
        f[0] = x.x, f[1] = x.y;
      }
    };

    // A row without a key so far has the reference PA_NONE, from which any score is a rise.
    float o[C::DT][RT][4], m[2 * RT], l[2 * RT];
#pragma unroll
    for (int x = 0; x < 2 * RT; ++x) m[x] = PA_NONE, l[x] = 0.f;
#pragma unroll
    for (int dt = 0; dt < C::DT; ++dt)
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) o[dt][i][c] = 0.f;

    for (int i = 0; i < steps; ++i) {
      const int base = r.first + (cur.step + i) * C::KEYS;
      const uint32_t k_at = ready();
      if (base >= r.len) {  // no key at all
        refill(false);
        ready();
        refill(true);
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
        const uint32_t at = k_at + (lane & 15) * C::ROWB + (((lane >> 4) ^ (lane & 7)) << 4);
        float s2[RT][4];  // two sums, so that a product waits for the last but one
#pragma unroll
        for (int j = 0; j < RT; ++j)
#pragma unroll
          for (int c = 0; c < 4; ++c) s2[j][c] = 0.f;
        constexpr int GROUP = C::KSTEPS < 8 || RT > 1 ? 4 : 8;
#pragma unroll
        for (int k0 = 0; k0 < C::KSTEPS; k0 += GROUP) {
          uint32_t k[GROUP][4];
#pragma unroll
          for (int ks = 0; ks < GROUP; ++ks) ldsm4((at ^ ((k0 + ks) % 4 * 32)) + (k0 + ks) / 4 * 128, k[ks]);
          if (k0 == 0) refill(false);  // its arithmetic fills the wait for the fragments
#pragma unroll
          for (int ks = 0; ks < GROUP; ++ks)
#pragma unroll
            for (int j = 0; j < RT; ++j) {
              uint32_t f[2];
              q_at(k0 + ks, j, f);
              if (ks & 1) mma16816<MBF16>(s2[j], k[ks], f[0], f[1]);
              else mma16816<MBF16>(s[0][j], k[ks], f[0], f[1]);
            }
        }
#pragma unroll
        for (int j = 0; j < RT; ++j)
#pragma unroll
          for (int c = 0; c < 4; ++c) s[0][j][c] += s2[j][c];
      } else {
#pragma unroll
        for (int part = 0; part < C::D / 64; ++part) {
          uint4 x[SN], y[SN];
#pragma unroll
          for (int n = 0; n < SN; ++n) {
            const uint32_t at = k_at + ring_at<C, false>(g, t4 + part * 4) + n * 16 * C::ROWB;
            x[n] = lds16(at), y[n] = lds16(at + 8 * C::ROWB);
          }
          if (part == 0) refill(false);  // its arithmetic fills the wait for the keys
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            uint32_t f[RT][2];
#pragma unroll
            for (int j = 0; j < RT; ++j) q_at(part * 4 + w, j, f[j]);
#pragma unroll
            for (int n = 0; n < SN; ++n) {
              uint32_t k[4];
              e4m3x4_to_h2x2(reinterpret_cast<const uint32_t*>(&x[n])[w], k[0], k[2]);
              e4m3x4_to_h2x2(reinterpret_cast<const uint32_t*>(&y[n])[w], k[1], k[3]);
#pragma unroll
              for (int j = 0; j < RT; ++j) mma16816<false>(s[n][j], k, f[j][0], f[j][1]);
            }
          }
        }
      }

      // ---- weights
      const bool whole = base >= all_lo && base + C::KEYS <= all_hi;  // every row sees every key
      if (!whole) {
#pragma unroll
        for (int x = 0; x < 2 * RT; ++x) {
          const int from = lo(pos[x]), to = hi(pos[x]);
#pragma unroll
          for (int n = 0; n < SN; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int key = base + n * 16 + h * 8 + g;
              if (key < from || key >= to) s[n][x >> 1][2 * h + (x & 1)] = unseen;
            }
        }
      }
      bool rise = false;
#pragma unroll
      for (int x = 0; x < 2 * RT; ++x)
#pragma unroll
        for (int n = 0; n < SN; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h) rise |= fmaf(s[n][x >> 1][2 * h + (x & 1)], factor(x), -m[x]) > RISE;
      if (__any_sync(~0u, rise)) {
#pragma unroll
        for (int x = 0; x < 2 * RT; ++x) {
          float top = -CUDART_INF_F;
#pragma unroll
          for (int n = 0; n < SN; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h) top = fmaxf(top, s[n][x >> 1][2 * h + (x & 1)] * factor(x));
          top = fmaxf(top, __shfl_xor_sync(~0u, top, 4));
          top = fmaxf(top, __shfl_xor_sync(~0u, top, 8));
          top = fmaxf(top, __shfl_xor_sync(~0u, top, 16));
          top -= BIAS;
          if (top > m[x]) {
            const float alpha = ex2(m[x] - top);
            m[x] = top;
            l[x] *= alpha;
#pragma unroll
            for (int dt = 0; dt < C::DT; ++dt) {
              o[dt][x >> 1][x & 1] *= alpha;
              o[dt][x >> 1][2 + (x & 1)] *= alpha;
            }
          }
        }
      }
      bool small = false;  // weights between 0 and PA_SMALL
#pragma unroll
      for (int x = 0; x < 2 * RT; ++x)
#pragma unroll
        for (int n = 0; n < SN; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float& v = s[n][x >> 1][2 * h + (x & 1)];
            v = ex2(fmaf(v, factor(x), -m[x]));
            l[x] += v;
            if constexpr (!MBF16) small |= __float_as_uint(v) - 1u < __float_as_uint(PA_SMALL) - 1u;
          }
      if constexpr (!MBF16) small = __any_sync(~0u, small);
      const uint32_t v_at = ready();
      refill(true);

      // ---- values, transposed: 16 dimensions by 8 rows a product
      uint32_t odd = 0;  // groups of 16 keys with values that are not finite, where some row does not see some key
      if (!whole && !newest) {
        constexpr uint32_t EXP = MBF16 ? 0x7F807F80u : 0x7C007C00u, ONE = MBF16 ? 0x00800080u : 0x04000400u;
#pragma unroll
        for (int kk = 0; kk < SN; ++kk) {
          bool any = false;
          each_v<C>(v_at, lane, kk, [&](int, const uint32_t (&v)[4]) {
#pragma unroll
            for (int c = 0; c < 4; ++c) any |= (((v[c] & EXP) + ONE) & 0x80008000u) != 0;
          });
          if (__any_sync(~0u, any)) odd |= 1u << kk;
        }
      }
      if (odd != 0) {
        PagedOdd<C> x;
#pragma unroll
        for (int j = 0; j < RT; ++j) {
          x.pos[2 * j] = pos[2 * j], x.pos[2 * j + 1] = pos[2 * j + 1];
#pragma unroll
          for (int c = 0; c < 4; ++c) {
#pragma unroll
            for (int dt = 0; dt < C::DT; ++dt) x.o[dt][j][c] = o[dt][j][c];
#pragma unroll
            for (int n = 0; n < SN; ++n) x.w[n][j][c] = s[n][j][c];
          }
        }
        paged_odd<C>(x, v_at, base, odd, a, r.len);
#pragma unroll
        for (int j = 0; j < RT; ++j)
#pragma unroll
          for (int dt = 0; dt < C::DT; ++dt)
#pragma unroll
            for (int c = 0; c < 4; ++c) o[dt][j][c] = x.o[dt][j][c];
      }
      auto products = [&](auto kind) {
        constexpr PagedKind K = decltype(kind)::value;
#pragma unroll
        for (int kk = 0; kk < SN; ++kk) {
          if ((odd >> kk & 1) != 0) continue;
          PagedWeights<K> w[RT];
#pragma unroll
          for (int j = 0; j < RT; ++j) w[j].set(s[kk][j]);
          each_v<C>(v_at, lane, kk, [&](int dt, const uint32_t (&v)[4]) {
            const PagedValues<K> x(v);
#pragma unroll
            for (int j = 0; j < RT; ++j) x.times(o[dt][j], w[j]);
          });
        }
      };
      if constexpr (MBF16) products(std::integral_constant<PagedKind, PAIR_BF16>());
      else if (!small) products(std::integral_constant<PagedKind, PAIR_F16>());
      else products(std::integral_constant<PagedKind, PAIR_TF32>());
    }

    // ---- the unit, or this worker's part of it, is done
    const bool from_start = cur.step == 0, to_end = cur.step + steps == r.steps, partial = !(from_start && to_end);
    const int part = (2 * worker + (first_segment ? 0 : 1)) * p.tracks + track;
#pragma unroll
    for (int x = 0; x < 2 * RT; ++x) {
      l[x] += __shfl_xor_sync(~0u, l[x], 4);
      l[x] += __shfl_xor_sync(~0u, l[x], 8);
      l[x] += __shfl_xor_sync(~0u, l[x], 16);
      if (m[x] == PA_NONE) m[x] = -CUDART_INF_F;
    }
    if (pool) {
      // The warps' parts meet in shared memory, in place of the rings, and each warp joins some fragments.
      cp_async_wait<0>();
      __syncwarp();
      const int active = min(wide, shares - static_cast<int>(blockIdx.x) * wide);  // teams
      auto own_o = [&](int w) { return reinterpret_cast<float4*>(smem + w * C::RING) + lane; };
      auto own_ml = [&](int w) { return reinterpret_cast<float4*>(smem + w * C::RING + C::FRAGS * 512) + lane; };
#pragma unroll
      for (int j = 0; j < RT; ++j) {
#pragma unroll
        for (int dt = 0; dt < C::DT; ++dt)
          own_o(warp)[(dt * RT + j) * 32] = make_float4(o[dt][j][0], o[dt][j][1], o[dt][j][2], o[dt][j][3]);
        own_ml(warp)[j * 32] = make_float4(m[2 * j], l[2 * j], m[2 * j + 1], l[2 * j + 1]);
      }
      asm volatile("bar.sync 1, %0;" ::"r"(active * p.tracks * 32) : "memory");
      const bool all = unit0 == cut.at(blockIdx.x * wide) &&
                       unit1 == cut.at(min((static_cast<int>(blockIdx.x) + 1) * wide, shares));
      const int64_t slot = 2 * static_cast<int64_t>(blockIdx.x) * wide * p.tracks + track;
#pragma unroll 1
      for (int f = team; f < C::FRAGS; f += active) {
        const int dt = f / RT, j = f % RT;
        PagedSum<1> sum;
        sum.clear();
#pragma unroll 1
        for (int w = 0; w < active; ++w) {
          const float4 u[1] = {own_o(w * p.tracks + track)[f * 32]};
          sum.add(own_ml(w * p.tracks + track)[j * 32], u);
        }
        if (j * 8 >= rows) continue;
        if (all) {
          paged_finish<C, 1>(a, sum.o, sum.m, sum.l, dt, r.s0, kv_head, row0 + j * 8, rows - j * 8, lane);
        } else if (j * 8 + 2 * t4 < rows) {
          reinterpret_cast<float4*>(p.part_o)[(slot * C::FRAGS + f) * 32 + lane] = make_float4(sum.o[0][0], sum.o[0][1], sum.o[0][2], sum.o[0][3]);
          if (dt == 0 && g == 0)
            *reinterpret_cast<float4*>(p.part_ml + (slot * C::ROWS + j * 8 + 2 * t4) * 2) = make_float4(sum.m[0], sum.l[0], sum.m[1], sum.l[1]);
        }
      }
      return;
    }
    if (partial) {
      float4* to = reinterpret_cast<float4*>(p.part_o) + static_cast<int64_t>(part) * C::FRAGS * 32 + lane;
#pragma unroll
      for (int j = 0; j < RT; ++j)
        if (j * 8 + 2 * t4 < rows) {
#pragma unroll
          for (int dt = 0; dt < C::DT; ++dt)
            to[(dt * RT + j) * 32] = make_float4(o[dt][j][0], o[dt][j][1], o[dt][j][2], o[dt][j][3]);
          if (g == 0)
            *reinterpret_cast<float4*>(p.part_ml + (static_cast<int64_t>(part) * C::ROWS + j * 8 + 2 * t4) * 2) =
                make_float4(m[2 * j], l[2 * j], m[2 * j + 1], l[2 * j + 1]);
        }
    } else {
#pragma unroll
      for (int j = 0; j < RT; ++j) {
        if (j * 8 >= rows) break;
        float f[C::DT][4];
#pragma unroll
        for (int dt = 0; dt < C::DT; ++dt)
#pragma unroll
          for (int c = 0; c < 4; ++c) f[dt][c] = o[dt][j][c];
        const float sum[2] = {l[2 * j], l[2 * j + 1]}, ref[2] = {m[2 * j], m[2 * j + 1]};
        paged_finish<C, C::DT>(a, f, ref, sum, 0, r.s0, kv_head, row0 + j * 8, rows - j * 8, lane);
      }
    }
    first_segment = false;
    t += steps;
    if (t < t1) cur.next_unit(a, heads);
  }
}

// Joins the parts of the units that borders between workers cut.  Of a unit of few parts a warp takes up to eight
// fragments of the output; of one of many (a long request has hundreds) a block takes a fragment, and its warps share the
// parts.  The kernel runs for a few microseconds, most of which its first pass through its own code takes: the
// loops stay rolled up (unrolled by 4 over parts and by 8 over fragments it took 24 us on 1776 units of two parts).
constexpr int PA_JOIN_WARPS = 16;
constexpr int PA_JOIN_MANY = 16;    // parts from which on a unit counts as one of many
constexpr int PA_JOIN_LOOK = 32;    // records that a block looks through for units of many parts, which it takes one by
                                    // one (16 requests, 8-bit, D = 64, 14 parts a unit: 71 us with 128 and 12, 49 so)

// Blocks of the join: those for units of few parts, then those for units of many.
template <typename C>
struct PagedJoinGrid {
  static constexpr int N = C::DT < 8 ? C::DT : 8;  // fragments a warp, of one 8-row tile
  static constexpr int SLICES = C::FRAGS / N;
  int few, many;
  __host__ __device__ explicit PagedJoinGrid(int records)
      : few((records + PA_JOIN_WARPS - 1) / PA_JOIN_WARPS * SLICES), many((records + PA_JOIN_LOOK - 1) / PA_JOIN_LOOK * C::FRAGS) {}
};

// Adds parts from, from + skip, ... of N fragments, U of them on their way at a time.
template <typename C, int N, int U>
__device__ __forceinline__ void paged_merge(const PagedAttnParams& p, const PagedJoin& d, PagedSum<N>& sum, int dt, int j, int from,
                                            int skip, int lane) {
  const int t4 = lane & 3, parts = j * 8 + 2 * t4 < d.rows ? d.parts() : 0;  // rows that there are none of have nothing to read
#pragma unroll 1
  for (int i = from; i < parts; i += U * skip) {
    float4 ml[U], u[U][N];
#pragma unroll
    for (int q = 0; q < U; ++q) {
      const int64_t slot = d.slot(min(i + q * skip, parts - 1));
      ml[q] = *reinterpret_cast<const float4*>(p.part_ml + (slot * C::ROWS + j * 8 + 2 * t4) * 2);
#pragma unroll
      for (int k = 0; k < N; ++k)
        u[q][k] = reinterpret_cast<const float4*>(p.part_o)[(slot * C::FRAGS + (dt + k) * C::RT + j) * 32 + lane];
    }
#pragma unroll
    for (int q = 0; q < U; ++q)
      if (i + q * skip < parts) sum.add(ml[q], u[q]);
  }
}

template <typename C>
__global__ void __launch_bounds__(PA_JOIN_WARPS * 32) paged_join_kernel(const __grid_constant__ PagedAttnParams p) {
  constexpr int RT = C::RT;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, records = p.grid * PA_WARPS;
  const PagedJoinGrid<C> grid(records);
  const PagedJoin* record = reinterpret_cast<const PagedJoin*>(p.desc);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (static_cast<int>(blockIdx.x) < grid.few) {
    constexpr int N = PagedJoinGrid<C>::N;
    const int slice = blockIdx.x % PagedJoinGrid<C>::SLICES, c = blockIdx.x / PagedJoinGrid<C>::SLICES * PA_JOIN_WARPS + warp;
    const int j = slice % RT, dt = slice / RT * N;
    if (c >= records) return;
    const PagedJoin d = record[c];
    if (d.parts() == 0 || d.parts() >= PA_JOIN_MANY || j * 8 >= d.rows) return;
    PagedSum<N> sum;
    sum.clear();
    paged_merge<C, N, 2>(p, d, sum, dt, j, 0, 1, lane);
    paged_finish<C, N>(p.a, sum.o, sum.m, sum.l, dt, d.s0, d.kv_head, d.row0 + j * 8, d.rows - j * 8, lane);
    return;
  }
  __shared__ float4 s_ml[PA_JOIN_WARPS][32], s_o[PA_JOIN_WARPS][32];
  const int index = blockIdx.x - grid.few, f = index % C::FRAGS, c0 = index / C::FRAGS * PA_JOIN_LOOK;
  const int j = f % RT, dt = f / RT;
  static_assert(PA_JOIN_LOOK == 32, "every warp looks for itself");
  int parts = 0;
  if (c0 + lane < records) parts = record[c0 + lane].parts();
  uint32_t left = __ballot_sync(~0u, parts >= PA_JOIN_MANY);
#pragma unroll 1
  while (left != 0) {  // the same for all warps
    const PagedJoin d = record[c0 + __ffs(left) - 1];
    left &= left - 1;
    if (j * 8 >= d.rows) continue;
    PagedSum<1> sum;
    sum.clear();
    paged_merge<C, 1, 4>(p, d, sum, dt, j, warp, PA_JOIN_WARPS, lane);
    s_ml[warp][lane] = make_float4(sum.m[0], sum.l[0], sum.m[1], sum.l[1]);
    s_o[warp][lane] = make_float4(sum.o[0][0], sum.o[0][1], sum.o[0][2], sum.o[0][3]);
    __syncthreads();
    if (warp == 0) {
#pragma unroll 1
      for (int v = 1; v < PA_JOIN_WARPS; ++v) {
        const float4 u[1] = {s_o[v][lane]};
        sum.add(s_ml[v][lane], u);
      }
      paged_finish<C, 1>(p.a, sum.o, sum.m, sum.l, dt, d.s0, d.kv_head, d.row0 + j * 8, d.rows - j * 8, lane);
    }
    __syncthreads();
  }
}

}  // namespace syn
