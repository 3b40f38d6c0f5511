// kvattn_tc.cu -- the shared pass of attention over a paged cache on the 5th-generation tensor cores:
// the queries of all sequences, stacked, against the prefix that they share.
//
// One block takes up to MT x 128 rows (tokens x heads of a key/value head's group) along its piece of
// the prefix, in steps of 64 positions.  Per step and 128 rows: S = Q K^T into 64 columns of tensor
// memory, one thread a row takes the row's maximum, exponentials and sum, writes P in the cache's type
// over S, and O += P V accumulates in tensor memory with P as the tensor-memory operand.  Two buffers of
// S a half of the rows, and two halves with MT = 2: products of one run while another is in its softmax,
// and both halves read the same tiles of K and V.  A row's reference maximum moves only when the maximum
// has grown by more than GROW (in log2 units); then O and the sum are rescaled, which after the first
// tiles is rare.  P goes to its product in two numbers of the cache's type where bytes bound (MT = 1) or the
// result is fp32, which a weight rounded to the type would not bear; else rounded to the type, 2^-8 (bf16) or
// 2^-11 (f16) of a weight at most, since the second product costs 185 -> 204 us (128 tokens behind 32k) and 188 -> 255
// (32 questions behind 8k).  Its sum l, S and O are fp32.
//
// Warps: 0 brings K and V by TMA (a box a page and 64 elements; 128-byte swizzle) through a ring of
// slots of 128 positions, one thread of 1 issues the products, 4..7 and 8..11 are the rows.  S, P:
// columns 128 x + 64 b of half x and buffer b; O: columns 256 + 128 x.  Tensor memory holds the whole
// accumulation, so shared memory is Q and the ring.
//
// Bound: 256 rows of head_dim 128 in 16 bits against 128 positions are 2 x 4 x 128 x 128 x 128 operations:
// 1.5 us of an SM at the rate of a large library product.  Measured: 2.4 to 2.6 us, the chain from the
// softmax's P through the issuing thread to the next S; the tensor pipe is busy 54 % of the time for 4085
// rows of each of 8 heads on 8k positions (149 us), 58 % for 512 rows of each on 32k (112 us on 90 SMs).
// Measured and not taken: steps of 128 (one buffer: 147 -> 160 us), a ring of 64 positions (twice the waits
// and commits: 140 -> 175), the halves' waits joined (175), exponentials by polynomial on 1/8 to 1/2 of the
// columns (+0 to +8 %), the halves' exponentials in turns, which keeps them out of phase (164 -> 172 us, 128
// behind 32k), the prefix brought into L2 two to four tiles ahead (no difference).
#include <cuda.h>
#include <cuda_runtime.h>

#include <cstring>

#include "capi_internal.h"
#include "kvattn.cuh"

namespace ex {
namespace {

constexpr int TC_THREADS = 384;

template <int DP, int MT>
struct TcLayout {
  static constexpr int HALF = TC_TILE * 128;           // 128 rows of 64 elements, swizzled: 16 KB
  static constexpr int SLOT = HALF * (DP / 64);        // a tile of K or V, or 128 rows of Q
  static constexpr int SLOTS = (208 * 1024 - MT * SLOT) / SLOT < 10 ? (208 * 1024 - MT * SLOT) / SLOT : 10;
  static constexpr int RING = MT * SLOT;
  static constexpr int BARS = RING + SLOTS * SLOT;
  static constexpr int N_BARS = 2 * SLOTS + 8 * 2 + 1;
  static constexpr int MISC = BARS + 8 * N_BARS;
  static constexpr int ALLOC = MISC + 16 + 1024;
  static_assert(ALLOC > 116 * 1024 && ALLOC <= 227 * 1024, "one block an SM, which then owns the tensor memory");
};

__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void tc_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// One product of the tensor pipe, D = A B or D += A B.  Descriptors come as their low words (the address
// and the leading offset); the high word is one constant.
constexpr uint32_t DESC_HI = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "mov.b64 da, {%1, %5};\n\t"
      "mov.b64 db, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(static_cast<int>(add)), "n"(DESC_HI)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "mov.b64 db, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(static_cast<int>(add)), "n"(DESC_HI)
      : "memory");
}

#define EX_R8(v, i) "=r"(v[i]), "=r"(v[i + 1]), "=r"(v[i + 2]), "=r"(v[i + 3]), "=r"(v[i + 4]), "=r"(v[i + 5]), "=r"(v[i + 6]), "=r"(v[i + 7])
#define EX_U8(v, i) "r"(v[i]), "r"(v[i + 1]), "r"(v[i + 2]), "r"(v[i + 3]), "r"(v[i + 4]), "r"(v[i + 5]), "r"(v[i + 6]), "r"(v[i + 7])

// 32 columns of the thread's row.
__device__ __forceinline__ void tc_ld32(uint32_t addr, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : EX_R8(v, 0), EX_R8(v, 8), EX_R8(v, 16), EX_R8(v, 24)
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tc_st32(uint32_t addr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::EX_U8(v, 0),
      EX_U8(v, 8), EX_U8(v, 16), EX_U8(v, 24), "r"(addr)
      : "memory");
}

// Rows of 128 bytes with the 128-byte swizzle, groups of eight 1024 bytes apart.  Read along the 64
// elements of a row (Q, K) the leading offset is not used; read across the rows (V) it is the distance
// to the next 64 elements.
__device__ __forceinline__ uint32_t sw128_desc(uint32_t addr, uint32_t leading) {  // the low word
  return (addr >> 4) | (leading >> 4) << 16;
}

// Pairs of fp32 in one instruction.
using f32x2 = unsigned long long;
__device__ __forceinline__ f32x2 two(float a, float b) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 one_by_one(f32x2 v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// The largest; NaN if any is.
__device__ __forceinline__ float max_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

__device__ __forceinline__ bool spin(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  if (mbar_try_wait(bar, parity)) return true;
  const unsigned long long t0 = global_ns();
  for (uint32_t i = 1;; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((i & 63u) == 0) {
      if (*abort_flag) return false;
      if (global_ns() - t0 > WAIT_LIMIT_NS) return false;
    }
  }
}

// A block of rows along consecutive tiles of the prefix, in steps of half a tile.
constexpr int STEP = TILE;
struct Segment {
  int kvh, row0, tile0, n, slot;
  int steps;  // the prefix's last half tile may be empty
};
__device__ __forceinline__ Segment segment_at(const TcCut& c, int at, int end, const AttnArgs& a, int shared) {
  Segment s;
  const int block = at / c.tiles;
  s.tile0 = at - block * c.tiles;
  s.n = min(c.tiles - s.tile0, end - at);
  s.kvh = block / c.lines;
  const int piece = blockIdx.x / a.pre_width, in_piece = blockIdx.x - piece * a.pre_width;
  s.row0 = ((block - s.kvh * c.lines) * a.pre_width + in_piece) * a.pre_rows;
  s.slot = piece - block * c.tiles / c.per;
  s.steps = min(2 * s.n, (shared - s.tile0 * TC_TILE + STEP - 1) / STEP);
  return s;
}

// FINE: P in two numbers of the type, a coarse and the rest.
template <typename T, int DP, int MT, bool FINE>
__global__ void __launch_bounds__(TC_THREADS, 1)
    attn_tc_kernel(const AttnArgs a, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
  using L = TcLayout<DP, MT>;
  constexpr int CH = DP / 8, NS = L::SLOTS;
  constexpr uint32_t FMT = exponent16<T>() == exponent16<__half>() ? 0u : 1u;
  // D fp32, A and B of the type, M = 128; N = 64 for S, DP for O, whose B is read across its rows
  constexpr uint32_t IDESC_S = (1u << 4) | (FMT << 7) | (FMT << 10) | ((uint32_t(STEP) >> 3) << 17) | ((128u >> 4) << 24);
  constexpr uint32_t IDESC_O = (1u << 4) | (FMT << 7) | (FMT << 10) | (1u << 16) | ((uint32_t(DP) >> 3) << 17) | ((128u >> 4) << 24);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::BARS);  // a ring slot's boxes landed
  uint64_t* empty = full + NS;                                   // the products that read it are done
  uint64_t* q_full = empty + NS;                                 // [half]: Q is in shared memory (128 threads)
  uint64_t* q_free = q_full + 2;                                 // [half]: the segment's sums have left Q's memory (4 warps)
  uint64_t* s_full = q_free + 2;                                 // [half][buffer]: S is in tensor memory
  uint64_t* p_full = s_full + 4;                                 // [half][buffer]: P is (4 warps)
  uint64_t* o_done = p_full + 4;                                 // [half][buffer]: the P V of a step is in O
  uint64_t* fin = o_done + 4;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::MISC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::MISC + 4);
  const int warp = __shfl_sync(0xFFFFFFFFu, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < NS; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 128);
      mbar_init(&q_free[i], 4);
      for (int j = 0; j < 2; ++j) {
        mbar_init(&s_full[2 * i + j], 1);
        mbar_init(&p_full[2 * i + j], 4);
        mbar_init(&o_done[2 * i + j], 1);
      }
    }
    mbar_init(fin, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512u)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_before();
  __syncthreads();
  tc_after();
  const uint32_t tmem = __shfl_sync(0xFFFFFFFFu, *tmem_slot, 0);
  pdl_enter_pair();

  const int shared = __shfl_sync(0xFFFFFFFFu, shared_of(a), 0);
  const TcCut cut = tc_cut(a, shared);
  const int begin = min(cut.total, static_cast<int>(blockIdx.x) / a.pre_width * cut.per), end = min(cut.total, begin + cut.per);

  if (warp == 0) {
    // K of tile 0, V of tile 0, K of tile 1, ...: the order in which the products need them
    const int32_t* table = a.c.table + static_cast<long long>(a.shared_seq) * a.c.max_pages;
    Ring<NS> ring;
    int issued = 0;
    bool ok = true;
    for (int at = begin; ok && at < end;) {
      const Segment g = segment_at(cut, at, end, a, shared);
      at += g.n;
      Pages pages(a.c, table, g.tile0 * TC_TILE, shared);
      for (int i = 0; ok && i < 2 * g.n; ++i) {
        const int p0 = (g.tile0 + (i >> 1)) * TC_TILE, page = pages.at(p0);
        ok = __all_sync(0xFFFFFFFFu, wait_or_abort(&empty[ring.slot], ring.phase ^ 1u, abort_flag)) != 0;
        if (!ok) break;
        bring_tile<DP, TC_TILE>(a.c, page, (i & 1) == 0 ? &kmap : &vmap, smem_u32(smem + L::RING + ring.slot * L::SLOT), g.kvh, p0,
                                shared, &full[ring.slot]);
        issued = min(issued + 1, NS);
        ring.next();
      }
    }
    if (lane == 0) {
      if (!ok) {
        *abort_flag = 1;
        atomicOr(a.c.status, ST_TIMEOUT_EMPTY);
      }
      drain<NS>(ring, issued, full, a.c.status);
    }
  } else if (warp == 1) {
    // One elected thread: each wait and each turn of a whole warp costs it about 100 ns between products.
    const uint32_t q_s = smem_u32(smem), ring_s = smem_u32(smem + L::RING);
    if (elect_one()) {
      Ring<NS> v;  // V of the tile in use; K of the next one is the place after it
      v.next();
      uint32_t segs = 0, par[2] = {0, 0};  // parity of either buffer's next P; constant indices only
      bool ok = true;
      auto there = [&](uint64_t* bar, uint32_t parity) { return spin(bar, parity, abort_flag); };
      // S of 64 positions, the first or last of a tile, into the buffer of that parity
      auto product_s = [&](int half, uint32_t kd, int b) {
        const uint32_t qd = sw128_desc(q_s + half * L::SLOT, 16);
#pragma unroll
        for (int k = 0; k < DP / 16; ++k) {
          const uint32_t off = ((k / 4) * L::HALF + (k % 4) * 32) >> 4;
          mma_ss(tmem + 128 * half + STEP * b, qd + off, kd + off + ((b * STEP * 128) >> 4), IDESC_S, k > 0);
        }
        tc_commit(&s_full[2 * half + b]);
      };
      for (int at = begin; ok && at < end; ++segs) {
        const Segment g = segment_at(cut, at, end, a, shared);
        at += g.n;
        Ring<NS> k = v;
        k.back();
        ok = there(&full[k.slot], k.phase);
#pragma unroll
        for (int h = 0; h < MT; ++h) ok = ok && there(&q_full[h], segs & 1u);
        if (!ok) break;
        tc_after();
        const uint32_t kd0 = sw128_desc(ring_s + k.slot * L::SLOT, 16);
#pragma unroll
        for (int h = 0; h < MT; ++h) product_s(h, kd0, 0);
        if (g.steps > 1)
#pragma unroll
          for (int h = 0; h < MT; ++h) product_s(h, kd0, 1);
        tc_commit(&empty[k.slot]);
        for (int j = 0; ok && j < g.steps; j += 2) {
          k.next();
          k.next();
          ok = there(&full[v.slot], v.phase);
          const uint32_t kd = sw128_desc(ring_s + k.slot * L::SLOT, 16), vd0 = sw128_desc(ring_s + v.slot * L::SLOT, L::HALF);
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            if (j + b >= g.steps) break;
            const bool more = j + b + 2 < g.steps;
#pragma unroll
            for (int h = 0; h < MT; ++h) {
              ok = ok && there(&p_full[2 * h + b], par[b]);
              if (!ok) break;
              tc_after();
              const uint32_t p_at = tmem + 128 * h + STEP * b;
#pragma unroll
              for (int s = 0; s < STEP / 16; ++s) {
                const uint32_t vs = vd0 + ((b * STEP * 128 + s * 2048) >> 4);
                mma_ts(tmem + 256 + 128 * h, p_at + 8 * s, vs, IDESC_O, b > 0 || s > 0 || j > 0);
                if constexpr (FINE) mma_ts(tmem + 256 + 128 * h, p_at + STEP / 2 + 8 * s, vs, IDESC_O, true);
              }
              tc_commit(&o_done[2 * h + b]);
              if (more && b == 0 && h == 0) ok = there(&full[k.slot], k.phase);
              if (!ok) break;
              if (more) product_s(h, kd, b);
            }
            par[b] ^= 1u;
          }
          tc_commit(&empty[v.slot]);  // both tiles' places are free once these products are done
          if (j + 2 < g.steps) tc_commit(&empty[k.slot]);
          v.next();
          v.next();
        }
      }
      if (!ok) {
        *abort_flag = 1;
        atomicOr(a.c.status, ST_TIMEOUT_FULL);
      }
      tc_commit(fin);  // all products are done before tensor memory is given back
      if (!mbar_wait(fin, 0)) atomicOr(a.c.status, ST_TIMEOUT_DRAIN);
    }
    __syncwarp();
  } else if (warp >= 4 && warp < 4 + 4 * MT) {
    const int half = (warp - 4) >> 2, r = threadIdx.x & 127;  // the thread's row of its half
    const uint32_t lane_base = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t o_at = lane_base + 256 + 128 * half;
    const int rows = a.n_tokens * a.rep, hd = a.c.hd;
    const float sc = fabsf(a.scale);
    const uint32_t flip = a.scale < 0.0f ? 0x80008000u : 0u;  // a negative scale: -Q, so that a maximum is a maximum
    uint32_t segs = 0, par[2] = {0, 0};  // parity of either buffer's next S; constant indices only
    Ring<NS> ring;  // V of the tile in use
    ring.next();
    bool ok = true;
    for (int at = begin; ok && at < end; ++segs) {
      const Segment g = segment_at(cut, at, end, a, shared);
      at += g.n;
      const int base_row = g.row0 + half * 128;
      {  // a thread takes one chunk of eight elements of every (128 / CH)th row
        constexpr int STEP = 128 / CH;
        const int ch = r % CH, dq = STEP / a.rep, dr = STEP - dq * a.rep;
        int tok = (base_row + r / CH) / a.rep, gh = base_row + r / CH - tok * a.rep;
        uint4 v[CH];
#pragma unroll
        for (int x = 0; x < CH; ++x) {
          v[x] = tok < a.n_tokens && ch * 8 < hd ? *reinterpret_cast<const uint4*>(
                                                       a.q + (static_cast<long long>(tok) * a.n_heads + g.kvh * a.rep + gh) * hd + ch * 8)
                                                 : make_uint4(0u, 0u, 0u, 0u);
          tok += dq;
          gh += dr;
          if (gh >= a.rep) {
            gh -= a.rep;
            ++tok;
          }
        }
        if (segs > 0) ok = __all_sync(0xFFFFFFFFu, wait_or_abort(&q_free[half], (segs - 1u) & 1u, abort_flag));
        if (!ok) break;
#pragma unroll
        for (int x = 0; x < CH; ++x) {
          const int qr = r / CH + x * STEP;
          v[x].x ^= flip;
          v[x].y ^= flip;
          v[x].z ^= flip;
          v[x].w ^= flip;
          *reinterpret_cast<uint4*>(smem + half * L::SLOT + (ch / 8) * L::HALF + qr * 128 + (((ch & 7) ^ (qr & 7)) << 4)) = v[x];
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      mbar_arrive(&q_full[half]);

      float m = -INFINITY, l = 0.0f;
      auto step = [&](const int j, const int b) {
        const uint32_t s_at = lane_base + 128 * half + STEP * b;
        ok = __all_sync(0xFFFFFFFFu, wait_or_abort(&s_full[2 * half + b], par[b], abort_flag)) != 0;
        if (!ok) return;
        par[b] ^= 1u;
        tc_after();
        uint32_t s[STEP];
        tc_ld32(s_at, s);
        tc_ld32(s_at + 32, s + 32);
        tc_wait_ld();
        const int valid = shared - g.tile0 * TC_TILE - j * STEP;
        if (valid < STEP) {
          // -inf times a scale of 0 is no number: scores of 0 then, as all are, whose weights of 2^P_SHIFT leave the
          // sum here (exactly) and meet values of 0 below
          const uint32_t off = sc == 0.0f ? 0u : 0xFF800000u;
          if (sc == 0.0f) l -= static_cast<float>((STEP - valid) << static_cast<int>(P_SHIFT));
#pragma unroll
          for (int c = 0; c < STEP; ++c)
            if (c >= valid) s[c] = off;
          if (half == 0) {
            // V past the prefix's end is what memory held: 0 for the product
            ok = __all_sync(0xFFFFFFFFu, wait_or_abort(&full[ring.slot], ring.phase, abort_flag)) != 0;
            if (!ok) return;
            uint8_t* vs = smem + L::RING + ring.slot * L::SLOT + b * (STEP * 128);
            for (int x = valid * 8 + r; x < STEP * 8; x += 128)
#pragma unroll
              for (int h = 0; h < DP / 64; ++h) *reinterpret_cast<uint4*>(vs + h * L::HALF + x * 16) = make_uint4(0u, 0u, 0u, 0u);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          }
        }
        float top[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) top[c] = max_nan(__uint_as_float(s[3 * c]), __uint_as_float(s[3 * c + 1]), __uint_as_float(s[3 * c + 2]));
#pragma unroll
        for (int c = 12; c < STEP; c += 2) top[(c >> 1) & 3] = max_nan(top[(c >> 1) & 3], __uint_as_float(s[c]), __uint_as_float(s[c + 1]));
        const float tm = max_nan(max_nan(top[0], top[1], top[2]), top[3], top[3]) * sc;
        if (j == 0) {
          m = tm;
        } else {
          const bool grow = !(tm <= m + GROW);  // a NaN too
          if (__any_sync(0xFFFFFFFFu, grow)) {
            // once the last step's product is in O, none runs on it until this step's P is there (the one
            // before the last was in O before this S, so that the barrier's parity says which)
            ok = __all_sync(0xFFFFFFFFu, wait_or_abort(&o_done[2 * half + (b ^ 1)], par[b ^ 1] ^ 1u, abort_flag)) != 0;
            if (!ok) return;
            tc_after();
            const float f = grow ? exp2f(m - tm) : 1.0f;
            l *= f;
            if (grow) m = tm;
#pragma unroll
            for (int c = 0; c < DP; c += 32) {
              uint32_t o[32];
              tc_ld32(o_at + c, o);
              tc_wait_ld();
#pragma unroll
              for (int x = 0; x < 32; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * f);
              tc_st32(o_at + c, o);
            }
          }
        }
        // scores of +inf make the row NaN (inf - inf), as a NaN does; a row of -inf so far has weights 0
        const float base = m == INFINITY ? NAN : (m == -INFINITY ? 0.0f : m) - P_SHIFT;
        const f32x2 scale2 = two(sc, sc), base2 = two(-base, -base);
        f32x2 sum[2] = {two(0.0f, 0.0f), two(0.0f, 0.0f)};
        uint32_t rest[FINE ? STEP / 2 : 1];
#pragma unroll
        for (int c = 0; c < STEP; c += 2) {
          const f32x2 x = fma2(two(__uint_as_float(s[c]), __uint_as_float(s[c + 1])), scale2, base2);
          const float2 y = one_by_one(x), p = make_float2(ex2(y.x), ex2(y.y));
          sum[(c >> 1) & 1] = add2(sum[(c >> 1) & 1], two(p.x, p.y));
          if constexpr (FINE)
            split16<T>(p.x, p.y, s[c >> 1], rest[c >> 1]);
          else
            s[c >> 1] = pack16<T>(p.x, p.y);
        }
        tc_st32(s_at, s);
        if constexpr (FINE) tc_st32(s_at + STEP / 2, rest);
        const float2 l01 = one_by_one(add2(sum[0], sum[1]));
        l += l01.x + l01.y;
        tc_wait_st();
        tc_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[2 * half + b]);
      };
      for (int j = 0; ok && j < g.steps; j += 2) {
        step(j, 0);
        if (ok && j + 1 < g.steps) step(j + 1, 1);
        ring.next();
        ring.next();
      }
      ok = ok && __all_sync(0xFFFFFFFFu, (g.steps & 1) != 0 ? wait_or_abort(&o_done[2 * half], par[0] ^ 1u, abort_flag)
                                                            : wait_or_abort(&o_done[2 * half + 1], par[1] ^ 1u, abort_flag));
      if (!ok) break;
      tc_after();
      const int rr = base_row + r;
      const int tok = min(rr, rows - 1) / a.rep;
      const long long row = static_cast<long long>(tok) * a.n_heads + g.kvh * a.rep + min(rr, rows - 1) - tok * a.rep;
      const long long part = static_cast<long long>(g.slot) * a.n_tokens * a.n_heads + row;
      if (rr < rows) a.part_ml[part] = make_float2(m, l);
      // a warp's 32 rows, 32 columns at a time, through Q's memory (its products are done), so that the
      // stores are whole rows; chunks of a row are swapped by the row
      uint8_t* mine = smem + half * L::SLOT + (warp & 3) * (L::SLOT / 4);
#pragma unroll
      for (int c = 0; c < DP; c += 32) {
        uint32_t o[32];
        __syncwarp();
        tc_ld32(o_at + c, o);
        tc_wait_ld();
#pragma unroll
        for (int x = 0; x < 8; ++x)
          *reinterpret_cast<uint4*>(mine + lane * 128 + ((x ^ (lane & 7)) << 4)) = make_uint4(o[4 * x], o[4 * x + 1], o[4 * x + 2], o[4 * x + 3]);
        __syncwarp();
#pragma unroll
        for (int y = 0; y < 8; ++y) {  // four rows of 32 columns
          const int q = 4 * y + (lane >> 3), ch = lane & 7;
          const long long to = __shfl_sync(0xFFFFFFFFu, part, q);
          const uint4 v = *reinterpret_cast<const uint4*>(mine + q * 128 + ((ch ^ (q & 7)) << 4));
          if (base_row + (warp & 3) * 32 + q < rows && c + 4 * ch < hd)
            *reinterpret_cast<uint4*>(a.part_o + to * hd + c + 4 * ch) = v;
        }
      }
      tc_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_free[half]);
    }
    if (!ok && lane == 0) {
      *abort_flag = 1;
      atomicOr(a.c.status, ST_TIMEOUT_FULL);
    }
  }

  __syncwarp();
  tc_before();
  __syncthreads();
  tc_after();
  if (warp == 1) {
    __syncwarp();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
}

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn kv_encode_tiled() {
  static EncodeTiledFn fn = nullptr;
  if (fn == nullptr) {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(p);
  }
  return fn;
}

}  // namespace

bool pool_map(CUtensorMap* map, const uint16_t* base, const KvView& c, uint32_t type) {
  EncodeTiledFn enc = kv_encode_tiled();
  if (enc == nullptr) return false;
  const int ps = 1 << c.ps_shift;
  const cuuint64_t dims[3] = {(cuuint64_t)c.hd, (cuuint64_t)c.n_kv * ps, (cuuint64_t)c.n_pages};
  const cuuint64_t strides[2] = {(cuuint64_t)c.hd * 2, (cuuint64_t)c.page_stride * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)(ps < TILE ? ps : TILE), 1};
  const cuuint32_t estr[3] = {1, 1, 1};
  return enc(map, type == TYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
             const_cast<uint16_t*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

namespace {

template <typename T, int DP, int MT, bool FINE>
cudaError_t launch_tc_as(const AttnArgs& a, uint32_t type, cudaStream_t st) {
  using L = TcLayout<DP, MT>;
  static const cudaError_t set = allow_smem(attn_tc_kernel<T, DP, MT, FINE>, L::ALLOC);
  if (set != cudaSuccess) return set;
  CUtensorMap kmap, vmap;
  if (!pool_map(&kmap, a.c.k + a.layer_off, a.c, type) || !pool_map(&vmap, a.c.v + a.layer_off, a.c, type)) return cudaErrorInvalidValue;
  return launch_dependent(attn_tc_kernel<T, DP, MT, FINE>, dim3(a.pre_ctas), dim3(TC_THREADS), L::ALLOC, st, a, kmap, vmap);
}

template <typename T, int DP>
cudaError_t launch_tc_rows(const AttnArgs& a, uint32_t type, cudaStream_t st) {
  if (a.pre_rows == 128) return launch_tc_as<T, DP, 1, true>(a, type, st);
  return a.out_f32 ? launch_tc_as<T, DP, 2, true>(a, type, st) : launch_tc_as<T, DP, 2, false>(a, type, st);
}

template <typename T>
cudaError_t launch_tc(const AttnArgs& a, uint32_t type, cudaStream_t st) {
  return a.c.hd <= 64 ? launch_tc_rows<T, 64>(a, type, st) : launch_tc_rows<T, 128>(a, type, st);
}

}  // namespace

cudaError_t launch_attn_tc(const AttnArgs& a, uint32_t type, cudaStream_t st) {
  return type == TYPE_F16 ? launch_tc<__half>(a, type, st) : launch_tc<__nv_bfloat16>(a, type, st);
}

}  // namespace ex
