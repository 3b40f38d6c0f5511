// kvattn_tc.cu -- the shared pass of attention over a paged cache on the 5th-generation tensor cores:
// the queries of all sequences, stacked, against the prefix that they share.
//
// One block takes up to MT x 128 rows (tokens x heads of a key/value head's group) along its piece of
// the prefix, 128 positions at a time.  Per tile and 128 rows: S = Q K^T into 128 columns of tensor
// memory, one thread a row takes the row's maximum, exponentials and sum, writes P in the cache's type
// over S, and O += P V accumulates in tensor memory with P as the tensor-memory operand.  With MT = 2
// the products of one half of the rows run while the other half is in its softmax, and both read the
// same tiles of K and V.  A row's reference maximum moves only when the maximum has grown by more than
// GROW (in log2 units); then O and the sum are rescaled, which after the first tiles is rare.
//
// Warps: 0 brings K and V by TMA (a box a page and 64 elements; 128-byte swizzle) through a ring of
// slots, 1 issues the products, 4..7 and 8..11 are the rows.  S, P: columns 128 x; O: columns
// 256 + 128 x of half x.  Tensor memory holds the whole accumulation, so shared memory is Q and the ring.
//
// Bound: per tile and 128 rows the two products take 2 x 512 cycles of the tensor pipe (head_dim 128)
// and the exponentials 1024 of the special-function units, beside 64 KB of K and V from L2 or HBM.
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
  static constexpr int N_BARS = 2 * SLOTS + 4 * 2 + 1;
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

__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(static_cast<int>(add))
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(static_cast<int>(add))
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
__device__ __forceinline__ uint64_t sw128_desc(uint32_t addr, uint32_t leading) {
  return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)(leading >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
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

// A place in the ring of slots, and the parity of its filling.
template <int NS>
struct Ring {
  int slot = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next() {
    if (++slot == NS) {
      slot = 0;
      phase ^= 1u;
    }
  }
};

// A block of rows along consecutive tiles of the prefix.
struct Segment {
  int kvh, row0, tile0, n, slot;
};
__device__ __forceinline__ Segment segment_at(const TcCut& c, long long at, long long end, int pre_rows) {
  Segment s;
  const long long block = at / c.tiles;
  s.tile0 = static_cast<int>(at - block * c.tiles);
  s.n = static_cast<int>(min(static_cast<long long>(c.tiles - s.tile0), end - at));
  s.kvh = static_cast<int>(block / c.row_blocks);
  s.row0 = static_cast<int>(block - static_cast<long long>(s.kvh) * c.row_blocks) * pre_rows;
  s.slot = static_cast<int>(blockIdx.x - block * c.tiles / c.per);
  return s;
}

template <typename T, int DP, int MT>
__global__ void __launch_bounds__(TC_THREADS, 1)
    attn_tc_kernel(const AttnArgs a, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
  using L = TcLayout<DP, MT>;
  constexpr int CH = DP / 8, NS = L::SLOTS;
  constexpr uint32_t FMT = exponent16<T>() == exponent16<__half>() ? 0u : 1u;
  // D fp32, A and B of the type, M = 128; N = 128 for S, DP for O, whose B is read across its rows
  constexpr uint32_t IDESC_S = (1u << 4) | (FMT << 7) | (FMT << 10) | ((128u >> 3) << 17) | ((128u >> 4) << 24);
  constexpr uint32_t IDESC_O = (1u << 4) | (FMT << 7) | (FMT << 10) | (1u << 16) | ((uint32_t(DP) >> 3) << 17) | ((128u >> 4) << 24);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::BARS);  // a ring slot's boxes landed
  uint64_t* empty = full + NS;                                   // the products that read it are done
  uint64_t* q_full = empty + NS;                                 // [half]: Q is in shared memory (128 threads)
  uint64_t* s_full = q_full + 2;                                 // [half]: S is in tensor memory
  uint64_t* p_full = s_full + 2;                                 // [half]: P is (128 threads)
  uint64_t* o_full = p_full + 2;                                 // [half]: the segment's O is
  uint64_t* fin = o_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::MISC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::MISC + 4);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < NS; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 128);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 128);
      mbar_init(&o_full[i], 1);
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
  const uint32_t tmem = *tmem_slot;
  pdl_enter_grid();

  const int shared = shared_of(a);
  const TcCut cut = tc_cut(a, shared);
  const long long begin = blockIdx.x * cut.per, end = min(cut.total, begin + cut.per);

  // registers: 384 x 168 at launch, from here on 128 x 64 and 256 x 216 (a row's 128 scores and 32 of O)
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
  if (warp == 0) {
    // K of tile 0, V of tile 0, K of tile 1, ...: the order in which the products need them
    const int box = min(1 << a.c.ps_shift, TC_TILE);  // positions a box holds
    const int32_t* table = a.c.table + static_cast<long long>(a.shared_seq) * a.c.max_pages;
    Ring<NS> ring;
    int issued = 0;  // slots filled, NS at most
    bool ok = true;
    for (long long at = begin; ok && at < end;) {
      const Segment g = segment_at(cut, at, end, a.pre_rows);
      at += g.n;
      for (int i = 0; ok && i < g.n; ++i) {
        const int p0 = (g.tile0 + i) * TC_TILE;
        const int boxes = (min(TC_TILE, shared - p0) + box - 1) / box;
        int page = 0;
        const int p = p0 + lane * box;
        if (lane < boxes) {
          page = table[p >> a.c.ps_shift];
          if (page < 0 || page >= a.c.n_pages) {
            atomicOr(a.c.status, ST_BAD_CACHE);
            page = 0;
          }
        }
        for (int kv = 0; kv < 2; ++kv, ring.next()) {
          const int slot = ring.slot;
          ok = __all_sync(0xFFFFFFFFu, wait_or_abort(&empty[slot], ring.phase ^ 1u, abort_flag));
          if (!ok) break;
          issued = min(issued + 1, NS);
          if (lane == 0) mbar_arrive_expect_tx(&full[slot], boxes * box * DP * 2);
          __syncwarp();
          if (lane < boxes) {
            const uint32_t dst = smem_u32(smem + L::RING + slot * L::SLOT) + lane * box * 128;
            const int y = (g.kvh << a.c.ps_shift) + (p & ((1 << a.c.ps_shift) - 1));
#pragma unroll
            for (int h = 0; h < DP / 64; ++h) tma_3d(dst + h * L::HALF, kv == 0 ? &kmap : &vmap, 64 * h, y, page, &full[slot]);
          }
        }
      }
    }
    if (lane == 0) {
      if (!ok) {
        *abort_flag = 1;
        atomicOr(a.c.status, ST_TIMEOUT_EMPTY);
      }
      bool drained = true;  // no copy may still be landing when the block exits
      for (int n = 0; n < issued; ++n) {  // the last filling of each slot, from the oldest
        const int back = issued - n;
        const int slot = ring.slot - back + (ring.slot < back ? NS : 0);
        if (!mbar_wait(&full[slot], ring.phase ^ (ring.slot < back ? 1u : 0u))) drained = false;
      }
      if (!drained) atomicOr(a.c.status, ST_TIMEOUT_DRAIN);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t q_s = smem_u32(smem), ring_s = smem_u32(smem + L::RING);
      Ring<NS> ring;
      uint32_t segs = 0, tiles_done = 0;
      bool ok = true;
      auto slot_ready = [&](const Ring<NS>& r) { return spin(&full[r.slot], r.phase, abort_flag); };
      auto product_s = [&](int half, int slot) {
        const uint64_t qd = sw128_desc(q_s + half * L::SLOT, 16), kd = sw128_desc(ring_s + slot * L::SLOT, 16);
#pragma unroll
        for (int k = 0; k < DP / 16; ++k) {
          const uint64_t off = static_cast<uint64_t>(((k / 4) * L::HALF + (k % 4) * 32) >> 4);
          mma_ss(tmem + 128 * half, qd + off, kd + off, IDESC_S, k > 0);
        }
        tc_commit(&s_full[half]);
      };
      for (long long at = begin; ok && at < end; ++segs) {
        const Segment g = segment_at(cut, at, end, a.pre_rows);
        at += g.n;
        ok = slot_ready(ring);
#pragma unroll
        for (int h = 0; h < MT; ++h) {
          ok = ok && spin(&q_full[h], segs & 1u, abort_flag);
          if (!ok) break;
          tc_after();
          product_s(h, ring.slot);
        }
        if (!ok) break;
        tc_commit(&empty[ring.slot]);
        ring.next();
        for (int i = 0; i < g.n; ++i, ++tiles_done) {
          const bool more = i + 1 < g.n;
          const Ring<NS> v = ring;
          ring.next();
          const Ring<NS> k = ring;
          if (more) ring.next();
          ok = slot_ready(v);
#pragma unroll
          for (int h = 0; h < MT; ++h) {
            ok = ok && spin(&p_full[h], tiles_done & 1u, abort_flag);
            if (!ok) break;
            tc_after();
            const uint64_t vd = sw128_desc(ring_s + v.slot * L::SLOT, L::HALF);
#pragma unroll
            for (int s = 0; s < TC_TILE / 16; ++s)
              mma_ts(tmem + 256 + 128 * h, tmem + 128 * h + 8 * s, vd + static_cast<uint64_t>((s * 2048) >> 4), IDESC_O, i > 0 || s > 0);
            if (more) {
              if (h == 0) ok = slot_ready(k);
              if (!ok) break;
              product_s(h, k.slot);
            } else {
              tc_commit(&o_full[h]);
            }
          }
          if (!ok) break;
          tc_commit(&empty[v.slot]);
          if (more) tc_commit(&empty[k.slot]);
        }
      }
      if (!ok) {
        *abort_flag = 1;
        atomicOr(a.c.status, ST_TIMEOUT_FULL);
      }
      tc_commit(fin);  // all products are done before tensor memory is given back
      if (!mbar_wait(fin, 0)) atomicOr(a.c.status, ST_TIMEOUT_DRAIN);
    }
  }
  } else if (warp < 4 + 4 * MT) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    const int half = (warp - 4) >> 2, r = threadIdx.x & 127;  // the thread's row of its half
    const uint32_t lane_base = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t s_at = lane_base + 128 * half, o_at = lane_base + 256 + 128 * half;
    const int rows = a.n_tokens * a.rep, hd = a.c.hd;
    const float sc = fabsf(a.scale);
    const uint32_t flip = a.scale < 0.0f ? 0x80008000u : 0u;  // a negative scale: -Q, so that a maximum is a maximum
    uint32_t segs = 0, tiles_done = 0;
    Ring<NS> ring;
    bool ok = true;
    for (long long at = begin; ok && at < end; ++segs) {
      const Segment g = segment_at(cut, at, end, a.pre_rows);
      at += g.n;
      const int base_row = g.row0 + half * 128;
#pragma unroll 4
      for (int x = r; x < 128 * CH; x += 128) {
        const int qr = x / CH, ch = x % CH, rr = base_row + qr;
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (rr < rows && ch * 8 < hd) {
          const int tok = rr / a.rep, head = g.kvh * a.rep + rr - tok * a.rep;
          v = *reinterpret_cast<const uint4*>(a.q + (static_cast<long long>(tok) * a.n_heads + head) * hd + ch * 8);
          v.x ^= flip;
          v.y ^= flip;
          v.z ^= flip;
          v.w ^= flip;
        }
        *reinterpret_cast<uint4*>(smem + half * L::SLOT + (ch / 8) * L::HALF + qr * 128 + (((ch & 7) ^ (qr & 7)) << 4)) = v;
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      mbar_arrive(&q_full[half]);

      float m = -INFINITY, l = 0.0f;
      for (int i = 0; i < g.n; ++i, ++tiles_done) {
        ok = __all_sync(0xFFFFFFFFu, wait_or_abort(&s_full[half], tiles_done & 1u, abort_flag));
        if (!ok) break;
        tc_after();
        uint32_t s[128];
#pragma unroll
        for (int c = 0; c < 128; c += 32) tc_ld32(s_at + c, s + c);
        tc_wait_ld();
        const int valid = shared - (g.tile0 + i) * TC_TILE;
        if (valid < TC_TILE) {
#pragma unroll
          for (int c = 0; c < 128; ++c)
            if (c >= valid) s[c] = 0xFF800000u;
        }
        float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < 128; ++c) top[c & 3] = fmaxf(top[c & 3], __uint_as_float(s[c]));
        const float tm = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * sc;
        if (i == 0) {
          m = tm;
        } else {
          const bool grow = tm > m + GROW || (m == -INFINITY && tm > m);
          if (__any_sync(0xFFFFFFFFu, grow)) {
            // the products before this S are done, and none is running on O
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
        const float base = (m == -INFINITY ? 0.0f : m) - P_SHIFT;
        float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c < 128; c += 2) {
          const float p0 = ex2(fmaf(__uint_as_float(s[c]), sc, -base)), p1 = ex2(fmaf(__uint_as_float(s[c + 1]), sc, -base));
          sum[(c >> 1) & 1] += p0;
          sum[2 + ((c >> 1) & 1)] += p1;
          s[c >> 1] = pack16<T>(p0, p1);
        }
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        tc_st32(s_at, s);
        tc_st32(s_at + 32, s + 32);
        ring.next();  // past K
        if (valid < TC_TILE && half == 0) {
          // V past the prefix's end is what memory held: 0 for the product
          ok = __all_sync(0xFFFFFFFFu, wait_or_abort(&full[ring.slot], ring.phase, abort_flag));
          if (!ok) break;
          uint8_t* vs = smem + L::RING + ring.slot * L::SLOT;
          for (int x = valid * 8 + r; x < TC_TILE * 8; x += 128)
#pragma unroll
            for (int h = 0; h < DP / 64; ++h) *reinterpret_cast<uint4*>(vs + h * L::HALF + x * 16) = make_uint4(0u, 0u, 0u, 0u);
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        ring.next();  // past V
        tc_wait_st();
        tc_before();
        mbar_arrive(&p_full[half]);
      }
      ok = ok && __all_sync(0xFFFFFFFFu, wait_or_abort(&o_full[half], segs & 1u, abort_flag));
      if (!ok) break;
      tc_after();
      const int rr = base_row + r;
      const int tok = min(rr, rows - 1) / a.rep;
      const long long row = static_cast<long long>(tok) * a.n_heads + g.kvh * a.rep + min(rr, rows - 1) - tok * a.rep;
      const long long part = static_cast<long long>(g.slot) * a.n_tokens * a.n_heads + row;
      if (rr < rows) a.part_ml[part] = make_float2(m, l);
#pragma unroll
      for (int c = 0; c < DP; c += 32) {
        uint32_t o[32];
        __syncwarp();
        tc_ld32(o_at + c, o);
        tc_wait_ld();
        if (rr < rows) {
          float4* dst = reinterpret_cast<float4*>(a.part_o + part * hd + c);
#pragma unroll
          for (int x = 0; x < 8; ++x)
            if (c + 4 * x < hd) dst[x] = make_float4(__uint_as_float(o[4 * x]), __uint_as_float(o[4 * x + 1]), __uint_as_float(o[4 * x + 2]),
                                 __uint_as_float(o[4 * x + 3]));
        }
      }
      __syncwarp();
      tc_before();
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

bool pool_map(CUtensorMap* map, const uint16_t* base, const KvView& c, uint32_t type, int most) {
  EncodeTiledFn enc = kv_encode_tiled();
  if (enc == nullptr) return false;
  const int ps = 1 << c.ps_shift;
  const cuuint64_t dims[3] = {(cuuint64_t)c.hd, (cuuint64_t)c.n_kv * ps, (cuuint64_t)c.n_pages};
  const cuuint64_t strides[2] = {(cuuint64_t)c.hd * 2, (cuuint64_t)c.page_stride * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)(ps < most ? ps : most), 1};
  const cuuint32_t estr[3] = {1, 1, 1};
  return enc(map, type == TYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
             const_cast<uint16_t*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

namespace {

template <typename T, int DP, int MT>
cudaError_t launch_tc_as(const AttnArgs& a, uint32_t type, cudaStream_t st) {
  using L = TcLayout<DP, MT>;
  static const cudaError_t set = cudaFuncSetAttribute(attn_tc_kernel<T, DP, MT>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::ALLOC);
  if (set != cudaSuccess) return set;
  CUtensorMap kmap, vmap;
  if (!pool_map(&kmap, a.c.k + a.layer_off, a.c, type, TC_TILE) || !pool_map(&vmap, a.c.v + a.layer_off, a.c, type, TC_TILE)) return cudaErrorInvalidValue;
  return launch_dependent(attn_tc_kernel<T, DP, MT>, dim3(a.pre_ctas), dim3(TC_THREADS), L::ALLOC, st, a, kmap, vmap);
}

template <typename T>
cudaError_t launch_tc(const AttnArgs& a, uint32_t type, cudaStream_t st) {
  if (a.c.hd <= 64) return a.pre_rows == 128 ? launch_tc_as<T, 64, 1>(a, type, st) : launch_tc_as<T, 64, 2>(a, type, st);
  return a.pre_rows == 128 ? launch_tc_as<T, 128, 1>(a, type, st) : launch_tc_as<T, 128, 2>(a, type, st);
}

}  // namespace

cudaError_t launch_attn_tc(const AttnArgs& a, uint32_t type, cudaStream_t st) {
  return type == TYPE_F16 ? launch_tc<__half>(a, type, st) : launch_tc<__nv_bfloat16>(a, type, st);
}

}  // namespace ex
