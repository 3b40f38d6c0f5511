// kvattn.cu -- attention of a batch's last tokens over a paged cache, with a prefix that all its
// sequences share read once.
//
// Mathematics.  The softmax of a row over a set of positions is the join of its parts: with, for each
// part, m = max s_j, l = sum 2^(s_j - m) and o = sum 2^(s_j - m) v_j (scores in log2 units), the whole
// is M = max m, L = sum l 2^(m - M), out = sum o 2^(m - M) / L.  So the queries of all sequences that
// share a prefix are stacked into one matrix against it (rows = tokens x heads of the group), each
// sequence's own positions are a second part, long parts are split further, and a last kernel joins.
//
// A row's mask is a number, the positions it sees.  Positions outside a block's range are loaded as
// zeros, so memory past a sequence's end may hold anything.  A sequence one of whose tokens sees less
// than the whole prefix takes no part in the shared pass: its own pass starts at position 0, which
// keeps the shared pass free of masks by row.
//
// Launches: the shared pass (kvattn_tc.cu; the rows kernel here for heads above 128 elements or at most
// 16 rows), beside it the own pass (kvattn_one.cu for single tokens, else the rows kernel here), then the
// join.  Floor: K and V of the prefix and of each sequence once, or 4 operations an element of K for each
// row.  Measured, 32 query heads on 8 of 128 elements, calls back to back with inputs in rotation: 128 single tokens
// behind a prefix of 32k with 33 to 2000 own positions in f16 189 us (floor 101, bytes), 32 behind 4k with up to 511
// in bf16 33 us (8, bytes; three kernels' latencies), 32 questions of 1 to 64 tokens behind 8k in f16 194 us (84,
// operations).  The same inputs for some milliseconds: 167, 32 and 182 to 191 us; the changes' figures below and in
// the other files are of that kind.
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <mutex>

#include "capi_internal.h"
#include "kv.cuh"
#include "kvattn.cuh"
#include "kvattn_mma.cuh"

namespace ex {
namespace {

constexpr int ROWS_THREADS = 160;

template <int DP, int WM>
struct RowsLayout {
  static constexpr int ROWS = 16 * WM;
  static constexpr int SLOTS = DP == 64 ? 6 : 3;
  static constexpr int HALF = TILE * 128;
  static constexpr int SLOT = HALF * (DP / 64);  // a tile of K, or of V
  static constexpr int Q_AT = SLOTS * SLOT;
  static constexpr int BARS = Q_AT + ROWS * DP * 2;
  static constexpr int JOIN_BYTES = WM == 1 ? 4 * 16 * DP * 4 : 0;  // over the ring, when it is done with
  static constexpr int ALLOC = BARS + 16 * SLOTS + 64 + 1024;
  static_assert(JOIN_BYTES <= SLOTS * SLOT, "the join fits the ring");
};

// Row r of entry e (or of the batch, in the prefix) against tiles [t_begin, t_end), by one warp: a lane has
// elements lane + 32 x, and a position it does not see is not read.
template <typename T>
__device__ __noinline__ void row_again(const AttnArgs& a, const Entry& e, int kvh, int r, int t_begin, int t_end, int pre, bool whole, int slot) {
  const int lane = threadIdx.x & 31, hd = a.c.hd, tok = e.t0 + r / a.rep;
  const long long row = static_cast<long long>(tok) * a.n_heads + kvh * a.rep + r % a.rep;
  const int hi = pre ? e.len : e.len - e.nq + r / a.rep + 1;
  const int32_t* table = a.c.table + static_cast<long long>(e.row) * a.c.max_pages;
  auto value = [&](const uint16_t* base, int p, int d) {
    const int page = min(max(table[p >> a.c.ps_shift], 0), a.c.n_pages - 1);
    const uint16_t* at = base + a.layer_off + page * a.c.page_stride +
                         ((static_cast<long long>(kvh) << a.c.ps_shift) + (p & ((1 << a.c.ps_shift) - 1))) * hd + d;
    return unpack16<T>(*at).x;
  };
  float m = -INFINITY, l = 0.0f, o[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
  for (int p = max(e.start, t_begin * TILE); p < min(hi, t_end * TILE); ++p) {
    float s = 0.0f;
    for (int d = lane; d < hd; d += 32) s = fmaf(unpack16<T>(a.q[row * hd + d]).x, value(a.c.k, p, d), s);
#pragma unroll
    for (int y = 16; y > 0; y >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, y);
    s *= a.scale;
    const float mn = fmaxf(m, s), base = mn == -INFINITY ? 0.0f : mn, f = exp2f(m - base), w = exp2f(s - base + P_SHIFT);
    m = mn;
    l = l * f + w;
#pragma unroll
    for (int x = 0; x < 8; ++x)
      if (lane + 32 * x < hd) o[x] = o[x] * f + w * value(a.c.v, p, lane + 32 * x);
  }
  const long long part = static_cast<long long>(slot) * a.n_tokens * a.n_heads + row;
#pragma unroll
  for (int x = 0; x < 8; ++x) {
    const int d = lane + 32 * x;
    if (d >= hd) continue;
    if (!whole) {
      a.part_o[part * hd + d] = o[x];
    } else {
      const float v = hi > 0 ? o[x] / l : 0.0f;
      if (a.out_f32)
        static_cast<float*>(a.out)[row * hd + d] = v;
      else
        static_cast<uint16_t*>(a.out)[row * hd + d] = round16<T>(v);
    }
  }
  if (!whole && lane == 0) a.part_ml[part] = make_float2(m, l);
}

// One block: 16 * WM rows of one key/value head against one part of the prefix (PRE) or of an entry's
// own positions.  Warp 4 brings K and V by TMA (128-byte swizzle; dims past head_dim read as 0).  Of the
// other four, with WM = 4 each has 16 rows and all positions of a tile, with WM = 1 all have the same 16
// rows and 16 positions of each tile, and join at the end.  P is rounded to the cache's type for its
// product, as the tensor cores take it, or (FINE: with WM = 1, where bytes bound, and where the result is fp32)
// goes in two numbers of the type; its sum l is of the unrounded values.  Fragments of warp products, since an own pass has few rows on few
// positions.  The own passes of 32 questions of 1 to 64 tokens on 64 to 200 positions: 41 us, bound by
// latency, a tile's two products and its softmax in turn in each warp.
template <typename T, int DP, int WM, bool FINE>
__global__ void __launch_bounds__(ROWS_THREADS, DP == 256 ? 1 : DP == 128 ? 2 : 3)
    attn_rows_kernel(const __grid_constant__ AttnArgs a, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const int pre) {
  using L = RowsLayout<DP, WM>;
  constexpr int ROWS = L::ROWS, NT = WM == 1 ? 2 : 8, CH = DP / 8, ST = L::SLOTS;
  extern __shared__ uint8_t smem_raw[];
  __shared__ int any_odd;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::BARS);
  uint64_t* empty = full + ST;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(empty + ST);
  if (threadIdx.x == 0) {
    for (int i = 0; i < ST; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 4);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  __syncthreads();
  if (pre)
    pdl_enter_pair();
  else
    own_enter(a);
  const uint32_t q_s = smem_u32(smem + L::Q_AT);
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int kvh = blockIdx.y, split = blockIdx.z;
  const int hd = a.c.hd, rep = a.rep;
  const int shared = shared_of(a);

  // the block's rows: tokens x heads of the group, from row r0 of entry e (or of the whole batch)
  Entry e{a.shared_seq, 0, a.n_tokens, shared, 0, true};
  int r0 = blockIdx.x * ROWS;
  if (!pre) {
    int i = blockIdx.x, blk = 0;
    const int per_entry = (rep + ROWS - 1) / ROWS;
    if (a.q_start == nullptr) {
      i = blockIdx.x / per_entry;
      blk = blockIdx.x - i * per_entry;
    } else {  // the entry whose blocks hold this one: a scan of the entries' block counts, a warp wide
      int before = 0, found = -1;
      for (int base = 0; base < a.n_batch && found < 0; base += 32) {
        int cnt = 0;
        if (base + lane < a.n_batch) {
          const Entry x = entry_of(a, base + lane, shared);
          cnt = (x.nq * rep + ROWS - 1) / ROWS;
        }
        int inc = cnt;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int y = __shfl_up_sync(0xFFFFFFFFu, inc, o);
          if (lane >= o) inc += y;
        }
        const uint32_t past = __ballot_sync(0xFFFFFFFFu, before + inc > static_cast<int>(blockIdx.x));
        if (past != 0) {
          const int src = __ffs(past) - 1;
          found = base + src;
          blk = blockIdx.x - (before + __shfl_sync(0xFFFFFFFFu, inc - cnt, src));
        }
        before += __shfl_sync(0xFFFFFFFFu, inc, 31);
      }
      if (found < 0) {
        own_leave(a);
        return;
      }
      i = found;
    }
    e = entry_of(a, i, shared);
    r0 = blk * ROWS;
  }
  const int n_rows = min(ROWS, e.nq * rep - r0);
  if (n_rows <= 0) {
    if (!pre) own_leave(a);
    return;
  }
  const bool whole = a.n_pre + a.n_own == 1;  // the only part there is: no join follows

  // what the rows see: row r is token r / rep; rows past the end see what the last one does
  const int last_tok = (r0 + n_rows - 1) / rep, first_tok = r0 / rep;
  const int block_hi = e.row < 0 ? 0 : pre ? shared : max(0, e.len - e.nq + last_tok + 1);
  const int block_lo_hi = e.row < 0 ? 0 : pre ? shared : max(0, e.len - e.nq + first_tok + 1);
  const Cut cut = pre ? cut_of(0, shared, a.n_pre) : cut_of(e.start, e.row < 0 ? 0 : e.len, a.n_own);
  if (split > 0 && split >= cut.used) {  // the join knows
    if (!pre) own_leave(a);
    return;
  }
  const int t_begin = cut.first + split * cut.per;
  const int t_end = min(min(t_begin + cut.per, cut.first + cut.tiles), (block_hi + TILE - 1) / TILE);
  if (w == 4) {
    const int32_t* table = a.c.table + static_cast<long long>(max(0, e.row)) * a.c.max_pages;
    Ring<ST> ring;
    int issued = 0;
    bool ok = true;
    Pages pages(a.c, table, t_begin * TILE, block_hi);
    for (int t = 2 * t_begin; t < 2 * t_end; ++t) {  // K of a tile, then its V
      const int p0 = (t >> 1) * TILE, page = pages.at(p0);
      ok = __all_sync(0xFFFFFFFFu, wait_or_abort(&empty[ring.slot], ring.phase ^ 1u, abort_flag)) != 0;
      if (!ok) break;
      bring_tile<DP, TILE>(a.c, page, (t & 1) == 0 ? &kmap : &vmap, smem_u32(smem + ring.slot * L::SLOT), kvh, p0, block_hi,
                           &full[ring.slot]);
      issued = min(issued + 1, ST);
      ring.next();
    }
    if (lane == 0) {
      if (!ok) {
        *abort_flag = 1;
        atomicOr(a.c.status, ST_TIMEOUT_EMPTY);
      }
      drain<ST>(ring, issued, full, a.c.status);
    }
    return;
  }

  const int wr = WM == 4 ? w * 16 : 0;  // the warp's rows of the block
  int hi[2], tok[2], head[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = r0 + min(wr + (lane >> 2) + 8 * h, n_rows - 1);
    tok[h] = e.t0 + r / rep;
    head[h] = kvh * rep + r % rep;
    hi[h] = e.row < 0 ? 0 : pre ? shared : e.len - e.nq + r / rep + 1;
  }
  {
    // a thread takes one chunk of eight elements of every (128 / CH)th row; rows past the end are 0
    constexpr int EACH = ROWS * CH / 128, STEP = ROWS / EACH;
    const int ch = threadIdx.x % CH;
    uint4 v[EACH];
    const int dq = STEP / rep, dr = STEP - dq * rep;
    int r = threadIdx.x / CH, tok_r = (r0 + r) / rep, g = r0 + r - tok_r * rep;
#pragma unroll
    for (int x = 0; x < EACH; ++x) {
      v[x] = ch * 8 < hd && r < n_rows ? *reinterpret_cast<const uint4*>(
                                             a.q + (static_cast<long long>(e.t0 + tok_r) * a.n_heads + kvh * rep + g) * hd + ch * 8)
                                       : make_uint4(0u, 0u, 0u, 0u);
      r += STEP;
      tok_r += dq;
      g += dr;
      if (g >= rep) {
        g -= rep;
        ++tok_r;
      }
    }
#pragma unroll
    for (int x = 0; x < EACH; ++x) {
      const int r = threadIdx.x / CH + x * STEP;
      *reinterpret_cast<uint4*>(smem + L::Q_AT + r * DP * 2 + ((ch ^ (r & 7)) << 4)) = v[x];
    }
  }
  named_bar_sync(1, 128);

  float o[DP / 8][4];
#pragma unroll
  for (int i = 0; i < DP / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
  const int kw = WM == 1 ? w * 16 : 0;  // the warp's positions of a tile
  const int g = lane >> 3, lr = lane & 7;

  // A given-up wait does not leave the loop: its barriers are all four warps'.  What follows it is void,
  // and the status says so.
  bool ok = true, odd = false;
  Ring<ST> ring;
  for (int t = t_begin; t < t_end; ++t) {
    ok = ok && __all_sync(0xFFFFFFFFu, wait_or_abort(&full[ring.slot], ring.phase, abort_flag));
    const uint32_t ks = smem_u32(smem + ring.slot * L::SLOT);
    const int k_slot = ring.slot;
    ring.next();
    uint8_t* vp = smem + ring.slot * L::SLOT;
    const uint32_t vs = smem_u32(vp);

    float s[NT][4];
#pragma unroll
    for (int i = 0; i < NT; ++i) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.0f;
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk) {
      uint32_t qa[4];
      const int qr = wr + lr + (g & 1) * 8, qc = 2 * kk + (g >> 1);
      ldsm4(qa, q_s + qr * DP * 2 + ((qc ^ (qr & 7)) << 4));
#pragma unroll
      for (int i = 0; i < NT; i += 2) {
        uint32_t kf[4];
        const int key = kw + i * 8 + lr + (g >> 1) * 8, ch = 2 * kk + (g & 1);
        ldsm4(kf, ks + (ch >> 3) * L::HALF + key * 128 + (((ch & 7) ^ (key & 7)) << 4));
        mma16816<T>(s[i], qa, kf[0], kf[1]);
        mma16816<T>(s[i + 1], qa, kf[2], kf[3]);
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&empty[k_slot]);
    const int p0 = t * TILE + kw;
    const bool masked = t * TILE < e.start || (t + 1) * TILE > block_lo_hi;
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        s[i][x] *= a.scale;
        if (masked) {
          const int p = p0 + i * 8 + (lane & 3) * 2 + (x & 1);
          if (p < e.start || p >= hi[x >> 1]) s[i][x] = -INFINITY;
        }
        top[x >> 1] = fmaxf(top[x >> 1], s[i][x]);
      }
    float base[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      top[h] = fmaxf(top[h], __shfl_xor_sync(0xFFFFFFFFu, top[h], 1));
      top[h] = fmaxf(top[h], __shfl_xor_sync(0xFFFFFFFFu, top[h], 2));
      const float mn = fmaxf(m[h], top[h]);
      base[h] = mn == -INFINITY ? 0.0f : mn;
      const float f = exp2f(m[h] - base[h]);
      l[h] *= f;
      m[h] = mn;
#pragma unroll
      for (int i = 0; i < DP / 8; ++i) {
        o[i][2 * h] *= f;
        o[i][2 * h + 1] *= f;
      }
    }
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        s[i][x] = ex2(s[i][x] - (base[x >> 1] - P_SHIFT));
        l[x >> 1] += s[i][x];
      }
    ok = ok && __all_sync(0xFFFFFFFFu, wait_or_abort(&full[ring.slot], ring.phase, abort_flag));
    // values that are no numbers, at positions that only some of the rows see
    if (masked && block_lo_hi < block_hi) {
      const int from = max(0, block_lo_hi - t * TILE), n = min(TILE, block_hi - t * TILE) - from;
      uint32_t most = 0;  // the largest magnitudes, as 16-bit integers
      for (int x = threadIdx.x; x < n * CH; x += 128) {
        const int key = from + x / CH, ch = x % CH;
        const uint4 v = *reinterpret_cast<const uint4*>(vp + (ch >> 3) * L::HALF + key * 128 + (((ch & 7) ^ (key & 7)) << 4));
        most = __vmaxu2(most, __vmaxu2(__vmaxu2(v.x & 0x7FFF7FFFu, v.y & 0x7FFF7FFFu), __vmaxu2(v.z & 0x7FFF7FFFu, v.w & 0x7FFF7FFFu)));
      }
      if ((most & 0xFFFFu) >= exponent16<T>() || (most >> 16) >= exponent16<T>()) odd = true;
    }
    // positions that are not the block's hold anything: their values count as 0
    const bool edge = t * TILE < e.start || (t + 1) * TILE > block_hi;
#pragma unroll
    for (int i = 0; i < NT; i += 2) {
      uint32_t pa[4], rest[4], keep[2] = {0xFFFFFFFFu, 0xFFFFFFFFu};
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const float p0v = s[i + (x >> 1)][2 * (x & 1)], p1v = s[i + (x >> 1)][2 * (x & 1) + 1];
        if constexpr (FINE)
          split16<T>(p0v, p1v, pa[x], rest[x]);
        else
          pa[x] = pack16<T>(p0v, p1v);
      }
      if (edge) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int p = p0 + (i + x) * 8 + (lane & 3) * 2;
          keep[x] = (p >= e.start && p < block_hi ? 0xFFFFu : 0u) | (p + 1 >= e.start && p + 1 < block_hi ? 0xFFFF0000u : 0u);
        }
      }
#pragma unroll
      for (int d = 0; d < DP / 16; ++d) {
        uint32_t vf[4];
        const int key = kw + i * 8 + lr + (g & 1) * 8, ch = 2 * d + (g >> 1);
        ldsm4t(vf, vs + (ch >> 3) * L::HALF + key * 128 + (((ch & 7) ^ (key & 7)) << 4));
        vf[0] &= keep[0];
        vf[1] &= keep[1];
        vf[2] &= keep[0];
        vf[3] &= keep[1];
        mma16816<T>(o[2 * d], pa, vf[0], vf[1]);
        mma16816<T>(o[2 * d + 1], pa, vf[2], vf[3]);
        if constexpr (FINE) {
          mma16816<T>(o[2 * d], rest, vf[0], vf[1]);
          mma16816<T>(o[2 * d + 1], rest, vf[2], vf[3]);
        }
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&empty[ring.slot]);
    ring.next();
  }
  if (!ok && lane == 0) {
    *abort_flag = 1;
    atomicOr(a.c.status, ST_TIMEOUT_FULL);
  }
  if (threadIdx.x == 0) any_odd = 0;
  named_bar_sync(1, 128);
  if (odd) any_odd = 1;
  named_bar_sync(1, 128);
  if (any_odd != 0) {
    // An infinity or NaN at a position that some rows do not see: its product with their weight of 0 has
    // spread to them.  Rare, so these rows are simply computed again, one position after the other.
    for (int r = w; r < n_rows; r += 4)
      row_again<T>(a, e, kvh, r0 + r, t_begin, t_end, pre, whole, (pre ? 0 : a.n_pre) + split);
    if (!pre) own_leave(a);
    return;
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    l[h] += __shfl_xor_sync(0xFFFFFFFFu, l[h], 1);
    l[h] += __shfl_xor_sync(0xFFFFFFFFu, l[h], 2);
  }

  const int slot = (pre ? 0 : a.n_pre) + split;
  const long long part = static_cast<long long>(slot) * a.n_tokens * a.n_heads;
  if constexpr (WM == 4) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (wr + (lane >> 2) + 8 * h >= n_rows) continue;
      const long long row = static_cast<long long>(tok[h]) * a.n_heads + head[h];
      if (!whole && (lane & 3) == 0) a.part_ml[part + row] = make_float2(m[h], l[h]);
#pragma unroll
      for (int i = 0; i < DP / 8; ++i) {
        const int d = i * 8 + (lane & 3) * 2;
        if (d >= hd) continue;
        if (whole)
          store_out<T>(a, row * hd + d, o[i][2 * h], o[i][2 * h + 1], l[h], hi[h] > 0);
        else
          *reinterpret_cast<float2*>(a.part_o + (part + row) * hd + d) = make_float2(o[i][2 * h], o[i][2 * h + 1]);
      }
    }
  } else {
    // join the four warps' positions: their m and l, then their sums through shared memory
    __shared__ float2 ml_s[4][16];
    float* o_s = reinterpret_cast<float*>(smem);
    if ((lane & 3) == 0) {
      ml_s[w][lane >> 2] = make_float2(m[0], l[0]);
      ml_s[w][(lane >> 2) + 8] = make_float2(m[1], l[1]);
    }
#pragma unroll
    for (int i = 0; i < DP / 8; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        *reinterpret_cast<float2*>(o_s + (w * 16 + (lane >> 2) + 8 * h) * DP + i * 8 + (lane & 3) * 2) =
            make_float2(o[i][2 * h], o[i][2 * h + 1]);
    named_bar_sync(1, 128);
    for (int x = threadIdx.x; x < n_rows * (DP / 2); x += 128) {
      const int r = x / (DP / 2), d = x % (DP / 2) * 2;
      float mm = -INFINITY;
#pragma unroll
      for (int y = 0; y < 4; ++y) mm = fmaxf(mm, ml_s[y][r].x);
      const float bs = mm == -INFINITY ? 0.0f : mm;
      float ll = 0.0f, o0 = 0.0f, o1 = 0.0f;
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const float f = exp2f(ml_s[y][r].x - bs);
        const float2 v = *reinterpret_cast<const float2*>(o_s + (y * 16 + r) * DP + d);
        ll += f * ml_s[y][r].y;
        o0 += f * v.x;
        o1 += f * v.y;
      }
      if (d >= hd) continue;
      const int rr = r0 + r;
      const long long row = static_cast<long long>(e.t0 + rr / rep) * a.n_heads + kvh * rep + rr % rep;
      const bool sees = e.row >= 0 && (pre || e.len - e.nq + rr / rep + 1 > 0);
      if (whole) {
        store_out<T>(a, row * hd + d, o0, o1, ll, sees);
      } else {
        *reinterpret_cast<float2*>(a.part_o + (part + row) * hd + d) = make_float2(o0, o1);
        if (d == 0) a.part_ml[part + row] = make_float2(mm, ll);
      }
    }
  }
  if (!pre) own_leave(a);
}

// Join the parts of each (token, head): a warp takes `heads` heads of a token, lane x elements 4 x ... and,
// in wide heads, 4 x + 128 ...  The parts' weights come first, a lane a part, then their sums AT_ONCE
// at a time: eight where rows are few and latency counts, else four.  Bound by latency (4096 rows of four
// parts: 10 to 15 us), with many rows by its instructions (32k rows: 27 us; issue slots 62 % in use).
template <typename T, bool WIDE, int AT_ONCE>
__global__ void __launch_bounds__(128) attn_join_kernel(const AttnArgs a, const int heads, const int per_token) {
  pdl_enter_grid();
  const int lane = threadIdx.x & 31, hd = a.c.hd;
  const int unit = static_cast<int>(blockIdx.x) * 4 + (threadIdx.x >> 5), t = unit / per_token;
  if (t >= a.n_tokens) return;
  int i = t;
  if (a.q_start != nullptr) {  // the last entry that starts at or before t: 32 of them at a time
    i = 0;
    for (int base = 0; base < a.n_batch; base += 32) {
      const bool at = base + lane < a.n_batch && a.q_start[base + lane] <= t;
      const uint32_t m = __ballot_sync(0xFFFFFFFFu, at);
      if (m != 0) i = base + 31 - __clz(m);
      if (m != 0xFFFFFFFFu) break;
    }
  }
  const int shared = shared_of(a);
  const Entry e = entry_of(a, i, shared);
  const bool sees = e.row >= 0 && t >= e.t0 && t < e.t0 + e.nq && e.len - e.nq + (t - e.t0) + 1 > 0;
  const int own_tiles = sees && a.own_ctas > 0 ? cut_of(e.start, e.len, 1).tiles : 0;
  const int n_rb = (a.rep + 15) / 16, per_entry = a.c.n_kv * n_rb;
  long long own_per = 1, own_first = 0;
  if (own_tiles > 0) {
    own_per = (static_cast<long long>(a.own_off[a.n_batch]) * per_entry + a.own_ctas - 1) / a.own_ctas;
    own_first = static_cast<long long>(a.own_off[i]) * per_entry;
  }
  const int own_slots = sees && a.own_ctas == 0 ? cut_of(e.start, e.len, a.n_own).used : 0;
  const TcCut pre = sees && e.shares && a.pre_rows > 0 ? tc_cut(a, shared) : TcCut{1, 1, 1, 1};
  const long long rows = static_cast<long long>(a.n_tokens) * a.n_heads;

  const int h0 = (unit - t * per_token) * heads;
  for (int head = h0; head < min(h0 + heads, a.n_heads); ++head) {
    const int kvh = head / a.rep, r = head - kvh * a.rep;
    const long long row = static_cast<long long>(t) * a.n_heads + head;
    int n_pre = 0, n_own = own_slots;
    long long cont = 0;  // single tokens: the row of the second own part
    if (sees && e.shares) {
      if (a.pre_rows > 0) {
        const int first = (kvh * pre.lines + (t * a.rep + r) / a.pre_rows / a.pre_width) * pre.tiles;
        n_pre = (first + pre.tiles - 1) / pre.per - first / pre.per + 1;
      } else {
        n_pre = cut_of(0, shared, a.n_pre).used;
      }
    }
    if (own_tiles > 0) {
      const long long first = own_first + static_cast<long long>(kvh * n_rb + r / 16) * own_tiles;
      const int c0 = static_cast<int>(first / own_per);
      n_own = static_cast<int>((first + own_tiles - 1) / own_per) - c0 + 1;
      cont = a.cont_row0 + static_cast<long long>(c0 + 1) * 16 + r % 16;
    }
    const int n = n_pre + n_own;
    auto row_of = [&](int x) {
      if (x < n_pre) return x * rows + row;
      x -= n_pre;
      return a.own_ctas > 0 && x > 0 ? cont + 16LL * (x - 1) : (a.n_pre + x) * rows + row;
    };
    float top = -INFINITY, l = 0.0f;
    float4 o[WIDE ? 2 : 1];
#pragma unroll
    for (int k = 0; k < (WIDE ? 2 : 1); ++k) o[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int b = 0; b < n; b += 32) {
      const float2 ml = b + lane < n ? a.part_ml[row_of(b + lane)] : make_float2(-INFINITY, 0.0f);
      float most = ml.x;
#pragma unroll
      for (int y = 16; y > 0; y >>= 1) most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, y));
      const float before = top;
      top = fmaxf(top, most);
      const float base = top == -INFINITY ? 0.0f : top;
      const float f = exp2f(ml.x - base), g = exp2f(before - base);
      float lw = f * ml.y;
#pragma unroll
      for (int y = 16; y > 0; y >>= 1) lw += __shfl_xor_sync(0xFFFFFFFFu, lw, y);
      l = l * g + lw;
#pragma unroll
      for (int k = 0; k < (WIDE ? 2 : 1); ++k) o[k] = make_float4(o[k].x * g, o[k].y * g, o[k].z * g, o[k].w * g);
      // a part that saw nothing may not have written its sums
      uint32_t some = __ballot_sync(0xFFFFFFFFu, ml.x != -INFINITY || ml.y != 0.0f);
      while (some != 0) {
        float4 v[AT_ONCE][WIDE ? 2 : 1];
        float w[AT_ONCE];
#pragma unroll
        for (int x = 0; x < AT_ONCE; ++x) {
          const int part = some != 0 ? __ffs(some) - 1 : -1;
          w[x] = __shfl_sync(0xFFFFFFFFu, f, max(part, 0));
          const float* src = a.part_o + row_of(b + max(part, 0)) * hd + lane * 4;
#pragma unroll
          for (int k = 0; k < (WIDE ? 2 : 1); ++k)
            v[x][k] = part >= 0 && lane * 4 + k * 128 < hd ? *reinterpret_cast<const float4*>(src + k * 128)
                                                           : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          if (part < 0) w[x] = 0.0f;
          some &= some - 1;
        }
#pragma unroll
        for (int x = 0; x < AT_ONCE; ++x)
#pragma unroll
          for (int k = 0; k < (WIDE ? 2 : 1); ++k) {
            o[k].x += w[x] * v[x][k].x;
            o[k].y += w[x] * v[x][k].y;
            o[k].z += w[x] * v[x][k].z;
            o[k].w += w[x] * v[x][k].w;
          }
      }
    }
#pragma unroll
    for (int k = 0; k < (WIDE ? 2 : 1); ++k) {
      const int d = lane * 4 + k * 128;
      if (d < hd) {
        store_out<T>(a, row * hd + d, o[k].x, o[k].y, l, sees);
        store_out<T>(a, row * hd + d + 2, o[k].z, o[k].w, l, sees);
      }
    }
  }
}

// How the work is divided: rows a block, and the parts of the prefix and of a sequence's own positions.
struct AttnPlan {
  int pre_wm, own_wm;
  int pre_blocks, own_blocks;
  int n_pre, n_own;
  int pre_rows, pre_ctas, pre_width;
  bool one;      // single tokens: kvattn_one.cu
  int own_ctas;
};

AttnPlan plan_of(int n_kv, int hd, bool ragged, int n_batch, int n_tokens, int n_heads, int shared_len, int max_len) {
  AttnPlan p{};
  const int sms = attn_sms();
  const int rep = n_heads / n_kv;
  const long long rows = static_cast<long long>(n_tokens) * rep;
  shared_len = std::max(0, std::min(shared_len, max_len));
  const int own_tiles = (std::max(0, max_len - shared_len) + TILE - 1) / TILE + 1;
  p.one = !ragged && hd <= 128 && n_batch <= ONE_MAX_BATCH;
  p.n_own = 1;
  const long long runs = static_cast<long long>(n_batch) * n_kv * ((rep + 15) / 16);  // of single tokens
  // short runs and no prefix: a block each, which needs no join; a tile takes a block about 0.5 us, a join 3
  const bool cut = p.one && (shared_len > 0 || own_tiles > 8) && runs * own_tiles <= INT_MAX;
  p.one = p.one && (cut || shared_len == 0);
  if (!p.one) {
    p.own_wm = rows <= 16LL * n_batch ? 1 : 4;
    const int own_rows = 16 * p.own_wm;
    p.own_blocks = static_cast<int>(ragged ? (rows + own_rows - 1) / own_rows + n_batch
                                           : static_cast<long long>(n_batch) * ((rep + own_rows - 1) / own_rows));
    // two blocks an SM: enough parts for two rounds of them, none shorter than two tiles
    const long long target = 4LL * sms, at_once = static_cast<long long>(p.own_blocks) * n_kv;
    p.n_own = static_cast<int>(std::max(1LL, std::min({(target + at_once - 1) / at_once, static_cast<long long>((own_tiles + 1) / 2),
                                                      static_cast<long long>(MAX_SLOTS)})));
  }
  if (shared_len > 0 && hd <= 128 && rows > 16 && (rows + 255) / 128 * n_kv * ((shared_len + TC_TILE - 1) / TC_TILE) < INT_MAX) {
    const int tiles = (shared_len + TC_TILE - 1) / TC_TILE;
    p.pre_rows = rows > 128 ? 256 : 128;
    const long long blocks = (rows + p.pre_rows - 1) / p.pre_rows * n_kv;
    // Beside single tokens the shared pass takes its share of the SMs, by measured costs of SM time: 2.6 us a tile of 256
    // rows, 1.6 of 128, 0.5 a tile of the own passes (taken half as long as they may be), and a tenth more, since the own
    // pass goes on where the shared one has ended.  128 behind 32k: 184 -> 169 us, 32 behind 4k: 37 -> 32.  The costs are
    // those of heads of 128; with the same numbers for 64 and 96 elements and pages of 16, 1.1 is within 5 % of the best
    // of 0.7 to 1.8 in eight of nine layouts, and 36.6 us against 31.3 (0.9) for 64 tokens of 12 heads on 2 of 96 behind
    // 8k.  Several tokens' own passes want all SMs after it instead (shares of 0.6 and 0.85 of them: 192 -> 256, 198 us).
    double share = 1.0;
    if (p.one) {
      const double pre = static_cast<double>(blocks) * tiles * (p.pre_rows == 256 ? 2.6 : 1.6);
      const double own = 0.25 * runs * own_tiles;
      share = std::min(1.0, std::max(0.35, 1.1 * pre / (pre + own)));
    }
    // The blocks of rows of a head go side by side along one piece where at least two pieces fit: with pieces of their
    // own, the two of 128 behind 32k read 254 MB from HBM of a prefix of 134.  165 -> 161 us there, 189 -> 187 with sixteen.
    const int limit = std::max(1, static_cast<int>(sms * share));
    const long long row_blocks = blocks / n_kv;
    p.pre_width = row_blocks <= limit / 2 ? static_cast<int>(row_blocks) : 1;
    const long long lines = blocks / p.pre_width;
    const int pieces = static_cast<int>(std::min(static_cast<long long>(limit / p.pre_width), lines * tiles));
    p.pre_ctas = pieces * p.pre_width;
    p.n_pre = static_cast<int>(std::min(static_cast<long long>(tiles), pieces / lines + 2));
  } else if (shared_len > 0) {
    p.pre_wm = rows <= 16 ? 1 : 4;
    p.pre_blocks = static_cast<int>((rows + 16 * p.pre_wm - 1) / (16 * p.pre_wm));
    const int tiles = (shared_len + TILE - 1) / TILE;
    const long long n = 2LL * sms / (static_cast<long long>(p.pre_blocks) * n_kv);
    p.n_pre = static_cast<int>(std::max(1LL, std::min({n, static_cast<long long>((tiles + 1) / 2), static_cast<long long>(MAX_SLOTS)})));
  }
  if (cut) {
    const int free_sms = p.pre_ctas < sms ? sms - p.pre_ctas : sms;
    p.own_ctas = static_cast<int>(std::min(static_cast<long long>(attn_one_blocks(hd, rep, n_batch, runs * own_tiles, free_sms)), runs * own_tiles));
  }
  return p;
}

// Rows of partial sums: a slot of every (token, head) for each part, and 16 for each block of the single tokens' line.
long long part_rows(const AttnPlan& p, int n_tokens, int n_heads) {
  const int slots = p.n_pre + p.n_own;
  if (slots == 1 && p.own_ctas == 0) return 0;
  return static_cast<long long>(slots) * n_tokens * n_heads + 16LL * p.own_ctas;
}

size_t up256(size_t n) { return (n + 255) & ~static_cast<size_t>(255); }

size_t work_bytes(const AttnPlan& p, int n_batch, int n_tokens, int n_heads, int hd) {
  const size_t rows = static_cast<size_t>(part_rows(p, n_tokens, n_heads));
  if (rows == 0) return 0;
  return up256(rows * 8) + up256(rows * hd * 4) + up256((static_cast<size_t>(n_batch) + 1) * 4);
}

template <typename T, int DP, int WM, bool FINE>
cudaError_t launch_rows_as(const AttnArgs& a, uint32_t type, int blocks, int splits, int pre, cudaStream_t st) {
  using L = RowsLayout<DP, WM>;
  static const cudaError_t set = allow_smem(attn_rows_kernel<T, DP, WM, FINE>, L::ALLOC);
  if (set != cudaSuccess) return set;
  CUtensorMap kmap, vmap;
  if (!pool_map(&kmap, a.c.k + a.layer_off, a.c, type) || !pool_map(&vmap, a.c.v + a.layer_off, a.c, type))
    return cudaErrorInvalidValue;
  return launch_dependent(attn_rows_kernel<T, DP, WM, FINE>, dim3(blocks, a.c.n_kv, splits), dim3(ROWS_THREADS), L::ALLOC, st, a, kmap, vmap, pre);
}

template <typename T, int DP>
cudaError_t launch_rows_of(const AttnArgs& a, uint32_t type, int wm, int blocks, int splits, int pre, cudaStream_t st) {
  if (wm == 1) return launch_rows_as<T, DP, 1, true>(a, type, blocks, splits, pre, st);
  return a.out_f32 ? launch_rows_as<T, DP, 4, true>(a, type, blocks, splits, pre, st)
                   : launch_rows_as<T, DP, 4, false>(a, type, blocks, splits, pre, st);
}

template <typename T>
cudaError_t launch_rows(const AttnArgs& a, uint32_t type, int wm, int blocks, int splits, int pre, cudaStream_t st) {
  return a.c.hd <= 64    ? launch_rows_of<T, 64>(a, type, wm, blocks, splits, pre, st)
         : a.c.hd <= 128 ? launch_rows_of<T, 128>(a, type, wm, blocks, splits, pre, st)
                         : launch_rows_of<T, 256>(a, type, wm, blocks, splits, pre, st);
}

template <typename T>
cudaError_t launch_attention_as(const AttnArgs& a, const AttnPlan& p, uint32_t type, cudaStream_t st) {
  if (p.pre_rows > 0) {
    const cudaError_t e = launch_attn_tc(a, type, st);
    if (e != cudaSuccess) return e;
  } else if (p.n_pre > 0) {
    const cudaError_t e = launch_rows<T>(a, type, p.pre_wm, p.pre_blocks, p.n_pre, 1, st);
    if (e != cudaSuccess) return e;
  }
  const cudaError_t e = p.one ? launch_attn_one(a, type, st) : launch_rows<T>(a, type, p.own_wm, p.own_blocks, p.n_own, 0, st);
  if (e != cudaSuccess || part_rows(p, a.n_tokens, a.n_heads) == 0) return e;
  // a head a warp while that leaves warps free, else several: what a token needs is looked up once for them
  const long long rows = static_cast<long long>(a.n_tokens) * a.n_heads;
  const int heads = rows <= 32LL * attn_sms() ? 1 : 4, per_token = (a.n_heads + heads - 1) / heads;
  const unsigned blocks = static_cast<unsigned>((static_cast<long long>(a.n_tokens) * per_token + 3) / 4);
  return launch_dependent(a.c.hd > 128 ? attn_join_kernel<T, true, 4> : heads == 1 ? attn_join_kernel<T, false, 8> : attn_join_kernel<T, false, 4>, dim3(blocks), dim3(128), 0, st, a,
                          heads, per_token);
}

}  // namespace
}  // namespace ex

extern "C" {

size_t edgexpu_cuda_kv_attention_work_bytes(const edgexpu_cuda_kv_cache* cache, int n_batch, int n_tokens, int n_heads,
                                            int shared_len, int max_len) {
  if (cache == nullptr || cache->n_kv < 1 || n_heads < 1 || n_heads % cache->n_kv != 0 || n_batch < 1 || n_tokens < 1 ||
      max_len < 1 || cache->head_dim < 1)
    return 0;
  // one token each may come with q_start or without: the larger of the two divisions
  const ex::AttnPlan p = ex::plan_of(cache->n_kv, cache->head_dim, true, n_batch, n_tokens, n_heads, shared_len, max_len);
  const ex::AttnPlan u = ex::plan_of(cache->n_kv, cache->head_dim, false, n_batch, n_tokens, n_heads, shared_len, max_len);
  return std::max(ex::work_bytes(p, n_batch, n_tokens, n_heads, cache->head_dim), ex::work_bytes(u, n_batch, n_tokens, n_heads, cache->head_dim));
}

int edgexpu_cuda_kv_attention_dev(const edgexpu_cuda_kv_cache* cache, int layer, const void* q, const int32_t* seqs,
                                  const int32_t* q_start, int n_batch, int n_tokens, int n_heads, int shared_seq,
                                  int shared_len, int max_len, float scale, void* out, uint32_t out_type, void* work,
                                  size_t work_size, void* stream) {
  std::lock_guard<std::recursive_mutex> lk(ex::api_mutex());
  if (!ex::api_ready(nullptr, 0)) return 0;
  ex::AttnArgs a{};
  if (!ex::kv_view(cache, "kv_attention", &a.c)) return 0;
  if (n_batch < 0 || n_tokens < 0 || n_heads < 1 || n_heads % a.c.n_kv != 0 || layer < 0 || layer >= a.c.n_layers)
    return ex::api_fail(nullptr, 0, "kv_attention: %d entries, %d tokens, %d heads over %d, layer %d of %d", n_batch, n_tokens,
                        n_heads, a.c.n_kv, layer, a.c.n_layers);
  if (n_tokens == 0) return 1;
  if (q == nullptr || seqs == nullptr || out == nullptr || n_batch < 1 || (q_start == nullptr && n_tokens != n_batch))
    return ex::api_fail(nullptr, 0, "kv_attention: invalid arguments (%d tokens of %d entries)", n_tokens, n_batch);
  if (out_type != ex::TYPE_F32 && out_type != cache->type)
    return ex::api_fail(nullptr, 0, "kv_attention: output type %u (F32, or the cache's %u)", out_type, cache->type);
  if (shared_len > 0 && (shared_seq < 0 || shared_seq >= a.c.n_seqs))
    return ex::api_fail(nullptr, 0, "kv_attention: shared sequence %d of %d", shared_seq, a.c.n_seqs);
  if (max_len < 1) return ex::api_fail(nullptr, 0, "kv_attention: max_len %d", max_len);
  if (((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15) != 0)
    return ex::api_fail(nullptr, 0, "kv_attention: q and out must be 16-byte aligned");
  const ex::AttnPlan p = ex::plan_of(a.c.n_kv, a.c.hd, q_start != nullptr, n_batch, n_tokens, n_heads, shared_len, max_len);
  const size_t need = ex::work_bytes(p, n_batch, n_tokens, n_heads, a.c.hd);
  const long long rows = static_cast<long long>(n_tokens) * n_heads;
  if (rows > INT_MAX || p.own_blocks < 0) return ex::api_fail(nullptr, 0, "kv_attention: %d tokens in one call", n_tokens);
  if (need > 0 && (work == nullptr || work_size < need || (reinterpret_cast<uintptr_t>(work) & 255) != 0))
    return ex::api_fail(nullptr, 0, "kv_attention: work memory of %zu bytes, 256-byte aligned, is needed (got %zu)", need,
                        work == nullptr ? static_cast<size_t>(0) : work_size);
  a.layer_off = layer * a.c.layer_stride;
  a.q = static_cast<const uint16_t*>(q);
  a.seqs = seqs;
  a.q_start = q_start;
  a.n_batch = n_batch;
  a.n_tokens = n_tokens;
  a.n_heads = n_heads;
  a.rep = n_heads / a.c.n_kv;
  a.shared_seq = shared_len > 0 ? shared_seq : 0;
  a.shared_len = std::max(0, std::min(shared_len, max_len));
  a.scale = scale * 1.4426950408889634f;
  a.n_pre = p.n_pre;
  a.n_own = p.n_own;
  a.pre_rows = p.pre_rows;
  a.pre_ctas = p.pre_ctas;
  a.pre_width = p.pre_width;
  a.own_ctas = p.own_ctas;
  const size_t parts = static_cast<size_t>(ex::part_rows(p, n_tokens, n_heads));
  uint8_t* at = static_cast<uint8_t*>(work);
  a.part_ml = reinterpret_cast<float2*>(at);
  a.part_o = reinterpret_cast<float*>(at + ex::up256(parts * 8));
  a.own_off = reinterpret_cast<int*>(at + ex::up256(parts * 8) + ex::up256(parts * a.c.hd * 4));
  a.cont_row0 = static_cast<long long>(p.n_pre + p.n_own) * rows;
  a.out = out;
  a.out_f32 = out_type == ex::TYPE_F32;
  a.beside = p.n_pre > 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = cache->type == ex::TYPE_F16 ? ex::launch_attention_as<__half>(a, p, cache->type, st)
                                                    : ex::launch_attention_as<__nv_bfloat16>(a, p, cache->type, st);
  if (e != cudaSuccess) return ex::api_fail(nullptr, 0, "kv_attention: %s", cudaGetErrorString(e));
  return 1;
}

}  // extern "C"
