// kvattn_one.cu -- attention over a paged cache for one new token of each sequence: the heads of a group
// against the sequence's own positions (all of them, or those past the shared prefix).
//
// The work is a line of tiles of 64 positions, (sequence, key/value head, up to 16 heads of the group,
// tile), cut into equal pieces for the blocks, so that ragged lengths load all blocks alike.  A piece
// that begins a sequence's run writes its sums to the run's own place, one that continues an earlier
// block's writes them to the block's place, and the join adds them up.  Where all runs are short every
// run is one block's, which writes the result itself.
//
// Warp 4 brings K and V by TMA (128-byte swizzle; dims past head_dim read as 0) through a ring that runs
// on from one run to the next; warps 0..3 take 16 positions of each tile each, with Q and O in
// registers, and meet only at a run's end.  P goes to its product in two numbers of the cache's type.
//
// Bound by HBM: K and V are read once, at (heads of the group) operations a byte.  128 sequences of 33 to
// 2000 own positions, 8 heads of 128 elements: 543 MB in 104 us on all SMs, 5.2 TB/s; 32 sequences of 1
// to 511: 45 MB in 21 us, where a block's first loads and its warps' join are a third.
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>

#include "capi_internal.h"
#include "kvattn.cuh"
#include "kvattn_mma.cuh"

namespace ex {
namespace {

constexpr int ONE_THREADS = 160;

template <int DP>
struct OneLayout {
  static constexpr int SLOTS = DP == 64 ? 10 : 6;
  static constexpr int HALF = TILE * 128;
  static constexpr int SLOT = HALF * (DP / 64);  // a tile of K, or of V
  static constexpr int BARS = SLOTS * SLOT;
  static constexpr int FIXED = BARS + 8 * 2 * SLOTS + 64;
};

// Dynamic shared memory: ring, barriers, the four warps' sums for a run's join, the runs' offsets.
template <int DP>
size_t one_smem(int rows, int n_batch, bool whole) {
  return OneLayout<DP>::FIXED + static_cast<size_t>(4) * rows * (DP + 2) * 4 + (whole ? 0 : (3 * n_batch + 1) * 4) + 1024;
}

struct Run {
  int entry, row, len, start, kvh, rb;  // rb: which 16 heads of the group
  int tile0, n;                         // this block's tiles of it, from position tile0 * TILE
  bool first;                           // the run begins here
};

template <typename T, int DP>
__global__ void __launch_bounds__(ONE_THREADS, 2)
    attn_one_kernel(const AttnArgs a, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
  using L = OneLayout<DP>;
  constexpr int ST = L::SLOTS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::BARS);
  uint64_t* empty = full + ST;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::BARS + 16 * ST);
  volatile int* quit = abort_flag + 1;  // a warp of the four gave up: all leave at the same run
  int* warp_sum = reinterpret_cast<int*>(smem + L::BARS + 16 * ST + 8);  // 5
  const int rows16 = min(16, a.rep), n_rb = (a.rep + 15) / 16;
  float* join_o = reinterpret_cast<float*>(smem + L::FIXED);             // [warp][rows16][DP]
  float* join_ml = join_o + 4 * rows16 * DP;                             // [warp][rows16][m, l]
  int* off = reinterpret_cast<int*>(join_ml + 4 * rows16 * 2);           // [n_batch + 1]: tiles before an entry's run
  int* lens = off + a.n_batch + 1;                                       // [n_batch]: its length, ~length where it shares the prefix
  int* table_row = lens + a.n_batch;                                     // [n_batch]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < ST; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 4);
    }
    *abort_flag = 0;
    *quit = 0;
    fence_mbar_init();
  }
  own_enter(a);
  const int shared = shared_of(a);
  const int per_entry = a.c.n_kv * n_rb;  // runs of an entry
  const bool whole = a.own_ctas == 0;
  long long begin = 0, end = 0;
  int first_entry = 0;
  if (whole) {
    first_entry = blockIdx.x / per_entry;
  } else {
    // every block counts the tiles of all entries; the first one leaves the counts for the join
    const int each = (a.n_batch + ONE_THREADS - 1) / ONE_THREADS, from = min(a.n_batch, static_cast<int>(threadIdx.x) * each);
    const int to = min(a.n_batch, from + each);
    int mine = 0;
    for (int i = from; i < to; ++i) {
      const Entry e = entry_of(a, i, shared);
      off[i] = mine;
      lens[i] = e.shares ? ~e.len : e.len;
      table_row[i] = e.row;
      mine += cut_of(e.start, e.len, 1).tiles;
    }
    int inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xFFFFFFFFu, inc, o);
      if (lane >= o) inc += y;
    }
    if (lane == 31) warp_sum[warp] = inc;
    __syncthreads();
    int before = inc - mine, all = 0;
#pragma unroll
    for (int w = 0; w < ONE_THREADS / 32; ++w) {
      if (w < warp) before += warp_sum[w];
      all += warp_sum[w];
    }
    for (int i = from; i < to; ++i) {
      off[i] += before;
      if (blockIdx.x == 0) a.own_off[i] = off[i];
    }
    if (threadIdx.x == 0) {
      off[a.n_batch] = all;
      if (blockIdx.x == 0) a.own_off[a.n_batch] = all;
    }
    const long long total = static_cast<long long>(all) * per_entry;
    const long long per = total <= INT_MAX / 2 ? (static_cast<int>(total) + a.own_ctas - 1) / a.own_ctas : (total + a.own_ctas - 1) / a.own_ctas;
    begin = blockIdx.x * per;
    end = min(total, begin + per);
  }
  __syncthreads();
  if (!whole && begin < end) {  // the last entry whose run begins at or before this piece
    int lo = 0, up = a.n_batch;
    while (up - lo > 1) {
      const int mid = (lo + up) / 2;
      if (static_cast<long long>(off[mid]) * per_entry <= begin) lo = mid;
      else up = mid;
    }
    first_entry = lo;
  }
  // The run at position `at` of the line, which lies in entry i or a later one.
  auto run_at = [&](long long at, int& i) {
    Run r;
    if (whole) {
      const Entry e = entry_of(a, first_entry, shared);
      r.entry = first_entry;
      r.row = e.row;
      r.len = e.len;
      r.start = e.start;
    } else {
      while (static_cast<long long>(off[i + 1]) * per_entry <= at) ++i;
      r.entry = i;
      r.row = table_row[i];
      r.len = lens[i] < 0 ? ~lens[i] : lens[i];
      r.start = lens[i] < 0 ? shared : 0;
    }
    const Cut cut = cut_of(r.start, r.len, 1);
    int which, t = 0;
    r.n = cut.tiles;
    if (whole) {
      which = blockIdx.x % per_entry;
    } else {
      const long long in = at - static_cast<long long>(off[i]) * per_entry;
      which = in <= INT_MAX ? static_cast<int>(in) / cut.tiles : static_cast<int>(in / cut.tiles);
      t = static_cast<int>(in - static_cast<long long>(which) * cut.tiles);
      r.n = static_cast<int>(min(static_cast<long long>(cut.tiles - t), end - at));
    }
    r.kvh = which / n_rb;
    r.rb = which - r.kvh * n_rb;
    r.tile0 = cut.first + t;
    r.first = t == 0;
    return r;
  };
  // `whole` blocks take one run, others all of their piece
  const long long stop = whole ? 1 : end;

  if (warp == 4) {
    Ring<ST> ring;
    int issued = 0, i = first_entry;
    bool ok = true;
    for (long long at = begin; ok && at < stop;) {
      const Run r = run_at(at, i);
      at += whole ? 1 : r.n;
      const int32_t* table = a.c.table + static_cast<long long>(max(0, r.row)) * a.c.max_pages;
      Pages pages(a.c, table, r.tile0 * TILE, r.len);
      for (int t = 2 * r.tile0; ok && t < 2 * (r.tile0 + r.n); ++t) {  // K of a tile, then its V
        const int p0 = (t >> 1) * TILE, page = pages.at(p0);
        ok = __all_sync(0xFFFFFFFFu, wait_or_abort(&empty[ring.slot], ring.phase ^ 1u, abort_flag)) != 0;
        if (!ok) break;
        bring_tile<DP, TILE>(a.c, page, (t & 1) == 0 ? &kmap : &vmap, smem_u32(smem + ring.slot * L::SLOT), r.kvh, p0, r.len,
                             &full[ring.slot]);
        issued = min(issued + 1, ST);
        ring.next();
      }
    }
    if (lane == 0) {
      if (!ok) {
        *abort_flag = 1;
        atomicOr(a.c.status, ST_TIMEOUT_EMPTY);
      }
      drain<ST>(ring, issued, full, a.c.status);
    }
  } else {
    const int g = lane >> 3, lr = lane & 7, kw = warp * 16, hd = a.c.hd;
    Ring<ST> ring;
    int i = first_entry;
    bool ok = true;
    for (long long at = begin; ok && at < stop;) {
      const Run r = run_at(at, i);
      at += whole ? 1 : r.n;
      const int n_rows = min(16, a.rep - r.rb * 16);
      const long long head0 = static_cast<long long>(r.entry) * a.n_heads + r.kvh * a.rep + r.rb * 16;
      uint32_t q[DP / 16][4];
#pragma unroll
      for (int kk = 0; kk < DP / 16; ++kk)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int row = (lane >> 2) + (x & 1) * 8, d = kk * 16 + (lane & 3) * 2 + (x >> 1) * 8;
          q[kk][x] = row < n_rows && d < hd ? *reinterpret_cast<const uint32_t*>(a.q + (head0 + row) * hd + d) : 0u;
        }
      float o[DP / 8][4];
#pragma unroll
      for (int x = 0; x < DP / 8; ++x) o[x][0] = o[x][1] = o[x][2] = o[x][3] = 0.0f;
      float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
      for (int t = r.tile0; t < r.tile0 + r.n; ++t) {
        ok = __all_sync(0xFFFFFFFFu, wait_or_abort(&full[ring.slot], ring.phase, abort_flag));
        if (!ok) break;
        const uint32_t ks = smem_u32(smem + ring.slot * L::SLOT);
        const Ring<ST> k = ring;
        ring.next();
        const uint32_t vs = smem_u32(smem + ring.slot * L::SLOT);
        const int p0 = t * TILE + kw;
        const bool in = p0 < r.len && p0 + 16 > r.start;
        float s[2][4] = {};
        if (in) {
#pragma unroll
          for (int kk = 0; kk < DP / 16; ++kk) {
            uint32_t kf[4];
            const int key = kw + lr + (g >> 1) * 8, ch = 2 * kk + (g & 1);
            ldsm4(kf, ks + (ch >> 3) * L::HALF + key * 128 + (((ch & 7) ^ (key & 7)) << 4));
            mma16816<T>(s[0], q[kk], kf[0], kf[1]);
            mma16816<T>(s[1], q[kk], kf[2], kf[3]);
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[k.slot]);
        ok = __all_sync(0xFFFFFFFFu, wait_or_abort(&full[ring.slot], ring.phase, abort_flag));
        if (!ok) break;
        if (in) {
          const bool edge = p0 < r.start || p0 + 16 > r.len;  // some of the 16 positions are not the run's
          uint32_t keep[2] = {0xFFFFFFFFu, 0xFFFFFFFFu};
          float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            if (edge) {
              const int p = p0 + n * 8 + (lane & 3) * 2;
              const bool in0 = p >= r.start && p < r.len, in1 = p + 1 >= r.start && p + 1 < r.len;
              keep[n] = (in0 ? 0xFFFFu : 0u) | (in1 ? 0xFFFF0000u : 0u);
            }
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              s[n][x] *= a.scale;
              if (((keep[n] >> ((x & 1) * 16)) & 1u) == 0) s[n][x] = -INFINITY;
              top[x >> 1] = fmaxf(top[x >> 1], s[n][x]);
            }
          }
          bool grow = false;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            top[h] = fmaxf(top[h], __shfl_xor_sync(0xFFFFFFFFu, top[h], 1));
            top[h] = fmaxf(top[h], __shfl_xor_sync(0xFFFFFFFFu, top[h], 2));
            grow = grow || top[h] > m[h] + GROW;
          }
          if (__any_sync(0xFFFFFFFFu, grow)) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float mn = top[h] > m[h] + GROW ? top[h] : m[h];
              const float f = mn == m[h] ? 1.0f : exp2f(m[h] - mn);
              m[h] = mn;
              l[h] *= f;
#pragma unroll
              for (int x = 0; x < DP / 8; ++x) {
                o[x][2 * h] *= f;
                o[x][2 * h + 1] *= f;
              }
            }
          }
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const float mm = m[x >> 1];
              s[n][x] = ex2(s[n][x] - ((mm == -INFINITY ? 0.0f : mm) - P_SHIFT));
              l[x >> 1] += s[n][x];
            }
          uint32_t pa[4], rest[4];  // P in two numbers of the type: bytes bound here, not products
#pragma unroll
          for (int x = 0; x < 4; ++x) split16<T>(s[x >> 1][2 * (x & 1)], s[x >> 1][2 * (x & 1) + 1], pa[x], rest[x]);
#pragma unroll
          for (int d = 0; d < DP / 16; ++d) {
            uint32_t vf[4];
            const int key = kw + lr + (g & 1) * 8, ch = 2 * d + (g >> 1);
            ldsm4t(vf, vs + (ch >> 3) * L::HALF + key * 128 + (((ch & 7) ^ (key & 7)) << 4));
            vf[0] &= keep[0];
            vf[1] &= keep[1];
            vf[2] &= keep[0];
            vf[3] &= keep[1];
            mma16816<T>(o[2 * d], pa, vf[0], vf[1]);
            mma16816<T>(o[2 * d + 1], pa, vf[2], vf[3]);
            mma16816<T>(o[2 * d], rest, vf[0], vf[1]);
            mma16816<T>(o[2 * d + 1], rest, vf[2], vf[3]);
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[ring.slot]);
        ring.next();
      }
      // join the four warps' positions; all of them get here, a given-up wait included
      if (!ok && lane == 0) {
        *quit = 1;
        *abort_flag = 1;
        atomicOr(a.c.status, ST_TIMEOUT_FULL);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        l[h] += __shfl_xor_sync(0xFFFFFFFFu, l[h], 1);
        l[h] += __shfl_xor_sync(0xFFFFFFFFu, l[h], 2);
        const int row = (lane >> 2) + 8 * h;
        if (row < n_rows) {
          if ((lane & 3) == 0) {
            join_ml[(warp * rows16 + row) * 2] = m[h];
            join_ml[(warp * rows16 + row) * 2 + 1] = l[h];
          }
#pragma unroll
          for (int x = 0; x < DP / 8; ++x)
            *reinterpret_cast<float2*>(join_o + (warp * rows16 + row) * DP + x * 8 + (lane & 3) * 2) = make_float2(o[x][2 * h], o[x][2 * h + 1]);
        }
      }
      named_bar_sync(1, 128);
      ok = *quit == 0;
      for (int x = threadIdx.x; x < n_rows * (DP / 4); x += 128) {
        const int row = x / (DP / 4), d = x % (DP / 4) * 4;
        float mm = -INFINITY;
#pragma unroll
        for (int w = 0; w < 4; ++w) mm = fmaxf(mm, join_ml[(w * rows16 + row) * 2]);
        const float base = mm == -INFINITY ? 0.0f : mm;
        float ll = 0.0f;
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float f = exp2f(join_ml[(w * rows16 + row) * 2] - base);
          const float4 u = *reinterpret_cast<const float4*>(join_o + (w * rows16 + row) * DP + d);
          ll += f * join_ml[(w * rows16 + row) * 2 + 1];
          v.x += f * u.x;
          v.y += f * u.y;
          v.z += f * u.z;
          v.w += f * u.w;
        }
        if (d >= hd) continue;
        if (whole) {
          store_out<T>(a, (head0 + row) * hd + d, v.x, v.y, ll, r.len > 0);
          store_out<T>(a, (head0 + row) * hd + d + 2, v.z, v.w, ll, r.len > 0);
        } else {
          const long long at_row = r.first ? static_cast<long long>(a.n_pre) * a.n_tokens * a.n_heads + head0 + row
                                           : a.cont_row0 + static_cast<long long>(blockIdx.x) * 16 + row;
          *reinterpret_cast<float4*>(a.part_o + at_row * hd + d) = v;
          if (d == 0) a.part_ml[at_row] = make_float2(mm, ll);
        }
      }
      named_bar_sync(1, 128);  // before the next run's sums
    }
  }
  own_leave(a);
}

// Two rounds of blocks: SMs do not get the same share of a busy memory, and the second round evens that out.
// Of the SMs that the shared pass leaves (32 behind 4k: one round 35.6 us, two 32.4), but no block gets more than 16
// tiles before there are two rounds of all SMs (128 sequences of 33 to 2000 positions: one round 185 us, two 182):
// where the shared pass leaves few, the blocks past the first round wait for its end and then have every SM (128
// behind 32k with up to 224 of their own and two SMs left: 16 blocks 321 us, 320 blocks 114).
template <int DP>
int blocks_of(int rep, int n_batch, long long tiles, int free_sms) {
  const size_t smem = one_smem<DP>(std::min(16, rep), n_batch, false);
  const int fit = std::max(1, std::min(static_cast<int>((228 * 1024) / (smem + 1024)), 2)), all = fit * attn_sms();
  return std::max(2 * fit * free_sms, static_cast<int>(std::min(2LL * all, (tiles + 15) / 16)));
}

template <typename T, int DP>
cudaError_t launch_one_as(const AttnArgs& a, uint32_t type, int blocks, cudaStream_t st) {
  static const cudaError_t set = allow_smem(attn_one_kernel<T, DP>, 200 * 1024);
  if (set != cudaSuccess) return set;
  CUtensorMap kmap, vmap;
  if (!pool_map(&kmap, a.c.k + a.layer_off, a.c, type) || !pool_map(&vmap, a.c.v + a.layer_off, a.c, type))
    return cudaErrorInvalidValue;
  return launch_dependent(attn_one_kernel<T, DP>, dim3(blocks), dim3(ONE_THREADS),
                          one_smem<DP>(std::min(16, a.rep), a.n_batch, a.own_ctas == 0), st, a, kmap, vmap);
}

}  // namespace

int attn_one_blocks(int hd, int rep, int n_batch, long long tiles, int free_sms) {
  return hd <= 64 ? blocks_of<64>(rep, n_batch, tiles, free_sms) : blocks_of<128>(rep, n_batch, tiles, free_sms);
}

cudaError_t launch_attn_one(const AttnArgs& a, uint32_t type, cudaStream_t st) {
  const int blocks = a.own_ctas > 0 ? a.own_ctas : a.n_batch * a.c.n_kv * ((a.rep + 15) / 16);
  if (type == TYPE_F16) return a.c.hd <= 64 ? launch_one_as<__half, 64>(a, type, blocks, st) : launch_one_as<__half, 128>(a, type, blocks, st);
  return a.c.hd <= 64 ? launch_one_as<__nv_bfloat16, 64>(a, type, blocks, st) : launch_one_as<__nv_bfloat16, 128>(a, type, blocks, st);
}

}  // namespace ex
