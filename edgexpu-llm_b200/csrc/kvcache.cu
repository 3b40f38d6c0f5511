// kvcache.cu -- a key/value cache in pages that many sequences share: taking, sharing, copying,
// packing and giving back pages, and the pass that norms, rotates and stores the heads of new tokens.
//
// State.  table[s][i] names the page of positions i * page_size ... of sequence s, refs[p] counts the
// rows that name page p, and a page with refs 0 is free.  All of it lives on the device, so a decode
// loop that takes pages can be a CUDA graph; the price is that finding free pages is a scan of refs.
#include <cuda_runtime.h>

#include <climits>
#include <cstring>
#include <mutex>

#include "capi_internal.h"
#include "kv.cuh"

namespace ex {
namespace {

constexpr int APPEND_MAX = 4096;  // entries of one append: four a thread of the one block that plans it
constexpr int PLAN_THREADS = 1024;
constexpr int WORK_HEAD = 16;     // ints: [0] the copies or moves that a plan found

// work: head | owner[n_seqs] | count[n_pages] | last[n_pages] | list[n_pages] | jobs[3 * n_seqs].
// A packing keeps its sources in count, its destinations in last and every page's new index in list.
struct Work {
  int32_t *head, *owner, *count, *last, *list, *jobs;
};
__host__ __device__ __forceinline__ Work work_of(const KvView& c) {
  Work w;
  w.head = c.work;
  w.owner = w.head + WORK_HEAD;
  w.count = w.owner + c.n_seqs;
  w.last = w.count + c.n_pages;
  w.list = w.last + c.n_pages;
  w.jobs = w.list + c.n_pages;
  return w;
}

// ---- giving back and sharing ------------------------------------------------------------------------

// One block a batch entry.  A page leaves its row by an exchange, so an entry that comes twice gives
// it back once.
__global__ void __launch_bounds__(128) kv_free_kernel(const KvView c, const int32_t* seqs, const int32_t* keep) {
  pdl_enter_grid();
  const int s = seqs[blockIdx.x];
  if (s < 0) return;
  if (s >= c.n_seqs) {
    if (threadIdx.x == 0) atomicOr(c.status, ST_BAD_CACHE);
    return;
  }
  const int len = max(0, c.lens[s]);
  const int kept = keep != nullptr ? min(max(0, keep[blockIdx.x]), len) : 0;
  const int end = min(kv_pages_of(c, len), c.max_pages);
  int32_t* row = c.table + static_cast<long long>(s) * c.max_pages;
  for (int i = kv_pages_of(c, kept) + threadIdx.x; i < end; i += blockDim.x) {
    const int p = atomicExch(&row[i], -1);
    if (p >= 0 && p < c.n_pages)
      atomicSub(&c.refs[p], 1);
    else if (p >= c.n_pages)
      atomicOr(c.status, ST_BAD_CACHE);
  }
  __syncthreads();
  if (threadIdx.x == 0) atomicMin(&c.lens[s], kept);
}

// One block a batch entry.  An entry is refused for what the batch alone shows (a destination that
// comes earlier too, a source that is a destination) or for a destination that holds tokens; no other
// entry writes what it reads then.
__global__ void __launch_bounds__(256) kv_fork_kernel(const KvView c, const int32_t* src, const int32_t* dst, int n) {
  pdl_enter_grid();
  const int b = blockIdx.x, s = src[b], d = dst[b];
  if (d < 0) return;
  int bad = s < 0 || s >= c.n_seqs || d >= c.n_seqs;
  const int held = bad ? 0 : c.lens[d], len = bad ? 0 : max(0, c.lens[s]);
  for (int j = threadIdx.x; j < n && !bad; j += blockDim.x) bad = (j < b && dst[j] == d) || dst[j] == s;
  bad = __syncthreads_or(bad || held != 0);
  if (bad) {
    if (threadIdx.x == 0) atomicOr(c.status, ST_BAD_CACHE);
    return;
  }
  const int pages = min(kv_pages_of(c, len), c.max_pages);
  const int32_t* from = c.table + static_cast<long long>(s) * c.max_pages;
  int32_t* to = c.table + static_cast<long long>(d) * c.max_pages;
  for (int i = threadIdx.x; i < pages; i += blockDim.x) {
    const int p = from[i];
    to[i] = p;
    if (p >= 0 && p < c.n_pages)
      atomicAdd(&c.refs[p], 1);
    else
      atomicOr(c.status, ST_BAD_CACHE);
  }
  if (threadIdx.x == 0) c.lens[d] = len;
}

// ---- block-wide scans ---------------------------------------------------------------------------------

// Exclusive sum of v over the block's threads in order; *total = the whole.  red: 33 numbers.
template <typename I>
__device__ __forceinline__ I block_scan(I v, I* red, I* total) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, nw = blockDim.x >> 5;
  I x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const I y = __shfl_up_sync(0xFFFFFFFFu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) red[w] = x;
  __syncthreads();
  if (w == 0) {
    I t = lane < nw ? red[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const I y = __shfl_up_sync(0xFFFFFFFFu, t, o);
      if (lane >= o) t += y;
    }
    red[lane] = t;
  }
  __syncthreads();
  const I r = x - v + (w > 0 ? red[w - 1] : 0);
  *total = red[nw - 1];
  __syncthreads();
  return r;
}

// The first `most` indices i in [from, to) with (refs[i] > 0) == live, ascending, into list (nullable).
// Returns how many there are up to where it stopped, which is after `most` of them.  All threads of the
// block call it.
__device__ int find_pages(const int32_t* refs, int from, int to, bool live, int most, int32_t* list, int* red) {
  constexpr int UN = 8;  // loads in flight a thread
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, nw = blockDim.x >> 5;
  int found = 0;
  for (int base = from; base < to && found < most; base += nw * 32 * UN) {
    const int b = base + w * 32 * UN + lane;
    uint32_t hit[UN];
    int mine = 0;
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      const int i = b + u * 32;
      const bool h = i < to && (refs[i] > 0) == live;
      hit[u] = __ballot_sync(0xFFFFFFFFu, h);
      mine += __popc(hit[u]);
    }
    int total;
    // every lane of a warp carries the warp's count; the first one enters it into the scan
    int off = block_scan(lane == 0 ? mine : 0, red, &total);
    off = found + __shfl_sync(0xFFFFFFFFu, off, 0);
    if (list != nullptr) {
#pragma unroll
      for (int u = 0; u < UN; ++u) {
        const int at = off + __popc(hit[u] & ((1u << lane) - 1u));
        if (((hit[u] >> lane) & 1u) != 0 && at < most) list[at] = b + u * 32;
        off += __popc(hit[u]);
      }
    }
    found += total;
  }
  return found;
}

// ---- taking -------------------------------------------------------------------------------------------

// One block: what each entry needs, the lowest free pages for it, and the last pages to be copied.  Bound by
// latency, a chain of dependent loads and block barriers.  FEW: at most 256 entries, one a thread; which
// entry names a sequence first and which rows of the batch share a last page is then found by comparing
// all pairs in shared memory, else by atomics in `work`.  Free and append, three kernels in a graph, of 16, 64, 128
// and 256 entries: 6.7, 7.6, 8.6 and 10.5 us by pairs, 10.3, 11.3, 11.8 and 12.9 in `work`; with a fork between them
// 10.0, 11.0, 12.9 and 16.0 against 13.7, 14.3, 16.0 and 16.4.
constexpr int APPEND_FEW = 256;
constexpr int LIST_SHARED = 2048;  // pages found, in shared memory up to so many

template <bool FEW>
__global__ void __launch_bounds__(PLAN_THREADS) kv_append_plan_kernel(const KvView c, const int32_t* seqs, const int32_t* n_new, int n,
                                                                      int32_t* pos, int32_t* missing) {
  constexpr int PER = FEW ? 1 : APPEND_MAX / PLAN_THREADS, MOST = FEW ? APPEND_FEW : APPEND_MAX;
  __shared__ int s_first[MOST], s_off[MOST + 1];  // an entry's first new column, its first place in the list
  __shared__ int s_seq[FEW ? MOST : 1], s_tail[FEW ? MOST : 1];
  __shared__ int s_list[FEW ? LIST_SHARED : 1];
  __shared__ int red[33];
  __shared__ long long red_need[33];
  __shared__ int n_jobs;
  const Work w = work_of(c);
  const int in_page = (1 << c.ps_shift) - 1;
  if (threadIdx.x == 0) n_jobs = 0;
  pdl_enter_grid();
  int seq[PER], len[PER], add[PER], tail[PER];  // tail: the page that holds the last tokens, when it has room; else -1
  bool ok[PER];
  // entries PER * thread ..., so that a scan over threads is a scan over the batch
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    const int b = threadIdx.x * PER + e;
    seq[e] = b < n ? seqs[b] : -1;
    add[e] = b < n ? n_new[b] : 0;
    ok[e] = seq[e] >= 0 && seq[e] < c.n_seqs;
    if (seq[e] >= c.n_seqs) atomicOr(c.status, ST_BAD_CACHE);
    len[e] = ok[e] ? c.lens[seq[e]] : 0;
    // a sequence belongs to the first entry that names it
    if constexpr (FEW) {
      if (b < n) s_seq[b] = seq[e];
    } else if (ok[e]) {
      w.owner[seq[e]] = INT_MAX;
    }
  }
  __syncthreads();
  if constexpr (FEW) {
    const int b = threadIdx.x;
    bool first = true;
    if (ok[0])
#pragma unroll 8
      for (int j = 0; j < b; ++j) first &= s_seq[j] != seq[0];
    if (ok[0] && !first) {
      ok[0] = false;
      atomicOr(c.status, ST_BAD_CACHE);
    }
  } else {
#pragma unroll
    for (int e = 0; e < PER; ++e)
      if (ok[e]) atomicMin(&w.owner[seq[e]], static_cast<int>(threadIdx.x) * PER + e);
    __syncthreads();
#pragma unroll
    for (int e = 0; e < PER; ++e)
      if (ok[e] && w.owner[seq[e]] != static_cast<int>(threadIdx.x) * PER + e) {
        ok[e] = false;
        atomicOr(c.status, ST_BAD_CACHE);
      }
  }
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    const int b = threadIdx.x * PER + e;
    tail[e] = -1;
    if (ok[e]) {
      bool fits = len[e] >= 0 && add[e] >= 0 && static_cast<long long>(len[e]) + add[e] <= (static_cast<long long>(c.max_pages) << c.ps_shift);
      if (fits && (len[e] & in_page) != 0 && add[e] > 0) {
        tail[e] = c.table[static_cast<long long>(seq[e]) * c.max_pages + (len[e] >> c.ps_shift)];
        if (tail[e] < 0 || tail[e] >= c.n_pages) {
          fits = false;
          tail[e] = -1;
        }
      }
      ok[e] = fits;
      if (!fits) atomicOr(c.status, ST_BAD_CACHE);
    }
    if constexpr (FEW) {
      if (b < n) s_tail[b] = tail[e];
    } else if (tail[e] >= 0) {
      w.count[tail[e]] = 0;
      w.last[tail[e]] = -1;
    }
  }
  __syncthreads();
  // a shared last page is copied, but for the last of the rows of the batch that share it when they are all its holders
  long long need = 0;  // rows of 2^27 pages: a batch's sum passes 32 bits
  int want[PER];
  bool split[PER];
  if constexpr (!FEW) {
#pragma unroll
    for (int e = 0; e < PER; ++e)
      if (tail[e] >= 0) {
        atomicAdd(&w.count[tail[e]], 1);
        atomicMax(&w.last[tail[e]], static_cast<int>(threadIdx.x) * PER + e);
      }
    __syncthreads();
  }
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    const int b = threadIdx.x * PER + e;
    split[e] = false;
    want[e] = 0;
    if (tail[e] >= 0) {
      const int r = c.refs[tail[e]];
      if (r > 1) {
        int sharers = 0, last = -1;
        if constexpr (FEW) {
#pragma unroll 8
          for (int j = 0; j < n; ++j) {
            const bool alike = s_tail[j] == tail[e];
            sharers += alike ? 1 : 0;
            last = alike ? j : last;
          }
        } else {
          sharers = w.count[tail[e]];
          last = w.last[tail[e]];
        }
        split[e] = !(sharers >= r && last == b);
      }
    }
    if (ok[e]) {
      s_first[b] = kv_pages_of(c, len[e]) - (split[e] ? 1 : 0);
      want[e] = kv_pages_of(c, len[e] + add[e]) - s_first[b];
      need += want[e];
    }
  }
  long long total;
  int off = static_cast<int>(block_scan(need, red_need, &total));  // read where the batch fits alone
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    const int b = threadIdx.x * PER + e;
    if (b < n) s_off[b] = off;
    off += want[e];
  }
  if (threadIdx.x == 0) s_off[n] = static_cast<int>(total);
  int32_t* list = FEW && total <= LIST_SHARED ? s_list : w.list;
  const int most = static_cast<int>(min(total, static_cast<long long>(c.n_pages)));  // places of the list
  const int found = total > 0 ? find_pages(c.refs, 0, c.n_pages, false, most, list, red) : 0;
  const bool fits = found >= total;
  __syncthreads();
  if (fits && total > 0) {  // a warp an entry: its pages into its row
    const int lane = threadIdx.x & 31;
    for (int b = threadIdx.x >> 5; b < n; b += blockDim.x >> 5) {
      const int at = s_off[b], take = s_off[b + 1] - at;
      if (take == 0) continue;
      int32_t* row = c.table + static_cast<long long>(seqs[b]) * c.max_pages + s_first[b];
      for (int i = lane; i < take; i += 32) {
        const int p = list[at + i];
        row[i] = p;
        c.refs[p] = 1;
      }
    }
  }
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    const int b = threadIdx.x * PER + e;
    if (b >= n) continue;
    const bool done = fits && ok[e];
    if (pos != nullptr) pos[b] = done ? len[e] : -1;
    if (!done) continue;
    c.lens[seq[e]] = len[e] + add[e];
    if (split[e]) {
      atomicSub(&c.refs[tail[e]], 1);
      const int j = atomicAdd(&n_jobs, 1);
      w.jobs[3 * j] = tail[e];
      w.jobs[3 * j + 1] = list[s_off[b]];
      w.jobs[3 * j + 2] = len[e] & in_page;
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    w.head[0] = n_jobs;
    if (missing != nullptr)
      *missing = fits ? 0 : static_cast<int>(min(total - found, static_cast<long long>(INT_MAX)));
    else if (!fits)
      atomicOr(c.status, ST_NO_PAGES);
  }
}

// ---- moving -------------------------------------------------------------------------------------------

constexpr int PIECE = 4096;  // bytes a warp copies at once: eight 16-byte loads a thread in flight

// Pages (or their first tokens) from src to dst, in every layer, in k and v.  The unit of work is a
// PIECE of one head of one page of one layer of one pool; warps take them in turn.  Bound by HBM.
//   stride 1: job i is src[i] -> dst[i], all tokens; stride 3: jobs[3i], jobs[3i + 1], jobs[3i + 2] tokens.
//   n_dev: the number of jobs, on the device; else n.
//   remap: afterwards table entries p >= *n_dev_live become remap[p] (a packing).
// A packing of 48 sequences of up to 4000 tokens (1.7 GB each way) 546 us, 95 % of a copy's rate; 128 copies of
// one last page (0.53 GB written, 4 MB read) 88 us.
struct MoveArgs {
  const int32_t* src;
  const int32_t* dst;
  int stride;
  int n;
  const int32_t* n_dev;
  const int32_t* n_live;
  const int32_t* remap;
};

__global__ void __launch_bounds__(256) kv_move_kernel(const KvView c, const MoveArgs a) {
  pdl_enter_grid();
  const int lane = threadIdx.x & 31;
  const long long warp = (static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
  const long long n_warps = (static_cast<long long>(gridDim.x) * blockDim.x) >> 5;
  const int n = a.n_dev != nullptr ? *a.n_dev : a.n;
  const int ps = 1 << c.ps_shift, head_bytes = ps * c.hd * 2;
  const int pieces = (head_bytes + PIECE - 1) / PIECE;
  const long long per_job = static_cast<long long>(c.n_layers) * 2 * c.n_kv * pieces;
  for (long long u = warp; u < n * per_job; u += n_warps) {
    const int job = static_cast<int>(u / per_job);
    int r = static_cast<int>(u - job * per_job);
    const int piece = r % pieces;
    r /= pieces;
    const int h = r % c.n_kv;
    r /= c.n_kv;
    const int layer = r >> 1;
    uint16_t* pool = (r & 1) != 0 ? c.v : c.k;
    const int from = a.src[job * a.stride], to = a.dst[job * a.stride];
    if (from < 0 || from >= c.n_pages || to < 0 || to >= c.n_pages) {
      if (lane == 0) atomicOr(c.status, ST_BAD_CACHE);
      continue;
    }
    const int bytes = a.stride == 3 ? a.src[job * 3 + 2] * c.hd * 2 : head_bytes;
    uint16_t* base = pool + layer * c.layer_stride + static_cast<long long>(h) * ps * c.hd;
    const uint4* s = reinterpret_cast<const uint4*>(base + from * c.page_stride);
    uint4* d = reinterpret_cast<uint4*>(base + to * c.page_stride);
    const int first = piece * (PIECE / 16) + lane, end = min(bytes, (piece + 1) * PIECE) / 16;
    uint4 x[PIECE / 512];
#pragma unroll
    for (int i = 0; i < PIECE / 512; ++i)
      if (first + i * 32 < end) x[i] = __ldcs(s + first + i * 32);
#pragma unroll
    for (int i = 0; i < PIECE / 512; ++i)
      if (first + i * 32 < end) __stcs(d + first + i * 32, x[i]);
  }
  if (a.remap != nullptr) {
    const int live = *a.n_live;
    const long long cells = static_cast<long long>(c.n_seqs) * c.max_pages, step = static_cast<long long>(gridDim.x) * blockDim.x;
    for (long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; i < cells; i += step) {
      const int p = c.table[i];
      if (p >= live) {
        if (p < c.n_pages)
          c.table[i] = a.remap[p];
        else
          atomicOr(c.status, ST_BAD_CACHE);
      }
    }
  }
}

// One block: the pages in use at or above their number L, the free ones below it, and the reference
// counts after the moves.
__global__ void __launch_bounds__(PLAN_THREADS) kv_compact_plan_kernel(const KvView c, int32_t* n_live) {
  pdl_enter_grid();
  __shared__ int red[33];
  const Work w = work_of(c);
  const int live = find_pages(c.refs, 0, c.n_pages, true, INT_MAX, nullptr, red);
  const int moves = find_pages(c.refs, live, c.n_pages, true, INT_MAX, w.count, red);
  find_pages(c.refs, 0, live, false, INT_MAX, w.last, red);
  for (int p = live + threadIdx.x; p < c.n_pages; p += blockDim.x) w.list[p] = p;
  __syncthreads();
  for (int i = threadIdx.x; i < moves; i += blockDim.x) {
    const int s = w.count[i], d = w.last[i];
    w.list[s] = d;
    c.refs[d] = c.refs[s];
    c.refs[s] = 0;
  }
  if (threadIdx.x == 0) {
    w.head[0] = moves;
    w.head[1] = live;
    if (n_live != nullptr) *n_live = live;
  }
}

cudaError_t launch_move(const KvView& c, const MoveArgs& a, long long jobs_at_most, cudaStream_t st) {
  const long long pieces = (static_cast<long long>(2 << c.ps_shift) * c.hd + PIECE - 1) / PIECE;
  const long long warps = jobs_at_most * c.n_layers * 2 * c.n_kv * pieces;
  long long blocks = (warps + 7) / 8;
  const long long most = 8LL * api_device_info().sm_count;  // 2048 threads an SM
  if (blocks > most) blocks = most;
  if (blocks < 1) blocks = 1;
  return launch_dependent(kv_move_kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, st, c, a);
}

// ---- norm, rotation and store of new tokens' heads ----------------------------------------------------

struct QkArgs {
  const float *q, *k, *v;
  long long qs, ks, vs;
  int n_tokens, n_heads, layer;
  const float *qw, *kw;
  float eps, inv_hd;
  const float* rope;
  int rope_positions, rot, halves;
  const int32_t *seqs, *pos;
  uint16_t* q_out;
};

constexpr int QK_WARPS = 8;
constexpr int QK_HEADS = 4;  // heads a group of lanes holds at once: their loads are all in flight together

// Pair (y0, y1) by the angle (c, s).
__device__ __forceinline__ void rotate(float& y0, float& y1, float c, float s) {
  const float a = y0 * c - y1 * s;
  y1 = y0 * s + y1 * c;
  y0 = a;
}

// Where the pairs of a head are turned: nowhere, in the lane that holds both (adjacent), between two lanes
// (halves, in whole chunks of four elements), or in shared memory (the other splits of a head).
enum class Turn { None, InLane, BetweenLanes, InShared };

// A group of GS lanes takes QK_HEADS heads of a token, all queries, all keys or all values, a lane V times
// four elements of each: the token's page, angles and weights are looked up once for them, and the sums of
// squares are fp32 over the group.  Bytes are 4 read and 2 written an element; at 8k tokens of 48 heads of
// 128 it is bound by the instructions it issues, about 110 a head and warp: 51 us (74 % of the issue slots, 60 %
// of HBM's rate; floor 47).  Wider blocks and fewer or more heads a group measured the same or slower.
template <typename T, int GS, int V, Turn TURN>
__global__ void __launch_bounds__(QK_WARPS * 32) qk_norm_rope_kernel(const KvView c, const QkArgs a, const int units) {
  pdl_enter_grid();
  constexpr int GROUPS = 32 / GS;
  extern __shared__ __align__(16) float rows[];  // [warp][group][QK_HEADS][GS * V * 4], for Turn::InShared
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, gl = lane % GS, gr = lane / GS;
  const unsigned unit = blockIdx.x * QK_WARPS + w, t = unit / static_cast<unsigned>(units);
  if (t >= static_cast<unsigned>(a.n_tokens)) return;
  const int nv = c.hd / 4, q_groups = (a.n_heads + QK_HEADS - 1) / QK_HEADS, k_groups = (c.n_kv + QK_HEADS - 1) / QK_HEADS;
  int group = static_cast<int>(unit - t * units) * GROUPS + gr;
  const bool is_q = group < q_groups, is_k = !is_q && group < q_groups + k_groups;
  const float* x = is_q ? a.q + t * a.qs : is_k ? a.k + t * a.ks : a.v + t * a.vs;
  const float* wt = is_q ? a.qw : is_k ? a.kw : nullptr;
  const int h0 = (is_q ? group : is_k ? group - q_groups : group - q_groups - k_groups) * QK_HEADS;
  const int n = min(QK_HEADS, (is_q ? a.n_heads : c.n_kv) - h0);  // heads of the group, none in a last one past the values
  float4 e[QK_HEADS][V];
  const float4* x4 = reinterpret_cast<const float4*>(x + h0 * c.hd) + gl;
#pragma unroll
  for (int i = 0; i < QK_HEADS; ++i)
#pragma unroll
    for (int u = 0; u < V; ++u) e[i][u] = i < n && gl + u * GS < nv ? __ldcs(x4 + i * nv + u * GS) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  const int s = a.seqs[t], p = a.pos[t];
  bool live = s >= 0 && p >= 0;
  int page = -1;
  if (live) {
    if (s < c.n_seqs && (p >> c.ps_shift) < c.max_pages && (TURN == Turn::None || p < a.rope_positions))
      page = c.table[static_cast<long long>(s) * c.max_pages + (p >> c.ps_shift)];
    if (page < 0 || page >= c.n_pages) {
      live = false;
      if (lane == 0) atomicOr(c.status, ST_BAD_CACHE);
    }
  }
  if (wt != nullptr || GROUPS > 1) {  // 1 / rms of each head, and the norm's weights
    float rms[QK_HEADS];
#pragma unroll
    for (int i = 0; i < QK_HEADS; ++i) {
      rms[i] = 0.0f;
#pragma unroll
      for (int u = 0; u < V; ++u) rms[i] += e[i][u].x * e[i][u].x + e[i][u].y * e[i][u].y + e[i][u].z * e[i][u].z + e[i][u].w * e[i][u].w;
    }
#pragma unroll
    for (int o = GS / 2; o > 0; o >>= 1)
#pragma unroll
      for (int i = 0; i < QK_HEADS; ++i) rms[i] += __shfl_xor_sync(0xFFFFFFFFu, rms[i], o);
    if (wt != nullptr) {
#pragma unroll
      for (int i = 0; i < QK_HEADS; ++i) rms[i] = rsqrtf(rms[i] * a.inv_hd + a.eps);
#pragma unroll
      for (int u = 0; u < V; ++u) {
        const float4 g = gl + u * GS < nv ? reinterpret_cast<const float4*>(wt)[gl + u * GS] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int i = 0; i < QK_HEADS; ++i) {
          e[i][u].x = e[i][u].x * rms[i] * g.x;
          e[i][u].y = e[i][u].y * rms[i] * g.y;
          e[i][u].z = e[i][u].z * rms[i] * g.z;
          e[i][u].w = e[i][u].w * rms[i] * g.w;
        }
      }
    }
  }

  const bool turned = live && (is_q || is_k);
  const float* cs = turned ? a.rope + static_cast<long long>(p) * a.rot : a.rope;
  const int half = a.rot / 2;
  if constexpr (TURN == Turn::InLane) {
#pragma unroll
    for (int u = 0; u < V; ++u) {
      const int j = gl + u * GS;
      if (turned && 4 * j < a.rot) {
        const bool both = 4 * j + 2 < a.rot;
        const float2 a0 = *reinterpret_cast<const float2*>(cs + 4 * j);
        const float2 a1 = both ? *reinterpret_cast<const float2*>(cs + 4 * j + 2) : make_float2(1.0f, 0.0f);
#pragma unroll
        for (int i = 0; i < QK_HEADS; ++i) rotate(e[i][u].x, e[i][u].y, a0.x, a0.y);
        if (both)
#pragma unroll
          for (int i = 0; i < QK_HEADS; ++i) rotate(e[i][u].z, e[i][u].w, a1.x, a1.y);
      }
    }
  } else if constexpr (TURN == Turn::BetweenLanes) {
    // V == 1 and half % 4 == 0: chunk j < half / 4 turns with chunk j + half / 4, half / 4 lanes on
    const int step = half / 4;
    const bool low = gl < step, in = turned && gl < 2 * step;
    float ang[8] = {1.0f, 0.0f, 1.0f, 0.0f, 1.0f, 0.0f, 1.0f, 0.0f};
    if (in) {
      const float2* at = reinterpret_cast<const float2*>(cs) + 4 * (low ? gl : gl - step);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 y = at[k];
        ang[2 * k] = y.x;
        ang[2 * k + 1] = low ? -y.y : y.y;  // y0 c - y1 s below, y1 c + y0 s above
      }
    }
    const int from = gr * GS + (low ? gl + step : gl < 2 * step ? gl - step : gl);
#pragma unroll
    for (int i = 0; i < QK_HEADS; ++i) {
      const float4 mine = e[i][0];
      float4 other;
      other.x = __shfl_sync(0xFFFFFFFFu, mine.x, from);
      other.y = __shfl_sync(0xFFFFFFFFu, mine.y, from);
      other.z = __shfl_sync(0xFFFFFFFFu, mine.z, from);
      other.w = __shfl_sync(0xFFFFFFFFu, mine.w, from);
      if (in) {
        e[i][0].x = mine.x * ang[0] + other.x * ang[1];
        e[i][0].y = mine.y * ang[2] + other.y * ang[3];
        e[i][0].z = mine.z * ang[4] + other.z * ang[5];
        e[i][0].w = mine.w * ang[6] + other.w * ang[7];
      }
    }
  } else if constexpr (TURN == Turn::InShared) {
    float* row = rows + (w * GROUPS + gr) * QK_HEADS * GS * V * 4;
#pragma unroll
    for (int i = 0; i < QK_HEADS; ++i)
#pragma unroll
      for (int u = 0; u < V; ++u) reinterpret_cast<float4*>(row + i * GS * V * 4)[gl + u * GS] = e[i][u];
    __syncwarp();
    for (int j = gl; j < half && turned; j += GS)
      for (int i = 0; i < n; ++i) rotate(row[i * GS * V * 4 + j], row[i * GS * V * 4 + j + half], cs[2 * j], cs[2 * j + 1]);
    __syncwarp();
#pragma unroll
    for (int i = 0; i < QK_HEADS; ++i)
#pragma unroll
      for (int u = 0; u < V; ++u) e[i][u] = reinterpret_cast<float4*>(row + i * GS * V * 4)[gl + u * GS];
  }

  if (!is_q && !live) return;
  // queries one head after the other, keys and values a page's head apart
  const int step = (is_q ? c.hd : c.hd << c.ps_shift) / 4;
  uint16_t* to = is_q ? a.q_out + (static_cast<long long>(t) * a.n_heads + h0) * c.hd
                      : (is_k ? c.k : c.v) + a.layer * c.layer_stride + page * c.page_stride +
                            ((static_cast<long long>(h0) << c.ps_shift) + (p & ((1 << c.ps_shift) - 1))) * c.hd;
  uint2* to2 = reinterpret_cast<uint2*>(to) + gl;
#pragma unroll
  for (int i = 0; i < QK_HEADS; ++i) {
#pragma unroll
    for (int u = 0; u < V; ++u)
      if (i < n && gl + u * GS < nv)
        to2[u * GS] = live ? make_uint2(pack16<T>(e[i][u].x, e[i][u].y), pack16<T>(e[i][u].z, e[i][u].w)) : make_uint2(0u, 0u);
    to2 += step;
  }
}

template <typename T, int GS, int V, Turn TURN>
cudaError_t launch_heads_as(const KvView& c, const QkArgs& a, cudaStream_t st) {
  const int groups = (a.n_heads + QK_HEADS - 1) / QK_HEADS + 2 * ((c.n_kv + QK_HEADS - 1) / QK_HEADS);
  const int units = (groups + 32 / GS - 1) / (32 / GS);  // warps a token
  const long long blocks = (static_cast<long long>(a.n_tokens) * units + QK_WARPS - 1) / QK_WARPS;
  if (blocks > INT_MAX / QK_WARPS) return cudaErrorInvalidValue;  // warps are counted in 32 bits
  constexpr size_t SMEM = TURN == Turn::InShared ? static_cast<size_t>(QK_WARPS) * 32 * V * QK_HEADS * 16 : 0;
  if (SMEM > 48 * 1024) {
    static const cudaError_t set = allow_smem(qk_norm_rope_kernel<T, GS, V, TURN>, SMEM);
    if (set != cudaSuccess) return set;
  }
  return launch_dependent(qk_norm_rope_kernel<T, GS, V, TURN>, dim3(static_cast<unsigned>(blocks)), dim3(QK_WARPS * 32), SMEM, st, c, a, units);
}

template <typename T, int GS, int V>
cudaError_t launch_heads_turned(const KvView& c, const QkArgs& a, cudaStream_t st) {
  if (a.rope == nullptr) return launch_heads_as<T, GS, V, Turn::None>(c, a, st);
  if (!a.halves) return launch_heads_as<T, GS, V, Turn::InLane>(c, a, st);
  if constexpr (V == 1)
    if (a.rot % 8 == 0) return launch_heads_as<T, GS, V, Turn::BetweenLanes>(c, a, st);
  return launch_heads_as<T, GS, V, Turn::InShared>(c, a, st);
}

template <typename T>
cudaError_t launch_heads(const KvView& c, const QkArgs& a, cudaStream_t st) {
  return c.hd <= 64    ? launch_heads_turned<T, 16, 1>(c, a, st)
         : c.hd <= 128 ? launch_heads_turned<T, 32, 1>(c, a, st)
                       : launch_heads_turned<T, 32, 2>(c, a, st);
}

bool aligned(const void* p, size_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

}  // namespace

int kv_view(const edgexpu_cuda_kv_cache* c, const char* who, KvView* view) {
  if (c == nullptr || c->k == nullptr || c->v == nullptr || c->table == nullptr || c->lens == nullptr || c->refs == nullptr)
    return api_fail(nullptr, 0, "%s: the cache or one of its arrays is NULL", who);
  if (c->type != TYPE_F16 && c->type != TYPE_BF16)
    return api_fail(nullptr, 0, "%s: cache type %u (F16 and BF16 are supported)", who, c->type);
  int shift = 0;
  while (shift < 8 && (1 << shift) < c->page_size) ++shift;
  if (c->page_size < 16 || (1 << shift) != c->page_size)
    return api_fail(nullptr, 0, "%s: page size %d (16, 32, 64, 128 or 256)", who, c->page_size);
  if (c->head_dim < 8 || c->head_dim > 256 || c->head_dim % 8 != 0)
    return api_fail(nullptr, 0, "%s: head_dim %d (a multiple of 8, 256 at most)", who, c->head_dim);
  if (c->n_layers < 1 || c->n_pages < 1 || c->n_kv < 1 || c->n_kv > 65535 || c->n_seqs < 1 || c->max_pages < 1)
    return api_fail(nullptr, 0, "%s: layers, pages, heads, sequences and columns must be positive", who);
  if ((static_cast<long long>(c->max_pages) << shift) > INT_MAX)
    return api_fail(nullptr, 0, "%s: a row of %d pages holds more than 2^31 - 1 positions", who, c->max_pages);
  const long long page = static_cast<long long>(c->n_kv) * c->page_size * c->head_dim;
  if (c->page_stride < page || c->page_stride % 8 != 0 || c->layer_stride < 0 || c->layer_stride % 8 != 0)
    return api_fail(nullptr, 0, "%s: strides %lld, %lld (multiples of 8; a page has %lld elements)", who,
                    static_cast<long long>(c->layer_stride), static_cast<long long>(c->page_stride), page);
  if (!aligned(c->k, 16) || !aligned(c->v, 16)) return api_fail(nullptr, 0, "%s: k and v must be 16-byte aligned", who);
  *view = KvView{static_cast<uint16_t*>(c->k), static_cast<uint16_t*>(c->v), c->layer_stride, c->page_stride, c->n_layers,
                 c->n_pages, shift, c->n_kv, c->head_dim, c->n_seqs, c->max_pages, c->table, c->lens, c->refs, c->work,
                 api_status_word()};
  return 1;
}

namespace {

// What every page call checks: a bound device, a cache, its scratch where the call needs it, a batch.
int page_call(const edgexpu_cuda_kv_cache* c, const char* who, bool scratch, int n, bool arrays, KvView* view) {
  if (!api_ready(nullptr, 0) || !kv_view(c, who, view)) return 0;
  if (scratch && c->work == nullptr) return api_fail(nullptr, 0, "%s: the cache has no work memory", who);
  if (n < 0 || !arrays) return api_fail(nullptr, 0, "%s: invalid arguments", who);
  return 1;
}

int launched(cudaError_t e, const char* who) {
  return e == cudaSuccess ? 1 : api_fail(nullptr, 0, "%s: %s", who, cudaGetErrorString(e));
}

}  // namespace
}  // namespace ex

extern "C" {

size_t edgexpu_cuda_kv_work_bytes(int n_pages, int n_seqs) {
  if (n_pages < 1 || n_seqs < 1) return 0;
  return (static_cast<size_t>(ex::WORK_HEAD) + 4 * static_cast<size_t>(n_seqs) + 3 * static_cast<size_t>(n_pages)) * 4;
}

int edgexpu_cuda_kv_append_dev(const edgexpu_cuda_kv_cache* cache, const int32_t* seqs, const int32_t* n_new, int n,
                               int32_t* pos, int32_t* missing, void* stream) {
  std::lock_guard<std::recursive_mutex> lk(ex::api_mutex());
  ex::KvView c;
  if (!ex::page_call(cache, "kv_append", true, n, n == 0 || (seqs != nullptr && n_new != nullptr), &c)) return 0;
  if (n > ex::APPEND_MAX) return ex::api_fail(nullptr, 0, "kv_append: %d entries (at most %d)", n, ex::APPEND_MAX);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e = ex::launch_dependent(n <= ex::APPEND_FEW ? ex::kv_append_plan_kernel<true> : ex::kv_append_plan_kernel<false>, dim3(1), dim3(ex::PLAN_THREADS), 0, st, c, seqs, n_new, n, pos, missing);
  if (e == cudaSuccess && n > 0) {
    const ex::Work w = ex::work_of(c);
    const ex::MoveArgs a{w.jobs, w.jobs + 1, 3, 0, w.head, nullptr, nullptr};
    e = ex::launch_move(c, a, n, st);
  }
  return ex::launched(e, "kv_append");
}

int edgexpu_cuda_kv_fork_dev(const edgexpu_cuda_kv_cache* cache, const int32_t* src, const int32_t* dst, int n, void* stream) {
  std::lock_guard<std::recursive_mutex> lk(ex::api_mutex());
  ex::KvView c;
  if (!ex::page_call(cache, "kv_fork", false, n, n == 0 || (src != nullptr && dst != nullptr), &c)) return 0;
  if (n == 0) return 1;
  return ex::launched(ex::launch_dependent(ex::kv_fork_kernel, dim3(n), dim3(256), 0, static_cast<cudaStream_t>(stream), c, src, dst, n),
                      "kv_fork");
}

int edgexpu_cuda_kv_free_dev(const edgexpu_cuda_kv_cache* cache, const int32_t* seqs, const int32_t* keep, int n, void* stream) {
  std::lock_guard<std::recursive_mutex> lk(ex::api_mutex());
  ex::KvView c;
  if (!ex::page_call(cache, "kv_free", false, n, n == 0 || seqs != nullptr, &c)) return 0;
  if (n == 0) return 1;
  return ex::launched(ex::launch_dependent(ex::kv_free_kernel, dim3(n), dim3(128), 0, static_cast<cudaStream_t>(stream), c, seqs, keep),
                      "kv_free");
}

int edgexpu_cuda_kv_copy_dev(const edgexpu_cuda_kv_cache* cache, const int32_t* src, const int32_t* dst, int n, void* stream) {
  std::lock_guard<std::recursive_mutex> lk(ex::api_mutex());
  ex::KvView c;
  if (!ex::page_call(cache, "kv_copy", false, n, n == 0 || (src != nullptr && dst != nullptr), &c)) return 0;
  if (n == 0) return 1;
  const ex::MoveArgs a{src, dst, 1, n, nullptr, nullptr, nullptr};
  return ex::launched(ex::launch_move(c, a, n, static_cast<cudaStream_t>(stream)), "kv_copy");
}

int edgexpu_cuda_kv_compact_dev(const edgexpu_cuda_kv_cache* cache, int32_t* n_live, void* stream) {
  std::lock_guard<std::recursive_mutex> lk(ex::api_mutex());
  ex::KvView c;
  if (!ex::page_call(cache, "kv_compact", true, 0, true, &c)) return 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const ex::Work w = ex::work_of(c);
  cudaError_t e = ex::launch_dependent(ex::kv_compact_plan_kernel, dim3(1), dim3(ex::PLAN_THREADS), 0, st, c, n_live);
  const ex::MoveArgs a{w.count, w.last, 1, 0, w.head, w.head + 1, w.list};
  if (e == cudaSuccess) e = ex::launch_move(c, a, c.n_pages, st);
  return ex::launched(e, "kv_compact");
}

int edgexpu_cuda_qk_norm_rope_dev(const edgexpu_cuda_kv_cache* cache, int layer, const float* q, const float* k,
                                  const float* v, int64_t q_stride, int64_t k_stride, int64_t v_stride, int n_tokens,
                                  int n_heads, const float* q_weight, const float* k_weight, float eps, const float* rope,
                                  int rope_positions, int rope_dims, int rope_pairing, const int32_t* seqs,
                                  const int32_t* pos, void* q_out, void* stream) {
  std::lock_guard<std::recursive_mutex> lk(ex::api_mutex());
  ex::KvView c;
  if (!ex::page_call(cache, "qk_norm_rope", false, n_tokens,
                     n_tokens == 0 || (q != nullptr && k != nullptr && v != nullptr && seqs != nullptr && pos != nullptr &&
                                       q_out != nullptr),
                     &c))
    return 0;
  if (layer < 0 || layer >= c.n_layers || n_heads < 1)
    return ex::api_fail(nullptr, 0, "qk_norm_rope: layer %d of %d, %d heads", layer, c.n_layers, n_heads);
  const int64_t qn = static_cast<int64_t>(n_heads) * c.hd, kn = static_cast<int64_t>(c.n_kv) * c.hd;
  if (q_stride < qn || k_stride < kn || v_stride < kn || q_stride % 4 != 0 || k_stride % 4 != 0 || v_stride % 4 != 0 ||
      !ex::aligned(q, 16) || !ex::aligned(k, 16) || !ex::aligned(v, 16) || !ex::aligned(q_out, 16))
    return ex::api_fail(nullptr, 0, "qk_norm_rope: rows must be 16-byte aligned and at least %lld and %lld floats apart",
                        static_cast<long long>(qn), static_cast<long long>(kn));
  if (rope != nullptr && (rope_positions < 1 || rope_dims < 2 || rope_dims > c.hd || rope_dims % 2 != 0))
    return ex::api_fail(nullptr, 0, "qk_norm_rope: a table of %d positions and %d dims for heads of %d", rope_positions, rope_dims, c.hd);
  if (!ex::aligned(q_weight, 16) || !ex::aligned(k_weight, 16) || !ex::aligned(rope, 8))
    return ex::api_fail(nullptr, 0, "qk_norm_rope: the norm weights must be 16-byte aligned, the table 8-byte");
  if (rope_pairing != EDGEXPU_CUDA_ROPE_ADJACENT && rope_pairing != EDGEXPU_CUDA_ROPE_HALVES)
    return ex::api_fail(nullptr, 0, "qk_norm_rope: pairing %d", rope_pairing);
  if (n_tokens == 0) return 1;
  const ex::QkArgs a{q, k, v, q_stride, k_stride, v_stride, n_tokens, n_heads, layer, q_weight, k_weight, eps, 1.0f / static_cast<float>(c.hd), rope,
                     rope_positions, rope_dims, rope_pairing == EDGEXPU_CUDA_ROPE_HALVES, seqs, pos,
                     static_cast<uint16_t*>(q_out)};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return ex::launched(cache->type == ex::TYPE_F16 ? ex::launch_heads<__half>(c, a, st) : ex::launch_heads<__nv_bfloat16>(c, a, st),
                      "qk_norm_rope");
}

}  // extern "C"
