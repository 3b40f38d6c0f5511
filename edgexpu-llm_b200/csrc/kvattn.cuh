// kvattn.cuh -- what the kernels of attention over a paged cache share (kvattn.cu, kvattn_one.cu,
// kvattn_tc.cu).
#pragma once

#include <cuda.h>

#include "capi_internal.h"
#include "kv.cuh"

namespace ex {

constexpr int TILE = 64;       // positions a tile, a multiple of 64 from position 0: a box of a page, 64 positions at most, never straddles two
constexpr int TILE_SHIFT = 6;
constexpr int MAX_SLOTS = 64;  // parts of a row in the shared pass, and in its own
// Softmax weights are kept 2^P_SHIFT times as large, in o and l alike, so that f16 holds the small
// weights of a long row in full: 2^-24 of the largest and more, where 2^-14 would be its limit.
constexpr float P_SHIFT = 10.0f;
constexpr float GROW = 5.0f;  // a reference maximum moves when the maximum is this much larger: weights stay below 2^15

struct AttnArgs {
  KvView c;
  long long layer_off;  // elements
  const uint16_t* q;
  const int32_t* seqs;
  const int32_t* q_start;
  int n_batch, n_tokens, n_heads, rep;
  int shared_seq, shared_len;
  float scale;       // times log2(e)
  int n_pre, n_own;  // parts of the shared prefix, and of a sequence's own positions
  int pre_rows;      // rows a block of the tensor-memory kernel's shared pass; 0: the rows kernel makes it
  int pre_ctas;      // its blocks
  int pre_width;     // blocks that share a piece of its line
  int own_ctas;      // blocks of the single-token kernel, whose line of work is cut into equal pieces; 0: a run each
  int* own_off;      // [n_batch + 1]: tiles of the line before each entry's run (by the kernel, for the join)
  long long cont_row0;  // row of part_o, part_ml where the blocks' 16 continuing rows begin
  float* part_o;     // [n_pre + n_own][token][head][hd]
  float2* part_ml;   // [n_pre + n_own][token][head]: m, l
  void* out;
  int out_f32;
  int beside;        // the own pass runs beside the shared pass, launched before it
};

// The own pass' way in and out: beside a shared pass it starts at once, and the last of its blocks waits
// for that pass, so that both are complete when it is.
__device__ __forceinline__ void own_enter(const AttnArgs& a) {
  if (a.beside)
    pdl_launch_next();
  else
    pdl_enter_grid();
}
__device__ __forceinline__ void own_leave(const AttnArgs& a) {
  if (a.beside && blockIdx.x == gridDim.x - 1 && blockIdx.y == gridDim.y - 1 && blockIdx.z == gridDim.z - 1) pdl_wait_previous();
}

// Positions of the prefix.
__device__ __forceinline__ int shared_of(const AttnArgs& a) {
  if (a.shared_len <= 0) return 0;
  const int held = min(a.c.lens[a.shared_seq], a.c.max_pages << a.c.ps_shift);
  return max(0, min(a.shared_len, held));
}

struct Entry {
  int row;         // of the table; -1: idle
  int t0, nq;      // its tokens
  int len;         // positions held
  int start;       // first position of its own pass
  bool shares;     // it takes part in the shared pass
};

__device__ __forceinline__ Entry entry_of(const AttnArgs& a, int i, int shared) {
  Entry e{-1, i, 1, 0, 0, false};
  if (a.q_start != nullptr) {
    e.t0 = a.q_start[i];
    e.nq = a.q_start[i + 1] - e.t0;
    if (e.t0 < 0 || e.nq < 0 || e.t0 > a.n_tokens || e.nq > a.n_tokens - e.t0) {
      atomicOr(a.c.status, ST_BAD_CACHE);
      e.t0 = e.nq = 0;
      return e;
    }
  }
  const int s = a.seqs[i];
  if (s < 0) return e;
  if (s >= a.c.n_seqs) {
    atomicOr(a.c.status, ST_BAD_CACHE);
    return e;
  }
  e.row = s;
  const int held = a.c.lens[s], most = a.c.max_pages << a.c.ps_shift;
  if (held < 0 || held > most) atomicOr(a.c.status, ST_BAD_CACHE);
  e.len = max(0, min(held, most));
  e.shares = shared > 0 && e.len - e.nq + 1 >= shared;
  e.start = e.shares ? shared : 0;
  return e;
}

// Tiles of a part: those of [start, end) cut into at most n parts of `per` tiles.
struct Cut {  // of the rows kernel
  int first, tiles, per, used;
};
__device__ __forceinline__ Cut cut_of(int start, int end, int n) {
  Cut c;
  c.first = start / TILE;
  c.tiles = end > start ? (end + TILE - 1) / TILE - c.first : 0;
  c.per = max(1, (c.tiles + n - 1) / n);
  c.used = (c.tiles + c.per - 1) / c.per;
  return c;
}

// The shared pass of the tensor-memory kernel.  (kv head, block of rows, tile of the prefix) is a line of
// work cut into equal pieces.  Where a few blocks of rows make up a head, pre_width blocks of the grid, one
// for each, take the same piece of the line (kv head, tile), so that what one of them brings from HBM the
// others find in L2; else pre_width is 1 and the blocks of rows are in the line.  A block of rows is divided
// over the pieces that touch it, and piece c's part of it is slot c - (the first such piece).
constexpr int TC_TILE = 128;  // positions
struct TcCut {
  int tiles, lines, total, per;  // lines: blocks of rows of a head that are in the line
};
__device__ __forceinline__ TcCut tc_cut(const AttnArgs& a, int shared) {
  TcCut c;
  c.tiles = (shared + TC_TILE - 1) / TC_TILE;
  c.lines = (a.n_tokens * a.rep + a.pre_rows - 1) / a.pre_rows / a.pre_width;
  c.total = c.lines * a.c.n_kv * c.tiles;
  const int pieces = a.pre_ctas / a.pre_width;
  c.per = (c.total + pieces - 1) / pieces;
  return c;
}

__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}

__device__ __forceinline__ void tma_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A layer of a pool as [page][head x slot][element], in boxes of 64 elements of at most 64 of a page's
// positions; elements past head_dim read as 0 (kvattn_tc.cu).
bool pool_map(CUtensorMap* map, const uint16_t* base, const KvView& c, uint32_t type);

// SMs for the division of the work: the device's, or a B200's before the library is bound to one, so that a work
// size asked for then holds.
inline int attn_sms() {
  const int n = api_device_info().sm_count;
  return n > 0 ? n : 148;
}

// Launch the single tokens' own pass (kvattn_one.cu), hd at most 128; its blocks where the line is cut.
constexpr int ONE_MAX_BATCH = 1024;  // what the runs need is in shared memory
cudaError_t launch_attn_one(const AttnArgs& a, uint32_t type, cudaStream_t st);
int attn_one_blocks(int hd, int rep, int n_batch, long long tiles, int free_sms);

// A place in a ring of slots, and the parity of its filling.
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
  __device__ __forceinline__ void back() {
    if (--slot < 0) {
      slot = NS - 1;
      phase ^= 1u;
    }
  }
};

// Wait for the last fillings of a ring that has got `issued` of them (NS or fewer count), `ring` being the
// place of the next: no copy may still be landing when a block exits.
template <int NS>
__device__ __forceinline__ void drain(const Ring<NS>& ring, int issued, uint64_t* full, uint32_t* status) {
  bool drained = true;
  for (int n = min(issued, NS); n > 0; --n) {
    const int s = ring.slot - n + (ring.slot < n ? NS : 0);
    if (!mbar_wait(&full[s], ring.phase ^ (ring.slot < n ? 1u : 0u))) drained = false;
  }
  if (!drained) atomicOr(status, ST_TIMEOUT_DRAIN);
}

// Page indices of a sequence's boxes (the rows of a page that one copy brings, 64 at most) ahead of their
// use by a warp: lane x has that of box `first` + x, and of 32 more, so that no look-up stands between the wait
// for a slot and the copies into it.
struct Pages {
  const int32_t* table;
  int ps_shift, box_shift, end, first, now, ahead;
  __device__ __forceinline__ Pages(const KvView& c, const int32_t* table, int p0, int end)
      : table(table), ps_shift(c.ps_shift), box_shift(min(c.ps_shift, TILE_SHIFT)), end(end), first(p0 >> box_shift) {
    now = look(first);
    ahead = look(first + 32);
  }
  __device__ __forceinline__ int look(int box) const {
    const long long p = static_cast<long long>(box + static_cast<int>(threadIdx.x & 31)) << box_shift;
    return p < end ? table[p >> ps_shift] : 0;
  }
  // For lane x, the page of the x-th box from position p on; p never falls and steps by less than 32 boxes.
  __device__ __forceinline__ int at(int p) {
    const int box = p >> box_shift;
    if (box >= first + 32) {
      now = ahead;
      first += 32;
      ahead = look(first + 32);
    }
    return __shfl_sync(0xFFFFFFFFu, now, (box - first + (threadIdx.x & 31)) & 31);
  }
};

// One warp: positions [p0, end) of head kvh, at most ROWS of them and from a multiple of ROWS, into a slot as
// ROWS rows of 128 bytes for each 64 elements, by boxes of rows; lane x names the page of the x-th box.  A lane
// brings its box where they are few.  Else one thread issues them all: a copy's operands are the warp's, so that 16
// copies of eight lanes took 1450 cycles, of one 1050 (pages of 16: 190 -> 181 us, 32 questions behind 8k; pages of
// 64, two boxes: 163 by lanes, 165 by one, 128 behind 32k).
template <int DP, int ROWS>
__device__ __forceinline__ void bring_tile(const KvView& c, int page, const CUtensorMap* map, uint32_t dst, int kvh, int p0, int end,
                                           uint64_t* bar) {
  const int lane = threadIdx.x & 31, box = min(1 << c.ps_shift, TILE), boxes = (min(ROWS, end - p0) + box - 1) / box;
  const int slot_mask = (1 << c.ps_shift) - 1, head_row = kvh << c.ps_shift;
  if (lane < boxes && (page < 0 || page >= c.n_pages)) {
    atomicOr(c.status, ST_BAD_CACHE);
    page = 0;
  }
  auto bring = [&](int x, int page_x) {
#pragma unroll
    for (int h = 0; h < DP / 64; ++h)
      tma_3d(dst + x * box * 128 + h * ROWS * 128, map, 64 * h, head_row + ((p0 + x * box) & slot_mask), page_x, bar);
  };
  if (boxes <= 2) {
    if (lane == 0) mbar_arrive_expect_tx(bar, boxes * box * DP * 2);
    __syncwarp();
    if (lane < boxes) bring(lane, page);
  } else {
    int pages[ROWS / 16];
#pragma unroll
    for (int x = 0; x < ROWS / 16; ++x) pages[x] = __shfl_sync(0xFFFFFFFFu, page, x);
    if (elect_one()) {
      mbar_arrive_expect_tx(bar, boxes * box * DP * 2);
#pragma unroll
      for (int x = 0; x < ROWS / 16; ++x)
        if (x < boxes) bring(x, pages[x]);
    }
  }
  __syncwarp();
}

// Launch the shared pass on the tensor cores' own memory (kvattn_tc.cu), hd at most 128.
cudaError_t launch_attn_tc(const AttnArgs& a, uint32_t type, cudaStream_t st);

}  // namespace ex
