// What the attention kernels over the paged frame cache share: the argument block and the division of the
// work among CTAs.
//
// The work is a list of items, one per (sequence, row tile, cache head): a row tile is up to `tpt` new frames
// with all `group` query heads that share the cache head. An item is a run of 64-key steps that covers the
// keys some row of it may see. Steps of all items form one line in the order (sequence, row tile, head,
// step); every worker (a CTA, a tile of one or a warp) takes an equal share of it, whatever the lengths are, so ragged
// batches, few heads over long caches and many heads over short ones all fill the GPU alike. Where a share ends inside
// an item the item's parts go to the workspace as (unnormalised sum, maximum, weight) per row and a second kernel joins
// them in the order of the keys, so results do not depend on timing. A worker owns two workspace slots: one for a first
// item begun by another, one for a last item that it begins and does not end.
// An item also costs its set-up and its epilogue, whatever its length: on the line its steps are preceded by run_cost
// places that stand for no step, so that shares of many short items come out as even as shares of few long ones.
// Each CTA derives the line from the device's lengths (a scan over the sequences); the host needs only bounds.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "sm100.cuh"

namespace trc {

constexpr int kCacheMaxSeqs = 2048;
constexpr int kCacheMaxGroup = 64;
constexpr int kCacheStep = 64;  // keys per step

// Programmatic dependent launch: every kernel here may start before the one in front of it on the stream has ended
// (its launch and set-up overlap that one's tail), lets its own successor do the same, and waits before it touches
// global memory.
__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_release() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// a / b for a >= 0, b > 0, the short way where both fit 32 bits
__device__ __forceinline__ int64_t div_pos(int64_t a, int64_t b) {
  return (a | b) >> 32 ? a / b : (int64_t)((uint32_t)a / (uint32_t)b);
}

struct CacheAttnArgs {
  const void* q;        // [n_tokens][hq][64] 16-bit, q_stride elements from token to token
  void* out;            // like q, out_stride
  int64_t q_stride, out_stride;
  const float* gates;   // [n_tokens][hq] fp32, or null
  const int32_t* table; // [n_seqs][table_stride] page numbers
  const int32_t* cu;    // [n_seqs + 1] first row of each sequence
  const int32_t* total; // [n_seqs] frames in the cache, the new ones included
  float* ws;
  int* status;
  int n_seqs, n_tokens, hq, hkv, group;
  int table_stride, page_log2, n_pages;
  int causal, window;   // window 0: unlimited
  int split;            // 1: shares may end inside an item
  int min_share;        // least steps of a share
  int run_cost;         // places of an item on the line besides its steps
  int whole_from;       // items stay whole where a share holds this many of the longest
  int rows_above, rows_upto;  // this launch's sequences: rows_above < new frames x group <= rows_upto
  int second;           // 1: launched behind a kernel of the same call that takes the other sequences
  float scale_log2;     // softmax scale x log2(e)
};

// The lengths and the first table lines into L2, before grid_wait: L2 is where earlier kernels' writes to them arrive.
__device__ __forceinline__ void cache_prefetch(const CacheAttnArgs& a) {
  const int64_t x = (int64_t)threadIdx.x * 32;
  if (x <= a.n_seqs) asm volatile("prefetch.global.L2 [%0];" ::"l"(a.cu + x));
  if (x < a.n_seqs) asm volatile("prefetch.global.L2 [%0];" ::"l"(a.total + x));
  if (x < (int64_t)a.n_seqs * a.table_stride) asm volatile("prefetch.global.L2 [%0];" ::"l"(a.table + x));
}

struct CacheSeq {
  int tok, n, total;  // first row, new frames, frames in the cache
};

// Sequence r, its lengths cut to the rows and the table. `bad` becomes true where they had to be: offsets that fall or
// leave the rows, or, for a sequence with new frames, a total that is negative or more than the table holds.
__device__ __forceinline__ CacheSeq cache_seq(const CacheAttnArgs& a, int r, bool& bad) {
  const int from = a.cu[r], to = a.cu[r + 1], total = a.total[r];
  const int room = (int)min((int64_t)a.table_stride << a.page_log2, (int64_t)1 << 30);
  CacheSeq s;
  s.tok = min(max(from, 0), a.n_tokens);
  s.n = min(max(to, s.tok), a.n_tokens) - s.tok;
  s.total = min(max(total, 0), room);
  bad |= from < 0 || to < from || to > a.n_tokens || (to > from && s.total != total);
  const int64_t rows = (int64_t)s.n * a.group;
  if (rows <= a.rows_above || rows > a.rows_upto) s.n = 0;  // another launch's
  return s;
}
__device__ __forceinline__ CacheSeq cache_seq(const CacheAttnArgs& a, int r) {
  bool bad = false;
  return cache_seq(a, r, bad);
}

// Keys [lo, hi) that new frame i of a sequence sees.
__device__ __forceinline__ int cache_hi(const CacheAttnArgs& a, const CacheSeq& s, int i) {
  return a.causal ? min(max(s.total - s.n + i + 1, 0), s.total) : s.total;
}
__device__ __forceinline__ int cache_lo(const CacheAttnArgs& a, const CacheSeq& s, int i) {
  return a.window ? max(s.total - s.n + i + 1 - a.window, 0) : 0;
}

// One item and its neighbours on the line.
struct CacheItem {
  int r, tile, head;  // sequence, row tile, cache head
  CacheSeq s;
  int tok0, ntok;     // its new frames (within the sequence)
  int lo, hi;         // keys that some row sees
  int t0, t1;         // its steps
  int64_t start;      // its place on the line

  __device__ __forceinline__ int places(const CacheAttnArgs& a) const { return t1 - t0 + a.run_cost; }
  __device__ __forceinline__ void set_tile(const CacheAttnArgs& a, int tpt) {
    tok0 = tile * tpt;
    ntok = min(tpt, s.n - tok0);
    hi = cache_hi(a, s, tok0 + ntok - 1);
    lo = min(cache_lo(a, s, tok0), hi);
    t0 = lo / kCacheStep;
    t1 = max((hi + kCacheStep - 1) / kCacheStep, t0 + 1);
  }
  // the item that holds place `at` (< the line's length); prefix: the line's scan over the sequences
  __device__ __forceinline__ void seek(const CacheAttnArgs& a, int tpt, const int64_t* prefix, int64_t at) {
    int x = 0, y = a.n_seqs;  // prefix[x] <= at < prefix[y]
    while (y - x > 1) {
      const int m = (x + y) >> 1;
      if (prefix[m] <= at) x = m; else y = m;
    }
    r = x;
    s = cache_seq(a, r);
    int64_t left = at - prefix[r];
    for (tile = 0;; ++tile) {
      set_tile(a, tpt);
      const int64_t all = (int64_t)places(a) * a.hkv;
      if (left < all) break;
      left -= all;
    }
    head = (int)div_pos(left, places(a));
    start = at - (left - (int64_t)head * places(a));
  }
  __device__ __forceinline__ void next(const CacheAttnArgs& a, int tpt) {
    start += places(a);
    if (++head < a.hkv) return;
    head = 0;
    if (tok0 + ntok < s.n) {
      ++tile;
    } else {
      tile = 0;
      do {
        if (++r >= a.n_seqs) return;  // the line's end: `start` equals its length
        s = cache_seq(a, r);
      } while (s.n == 0);
    }
    set_tile(a, tpt);
  }
};

// A CTA's share of a line of `length` steps.
__device__ __forceinline__ int64_t cache_share(const CacheAttnArgs& a, int64_t length, int ctas) {
  return max(div_pos(length + ctas - 1, ctas), (int64_t)a.min_share);
}

// The line's scan, by all `threads` threads of the CTA: prefix[r] = places before sequence r, prefix[n_seqs] =
// the line's length. Returns whether shares end inside items: not where the host rules it out, nor where a share
// holds whole_from of the longest items (whole items are then at most 1 / whole_from uneven, nothing is joined).
// Block 0 reports lengths that do not fit. `part` holds 32 int64 of scratch. Ends with a CTA barrier.
__device__ __forceinline__ bool cache_scan(const CacheAttnArgs& a, int tpt, int threads, int ctas, int64_t* prefix,
                                           int64_t* part) {
  const int per = (a.n_seqs + threads - 1) / threads;
  const int r0 = min((int)threadIdx.x * per, a.n_seqs), r1 = min(r0 + per, a.n_seqs);
  int64_t sum = 0;
  int longest = 0;
  bool bad = false;
  for (int r = r0; r < r1; ++r) {
    CacheItem it;
    it.s = cache_seq(a, r, bad);
    int64_t steps = 0;
    for (it.tile = 0; it.tile * tpt < it.s.n; ++it.tile) {
      it.set_tile(a, tpt);
      steps += it.places(a);
      longest = max(longest, it.places(a));
    }
    prefix[r] = sum;
    sum += steps * a.hkv;
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t scan = sum;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t o = __shfl_up_sync(0xffffffffu, scan, d);
    if (lane >= d) scan += o;
  }
  if (lane == 31) part[warp] = scan;
  __syncthreads();
  int64_t before = scan - sum, length = 0;
  for (int w = 0; w < threads / 32; ++w) {
    if (w < warp) before += part[w];
    length += part[w];
  }
  for (int r = r0; r < r1; ++r) prefix[r] += before;
  if (threadIdx.x == 0) prefix[a.n_seqs] = length;
  const bool divided = __syncthreads_or(a.split && longest * (int64_t)a.whole_from > cache_share(a, length, ctas));
  if (bad && blockIdx.x == 0) record_error(a.status, kErrBadArgs);
  return divided;
}

// The runs of steps that one worker works on, in order.
struct CacheWalk {
  CacheItem it;
  int64_t s0, s1;  // the worker's share of the line
  int a0, a1;      // the run's steps [a0, a1) within the item
  bool split, valid;

  __device__ __forceinline__ void begin(const CacheAttnArgs& a, int tpt, const int64_t* prefix, int worker, int workers,
                                        bool divided) {
    const int64_t length = prefix[a.n_seqs], w = cache_share(a, length, workers);
    split = divided;
    s0 = min(length, (int64_t)worker * w);
    s1 = min(length, s0 + w);
    valid = s0 < s1;
    if (!valid) return;
    it.seek(a, tpt, prefix, s0);
    if (!split && it.start < s0) it.next(a, tpt);  // whole items go to the worker whose share holds their start
    settle(a, tpt);
  }
  __device__ __forceinline__ void advance(const CacheAttnArgs& a, int tpt) {
    it.next(a, tpt);
    settle(a, tpt);
  }
  // the next item from `it` on of which a step lies in the share
  __device__ __forceinline__ void settle(const CacheAttnArgs& a, int tpt) {
    for (;; it.next(a, tpt)) {
      valid = it.start < s1;
      if (!valid) return;
      a0 = it.t0;
      a1 = it.t1;
      if (!split) return;
      const int64_t first = it.start + a.run_cost;  // place of step t0
      a0 += (int)max(s0 - first, (int64_t)0);
      a1 = (int)min((int64_t)a1, it.t0 + max(s1 - first, (int64_t)0));
      if (a0 < a1) return;
    }
  }
  __device__ __forceinline__ bool whole() const { return a0 == it.t0 && a1 == it.t1; }
  __device__ __forceinline__ int slot() const { return a0 == it.t0 ? 1 : 0; }  // of a run that is not whole
  // workers on this item, when it is begun here and not ended
  __device__ __forceinline__ int parts(const CacheAttnArgs& a) const {
    const int64_t w = s1 - s0;  // a share that an item outlasts is not the line's last, so it is a full one
    return 1 + (int)div_pos(it.start + it.places(a) - 1 - s0, w);
  }
};

// Workspace: for each worker a record of the item that it begins and does not end, then the slots. Slot
// (2 worker + which) holds a run's sums, 64 per row, then [rows][2] (maximum in log2 units, weight). The sums are
// [rows][64] where lanes hold columns (cache_rows_kernel) and [16][rows][4] where they hold rows (cache_tiles_kernel).
struct CacheRecord {
  int parts;  // workers on the item; 0: there is none
  int tok, ntok, head;
};
__host__ __device__ __forceinline__ int64_t cache_slot_floats(int rows) { return (int64_t)rows * 66; }
__host__ __device__ __forceinline__ int64_t cache_workspace_floats(int rows, int ctas) {
  return 4ll * ctas + 2ll * ctas * cache_slot_floats(rows);
}
__device__ __forceinline__ CacheRecord* cache_record(const CacheAttnArgs& a, int cta) {
  return reinterpret_cast<CacheRecord*>(a.ws) + cta;
}
__device__ __forceinline__ float* cache_slot(const CacheAttnArgs& a, int rows, int ctas, int slot) {
  return a.ws + 4ll * ctas + cache_slot_floats(rows) * slot;
}

}  // namespace trc
