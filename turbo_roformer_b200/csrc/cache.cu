// The frame cache of live input (declared in include/trcuda.h): block tables and slots from sequence lengths
// (trc_cache_plan), rotary q/k and plain v into the pages (trc_cache_append), and the attention of new frames
// over the pages (trc_cache_attention).
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <limits.h>
#include <math.h>
#include <stdint.h>
#include <stdio.h>

#include <atomic>

#include "../../include/trcuda.h"
#include "cache_attention.cuh"
#include "cache_attention_tiles.cuh"
#include "cache_sched.cuh"
#include "internal.h"

namespace trc {

static_assert(kCacheMaxSeqs == TRC_CACHE_MAX_SEQS && kCacheMaxGroup == TRC_CACHE_MAX_GROUP, "include/trcuda.h");

namespace {

// Launches with programmatic dependence on the kernel in front (every kernel of this file waits on the device before
// it touches memory) and counts the launch.
template <typename... Params, typename... Args>
int launch(const char* what, void (*kern)(Params...), dim3 grid, int threads, int smem, cudaStream_t st,
           const Args&... args) {
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = st;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, Params(args)...);
  if (e != cudaSuccess) {
    char buf[160];
    snprintf(buf, sizeof(buf), "%s launch failed: %s", what, cudaGetErrorString(e));
    return set_last_error(TRC_E_CUDA, buf);
  }
  count_launches(1);
  return TRC_OK;
}

int page_log2_of(int page) {
  switch (page) {
    case 16: return 4;
    case 32: return 5;
    case 64: return 6;
    case 128: return 7;
    default: return -1;
  }
}

// Memory that a call reads or writes.
struct Span {
  const void* at;
  int64_t bytes;
};
bool overlap(const Span& a, const Span& b) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a.at), y = reinterpret_cast<uintptr_t>(b.at);
  return a.bytes > 0 && b.bytes > 0 && x < y + (uintptr_t)b.bytes && y < x + (uintptr_t)a.bytes;
}
// Whether one of the first `written` spans shares memory with another span.
template <int N>
bool overlap(const Span (&spans)[N], int written) {
  for (int i = 0; i < written; ++i)
    for (int k = i + 1; k < N; ++k)
      if (overlap(spans[i], spans[k])) return true;
  return false;
}

// Rows `width` bytes long, `stride` bytes apart.
struct Rows {
  const void* at;
  int64_t stride, width;
  Span span(int64_t n) const {
    const int64_t reach = (n - 1) * stride;  // negative: the first row lies last
    return {static_cast<const char*>(at) + (reach < 0 ? reach : 0), (reach < 0 ? -reach : reach) + width};
  }
};
// Whether any of n rows of a and n of b share memory. Rows of one stride may lie between each other's (columns of a
// wider buffer); of different strides they count as overlapping where their spans do. a.stride >= a.width.
bool overlap(const Rows& a, const Rows& b, int64_t n) {
  if (!overlap(a.span(n), b.span(n))) return false;
  if (n == 1 || a.stride != b.stride) return true;
  const int64_t apart = (int64_t)(reinterpret_cast<uintptr_t>(b.at) - reinterpret_cast<uintptr_t>(a.at));
  const int64_t d = ((apart % a.stride) + a.stride) % a.stride;  // where in a row of a, or behind it, rows of b begin
  return d < a.width || d + b.width > a.stride;
}

// ------------------------------------------------------------------------------------------------ plan
// Every block repeats the scan over the sequences (two 64-bit sums per thread) and then takes its part of two
// flat ranges: the fresh pages (each finds its sequence by a search in the scan) and the rows, four at a time (one
// search, then onwards; vector stores). Nothing is exchanged between blocks, so one launch serves any batch: a row's
// page is either fresh (read from the free list, not from the table that another block is writing) or was in the table
// before. Lengths and sums sit in shared memory. A push of 8 streams takes 4 us, the launch and the scan's latency; one
// of 4,001 sequences and a million rows 11 to 15 us (8.9 MB: 1.4 us of HBM): 59 % of the issue slots, every row finds
// its own page.
struct PlanArgs {
  const int32_t* cached;
  const int32_t* fresh;  // new lengths
  const int32_t* free_pages;
  int32_t* table;
  int32_t *cu, *total, *slots, *positions, *counts;
  int n_seqs, page_log2, n_free, table_stride, capacity;
};

constexpr int kPlanThreads = 1024;

// frames <= 2^30
__device__ __forceinline__ int pages_of(int frames, int page_log2) {
  return (frames + (1 << page_log2) - 1) >> page_log2;
}

// last x in [0, n) with v[x] <= at, for ascending v with v[0] <= at
__device__ __forceinline__ int last_upto(const int32_t* v, int n, int at) {
  int x = 0, y = n;
  while (y - x > 1) {
    const int m = (x + y) >> 1;
    if (v[m] <= at) x = m; else y = m;
  }
  return x;
}

// A sequence's lengths, 0 and 0 (and true) where they are bad.
__device__ __forceinline__ bool plan_lengths(const PlanArgs& a, int r, int& c, int& n) {
  c = a.cached[r];
  n = a.fresh[r];
  const bool bad = c < 0 || n < 0 || (int64_t)c + n > (1 << 30);
  if (bad) c = n = 0;
  return bad;
}

__global__ void __launch_bounds__(kPlanThreads) cache_plan_kernel(const __grid_constant__ PlanArgs a) {
  extern __shared__ int32_t plan_smem[];
  int32_t* cu = plan_smem;                   // [n_seqs + 1] rows before each sequence
  int32_t* base = cu + a.n_seqs + 1;         // [n_seqs + 1] fresh pages before each sequence
  int32_t* cached = base + a.n_seqs + 1;     // [n_seqs] frames it has, 0 where the lengths are bad
  __shared__ int64_t part[2][kPlanThreads / 32];
  __shared__ int flags;
  if (threadIdx.x == 0) flags = 0;
  grid_wait();
  grid_release();
  // the new lengths pass through cu
  int bad = 0;
  for (int r = threadIdx.x; r < a.n_seqs; r += kPlanThreads) {
    int c, n;
    if (plan_lengths(a, r, c, n)) bad |= TRC_CACHE_BAD_LENGTH;
    cached[r] = c;
    cu[r] = n;
    if (pages_of(c + n, a.page_log2) > a.table_stride) bad |= TRC_CACHE_TABLE_FULL;
  }
  __syncthreads();
  // an odd number of sequences per thread: neighbours' strides then miss each other's banks
  const int per = ((a.n_seqs + kPlanThreads - 1) / kPlanThreads) | 1;
  const int r0 = min((int)threadIdx.x * per, a.n_seqs), r1 = min(r0 + per, a.n_seqs);
  int64_t rows = 0, pages = 0;
  auto pages_for = [&](int c, int n) { return pages_of(c + n, a.page_log2) - pages_of(c, a.page_log2); };
  for (int r = r0; r < r1; ++r) {
    rows += cu[r];
    pages += pages_for(cached[r], cu[r]);
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t rs = rows, ps = pages;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t x = __shfl_up_sync(0xffffffffu, rs, d), y = __shfl_up_sync(0xffffffffu, ps, d);
    if (lane >= d) {
      rs += x;
      ps += y;
    }
  }
  if (lane == 31) {
    part[0][warp] = rs;
    part[1][warp] = ps;
  }
  __syncthreads();
  static_assert(kPlanThreads == 1024, "one warp scans the warps' sums");
  if (warp < 2) {
    int64_t x = part[warp][lane];
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, x, d);
      if (lane >= d) x += y;
    }
    part[warp][lane] = x;
  }
  __syncthreads();
  rs += (warp ? part[0][warp - 1] : 0) - rows;
  ps += (warp ? part[1][warp - 1] : 0) - pages;
  const int64_t all_rows = part[0][31], all_pages = part[1][31];
  for (int r = r0; r < r1; ++r) {
    const int n = cu[r];
    cu[r] = (int)min(rs, (int64_t)INT_MAX);
    base[r] = (int)min(ps, (int64_t)INT_MAX);
    rs += n;
    ps += pages_for(cached[r], n);
  }
  const int live_rows = (int)min(all_rows, (int64_t)INT_MAX), live_pages = (int)min(all_pages, (int64_t)INT_MAX);
  if (threadIdx.x == 0) {
    cu[a.n_seqs] = live_rows;
    base[a.n_seqs] = live_pages;
  }
  if (blockIdx.x == 0) {
    if (all_rows > a.capacity) bad |= TRC_CACHE_ROWS_FULL;
    if (all_pages > a.n_free) bad |= TRC_CACHE_NO_PAGES;
    if (bad) atomicOr(&flags, bad);
  }
  __syncthreads();
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    a.counts[0] = min(live_pages, a.n_free);
    a.counts[1] = flags;
  }
  const int stride = gridDim.x * kPlanThreads, first = blockIdx.x * kPlanThreads + threadIdx.x;
  for (int r = first; r <= a.n_seqs; r += stride) {
    a.cu[r] = cu[r];
    if (r < a.n_seqs) {
      int c, n;
      plan_lengths(a, r, c, n);
      a.total[r] = c + n;
    }
  }
  // fresh pages into the table
  const int64_t given = min(live_pages, a.n_free);
  for (int64_t e = first; e < given; e += stride) {
    const int r = last_upto(base, a.n_seqs, (int)e);
    const int64_t column = (int64_t)pages_of(cached[r], a.page_log2) + (e - base[r]);
    if (column < a.table_stride) a.table[(int64_t)r * a.table_stride + column] = a.free_pages[e];
  }
  // entries that the free list no longer serves, a warp per sequence: the work is the table's, whatever the lengths are
  if (all_pages > a.n_free) {
    for (int r = first >> 5; r < a.n_seqs; r += stride >> 5) {
      int c, n;
      plan_lengths(a, r, c, n);
      const int need = min(pages_of(c + n, a.page_log2), a.table_stride);
      for (int64_t column = (int64_t)pages_of(c, a.page_log2) + max(a.n_free - base[r], 0) + lane; column < need;
           column += 32)
        a.table[(int64_t)r * a.table_stride + column] = -1;
    }
  }
  // rows: position and slot, four to a thread
  auto store4 = [&](int32_t* to, int64_t row0, const int(&v)[4]) {
    if ((reinterpret_cast<uintptr_t>(to) & 15) == 0 && row0 + 4 <= a.capacity) {
      *reinterpret_cast<int4*>(to + row0) = make_int4(v[0], v[1], v[2], v[3]);
    } else {
      for (int i = 0; i < 4 && row0 + i < a.capacity; ++i) to[row0 + i] = v[i];
    }
  };
  for (int64_t row0 = 4ll * first; row0 < a.capacity; row0 += 4ll * stride) {
    int pos[4], slot[4];
    int r = row0 < live_rows ? last_upto(cu, a.n_seqs, (int)row0) : 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t row = row0 + i;
      pos[i] = 0;
      slot[i] = -1;
      if (row >= live_rows) continue;
      while (cu[r + 1] <= row) ++r;
      const int c = cached[r];
      pos[i] = c + (int)(row - cu[r]);
      const int column = pos[i] >> a.page_log2, held = pages_of(c, a.page_log2);
      int page = -1;
      if (column < a.table_stride) {
        if (column < held) {
          page = a.table[(int64_t)r * a.table_stride + column];
        } else {
          const int64_t e = (int64_t)base[r] + (column - held);
          if (e < a.n_free) page = a.free_pages[e];
        }
      }
      if (page >= 0 && page <= (INT_MAX >> a.page_log2))
        slot[i] = (page << a.page_log2) + (pos[i] & ((1 << a.page_log2) - 1));
    }
    store4(a.positions, row0, pos);
    store4(a.slots, row0, slot);
  }
}

// ------------------------------------------------------------------------------------------------ append
// HBM bound: each element is read once and written once. Eight lanes own a head row (64 elements, 16 bytes = 4 rotary
// pairs each). A block takes one band of up to 16 consecutive frames, and each thread one frame of it and every
// 32 / frames-th head row, so that
//   * its four angles (position x frequency in fp64, reduced to half turns, because fp32 loses the angle of far
//     positions) are computed once, while its first loads travel, and stay in registers for all its heads;
//   * the 128-byte rows that a head's frames write to a page lie one behind the other.
// 1,700 frames of 62 bands x 24 head rows with gates (653 MB): 115 us, 5.7 TB/s, 0.87 of the copy rate; one thread per
// vector of a flat run, the angles in shared memory, took 187 us (184 instructions per vector).
constexpr int kAppendThreads = 256;
constexpr int kAppendFlight = 4;  // head rows per thread in flight
constexpr int kAppendFrames = 16;

struct AppendArgs {
  const void* qkv;
  int64_t tok_stride, band_stride;  // elements
  const int32_t *positions, *slots;
  const float* freqs;
  void *q, *k, *v;
  int64_t q_stride;
  float* gates;
  int* status;
  int n_tokens, bands, heads, kv_heads, page_log2;
  int64_t n_slots;
  int frames;  // frames of a block: 1, 2, 4, 8 or 16
};

template <typename T>
struct Vec8;
template <>
struct Vec8<__half> {
  __device__ static float2 to_f2(uint32_t u) { return __half22float2(*reinterpret_cast<__half2*>(&u)); }
  __device__ static float to_f(__half x) { return __half2float(x); }
};
template <>
struct Vec8<__nv_bfloat16> {
  __device__ static float2 to_f2(uint32_t u) { return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&u)); }
  __device__ static float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
};

template <typename T>
__global__ void __launch_bounds__(kAppendThreads) cache_append_kernel(const __grid_constant__ AppendArgs a) {
  grid_wait();
  grid_release();
  const int band = blockIdx.x, tok0 = blockIdx.y * a.frames;
  const int slot_id = threadIdx.x >> 3, d = (threadIdx.x & 7) * 8;  // of 32 head rows at a time; first element
  const int f = slot_id & (a.frames - 1), step = 32 / a.frames;
  const int tok = tok0 + f, rows = a.heads + 2 * a.kv_heads;
  if (tok >= a.n_tokens) return;
  const T* band_row = static_cast<const T*>(a.qkv) + tok * a.tok_stride + band * a.band_stride;
  const T* src = band_row + d;
  int row = slot_id / a.frames;
  uint4 data[kAppendFlight];
  auto load = [&](int r) {
#pragma unroll
    for (int i = 0; i < kAppendFlight; ++i)
      if (r + i * step < rows) data[i] = __ldcs(reinterpret_cast<const uint4*>(src + (r + i * step) * 64));
  };
  load(row);
  const int slot = a.slots[tok];
  if (slot < 0) return;  // a row of padding
  float2 turn[4] = {{1.f, 0.f}, {1.f, 0.f}, {1.f, 0.f}, {1.f, 0.f}};
  if (a.freqs) {
    const double pos = a.positions[tok];
    const float4 w = *reinterpret_cast<const float4*>(a.freqs + (d >> 1));
    const float fr[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      // half turns: the angle over pi, modulo 2; fp64 keeps 1e-9 of a turn up to 5e7 frames and 2.6e-8 up to 2^30, as
      // many bits as an fp64 product position x frequency has
      const double h = pos * (double)fr[p] * 0.31830988618379067154;
      sincospif((float)(h - 2.0 * rint(0.5 * h)), &turn[p].y, &turn[p].x);
    }
  }
  const bool known = slot < a.n_slots;
  if (!known) record_error(a.status, kErrBadArgs);
  // where head row r of q, k and v goes: the cache's rows are a page apart
  const int64_t page_row = ((((int64_t)(slot >> a.page_log2) * a.bands + band) * a.kv_heads) << a.page_log2) +
                           (slot & ((1 << a.page_log2) - 1));
  T* const q = static_cast<T*>(a.q) + tok * a.q_stride + (int64_t)band * a.heads * 64 + d;
  T* const k = static_cast<T*>(a.k) + page_row * 64 + d - ((int64_t)a.heads << (a.page_log2 + 6));
  T* const v = static_cast<T*>(a.v) + page_row * 64 + d - ((int64_t)(a.heads + a.kv_heads) << (a.page_log2 + 6));
  for (; row < rows; row += kAppendFlight * step) {
#pragma unroll
    for (int i = 0; i < kAppendFlight; ++i) {
      const int r = row + i * step;
      if (r >= rows) break;
      uint4 u = data[i];
      if (r < a.heads + a.kv_heads && a.freqs) {
        uint32_t* w = reinterpret_cast<uint32_t*>(&u);
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          const float2 y = Vec8<T>::to_f2(w[p]), t = turn[p];
          w[p] = OperandType<T>::pack2(y.x * t.x - y.y * t.y, y.y * t.x + y.x * t.y);
        }
      }
      if (r < a.heads)
        *reinterpret_cast<uint4*>(q + r * 64) = u;
      else if (known)
        *reinterpret_cast<uint4*>((r < a.heads + a.kv_heads ? k : v) + ((int64_t)r << (a.page_log2 + 6))) = u;
    }
    if (row + kAppendFlight * step < rows) load(row + kAppendFlight * step);
  }
  if (a.gates) {
    const T* logits = band_row + rows * 64;
    float* g = a.gates + ((int64_t)tok * a.bands + band) * a.heads;
    for (int h = slot_id / a.frames * 8 + (threadIdx.x & 7); h < a.heads; h += step * 8)
      g[h] = 1.0f / (1.0f + expf(-Vec8<T>::to_f(logits[h])));
  }
}

// ------------------------------------------------------------------------------------------------ attention
// SMs of the current device (asked once per device), 0 on failure.
int sm_count() {
  static std::atomic<int> known[64];
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  if ((n = known[dev & 63].load(std::memory_order_relaxed))) return n;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
  known[dev & 63].store(n, std::memory_order_relaxed);
  return n;
}

// Which kernel takes a sequence, by its rows per cache head (new frames x query heads that share it). A call's time
// with 496 heads over 1,700 frames, us (HBM floor 33 us for one row, 38 us for 128; tensor floor 60 us for 384):
//   rows                         1   16   20   32   40   64  128  200  256  384  768
//   cache_rows_kernel           45   49   56   59
//   cache_tiles_kernel                    68   68   70   70   75  120  126  176  326
//   cache_tiles_kernel, shared            95   96   96   97  100  128  136  158  293
constexpr int kFewRows = 32;        // cache_rows_kernel
constexpr int kSeparateRows = 256;  // cache_tiles_kernel with separate tiles; above it with shared ones
constexpr int kCtasPerSm = 2;     // of cache_rows_kernel

// The launches of a call and where their parts go in the workspace.
struct Layout {
  int rows;            // of cache_rows_kernel's tiles
  int workers;         // its warps
  bool tiles, shared;  // whether cache_tiles_kernel follows, and how
  int workers2, rows2;
  int64_t floats, floats2;  // workspace of the two
};
Layout layout_of(int max_new, int group, int sms) {
  const int64_t most = (int64_t)(max_new > 0 ? max_new : 1) * group;
  Layout l;
  l.rows = most <= 16 ? 16 : kFewRows;
  l.workers = kCtasPerSm * sms * kCrWarps;
  l.tiles = most > kFewRows;
  l.shared = most > kSeparateRows;
  l.workers2 = !l.tiles ? 0 : l.shared ? sms : sms * kCtTiles;
  l.rows2 = l.shared ? CtSmem<true>::kRows : CtSmem<false>::kRows;
  l.floats = cache_workspace_floats(l.rows, l.workers);
  l.floats2 = l.tiles ? cache_workspace_floats(l.rows2, l.workers2) : 0;
  return l;
}

// Dynamic shared-memory opt-in, once per kernel and device (`done`: one object per kernel).
template <typename Kern>
int allow_smem(Kern kern, int bytes, std::atomic<unsigned long long>& done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  const unsigned long long bit = 1ull << (dev & 63);
  if (e == cudaSuccess && !(done.load(std::memory_order_relaxed) & bit)) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) done.fetch_or(bit);
  }
  return e == cudaSuccess ? TRC_OK : set_last_error(TRC_E_CUDA, cudaGetErrorString(e));
}

template <typename T, int MT>
int launch_rows(const CUtensorMap& mk, const CUtensorMap& mv, const CacheAttnArgs& a, int workers, cudaStream_t st) {
  static std::atomic<unsigned long long> done{0};
  const int rc = allow_smem(cache_rows_kernel<T, MT>, CrSmem::bytes(kCacheMaxSeqs), done);
  if (rc) return rc;
  return launch("cache attention", cache_rows_kernel<T, MT>, dim3(workers / kCrWarps), 32 * kCrWarps,
                CrSmem::bytes(a.n_seqs), st, mk, mv, a);
}

// The tcgen05 kernels move registers between their warpgroups (setmaxnreg): the split must fit in what the launch
// gives the block, or the softmax warps' increase would never be granted.
template <typename Kern>
int check_registers(Kern kern, int threads, int wanted, std::atomic<int>& regs) {
  if (regs.load() == 0) {
    cudaFuncAttributes fa;
    const cudaError_t e = cudaFuncGetAttributes(&fa, kern);
    if (e != cudaSuccess) return set_last_error(TRC_E_CUDA, cudaGetErrorString(e));
    regs.store(fa.numRegs);
  }
  return wanted > threads * regs.load()
             ? set_last_error(TRC_E_CUDA, "cache attention: register split larger than the launch's registers")
             : TRC_OK;
}

// Q as (64, heads, rows): boxes of a cache head's query heads for the frames of a tile.
template <typename T>
int map_q(const CacheAttnArgs& a, CUtensorMap& mq) {
  const uint64_t dims[3] = {64, (uint64_t)a.hq, (uint64_t)a.n_tokens};
  const uint64_t strides[2] = {128, 2 * (uint64_t)(a.n_tokens > 1 ? a.q_stride : (int64_t)a.hq * 64)};
  const uint32_t box[3] = {64, (uint32_t)a.group, (uint32_t)(128 / a.group)};
  return make_tensor_map(&mq, OperandType<T>::kFormat, a.q, 3, dims, strides, box);
}

template <typename T, bool SHARED>
int launch_tiles(const CUtensorMap& mk, const CUtensorMap& mv, const CacheAttnArgs& a, int sms, cudaStream_t st) {
  using S = CtSmem<SHARED>;
  auto kern = cache_tiles_kernel<T, SHARED>;
  static std::atomic<unsigned long long> done{0};
  static std::atomic<int> regs{0};
  CUtensorMap mq;
  int rc = allow_smem(kern, S::bytes(kCacheMaxSeqs), done);
  if (!rc) rc = check_registers(kern, S::kThreads, S::kRegs, regs);
  if (!rc) rc = map_q<T>(a, mq);
  return rc ? rc
            : launch("cache attention (tiles)", kern, dim3(sms), S::kThreads, S::bytes(a.n_seqs), st, mq, mk, mv, a);
}

template <typename T>
int launch_cache_attention(const Layout& l, int page, const void* k, const void* v, CacheAttnArgs a, int sms,
                           cudaStream_t st) {
  const int prec = OperandType<T>::kFormat;
  const uint64_t dims[2] = {64, (uint64_t)a.n_pages * a.hkv * page};
  const uint64_t strides[1] = {128};
  auto maps = [&](int keys, CUtensorMap& mk, CUtensorMap& mv) {
    const uint32_t box[2] = {64, (uint32_t)(page < keys ? page : keys)};
    const int rc = make_tensor_map(&mk, prec, k, 2, dims, strides, box);
    return rc ? rc : make_tensor_map(&mv, prec, v, 2, dims, strides, box);
  };
  CUtensorMap mk, mv;
  int rc;
  float* const ws2 = a.ws ? a.ws + l.floats : nullptr;
  if (l.tiles) {
    CacheAttnArgs b = a;
    b.rows_above = kFewRows;
    b.rows_upto = INT_MAX;
    b.run_cost = l.shared ? 3 : 4;  // a run's start and end, in steps (one less: a ragged batch 88 instead of 85 us)
    b.whole_from = 6;  // a divided tile leaves 34 KB or more in the workspace
    b.ws = ws2;
    if ((rc = maps(kCacheStep, mk, mv))) return rc;
    rc = l.shared ? launch_tiles<T, true>(mk, mv, b, sms, st) : launch_tiles<T, false>(mk, mv, b, sms, st);
    if (rc) return rc;
  }
  a.run_cost = 1;
  a.whole_from = 16;
  a.rows_above = 0;
  a.rows_upto = l.tiles ? kFewRows : INT_MAX;
  a.second = l.tiles;
  if ((rc = maps(kCrKeys, mk, mv))) return rc;
  rc = l.rows == 16 ? launch_rows<T, 1>(mk, mv, a, l.workers, st) : launch_rows<T, 2>(mk, mv, a, l.workers, st);
  if (rc) return rc;
  if (!a.split) return TRC_OK;
  const CacheJoin j = {l.workers, l.rows, l.rows2, ws2};
  return launch("cache attention join", cache_join_kernel<T>, dim3(l.workers + kJoinBlocks * l.workers2), 256, 0, st,
                a, j);
}

}  // namespace
}  // namespace trc

using trc::set_last_error;

extern "C" {

int trc_cache_plan(const int32_t* d_cached, const int32_t* d_new, int n_seqs, int page, const int32_t* d_free,
                   int n_free, int32_t* d_table, int table_stride, int max_rows, int32_t* d_cu, int32_t* d_total,
                   int32_t* d_slots, int32_t* d_positions, int32_t* d_counts, void* stream) {
  if (!d_cached || !d_new || !d_table || !d_cu || !d_total || !d_counts || (n_free > 0 && !d_free) ||
      (max_rows > 0 && (!d_slots || !d_positions)))
    return set_last_error(TRC_E_INVALID, "cache plan: null argument");
  if (n_seqs < 1 || n_seqs > TRC_CACHE_PLAN_MAX_SEQS)
    return set_last_error(TRC_E_INVALID, "cache plan: 1 to TRC_CACHE_PLAN_MAX_SEQS sequences");
  const int lp = trc::page_log2_of(page);
  if (lp < 0) return set_last_error(TRC_E_INVALID, "cache plan: page must be 16, 32, 64 or 128 frames");
  if (n_free < 0 || table_stride < 1 || max_rows < 0)
    return set_last_error(TRC_E_INVALID, "cache plan: bad sizes");
  // every block reads all lengths while others already write
  const trc::Span spans[] = {{d_table, 4ll * n_seqs * table_stride},
                             {d_cu, 4ll * (n_seqs + 1)},
                             {d_total, 4ll * n_seqs},
                             {d_slots, 4ll * max_rows},
                             {d_positions, 4ll * max_rows},
                             {d_counts, 8},
                             {d_cached, 4ll * n_seqs},
                             {d_new, 4ll * n_seqs},
                             {d_free, 4ll * n_free}};
  if (trc::overlap(spans, 6))
    return set_last_error(TRC_E_INVALID, "cache plan: what is written overlaps another argument");
  trc::PlanArgs a;
  a.cached = d_cached;
  a.fresh = d_new;
  a.free_pages = d_free;
  a.table = d_table;
  a.cu = d_cu;
  a.total = d_total;
  a.slots = d_slots;
  a.positions = d_positions;
  a.counts = d_counts;
  a.n_seqs = n_seqs;
  a.page_log2 = lp;
  a.n_free = n_free;
  a.table_stride = table_stride;
  a.capacity = max_rows;
  const int sms = trc::sm_count();
  if (!sms) return set_last_error(TRC_E_CUDA, "cache plan: no current CUDA device");
  const int smem = (3 * n_seqs + 2) * 4;
  static std::atomic<unsigned long long> done{0};
  int dev = 0;
  cudaGetDevice(&dev);
  if (!(done.load(std::memory_order_relaxed) >> (dev & 63) & 1)) {
    const cudaError_t e = cudaFuncSetAttribute(trc::cache_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               (3 * TRC_CACHE_PLAN_MAX_SEQS + 2) * 4);
    if (e != cudaSuccess) return set_last_error(TRC_E_CUDA, cudaGetErrorString(e));
    done.fetch_or(1ull << (dev & 63));
  }
  // a thread for every four rows
  const int64_t most = (int64_t)max_rows / 4 + 1;
  const int blocks = (int)((most + trc::kPlanThreads - 1) / trc::kPlanThreads);
  return trc::launch("cache plan", trc::cache_plan_kernel, dim3(blocks < sms ? blocks : sms), trc::kPlanThreads,
                     smem, (cudaStream_t)stream, a);
}

int trc_cache_append(int precision, const void* d_qkv, int64_t row_stride, int64_t band_stride, int n_rows, int bands,
                     int heads, int kv_heads, const int32_t* d_positions, const int32_t* d_slots, const float* d_freqs,
                     int page, int n_pages, void* d_q, int64_t q_stride, void* d_k, void* d_v, float* d_gates,
                     int* d_status, void* stream) {
  if (precision != TRC_PREC_FP16 && precision != TRC_PREC_BF16)
    return set_last_error(TRC_E_INVALID, "cache append: precision must be TRC_PREC_FP16 or TRC_PREC_BF16");
  if (n_rows < 0 || bands < 1 || heads < 1 || kv_heads < 1 || heads % kv_heads || bands > 4096 || heads > 4096 ||
      n_pages < 1)
    return set_last_error(TRC_E_INVALID, "cache append: bad sizes");
  const int lp = trc::page_log2_of(page);
  if (lp < 0) return set_last_error(TRC_E_INVALID, "cache append: page must be 16, 32, 64 or 128 frames");
  if (!n_rows) return TRC_OK;
  if (!d_qkv || !d_positions || !d_slots || !d_q || !d_k || !d_v)
    return set_last_error(TRC_E_INVALID, "cache append: null argument");
  const int64_t width = (int64_t)(heads + 2 * kv_heads) * 64 + (d_gates ? heads : 0);
  if (row_stride % 8 || band_stride % 8 || q_stride % 8 || reinterpret_cast<uintptr_t>(d_qkv) % 16 ||
      reinterpret_cast<uintptr_t>(d_q) % 16 || reinterpret_cast<uintptr_t>(d_k) % 16 ||
      reinterpret_cast<uintptr_t>(d_v) % 16 || reinterpret_cast<uintptr_t>(d_freqs) % 16)
    return set_last_error(TRC_E_INVALID, "cache append: rows (and d_freqs) must start on 16-byte boundaries");
  if ((bands > 1 && band_stride < width) || (n_rows > 1 && q_stride < (int64_t)bands * heads * 64))
    return set_last_error(TRC_E_INVALID, "cache append: strides shorter than the rows");
  if (n_rows > 1 << 20 || (n_rows + trc::kAppendFrames - 1) / trc::kAppendFrames > 65535)  // the grid's second axis
    return set_last_error(TRC_E_INVALID, "cache append: more than 1,048,560 rows");
  // threads write what others have yet to read; only a row's q may take the place of the q it is made from
  const int64_t qkv_width = 2 * ((bands - 1) * band_stride + width), page_bytes = 128ll * bands * kv_heads * page;
  const int64_t pool = n_pages > (1ll << 62) / page_bytes ? 1ll << 62 : n_pages * page_bytes;
  const trc::Rows from = {d_qkv, 2 * row_stride, qkv_width}, to = {d_q, 2 * q_stride, 128ll * bands * heads};
  const trc::Span spans[] = {{d_k, pool},
                             {d_v, pool},
                             {d_gates, d_gates ? 4ll * n_rows * bands * heads : 0},
                             to.span(n_rows),
                             from.span(n_rows),
                             {d_positions, 4ll * n_rows},
                             {d_slots, 4ll * n_rows},
                             {d_freqs, d_freqs ? 128 : 0}};
  const bool in_place =
      d_q == d_qkv && bands == 1 && (n_rows == 1 || (q_stride == row_stride && row_stride >= width));
  if (trc::overlap(spans, 3) || trc::overlap(to.span(n_rows), spans[5]) || trc::overlap(to.span(n_rows), spans[6]) ||
      trc::overlap(to.span(n_rows), spans[7]) || (!in_place && trc::overlap(to, from, n_rows)))
    return set_last_error(TRC_E_INVALID, "cache append: what is written overlaps another argument");
  trc::AppendArgs a;
  a.qkv = d_qkv;
  a.tok_stride = row_stride;
  a.band_stride = band_stride;
  a.positions = d_positions;
  a.slots = d_slots;
  a.freqs = d_freqs;
  a.q = d_q;
  a.k = d_k;
  a.v = d_v;
  a.q_stride = q_stride;
  a.gates = d_gates;
  a.status = d_status;
  a.n_tokens = n_rows;
  a.bands = bands;
  a.heads = heads;
  a.kv_heads = kv_heads;
  a.page_log2 = lp;
  a.n_slots = (int64_t)n_pages << lp;
  const int sms = trc::sm_count();
  if (!sms) return set_last_error(TRC_E_CUDA, "cache append: no current CUDA device");
  // the most frames per block that leave eight blocks per SM
  a.frames = trc::kAppendFrames;
  while (a.frames > 1 && (int64_t)((n_rows + a.frames - 1) / a.frames) * bands < 8ll * sms) a.frames /= 2;
  cudaStream_t st = (cudaStream_t)stream;
  auto kern = precision == TRC_PREC_FP16 ? trc::cache_append_kernel<__half> : trc::cache_append_kernel<__nv_bfloat16>;
  return trc::launch("cache append", kern, dim3(bands, (n_rows + a.frames - 1) / a.frames), trc::kAppendThreads, 0, st,
                     a);
}

int64_t trc_cache_workspace(int max_new, int heads, int kv_heads) {
  if (max_new < 0 || kv_heads < 1 || heads < kv_heads || heads % kv_heads ||
      heads / kv_heads > trc::kCacheMaxGroup)
    return set_last_error(TRC_E_INVALID, "cache workspace: bad sizes");
  const int sms = trc::sm_count();
  if (!sms) return set_last_error(TRC_E_CUDA, "cache workspace: no current CUDA device");
  const trc::Layout l = trc::layout_of(max_new, heads / kv_heads, sms);
  return 4 * (l.floats + l.floats2);
}

int trc_cache_attention(int precision, const void* d_q, int64_t q_stride, const void* d_k, const void* d_v,
                        const int32_t* d_table, int table_stride, const int32_t* d_cu, const int32_t* d_total,
                        int n_seqs, int n_rows, int max_new, int max_total, int heads, int kv_heads, int page,
                        int n_pages, int causal, int window, float scale, const float* d_gates, void* d_out,
                        int64_t out_stride, void* d_workspace, int64_t workspace_bytes, int* d_status, void* stream) {
  if (precision != TRC_PREC_FP16 && precision != TRC_PREC_BF16)
    return set_last_error(TRC_E_INVALID, "cache attention: precision must be TRC_PREC_FP16 or TRC_PREC_BF16");
  if (n_seqs < 1 || n_seqs > TRC_CACHE_MAX_SEQS)
    return set_last_error(TRC_E_INVALID, "cache attention: 1 to TRC_CACHE_MAX_SEQS sequences");
  if (n_rows < 0 || n_rows > 1 << 30 || max_new < 0 || max_total < 0 || heads < 1 || kv_heads < 1 ||
      heads % kv_heads || n_pages < 1 || table_stride < 1 || window < 0)
    return set_last_error(TRC_E_INVALID, "cache attention: bad sizes");
  if (heads / kv_heads > trc::kCacheMaxGroup)
    return set_last_error(TRC_E_INVALID, "cache attention: more than TRC_CACHE_MAX_GROUP query heads per cache head");
  if (heads > INT_MAX / 64)  // offsets within a row are 32-bit
    return set_last_error(TRC_E_INVALID, "cache attention: rows of 2^31 elements or more");
  const int lp = trc::page_log2_of(page);
  if (lp < 0) return set_last_error(TRC_E_INVALID, "cache attention: page must be 16, 32, 64 or 128 frames");
  // TMA addresses the pool by rows with 32-bit coordinates, and reads its zero fill just behind it
  if (((int64_t)n_pages * kv_heads << lp) > INT_MAX - 256)
    return set_last_error(TRC_E_INVALID, "cache attention: pool larger than 2^31 head rows");
  if (!(scale > 0.f) || !isfinite(scale))
    return set_last_error(TRC_E_INVALID, "cache attention: scale must be positive and finite");
  if (!n_rows) return TRC_OK;
  if (!d_q || !d_k || !d_v || !d_table || !d_cu || !d_total || !d_out)
    return set_last_error(TRC_E_INVALID, "cache attention: null argument");
  if (q_stride % 8 || out_stride % 8 || reinterpret_cast<uintptr_t>(d_q) % 16 ||
      reinterpret_cast<uintptr_t>(d_out) % 16 || reinterpret_cast<uintptr_t>(d_k) % 16 ||
      reinterpret_cast<uintptr_t>(d_v) % 16)
    return set_last_error(TRC_E_INVALID, "cache attention: rows must start on 16-byte boundaries");
  if (n_rows > 1 && (q_stride < (int64_t)heads * 64 || out_stride < (int64_t)heads * 64))
    return set_last_error(TRC_E_INVALID, "cache attention: strides shorter than the rows");
  const trc::Rows to = {d_out, 2 * out_stride, 128ll * heads};
  const int64_t pool = 128ll * n_pages * kv_heads * page;
  const trc::Span spans[] = {to.span(n_rows),
                             {d_workspace, d_workspace ? workspace_bytes : 0},
                             {d_k, pool},
                             {d_v, pool},
                             {d_table, 4ll * n_seqs * table_stride},
                             {d_cu, 4ll * (n_seqs + 1)},
                             {d_total, 4ll * n_seqs},
                             {d_gates, d_gates ? 4ll * n_rows * heads : 0}};
  const trc::Rows from = {d_q, 2 * q_stride, 128ll * heads};
  if (trc::overlap(spans, 2) || trc::overlap(spans[1], from.span(n_rows)) || trc::overlap(to, from, n_rows))
    return set_last_error(TRC_E_INVALID, "cache attention: what is written overlaps another argument");
  const int sms = trc::sm_count();
  if (!sms) return set_last_error(TRC_E_CUDA, "cache attention: no current CUDA device");
  trc::CacheAttnArgs a;
  a.q = d_q;
  a.out = d_out;
  a.q_stride = q_stride;
  a.out_stride = out_stride;
  a.gates = d_gates;
  a.table = d_table;
  a.cu = d_cu;
  a.total = d_total;
  a.ws = static_cast<float*>(d_workspace);
  a.status = d_status;
  a.n_seqs = n_seqs;
  a.n_tokens = n_rows;
  a.hq = heads;
  a.hkv = kv_heads;
  a.group = heads / kv_heads;
  a.table_stride = table_stride;
  a.page_log2 = lp;
  a.n_pages = n_pages;
  a.causal = causal != 0;
  a.window = window > 1 << 30 ? 0 : window;  // longer than any sequence
  a.second = 0;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.split = max_total > TRC_CACHE_MAX_WHOLE;
  a.min_share = a.split ? 2 : 1;  // steps: a part of less than 128 keys costs more to join than it saves
  const trc::Layout l = trc::layout_of(max_new, a.group, sms);
  if (a.split && (!d_workspace || reinterpret_cast<uintptr_t>(d_workspace) % 16 ||
                  workspace_bytes < 4 * (l.floats + l.floats2)))
    return set_last_error(TRC_E_INVALID, "cache attention: workspace missing or smaller than trc_cache_workspace");
  cudaStream_t st = (cudaStream_t)stream;
  return precision == TRC_PREC_FP16
             ? trc::launch_cache_attention<__half>(l, page, d_k, d_v, a, sms, st)
             : trc::launch_cache_attention<__nv_bfloat16>(l, page, d_k, d_v, a, sms, st);
}

}  // extern "C"
