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

// ------------------------------------------------------------------------------------------------ plan
// Every block repeats the scan over the sequences (two 64-bit sums per thread) and then takes its part of two
// flat ranges: the fresh pages (each finds its sequence by a search in the scan) and the rows. Nothing is
// exchanged between blocks, so one launch serves any batch: a row's page is either fresh (read from the free
// list, not from the table that another block is writing) or was in the table before.
struct PlanArgs {
  const int32_t* cached;
  const int32_t* fresh;  // new lengths
  const int32_t* free_pages;
  int32_t* table;
  int32_t *cu, *total, *slots, *positions, *counts;
  int n_seqs, page_log2, n_free, table_stride, capacity;
};

constexpr int kPlanThreads = 512;

__device__ __forceinline__ int pages_of(int64_t frames, int page_log2) {
  return (int)((frames + (1 << page_log2) - 1) >> page_log2);
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

__global__ void __launch_bounds__(kPlanThreads) cache_plan_kernel(const __grid_constant__ PlanArgs a) {
  extern __shared__ int32_t plan_smem[];
  int32_t* cu = plan_smem;                 // [n_seqs + 1] rows before each sequence
  int32_t* base = plan_smem + a.n_seqs + 1;  // [n_seqs + 1] fresh pages before each sequence
  __shared__ int64_t part[2][kPlanThreads / 32];
  __shared__ int flags;
  if (threadIdx.x == 0) flags = 0;
  grid_wait();
  grid_release();
  const int per = (a.n_seqs + kPlanThreads - 1) / kPlanThreads;
  const int r0 = min((int)threadIdx.x * per, a.n_seqs), r1 = min(r0 + per, a.n_seqs);
  int64_t rows = 0, pages = 0;
  int bad = 0;
  auto lengths = [&](int r, int& c, int& n) {
    c = a.cached[r];
    n = a.fresh[r];
    if (c < 0 || n < 0 || (int64_t)c + n > (1 << 30)) {
      bad |= TRC_CACHE_BAD_LENGTH;
      c = n = 0;
    }
  };
  for (int r = r0; r < r1; ++r) {
    int c, n;
    lengths(r, c, n);
    rows += n;
    pages += pages_of((int64_t)c + n, a.page_log2) - pages_of(c, a.page_log2);
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
  rs -= rows;
  ps -= pages;
  int64_t all_rows = 0, all_pages = 0;
#pragma unroll
  for (int w = 0; w < kPlanThreads / 32; ++w) {
    if (w < warp) {
      rs += part[0][w];
      ps += part[1][w];
    }
    all_rows += part[0][w];
    all_pages += part[1][w];
  }
  for (int r = r0; r < r1; ++r) {
    int c, n;
    lengths(r, c, n);
    cu[r] = (int)min(rs, (int64_t)INT_MAX);
    base[r] = (int)min(ps, (int64_t)INT_MAX);
    rs += n;
    ps += pages_of((int64_t)c + n, a.page_log2) - pages_of(c, a.page_log2);
    if (blockIdx.x == 0) {
      a.cu[r] = cu[r];
      a.total[r] = c + n;
      if (pages_of((int64_t)c + n, a.page_log2) > a.table_stride) bad |= TRC_CACHE_TABLE_FULL;
    }
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
    a.cu[a.n_seqs] = live_rows;
    a.counts[0] = min(live_pages, a.n_free);
    a.counts[1] = flags;
  }

  const int stride = gridDim.x * kPlanThreads, first = blockIdx.x * kPlanThreads + threadIdx.x;
  // fresh pages into the table
  for (int64_t e = first; e < live_pages; e += stride) {
    const int r = last_upto(base, a.n_seqs, (int)e);
    int c, n;
    lengths(r, c, n);
    const int64_t column = (int64_t)pages_of(c, a.page_log2) + (e - base[r]);
    if (column < a.table_stride)
      a.table[(int64_t)r * a.table_stride + column] = e < a.n_free ? a.free_pages[e] : -1;
  }
  // rows: position and slot
  for (int64_t row = first; row < a.capacity; row += stride) {
    int pos = 0, slot = -1;
    if (row < live_rows) {
      const int r = last_upto(cu, a.n_seqs, (int)row);
      int c, n;
      lengths(r, c, n);
      pos = c + (int)(row - cu[r]);
      const int column = pos >> a.page_log2, held = pages_of(c, a.page_log2);
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
        slot = (page << a.page_log2) + (pos & ((1 << a.page_log2) - 1));
    }
    a.positions[row] = pos;
    a.slots[row] = slot;
  }
}

// ------------------------------------------------------------------------------------------------ append
// One thread per 16-byte vector (8 elements = 4 rotary pairs) of the rows, kAppendVecs vectors per thread in
// flight; HBM bound (each element is read once and written once). A block takes a flat run of vectors, which may
// span many short rows or a part of a long one; the angles of its frames (position x frequency in fp64, reduced
// to half turns, because fp32 loses the angle of far positions) are computed once per block and shared by all
// heads.
constexpr int kAppendThreads = 256;
constexpr int kAppendVecs = 4;
constexpr int kAppendRun = kAppendThreads * kAppendVecs;
// frames that a run can touch: a frame has at least 24 vectors (one q, k and v head)
constexpr int kAppendFrames = kAppendRun / 24 + 2;

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
  int band_vecs, vecs;        // 16-byte vectors per band and per frame
  uint32_t band_mul, frame_mul;  // x / d = umulhi(x, mul) for the x that occur (see div_mul)
};

// umulhi(x, ceil(2^32 / d)) = x / d for x * d < 2^32 (the error x (mul d - 2^32) / (2^32 d) stays below 1 / d)
uint32_t div_mul(uint32_t d) { return d == 1 ? 0u : (uint32_t)((0x100000000ull + d - 1) / d); }
__device__ __forceinline__ uint32_t div_by(uint32_t x, uint32_t mul) { return mul ? __umulhi(x, mul) : x; }

template <typename T>
struct Vec8;
template <>
struct Vec8<__half> {
  __device__ static float2 to_f2(uint32_t u) { return __half22float2(*reinterpret_cast<__half2*>(&u)); }
};
template <>
struct Vec8<__nv_bfloat16> {
  __device__ static float2 to_f2(uint32_t u) { return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&u)); }
};

template <typename T>
__global__ void __launch_bounds__(kAppendThreads) cache_append_kernel(const __grid_constant__ AppendArgs a) {
  __shared__ float2 turn[kAppendFrames][32];  // (cos, sin) of each frame and pair
  grid_wait();
  grid_release();
  const int64_t run0 = (int64_t)blockIdx.x * kAppendRun;
  const int frame0 = (int)(run0 / a.vecs);
  const uint32_t rem0 = (uint32_t)(run0 - (int64_t)frame0 * a.vecs);

  // the run's loads first: the angles are computed while they travel
  uint4 data[kAppendVecs];
  int frame[kAppendVecs], band[kAppendVecs], sub[kAppendVecs];
#pragma unroll
  for (int i = 0; i < kAppendVecs; ++i) {
    const uint32_t x = rem0 + i * kAppendThreads + threadIdx.x;
    const uint32_t f = div_by(x, a.frame_mul);
    const uint32_t in = x - f * a.vecs;
    const uint32_t b = div_by(in, a.band_mul);
    frame[i] = (int)f;
    band[i] = (int)b;
    sub[i] = (int)(in - b * a.band_vecs);
    const int64_t tok = (int64_t)frame0 + f;
    data[i] = make_uint4(0, 0, 0, 0);
    if (tok >= a.n_tokens || a.slots[tok] < 0) {
      frame[i] = -1;  // behind the last row, or a row of padding
    } else {
      const T* src = static_cast<const T*>(a.qkv) + tok * a.tok_stride + b * a.band_stride + (int64_t)sub[i] * 8;
      const int gate0 = (a.heads + 2 * a.kv_heads) * 8;
      if (sub[i] < gate0 || (sub[i] - gate0) * 8 + 8 <= a.heads) {
        data[i] = __ldcs(reinterpret_cast<const uint4*>(src));
      } else {  // the last gates: no reads behind them
        uint16_t tail[8] = {};
        for (int e = 0; e < a.heads - (sub[i] - gate0) * 8; ++e) tail[e] = reinterpret_cast<const uint16_t*>(src)[e];
        data[i] = make_uint4(tail[0] | (uint32_t)tail[1] << 16, tail[2] | (uint32_t)tail[3] << 16,
                             tail[4] | (uint32_t)tail[5] << 16, tail[6] | (uint32_t)tail[7] << 16);
      }
    }
  }
  const int frames = (int)div_by(rem0 + kAppendRun - 1, a.frame_mul) + 1;
  for (int x = threadIdx.x; x < frames * 32; x += kAppendThreads) {
    const int64_t tok = (int64_t)frame0 + (x >> 5);
    float2 t = make_float2(1.f, 0.f);
    if (a.freqs && tok < a.n_tokens) {
      // half turns: the angle over pi, modulo 2; fp64 keeps 1e-9 of a turn at positions past 2^30
      const double h = (double)a.positions[tok] * (double)a.freqs[x & 31] * 0.31830988618379067154;
      sincospif((float)(h - 2.0 * rint(0.5 * h)), &t.y, &t.x);
    }
    turn[x >> 5][x & 31] = t;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kAppendVecs; ++i) {
    if (frame[i] < 0) continue;
    const int64_t tok = (int64_t)frame0 + frame[i];
    const int head = sub[i] >> 3, d = (sub[i] & 7) * 8;
    uint32_t u[4] = {data[i].x, data[i].y, data[i].z, data[i].w};
    if (head < a.heads + a.kv_heads && a.freqs) {
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        const float2 x = Vec8<T>::to_f2(u[p]), t = turn[frame[i]][(d >> 1) + p];
        u[p] = OperandType<T>::pack2(x.x * t.x - x.y * t.y, x.y * t.x + x.x * t.y);
      }
    }
    const uint4 out = make_uint4(u[0], u[1], u[2], u[3]);
    if (head < a.heads) {
      T* dst = static_cast<T*>(a.q) + tok * a.q_stride + ((int64_t)band[i] * a.heads + head) * 64 + d;
      *reinterpret_cast<uint4*>(dst) = out;
    } else if (head < a.heads + 2 * a.kv_heads) {
      const int64_t slot = a.slots[tok];
      if (slot >= a.n_slots) {
        record_error(a.status, kErrBadArgs);
        continue;
      }
      const bool is_v = head >= a.heads + a.kv_heads;
      const int64_t kvh = (int64_t)band[i] * a.kv_heads + head - a.heads - (is_v ? a.kv_heads : 0);
      const int64_t page = slot >> a.page_log2, in_page = slot & ((1 << a.page_log2) - 1);
      T* dst = static_cast<T*>(is_v ? a.v : a.k) +
               ((((page * a.bands * a.kv_heads + kvh) << a.page_log2) + in_page) * 64 + d);
      *reinterpret_cast<uint4*>(dst) = out;
    } else {
      const int h0 = (sub[i] - (a.heads + 2 * a.kv_heads) * 8) * 8;
      float* dst = a.gates + (tok * a.bands + band[i]) * a.heads + h0;
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        const float2 x = Vec8<T>::to_f2(u[p]);
        if (h0 + 2 * p < a.heads) dst[2 * p] = 1.0f / (1.0f + expf(-x.x));
        if (h0 + 2 * p + 1 < a.heads) dst[2 * p + 1] = 1.0f / (1.0f + expf(-x.y));
      }
    }
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

// Which kernel takes a sequence, by its rows per cache head (new frames x query heads that share it). Measured with
// 496 heads over 1,700 frames (us; HBM floor 34-43 us):
//   rows                        16   20   28   40   64  128  200  256  384
//   cache_rows_kernel           ROWS_FIGURES
//   cache_tiles_kernel          SEPARATE_FIGURES
//   cache_tiles_kernel, shared  SHARED_FIGURES
constexpr int kFewRows = 32;      // cache_rows_kernel
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
  int rc = maps(kCrKeys, mk, mv);
  if (rc) return rc;
  float* const ws2 = a.ws ? a.ws + l.floats : nullptr;
  a.rows_above = 0;
  a.rows_upto = l.tiles ? kFewRows : INT_MAX;
  rc = l.rows == 16 ? launch_rows<T, 1>(mk, mv, a, l.workers, st) : launch_rows<T, 2>(mk, mv, a, l.workers, st);
  if (rc) return rc;
  if (l.tiles) {
    CacheAttnArgs b = a;
    b.rows_above = kFewRows;
    b.rows_upto = INT_MAX;
    b.ws = ws2;
    if ((rc = maps(kCacheStep, mk, mv))) return rc;
    rc = l.shared ? launch_tiles<T, true>(mk, mv, b, sms, st) : launch_tiles<T, false>(mk, mv, b, sms, st);
    if (rc) return rc;
  }
  if (!a.split) return TRC_OK;
  const CacheJoin j = {l.workers, l.rows, l.rows2, ws2};
  return launch("cache attention join", cache_join_kernel<T>, dim3(l.workers + l.workers2, l.tiles ? 4 : 1), 256, 0, st,
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
  const int smem = 2 * (n_seqs + 1) * 4;
  static std::atomic<unsigned long long> done{0};
  int dev = 0;
  cudaGetDevice(&dev);
  if (!(done.load(std::memory_order_relaxed) >> (dev & 63) & 1)) {
    const cudaError_t e = cudaFuncSetAttribute(trc::cache_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               2 * (TRC_CACHE_PLAN_MAX_SEQS + 1) * 4);
    if (e != cudaSuccess) return set_last_error(TRC_E_CUDA, cudaGetErrorString(e));
    done.fetch_or(1ull << (dev & 63));
  }
  // blocks for the rows; the fresh pages are at most as many plus one per sequence
  const int64_t most = (int64_t)max_rows + n_seqs;
  const int blocks = (int)((most + trc::kPlanThreads - 1) / trc::kPlanThreads);
  return trc::launch("cache plan", trc::cache_plan_kernel, dim3(blocks < 2 * sms ? blocks : 2 * sms), trc::kPlanThreads,
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
      reinterpret_cast<uintptr_t>(d_v) % 16)
    return set_last_error(TRC_E_INVALID, "cache append: rows must start on 16-byte boundaries");
  if ((bands > 1 && band_stride < width) || (n_rows > 1 && q_stride < (int64_t)bands * heads * 64))
    return set_last_error(TRC_E_INVALID, "cache append: strides shorter than the rows");
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
  a.band_vecs = (heads + 2 * kv_heads) * 8 + (d_gates ? (heads + 7) / 8 : 0);
  const int64_t vecs = (int64_t)bands * a.band_vecs;
  // div_mul's range: an index below vecs + a run, times the divisor
  if ((vecs + trc::kAppendRun) * vecs >= (int64_t)1 << 32)
    return set_last_error(TRC_E_INVALID, "cache append: bands x heads too large");
  a.vecs = (int)vecs;
  a.band_mul = trc::div_mul((uint32_t)a.band_vecs);
  a.frame_mul = trc::div_mul((uint32_t)vecs);
  const int64_t blocks = ((int64_t)n_rows * vecs + trc::kAppendRun - 1) / trc::kAppendRun;
  if (blocks > INT_MAX) return set_last_error(TRC_E_INVALID, "cache append: too many rows");
  cudaStream_t st = (cudaStream_t)stream;
  auto kern = precision == TRC_PREC_FP16 ? trc::cache_append_kernel<__half> : trc::cache_append_kernel<__nv_bfloat16>;
  return trc::launch("cache append", kern, dim3((unsigned)blocks), trc::kAppendThreads, 0, st, a);
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
