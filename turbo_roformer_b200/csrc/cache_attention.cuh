// Attention of a few new frames over the paged cache: O = gate * softmax(scale Q K^T) V with the rows of one
// (sequence, cache head) against all its keys, for up to 32 rows at a time (new frames x query heads that share
// the cache head).
//
// With few rows the work is reading K and V: 256 bytes per key and head against 4 x 64 flop per row, so HBM bounds it,
// and a 128-row tcgen05 tile would be mostly padding whose softmax still takes a thread per row. mma.sync m16n8k16
// tiles follow the row count in steps of 16 and keep scores, weights and sums in registers.
//   * Every warp is a worker with its own share of the line (cache_sched.cuh) and its own ring of 32-key tiles, which
//     TMA fills straight from the pages (a page's rows of one head are contiguous: one box per page and tile, 128-byte
//     swizzle). It refills a stage itself as soon as it has read it: no producer, no barrier between warps. 24 KB in
//     flight per warp, eight warps per SM, cover HBM's latency. Consecutive workers sit in different CTAs, so that few
//     of them spread over the SMs.
//   * Running maximum raised only past 2^8 (kRescaleThreshold): a lane compares its own scores with it, and only if
//     some lane of the warp exceeds it are maxima exchanged and sums rescaled.
//   * Weights are rounded to the 16-bit type for the product with V (relative error at most half a step each, averaged
//     over the keys); their sum is taken in fp32 before that rounding.
//   * Keys outside [lo, hi) of the item: K's scores are replaced (never added to) and V's fragments zeroed, so
//     whatever a page holds behind a sequence's end, NaN included, does not reach a sum.
// Measured: 300,000 frames x 8 heads, one row (614 MB): 106 us, 5.8 TB/s, 0.88 of the copy rate; 1,700 frames x 496
// heads (216 MB): 45 us with 5 us of set-up and 3 us of the join. What is left is the end: equal shares finish between
// 75 and 102 us on different SMs. With a CTA per worker whose warps join at every run's end, ragged pushes of 5 x 496
// heads took 152 us instead of 117.
// Every wait is bounded (sm100.cuh); after one gave up the status word tells the host.
#pragma once

#include "attention.cuh"  // kRescaleThreshold
#include "cache_sched.cuh"

namespace trc {

__device__ __forceinline__ void ldmatrix_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

// D (16 x 8, fp32) += A (16 x 16) B (16 x 8), 16-bit operands
template <typename T>
__device__ __forceinline__ void mma_m16n8k16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma_m16n8k16<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                                     uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
               "{%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma_m16n8k16<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                                            uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
               "{%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

constexpr int kCrWarps = 4;
constexpr int kCrKeys = 32;   // keys of a tile
constexpr int kCrStages = 3;  // tiles in a warp's ring

// Shared memory: a ring per warp (K then V of each stage), barriers, scan.
struct CrSmem {
  static constexpr int kTile = kCrKeys * 128;
  static constexpr int kStage = 2 * kTile;
  static constexpr int kBar = kCrWarps * kCrStages * kStage;
  static constexpr int kScan = kBar + kCrWarps * kCrStages * 8 + 16 + 32 * 8;
  static constexpr int bytes(int n_seqs) { return kScan + (n_seqs + 1) * 8 + 1024; }
};

template <typename T, int MT>
__global__ void __launch_bounds__(32 * kCrWarps, 2)
    cache_rows_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                      const __grid_constant__ CacheAttnArgs args) {
  using S = CrSmem;
  constexpr int kRows = 16 * MT;
  constexpr int NT = kCrKeys / 8;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::kBar);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars + kCrWarps * kCrStages);
  int64_t* part = reinterpret_cast<int64_t*>(bars + kCrWarps * kCrStages + 2);
  int64_t* prefix = reinterpret_cast<int64_t*>(smem + S::kScan);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint64_t* full = bars + warp * kCrStages;
  uint8_t* ring = smem + warp * kCrStages * S::kStage;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kCrWarps * kCrStages; ++i) mbar_init(&bars[i], 1);
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&map_k);
    tma_prefetch_desc(&map_v);
  }
  // Behind a cache_tiles_kernel this launch need not wait to begin: that one's blocks have all waited for what came
  // before them, and it takes other rows and another workspace. It fills the SMs that the other leaves, and waits for
  // it at its own end, so that whatever follows has both behind it.
  cache_prefetch(args);
  if (!args.second) grid_wait();
  grid_release();
  const int tpt = kRows / args.group;
  // its barriers cover the initialisation above
  const int workers = gridDim.x * kCrWarps, worker = warp * gridDim.x + blockIdx.x;
  const bool split = cache_scan(args, tpt, 32 * kCrWarps, workers, prefix, part);

  CacheWalk cons;
  cons.begin(args, tpt, prefix, worker, workers, split);
  if (args.split && lane == 0) cache_record(args, worker)->parts = 0;
  if (!cons.valid) {
    if (args.second) grid_wait();
    return;
  }
  bool ok = true;

  // ---- loads. The warp's next tile: pj of a run that ends before tile p_end and sees keys [p_lo, p_hi); lane b holds
  // the page of its box b (read a tile ahead of its use; -1: no row sees a key of the box). pj < 0: no more.
  const int box = min(1 << args.page_log2, kCrKeys), boxes = kCrKeys / box;  // keys per box, boxes per tile
  const int in_page = (1 << args.page_log2) - 1;
  const int nowhere = (args.n_pages * args.hkv) << args.page_log2;  // behind the pool: TMA's zero fill
  constexpr int kPer = kCacheStep / kCrKeys;
  auto tiles_begin = [&](const CacheWalk& w) { return max(w.a0 * kPer, w.it.lo / kCrKeys); };
  auto tiles_end = [&](const CacheWalk& w) { return min(w.a1 * kPer, (w.it.hi + kCrKeys - 1) / kCrKeys); };
  CacheWalk prod = cons;
  int pj = -1, p_end = 0, p_lo = 0, p_hi = 0, p_head = 0, p_page = -1;
  const int32_t* p_table = nullptr;
  auto look_up = [&]() {
    const int key = pj * kCrKeys + lane * box;
    p_page = -1;
    if (lane < boxes && key < p_hi && key + box > p_lo) p_page = p_table[key >> args.page_log2];
  };
  auto enter = [&]() {  // the first run from `prod` on that has a tile
    for (pj = -1; prod.valid; prod.advance(args, tpt)) {
      pj = tiles_begin(prod);
      p_end = tiles_end(prod);
      if (pj < p_end) {
        p_lo = prod.it.lo;
        p_hi = prod.it.hi;
        p_head = prod.it.head;
        p_table = args.table + (int64_t)prod.it.r * args.table_stride;
        prod.advance(args, tpt);
        look_up();
        return;
      }
      pj = -1;
    }
  };
  int p_st = 0, issued = 0;
  auto issue = [&]() {
    if (pj < 0) return;
    if (lane == 0) mbar_arrive_expect_tx(&full[p_st], S::kStage);
    __syncwarp();
    if (lane < boxes) {
      const int key = pj * kCrKeys + lane * box;
      int y = nowhere;
      if ((unsigned)p_page < (unsigned)args.n_pages)
        y = ((p_page * args.hkv + p_head) << args.page_log2) + (key & in_page);
      else if (key < p_hi && key + box > p_lo)
        record_error(args.status, kErrBadArgs);
      uint8_t* dst = ring + p_st * S::kStage + lane * box * 128;
      tma_load_2d(dst, &map_k, &full[p_st], 0, y);
      tma_load_2d(dst + S::kTile, &map_v, &full[p_st], 0, y);
    }
    p_st = p_st == kCrStages - 1 ? 0 : p_st + 1;
    ++issued;
    if (++pj < p_end)
      look_up();
    else
      enter();
  };
  enter();
  for (int i = 0; i < kCrStages; ++i) issue();

  const int g4 = lane >> 2, c2 = (lane & 3) * 2;
  // ldmatrix addresses within a tile: row r's 16-byte chunk c lies at chunk c ^ (r % 8)
  const uint32_t k_off = (lane & 7) * 128 + (((lane >> 3) ^ (lane & 7)) << 4);
  const uint32_t v_off = (((lane >> 3) & 1) * 8 + (lane & 7)) * 128 + (((lane >> 4) ^ (lane & 7)) << 4) + S::kTile;
  const float2 scale2 = make_float2(args.scale_log2, args.scale_log2);
  int st = 0;
  uint32_t phase = 0;
  for (; cons.valid; cons.advance(args, tpt)) {
    const CacheItem& it = cons.it;
    // ---- this lane's rows: row = (frame of the tile) * group + query head within the group
    uint32_t qf[MT][4][4];
    int lo[MT][2], hi[MT][2];
    int64_t row_out[MT][2];
    float gate[MT][2];
    int hi_min = INT_MAX, lo_max = 0;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int row = mt * 16 + h * 8 + g4;
        const int i = row / args.group, head = it.head * args.group + (row - i * args.group);
        const bool live = i < it.ntok;
        const int64_t tok = it.s.tok + it.tok0 + i;
        const T* src = static_cast<const T*>(args.q) + tok * args.q_stride + head * 64;
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          qf[mt][kk][h] = live ? *reinterpret_cast<const uint32_t*>(src + kk * 16 + c2) : 0u;
          qf[mt][kk][2 + h] = live ? *reinterpret_cast<const uint32_t*>(src + kk * 16 + 8 + c2) : 0u;
        }
        hi[mt][h] = live ? cache_hi(args, it.s, it.tok0 + i) : INT_MAX;
        lo[mt][h] = live ? cache_lo(args, it.s, it.tok0 + i) : 0;
        hi_min = min(hi_min, hi[mt][h]);
        lo_max = max(lo_max, lo[mt][h]);
        row_out[mt][h] = live ? tok * args.out_stride + head * 64 : -1;
        gate[mt][h] = live && args.gates ? args.gates[tok * args.hq + head] : 1.f;
      }
    hi_min = __reduce_min_sync(0xffffffffu, hi_min);
    lo_max = __reduce_max_sync(0xffffffffu, lo_max);

    float o[MT][8][4], m_run[MT][2], shift[MT][2];
    float2 l2[MT][2];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
      for (int n = 0; n < 8; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[mt][n][i] = 0.f;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        m_run[mt][h] = -INFINITY;
        shift[mt][h] = 0.f;
        l2[mt][h] = make_float2(0.f, 0.f);
      }
    }

    const int tend = tiles_end(cons);
    for (int t = tiles_begin(cons); t < tend && ok; ++t) {
      ok = mbar_wait_warp(&full[st], phase, args.status, kErrWaitMma, abort_flag);
      if (!ok) break;
      const uint32_t base = smem_u32(ring) + st * S::kStage;
      const int key0 = t * kCrKeys;
      // ---- S = Q K^T
      float s[MT][NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        uint32_t b[2][4];
        ldmatrix_x4(base + n * 1024 + k_off, b[0]);
        ldmatrix_x4(base + n * 1024 + (k_off ^ 64), b[1]);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
          for (int i = 0; i < 4; ++i) s[mt][n][i] = 0.f;
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            mma_m16n8k16<T>(s[mt][n], qf[mt][kk], b[kk >> 1][(kk & 1) * 2], b[kk >> 1][(kk & 1) * 2 + 1]);
        }
      }
      if (key0 + kCrKeys > hi_min || key0 < lo_max) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int key = key0 + n * 8 + c2 + (i & 1), h = i >> 1;
              if (key >= hi[mt][h] || key < lo[mt][h]) s[mt][n][i] = -INFINITY;
            }
      }
      // ---- running maximum: this lane's scores against it
      float m_new[MT][2];
      bool need = false;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float m = fmaxf(s[mt][0][2 * h], s[mt][0][2 * h + 1]);
#pragma unroll
          for (int n = 1; n < NT; ++n) m = fmax3(m, s[mt][n][2 * h], s[mt][n][2 * h + 1]);
          m_new[mt][h] = m * args.scale_log2;
          need |= m_new[mt][h] > m_run[mt][h] + kRescaleThreshold;
        }
      if (__any_sync(0xffffffffu, need)) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float m = m_new[mt][h];  // the row's: over its four lanes
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
            if (m > m_run[mt][h] + kRescaleThreshold) {
              // from -inf, before the first visible key: sum and weight are zero, 2^-inf = 0 keeps them
              const float alpha = ex2_approx(m_run[mt][h] - m);
              m_run[mt][h] = m;
              shift[mt][h] = -m;
              l2[mt][h].x *= alpha;
              l2[mt][h].y *= alpha;
#pragma unroll
              for (int n = 0; n < 8; ++n) {
                o[mt][n][2 * h] *= alpha;
                o[mt][n][2 * h + 1] *= alpha;
              }
            }
          }
      }
      // ---- weights, and O += P V
      const bool edge = key0 + kCrKeys > it.hi || key0 < it.lo;
#pragma unroll
      for (int ks = 0; ks < kCrKeys / 16; ++ks) {
        uint32_t p[MT][4];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float* x = &s[mt][2 * ks + half][2 * h];
              const float2 e = __ffma2_rn(make_float2(x[0], x[1]), scale2, make_float2(shift[mt][h], shift[mt][h]));
              const float2 w = make_float2(ex2_approx(e.x), ex2_approx(e.y));
              l2[mt][h] = __fadd2_rn(l2[mt][h], w);
              p[mt][half * 2 + h] = OperandType<T>::pack2(w.x, w.y);
            }
#pragma unroll
        for (int dp = 0; dp < 4; ++dp) {
          uint32_t b[4];
          ldmatrix_x4_trans(base + ks * 2048 + (v_off ^ (dp * 32)), b);
          if (edge) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int key = key0 + ks * 16 + (i & 1) * 8 + c2;
              uint32_t keep = 0;
              if (key >= it.lo && key < it.hi) keep |= 0x0000ffffu;
              if (key + 1 >= it.lo && key + 1 < it.hi) keep |= 0xffff0000u;
              b[i] &= keep;
            }
          }
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            mma_m16n8k16<T>(o[mt][dp * 2], p[mt], b[0], b[1]);
            mma_m16n8k16<T>(o[mt][dp * 2 + 1], p[mt], b[2], b[3]);
          }
        }
      }
      if (++st == kCrStages) {
        st = 0;
        phase ^= 1;
      }
      __syncwarp();
      issue();
    }
    // ---- a row's weight over its four lanes
    float l_run[MT][2];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float l = l2[mt][h].x + l2[mt][h].y;
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l_run[mt][h] = l + __shfl_xor_sync(0xffffffffu, l, 2);
      }
    if (!ok) break;
    // ---- results, or this run's part of them
    const bool whole = cons.whole();
    float* slot = whole ? nullptr : cache_slot(args, kRows, workers, 2 * worker + cons.slot());
    if (!whole && cons.slot() == 1 && lane == 0)
      *cache_record(args, worker) = {cons.parts(args), it.s.tok + it.tok0, it.ntok, it.head};
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (row_out[mt][h] < 0) continue;
        if (whole) {
          const float f = l_run[mt][h] == 0.f ? 0.f : gate[mt][h] / l_run[mt][h];  // no visible key: zero
          T* dst = static_cast<T*>(args.out) + row_out[mt][h] + c2;
#pragma unroll
          for (int n = 0; n < 8; ++n)
            *reinterpret_cast<uint32_t*>(dst + n * 8) =
                OperandType<T>::pack2(o[mt][n][2 * h] * f, o[mt][n][2 * h + 1] * f);
        } else {
          const int row = mt * 16 + h * 8 + g4;
          float* dst = slot + row * 64 + c2;
#pragma unroll
          for (int n = 0; n < 8; ++n)
            *reinterpret_cast<float2*>(dst + n * 8) = make_float2(o[mt][n][2 * h], o[mt][n][2 * h + 1]);
          if (c2 == 0)
            *reinterpret_cast<float2*>(slot + kRows * 64 + row * 2) = make_float2(m_run[mt][h], l_run[mt][h]);
        }
      }
  }
  // after a wait that gave up, copies may still be in flight: let them land before shared memory is given back
  if (!ok && lane == 0) {
    const uint64_t t0 = global_ns();
    for (int k = max(0, issued - kCrStages); k < issued; ++k)
      while (!mbar_try_wait(&full[k % kCrStages], (uint32_t)(k / kCrStages) & 1) && global_ns() - t0 < kWaitLimitNs) {
      }
  }
  if (args.second) grid_wait();
}

// Joins the parts of items that were divided among workers, for the workers of cache_rows_kernel (0 .. workers - 1) and,
// behind them, those of cache_tiles_kernel, with a workspace of its own. A block takes the item that its worker began
// and did not end, if there is one. Few rows: a warp takes a row at a time and reads two parts at once (16 lanes x 4
// dims each); where an item has few rows in many parts, 2, 4 or 8 warps share a row and meet in shared memory. Tiles:
// kJoinBlocks blocks share an item, a thread takes 4 dims of a row, consecutive threads consecutive rows.
constexpr int kJoinBlocks = 8;
struct CacheJoin {
  int workers, rows;  // of the first launch; rows of its slots
  int rows2;
  float* ws2;
};
struct JoinSum {
  float m, l;
  float4 o;
  __device__ __forceinline__ void add(float m2, float l2, float4 x) {
    const float mn = fmaxf(m, m2);
    const float f1 = mn == -INFINITY ? 1.f : ex2_approx(m - mn), f2 = mn == -INFINITY ? 1.f : ex2_approx(m2 - mn);
    m = mn;
    l = l * f1 + l2 * f2;
    o = make_float4(o.x * f1 + x.x * f2, o.y * f1 + x.y * f2, o.z * f1 + x.z * f2, o.w * f1 + x.w * f2);
  }
};
// dims d .. d + 3 of a joined row
template <typename T>
__device__ __forceinline__ void join_store(const CacheAttnArgs& args, const CacheRecord& rec, int row, int d,
                                           const JoinSum& s) {
  const int i = row / args.group, head = rec.head * args.group + (row - i * args.group);
  const int64_t tok = rec.tok + i;
  const float gate = args.gates ? args.gates[tok * args.hq + head] : 1.f;
  const float f = s.l == 0.f ? 0.f : gate / s.l;  // no visible key: zero
  uint2 u;
  u.x = OperandType<T>::pack2(s.o.x * f, s.o.y * f);
  u.y = OperandType<T>::pack2(s.o.z * f, s.o.w * f);
  *reinterpret_cast<uint2*>(static_cast<T*>(args.out) + tok * args.out_stride + head * 64 + d) = u;
}
template <typename T>
__global__ void __launch_bounds__(256) cache_join_kernel(const __grid_constant__ CacheAttnArgs first,
                                                         const __grid_constant__ CacheJoin j) {
  __shared__ float4 meet_o[8][16];
  __shared__ float2 meet_ml[8][16];
  grid_wait();
  grid_release();
  CacheAttnArgs args = first;
  int worker = blockIdx.x, workers = j.workers, tile_rows = j.rows, y = 0, ny = 1;
  if (worker >= j.workers) {  // kJoinBlocks per worker of the second launch
    ny = kJoinBlocks;
    y = (worker - j.workers) % ny;
    worker = (worker - j.workers) / ny;
    workers = ((int)gridDim.x - j.workers) / ny;
    tile_rows = j.rows2;
    args.ws = j.ws2;
  }
  const CacheRecord rec = *cache_record(args, worker);
  if (rec.parts == 0) return;
  const int rows = rec.ntok * args.group;
  if (ny > 1) {
    const int padded = (rows + 31) & ~31;
    for (int x = y * 256 + threadIdx.x; x < 16 * padded; x += ny * 256) {
      const int k = x / padded, row = x - k * padded;
      if (row >= rows) continue;
      JoinSum s = {-INFINITY, 0.f, make_float4(0.f, 0.f, 0.f, 0.f)};
#pragma unroll 4
      for (int p = 0; p < rec.parts; ++p) {
        const float* src = cache_slot(args, tile_rows, workers, 2 * (worker + p) + (p == 0 ? 1 : 0));
        const float2 ml = *reinterpret_cast<const float2*>(src + tile_rows * 64 + row * 2);
        s.add(ml.x, ml.y, *reinterpret_cast<const float4*>(src + (k * tile_rows + row) * 4));
      }
      join_store<T>(args, rec, row, k * 4, s);
    }
    return;
  }
  const int share = rec.parts <= 4 || rows > 4 ? 1 : rows > 2 ? 2 : rows > 1 ? 4 : 8;  // warps per row
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int sub = lane >> 4, d = (lane & 15) * 4;
  const int per = 8 / share;  // rows of a block at a time
  for (int row0 = y * per; row0 < rows; row0 += ny * per) {
    const int row = row0 + warp / share;
    JoinSum s = {-INFINITY, 0.f, make_float4(0.f, 0.f, 0.f, 0.f)};
    if (row < rows) {
#pragma unroll 4
      for (int p = warp % share * 2 + sub; p < rec.parts; p += 2 * share) {
        const float* src = cache_slot(args, tile_rows, workers, 2 * (worker + p) + (p == 0 ? 1 : 0));
        const float2 ml = *reinterpret_cast<const float2*>(src + tile_rows * 64 + row * 2);
        s.add(ml.x, ml.y, *reinterpret_cast<const float4*>(src + row * 64 + d));
      }
      const float m2 = __shfl_xor_sync(0xffffffffu, s.m, 16), l2 = __shfl_xor_sync(0xffffffffu, s.l, 16);
      float4 x;
      x.x = __shfl_xor_sync(0xffffffffu, s.o.x, 16);
      x.y = __shfl_xor_sync(0xffffffffu, s.o.y, 16);
      x.z = __shfl_xor_sync(0xffffffffu, s.o.z, 16);
      x.w = __shfl_xor_sync(0xffffffffu, s.o.w, 16);
      s.add(m2, l2, x);
    }
    if (share > 1) {
      if (sub == 0) {
        meet_o[warp][lane] = s.o;
        meet_ml[warp][lane] = make_float2(s.m, s.l);
      }
      __syncthreads();
      if (warp % share == 0 && sub == 0)
        for (int w = warp + 1; w < warp + share; ++w) s.add(meet_ml[w][lane].x, meet_ml[w][lane].y, meet_o[w][lane]);
      __syncthreads();
    }
    if (row < rows && warp % share == 0 && sub == 0) join_store<T>(args, rec, row, d, s);
  }
}

}  // namespace trc
