// Attention of a few new frames over the paged cache: O = gate * softmax(scale Q K^T) V with the rows of one
// (sequence, cache head) against all its keys, for up to 128 rows at a time (new frames x query heads that share
// the cache head).
//
// With few rows the work is reading K and V: 256 bytes per key and head against 4 x 64 flop per row, so below
// about 200 rows HBM bounds it, and a 128-row tcgen05 tile would be mostly padding whose softmax still takes a
// thread per row. mma.sync m16n8k16 tiles follow the row count in steps of 16 and keep scores, weights and sums
// in registers. K and V tiles arrive by TMA straight from the pages (a page's rows of one head are contiguous:
// one box per page and tile) into a ring of 128-byte-swizzled stages, enough in flight per SM to cover HBM's
// latency.
//   * WM warps share a tile's keys, 16 x MT rows each; WK groups of them take different key tiles, each with a
//     ring of its own, and join at the end of a run through shared memory (a fixed tree, no atomics).
//   * Running maximum raised only past 2^8 (kRescaleThreshold); weights rounded to the 16-bit type for the
//     product with V (relative error at most half a step each, averaged over the keys), their sum kept in fp32
//     before that rounding.
//   * Keys outside [lo, hi) of the item: K's scores are replaced (never added to) and V's fragments zeroed, so
//     whatever a page holds behind a sequence's end, NaN included, does not reach a sum.
// Every wait is bounded (sm100.cuh); a warp whose wait gave up goes on without waiting, so that the CTA's
// barriers still meet, and the status word tells the host.
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

// Shared memory of the kernel: per group ST stages of KT keys (K then V), the join's scratch, barriers, scan.
template <int MT, int WM, int WK, int KT, int ST>
struct CacheRowsSmem {
  static constexpr int kTile = KT * 128;
  static constexpr int kStage = 2 * kTile;
  static constexpr int kRing = WK * ST * kStage;
  // half of the groups hand their rows over at a time: MT x 32 sums and 4 MT statistics per lane
  static constexpr int kJoin = WK > 1 ? (WK / 2) * WM * MT * (32 + 4) * 32 * 4 : 0;
  static constexpr int kBar = kRing + kJoin;
  static constexpr int kScan = kBar + 2 * WK * ST * 8 + 16 + 32 * 8;
  static constexpr int bytes(int n_seqs) { return kScan + (n_seqs + 1) * 8 + 1024; }
};

template <typename T, int MT, int WM, int WK, int KT, int ST>
__global__ void __launch_bounds__(32 * WM * WK, 2)
    cache_rows_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                      const __grid_constant__ CacheAttnArgs args) {
  using S = CacheRowsSmem<MT, WM, WK, KT, ST>;
  constexpr int kThreads = 32 * WM * WK;
  constexpr int kRows = 16 * MT * WM;
  constexpr int NT = KT / 8;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::kBar);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars + 2 * WK * ST);
  int64_t* part = reinterpret_cast<int64_t*>(bars + 2 * WK * ST + 2);
  int64_t* prefix = reinterpret_cast<int64_t*>(smem + S::kScan);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int wm = warp % WM, wk = warp / WM;
  uint64_t* full = bars + wk * ST;
  uint64_t* empty = bars + (WK + wk) * ST;
  uint8_t* ring = smem + wk * ST * S::kStage;
  if (threadIdx.x == 0) {
    for (int i = 0; i < WK * ST; ++i) {
      mbar_init(&bars[i], 1);
      mbar_init(&bars[WK * ST + i], WM);
    }
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&map_k);
    tma_prefetch_desc(&map_v);
  }
  const int tpt = kRows / args.group;
  const bool split = cache_scan(args, tpt, kThreads, gridDim.x, prefix, part);  // its barriers cover the above

  CacheWalk cons;
  cons.begin(args, tpt, prefix, blockIdx.x, gridDim.x, split);
  if (args.split && threadIdx.x == 0) cache_record(args, blockIdx.x)->parts = 0;
  if (!cons.valid) return;
  bool ok = true;

  // ---- loads: the group's first warp walks the same runs ahead of the products
  const int box = min(1 << args.page_log2, KT), boxes = KT / box;  // keys per box, boxes per tile
  CacheWalk prod = cons;
  int issued = 0, page_next = -1;
  // key tile (of KT keys) within the run, by group
  auto tiles_begin = [&](const CacheWalk& w) { return max(w.a0 * (kCacheStep / KT), w.it.lo / KT); };
  auto tiles_end = [&](const CacheWalk& w) { return min(w.a1 * (kCacheStep / KT), (w.it.hi + KT - 1) / KT); };
  int prod_tile = tiles_begin(prod) + wk;
  auto settle = [&]() {  // the next run in which this group has a tile
    while (prod.valid && prod_tile >= tiles_end(prod)) {
      prod.advance(args, tpt);
      if (prod.valid) prod_tile = tiles_begin(prod) + wk;
    }
  };
  auto fetch_page = [&]() {  // lane b: the page of box b of the next tile (loaded a tile ahead of its use)
    page_next = -1;
    if (prod.valid && lane < boxes) {
      const int key = prod_tile * KT + lane * box;
      if (key < prod.it.hi && key + box > prod.it.lo)
        page_next = args.table[(int64_t)prod.it.r * args.table_stride + (key >> args.page_log2)];
    }
  };
  auto issue = [&]() {
    if (!prod.valid) return;
    const int st = issued % ST;
    if (WM > 1 && issued >= ST && ok)
      ok = mbar_wait_warp(&empty[st], (uint32_t)(issued / ST - 1) & 1, args.status, kErrWaitProducer, abort_flag);
    if (!ok) return;
    if (lane == 0) mbar_arrive_expect_tx(&full[st], S::kStage);
    __syncwarp();
    if (lane < boxes) {
      const int key = prod_tile * KT + lane * box;
      // a box that no row sees, or whose page number is bad, reads the zero fill behind the pool
      int64_t y = (int64_t)args.n_pages * args.hkv << args.page_log2;
      if (page_next >= 0 && page_next < args.n_pages)
        y = (((int64_t)page_next * args.hkv + prod.it.head) << args.page_log2) + (key & ((1 << args.page_log2) - 1));
      else if (key < prod.it.hi && key + box > prod.it.lo)
        record_error(args.status, kErrBadArgs);
      uint8_t* dst = ring + st * S::kStage + lane * box * 128;
      tma_load_2d(dst, &map_k, &full[st], 0, (int)y);
      tma_load_2d(dst + S::kTile, &map_v, &full[st], 0, (int)y);
    }
    ++issued;
    prod_tile += WK;
    settle();
    fetch_page();
  };
  if (wm == 0) {
    settle();
    fetch_page();
    for (int i = 0; i < ST; ++i) issue();
  }

  const int g4 = lane >> 2, c2 = (lane & 3) * 2;
  int used = 0;
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
        const int row = (wm * MT + mt) * 16 + h * 8 + g4;
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

    float o[MT][8][4], m_run[MT][2], l_run[MT][2];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
      for (int n = 0; n < 8; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[mt][n][i] = 0.f;
      m_run[mt][0] = m_run[mt][1] = -INFINITY;
      l_run[mt][0] = l_run[mt][1] = 0.f;
    }

    const int tend = tiles_end(cons);
    for (int t = tiles_begin(cons) + wk; t < tend; t += WK) {
      const int st = used % ST;
      if (ok) ok = mbar_wait_warp(&full[st], (uint32_t)(used / ST) & 1, args.status, kErrWaitMma, abort_flag);
      const uint32_t kbase = smem_u32(ring + st * S::kStage), vbase = kbase + S::kTile;
      const int key0 = t * KT;
      // ---- S = Q K^T
      float s[MT][NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        uint32_t b[2][4];
        const int row = n * 8 + (lane & 7), c = lane >> 3;
        ldmatrix_x4(kbase + row * 128 + ((c ^ (row & 7)) << 4), b[0]);
        ldmatrix_x4(kbase + row * 128 + (((c + 4) ^ (row & 7)) << 4), b[1]);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
          for (int i = 0; i < 4; ++i) s[mt][n][i] = 0.f;
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            mma_m16n8k16<T>(s[mt][n], qf[mt][kk], b[kk >> 1][(kk & 1) * 2], b[kk >> 1][(kk & 1) * 2 + 1]);
        }
      }
      if (key0 + KT > hi_min || key0 < lo_max) {
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
      // ---- running maximum
      float m_new[MT][2];
      bool need = false;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float m = fmaxf(s[mt][0][2 * h], s[mt][0][2 * h + 1]);
#pragma unroll
          for (int n = 1; n < NT; ++n) m = fmax3(m, s[mt][n][2 * h], s[mt][n][2 * h + 1]);
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
          m *= args.scale_log2;
          const bool up = m > m_run[mt][h] + kRescaleThreshold;
          m_new[mt][h] = up ? m : m_run[mt][h];
          need |= up;
        }
      if (__any_sync(0xffffffffu, need)) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            // -inf only before the first visible key, where sum and weight are zero: 2^-inf = 0 keeps them
            const float alpha = m_new[mt][h] == m_run[mt][h] ? 1.f : ex2_approx(m_run[mt][h] - m_new[mt][h]);
            m_run[mt][h] = m_new[mt][h];
            l_run[mt][h] *= alpha;
#pragma unroll
            for (int n = 0; n < 8; ++n) {
              o[mt][n][2 * h] *= alpha;
              o[mt][n][2 * h + 1] *= alpha;
            }
          }
      }
      // ---- weights, and O += P V
      const bool edge = key0 + KT > it.hi || key0 < it.lo;
      float shift[MT][2];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int h = 0; h < 2; ++h) shift[mt][h] = m_run[mt][h] == -INFINITY ? 0.f : -m_run[mt][h];
#pragma unroll
      for (int ks = 0; ks < KT / 16; ++ks) {
        uint32_t p[MT][4];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float x = ex2_approx(fmaf(s[mt][2 * ks + half][2 * h], args.scale_log2, shift[mt][h]));
              const float y = ex2_approx(fmaf(s[mt][2 * ks + half][2 * h + 1], args.scale_log2, shift[mt][h]));
              l_run[mt][h] += x + y;
              p[mt][half * 2 + h] = OperandType<T>::pack2(x, y);
            }
#pragma unroll
        for (int dp = 0; dp < 4; ++dp) {
          uint32_t b[4];
          const int row = ks * 16 + ((lane >> 3) & 1) * 8 + (lane & 7), c = dp * 2 + (lane >> 4);
          ldmatrix_x4_trans(vbase + row * 128 + ((c ^ (row & 7)) << 4), b);
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
      ++used;
      __syncwarp();
      if (WM > 1) {
        if (lane == 0) mbar_arrive(&empty[st]);
        // a tile late, so that the group's other warps need not have finished this one
        if (wm == 0 && used >= 2 && issued < used - 1 + ST) issue();
      } else {
        issue();
      }
    }
    // ---- a row's weight over its four lanes
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        l_run[mt][h] += __shfl_xor_sync(0xffffffffu, l_run[mt][h], 1);
        l_run[mt][h] += __shfl_xor_sync(0xffffffffu, l_run[mt][h], 2);
      }
    // ---- join the groups: the upper half hands its rows to the lower half until one group is left
    if (WK > 1) {
      float* join = reinterpret_cast<float*>(smem + S::kRing) + (wm * MT * 36) * 32 + lane;
#pragma unroll
      for (int half = WK / 2; half >= 1; half >>= 1) {
        float* at = join + (size_t)(wk & (half - 1)) * WM * MT * 36 * 32;
        if (wk >= half && wk < 2 * half) {
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
            for (int i = 0; i < 32; ++i) at[(mt * 36 + i) * 32] = o[mt][i >> 2][i & 3];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              at[(mt * 36 + 32 + h) * 32] = m_run[mt][h];
              at[(mt * 36 + 34 + h) * 32] = l_run[mt][h];
            }
          }
        }
        __syncthreads();
        if (wk < half) {
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float m2 = at[(mt * 36 + 32 + h) * 32], l2 = at[(mt * 36 + 34 + h) * 32];
              const float m = fmaxf(m_run[mt][h], m2);
              const float f1 = m == -INFINITY ? 1.f : ex2_approx(m_run[mt][h] - m);
              const float f2 = m == -INFINITY ? 1.f : ex2_approx(m2 - m);
              m_run[mt][h] = m;
              l_run[mt][h] = l_run[mt][h] * f1 + l2 * f2;
#pragma unroll
              for (int n = 0; n < 8; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                  o[mt][n][2 * h + e] = o[mt][n][2 * h + e] * f1 + at[(mt * 36 + n * 4 + 2 * h + e) * 32] * f2;
            }
        }
        __syncthreads();
      }
    }
    // ---- results, or this run's part of them
    if (wk == 0) {
      const bool whole = cons.whole();
      float* slot = whole ? nullptr : cache_slot(args, kRows, gridDim.x, 2 * blockIdx.x + cons.slot());
      if (!whole && cons.slot() == 1 && threadIdx.x == 0)
        *cache_record(args, blockIdx.x) = {cons.parts(), it.s.tok + it.tok0, it.ntok, it.head};
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
            const int row = (wm * MT + mt) * 16 + h * 8 + g4;
            float* dst = slot + row * 64 + c2;
#pragma unroll
            for (int n = 0; n < 8; ++n)
              *reinterpret_cast<float2*>(dst + n * 8) = make_float2(o[mt][n][2 * h], o[mt][n][2 * h + 1]);
            if (c2 == 0)
              *reinterpret_cast<float2*>(slot + kRows * 64 + row * 2) = make_float2(m_run[mt][h], l_run[mt][h]);
          }
        }
    }
  }
  // after a wait that gave up, copies may still be in flight: let them land before shared memory is given back
  if (!ok && wm == 0 && lane == 0) {
    const uint64_t t0 = global_ns();
    for (int k = max(0, issued - ST); k < issued; ++k)
      while (!mbar_try_wait(&full[k % ST], (uint32_t)(k / ST) & 1) && global_ns() - t0 < kWaitLimitNs) {
      }
  }
}

// Joins the parts of items that were divided among CTAs. Blocks (c, y) take the item that CTA c began and did not
// end, if there is one; their warps take its rows in turn. A warp reads two parts at a time (16 lanes x 4 dims).
template <typename T>
__global__ void __launch_bounds__(256) cache_join_kernel(const __grid_constant__ CacheAttnArgs args, int tile_rows) {
  const int ctas = gridDim.x;
  const CacheRecord rec = *cache_record(args, blockIdx.x);
  if (rec.parts == 0) return;
  const int lane = threadIdx.x & 31, sub = lane >> 4, d = (lane & 15) * 4;
  for (int row = blockIdx.y * 8 + (threadIdx.x >> 5); row < rec.ntok * args.group; row += gridDim.y * 8) {
    float m = -INFINITY, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int p = sub; p < rec.parts; p += 2) {
      const float* src = cache_slot(args, tile_rows, ctas, 2 * (blockIdx.x + p) + (p == 0 ? 1 : 0));
      const float2 ml = *reinterpret_cast<const float2*>(src + tile_rows * 64 + row * 2);
      const float4 x = *reinterpret_cast<const float4*>(src + row * 64 + d);
      const float mn = fmaxf(m, ml.x);
      const float f1 = mn == -INFINITY ? 1.f : ex2_approx(m - mn), f2 = mn == -INFINITY ? 1.f : ex2_approx(ml.x - mn);
      m = mn;
      l = l * f1 + ml.y * f2;
      o = make_float4(o.x * f1 + x.x * f2, o.y * f1 + x.y * f2, o.z * f1 + x.z * f2, o.w * f1 + x.w * f2);
    }
    const float m2 = __shfl_xor_sync(0xffffffffu, m, 16), l2 = __shfl_xor_sync(0xffffffffu, l, 16);
    const float mn = fmaxf(m, m2);
    const float f1 = mn == -INFINITY ? 1.f : ex2_approx(m - mn), f2 = mn == -INFINITY ? 1.f : ex2_approx(m2 - mn);
    l = l * f1 + l2 * f2;
    o.x = o.x * f1 + __shfl_xor_sync(0xffffffffu, o.x, 16) * f2;
    o.y = o.y * f1 + __shfl_xor_sync(0xffffffffu, o.y, 16) * f2;
    o.z = o.z * f1 + __shfl_xor_sync(0xffffffffu, o.z, 16) * f2;
    o.w = o.w * f1 + __shfl_xor_sync(0xffffffffu, o.w, 16) * f2;
    if (sub == 0) {
      const int i = row / args.group, head = rec.head * args.group + (row - i * args.group);
      const int64_t tok = rec.tok + i;
      const float gate = args.gates ? args.gates[tok * args.hq + head] : 1.f;
      const float f = l == 0.f ? 0.f : gate / l;
      uint2 u;
      u.x = OperandType<T>::pack2(o.x * f, o.y * f);
      u.y = OperandType<T>::pack2(o.z * f, o.w * f);
      *reinterpret_cast<uint2*>(static_cast<T*>(args.out) + tok * args.out_stride + head * 64 + d) = u;
    }
  }
}

}  // namespace trc
