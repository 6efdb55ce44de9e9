// Attention of many new frames over the paged cache on tcgen05: sequences whose push has more than 128 rows per
// cache head (new frames x query heads that share it), where the products and the exponentials bound the work and
// not the reading of K and V.
//
// The pipeline is the time attention's (attention_time.cuh: three 128-row query tiles share 64-key stages, S = Q K^T
// and O += P V in TMEM, one softmax thread per row, registers moved to the softmax warpgroups), with what the cache
// adds:
//   * Work comes in runs (cache_sched.cuh). Warp 0 alone walks the CTA's share of the line; it hands each run to the
//     other warps as a descriptor in shared memory that travels with the run's Q buffer (same barriers), and loads
//     the key stages from the pages, one TMA box per page and stage, page numbers read a stage ahead.
//   * A tile of 128 rows holds 128 / group frames with all query heads of one cache head (row = frame * group +
//     head): one 3-D box of Q. Tiles have key ranges of their own within the run (causal, window): a tile takes
//     part in the stages of its range and only releases the others.
//   * V rows outside the item's keys (behind the sequence's end, before the window) are zeroed in shared memory
//     before the stage is handed on, because the tensor core multiplies them by zero weights and pages hold
//     anything there; scores are replaced per row.
//   * A run that is not a whole item leaves its rows' sums, maxima and weights in the workspace for the join.
#pragma once

#include "attention_time.cuh"
#include "cache_sched.cuh"

namespace trc {

constexpr int kClRows = 128 * kTaTiles;

// What the producer tells the other warps of a run.
struct CacheRun {
  int tok, ntok;    // first row (of all rows) and frames of the item
  int pos0, total;  // frame number of its first frame (negative: see nothing if causal), frames in the cache
  int a0, a1;       // 64-key steps of the run
  int head;         // cache head; -1: no more runs
  int slot;         // workspace slot, -1 for a whole item
};

struct ClSmem {
  static constexpr int kTileQ = TaSmem::kTileQ;
  static constexpr int kTileKV = TaSmem::kTileKV;
  static constexpr int kQ = 0;
  static constexpr int kKV = kQ + 2 * kTaTiles * kTileQ;
  static constexpr int kScale = kKV + 2 * kTaKvStages * kTileKV;
  static constexpr int kRun = kScale + kTaTiles * 128 * 4;  // [2] CacheRun
  static constexpr int kBar = kRun + 64;
  static constexpr int kScan = kBar + 512 + 256;
  static constexpr int bytes(int n_seqs) { return kScan + (n_seqs + 1) * 8 + 1024; }
  static_assert(sizeof(CacheRun) == 32 && kScan + (kCacheMaxSeqs + 1) * 8 + 1024 <= 232448, "shared memory per CTA");
};

template <typename TIn>
__global__ void __launch_bounds__(kTaThreads, 1)
    cache_long_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                      const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CacheAttnArgs args) {
  using S = ClSmem;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::kBar);
  uint64_t* q_full = bars;                  // [2] a run: descriptor and Q
  uint64_t* q_empty = q_full + 2;           // [2]
  uint64_t* kv_full = q_empty + 2;          // [stages]
  uint64_t* kv_empty = kv_full + kTaKvStages;
  uint64_t* s_full = kv_empty + kTaKvStages;  // [3]
  uint64_t* s_free = s_full + kTaTiles;
  uint64_t* p_full = s_free + kTaTiles;
  uint64_t* p_free = p_full + kTaTiles;
  uint64_t* o_free = p_free + kTaTiles;
  uint64_t* raw = o_free + kTaTiles;        // a stage whose V rows are still to be zeroed
  uint64_t* drain = raw + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int64_t* part = reinterpret_cast<int64_t*>(smem + S::kBar + 512);
  int64_t* prefix = reinterpret_cast<int64_t*>(smem + S::kScan);
  CacheRun* runs = reinterpret_cast<CacheRun*>(smem + S::kRun);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int tile_frames = 128 / args.group;

  if (threadIdx.x == 0) {
    for (int b = 0; b < 2; ++b) {
      mbar_init(&q_full[b], 1);
      mbar_init(&q_empty[b], kTaTiles + 4 * kTaTiles);  // issuers and softmax warps
    }
    for (int x = 0; x < kTaTiles; ++x) {
      mbar_init(&s_full[x], 1);
      mbar_init(&s_free[x], 4);
      mbar_init(&p_full[x], 4);
      mbar_init(&p_free[x], 1);
      mbar_init(&o_free[x], 4);
    }
    for (int s = 0; s < kTaKvStages; ++s) {
      mbar_init(&kv_full[s], 1);
      mbar_init(&kv_empty[s], kTaTiles);
    }
    mbar_init(raw, 1);
    mbar_init(drain, kTaTiles);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&map_q);
    tma_prefetch_desc(&map_k);
    tma_prefetch_desc(&map_v);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  const bool split = cache_scan(args, kTaTiles * tile_frames, kTaThreads, gridDim.x, prefix, part);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  // steps [b, e) of tile x within a run; empty for a tile without rows or without visible keys
  auto tile_steps = [&](const CacheRun& run, int x, int& b, int& e) {
    const int i0 = x * tile_frames, i1 = min(i0 + tile_frames, run.ntok);
    b = e = run.a0;
    if (i0 >= i1) return;
    const int hi = args.causal ? min(max(run.pos0 + i1, 0), run.total) : run.total;
    const int lo = min(args.window ? max(run.pos0 + i0 + 1 - args.window, 0) : 0, hi);
    if (lo == hi) return;
    b = max(lo / kCacheStep, run.a0);
    e = max(min((hi + kCacheStep - 1) / kCacheStep, run.a1), b);
  };

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kTaRegsLow) : "memory");
    if (warp == 0) {
      // ------------------------------------------------------------------ producer: runs, Q, key stages
      const int page = 1 << args.page_log2, box = min(page, kCacheStep), boxes = kCacheStep / box;
      int kvc = 0, local = 0, raws = 0;
      bool ok = true;
      CacheWalk w;
      w.begin(args, kTaTiles * tile_frames, prefix, blockIdx.x, gridDim.x, split);
      if (args.split && lane == 0) cache_record(args, blockIdx.x)->parts = 0;
      for (;; ++local) {
        const int qb = local & 1;
        ok = mbar_wait_warp(&q_empty[qb], ((uint32_t)(local >> 1) & 1) ^ 1, args.status, kErrWaitProducer, abort_flag);
        if (!ok) break;
        if (!w.valid) {
          if (lane == 0) {
            runs[qb].head = -1;
            mbar_arrive(&q_full[qb]);
          }
          break;
        }
        const CacheItem& it = w.it;
        if (lane == 0) {
          CacheRun run;
          run.tok = it.s.tok + it.tok0;
          run.ntok = it.ntok;
          run.pos0 = it.s.total - it.s.n + it.tok0;
          run.total = it.s.total;
          run.a0 = w.a0;
          run.a1 = w.a1;
          run.head = it.head;
          run.slot = w.whole() ? -1 : 2 * (int)blockIdx.x + w.slot();
          runs[qb] = run;
          if (!w.whole() && w.slot() == 1)
            *cache_record(args, blockIdx.x) = {w.parts(), run.tok, run.ntok, run.head};
          const int tiles = (it.ntok + tile_frames - 1) / tile_frames;
          mbar_arrive_expect_tx(&q_full[qb], tiles * tile_frames * args.group * 128);
          uint8_t* qbuf = smem + S::kQ + qb * kTaTiles * S::kTileQ;
          for (int x = 0; x < tiles; ++x)
            tma_load_3d(qbuf + x * S::kTileQ, &map_q, &q_full[qb], 0, it.head * args.group, run.tok + x * tile_frames);
        }
        __syncwarp();
        // lane b: page of box b of a step, -1 where no row sees a key of it
        auto page_of = [&](int j) {
          const int key = j * kCacheStep + lane * box;
          if (lane >= boxes || j >= w.a1 || key >= it.hi || key + box <= it.lo) return -1;
          const int p = args.table[(int64_t)it.r * args.table_stride + (key >> args.page_log2)];
          if (p < 0 || p >= args.n_pages) {
            record_error(args.status, kErrBadArgs);
            return -1;
          }
          return p;
        };
        int next = page_of(w.a0);
        for (int j = w.a0; j < w.a1; ++j, ++kvc) {
          const int st = kvc % kTaKvStages;
          const int p = next;
          next = page_of(j + 1);
          ok = mbar_wait_warp(&kv_empty[st], ((uint32_t)(kvc / kTaKvStages) & 1) ^ 1, args.status, kErrWaitProducer,
                              abort_flag);
          if (!ok) break;
          uint8_t* kb = smem + S::kKV + st * 2 * S::kTileKV;
          const int key0 = j * kCacheStep;
          const bool edge = key0 < it.lo || key0 + kCacheStep > it.hi;
          uint64_t* bar = edge ? raw : &kv_full[st];
          if (lane == 0) mbar_arrive_expect_tx(bar, 2 * S::kTileKV);
          __syncwarp();
          if (lane < boxes) {
            // behind the pool: TMA's zero fill
            int64_t y = (int64_t)args.n_pages * args.hkv << args.page_log2;
            if (p >= 0) y = (((int64_t)p * args.hkv + it.head) << args.page_log2) + ((key0 + lane * box) & (page - 1));
            tma_load_2d(kb + lane * box * 128, &map_k, bar, 0, (int)y);
            tma_load_2d(kb + S::kTileKV + lane * box * 128, &map_v, bar, 0, (int)y);
          }
          if (edge) {
            ok = mbar_wait_warp(raw, (uint32_t)raws++ & 1, args.status, kErrWaitProducer, abort_flag);
            if (!ok) break;
            for (int x = lane; x < kCacheStep * 8; x += 32) {  // 16-byte chunks; the swizzle stays within a row
              const int key = key0 + (x >> 3);
              if (key < it.lo || key >= it.hi)
                *reinterpret_cast<uint4*>(kb + S::kTileKV + x * 16) = make_uint4(0, 0, 0, 0);
            }
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&kv_full[st]);
          }
        }
        if (!ok) break;
        w.advance(args, kTaTiles * tile_frames);
      }
      if (!ok && lane == 0) {
        // a wait gave up: let the copies in flight land before shared memory is given back
        const uint64_t t0 = global_ns();
        for (int k = max(0, kvc - kTaKvStages); k < kvc; ++k)
          while (!mbar_try_wait(&kv_full[k % kTaKvStages], (uint32_t)(k / kTaKvStages) & 1) &&
                 global_ns() - t0 < kWaitLimitNs) {
          }
        if (raws)
          while (!mbar_try_wait(raw, (uint32_t)(raws - 1) & 1) && global_ns() - t0 < kWaitLimitNs) {
          }
        for (int k = max(0, local - 1); k <= local; ++k)
          while (!mbar_try_wait(&q_full[k & 1], (uint32_t)(k >> 1) & 1) && global_ns() - t0 < kWaitLimitNs) {
          }
      }
    } else {
      // ------------------------------------------------------------------ MMA issuers, one per query tile
      if (lane == 0) {
        const int x = warp - 1;
        const uint32_t idesc_qk = idesc_f16(128, 64, OperandType<TIn>::kFormat, 0, 0);
        const uint32_t idesc_pv = idesc_f16(128, 64, OperandType<TIn>::kFormat, 0, 1);  // V is MN-major
        const uint32_t tS = tmem_base + ta_col_s(x), tP = tmem_base + ta_col_p(x), tO = tmem_base + ta_col_o(x);
        const uint64_t q_desc0 = sdesc_sw128(smem_u32(smem + S::kQ + x * S::kTileQ), 16, 1024);
        const uint64_t k_desc0 = sdesc_sw128(smem_u32(smem + S::kKV), 16, 1024);
        const uint64_t v_desc0 = sdesc_sw128(smem_u32(smem + S::kKV + S::kTileKV), 8192, 1024);
        constexpr uint32_t kStepKV = (2 * S::kTileKV) >> 4;
        constexpr uint32_t kStepQ = (kTaTiles * S::kTileQ) >> 4;
        int kvc = 0, active = 0;  // kvc: stage count at the run's first step; active: runs worked on (o_free phases)
        uint32_t g = 0;
        bool ok = true;
        auto wait = [&](uint64_t* bar, uint32_t parity) {
          if (ok && !mbar_wait(bar, parity, args.status, kErrWaitMma, abort_flag)) ok = false;
          return ok;
        };
        for (int local = 0; ok; ++local) {
          const int qb = local & 1;
          if (!wait(&q_full[qb], (uint32_t)(local >> 1) & 1)) break;
          const CacheRun run = runs[qb];
          if (run.head < 0) break;
          int b, e;
          tile_steps(run, x, b, e);
          const uint64_t qd = q_desc0 + (uint64_t)(qb * kStepQ);
          auto pass = [&](int j0, int j1) {  // stages of other tiles' keys: released once filled
            for (int j = j0; j < j1 && ok; ++j) {
              const int idx = kvc + j - run.a0;
              if (wait(&kv_full[idx % kTaKvStages], (uint32_t)(idx / kTaKvStages) & 1))
                mbar_arrive(&kv_empty[idx % kTaKvStages]);
            }
          };
          auto issue_s = [&](int j) {
            const int idx = kvc + j - run.a0;
            const int st = idx % kTaKvStages;
            if (!wait(&kv_full[st], (uint32_t)(idx / kTaKvStages) & 1)) return;
            tc_fence_after();
            const uint64_t kd = k_desc0 + (uint64_t)(st * kStepKV);
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) mma_f16_ss(tS, qd + 2 * kk, kd + 2 * kk, idesc_qk, kk > 0 ? 1u : 0u);
            mma_commit(&s_full[x]);
            if (j == e - 1) mma_commit(&q_empty[qb]);
          };
          auto issue_pv = [&](int j) {
            if (!wait(&p_full[x], g & 1u)) return;
            if (j == b && active > 0 && !wait(&o_free[x], (uint32_t)(active - 1) & 1)) return;
            tc_fence_after();
            const int st = (kvc + j - run.a0) % kTaKvStages;
            const uint64_t vd = v_desc0 + (uint64_t)(st * kStepKV);
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              mma_f16_ts(tO, tP + kk * 8, vd + kk * (2048 >> 4), idesc_pv, (j > b || kk > 0) ? 1u : 0u);
            mma_commit(&p_free[x]);
            mma_commit(&kv_empty[st]);
          };
          if (b == e) {
            mbar_arrive(&q_empty[qb]);
            pass(run.a0, run.a1);
          } else {
            pass(run.a0, b);
            if (g > 0 && !wait(&s_free[x], (g - 1) & 1u)) break;
            issue_s(b);
            for (int j = b; j < e && ok; ++j, ++g) {
              if (j + 1 < e && wait(&s_free[x], g & 1u)) issue_s(j + 1);
              issue_pv(j);
            }
            pass(e, run.a1);
            ++active;
          }
          kvc += run.a1 - run.a0;
        }
        mma_commit(drain);
        const uint64_t t0 = global_ns();
        while (!mbar_try_wait(drain, 0) && global_ns() - t0 < kWaitLimitNs) {
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kTaRegsHigh) : "memory");
    // ------------------------------------------------------------------ softmax + epilogue (warps 4-15)
    const int x = (warp - 4) >> 2;
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;
    const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
    const uint32_t tS = tmem_base + lane_off + ta_col_s(x);
    const uint32_t tP = tmem_base + lane_off + ta_col_p(x);
    const uint32_t tO = tmem_base + lane_off + ta_col_o(x);
    float* row_scale = reinterpret_cast<float*>(smem + S::kScale) + x * 128 + r;
    const int frame = r / args.group, sub = r - frame * args.group;  // of this row within its tile
    const int i = x * tile_frames + frame;                          // frame within the item
    uint32_t g = 0;
    // the last run's row, whose epilogue is deferred: where it goes (nothing if null) and whether it is a part
    void* dst = nullptr;
    bool dst_part = false, pending = false;
    auto finish = [&]() {
      const float scale = dst_part ? 1.f : *row_scale;
#pragma unroll 1
      for (int hc = 0; hc < 2; ++hc) {
        float o[32];
        tmem_ld32(tO + hc * 32, o);
        if (hc == 1) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&o_free[x]);
        }
        if (dst) {
          if (dst_part) {
            float4* d = static_cast<float4*>(dst) + hc * 8;
#pragma unroll
            for (int k = 0; k < 8; ++k) d[k] = make_float4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
          } else {
#pragma unroll
            for (int k = 0; k < 32; ++k) o[k] *= scale;
            store32<TIn>(static_cast<TIn*>(dst) + hc * 32, o);
          }
        }
      }
      pending = false;
    };
    bool ok = true;
    for (int local = 0; ok; ++local) {
      const int qb = local & 1;
      if (!(ok = mbar_wait_warp(&q_full[qb], (uint32_t)(local >> 1) & 1, args.status, kErrWaitSoftmax, abort_flag))) break;
      const CacheRun run = runs[qb];
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_empty[qb]);
      if (run.head < 0) break;
      int b, e;
      tile_steps(run, x, b, e);
      const bool live = frame < tile_frames && i < run.ntok;
      const int64_t tok = run.tok + i;
      const int head = run.head * args.group + sub;
      TIn* row_out = static_cast<TIn*>(args.out) + tok * args.out_stride + head * 64;
      float* slot = run.slot < 0 ? nullptr : cache_slot(args, kClRows, gridDim.x, run.slot);
      const int slot_row = i * args.group + sub;  // as the join counts them
      if (b == e) {
        // nothing to add: zeros, or an empty part
        if (live) {
          if (slot) {
            *reinterpret_cast<float2*>(slot + kClRows * 64 + slot_row * 2) = make_float2(-INFINITY, 0.f);
#pragma unroll 1
            for (int k = 0; k < 16; ++k)
              reinterpret_cast<float4*>(slot + slot_row * 64)[k] = make_float4(0.f, 0.f, 0.f, 0.f);
          } else {
#pragma unroll 1
            for (int k = 0; k < 8; ++k) reinterpret_cast<uint4*>(row_out)[k] = make_uint4(0, 0, 0, 0);
          }
        }
        continue;
      }
      const bool warp_live = __any_sync(0xffffffffu, live);
      const float gate = live && args.gates ? args.gates[tok * args.hq + head] : 1.f;
      // rows without a frame take any keys; nothing of them is stored
      const int hi = !live ? INT_MAX : args.causal ? min(max(run.pos0 + i + 1, 0), run.total) : run.total;
      const int lo = live && args.window ? max(run.pos0 + i + 1 - args.window, 0) : 0;
      float m_run = -INFINITY, l_run = 0.f;
      for (int j = b; j < e; ++j, ++g) {
        if (!(ok = mbar_wait_warp(&s_full[x], g & 1u, args.status, kErrWaitSoftmax, abort_flag))) break;
        tc_fence_after();
        if (!warp_live) {
          // no row of this warp exists: its part of P may hold anything, it only reaches its own rows of O. The
          // arrival for this step's P still waits for the previous step's product, or it would count for that step.
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&s_free[x]);
          if (g > 0 &&
              !(ok = mbar_wait_warp(&p_free[x], (g - 1) & 1u, args.status, kErrWaitSoftmax, abort_flag)))
            break;
          tc_fence_after();
          if (j == b && pending) finish();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_full[x]);
          continue;
        }
        float sc[64];
        tmem_ld64(tS, sc);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_free[x]);
        const int kmax = hi - j * 64, kmin = lo - j * 64;
        if (kmax < 64 || kmin > 0) {
#pragma unroll
          for (int k = 0; k < 64; ++k)
            if (k >= kmax || k < kmin) sc[k] = -INFINITY;
        }
        float mx4[4] = {sc[0], sc[1], sc[2], sc[3]};
#pragma unroll
        for (int k = 4; k < 60; k += 8) {
          mx4[0] = fmax3(mx4[0], sc[k], sc[k + 4]);
          mx4[1] = fmax3(mx4[1], sc[k + 1], sc[k + 5]);
          mx4[2] = fmax3(mx4[2], sc[k + 2], sc[k + 6]);
          mx4[3] = fmax3(mx4[3], sc[k + 3], sc[k + 7]);
        }
        const float m_tile =
            fmaxf(fmax3(mx4[0], mx4[1], sc[60]), fmax3(mx4[2], mx4[3], fmax3(sc[61], sc[62], sc[63]))) *
            args.scale_log2;
        bool rescale = false;
        float alpha = 1.0f;
        if (j == b) {
          m_run = m_tile;
        } else {
          // from -inf (no visible key so far): O and the weight are zero, 2^-inf = 0 keeps them
          const bool need = m_tile > m_run + kRescaleThreshold;
          rescale = __any_sync(0xffffffffu, need);
          if (need) {
            alpha = ex2_approx(m_run - m_tile);
            m_run = m_tile;
          }
        }
        const float shift = m_run == -INFINITY ? 0.f : -m_run;
        const float2 scale2 = make_float2(args.scale_log2, args.scale_log2);
        const float2 shift2 = make_float2(shift, shift);
        float2 l2 = make_float2(0.f, 0.f);
        auto exp_chunk = [&](int c, uint32_t(&packed)[16]) {
#pragma unroll
          for (int k = 0; k < 32; k += 2) {
            const int at = c * 32 + k;
            const float2 xv = __ffma2_rn(make_float2(sc[at], sc[at + 1]), scale2, shift2);
            const float2 pv = (k & 7) == 6 ? ex2_poly2(xv) : make_float2(ex2_approx(xv.x), ex2_approx(xv.y));
            l2 = __fadd2_rn(l2, pv);
            packed[k >> 1] = OperandType<TIn>::pack2(pv.x, pv.y);
          }
        };
        {
          uint32_t packed[16];
          exp_chunk(0, packed);
          if (g > 0 &&
              !(ok = mbar_wait_warp(&p_free[x], (g - 1) & 1u, args.status, kErrWaitSoftmax, abort_flag)))
            break;
          tc_fence_after();
          if (rescale) {
#pragma unroll 1
            for (int h = 0; h < 4; ++h) {
              float o[16];
              uint32_t u[16];
              tmem_ld16(tO + h * 16, o);
#pragma unroll
              for (int k = 0; k < 16; ++k) u[k] = __float_as_uint(o[k] * alpha);
              tmem_st16(tO + h * 16, u);
            }
          }
          tmem_st16(tP, packed);
        }
        {
          uint32_t packed[16];
          exp_chunk(1, packed);
          tmem_st16(tP + 16, packed);
        }
        l_run = l_run * alpha + (l2.x + l2.y);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[x]);
        if (j == b && pending) finish();
      }
      if (!ok) break;
      // a row that saw no key: ex2_poly2 makes 2^-126 of a hidden score, so its weight is set to zero here
      if (m_run == -INFINITY) l_run = 0.f;
      *row_scale = l_run == 0.f ? 0.f : gate / l_run;
      dst_part = slot != nullptr;
      dst = !live ? nullptr : slot ? static_cast<void*>(slot + slot_row * 64) : static_cast<void*>(row_out);
      if (slot && live) *reinterpret_cast<float2*>(slot + kClRows * 64 + slot_row * 2) = make_float2(m_run, l_run);
      pending = true;
    }
    if (ok && pending && mbar_wait_warp(&p_free[x], (g - 1) & 1u, args.status, kErrWaitSoftmax, abort_flag)) {
      tc_fence_after();
      finish();
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

}  // namespace trc
