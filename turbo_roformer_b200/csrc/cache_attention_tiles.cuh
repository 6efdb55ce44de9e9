// Attention of many new frames over the paged cache on tcgen05: sequences whose push has more rows per cache head (new
// frames x query heads that share it) than the mma.sync kernel serves best.
//
// As in the time attention (attention_time.cuh) a CTA works on three 128-row query tiles: S = Q K^T (N = 64) and
// O += P V in TMEM, one softmax thread per row, the next S during the exponentials, registers moved to the softmax
// warpgroups. A tile holds 128 / group frames with all query heads of one cache head (row = frame * group + head): one
// 3-D TMA box of Q. K and V come from the pages, one box per page and stage, page numbers read a step ahead.
//   * SHARED: the three tiles are one item's (up to 384 rows of one sequence and cache head) and share its key stages:
//     one channel, one producer. Tiles have key ranges of their own within the run (causal, window): a tile takes part
//     in the steps of its range and only releases the others.
//   * Otherwise each tile is a channel of its own, a worker with its own share of the line, items of one tile and own
//     stages. Pushes of up to 256 rows keep all three tiles busy this way, where the shared form would leave one or two
//     idle (128 rows of 496 heads over 1,700 frames: 75 against 100 us, 256: 126 against 136); longer ones are faster
//     shared, which loads a third of the key bytes (384 rows: 158 against 176 us).
//   * Producers and MMA issuers are warps of their own: issuing a step's products takes 750 cycles of its 2,400 (the
//     tensor pipe is shared by the three). Issuers stay whole warps and elect a lane for the MMAs and commits (5 % over
//     a single lane that runs the whole role). Keys and values have stages of their own, K
//     freed by S, V by P V.
//   * V rows outside the item's keys (behind the sequence's end, before the window) are zeroed in shared memory by the
//     producer before it hands the stage on, because pages hold anything there and 0 x NaN is NaN; scores are replaced
//     per row, behind one vote per step.
//   * A run that is not a whole item leaves its rows' sums, maxima and weights in the workspace for the join.
// Measured: a step of three shared tiles takes 2,400 cycles and of three separate ones 3,300 to 3,600, a run's start
// and end about three steps, a launch 12 us up to its first weights. 1,701 frames x 496 heads: 650 to 680 us under the
// power cap. A step's time is neither the exponentials' nor the products' alone: without any exponential it is a fifth
// less, with a quarter of the products the same. It is the chain from S to P to the next product, of which three tiles
// hide a part (384 rows: issue slots 52 % used, tensor pipe 32 %, MUFU 58 %). The time attention, which does the same
// products and exponentials without pages, masks and a divided line, takes 0.89 of this time (1,701 frames x 232
// heads: 264 and 296 us in turn). Why separate tiles need 40 % more cycles per step than shared ones is not located:
// each run waits for its one Q buffer, and the softmax has 112 registers instead of 144.
// Roles: warps 0-2 MMA issuers of tiles 0-2, warp 3 owns TMEM, producers, softmax + epilogue (CtSmem).
#pragma once

#include "attention_time.cuh"
#include "cache_sched.cuh"

namespace trc {

constexpr int kCtTiles = 3;
constexpr int kCtRuns = 4;  // descriptors: run r's is written once every warp is done with run r - kQBufs - 1's

// A run, as the producer tells the issuers and softmax warps.
struct CacheRun {
  int tok, ntok;    // first row (of all rows) and frames of the item
  int pos0, total;  // frame number of its first frame (negative: sees nothing if causal), frames in the cache
  int a0, a1;       // 64-key steps of the run
  int head;         // cache head; -1: no more runs
  int slot;         // workspace slot, -1 for a whole item
  int lo, hi;       // keys that some row sees
  int seq;          // sequence
  int unused;
};

template <bool SHARED>
struct CtSmem {
  static constexpr int kChannels = SHARED ? 1 : kCtTiles;
  static constexpr int kTilesPer = SHARED ? kCtTiles : 1;  // tiles of a channel
  static constexpr int kQBufs = SHARED ? 2 : 1;
  static constexpr int kStages = SHARED ? 6 : 3;           // of K, and of V, per channel
  static constexpr int kRows = 128 * kTilesPer;            // rows of an item
  static constexpr int kTileQ = 128 * 64 * 2;
  static constexpr int kTileKV = 64 * 64 * 2;
  static constexpr int kQ = 0;                                                          // [bufs][tiles]
  static constexpr int kKV = kQ + kQBufs * kCtTiles * kTileQ;                              // [channels][K, V][stages]
  static constexpr int kScale = kKV + kChannels * 2 * kStages * kTileKV;                // [tiles][128] fp32
  static constexpr int kOut = kScale + kCtTiles * 128 * 4;                              // [softmax warps][8 rows]
  static constexpr int kRun = kOut + 4 * kCtTiles * 1024;                               // [channels][kCtRuns]
  static constexpr int kWalk = kRun + kChannels * kCtRuns * (int)sizeof(CacheRun);      // [channels] CacheWalk
  static constexpr int kBar = kWalk + kChannels * 128;
  static constexpr int kScan = kBar + 768 + 256;
  static constexpr int bytes(int n_seqs) { return kScan + (n_seqs + 1) * 8 + 1024; }
  // Warps 0-2 issue; the producers are warp 3 (shared) or warps 4-6; then twelve softmax warps. Registers per thread
  // after setmaxnreg add up to what the launch gives (checked before it): 512 x 128 = 128 x 80 + 384 x 144, or
  // 640 x 96 = 128 x 72 + 128 x 72 + 384 x 112. The issuers and producers need theirs: with 40 and 56 (128 for the
  // softmax) they spill inside their loops, and 100 rows over 1,700 frames take 7 % longer.
  static constexpr int kProducer0 = SHARED ? 3 : 4;
  static constexpr int kSoftmax0 = SHARED ? 4 : 8;
  static constexpr int kThreads = 32 * (kSoftmax0 + 4 * kCtTiles);
  static constexpr int kRegsIssue = SHARED ? 80 : 72;
  static constexpr int kRegsLoad = 72;
  static constexpr int kRegsSoftmax = SHARED ? 144 : 112;
  static constexpr int kRegs = 128 * (kRegsIssue + (SHARED ? 0 : kRegsLoad) + 3 * kRegsSoftmax);
  static_assert(kBar % 8 == 0 && kScan % 8 == 0, "alignment");
  static_assert(kScan + (kCacheMaxSeqs + 1) * 8 + 1024 <= 232448, "shared memory per CTA");
};

// A warp's rows of O from TMEM to where they go (thread = row, dst null: nowhere), and the accumulator's release. A
// function of its own, because inlined into the softmax loop its registers cost every step a fifth.
template <typename TIn, int ROWS>
__device__ __noinline__ void ct_finish(uint32_t t_o, void* dst, bool is_part, float scale, uint8_t* stage,
                                       uint64_t* o_free) {
  const int lane = threadIdx.x & 31;
  if (is_part) {
    // a part: 4 dims of 32 consecutive rows per store
#pragma unroll 1
    for (int hc = 0; hc < 2; ++hc) {
      float o[32];
      tmem_ld32(t_o + hc * 32, o);
      float4* d = static_cast<float4*>(dst) + hc * 8 * ROWS;
      if (dst) {
#pragma unroll
        for (int k = 0; k < 8; ++k) d[k * ROWS] = make_float4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
      }
    }
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(o_free);
    return;
  }
  // results: eight rows at a time through shared memory, so that a store instruction writes whole 128-byte rows (a
  // thread's own row in 16-byte pieces would touch 32 lines per instruction)
  uint32_t u[32];
#pragma unroll
  for (int hc = 0; hc < 2; ++hc) {
    float o[32];
    tmem_ld32(t_o + hc * 32, o);
#pragma unroll
    for (int k = 0; k < 16; ++k) u[hc * 16 + k] = OperandType<TIn>::pack2(o[2 * k] * scale, o[2 * k + 1] * scale);
  }
  tc_fence_before();
  __syncwarp();
  if (lane == 0) mbar_arrive(o_free);
#pragma unroll 1
  for (int q = 0; q < 4; ++q) {
    if ((lane >> 3) == q) {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        *reinterpret_cast<uint4*>(stage + (lane & 7) * 128 + ((k ^ (lane & 7)) << 4)) =
            make_uint4(u[4 * k], u[4 * k + 1], u[4 * k + 2], u[4 * k + 3]);
    }
    __syncwarp();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r8 = h * 4 + (lane >> 3), k = lane & 7;
      uint4* to = reinterpret_cast<uint4*>(__shfl_sync(0xffffffffu, reinterpret_cast<uint64_t>(dst), q * 8 + r8));
      const uint4 v = *reinterpret_cast<const uint4*>(stage + r8 * 128 + ((k ^ r8) << 4));
      if (to) to[k] = v;
    }
    __syncwarp();
  }
}

template <typename TIn, bool SHARED>
__global__ void __launch_bounds__(CtSmem<SHARED>::kThreads, 1)
    cache_tiles_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                       const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CacheAttnArgs args) {
  using S = CtSmem<SHARED>;
  constexpr int kCh = S::kChannels, kStages = S::kStages, kBufs = S::kQBufs;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::kBar);
  uint64_t* q_full = bars;                   // [channels][bufs] a run: descriptor and Q
  uint64_t* q_empty = q_full + kCh * kBufs;
  uint64_t* k_full = q_empty + kCh * kBufs;  // [channels][stages], and so on
  uint64_t* v_full = k_full + kCh * kStages;
  uint64_t* k_empty = v_full + kCh * kStages;
  uint64_t* v_empty = k_empty + kCh * kStages;
  uint64_t* s_full = v_empty + kCh * kStages;  // [tiles]
  uint64_t* s_free = s_full + kCtTiles;
  uint64_t* p_full = s_free + kCtTiles;
  uint64_t* p_free = p_full + kCtTiles;
  uint64_t* o_free = p_free + kCtTiles;
  uint64_t* drain = o_free + kCtTiles;
  uint64_t* raw = drain + kCtTiles;            // [channels] values that are still to be zeroed in part
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(raw + kCh);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int64_t* part = reinterpret_cast<int64_t*>(smem + S::kBar + 768);
  int64_t* prefix = reinterpret_cast<int64_t*>(smem + S::kScan);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int tile_frames = 128 / args.group;  // frames of a tile
  const int tpt = S::kTilesPer * tile_frames, workers = gridDim.x * kCh;

  if (threadIdx.x == 0) {
    for (int c = 0; c < kCh * kBufs; ++c) {
      mbar_init(&q_full[c], 1);
      if (c < kCh) mbar_init(&raw[c], 1);
      mbar_init(&q_empty[c], 5 * S::kTilesPer);  // a tile's issuer, and its softmax warps once they have the run
    }
    for (int s = 0; s < kCh * kStages; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&v_full[s], 1);
      mbar_init(&k_empty[s], S::kTilesPer);
      mbar_init(&v_empty[s], S::kTilesPer);
    }
    for (int x = 0; x < kCtTiles; ++x) {
      mbar_init(&s_full[x], 1);
      mbar_init(&s_free[x], 4);
      mbar_init(&p_full[x], 4);
      mbar_init(&p_free[x], 1);
      mbar_init(&o_free[x], 4);
      mbar_init(&drain[x], 1);
    }
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&map_q);
    tma_prefetch_desc(&map_k);
    tma_prefetch_desc(&map_v);
  }
  cache_prefetch(args);
  if (warp == 3) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  grid_wait();
  grid_release();
  const bool split = cache_scan(args, tpt, S::kThreads, workers, prefix, part);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  // steps [b, e) of tile x within a run: the run's, or in a shared one those in which a row of the tile sees a key
  auto tile_steps = [&](const CacheRun& run, int x, int& b, int& e) {
    b = run.a0;
    e = run.a1;
    if (!SHARED) return;
    const int i0 = x * tile_frames, i1 = min(i0 + tile_frames, run.ntok);
    const int hi = args.causal ? min(max(run.pos0 + i1, 0), run.total) : run.total;
    const int lo = min(args.window ? max(run.pos0 + i0 + 1 - args.window, 0) : 0, hi);
    b = min(max(lo / kCacheStep, run.a0), run.a1);  // its range may begin behind the run
    e = i0 >= i1 || lo == hi ? b : max(min((hi + kCacheStep - 1) / kCacheStep, run.a1), b);
  };

  if (warp < S::kSoftmax0) {
    if (warp < 4)
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(S::kRegsIssue) : "memory");
    else
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(S::kRegsLoad) : "memory");
    if (warp < kCtTiles) {
      // ------------------------------------------------------------------ MMA issuer of tile x
      const int x = warp, c = SHARED ? 0 : x;
      const CacheRun* runs = reinterpret_cast<const CacheRun*>(smem + S::kRun) + c * kCtRuns;
      const uint32_t k_ring = smem_u32(smem + S::kKV + c * 2 * kStages * S::kTileKV);
      uint64_t* kf = k_full + c * kStages;
      uint64_t* vf = v_full + c * kStages;
      uint64_t* ke = k_empty + c * kStages;
      uint64_t* ve = v_empty + c * kStages;
      const uint32_t idesc_qk = idesc_f16(128, 64, OperandType<TIn>::kFormat, 0, 0);
      const uint32_t idesc_pv = idesc_f16(128, 64, OperandType<TIn>::kFormat, 0, 1);  // V is MN-major
      const uint32_t tS = tmem_base + ta_col_s(x), tP = tmem_base + ta_col_p(x), tO = tmem_base + ta_col_o(x);
      const uint64_t q_desc0 = sdesc_sw128(smem_u32(smem + S::kQ + x * S::kTileQ), 16, 1024);
      const uint64_t k_desc = sdesc_sw128(k_ring, 16, 1024);
      const uint64_t v_desc = sdesc_sw128(k_ring + kStages * S::kTileKV, 8192, 1024);
      uint32_t n = 0;            // the tile's steps so far
      uint32_t active = 0;       // its runs of at least one step
      int ks = 0, vs = 0;        // stages of the next S and P V
      uint32_t kp = 0, vp = 0;   // and their phases
      bool ok = true;
      auto wait = [&](uint64_t* bar, uint32_t parity) {
        if (ok && !mbar_wait_warp(bar, parity, args.status, kErrWaitMma, abort_flag)) ok = false;
        return ok;
      };
      auto next_stage = [&](int& st, uint32_t& phase) {
        if (++st == kStages) {
          st = 0;
          phase ^= 1;
        }
      };
      auto pass = [&](int steps) {  // steps of other tiles' keys: released once filled
        for (; steps > 0 && ok; --steps) {
          if (!wait(&kf[ks], kp)) return;
          if (lane == 0) mbar_arrive(&ke[ks]);
          next_stage(ks, kp);
          if (!wait(&vf[vs], vp)) return;
          if (lane == 0) mbar_arrive(&ve[vs]);
          next_stage(vs, vp);
        }
      };
      int qb = 0;                // the run's Q buffer
      auto issue_s = [&](bool last) {
        if (!wait(&kf[ks], kp)) return;
        tc_fence_after();
        const uint64_t qd = q_desc0 + (uint64_t)(qb * (kCtTiles * S::kTileQ >> 4));
        const uint64_t kd = k_desc + (uint64_t)(ks * (S::kTileKV >> 4));
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) mma_f16_ss(tS, qd + 2 * kk, kd + 2 * kk, idesc_qk, kk > 0 ? 1u : 0u);
          mma_commit(&s_full[x]);
          mma_commit(&ke[ks]);
          if (last) mma_commit(&q_empty[c * kBufs + qb]);
        }
        __syncwarp();
        next_stage(ks, kp);
      };
      for (int r = 0; ok; ++r) {
        qb = r % kBufs;
        if (!wait(&q_full[c * kBufs + qb], (uint32_t)(r / kBufs) & 1)) break;
        const CacheRun& run = runs[r % kCtRuns];
        if (run.head < 0) break;
        int b, e;
        tile_steps(run, x, b, e);
        const int after = run.a1 - e;
        if (SHARED) {
          pass(b - run.a0);
          if (b == e && lane == 0) mbar_arrive(&q_empty[c * kBufs + qb]);
        }
        if (b < e) {
          issue_s(e - b == 1);  // the softmax warps have taken S(n - 1): waited for below
          for (int j = b; j < e && ok; ++j, ++n) {
            if (!wait(&s_free[x], n & 1u)) break;
            if (j + 1 < e) issue_s(j + 2 == e);
            if (!wait(&vf[vs], vp) || !wait(&p_full[x], n & 1u)) break;
            if (j == b && active > 0 && !wait(&o_free[x], (active - 1) & 1)) break;
            tc_fence_after();
            const uint64_t vd = v_desc + (uint64_t)(vs * (S::kTileKV >> 4));
            if (elect_one()) {
#pragma unroll
              for (int kk = 0; kk < 4; ++kk)
                mma_f16_ts(tO, tP + kk * 8, vd + kk * (2048 >> 4), idesc_pv, (j > b || kk > 0) ? 1u : 0u);
              mma_commit(&p_free[x]);
              mma_commit(&ve[vs]);
            }
            __syncwarp();
            next_stage(vs, vp);
          }
          ++active;
        }
        if (SHARED) pass(after);
      }
      __syncwarp();
      if (elect_one()) mma_commit(&drain[x]);
      __syncwarp();
      const uint64_t t0 = global_ns();
      while (!mbar_try_wait(&drain[x], 0) && global_ns() - t0 < kWaitLimitNs) {
      }
    }
    if (warp >= S::kProducer0 && warp < S::kProducer0 + kCh) {
      // ------------------------------------------------------------------ producer of channel c: runs, Q, K, V
      const int c = warp - S::kProducer0, worker = blockIdx.x * kCh + c;
      CacheRun* runs = reinterpret_cast<CacheRun*>(smem + S::kRun) + c * kCtRuns;
      uint8_t* k_ring = smem + S::kKV + c * 2 * kStages * S::kTileKV;
      uint8_t* v_ring = k_ring + kStages * S::kTileKV;
      const int page = 1 << args.page_log2, box = min(page, kCacheStep), boxes = kCacheStep / box;
      const int nowhere = (args.n_pages * args.hkv) << args.page_log2;  // behind the pool: TMA's zero fill
      // the walk lives in shared memory, lane 0's: it takes more registers than the loads have to spare
      CacheWalk& w = *reinterpret_cast<CacheWalk*>(smem + S::kWalk + c * 128);
      static_assert(sizeof(CacheWalk) <= 128, "layout");
      if (lane == 0) {
        CacheWalk first;
        first.begin(args, tpt, prefix, worker, workers, split);
        w = first;
        if (args.split) cache_record(args, worker)->parts = 0;
      }
      bool ok = true;
      int k_count = 0, v_count = 0, r = 0;
      auto wait = [&](uint64_t* bar, uint32_t parity) {
        if (ok) ok = mbar_wait_warp(bar, parity, args.status, kErrWaitProducer, abort_flag);
        return ok;
      };
      auto request = [&](const CUtensorMap& map, uint8_t* dst, uint64_t* bar, int y) {
        if (lane == 0) mbar_arrive_expect_tx(bar, S::kTileKV);
        __syncwarp();
        if (lane < boxes) tma_load_2d(dst + lane * box * 128, &map, bar, 0, y);
      };
      auto request_k = [&](int y) {
        const int st = k_count % kStages;
        if (!wait(&k_empty[c * kStages + st], ((uint32_t)(k_count / kStages) & 1) ^ 1)) return;
        request(map_k, k_ring + st * S::kTileKV, &k_full[c * kStages + st], y);
        ++k_count;
      };
      int raws = 0;
      // the values of step j, whose item sees keys [lo, hi)
      auto request_v = [&](int y, int j, int lo, int hi) {
        const int st = v_count % kStages, key0 = j * kCacheStep;
        uint64_t* full = &v_full[c * kStages + st];
        uint8_t* dst = v_ring + st * S::kTileKV;
        if (!wait(&v_empty[c * kStages + st], ((uint32_t)(v_count / kStages) & 1) ^ 1)) return;
        if (key0 >= lo && key0 + kCacheStep <= hi) {
          request(map_v, dst, full, y);
        } else {
          // rows that no row of the item may see: zero (the other stages cover the time this takes)
          request(map_v, dst, &raw[c], y);
          if (!wait(&raw[c], (uint32_t)raws++ & 1)) return;
          // 16-byte chunks; the swizzle stays within a row
          for (int k = lane; k < (lo - key0) * 8; k += 32)
            *reinterpret_cast<uint4*>(dst + k * 16) = make_uint4(0, 0, 0, 0);
          for (int k = max(hi - key0, 0) * 8 + lane; k < kCacheStep * 8; k += 32)
            *reinterpret_cast<uint4*>(dst + k * 16) = make_uint4(0, 0, 0, 0);
          fence_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(full);
        }
        ++v_count;
      };
      int v_y = -1;  // pool row (lane b: of box b) of the step whose values are requested next
      for (;; ++r) {
        const int qb = c * kBufs + r % kBufs;
        CacheRun& run = runs[r % kCtRuns];
        if (lane == 0) {
          run.head = -1;
          if (w.valid) {
            run.tok = w.it.s.tok + w.it.tok0;
            run.ntok = w.it.ntok;
            run.pos0 = w.it.s.total - w.it.s.n + w.it.tok0;
            run.total = w.it.s.total;
            run.a0 = w.a0;
            run.a1 = w.a1;
            run.head = w.it.head;
            run.slot = w.whole() ? -1 : 2 * worker + w.slot();
            run.lo = w.it.lo;
            run.hi = w.it.hi;
            run.seq = w.it.r;
            if (run.slot >= 0 && w.slot() == 1)
              *cache_record(args, worker) = {w.parts(args), run.tok, run.ntok, run.head};
            // one buffer: Q is asked for only once its predecessor is done with; until then it comes as far as L2
            if (kBufs == 1) tma_prefetch_3d(&map_q, 0, run.head * args.group, run.tok);
          }
        }
        __syncwarp();
        if (r >= kBufs && !wait(&q_empty[qb], (uint32_t)(r / kBufs - 1) & 1)) break;
        if (lane == 0) {
          if (run.head < 0) {
            mbar_arrive(&q_full[qb]);
          } else {
            const int tiles = SHARED ? (run.ntok + tile_frames - 1) / tile_frames : 1;
            mbar_arrive_expect_tx(&q_full[qb], tiles * tile_frames * args.group * 128);
            for (int x = 0; x < tiles; ++x)
              tma_load_3d(smem + S::kQ + (r % kBufs * kCtTiles + (SHARED ? x : c)) * S::kTileQ, &map_q, &q_full[qb], 0,
                          run.head * args.group, run.tok + x * tile_frames);
          }
        }
        __syncwarp();
        const int hi = run.hi, lo = run.lo, head = run.head, a0 = run.a0, a1 = run.a1;
        if (head < 0) break;
        const int32_t* table = args.table + (int64_t)run.seq * args.table_stride;
        auto look_up = [&](int j) {  // lane b: page of box b; -1: no row sees a key of it
          const int key = j * kCacheStep + lane * box;
          return lane < boxes && j < a1 && key < hi && key + box > lo ? table[key >> args.page_log2] : -1;
        };
        int p = look_up(a0);
        for (int j = a0; j < a1 && ok; ++j) {
          const int next = look_up(j + 1);  // a step ahead of its use
          const int key = j * kCacheStep + lane * box;
          int y = nowhere;
          if (p >= 0 && p < args.n_pages)
            y = ((p * args.hkv + head) << args.page_log2) + (key & (page - 1));
          else if (lane < boxes && key < hi && key + box > lo)
            record_error(args.status, kErrBadArgs);
          p = next;
          request_k(y);
          if (j > a0) request_v(v_y, j - 1, lo, hi);  // a step behind the keys: their stage falls free later
          v_y = y;
        }
        // the run's last values before its successor's Q, which waits for this run's last S
        request_v(v_y, a1 - 1, lo, hi);
        if (!ok) {
          ++r;
          break;
        }
        if (lane == 0) {
          CacheWalk next = w;
          next.advance(args, tpt);
          w = next;
        }
      }
      if (!ok && lane == 0) {
        // a wait gave up: let the copies in flight land before shared memory is given back
        const uint64_t t0 = global_ns();
        auto land = [&](uint64_t* b, int count) {
          for (int k = max(0, count - kStages); k < count; ++k)
            while (!mbar_try_wait(&b[k % kStages], (uint32_t)(k / kStages) & 1) && global_ns() - t0 < kWaitLimitNs) {
            }
        };
        land(k_full + c * kStages, k_count);
        land(v_full + c * kStages, v_count);
        if (raws)
          while (!mbar_try_wait(&raw[c], (uint32_t)(raws - 1) & 1) && global_ns() - t0 < kWaitLimitNs) {
          }
        for (int k = max(0, r - kBufs); k < r; ++k)
          while (!mbar_try_wait(&q_full[c * kBufs + k % kBufs], (uint32_t)(k / kBufs) & 1) &&
                 global_ns() - t0 < kWaitLimitNs) {
          }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(S::kRegsSoftmax) : "memory");
    // ------------------------------------------------------------------ softmax + epilogue
    const int x = (warp - S::kSoftmax0) >> 2, c = SHARED ? 0 : x;
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
    const uint32_t tS = tmem_base + lane_off + ta_col_s(x);
    const uint32_t tP = tmem_base + lane_off + ta_col_p(x);
    const uint32_t tO = tmem_base + lane_off + ta_col_o(x);
    const CacheRun* runs = reinterpret_cast<const CacheRun*>(smem + S::kRun) + c * kCtRuns;
    float* row_scale = reinterpret_cast<float*>(smem + S::kScale) + x * 128 + row;
    const int frame = row / args.group, sub = row - frame * args.group;  // frame of the tile, query head of the group
    const int i = (SHARED ? x * tile_frames : 0) + frame;                // frame of the item
    uint32_t g = 0;                                                      // the tile's steps so far
    // the last run's row, whose epilogue is deferred: where it goes (nowhere if null), and whether it is a part
    void* dst = nullptr;
    bool dst_part = false, pending = false;
    uint8_t* out_stage = smem + S::kOut + (warp - S::kSoftmax0) * 1024;
    auto finish = [&]() {
      ct_finish<TIn, S::kRows>(tO, dst, dst_part, *row_scale, out_stage, &o_free[x]);
      pending = false;
    };
    bool ok = true;
    for (int r = 0; ok; ++r) {
      const int qb = c * kBufs + r % kBufs;
      if (!(ok = mbar_wait_warp(&q_full[qb], (uint32_t)(r / kBufs) & 1, args.status, kErrWaitSoftmax, abort_flag)))
        break;
      const CacheRun run = runs[r % kCtRuns];
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_empty[qb]);
      if (run.head < 0) break;
      const bool live = frame < tile_frames && i < run.ntok;
      const int64_t tok = run.tok + i;
      const int head = run.head * args.group + sub;
      const int slot_row = i * args.group + sub;  // as the join counts them
      int b, e;
      tile_steps(run, x, b, e);
      if (SHARED && b == e) {
        // nothing to add: zeros, or an empty part
        if (live) {
          if (run.slot >= 0) {
            float* slot = cache_slot(args, S::kRows, workers, run.slot);
            *reinterpret_cast<float2*>(slot + S::kRows * 64 + slot_row * 2) = make_float2(-INFINITY, 0.f);
#pragma unroll 1
            for (int k = 0; k < 16; ++k)
              reinterpret_cast<float4*>(slot)[k * S::kRows + slot_row] = make_float4(0.f, 0.f, 0.f, 0.f);
          } else {
            TIn* to = static_cast<TIn*>(args.out) + tok * args.out_stride + head * 64;
#pragma unroll 1
            for (int k = 0; k < 8; ++k) reinterpret_cast<uint4*>(to)[k] = make_uint4(0, 0, 0, 0);
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
        if (__any_sync(0xffffffffu, j * 64 + 64 > hi || j * 64 < lo)) {  // some row does not see all keys
          const int kmax = hi - j * 64, kmin = lo - j * 64;
#pragma unroll
          for (int k = 0; k < 64; ++k)
            if (k >= kmax || k < kmin) sc[k] = -INFINITY;
        }
        // A visible score of NaN or +inf makes the row NaN, through its maximum: the polynomial would lose a NaN.
        float mx4[4] = {sc[0], sc[1], sc[2], sc[3]};
#pragma unroll
        for (int k = 4; k < 60; k += 8) {
          mx4[0] = fmax3_nan(mx4[0], sc[k], sc[k + 4]);
          mx4[1] = fmax3_nan(mx4[1], sc[k + 1], sc[k + 5]);
          mx4[2] = fmax3_nan(mx4[2], sc[k + 2], sc[k + 6]);
          mx4[3] = fmax3_nan(mx4[3], sc[k + 3], sc[k + 7]);
        }
        const float m_tile = fmax3_nan(fmax3_nan(mx4[0], mx4[1], sc[60]), fmax3_nan(mx4[2], mx4[3], sc[61]),
                                       fmax3_nan(sc[62], sc[63], sc[63])) *
                             args.scale_log2;
        bool rescale = false;
        float alpha = 1.0f;
        if (j == b) {
          m_run = m_tile < INFINITY ? m_tile : NAN;
        } else {
          // from -inf (no visible key so far): O and the weight are zero, 2^-inf = 0 keeps them
          const bool need = live && !(m_tile <= m_run + kRescaleThreshold);
          rescale = __any_sync(0xffffffffu, need);
          if (need) {
            const float m_next = m_tile < INFINITY ? m_tile : NAN;
            alpha = ex2_approx(m_run - m_next);
            m_run = m_next;
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
            // one pair in eight on the FMA pipe; one in four is 1.5 % slower, the polynomial being more instructions
            const float2 pv = (k & 15) == 14 ? ex2_poly2(xv) : make_float2(ex2_approx(xv.x), ex2_approx(xv.y));
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
      // a row that saw no key: ex2_poly2 makes 2^-134.6 of a hidden score, so its weight is set to zero here
      if (m_run == -INFINITY) l_run = 0.f;
      *row_scale = l_run == 0.f ? 0.f : gate / l_run;
      dst_part = run.slot >= 0;
      dst = nullptr;
      if (live) {
        if (dst_part) {
          float* slot = cache_slot(args, S::kRows, workers, run.slot);
          *reinterpret_cast<float2*>(slot + S::kRows * 64 + slot_row * 2) = make_float2(m_run, l_run);
          dst = slot + slot_row * 4;
        } else {
          dst = static_cast<TIn*>(args.out) + tok * args.out_stride + head * 64;
        }
      }
      pending = true;
    }
    if (ok && pending && mbar_wait_warp(&p_free[x], (g - 1) & 1u, args.status, kErrWaitSoftmax, abort_flag)) {
      tc_fence_after();
      finish();
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 3) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

}  // namespace trc
