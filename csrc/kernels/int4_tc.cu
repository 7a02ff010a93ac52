// Products with 4-bit weights (int4.cuh) on tcgen05: y[r, f] = sum over groups j of scale[f, j] * ( sum_{k in j} x[r, k] (code[f, k] - zero[f, j]) ).
//
// Weights are the M side (128 rows of a tile), NT rows of x the N side. A CTA walks tiles, or with few of them owns a piece of the K of one (the CTAs of
// a cluster share the tile). Roles, one pipeline:
//   producer    one bulk copy per step (codes, scales and zeros of 128 rows x 128 of K are one run) and TMA tiles of x into a ring of shared-memory
//               stages
//   gatherers   two warps that copy the rows of x which src_row names, 16 bytes a lane (tile::gather4 takes 55 to 80 cycles for four rows of 128 bytes:
//               it bounded experts at 250 us where these take 160)
//   converters  a thread owns a row: eight codes of a word become four bf16 pairs code - zero (exact), 64 of K a slot, written to tensor
//               memory as the A operand
//   MMA         one thread; every group of K has an accumulator of its own (a ring of them)
//   epilogue    takes a group's accumulator out of tensor memory, multiplies it by the row's scale and adds it to its registers, fp32
// So no rounding happens before the result, whatever the scales are. (Scaled weights rounded to bf16 would need neither the ring nor the second sum,
// but double the error of a product, and more for a gate / up pair.)
// What bounds it. A step (128 weight rows x 128 of K) takes, at 1.9 GHz:
//   128 rows of x       about 1030 cycles of the SM's one CTA, 512 of them MMAs. No unit is full: the tensor pipe is active 54 % of the time, 64 % of the issue
//                       slots are used, and 11.2 TB/s of operands leave L2 (41 KB a step: x comes again for each 128 features), 42 % of what it can hand over.
//                       With the conversion, the drains and seven of eight MMAs left out, but all the loads, a step still took 870.
//   32 rows, gathered   about 1560 cycles of a CTA, two of which share the SM: 780 a step. The two warps that copy the rows bound it.
//   16 rows, two tiles  about 2800 cycles of a CTA for two tiles, two CTAs to an SM: 700 a tile's step; the weights' share of HBM is 365 to 390.
// So with up to 64 rows two CTAs share an SM, with 16 rows two tiles of weights a step, handovers are whole steps, and tests of barriers are issued before
// their answers are needed. Measured: 1000 rows of gate / up 37888 x 3584 244 us (1.1 PFLOP/s), 4096 rows over 8 experts of 4096 x 14336 468 us (1.0
// PFLOP/s); called for seconds on end, when the power cap holds the clock at 1.55 to 1.6 GHz, 290 and 556 us (0.94 and 0.86). 13 rows of 152064 x 3584 84 us
// (3.6 TB/s), 128 rows over 8 experts of 28672 x 4096, gathered, 160 us (3.0 TB/s).
// Pieces of a tile meet in distributed shared memory in rank order: the result does not depend on timing, and no memory outlives the call.
#include "int4.cuh"
#include "launch.cuh"
#include <cooperative_groups.h>
#include <cuda.h>

namespace skein {

int make_tmap_2d(CUtensorMap* out, const void* base, uint64_t rows, uint64_t k_elems, uint64_t ld, int elem_bytes, uint32_t box_rows);   // gemm_ws.cu

constexpr int IT_MAX_STAGES = 8;
constexpr int IT_SCALES = 8;             // steps of the ring of scales
constexpr int IT_BAND = 12;              // feature tiles of a band in which the row tiles run (L2 keeps a band's weights)

struct Int4Tc {
  const __nv_bfloat16* x;
  const int* src_row;
  const uint8_t* w;
  const void* residual;
  void* out;
  const int *counts, *offsets;
  int* status;
  long long x_ld, out_ld;
  int rows, x_rows, E, F, K, strips, steps, w_tiles, m_tiles, split, least, stages, flags;   // split: CTAs of a cluster, least: steps of a piece; flags: 1 pair, 2 fp16 scales, 4 fp32 output, 8 zeros
  uint64_t budget_ns;
};

// 16 bytes of a gathered row; bytes = 0: zeros
__device__ __forceinline__ void it_copy16(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
// The barrier hears of this thread's copies when they are complete: one arrival of its count.
__device__ __forceinline__ void it_copy_arrive(uint32_t bar) { asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void it_copy_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// Bounded wait of a thread.
__device__ __forceinline__ bool it_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, uint64_t budget_ns) {
  uint64_t t0 = 0;
#pragma unroll 1
  for (uint32_t n = 1;; ++n) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((n & 255) == 0) {
      if (t0 == 0) t0 = global_timer_ns();
      if (*abort_flag || global_timer_ns() - t0 > budget_ns) return false;
    }
  }
}
// The same of a warp, with the same answer for every lane, so that a warp leaves a role together. seen: the lane knows already (it_peek).
__device__ __forceinline__ bool it_warp_wait(uint32_t seen, uint32_t bar, uint32_t parity, volatile int* abort_flag, uint64_t budget_ns) {
  if (!seen) seen = it_wait(bar, parity, abort_flag, budget_ns);
  return __all_sync(0xffffffffu, seen);
}
// Looks at a phase without waiting, well before the answer is needed: a wait on a phase that is long complete takes a hundred cycles and more. Only for
// a phase whose predecessor on that barrier the asking role has seen complete.
__device__ __forceinline__ uint32_t it_peek(uint32_t bar, uint32_t parity) { return mbar_test_wait(bar, parity) ? 1u : 0u; }

// a += b * s on two neighbours at a time
__device__ __forceinline__ void it_fma2(uint64_t& a, uint32_t b0, uint32_t b1, uint64_t s) {
  asm("{\n\t.reg .b64 b;\n\tmov.b64 b, {%1, %2};\n\tfma.rn.f32x2 %0, b, %3, %0;\n\t}" : "+l"(a) : "r"(b0), "r"(b1), "l"(s));
}
__device__ __forceinline__ uint64_t it_pack(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 it_unpack(uint64_t a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a));
  return r;
}

// Shape of a launch. SUB: tiles of 128 weight rows that a CTA takes at a time.
template <int NT, int SUB>
struct ItShape {
  static constexpr bool ONE = NT == 128;                   // one CTA per SM, 512 columns; else two with 256 each
  static constexpr int CONV_WARPS = NT == 64 ? 4 : 8, EPI_WARPS = NT >= 64 ? 8 : 4;
  static constexpr int GROUPS = CONV_WARPS / 4 / SUB;      // of converters that take the steps in turn
  static constexpr int THREADS = 32 * (4 + CONV_WARPS + EPI_WARPS);       // warp 0 produces, 1 issues, 2 and 3 gather
  static constexpr int ACC = NT;                           // columns of an accumulator
  static constexpr int BUFS = NT == 16 ? 4 : ONE ? 3 : 2;
  static constexpr int SLOTS = SUB == 2 ? 1 : NT <= 32 ? 3 : 2;           // of a converted step, 64 columns for each tile
  static constexpr int COLS = ONE ? 512 : 256;
  static constexpr int EPI_COLS = NT / (EPI_WARPS / 4);    // columns that an epilogue warp takes, of every tile
  // Scales of the steps that are converted and not drained: a converter that writes those of step s + IT_SCALES has seen the MMAs of step s + IT_SCALES
  // - SLOTS done, which began after the epilogue had freed the accumulators of step s + IT_SCALES - SLOTS - BUFS, and had read their scales before
  static_assert(SLOTS + BUFS < IT_SCALES, "the ring of scales");
  static_assert(SUB * (BUFS * ACC + SLOTS * 64) <= COLS && GROUPS * 4 * SUB == CONV_WARPS, "tensor memory");
};

// What a CTA does: `items` tiles, the last of them `last` with steps s0 .. s1 of it (of the others all) and `share` CTAs of a cluster on it
struct ItPlan { int items, last, s0, s1, share, mine, n_steps; };

template <int NT, int GP, int SUB>
__global__ void __launch_bounds__(ItShape<NT, SUB>::THREADS, ItShape<NT, SUB>::ONE ? 1 : 2) int4_tc_kernel(const __grid_constant__ CUtensorMap tmX, const Int4Tc p) {
  namespace cg = cooperative_groups;
  using S = ItShape<NT, SUB>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bar_full[IT_MAX_STAGES], bar_empty[IT_MAX_STAGES], bar_cfull[S::SLOTS], bar_cempty[S::SLOTS], bar_dfull[S::BUFS], bar_dempty[S::BUFS];
  __shared__ uint32_t tmem_base_smem;
  __shared__ int abort_flag;
  __shared__ ItPlan plan;
  __shared__ float scales[IT_SCALES][GP][SUB * 128];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const bool zeros = p.flags & 8;
  const int rec = i4_record(GP, zeros);
  constexpr int X_BYTES = NT * 256;
  const int w_bytes = (rec + 1023) & ~1023, stage_bytes = X_BYTES + SUB * w_bytes;

  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int s = 0; s < p.stages; ++s) { mbar_init(smem_u32(&bar_full[s]), p.src_row != nullptr ? 65 : 1); mbar_init(smem_u32(&bar_empty[s]), 1); }
    for (int s = 0; s < S::SLOTS; ++s) { mbar_init(smem_u32(&bar_cfull[s]), 4 * SUB); mbar_init(smem_u32(&bar_cempty[s]), 1); }
    for (int b = 0; b < S::BUFS; ++b) { mbar_init(smem_u32(&bar_dfull[b]), 1); mbar_init(smem_u32(&bar_dempty[b]), S::EPI_WARPS); }
    fence_mbar_init();
  }
  if (warp == 1) { tmem_alloc(smem_u32(&tmem_base_smem), S::COLS); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = tmem_base_smem;
  pdl_trigger();
  pdl_wait();

  // ---- the tiles: experts in order, in each bands of feature tiles, in a band the feature tile runs fastest. pre: tiles before an expert
  int* pre = reinterpret_cast<int*>(smem_raw + (smem_base - smem_u32(smem_raw)) + p.stages * stage_bytes);
  int *cnt = pre + p.E + 1, *off = cnt + p.E;
  if (warp == 0) {
    int run = 0;
    for (int e0 = 0; e0 < p.E; e0 += 32) {
      int c = 0, o = 0;
      if (e0 + lane < p.E) {
        c = p.rows;
        if (p.counts != nullptr) {
          c = p.counts[e0 + lane];
          o = p.offsets[e0 + lane];
          if (o < 0 || c < 0 || c > p.rows - o) {
            if (c != 0) report_status(p.status, ST_BAD_INDEX, e0 + lane);
            c = 0;
          }
        }
      }
      const int mine = p.m_tiles * ((c + NT - 1) / NT);
      int inc = mine;
      for (int d = 1; d < 32; d <<= 1) { const int v = __shfl_up_sync(0xffffffffu, inc, d); if (lane >= d) inc += v; }
      if (e0 + lane < p.E) { pre[e0 + lane] = run + inc - mine; cnt[e0 + lane] = c; off[e0 + lane] = o; }
      run += __shfl_sync(0xffffffffu, inc, 31);
    }
    if (lane == 0) pre[p.E] = run;
    // (tiles that share their K have a place each; more of them are rows that belong to several experts)
    if (SUB == 1 && p.split > 1 && lane == 0 && run > (int)gridDim.x / p.split) report_status(p.status, ST_BAD_INDEX, p.E);
    // A CTA walks whole tiles, every role at its own pace: the next tile's steps begin while the last one's results are stored. With two tiles a step
    // what does not fill a round is shared: `share` CTAs of a cluster take a piece of K each.
    if (SUB == 2 && lane == 0) {
      const int grid = (int)gridDim.x, me = (int)blockIdx.x, rounds = run / grid, left = run - rounds * grid;
      int share = 1;
      while (share < p.split && left * share * 2 <= grid && p.steps >= p.least * share * 2) share *= 2;
      const int rank = me % share;
      const bool more = me / share < left;
      plan.items = rounds + more;
      plan.last = more ? rounds * grid + me / share : me + (rounds - 1) * grid;
      plan.s0 = more ? (int)((long long)p.steps * rank / share) : 0;
      plan.s1 = more ? (int)((long long)p.steps * (rank + 1) / share) : p.steps;
      plan.share = share;
      plan.mine = more && share > 1;
      plan.n_steps = (plan.items - 1) * p.steps + plan.s1 - plan.s0;
    }
  }
  __syncthreads();
  // The other shapes, which the plan would cost registers in their loops (3 to 8 %), take tiles `hop` apart from `first`, the same steps of each; the CTAs
  // of a cluster share all of theirs (one).
  const int total = pre[p.E], rank_of = SUB == 2 ? 0 : (int)blockIdx.x % p.split, first = SUB == 2 ? (int)blockIdx.x : (int)blockIdx.x / p.split;
  const int hop = SUB == 2 ? (int)gridDim.x : (int)gridDim.x / p.split, end = SUB == 2 ? first + plan.items * hop : p.split > 1 ? min(total, hop) : total;
  const int s0 = SUB == 2 ? 0 : (int)((long long)p.steps * rank_of / p.split), s1 = SUB == 2 ? p.steps : (int)((long long)p.steps * (rank_of + 1) / p.split);
  struct Item { int u, s0, s1; };
  auto item_at = [&](int u) {
    if (SUB == 2 && u + hop >= end) return Item{plan.last, plan.s0, plan.s1};
    return Item{u, s0, s1};
  };
  struct Tile { int e, m, row0, valid; };
  auto tile_at = [&](int u, int& e) {        // e: the expert of the role's tile before
    while (u >= pre[e + 1]) ++e;
    const int r = u - pre[e], nt = (cnt[e] + NT - 1) / NT, band = r / (IT_BAND * nt), rb = r - band * IT_BAND * nt, bm = min(IT_BAND, p.m_tiles - band * IT_BAND), n = rb / bm;
    return Tile{e, band * IT_BAND + rb - n * bm, off[e] + n * NT, min(NT, cnt[e] - n * NT)};
  };
  uint64_t acc[SUB][S::EPI_COLS / 2];        // two columns each
  const bool pair = p.flags & 1, f32 = p.flags & 4;
  auto store = [&](size_t at, float y) {
    if (f32) ((float*)p.out)[at] = p.residual ? y + ((const float*)p.residual)[at] : y;
    else ((__nv_bfloat16*)p.out)[at] = __float2bfloat16(p.residual ? y + __bfloat162float(((const __nv_bfloat16*)p.residual)[at]) : y);
  };
  // Of a pair the gate's lane finishes the first of two columns and the up's the second.
  auto of_pair = [&](float a, float b) {
    const bool up = lane & 8;
    const float other = __shfl_xor_sync(0xffffffffu, up ? a : b, 8), g = up ? other : a, u = up ? b : other;
    return silu(g) * u;
  };

  if (first < end) {
    if (warp == 0) {
      // ================= producer =================
      if (elect_one()) {
        if (p.src_row == nullptr) tma_prefetch_desc(&tmX);
        const uint64_t keep = l2_policy_evict_last();
        int st = 0, e = 0;
        uint32_t ph = 0;
        bool ok = true;
        for (int u = first; u < end && ok; u += hop) {
          const Item it = item_at(u);
          const Tile tl = tile_at(it.u, e);
          // (behind the last tile that one again, for nothing)
          const uint8_t* w = p.w + ((size_t)tl.e * p.w_tiles + tl.m * SUB) * p.steps * rec;
          const size_t second = tl.m * SUB + 1 < p.w_tiles ? (size_t)p.steps * rec : 0;
          for (int s = it.s0; s < it.s1; ++s) {
            if (!it_wait(smem_u32(&bar_empty[st]), ph ^ 1, &abort_flag, p.budget_ns)) {
              report_status(p.status, ST_TIMEOUT_SMEM_EMPTY, blockIdx.x);
              abort_flag = 1;
              ok = false;
              break;
            }
            const uint32_t full = smem_u32(&bar_full[st]), at = smem_base + st * stage_bytes;
            mbar_expect_tx(full, (p.src_row == nullptr ? X_BYTES : 0) + SUB * rec);
            bulk_load_1d(at + X_BYTES, w + (size_t)s * rec, rec, full);
            if (SUB == 2) bulk_load_1d(at + X_BYTES + w_bytes, w + second + (size_t)s * rec, rec, full);
            if (p.src_row == nullptr) {
              tma_load_2d(at, &tmX, full, s * I4_STEP, tl.row0, keep);
              tma_load_2d(at + NT * 128, &tmX, full, s * I4_STEP + 64, tl.row0, keep);
            }
            if (++st == p.stages) { st = 0; ph ^= 1; }
          }
        }
      }
      __syncwarp();
    } else if (warp == 1) {
      // ================= MMA =================
      if (elect_one()) {
        const uint32_t idesc = umma_idesc(1, 1, 128, NT);
        int st = 0, slot = 0, buf = 0;
        uint32_t sph = 0, bph = 0, seen_c = 0, seen_d = 0;
        bool ok = true;
        for (int u = first; u < end && ok; u += hop)
        for (int s = item_at(u).s0, to = item_at(u).s1; s < to; ++s) {
          // (the converters have seen the stage arrive, x included)
          if (!seen_c && !it_wait(smem_u32(&bar_cfull[slot]), sph, &abort_flag, p.budget_ns)) { report_status(p.status, ST_TIMEOUT_SMEM_FULL, blockIdx.x); abort_flag = 1; ok = false; break; }
          const uint32_t at = smem_base + st * stage_bytes;
          const uint64_t dx0 = umma_desc_sw128(at), dx1 = umma_desc_sw128(at + NT * 128);
          const uint32_t a_tmem = tmem_base + SUB * (S::BUFS * S::ACC + slot * 64);
          const uint32_t cempty = smem_u32(&bar_cempty[slot]), empty = smem_u32(&bar_empty[st]);
          if (++slot == S::SLOTS) { slot = 0; sph ^= 1; }
          if (++st == p.stages) st = 0;
#pragma unroll
          for (int g = 0; g < GP; ++g) {
            if (!seen_d && !it_wait(smem_u32(&bar_dempty[buf]), bph ^ 1, &abort_flag, p.budget_ns)) {
              report_status(p.status, ST_TIMEOUT_TMEM_EMPTY, blockIdx.x);
              ok = false;
              break;
            }
            tc_fence_after();
            constexpr int PER = 8 / GP;              // MMAs of a group
#pragma unroll
            for (int sub = 0; sub < SUB; ++sub)
#pragma unroll
              for (int i = 0; i < PER; ++i) {
                const int k = g * PER + i;
                mma_f16_ts(tmem_base + (buf * SUB + sub) * S::ACC, a_tmem + sub * 64 + 8 * k, (k < 4 ? dx0 : dx1) + 2 * (k & 3), idesc, i > 0 ? 1u : 0u);
              }
            tc_commit(smem_u32(&bar_dfull[buf]));
            if (++buf == S::BUFS) { buf = 0; bph ^= 1; }
            seen_d = it_peek(smem_u32(&bar_dempty[buf]), bph ^ 1);
          }
          if (!ok) { abort_flag = 1; break; }
          seen_c = it_peek(smem_u32(&bar_cfull[slot]), sph);
          tc_commit(cempty);
          tc_commit(empty);
        }
      }
      __syncwarp();
    } else if (warp < 4) {
      // ================= rows that src_row names: 16 lanes copy one, two warps four at a time, swizzled as TMA would =================
      if (NT < 128 && p.src_row != nullptr) {
        const int half = lane >> 4, c = lane & 15, first_row = 2 * (warp - 2) + half;
        int st = 0, e = 0;
        uint32_t ph = 0;
        bool ok = true;
        for (int u = first; u < end && ok; u += hop) {
          const Item it = item_at(u);
          const Tile tl = tile_at(it.u, e);
          // A lane looks one of its warp's rows up. Where the rows begin is kept for the tile; of tiles of 64, which have no registers for it, computed
          // for eight copies at a time (one chain from shuffle to copy is 70 cycles).
          const int mine = 4 * (lane >> 1) + 2 * (warp - 2) + (lane & 1);
          int from = 0;
          if (mine < tl.valid) {
            const int row = p.src_row[tl.row0 + mine];
            if (row < 0 || row >= p.x_rows) report_status(p.status, ST_BAD_INDEX, row);
            else from = row;
          }
          constexpr int PASSES = NT < 128 ? NT / 4 : 1, KEPT = PASSES < 8 ? PASSES : 8;
          const __nv_bfloat16* src[KEPT];
#pragma unroll
          for (int i = 0; i < KEPT && PASSES == KEPT; ++i) src[i] = p.x + (size_t)__shfl_sync(0xffffffffu, from, 2 * i + half) * p.x_ld;
          for (int s = it.s0; s < it.s1; ++s) {
            if (!it_warp_wait(0, smem_u32(&bar_empty[st]), ph ^ 1, &abort_flag, p.budget_ns)) {
              if (lane == 0) { report_status(p.status, ST_TIMEOUT_SMEM_EMPTY, blockIdx.x); abort_flag = 1; }
              ok = false;
              break;
            }
            const int k = s * I4_STEP + c * 8;             // (behind K zeros, as their scales are)
            const int at_k = k < p.K ? k : 0;
            const __nv_bfloat16* x = p.x + at_k;
            const uint32_t bytes = k < p.K ? 16 : 0, to = smem_base + st * stage_bytes + (c >> 3) * NT * 128 + first_row * 128;
#pragma unroll
            for (int i0 = 0; i0 < PASSES; i0 += KEPT) {
              if (PASSES > KEPT) {
                if (4 * i0 >= tl.valid) break;
#pragma unroll
                for (int i = 0; i < KEPT; ++i) src[i] = x + (size_t)__shfl_sync(0xffffffffu, from, 2 * (i0 + i) + half) * p.x_ld;
              }
#pragma unroll
              for (int i = 0; i < KEPT; ++i) {
                const int at = 4 * (i0 + i);
                // (rows of the stage behind the tile's last stay what they were: no result has them)
                if (at + first_row < tl.valid) it_copy16(to + at * 128 + (((c & 7) ^ ((at + first_row) & 7)) << 4), PASSES > KEPT ? src[i] : src[i] + at_k, bytes);
              }
            }
            it_copy_arrive(smem_u32(&bar_full[st]));
            if (++st == p.stages) { st = 0; ph ^= 1; }
          }
        }
        it_copy_wait_all();
      }
    } else if (warp >= 4 && warp < 4 + S::CONV_WARPS) {
      // ================= converters: row r of the tile; of eight warps four take a tile each, or the two groups the steps in turn =================
      constexpr int GROUPS = S::GROUPS;
      const int r = (warp & 3) * 32 + lane, sub = (warp - 4) / 4 % SUB, group = (warp - 4) / (4 * SUB);
      const uint32_t lane_tmem = (uint32_t)((warp & 3) * 32) << 16;
      const int in_stage = X_BYTES + sub * w_bytes + (r >> 4) * I4_CODES + (r & 7) * 16 + ((r >> 3) & 1) * 8, row_at = (r >> 4) * 8 + (r & 7), odd = (r >> 3) & 1;
      const int zero_at = X_BYTES + sub * w_bytes + i4_zeros(GP) + row_at * GP * 2 + odd, scale_at = X_BYTES + sub * w_bytes + I4_SCALES + row_at * GP * 4 + odd * 2;
      int st = group, slot = group;
      uint32_t ph = 0, sph = 0, seen = 0;
      // (a step is a step here, whatever tile it belongs to)
      const int n_steps = SUB == 2 ? plan.n_steps : (end - first + hop - 1) / hop * (s1 - s0);
      for (int s = group; s < n_steps; s += GROUPS) {
        if (!it_warp_wait(seen, smem_u32(&bar_full[st]), ph, &abort_flag, p.budget_ns)) {
          if (lane == 0) { report_status(p.status, ST_TIMEOUT_SMEM_FULL, blockIdx.x); abort_flag = 1; }
          break;
        }
        const uint8_t* at = smem_raw + (smem_base - smem_u32(smem_raw)) + st * stage_bytes;
        const uint32_t to = tmem_base + SUB * (S::BUFS * S::ACC + slot * 64) + sub * 64 + lane_tmem, cfull = smem_u32(&bar_cfull[slot]), cempty = smem_u32(&bar_cempty[slot]);
        uint32_t free_slot = it_peek(cempty, sph ^ 1);
        const uint32_t sph_now = sph;
        slot += GROUPS;
        if (slot >= S::SLOTS) { slot -= S::SLOTS; sph ^= 1; }
        st += GROUPS;                         // (two groups, an even number of stages: a group sees every phase of its own)
        if (st >= p.stages) { st -= p.stages; ph ^= 1; }
        // With registers for it the whole step is ready before the slot is asked for: what follows the wait is in the chain slot - MMAs - slot.
        constexpr int READY = S::ONE ? 2 : 1;       // halves of a step
        bool ok = true;
#pragma unroll
        for (int j0 = 0; j0 < 2; j0 += READY) {
          uint32_t v[READY][32];
#pragma unroll
          for (int i = 0; i < READY; ++i) {
            const int j = j0 + i;
            uint2 c[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) c[t] = *reinterpret_cast<const uint2*>(at + in_stage + j * 512 + t * 128);
            uint32_t base[2] = {I4_EIGHT, I4_EIGHT};
            if (zeros) {
              base[0] = i4_zero(at[zero_at + (GP == 1 ? 0 : GP == 2 ? j : 2 * j) * 2]);
              base[1] = GP == 4 ? i4_zero(at[zero_at + (2 * j + 1) * 2]) : base[0];
            }
#pragma unroll
            for (int t = 0; t < 4; ++t) {
              i4_expand(c[t].x, base[0], v[i] + t * 4);
              i4_expand(c[t].y, base[1], v[i] + 16 + t * 4);
            }
          }
          if (j0 == 0) {
            float sc[GP];
#pragma unroll
            for (int g = 0; g < GP; ++g) sc[g] = i4_scale(*reinterpret_cast<const uint16_t*>(at + scale_at + g * 4), p.flags & 2);
            if (!it_warp_wait(free_slot, cempty, sph_now ^ 1, &abort_flag, p.budget_ns)) {
              if (lane == 0) { report_status(p.status, ST_TIMEOUT_SMEM_EMPTY, blockIdx.x); abort_flag = 1; }
              ok = false;
              break;
            }
            tc_fence_after();
#pragma unroll
            for (int g = 0; g < GP; ++g) scales[s & (IT_SCALES - 1)][g][sub * 128 + r] = sc[g];
          }
#pragma unroll
          for (int i = 0; i < READY; ++i) {
            tmem_st16(to + (j0 + i) * 32, v[i]);
            tmem_st16(to + (j0 + i) * 32 + 16, v[i] + 16);
          }
        }
        if (!ok) break;
        seen = it_peek(smem_u32(&bar_full[st]), ph);
        // gathered rows are ordinary writes, which this thread has seen complete: from here on the MMAs see them too. (The gatherers would wait in the
        // fence for the copies that they have only begun.)
        if (p.src_row != nullptr) fence_proxy_async_smem();
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(cfull);
      }
    } else if (warp >= 4) {
      // ================= epilogue: row r, columns col0 .. + EPI_COLS =================
      const int r = (warp & 3) * 32 + lane, part = (warp - 4 - S::CONV_WARPS) >> 2, col0 = part * S::EPI_COLS;
      const uint32_t lane_tmem = (uint32_t)((warp & 3) * 32) << 16;
      int buf = 0, it = 0, e = 0;
      uint32_t bph = 0, seen = 0;
      bool ok = true;
      for (int u = first; u < end; u += hop) {
        const Item now = item_at(u);
#pragma unroll
        for (int h = 0; h < SUB; ++h)
#pragma unroll
          for (int c = 0; c < S::EPI_COLS / 2; ++c) acc[h][c] = 0ull;
        for (int s = now.s0; s < now.s1 && ok; ++s, ++it) {
#pragma unroll
          for (int g = 0; g < GP; ++g) {
            if (!it_warp_wait(seen, smem_u32(&bar_dfull[buf]), bph, &abort_flag, p.budget_ns)) {
              if (lane == 0) { report_status(p.status, ST_TIMEOUT_TMEM_FULL, blockIdx.x); abort_flag = 1; }
              ok = false;
              break;
            }
            tc_fence_after();
            const uint32_t from = tmem_base + buf * SUB * S::ACC + col0 + lane_tmem, dempty = smem_u32(&bar_dempty[buf]);
            if (++buf == S::BUFS) { buf = 0; bph ^= 1; }
            // (written before the arrival that let the step's MMAs begin)
            uint64_t s2[SUB];
#pragma unroll
            for (int h = 0; h < SUB; ++h) {
              const float sc = *reinterpret_cast<volatile float*>(&scales[it & (IT_SCALES - 1)][g][h * 128 + r]);
              s2[h] = it_pack(sc, sc);
            }
            constexpr int COLS_ALL = SUB * S::EPI_COLS, AT_ONCE = S::EPI_COLS < 32 ? 16 : 32;
#pragma unroll
            for (int c0 = 0; c0 < COLS_ALL; c0 += AT_ONCE) {
              uint32_t v[AT_ONCE];
#pragma unroll
              for (int c = 0; c < AT_ONCE; c += 16) tmem_ld16(from + c0 + c, v + c);
              tmem_ld_wait();
              if (c0 + AT_ONCE == COLS_ALL) {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(dempty);
                seen = it_peek(smem_u32(&bar_dfull[buf]), bph);
              }
#pragma unroll
              for (int c = 0; c < AT_ONCE; c += 2) it_fma2(acc[(c0 + c) / S::EPI_COLS][(c0 + c) % S::EPI_COLS / 2], v[c], v[c + 1], s2[(c0 + c) / S::EPI_COLS]);
            }
          }
        }
        if (!ok || (SUB == 2 ? plan.mine && u + hop >= end : p.split > 1)) break;
        const Tile tl = tile_at(now.u, e);
        // (MMAs of the next tile wait for these warps once the accumulators are full: what is the same for all columns stays out of the loops)
#pragma unroll
        for (int h = 0; h < SUB; ++h) {
          const int m = tl.m * SUB + h, f = pair ? (m * 8 + (r >> 4)) * 8 + (r & 7) : m * 128 + r, mine = pair ? (lane >> 3) & 1 : 0;
          const int left = f < p.F ? tl.valid - col0 - mine : 0;
          const size_t at = (size_t)(tl.row0 + col0 + mine) * p.out_ld + f;
          if (pair) {
            __nv_bfloat16* to = (__nv_bfloat16*)p.out + at;
#pragma unroll
            for (int c = 0; c < S::EPI_COLS; c += 2) {
              const float2 v = it_unpack(acc[h][c / 2]);
              const float y = of_pair(v.x, v.y);
              if (c < left) *to = __float2bfloat16(y);
              to += 2 * p.out_ld;
            }
          } else if (NT <= 32 && f32 && p.residual == nullptr) {        // (logits of a step)
            float* to = (float*)p.out + at;
#pragma unroll
            for (int c = 0; c < S::EPI_COLS; c += 2) {
              const float2 v = it_unpack(acc[h][c / 2]);
              if (c < left) *to = v.x;
              to += p.out_ld;
              if (c + 1 < left) *to = v.y;
              to += p.out_ld;
            }
          } else if (!f32 && p.residual == nullptr) {
            __nv_bfloat16* to = (__nv_bfloat16*)p.out + at;
#pragma unroll
            for (int c = 0; c < S::EPI_COLS; c += 2) {
              const float2 v = it_unpack(acc[h][c / 2]);
              if (c < left) *to = __float2bfloat16(v.x);
              to += p.out_ld;
              if (c + 1 < left) *to = __float2bfloat16(v.y);
              to += p.out_ld;
            }
          } else {
#pragma unroll
            for (int c = 0; c < S::EPI_COLS; c += 2) {
              const float2 v = it_unpack(acc[h][c / 2]);
              if (c < left) store(at + (size_t)c * p.out_ld, v.x);
              if (c + 1 < left) store(at + (size_t)(c + 1) * p.out_ld, v.y);
            }
          }
        }
      }
    }
  }

  // ---- the pieces of a tile: every CTA finishes NT / share columns, summed in rank order
  const int share = SUB == 2 ? plan.share : p.split;
  if (share > 1) {        // (of every CTA or none)
    const bool epi = (SUB == 2 ? plan.mine : first < end) && warp >= 4 + S::CONV_WARPS;
    const int rank = SUB == 2 ? (int)blockIdx.x % share : rank_of;
    const int r = (warp & 3) * 32 + lane, part = (warp - 4 - S::CONV_WARPS) >> 2, col0 = part * S::EPI_COLS;
    const int slice = NT / share, base = (int)blockIdx.x % p.split - rank;      // base: the group's first CTA in the cluster
    float* recv = reinterpret_cast<float*>(smem_raw + (smem_base - smem_u32(smem_raw)));      // [rank][tile][slice][128], on stages that nothing reads any more
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    if (epi) {
#pragma unroll
      for (int h = 0; h < SUB; ++h)
#pragma unroll
        for (int c = 0; c < S::EPI_COLS; c += 2) {       // (a slice is an even number of columns)
          const float2 v = it_unpack(acc[h][c / 2]);
          float* to = cluster.map_shared_rank(recv, base + (col0 + c) / slice) + ((rank * SUB + h) * slice + (col0 + c) % slice) * 128 + r;
          to[0] = v.x;
          to[128] = v.y;
        }
    }
    cluster.sync();
    if (epi && abort_flag == 0) {
      int e = 0;
      const Tile tl = tile_at(SUB == 2 ? plan.last : first, e);
      for (int h = 0; h < SUB; ++h) {
        const int m = tl.m * SUB + h, f = pair ? (m * 8 + (r >> 4)) * 8 + (r & 7) : m * 128 + r;
        for (int c = part * 2; c < slice; c += S::EPI_WARPS / 2) {
          const int col = rank * slice + c;
          if (col >= tl.valid) break;
          float a = 0.f, b = 0.f;
          for (int q = 0; q < share; ++q) {
            a += recv[((q * SUB + h) * slice + c) * 128 + r];
            b += recv[((q * SUB + h) * slice + c + 1) * 128 + r];
          }
          if (pair) {
            const float y = of_pair(a, b);
            const int own = col + ((lane >> 3) & 1);
            if (f < p.F && own < tl.valid) store((size_t)(tl.row0 + own) * p.out_ld + f, y);
          } else if (f < p.F) {
            store((size_t)(tl.row0 + col) * p.out_ld + f, a);
            if (col + 1 < tl.valid) store((size_t)(tl.row0 + col + 1) * p.out_ld + f, b);
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (abort_flag) {       // copies may still be on their way into this CTA's shared memory
    const uint64_t t0 = global_timer_ns();
    while (global_timer_ns() - t0 < 200000) __nanosleep(1000);
  }
  if (warp == 1) { tc_fence_after(); tmem_dealloc(tmem_base, S::COLS); }
}

template <int NT, int GP, int SUB>
static int launch_tc(const CUtensorMap& tmX, Int4Tc p, int tiles, cudaStream_t s) {
  using S = ItShape<NT, SUB>;
  static PerDevice allowed;
  const int list = 4 * (3 * p.E + 1), room = (S::ONE ? 224 : 112) * 1024 - IT_SCALES * GP * 512 * SUB - 2048;     // (beside the static part)
  const int stage = NT * 256 + SUB * ((i4_record(GP, p.flags & 8) + 1023) & ~1023);
  p.stages = (room - 1024 - list) / stage;
  if (p.stages > IT_MAX_STAGES) p.stages = IT_MAX_STAGES;
  if (S::GROUPS == 2) p.stages &= ~1;        // every stage belongs to one group of converters
  if (p.stages < 2) return -1;
  const cudaError_t e = allow_smem(allowed, (const void*)int4_tc_kernel<NT, GP, SUB>, room);
  if (e != cudaSuccess) return (int)e;
  cudaLaunchConfig_t cfg{};
  const int places = S::ONE ? 148 : 296;
  const bool walk = p.split == 1;
  // CTAs that stay. Of a dense product whose last round would leave half of them idle they come in pairs, which share its tiles (13 rows of 152064 x 3584: 83
  // us, 93 without; not experts, whose tiles the host cannot count and whose unequal CTAs pairs slow down: 48 tokens of 64 experts 37 us, 31 without).
  if (SUB == 2 && p.counts == nullptr && tiles > places && tiles % places != 0 && tiles % places <= places / 2) {
    p.split = 2;
    p.least = 4;
  }
  cfg.blockDim = dim3(S::THREADS);
  cfg.dynamicSmemBytes = (size_t)p.stages * stage + 1024 + list;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = p.split;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  cfg.gridDim = dim3((unsigned)(walk ? min(tiles, places) : tiles * p.split));
  return (int)cudaLaunchKernelEx(&cfg, int4_tc_kernel<NT, GP, SUB>, tmX, p);
}
template <int NT, int SUB>
static int launch_tc_group(const CUtensorMap& tmX, const Int4Tc& p, int group, int tiles, cudaStream_t s) {
  return group == 128 ? launch_tc<NT, 1, SUB>(tmX, p, tiles, s) : group == 64 ? launch_tc<NT, 2, SUB>(tmX, p, tiles, s) : launch_tc<NT, 4, SUB>(tmX, p, tiles, s);
}

}  // namespace skein

// Arguments as skein_int4_rows (int4_rows.cu); x and its rows on 16-byte boundaries. n_tile (16, 32, 64 or 128) rows of a tile, split CTAs that share
// the K of one (1, 2, 4 or 8); 0: by the rules here from rows_hint, the rows expected of an expert. Returns -1 for what it does not take.
extern "C" int skein_int4_tc(const void* x, long long x_ld, const int* src_row, const void* w, const void* residual, void* out, long long out_ld,
                             const int* counts, const int* offsets, int rows, int x_rows, int E, int F, int K, int group, int rows_hint, int flags, int n_tile,
                             int split, int* status, void* stream) {
  using namespace skein;
  if (rows == 0) return 0;
  if (rows < 0 || x_rows < 1 || E < 1 || E > 1024 || F < 1 || K < 32 || K % group != 0 || (group != 32 && group != 64 && group != 128)) return -1;
  if (x_ld % 8 != 0 || (uintptr_t)x % 16 != 0 || (uintptr_t)w % 16 != 0) return -1;
  if (n_tile == 0) {
    // experts' rows differ: room for a quarter more than their mean, as a second tile of an expert converts its weights again. Measured, us, tiles of
    // 16 / 32 / 64 rows: 28672 x 4096, 8 experts, mean 8 125 / 157 / 199, mean 16 179 / 160 / 199, mean 24 223 / 208 / 226; 2048 x 1408, 64 experts, mean
    // 4.5 31 / 38 / 46, mean 12 45 / 42 / 51, mean 37 81 / 70 / 65.
    const int want = counts == nullptr ? rows_hint : rows_hint + rows_hint / 4;
    n_tile = want <= 16 ? 16 : want <= 32 ? 32 : want <= 64 ? 64 : 128;
  }
  if (n_tile != 16 && n_tile != 32 && n_tile != 64 && n_tile != 128) return -1;
  // Gathered rows take two warps of a CTA as long as the MMAs of 128: two CTAs with 64 are as quick (28672 x 4096, 8 experts, mean 64 353 us and 413, mean 250
  // 1031 and 1066).
  if (src_row != nullptr && n_tile == 128) n_tile = 64;
  Int4Tc p;
  p.x = (const __nv_bfloat16*)x; p.x_ld = x_ld; p.src_row = src_row; p.w = (const uint8_t*)w; p.residual = residual; p.out = out; p.counts = counts; p.offsets = offsets; p.status = status;
  p.out_ld = out_ld; p.rows = rows; p.x_rows = x_rows; p.E = E; p.F = F; p.K = K; p.flags = flags;
  p.strips = flags & 1 ? (F + 7) / 8 : (F + 15) / 16;
  p.steps = (K + I4_STEP - 1) / I4_STEP;
  p.w_tiles = (p.strips + 7) / 8;
  p.budget_ns = (uint64_t)gemm_wait_budget_ms() * 1000000ull;
  // row tiles at most (an expert's last one may be part empty), and those to expect
  const long long row_tiles = counts == nullptr ? (rows + n_tile - 1) / n_tile : (rows + (long long)(n_tile - 1) * (E < rows ? E : rows)) / n_tile;
  const long long expect_rows = counts == nullptr ? row_tiles : rows < E ? (long long)rows : (long long)E * ((rows_hint + n_tile - 1) / n_tile);
  // Two tiles of 16 rows at a time from where one each fills the GPU (1408 x 2048 pairs, 64 experts, mean 4.5: 79 us one at a time, 65 two; 152064 x 3584 100
  // and 83; but 18944 x 2048, 148 tiles, 12.1 and 16.2).
  const bool two = n_tile == 16 && split <= 1 && p.w_tiles * expect_rows >= 296;
  p.m_tiles = two ? (p.w_tiles + 1) / 2 : p.w_tiles;
  const long long tiles = row_tiles * p.m_tiles;
  if (split == 0) {
    // Pieces until every place on the GPU has a CTA, while they keep eight steps, or four where there is less than one CTA per SM (16 rows of 4096 x 4096:
    // 12.7 us in two pieces, 10.1 in four of eight steps, 10.7 in eight; 1024 x 4096 11.9 in four, 9.3 in eight; 4096 x 14336 18.6 and 17.6).
    const long long expect = p.m_tiles * expect_rows;
    const int slots = 148 * (n_tile == 128 ? 1 : 2);
    split = 1;
    while (!two && split < 8 && expect * split * 2 <= slots && p.steps / (split * 2) >= (expect * split * 2 <= 148 ? 4 : 8)) split *= 2;
  }
  if (split != 1 && split != 2 && split != 4 && split != 8) return -1;
  if (tiles * split > 0x7fffffffll) return -1;
  p.split = split;
  p.least = 0;
  CUtensorMap tmX{};
  if (src_row == nullptr) {
    const int rc = make_tmap_2d(&tmX, x, (uint64_t)x_rows, (uint64_t)K, (uint64_t)x_ld, 2, n_tile);
    if (rc) return rc;
  }
  cudaStream_t s = (cudaStream_t)stream;
  switch (n_tile) {
    case 16: return two ? launch_tc_group<16, 2>(tmX, p, group, (int)tiles, s) : launch_tc_group<16, 1>(tmX, p, group, (int)tiles, s);
    case 32: return launch_tc_group<32, 1>(tmX, p, group, (int)tiles, s);
    case 64: return launch_tc_group<64, 1>(tmX, p, group, (int)tiles, s);
    default: return launch_tc_group<128, 1>(tmX, p, group, (int)tiles, s);
  }
}
