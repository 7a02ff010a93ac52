// Products of few rows with 4-bit weights (int4.cuh): a decode step's dense projections and its experts.
//
//   y[r, f] = sum over groups j of scale[f, j] * ( sum_{k in j} x[r, k] (code[f, k] - zero[f, j]) )
//
// With a few rows the weights' bytes bound the time, and what has to be done for each of them besides. A warp reads a step of a strip (16 rows x 128 of
// K) with two 16-byte loads per lane, turns the codes into bf16 (exact, nine instructions per word of eight) and multiplies them
// with mma.sync m16n8k16 against eight rows of x in shared memory. A group's sum is fp32 and is scaled in fp32, so nothing is rounded before the result.
// A CTA per SM stays for the launch. WK of its 16 warps make a team that shares the K of a strip (a warp every WK-th step) and walks its run of strips;
// the loads of the next four steps, the next strip's among them, are always on their way. The team's sums meet in shared memory and are added up in warp order
// a strip later, so that no warp waits for the slowest. The runs are equal shares of all strips that some row goes to, whatever expert they belong to.
// What bounds it: the instructions. A step of a strip is about 150 of them, 72 for the codes and 8 products, and the 16 warps that the registers leave
// room for issue half of the cycles (28672 x 8192 gate / up, one row: 63 us, 3.9 TB/s, where HBM would take 38). Tried and not kept: the codes as
// subnormal operands of the products without a multiply-add, with scaled rows of x and their sums for the zeros (63 us, but 232 against 139 for 13 rows
// of 152064 x 3584); two strips per warp (62 and 182); a ring in shared memory filled with cp.async (72 and 148).
#include "int4.cuh"
#include "launch.cuh"

namespace skein {

constexpr int IR_WARPS = 16, IR_THREADS = 32 * IR_WARPS;
constexpr int IR_DEPTH = 4;             // steps whose codes are in flight
constexpr int IR_MAX_E = 1024;
constexpr int IR_SMEM = 184 * 1024;     // for the rows of x

struct Int4Rows {
  const __nv_bfloat16* x;
  const int* src_row;
  const uint8_t* w;
  const void* residual;
  void* out;
  const int *counts, *offsets;
  int* status;
  long long x_ld, out_ld;
  uint64_t budget_ns;
  int rows, x_rows, E, F, K, strips, steps, out_f32, vec, pair, x_stage;   // x_stage: rows of a tile (8, or as many as fit a team's shared memory)
};

// bytes of a row of x in shared memory: 64 past a multiple of 128, so that eight rows x 64 bytes lie in different banks
__host__ __device__ constexpr int ir_x_row(int steps) { return steps * I4_STEP * 2 + 64; }

// eight neighbours of a row of x from k on, zero past its end
__device__ __forceinline__ uint4 ir_load_x(const __nv_bfloat16* row, int k, int K, int vec) {
  uint4 v = make_uint4(0, 0, 0, 0);
  if (k >= K) return v;
  if (vec) return __ldg(reinterpret_cast<const uint4*>(row + k));   // K is a multiple of 8
  const unsigned short* s = reinterpret_cast<const unsigned short*>(row + k);
  v.x = s[0] | (uint32_t)s[1] << 16; v.y = s[2] | (uint32_t)s[3] << 16;
  v.z = s[4] | (uint32_t)s[5] << 16; v.w = s[6] | (uint32_t)s[7] << 16;
  return v;
}
template <int THREADS>
__device__ __forceinline__ void ir_team_sync(int team) {
  if constexpr (THREADS == 32) __syncwarp();
  else asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "n"(THREADS) : "memory");
}
// the first product of a group: no sum to add to
__device__ __forceinline__ void ir_mma0(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
               : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void ir_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <int GP, bool ZERO>
struct Int4Step {       // a lane's part of a step of one strip
  uint4 c[2];
  uint32_t s[GP];       // scales of rows g and g + 8
  uint16_t z[ZERO ? GP : 1];
  __device__ __forceinline__ void load(const uint8_t* codes, const uint8_t* scales, const uint8_t* zeros) {
    c[0] = __ldcs(reinterpret_cast<const uint4*>(codes));
    c[1] = __ldcs(reinterpret_cast<const uint4*>(codes + 512));
    if constexpr (GP == 1) s[0] = __ldcs(reinterpret_cast<const uint32_t*>(scales));
    if constexpr (GP == 2) { const uint2 v = __ldcs(reinterpret_cast<const uint2*>(scales)); s[0] = v.x; s[1] = v.y; }
    if constexpr (GP == 4) { const uint4 v = __ldcs(reinterpret_cast<const uint4*>(scales)); s[0] = v.x; s[1] = v.y; s[2] = v.z; s[3] = v.w; }
    if constexpr (ZERO) {
      if constexpr (GP == 1) z[0] = __ldcs(reinterpret_cast<const uint16_t*>(zeros));
      if constexpr (GP == 2) { const ushort2 v = __ldcs(reinterpret_cast<const ushort2*>(zeros)); z[0] = v.x; z[1] = v.y; }
      if constexpr (GP == 4) { const ushort4 v = __ldcs(reinterpret_cast<const ushort4*>(zeros)); z[0] = v.x; z[1] = v.y; z[2] = v.z; z[3] = v.w; }
    }
  }
};

template <int GP, bool ZERO, bool HALF, int WK>
__global__ void __launch_bounds__(IR_THREADS, 1) int4_rows_kernel(const __grid_constant__ Int4Rows p) {
  constexpr int TEAMS = IR_WARPS / WK, REC = i4_record(GP, ZERO);
  extern __shared__ __align__(16) uint8_t x_smem[];
  __shared__ float4 sums[2][IR_WARPS][32];
  __shared__ int pre[IR_MAX_E + 1], cnt[IR_MAX_E];      // row tiles before an expert, its rows
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  __shared__ __align__(8) uint64_t bar[TEAMS];          // a team's sums of a strip are parked
  __shared__ int abort_flag;
  const int team = warp / WK, part = warp % WK;
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int i = 0; i < TEAMS; ++i) mbar_init(smem_u32(&bar[i]), WK);
    fence_mbar_init();
  }
  pdl_trigger();
  pdl_wait();
  if (warp == 0) {
    int run = 0;
    for (int e0 = 0; e0 < p.E; e0 += 32) {
      int c = 0;
      if (e0 + lane < p.E) {
        c = p.rows;
        if (p.counts != nullptr) {
          const int first = p.offsets[e0 + lane];
          c = p.counts[e0 + lane];
          if (first < 0 || c < 0 || c > p.rows - first) {
            if (c != 0) report_status(p.status, ST_BAD_INDEX, e0 + lane);
            c = 0;
          }
        }
      }
      const int tiles = (c + p.x_stage - 1) / p.x_stage;
      int inc = tiles;
      for (int o = 1; o < 32; o <<= 1) { const int v = __shfl_up_sync(0xffffffffu, inc, o); if (lane >= o) inc += v; }
      if (e0 + lane < p.E) { pre[e0 + lane] = run + inc - tiles; cnt[e0 + lane] = c; }
      run += __shfl_sync(0xffffffffu, inc, 31);
    }
    if (lane == 0) pre[p.E] = run;
  }
  __syncthreads();
  // the team's run of units (row tile, strip), strips fastest
  const int who = blockIdx.x * TEAMS + team, teams = gridDim.x * TEAMS;
  const int u0 = (int)((long long)pre[p.E] * p.strips * who / teams), u1 = (int)((long long)pre[p.E] * p.strips * (who + 1) / teams);
  const int mine = (p.steps - part + WK - 1) / WK;       // steps of a strip that this warp takes (at least one: WK <= steps)
  // cursor of the loads, ahead of the products
  const size_t matrix = (size_t)((p.strips + 7) / 8) * p.steps * REC;
  int le = 0, lleft = u1 - u0, ltile = u0 / p.strips, lstrip = u0 - ltile * p.strips, li = 0;
  const uint8_t *lc = nullptr, *ls = nullptr, *lz = nullptr;
  auto seek = [&]() {
    while (ltile >= pre[le + 1]) ++le;
    const uint8_t* at = p.w + le * matrix + ((size_t)(lstrip >> 3) * p.steps + part) * REC;
    const int row = (lstrip & 7) * 8 + g;
    lc = at + (lstrip & 7) * I4_CODES + (t * 8 + g) * 16;
    ls = at + I4_SCALES + row * GP * 4;
    if constexpr (ZERO) lz = at + i4_zeros(GP) + row * GP * 2;
  };
  if (lleft > 0) seek();
  Int4Step<GP, ZERO> buf[IR_DEPTH];
  auto load = [&](Int4Step<GP, ZERO>& b) {
    if (lleft <= 0) return;
    b.load(lc, ls, lz);
    if (++li < mine) {
      lc += WK * REC;
      ls += WK * REC;
      if constexpr (ZERO) lz += WK * REC;
    } else {
      li = 0;
      if (++lstrip == p.strips) { lstrip = 0; ++ltile; }
      if (--lleft > 0) seek();
    }
  };
#pragma unroll
  for (int d = 0; d < IR_DEPTH; ++d) load(buf[d]);

  const int x_row = ir_x_row(p.steps);
  uint8_t* x_team = x_smem + (size_t)team * p.x_stage * x_row;
  int e = 0, i = 0, n_done = 0, valid = 0, row0 = 0, old_valid = 0, old_row0 = 0, old_strip = 0;
  int left = u1 - u0, tile = u0 / p.strips, staged = -1, strip = u0 - tile * p.strips;
  const uint8_t* xb = nullptr;
  float acc[4];
  // adds up the team's sums of the strip before (its turn goes round the warps) and stores them
  auto finish = [&]() {
    if ((n_done - 1) % WK != part) return;
    float4 (*parked)[32] = sums[(n_done - 1) & 1] + team * WK;
    float4 v = parked[0][lane];
#pragma unroll
    for (int w = 1; w < WK; ++w) {
      const float4 o = parked[w][lane];
      v.x += o.x; v.y += o.y; v.z += o.z; v.w += o.w;
    }
    // v: (row g, x rows 2t and 2t + 1), (row g + 8, the same)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int r = 2 * t + j;
      if (r >= old_valid) continue;
      const float a = 64.f * (j ? v.y : v.x), b = 64.f * (j ? v.w : v.z);       // (the codes were 64ths)
      const size_t to = (size_t)(old_row0 + r) * p.out_ld;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (p.pair && h) continue;
        const int f = p.pair ? old_strip * 8 + g : old_strip * 16 + g + 8 * h;
        if (f >= p.F) continue;
        const float y = p.pair ? silu(a) * b : h ? b : a;
        if (p.out_f32) ((float*)p.out)[to + f] = p.residual ? y + ((const float*)p.residual)[to + f] : y;
        else ((__nv_bfloat16*)p.out)[to + f] = __float2bfloat16(p.residual ? y + __bfloat162float(((const __nv_bfloat16*)p.residual)[to + f]) : y);
      }
    }
  };
  while (left > 0) {
#pragma unroll
    for (int d = 0; d < IR_DEPTH; ++d) {
      if (left <= 0) break;
      if (i == 0) {
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[k] = 0.f;
        if (staged != tile) {      // the rows of x of this tile
          while (tile >= pre[e + 1]) ++e;
          const int first = (tile - pre[e]) * p.x_stage, base = p.counts != nullptr ? p.offsets[e] : 0;
          valid = min(p.x_stage, cnt[e] - first);
          row0 = base + first;
          const int chunks = p.steps * (I4_STEP / 8);
          if (staged >= 0) ir_team_sync<WK * 32>(team);      // every warp is past its products with the rows before
          // all threads of the team over the rows' 16-byte pieces, four loads at a time
          for (int i0 = part * 32 + lane; i0 < valid * chunks; i0 += 4 * WK * 32) {
            uint4 v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int at = i0 + k * WK * 32, r = at / chunks, c = at - r * chunks;
              v[k] = make_uint4(0, 0, 0, 0);
              if (r < valid) {
                const int from = p.src_row != nullptr ? p.src_row[row0 + r] : row0 + r;
                if (from >= 0 && from < p.x_rows) v[k] = ir_load_x(p.x + (size_t)from * p.x_ld, c * 8, p.K, p.vec);
                else if (c == 0) report_status(p.status, ST_BAD_INDEX, from);
              }
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int at = i0 + k * WK * 32, r = at / chunks, c = at - r * chunks;
              if (r < valid) *reinterpret_cast<uint4*>(x_team + (size_t)r * x_row + c * 16) = v[k];
            }
          }
          staged = tile;
          xb = x_team + (size_t)min(g, valid - 1) * x_row + t * 16 + part * I4_STEP * 2;
          ir_team_sync<WK * 32>(team);
        }
      }
      const int at = i * (WK * I4_STEP * 2);
      constexpr int per = 4 / GP;               // quarters of a step in a group
      float part_sum[4];
      uint32_t lo[4], hi[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {             // 32 of K each
        const int grp = q / per;
        const uint4 c = buf[d].c[q >> 1];
        i4_expand(q & 1 ? c.y : c.x, ZERO ? i4_zero(buf[d].z[ZERO ? grp : 0] & 0xff) : I4_EIGHT, lo);
        i4_expand(q & 1 ? c.w : c.z, ZERO ? i4_zero(buf[d].z[ZERO ? grp : 0] >> 8) : I4_EIGHT, hi);
        const uint4 b = *reinterpret_cast<const uint4*>(xb + at + q * 64);
        if (q % per == 0) ir_mma0(part_sum, lo[0], hi[0], lo[1], hi[1], b.x, b.y);
        else ir_mma(part_sum, lo[0], hi[0], lo[1], hi[1], b.x, b.y);
        ir_mma(part_sum, lo[2], hi[2], lo[3], hi[3], b.z, b.w);
        if (q % per == per - 1) {
          float sl, sh;
          if constexpr (HALF) { const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&buf[d].s[grp])); sl = f.x; sh = f.y; }
          else { sl = __uint_as_float(buf[d].s[grp] << 16); sh = __uint_as_float(buf[d].s[grp] & 0xffff0000u); }
          acc[0] += sl * part_sum[0]; acc[1] += sl * part_sum[1];
          acc[2] += sh * part_sum[2]; acc[3] += sh * part_sum[3];
        }
      }
      load(buf[d]);
      if (++i < mine) continue;
      // The strip is done: the sums of the one before are complete and added up, then this one's are parked in the other half. Whoever parks those of
      // strip n + 2 has seen all warps arrive with n + 1, which they do after they have added up n.
      i = 0;
      --left;
      if (n_done > 0) {
        if (WK > 1 && !mbar_wait(smem_u32(&bar[team]), (n_done - 1) & 1, &abort_flag, p.budget_ns)) { report_status(p.status, ST_TIMEOUT_SMEM_FULL, blockIdx.x); abort_flag = 1; }
        __syncwarp();
        finish();
      }
      sums[n_done & 1][warp][lane] = make_float4(acc[0], acc[1], acc[2], acc[3]);
      __syncwarp();
      if (WK > 1 && lane == 0) mbar_arrive(smem_u32(&bar[team]));
      ++n_done;
      old_valid = valid;
      old_row0 = row0;
      old_strip = strip;
      if (++strip == p.strips) { strip = 0; ++tile; }
    }
  }
  if (n_done > 0) {
    if (WK > 1 && !mbar_wait(smem_u32(&bar[team]), (n_done - 1) & 1, &abort_flag, p.budget_ns)) report_status(p.status, ST_TIMEOUT_SMEM_FULL, blockIdx.x);
    __syncwarp();
    finish();
  }
}

template <int GP, bool ZERO, bool HALF, int WK>
static int launch_rows(Int4Rows p, cudaStream_t s) {
  static PerDevice allowed;
  constexpr int TEAMS = IR_WARPS / WK;
  p.x_stage = min(8, p.rows);
  while (p.x_stage > 0 && TEAMS * (p.x_stage * ir_x_row(p.steps)) > IR_SMEM) --p.x_stage;
  if (p.x_stage < 1 || ((long long)p.rows / p.x_stage + min(p.E, p.rows)) * p.strips > 0x7fffffffll) return -1;
  const cudaError_t e = allow_smem(allowed, (const void*)int4_rows_kernel<GP, ZERO, HALF, WK>, IR_SMEM);
  if (e != cudaSuccess) return (int)e;
  return (int)launch_pdl(int4_rows_kernel<GP, ZERO, HALF, WK>, dim3(148), dim3(IR_THREADS), (size_t)TEAMS * (p.x_stage * ir_x_row(p.steps)), s, p);
}
// Warps of a team: as many as leave each three steps or more of a strip, and more where its rows of x do not fit a smaller team's shared memory or the
// strips are few (one row of 4096 x 4096, 256 strips: 7.3 us with 8 warps, 7.7 with 16, but four rows 8.9 and 8.8, and 1024 x 4096 5.9 and 5.3;
// 28672 x 4096 25.2 and 27.7; 2048 x 1408 over experts 32.7 with 4, 34.8 with 8).
template <int GP, bool ZERO, bool HALF>
static int pick_team(const Int4Rows& p, int team, cudaStream_t s) {
  const int x = min(8, p.rows) * ir_x_row(p.steps);
  const long long strips = (long long)p.strips * min(p.E, p.rows);
  if (team == 0)
    team = p.steps >= 48 || (p.steps >= 24 && strips <= 296 && (p.rows > 2 || strips <= 148)) || (p.steps >= 16 && x > IR_SMEM / 2)  ? 16
           : p.steps >= 24 || (p.steps >= 8 && x > IR_SMEM / 4) ? 8
           : p.steps >= 4                                       ? 4
                                                                : 1;
  if (team > p.steps) return -1;
  switch (team) {
    case 16: return launch_rows<GP, ZERO, HALF, 16>(p, s);
    case 8: return launch_rows<GP, ZERO, HALF, 8>(p, s);
    case 4: return launch_rows<GP, ZERO, HALF, 4>(p, s);
    case 1: return launch_rows<GP, ZERO, HALF, 1>(p, s);
    default: return -1;
  }
}
template <int GP>
static int pick_form(const Int4Rows& p, bool zero, bool half, int team, cudaStream_t s) {
  if (zero) return half ? pick_team<GP, true, true>(p, team, s) : pick_team<GP, true, false>(p, team, s);
  return half ? pick_team<GP, false, true>(p, team, s) : pick_team<GP, false, false>(p, team, s);
}
static int pick_group(const Int4Rows& p, int group, bool zero, bool half, int team, cudaStream_t s) {
  return group == 128 ? pick_form<1>(p, zero, half, team, s) : group == 64 ? pick_form<2>(p, zero, half, team, s) : pick_form<4>(p, zero, half, team, s);
}

}  // namespace skein

// x [x_rows, x_ld] bf16 (row r of the product reads row src_row[r], or r); w as in int4.cuh; out and residual [rows, out_ld] bf16
// or fp32. counts / offsets null: one matrix for all rows. rows_hint is for the other kernel. flags: 1 pair, 2 fp16 scales, 4 fp32 output, 8 zeros.
// team: warps that share a strip (1, 4, 8 or 16, at most its steps), 0: by the rule above. Returns -1 for what it does not take (more than IR_MAX_E experts,
// a weight off 16-byte boundaries, or a row of x past the shared memory: K of 94,000).
extern "C" int skein_int4_rows(const void* x, long long x_ld, const int* src_row, const void* w, const void* residual, void* out, long long out_ld,
                               const int* counts, const int* offsets, int rows, int x_rows, int E, int F, int K, int group, int /*rows_hint*/, int flags, int team,
                               int* status, void* stream) {
  using namespace skein;
  if (rows == 0) return 0;
  if (rows < 0 || E < 1 || E > IR_MAX_E || F < 1 || K < 32 || K % group != 0 || (group != 32 && group != 64 && group != 128)) return -1;
  if ((uintptr_t)w % 16 != 0) return -1;
  Int4Rows p;
  p.x = (const __nv_bfloat16*)x; p.src_row = src_row; p.w = (const uint8_t*)w; p.residual = residual; p.out = out; p.counts = counts;
  p.offsets = offsets; p.status = status; p.x_ld = x_ld; p.out_ld = out_ld; p.rows = rows; p.x_rows = x_rows; p.E = E; p.F = F; p.K = K;
  p.budget_ns = (uint64_t)gemm_wait_budget_ms() * 1000000ull;
  p.pair = flags & 1;
  p.strips = p.pair ? (F + 7) / 8 : (F + 15) / 16;
  p.steps = (K + I4_STEP - 1) / I4_STEP;
  p.out_f32 = (flags >> 2) & 1;
  p.vec = x_ld % 8 == 0 && (uintptr_t)x % 16 == 0;
  cudaStream_t s = (cudaStream_t)stream;
  return pick_group(p, group, flags & 8, flags & 2, team, s);
}
