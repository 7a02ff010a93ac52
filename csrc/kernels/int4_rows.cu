// Products of few rows with 4-bit weights (int4.cuh): a decode step's dense projections and its experts.
//
//   y[r, f] = sum over groups j of scale[f, j] * ( sum_{k in j} x[r, k] (code[f, k] - zero[f, j]) )
//
// With a few rows the weights' bytes bound the time, and what has to be done for each of them besides. A warp reads 16 rows of a strip x 128
// of K with two 16-byte loads per lane, turns the codes into bf16 whole numbers (exact, three instructions per pair) and multiplies them
// with mma.sync m16n8k16 against eight rows of x, whose fragments it reads through L1 in the order of the codes. A group's sum is fp32 and is
// scaled in fp32, so nothing is rounded before the result. The warps of a unit share K and add their sums in shared memory in warp order.
#include "int4.cuh"
#include "launch.cuh"

namespace skein {

constexpr int IR_WARPS = 8, IR_THREADS = 32 * IR_WARPS;
constexpr int IR_DEPTH = 4;      // steps whose codes are in flight

struct Int4Rows {
  const __nv_bfloat16* x;
  const int* src_row;
  const uint8_t* w;
  const void* residual;
  void* out;
  const int *counts, *offsets;
  int* status;
  long long x_ld, out_ld;
  int rows, x_rows, F, K, strips, steps, scale_half, out_f32, vec;
};

// eight neighbours of a row of x from k on, zero past its end
__device__ __forceinline__ uint4 ir_load_x(const __nv_bfloat16* row, int k, int K, int vec) {
  uint4 v = make_uint4(0, 0, 0, 0);
  if (row == nullptr || k >= K) return v;
  if (vec) return *reinterpret_cast<const uint4*>(row + k);   // K is a multiple of 8
  const unsigned short* s = reinterpret_cast<const unsigned short*>(row + k);
  v.x = s[0] | (uint32_t)s[1] << 16; v.y = s[2] | (uint32_t)s[3] << 16;
  v.z = s[4] | (uint32_t)s[5] << 16; v.w = s[6] | (uint32_t)s[7] << 16;
  return v;
}
__device__ __forceinline__ void ir_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <int GP, bool ZERO>
struct Int4Step {       // a lane's part of a step of one strip
  uint4 c[2];
  uint32_t s[GP];       // scales of rows g and g + 8
  uint16_t z[GP];
  __device__ __forceinline__ void load(const uint8_t* rec, int strip, int lane) {
    const int g = lane >> 2;
    const uint8_t* at = rec + strip * I4_CODES + ((lane & 3) * 8 + g) * 16;
    c[0] = __ldcs(reinterpret_cast<const uint4*>(at));
    c[1] = __ldcs(reinterpret_cast<const uint4*>(at + 512));
    const uint32_t* sp = reinterpret_cast<const uint32_t*>(rec + I4_SCALES) + (strip * 8 + g) * GP;
    if constexpr (GP == 1) s[0] = __ldg(sp);
    if constexpr (GP == 2) { const uint2 v = __ldg(reinterpret_cast<const uint2*>(sp)); s[0] = v.x; s[1] = v.y; }
    if constexpr (GP == 4) { const uint4 v = __ldg(reinterpret_cast<const uint4*>(sp)); s[0] = v.x; s[1] = v.y; s[2] = v.z; s[3] = v.w; }
    if constexpr (ZERO) {
      const uint16_t* zp = reinterpret_cast<const uint16_t*>(rec + i4_zeros(GP)) + (strip * 8 + g) * GP;
      if constexpr (GP == 1) z[0] = __ldg(zp);
      if constexpr (GP == 2) { const ushort2 v = __ldg(reinterpret_cast<const ushort2*>(zp)); z[0] = v.x; z[1] = v.y; }
      if constexpr (GP == 4) { const ushort4 v = __ldg(reinterpret_cast<const ushort4*>(zp)); z[0] = v.x; z[1] = v.y; z[2] = v.z; z[3] = v.w; }
    }
  }
};

// grid (strips / units of a CTA, experts, tiles of 8 NT rows of an expert, which a CTA walks with that stride). WK warps share a strip's K.
template <int NT, int GP, bool ZERO, bool PAIR, int WK>
__global__ void __launch_bounds__(IR_THREADS) int4_rows_kernel(const Int4Rows p) {
  constexpr int UNITS = IR_WARPS / WK;
  __shared__ float4 sums[IR_WARPS][NT][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int unit = warp / WK, part = warp % WK, strip = blockIdx.x * UNITS + unit, e = blockIdx.y;
  pdl_trigger();
  pdl_wait();
  int first = 0, count = p.rows;
  if (p.counts != nullptr) {
    first = p.offsets[e];
    count = p.counts[e];
    if (first < 0 || count < 0 || count > p.rows - first) {
      if (threadIdx.x == 0 && count != 0) report_status(p.status, ST_BAD_INDEX, e);
      count = 0;
    }
  }
  const bool live = strip < p.strips;
  constexpr int REC = i4_record(GP, ZERO);
  const uint8_t* tile_w = p.w + ((size_t)e * ((p.strips + 7) / 8) + (live ? strip >> 3 : 0)) * p.steps * REC;
  for (int tile = blockIdx.z; tile * 8 * NT < count; tile += gridDim.z) {
    const __nv_bfloat16* row[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = tile * 8 * NT + n * 8 + g;
      row[n] = nullptr;
      if (r < count) {
        const int from = p.src_row != nullptr ? p.src_row[first + r] : first + r;
        if (from >= 0 && from < p.x_rows) row[n] = p.x + (size_t)from * p.x_ld;
        else report_status(p.status, ST_BAD_INDEX, from);
      }
    }
    float acc[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[n][i] = 0.f;
    Int4Step<GP, ZERO> buf[IR_DEPTH];
#pragma unroll
    for (int d = 0; d < IR_DEPTH; ++d)
      if (live && part + d * WK < p.steps) buf[d].load(tile_w + (size_t)(part + d * WK) * REC, strip & 7, lane);
    for (int s0 = part; s0 < p.steps; s0 += IR_DEPTH * WK) {
#pragma unroll
      for (int d = 0; d < IR_DEPTH; ++d) {
        const int step = s0 + d * WK;
        if (step >= p.steps || !live) break;
        const Int4Step<GP, ZERO> cur = buf[d];
        if (step + IR_DEPTH * WK < p.steps) buf[d].load(tile_w + (size_t)(step + IR_DEPTH * WK) * REC, strip & 7, lane);
        float part_sum[NT][4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {             // 32 of K each
          const int grp = q * GP / 4;
          if (q * GP % 4 == 0)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int i = 0; i < 4; ++i) part_sum[n][i] = 0.f;
          const uint4 c = cur.c[q >> 1];
          uint32_t lo[4], hi[4];
          i4_expand(q & 1 ? c.y : c.x, i4_base(ZERO ? cur.z[grp] & 0xff : 8), lo);
          i4_expand(q & 1 ? c.w : c.z, i4_base(ZERO ? cur.z[grp] >> 8 : 8), hi);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const uint4 b = ir_load_x(row[n], step * I4_STEP + q * 32 + t * 8, p.K, p.vec);
            ir_mma(part_sum[n], lo[0], hi[0], lo[1], hi[1], b.x, b.y);
            ir_mma(part_sum[n], lo[2], hi[2], lo[3], hi[3], b.z, b.w);
          }
          if ((q + 1) * GP % 4 == 0) {
            const float sl = i4_scale(cur.s[grp] & 0xffff, p.scale_half), sh = i4_scale(cur.s[grp] >> 16, p.scale_half);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              acc[n][0] += sl * part_sum[n][0]; acc[n][1] += sl * part_sum[n][1];
              acc[n][2] += sh * part_sum[n][2]; acc[n][3] += sh * part_sum[n][3];
            }
          }
        }
      }
    }
    __syncthreads();              // the sums of the tile before are read
#pragma unroll
    for (int n = 0; n < NT; ++n) sums[warp][n][lane] = make_float4(acc[n][0], acc[n][1], acc[n][2], acc[n][3]);
    __syncthreads();
    for (int n = part; n < NT; n += WK) {
      float4 v = sums[unit * WK][n][lane];
#pragma unroll
      for (int w = 1; w < WK; ++w) {
        const float4 o = sums[unit * WK + w][n][lane];
        v.x += o.x; v.y += o.y; v.z += o.z; v.w += o.w;
      }
      // v: (row g, x rows 2t and 2t + 1), (row g + 8, the same)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int r = tile * 8 * NT + n * 8 + 2 * t + j;
        if (r >= count || !live) continue;
        const float a = j ? v.y : v.x, b = j ? v.w : v.z;
        const size_t at = (size_t)(first + r) * p.out_ld;
#pragma unroll
        for (int h = 0; h < (PAIR ? 1 : 2); ++h) {
          const int f = PAIR ? strip * 8 + g : strip * 16 + g + 8 * h;
          if (f >= p.F) continue;
          float y = PAIR ? silu(a) * b : h ? b : a;
          if (p.out_f32) ((float*)p.out)[at + f] = p.residual ? y + ((const float*)p.residual)[at + f] : y;
          else ((__nv_bfloat16*)p.out)[at + f] = __float2bfloat16(p.residual ? y + __bfloat162float(((const __nv_bfloat16*)p.residual)[at + f]) : y);
        }
      }
    }
  }
}

template <int NT, int GP, bool ZERO, bool PAIR, int WK>
static int launch_rows(const Int4Rows& p, int E, int tiles, cudaStream_t s) {
  constexpr int UNITS = IR_WARPS / WK;
  return (int)launch_pdl(int4_rows_kernel<NT, GP, ZERO, PAIR, WK>, dim3((p.strips + UNITS - 1) / UNITS, E, tiles), dim3(IR_THREADS), 0, s, p);
}
template <int NT, int GP, bool ZERO>
static int pick_pair(const Int4Rows& p, bool pair, int E, int tiles, cudaStream_t s) {
  return pair ? launch_rows<NT, GP, ZERO, true, 8>(p, E, tiles, s) : launch_rows<NT, GP, ZERO, false, 8>(p, E, tiles, s);
}
template <int NT>
static int pick_group(const Int4Rows& p, int group, bool zero, bool pair, int E, int tiles, cudaStream_t s) {
  if (group == 128) return zero ? pick_pair<NT, 1, true>(p, pair, E, tiles, s) : pick_pair<NT, 1, false>(p, pair, E, tiles, s);
  if (group == 64) return zero ? pick_pair<NT, 2, true>(p, pair, E, tiles, s) : pick_pair<NT, 2, false>(p, pair, E, tiles, s);
  return zero ? pick_pair<NT, 4, true>(p, pair, E, tiles, s) : pick_pair<NT, 4, false>(p, pair, E, tiles, s);
}

}  // namespace skein

// x [x_rows, x_ld] bf16 (row r of the product reads row src_row[r], or r); w as in int4.cuh; out and residual [rows, out_ld] bf16
// or fp32. counts / offsets null: one matrix for all rows. tiles: tiles of rows that an expert's CTAs are dealt over (each walks its share).
// flags: 1 pair, 2 fp16 scales, 4 fp32 output, 8 zeros.
extern "C" int skein_int4_rows(const void* x, long long x_ld, const int* src_row, const void* w, const void* residual, void* out, long long out_ld, const int* counts, const int* offsets, int rows, int x_rows,
                               int E, int F, int K, int group, int rows_hint, int flags, int* status, void* stream) {
  using namespace skein;
  if (rows == 0) return 0;
  if (rows < 0 || E < 1 || E > 65535 || F < 1 || K < 32 || K % group != 0 || (group != 32 && group != 64 && group != 128)) return -1;
  Int4Rows p;
  p.x = (const __nv_bfloat16*)x; p.src_row = src_row; p.w = (const uint8_t*)w; p.residual = residual; p.out = out; p.counts = counts; p.offsets = offsets; p.status = status;
  p.x_ld = x_ld; p.out_ld = out_ld; p.rows = rows; p.x_rows = x_rows; p.F = F; p.K = K;
  const bool pair = flags & 1;
  p.strips = pair ? (F + 7) / 8 : (F + 15) / 16;
  p.steps = (K + I4_STEP - 1) / I4_STEP;
  p.scale_half = (flags >> 1) & 1; p.out_f32 = (flags >> 2) & 1;
  p.vec = x_ld % 8 == 0 && (uintptr_t)x % 16 == 0;
  const int per = rows_hint < 1 ? 1 : rows_hint;
  const int nt = per <= 8 ? 1 : 2;
  int tiles = (per + 8 * nt - 1) / (8 * nt);
  if (tiles > 65535) tiles = 65535;
  cudaStream_t s = (cudaStream_t)stream;
  return nt == 1 ? pick_group<1>(p, group, flags & 8, pair, E, tiles, s) : pick_group<2>(p, group, flags & 8, pair, E, tiles, s);
}
