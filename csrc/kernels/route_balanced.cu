// Choice of experts by scores with a bias that balances their load, and the expert-sorted layout of the chosen (token, slot) pairs.
//
//   s = sigmoid(z) or softmax(z) of a token's logits;   c = s + bias
//   worth of a group of neighbouring experts = the sum of its best one or two c; the `keep` best groups are eligible
//   the `top` largest c among them are chosen (ties to the lower index, of groups too), with weights scale * s / (sum of the chosen s + 1e-20)
//
// The bias steers the choice only. Scores are 64-bit: the choices of a step decide which rows meet which weights, and experts whose scores differ by
// less than the error of a 32-bit exponential would be chosen by the build that computes them (with 256 experts one token in about 3000). A GPU of
// this kind has the 64-bit rate for it. A logit that is not a number counts as the lowest; logits and choices are clamped to +-3e38, so that no
// input makes an index invalid.
//
// A warp owns a token; choices are kept as ordered 64-bit integers, a round of the choice is a maximum over the lanes' upper halves (one instruction)
// and, where several lanes have it, over the lower halves and indices. The layout is a counting sort that keeps the tokens' order: for every
// expert a CTA has one bit per token of its tile, so that a pair's place among the tile's is a count of bits, whatever order the warps came in.
// Up to 256 tokens the tiles are the CTAs of one cluster, which add their counts up in distributed shared memory; beyond, the first
// kernel leaves the tiles' counts in memory and a second one finishes the places.
#include "launch.cuh"
#include "ptx.cuh"
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <math.h>

namespace skein {

constexpr int RB_MAX_E = 512, RB_MAX_TOP = 16, RB_MAX_GROUPS = 64;
constexpr int RB_CLUSTER = 8, RB_CLUSTER_TOKENS = 256;
constexpr int RB_TILE = 32;              // tokens of a tile at least (a word of the bit masks)
constexpr int RB_MAX_TILES = 256;
constexpr int RB_MAX_WORDS = 48;

struct RouteBalanced {
  const void* logits;
  const float* bias;
  int* ids;
  float* w;
  int *counts, *offsets, *row_of, *src_token;
  uint16_t* tile_counts;   // [E][tiles_ld]
  long long ld;
  int T, E, top, groups, keep, group_best, renorm, sigmoid, bf16, e_first, e_count, per_tile, tiles, tiles_ld;
  float scale;
};

// order of doubles as order of unsigned integers
__device__ __forceinline__ unsigned long long rb_key(double v) {
  const long long b = __double_as_longlong(v);
  return (unsigned long long)b ^ (b < 0 ? ~0ull : 1ull << 63);
}
__device__ __forceinline__ double rb_clamp(double v) { return v != v ? -3e38 : fmin(fmax(v, -3e38), 3e38); }

// The lane whose key is the largest, ties to the lowest index; idx of the winner on every lane (keys of 0 are no candidates).
__device__ __forceinline__ int rb_argmax(unsigned long long key, int idx) {
  const unsigned hi = (unsigned)(key >> 32);
  const unsigned mh = __reduce_max_sync(0xffffffffu, hi);
  unsigned who = __ballot_sync(0xffffffffu, hi == mh);
  if (who & (who - 1)) {
    const unsigned lo = hi == mh ? (unsigned)key : 0u;
    const unsigned ml = __reduce_max_sync(0xffffffffu, lo);
    return (int)__reduce_min_sync(0xffffffffu, hi == mh && lo == ml ? (unsigned)idx : 0x7fffffffu);
  }
  return __shfl_sync(0xffffffffu, idx, __ffs(who) - 1);
}

// A warp's token: ids and weights to global memory, the tile's bit of every chosen expert. pool: E doubles of this warp.
template <int PER>
__device__ __forceinline__ void rb_token(const RouteBalanced& p, int t, int slot, double* pool, uint32_t* masks, int words) {
  const int lane = threadIdx.x & 31;
  double s[PER], mx = -3e38;
  unsigned long long key[PER];
#pragma unroll
  for (int q = 0; q < PER; ++q) {
    const int e = q * 32 + lane;
    s[q] = 0.0;
    if (e < p.E) {
      const size_t at = (size_t)t * p.ld + e;
      const float z = p.bf16 ? __bfloat162float(((const __nv_bfloat16*)p.logits)[at]) : ((const float*)p.logits)[at];
      s[q] = rb_clamp((double)z);
      mx = fmax(mx, s[q]);
    }
  }
  if (p.sigmoid) {
#pragma unroll
    for (int q = 0; q < PER; ++q) s[q] = 1.0 / (1.0 + exp(-s[q]));
  } else {
    for (int o = 16; o > 0; o >>= 1) mx = fmax(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    double den = 0.0;
#pragma unroll
    for (int q = 0; q < PER; ++q) {
      s[q] = q * 32 + lane < p.E ? exp(s[q] - mx) : 0.0;
      den += s[q];
    }
    for (int o = 16; o > 0; o >>= 1) den += __shfl_xor_sync(0xffffffffu, den, o);
#pragma unroll
    for (int q = 0; q < PER; ++q) s[q] /= den;
  }
#pragma unroll
  for (int q = 0; q < PER; ++q) {
    const int e = q * 32 + lane;
    const double c = e < p.E ? rb_clamp(p.bias != nullptr ? s[q] + (double)p.bias[e] : s[q]) : 0.0;
    key[q] = e < p.E ? rb_key(c) : 0ull;
    if (p.keep < p.groups && e < p.E) pool[e] = c;
  }
  if (p.keep < p.groups) {
    __syncwarp();
    const int per = p.E / p.groups;
    unsigned long long worth[RB_MAX_GROUPS / 32], kept = 0;
#pragma unroll
    for (int h = 0; h < RB_MAX_GROUPS / 32; ++h) {
      const int grp = h * 32 + lane;
      worth[h] = 0ull;
      if (grp < p.groups) {
        double b1 = -INFINITY, b2 = -INFINITY;
        for (int i = 0; i < per; ++i) {
          const double c = pool[grp * per + i];
          if (c > b1) { b2 = b1; b1 = c; }
          else if (c > b2) b2 = c;
        }
        worth[h] = rb_key(p.group_best > 1 && per > 1 ? b1 + b2 : b1);
      }
    }
    for (int k = 0; k < p.keep; ++k) {
      const bool up = p.groups > 32 && worth[1] > worth[0];       // the lower group where both are equal
      const int got = rb_argmax(up ? worth[1] : worth[0], up ? 32 + lane : lane);
      kept |= 1ull << got;
      if ((got & 31) == lane) worth[got >> 5] = 0ull;
    }
#pragma unroll
    for (int q = 0; q < PER; ++q) {
      const int e = q * 32 + lane;
      if (e < p.E && !((kept >> (e / per)) & 1ull)) key[q] = 0ull;
    }
    __syncwarp();                // the pool is free for the warp's next token
  }
  int my_id = 0;
  double my_s = 0.0, sum = 0.0;
  for (int j = 0; j < p.top; ++j) {
    unsigned long long best = key[0];
    int bq = 0;
#pragma unroll
    for (int q = 1; q < PER; ++q) if (key[q] > best) { best = key[q]; bq = q; }
    const int e = rb_argmax(best, bq * 32 + lane);
    double mine = 0.0;
#pragma unroll
    for (int q = 0; q < PER; ++q) if (q * 32 + lane == e) { mine = s[q]; key[q] = 0ull; }
    const double got = __shfl_sync(0xffffffffu, mine, e & 31);
    sum += got;
    if (lane == j) { my_id = e; my_s = got; }
  }
  if (lane < p.top) {
    const size_t at = (size_t)t * p.top + lane;
    p.ids[at] = my_id;
    p.w[at] = (float)(my_s * (double)p.scale / (p.renorm ? sum + 1e-20 : 1.0));
    atomicOr(&masks[my_id * words + (slot >> 5)], 1u << (slot & 31));
  }
}

// Exclusive sums of total[0 .. E) into off[0 .. E], by the first warp.
__device__ __forceinline__ void rb_scan(const int* total, int* off, int E) {
  const int lane = threadIdx.x & 31;
  int run = 0;
  for (int e0 = 0; e0 < E; e0 += 32) {
    const int v = e0 + lane < E ? total[e0 + lane] : 0;
    int inc = v;
    for (int o = 1; o < 32; o <<= 1) { const int u = __shfl_up_sync(0xffffffffu, inc, o); if (lane >= o) inc += u; }
    if (e0 + lane < E) off[e0 + lane] = run + inc - v;
    run += __shfl_sync(0xffffffffu, inc, 31);
  }
  if (lane == 0) off[E] = run;
}

__device__ __forceinline__ int rb_rank(const uint32_t* masks, int words, int e, int slot) {
  int r = __popc(masks[e * words + (slot >> 5)] & ((1u << (slot & 31)) - 1u));
  for (int w = 0; w < (slot >> 5); ++w) r += __popc(masks[e * words + w]);
  return r;
}

// Places of a tile's pairs: base[e] is the first row of its pairs of expert e.
__device__ __forceinline__ void rb_place(const RouteBalanced& p, int t0, int n_tokens, const uint32_t* masks, int words, const int* base) {
  for (int i = threadIdx.x; i < n_tokens * p.top; i += blockDim.x) {
    const int slot = i / p.top, e = p.ids[(size_t)t0 * p.top + i];
    const bool mine = e >= p.e_first && e < p.e_first + p.e_count;
    const int row = mine ? base[e] + rb_rank(masks, words, e, slot) : -1;
    p.row_of[(size_t)t0 * p.top + i] = row;
    if (mine) p.src_token[row] = t0 + slot;
  }
}

// One cluster (or one CTA): every CTA a tile of at most 32 tokens, a warp per token. Dynamic shared memory: the warps' pools.
template <int PER>
__global__ void __launch_bounds__(1024) route_balanced_cluster_kernel(const RouteBalanced p) {
  namespace cg = cooperative_groups;
  extern __shared__ double pool[];
  __shared__ uint32_t masks[RB_MAX_E];
  __shared__ int cnt[RB_MAX_E], base[RB_MAX_E], total[RB_MAX_E], off[RB_MAX_E + 1];
  cg::cluster_group cluster = cg::this_cluster();
  const int n = gridDim.x, rank = blockIdx.x, t0 = rank * p.per_tile, warp = threadIdx.x >> 5;
  const int n_tokens = max(0, min(p.per_tile, p.T - t0));
  for (int e = threadIdx.x; e < p.E; e += blockDim.x) masks[e] = 0u;
  pdl_trigger();
  pdl_wait();
  __syncthreads();
  if (warp < n_tokens) rb_token<PER>(p, t0 + warp, warp, pool + (size_t)warp * p.E, masks, 1);
  __syncthreads();
  for (int e = threadIdx.x; e < p.E; e += blockDim.x) cnt[e] = e >= p.e_first && e < p.e_first + p.e_count ? __popc(masks[e]) : 0;
  if (n > 1) cluster.sync(); else __syncthreads();
  for (int e = threadIdx.x; e < p.E; e += blockDim.x) {
    int before = 0, all = 0;
    for (int c = 0; c < n; ++c) {
      const int v = n > 1 ? cluster.map_shared_rank(cnt, c)[e] : cnt[e];
      before += c < rank ? v : 0;
      all += v;
    }
    base[e] = before;
    total[e] = all;
  }
  __syncthreads();
  if (warp == 0) rb_scan(total, off, p.E);
  __syncthreads();
  for (int e = threadIdx.x; e < p.E; e += blockDim.x) {
    base[e] += off[e];
    if (rank == 0) { p.counts[e] = total[e]; p.offsets[e] = off[e]; }
  }
  if (rank == 0 && threadIdx.x == 0) p.offsets[p.E] = off[p.E];
  __syncthreads();
  rb_place(p, t0, n_tokens, masks, 1, base);
  if (n > 1) cluster.sync();      // nobody leaves while its counts are read
}

// Many tokens, first kernel: the choices of a tile, its counts and, in row_of, the pairs' places among the tile's.
template <int PER>
__global__ void __launch_bounds__(512) route_balanced_tile_kernel(const RouteBalanced p) {
  extern __shared__ double pool[];
  const int words = (p.per_tile + 31) / 32, n_warps = blockDim.x >> 5, warp = threadIdx.x >> 5;
  uint32_t* masks = reinterpret_cast<uint32_t*>(pool + (size_t)n_warps * p.E);
  const int t0 = blockIdx.x * p.per_tile, n_tokens = max(0, min(p.per_tile, p.T - t0));
  for (int i = threadIdx.x; i < p.E * words; i += blockDim.x) masks[i] = 0u;
  pdl_wait();
  __syncthreads();
  for (int i = warp; i < n_tokens; i += n_warps) rb_token<PER>(p, t0 + i, i, pool + (size_t)warp * p.E, masks, words);
  __syncthreads();
  for (int e = threadIdx.x; e < p.E; e += blockDim.x) {
    int c = 0;
    for (int w = 0; w < words; ++w) c += __popc(masks[e * words + w]);
    p.tile_counts[(size_t)e * p.tiles_ld + blockIdx.x] = (uint16_t)(e >= p.e_first && e < p.e_first + p.e_count ? c : 0);
  }
  for (int i = threadIdx.x; i < n_tokens * p.top; i += blockDim.x)
    p.row_of[(size_t)t0 * p.top + i] = rb_rank(masks, words, p.ids[(size_t)t0 * p.top + i], i / p.top);
  pdl_trigger();
}

// Second kernel: the tiles' counts become bases, the places become rows.
__global__ void __launch_bounds__(512) route_balanced_place_kernel(const RouteBalanced p) {
  __shared__ int base[RB_MAX_E], total[RB_MAX_E], off[RB_MAX_E + 1];
  pdl_wait();
  const int tile = blockIdx.x;
  for (int e = threadIdx.x; e < p.E; e += blockDim.x) {
    const uint4* row = reinterpret_cast<const uint4*>(p.tile_counts + (size_t)e * p.tiles_ld);   // eight tiles each
    int before = 0, all = 0;
    for (int b = 0; b * 8 < p.tiles; ++b) {
      const uint4 v = row[b];
      const uint32_t r[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int at = b * 8 + i;
        const int c = at < p.tiles ? (int)((r[i >> 1] >> (16 * (i & 1))) & 0xffffu) : 0;
        before += at < tile ? c : 0;
        all += c;
      }
    }
    base[e] = before;
    total[e] = all;
  }
  __syncthreads();
  if (threadIdx.x < 32) rb_scan(total, off, p.E);
  __syncthreads();
  for (int e = threadIdx.x; e < p.E; e += blockDim.x) {
    base[e] += off[e];
    if (tile == 0) { p.counts[e] = total[e]; p.offsets[e] = off[e]; }
  }
  if (tile == 0 && threadIdx.x == 0) p.offsets[p.E] = off[p.E];
  __syncthreads();
  const int t0 = tile * p.per_tile, n_tokens = max(0, min(p.per_tile, p.T - t0));
  for (int i = threadIdx.x; i < n_tokens * p.top; i += blockDim.x) {
    const size_t at = (size_t)t0 * p.top + i;
    const int e = p.ids[at];
    const bool mine = e >= p.e_first && e < p.e_first + p.e_count;
    const int row = mine ? base[e] + p.row_of[at] : -1;
    p.row_of[at] = row;
    if (mine) p.src_token[row] = t0 + i / p.top;
  }
}

__global__ void route_balanced_empty_kernel(const RouteBalanced p) {
  for (int e = threadIdx.x; e <= p.E; e += blockDim.x) { p.offsets[e] = 0; if (e < p.E) p.counts[e] = 0; }
}

static int rb_tiles(int T, int* per_tile) {
  int per = RB_TILE;
  if ((T + per - 1) / per > RB_MAX_TILES) per = ((T + RB_MAX_TILES - 1) / RB_MAX_TILES + 31) / 32 * 32;
  *per_tile = per;
  return (T + per - 1) / per;
}

template <int PER>
static int rb_launch(RouteBalanced p, cudaStream_t s) {
  if (p.T <= RB_CLUSTER_TOKENS) {
    static PerDevice allowed;
    const int n = p.T <= 8 ? 1 : RB_CLUSTER;
    p.per_tile = (p.T + n - 1) / n;
    const size_t smem = p.keep < p.groups ? (size_t)p.per_tile * p.E * sizeof(double) : 0;
    if (smem > 36 * 1024) {
      const cudaError_t e = allow_smem(allowed, (const void*)route_balanced_cluster_kernel<PER>, 32 * RB_MAX_E * (int)sizeof(double));
      if (e != cudaSuccess) return (int)e;
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(n);
    cfg.blockDim = dim3(32 * max(p.per_tile, 4));
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = n;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return (int)cudaLaunchKernelEx(&cfg, route_balanced_cluster_kernel<PER>, p);
  }
  static PerDevice allowed;
  p.tiles = rb_tiles(p.T, &p.per_tile);
  p.tiles_ld = (p.tiles + 7) / 8 * 8;
  const int words = (p.per_tile + 31) / 32, warps = 16;
  const size_t smem = (size_t)warps * p.E * sizeof(double) + (size_t)p.E * words * 4;
  cudaError_t e = allow_smem(allowed, (const void*)route_balanced_tile_kernel<PER>, 16 * RB_MAX_E * (int)sizeof(double) + RB_MAX_E * RB_MAX_WORDS * 4);
  if (e != cudaSuccess) return (int)e;
  e = launch_pdl(route_balanced_tile_kernel<PER>, dim3(p.tiles), dim3(32 * warps), smem, s, p);
  if (e != cudaSuccess) return (int)e;
  return (int)launch_pdl_if(true, route_balanced_place_kernel, dim3(p.tiles), dim3(512), 0, s, p);
}

}  // namespace skein

// Bytes of scratch (16-byte aligned) that a call needs; -1 for more tokens than the kernels take.
extern "C" long long skein_route_balanced_scratch(int T, int E) {
  using namespace skein;
  if (T <= RB_CLUSTER_TOKENS) return 0;
  int per;
  const int tiles = rb_tiles(T, &per);
  return per > RB_MAX_WORDS * 32 ? -1 : (long long)E * ((tiles + 7) / 8 * 8) * 2;
}

// logits [T, ld] fp32 or bf16 (bf16 != 0); bias [E] fp32 or null. ids / w [T, top], counts [E], offsets [E + 1], row_of / src_token [T * top].
extern "C" int skein_route_balanced(const void* logits, long long ld, int bf16, const float* bias, int T, int E, int top, int groups, int keep,
                                    int group_best, int renorm, int sigmoid, float scale, int e_first, int e_count, int* ids, float* w, int* counts,
                                    int* offsets, int* row_of, int* src_token, void* scratch, void* stream) {
  using namespace skein;
  if (T < 0 || E < 1 || E > RB_MAX_E || top < 1 || top > RB_MAX_TOP || groups < 1 || groups > RB_MAX_GROUPS || E % groups != 0 || keep < 1 ||
      keep > groups || top > keep * (E / groups) || group_best < 1 || group_best > 2 || e_first < 0 || e_count < 0 || e_first + e_count > E)
    return -1;
  if (skein_route_balanced_scratch(T, E) < 0 || (skein_route_balanced_scratch(T, E) > 0 && scratch == nullptr)) return -2;
  RouteBalanced p{logits, bias, ids, w, counts, offsets, row_of, src_token, (uint16_t*)scratch, ld, T, E, top, groups, keep, group_best, renorm, sigmoid, bf16,
                  e_first, e_count, 0, 0, 0, scale};
  cudaStream_t s = (cudaStream_t)stream;
  if (T == 0) {
    route_balanced_empty_kernel<<<1, 256, 0, s>>>(p);
    return (int)cudaGetLastError();
  }
  if (E <= 64) return rb_launch<2>(p, s);
  if (E <= 128) return rb_launch<4>(p, s);
  if (E <= 256) return rb_launch<8>(p, s);
  return rb_launch<16>(p, s);
}
