// Choice of experts by scores with a bias that balances their load, and the expert-sorted layout of the chosen (token, slot) pairs.
//
//   s = sigmoid(z) or softmax(z) of a token's logits;   c = s + bias
//   worth of a group of neighbouring experts = the sum of its best one or two c; the `keep` best groups are eligible
//   the `top` largest c among them are chosen (ties to the lower index, of groups too), with weights scale * s / (sum of the chosen s + 1e-20)
//
// The bias steers the choice only. Scores are 64-bit: the choices of a step decide which rows meet which weights, and experts whose scores differ by
// less than the error of a 32-bit exponential would be chosen by the build that computes them (with 256 experts one token in about 3000). A GPU of
// this kind has the 64-bit rate for it. A logit that is not a number counts as the lowest; logits and biases are clamped to +-3e38, so that no
// input makes an index invalid. (Compiled without fast-math, which would take subnormal biases and weights for zero.)
//
// A warp owns a token. Choices are kept as ordered 64-bit integers, all bits of them; a lane sorts its own with their places beside them, and a round of the
// choice is a maximum over the lanes' heads: one instruction on the upper halves, two more where several lanes have the largest, and a minimum of the
// places where they are equal. Without the order a round compared all of them again (4096 tokens, 256 experts:
// 3250 instructions per token, 35 us). The layout is a counting sort that keeps the tokens' order: for every expert a CTA has one bit per token of its
// tile, so that a pair's place among the tile's is a count of bits, whatever order the warps came in. Up to 256 tokens the tiles are the CTAs of one
// cluster, which add their counts up in distributed shared memory; beyond, the first kernel leaves the tiles' counts in memory and a second one
// finishes the places. One token takes 6.7 us with 128 experts, 64 tokens 7.2 with 64, 12.7 with 256 and 19.5 with 512, 4096 tokens of 256 26.1.
// What bounds it. A token of 256 experts is about 2250 instructions of its warp (2500 in a cluster). With 64 tokens they wait for one another, 11.7 cycles each,
// with two warps on a scheduler: the chain is the time. With 4096 the eight warps of a scheduler fill 57 % of its issue slots (64 registers a thread allow
// no more of them), which is 10 to 15 us; the second kernel, whose CTAs read all tiles' counts, waits for memory for most of the rest (31 of 39 cycles per
// instruction), in part behind the first.
#include "launch.cuh"
#include "ptx.cuh"
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <math.h>

namespace skein {

constexpr int RB_MAX_E = 512, RB_MAX_TOP = 16, RB_MAX_GROUPS = 64;
constexpr int RB_CLUSTER = 8, RB_CLUSTER_TOKENS = 256;
constexpr int RB_TILE = 32;              // tokens of a tile at least: a warp each
constexpr int RB_MAX_TILES = 148;        // (every CTA of the second kernel reads all tiles' counts: 4096 tokens of 256 experts in 256 tiles took 36 us, in 128 28)
constexpr int RB_MAX_WORDS = 48;

struct RouteBalanced {
  const void* logits;
  const float* bias;
  int* ids;
  float* w;
  int *counts, *offsets, *row_of, *src_token;
  uint16_t* tile_counts;   // [tiles][E, rounded up to an even number]
  long long ld;
  uint32_t per_inverse;    // 2^32 over the experts of a group, rounded up: e * per_inverse >> 32 is the group of e < 512 (more than one of them)
  int T, E, top, groups, keep, group_best, renorm, sigmoid, bf16, e_first, e_count, per_tile, tiles;
  float scale;
};

// order of doubles as order of unsigned integers
__device__ __forceinline__ unsigned long long rb_key(double v) {
  const long long b = __double_as_longlong(v);
  return (unsigned long long)b ^ (b < 0 ? ~0ull : 1ull << 63);
}
// (fmaxf gives its other operand for one that is not a number)
__device__ __forceinline__ float rb_clamp(float v) { return fminf(fmaxf(v, -3e38f), 3e38f); }
__device__ __forceinline__ double rb_max(double a, double b) { return a > b ? a : b; }
__device__ __forceinline__ double rb_min(double a, double b) { return a > b ? b : a; }

// The lane whose key is the largest; of several the one with the lowest place, of those the lowest lane.
__device__ __forceinline__ int rb_first(unsigned long long key, unsigned place) {
  const unsigned hi = (unsigned)(key >> 32), mh = __reduce_max_sync(0xffffffffu, hi);
  unsigned who = __ballot_sync(0xffffffffu, hi == mh);
  if (who & (who - 1)) {
    const unsigned lo = hi == mh ? (unsigned)key : 0u, ml = __reduce_max_sync(0xffffffffu, lo);
    const bool in = hi == mh && lo == ml;
    who = __ballot_sync(0xffffffffu, in);
    if (who & (who - 1)) {
      const unsigned at = in ? place : ~0u, first = __reduce_min_sync(0xffffffffu, at);
      who = __ballot_sync(0xffffffffu, in && at == first);
    }
  }
  return __ffs(who) - 1;
}
// Descending order of N (a power of two) keys, equal ones by their places: Batcher's odd-even merges, which have fewer exchanges than bitonic ones (19 for 24
// with 8 keys, 63 for 80 with 16).
template <int N>
__device__ __forceinline__ void rb_sort(unsigned long long (&k)[N], unsigned (&place)[N]) {
#pragma unroll
  for (int run = 1; run < N; run *= 2)
#pragma unroll
    for (int hop = run; hop > 0; hop /= 2)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int j = i + hop;
        if (i < hop % run || ((i - hop % run) & hop) || j >= N || i / (2 * run) != j / (2 * run)) continue;
        const bool turn = k[j] > k[i] || (k[j] == k[i] && place[j] < place[i]);
        const unsigned long long a = turn ? k[j] : k[i], b = turn ? k[i] : k[j];
        const unsigned c = turn ? place[j] : place[i], d = turn ? place[i] : place[j];
        k[i] = a;
        k[j] = b;
        place[i] = c;
        place[j] = d;
      }
}

__device__ __forceinline__ double rb_logit(const RouteBalanced& p, int t, int e) {
  const size_t at = (size_t)t * p.ld + e;
  return (double)rb_clamp(p.bf16 ? __bfloat162float(((const __nv_bfloat16*)p.logits)[at]) : ((const float*)p.logits)[at]);
}

// A warp's token: ids and weights to global memory, the tile's bit of every chosen expert. pool: 32 PER doubles of this warp.
template <int PER>
__device__ __forceinline__ void rb_token(const RouteBalanced& p, int t, int slot, double* pool, uint32_t* masks, int words) {
  const int lane = threadIdx.x & 31;
  double s[PER], mx = (double)-3e38f, den = 1.0;
  unsigned long long key[PER];
#pragma unroll
  for (int q = 0; q < PER; ++q) {
    const int e = q * 32 + lane;
    s[q] = e < p.E ? rb_logit(p, t, e) : (double)-3e38f;
    mx = rb_max(mx, s[q]);
  }
  if (p.sigmoid) {
#pragma unroll
    for (int q = 0; q < PER; ++q) s[q] = 1.0 / (1.0 + exp(-s[q]));
  } else {
    for (int o = 16; o > 0; o >>= 1) mx = rb_max(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    den = 0.0;
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
    key[q] = 0ull;
    if (e < p.E) {
      const double c = p.bias != nullptr ? s[q] + (double)rb_clamp(p.bias[e]) : s[q];
      key[q] = rb_key(c);
      if (p.keep < p.groups) pool[e] = c;
    }
  }
  if (p.keep < p.groups) {
    __syncwarp();
    const int per = p.E / p.groups;
    unsigned long long worth[RB_MAX_GROUPS / 32], kept = 0;
    worth[0] = worth[1] = 0ull;
    // Lanes of a group: as many as there are for all groups. They take its members in turn, each group from another place on (neighbouring groups begin in
    // the same bank), and join their two best.
    int share_log = 5;
    while (share_log > 0 && p.groups << share_log > 32) --share_log;
    const int share = 1 << share_log;
    const int sub = lane & (share - 1), turns = (per + share - 1) >> share_log;
#pragma unroll
    for (int h = 0; h < RB_MAX_GROUPS / 32; ++h) {
      if (h * 32 >= p.groups) break;
      const int grp = h * 32 + (lane >> share_log);
      double b1 = -INFINITY, b2 = -INFINITY;
      if (grp < p.groups) {
        int k = grp % turns;
        for (int n = 0; n < turns; ++n) {
          const int i = k * share + sub;
          if (++k == turns) k = 0;
          const double c = i < per ? pool[grp * per + i] : -INFINITY;
          b2 = rb_max(b2, rb_min(b1, c));
          b1 = rb_max(b1, c);
        }
      }
      for (int o = 1; o < share; o <<= 1) {
        const double c1 = __shfl_xor_sync(0xffffffffu, b1, o), c2 = __shfl_xor_sync(0xffffffffu, b2, o);
        b2 = rb_max(rb_max(b2, c2), rb_min(b1, c1));
        b1 = rb_max(b1, c1);
      }
      // (to lane grp % 32, which owns the group from here on)
      const unsigned long long v = grp < p.groups ? rb_key(p.group_best > 1 && per > 1 ? b1 + b2 : b1) : 0ull;
      const unsigned long long mine = __shfl_sync(0xffffffffu, v, (lane * share) & 31);
      worth[h] = h * 32 + lane < p.groups ? mine : 0ull;
    }
    for (int k = 0; k < p.keep; ++k) {
      // the lower group where two are equal: of a lane's two the first, of several lanes' first ones the lowest before any second one
      const unsigned long long first = worth[0], second = p.groups > 32 ? worth[1] : 0ull;
      const int l = rb_first(first > second ? first : second, 0u);
      const bool up = __shfl_sync(0xffffffffu, first >= second ? 0 : 1, l);
      int got = l + (up ? 32 : 0);
      if (p.groups > 32) {
        const unsigned long long best = __shfl_sync(0xffffffffu, first > second ? first : second, l);
        const unsigned in_first = __ballot_sync(0xffffffffu, first == best);
        if (in_first) got = __ffs(in_first) - 1;
      }
      kept |= 1ull << got;
      if (got == lane) worth[0] = 0ull;
      if (got == lane + 32) worth[1] = 0ull;
    }
#pragma unroll
    for (int q = 0; q < PER; ++q) {
      const int e = q * 32 + lane;
      const int of = per == 1 ? e : (int)__umulhi(e, p.per_inverse);
      if (e < p.E && !((kept >> of) & 1ull)) key[q] = 0ull;
    }
  }
  unsigned place[PER];
#pragma unroll
  for (int q = 0; q < PER; ++q) place[q] = q;
  rb_sort<PER>(key, place);
  unsigned long long places = 0;       // four bits each, in order
#pragma unroll
  for (int q = 0; q < PER; ++q) places |= (unsigned long long)place[q] << (4 * q);
  __syncwarp();                // the pool's choices are read
  unsigned long long* list = reinterpret_cast<unsigned long long*>(pool);
#pragma unroll
  for (int q = 1; q < PER; ++q) list[q * 32 + lane] = key[q];
  unsigned long long head = key[0];
  int next = 1, my_id = 0;
  for (int j = 0; j < p.top; ++j) {
    const unsigned at = (unsigned)places & 15u;
    const int l = rb_first(head, at);
    const int e = (int)__shfl_sync(0xffffffffu, at, l) * 32 + l;
    if (lane == l) {
      head = next < PER ? list[next * 32 + lane] : 0ull;
      places >>= 4;
      ++next;
    }
    if (lane == j) my_id = e;
  }
  // the chosen scores, once more from the logits
  double mine = 0.0;
  if (lane < p.top) {
    const double z = rb_logit(p, t, my_id);
    mine = p.sigmoid ? 1.0 / (1.0 + exp(-z)) : exp(z - mx) / den;
  }
  double sum = mine;
  for (int o = 1; o < RB_MAX_TOP; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane < p.top) {
    const size_t at = (size_t)t * p.top + lane;
    p.ids[at] = my_id;
    p.w[at] = (float)(mine * (double)p.scale / (p.renorm ? sum + 1e-20 : 1.0));
    atomicOr(&masks[my_id * words + (slot >> 5)], 1u << (slot & 31));
  }
  __syncwarp();                // the pool is free for the warp's next token
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
  if (warp < n_tokens) rb_token<PER>(p, t0 + warp, warp, pool + (size_t)warp * PER * 32, masks, 1);
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
__global__ void __launch_bounds__(1024) route_balanced_tile_kernel(const RouteBalanced p) {
  extern __shared__ double pool[];
  const int words = (p.per_tile + 31) / 32, n_warps = blockDim.x >> 5, warp = threadIdx.x >> 5;
  uint32_t* masks = reinterpret_cast<uint32_t*>(pool + (size_t)n_warps * PER * 32);
  const int t0 = blockIdx.x * p.per_tile, n_tokens = max(0, min(p.per_tile, p.T - t0));
  for (int i = threadIdx.x; i < p.E * words; i += blockDim.x) masks[i] = 0u;
  pdl_wait();
  __syncthreads();
  for (int i = warp; i < n_tokens; i += n_warps) rb_token<PER>(p, t0 + i, i, pool + (size_t)warp * PER * 32, masks, words);
  __syncthreads();
  for (int e = threadIdx.x; e < p.E; e += blockDim.x) {
    int c = 0;
    for (int w = 0; w < words; ++w) c += __popc(masks[e * words + w]);
    p.tile_counts[(size_t)blockIdx.x * ((p.E + 1) & ~1) + e] = (uint16_t)(e >= p.e_first && e < p.e_first + p.e_count ? c : 0);
  }
  if ((p.E & 1) && threadIdx.x == 0) p.tile_counts[(size_t)blockIdx.x * (p.E + 1) + p.E] = 0;
  for (int i = threadIdx.x; i < n_tokens * p.top; i += blockDim.x)
    p.row_of[(size_t)t0 * p.top + i] = rb_rank(masks, words, p.ids[(size_t)t0 * p.top + i], i / p.top);
  pdl_trigger();
}

// Second kernel: the tiles' counts become bases, the places become rows.
__global__ void __launch_bounds__(512) route_balanced_place_kernel(const RouteBalanced p) {
  __shared__ int base[RB_MAX_E + 1], total[RB_MAX_E + 1], off[RB_MAX_E + 1];
  const int tile = blockIdx.x, words = (p.E + 1) / 2, parts = blockDim.x / words;      // (at most 256 words)
  for (int e = threadIdx.x; e <= p.E; e += blockDim.x) base[e] = total[e] = 0;
  __syncthreads();
  pdl_wait();
  // two experts per thread, the tiles dealt over the parts of the block
  const int w = threadIdx.x % words, part = threadIdx.x / words;
  if (part < parts) {
    const uint32_t* at = reinterpret_cast<const uint32_t*>(p.tile_counts) + w;
    int before[2] = {0, 0}, all[2] = {0, 0};
#pragma unroll 8
    for (int i = part; i < p.tiles; i += parts) {
      const uint32_t v = at[(size_t)i * words];
      const int lo = (int)(v & 0xffffu), hi = (int)(v >> 16);
      all[0] += lo; all[1] += hi;
      if (i < tile) { before[0] += lo; before[1] += hi; }
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) { atomicAdd(&base[2 * w + k], before[k]); atomicAdd(&total[2 * w + k], all[k]); }
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
  if ((T + per - 1) / per > RB_MAX_TILES) per = (T + RB_MAX_TILES - 1) / RB_MAX_TILES;
  *per_tile = per;
  return (T + per - 1) / per;
}

template <int PER>
static int rb_launch(RouteBalanced p, cudaStream_t s) {
  if (p.T <= RB_CLUSTER_TOKENS) {
    static PerDevice allowed;
    const int n = p.T <= 8 ? 1 : RB_CLUSTER;
    p.per_tile = (p.T + n - 1) / n;
    const size_t smem = (size_t)p.per_tile * PER * 32 * sizeof(double);
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
  const int words = (p.per_tile + 31) / 32, warps = 32;
  const size_t smem = (size_t)warps * PER * 32 * sizeof(double) + (size_t)p.E * words * 4;
  cudaError_t e = allow_smem(allowed, (const void*)route_balanced_tile_kernel<PER>, 32 * PER * 32 * (int)sizeof(double) + PER * 32 * RB_MAX_WORDS * 4);
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
  return per > RB_MAX_WORDS * 32 ? -1 : (long long)tiles * ((E + 1) & ~1) * 2;
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
  RouteBalanced p{logits, bias, ids, w, counts, offsets, row_of, src_token, (uint16_t*)scratch, ld, (uint32_t)((0x100000000ull + E / groups - 1) / (E / groups)), T, E, top, groups, keep, group_best, renorm, sigmoid, bf16,
                  e_first, e_count, 0, 0, scale};
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
