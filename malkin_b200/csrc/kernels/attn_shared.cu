// Attention of a decoding batch whose requests share prefixes, over the int8 cache (mk_attention_shared).
//
// A token's keys are the prefix rows of its group, the first n_keys rows of its own sequence, and its ancestors' rows in
// a draft tree. The prefix part is computed once per group for the rows (tokens x query heads of one KV head) of all its
// requests, so its K and V are read once for up to 128 rows; the own part once per run of tokens with the same sequence.
// Softmax parts are joined from (maximum, sum, unnormalised output) triples in fp32.
//
//   k_shared_plan     one CTA: tiles of at most 128 rows over (group, prefix) and (run, own rows); the blocks of 64 keys of
//                     all (tile, KV head) units form one line that is cut into equal pieces, one per CTA of the next kernel
//   k_shared_attend   two CTAs per SM, each walks its piece: int8 rows to 16-bit tiles in shared memory, S = Q K^T and
//                     O += P V on tcgen05, a partial triple per (unit, piece)
//   k_shared_join     a warp per (token, head): joins its partial triples and the ancestors' few keys
//
// int8 values are exact in both 16-bit types. Row scales of K (with scale and log2 e) multiply the scores, those of V the
// weights. P V is in fp16 whatever q's type: a weight x scale is rounded by 2^-11 of itself (bf16 would lose 2^-8, which is
// what an fp16 output would then be off by). To stay in fp16's range the row's reference exponent is not the largest score
// but that plus the exponent of the block's largest V scale, less 6: products are at most 2^15, and full precision reaches
// down to 2^-20 of the largest. Sums and outputs carry the same reference, so it cancels.
// Bound: HBM for one tile of rows a group (128 rows: 65.5 kFLOP against 264 bytes a key and head, the machine's balance),
// the tensor pipe and the conversion above that.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "kernels.hpp"
#include "tcgen05.cuh"
#include "types16.cuh"

namespace mkb {

namespace {

constexpr int kTileRows = 128;
constexpr int kBlock = 64;         // keys
constexpr int kMinBlocks = 2;      // of a CTA's piece
constexpr int kPlanThreads = 1024;
constexpr int kAttendThreads = 384;  // warpgroups: softmax, conversion, MMA (one thread)
constexpr int kRegsSoftmax = 128, kRegsConvert = 88, kRegsMma = 24;  // sum: 3 x the 80 of the launch
constexpr int kCtasPerSm = 2;
constexpr float kRaiseMax = 8.0f;   // a row's reference is raised when it is to grow by more (exponents of 2)
constexpr float kHeadroom = 6.0f;   // of it below the largest weight x scale
constexpr int kLeastExp = -40;      // of a block's largest V scale: blocks of zeros must not push the sums out of range

struct Tile {
  int32_t t0, nt;      // tokens
  int32_t base, len;   // key rows
  int32_t blocks;      // of 64 keys
  int32_t own;         // 1: each token sees its own n_keys of them
  int64_t first;       // blocks of all KV heads before this tile
  int64_t row;         // first partial row
};
struct PlanHead {
  int32_t tiles;
  int32_t per;       // blocks of a piece
  int64_t total;     // blocks of all units
};

struct SharedWs {  // the workspace's parts
  PlanHead* head;
  Tile* tile;
  int32_t* tok_pre;  // [n] tile of the token's prefix, -1: none
  int32_t* tok_own;  // [n]
  int32_t* group_tile;  // [n_groups]
  float2* ml;        // [rows] reference (exponent of 2), sum
  float* o;          // [rows][D]
  int64_t rows;
  int prefix_tiles;  // room for tiles over prefixes
};

__host__ __device__ inline int64_t pieces_bound(int blocks, int per) { return (blocks + per - 1) / per + 1; }

struct WsLayout {
  int64_t prefix_tiles, tiles, rows, head, tile, pre, own, group, ml, o, bytes;
};
WsLayout ws_layout(int n, int H, int KV, int D, int n_groups, int ctas) {
  const int per_tile = kTileRows / (H / KV);  // tokens
  WsLayout w;
  w.prefix_tiles = n / per_tile + n_groups;  // a group of x tokens has at most x / per_tile + 1
  w.tiles = w.prefix_tiles + n;
  // whole pieces (at most one per CTA and one more) of at most 128 rows, and two part pieces per unit and segment
  w.rows = static_cast<int64_t>(ctas + 1) * kTileRows + 4 * static_cast<int64_t>(n) * H;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t p = at;
    at = (at + bytes + 255) / 256 * 256;
    return p;
  };
  w.head = take(sizeof(PlanHead));
  w.tile = take((w.tiles + 1) * static_cast<int64_t>(sizeof(Tile)));
  w.pre = take(static_cast<int64_t>(n) * 4);
  w.own = take(static_cast<int64_t>(n) * 4);
  w.group = take(static_cast<int64_t>(n_groups) * 4);
  w.ml = take(w.rows * 8);
  w.o = take(w.rows * D * 4);
  w.bytes = at;
  return w;
}

// ---------------- plan ----------------
template <typename V>
__device__ __forceinline__ V block_scan_sum(V v, V* part, V& total) {  // inclusive; part: 33 shared values
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const V y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += y;
  }
  __syncthreads();
  if (lane == 31) part[warp] = v;
  __syncthreads();
  if (warp == 0) {
    V w = part[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const V y = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += y;
    }
    part[lane] = w;
  }
  __syncthreads();
  total = part[31];
  return v + (warp ? part[warp - 1] : V(0));
}

__device__ __forceinline__ int block_scan_max(int v, int* part) {  // inclusive
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v = max(v, y);
  }
  __syncthreads();
  if (lane == 31) part[warp] = v;
  __syncthreads();
  if (warp == 0) {
    int w = part[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w = max(w, y);
    }
    part[lane] = w;
  }
  __syncthreads();
  return warp ? max(v, part[warp - 1]) : v;
}

// Keys of the token in its own sequence, 0 when the table leaves the cache.
__device__ __forceinline__ int own_keys(const SharedArgs& a, int t, bool* bad) {
  const int64_t base = a.kv_base[t], keys = a.n_keys[t];
  if (base < 0 || keys < 0 || base + keys > a.n_rows) {
    if (bad) *bad = true;
    return 0;
  }
  return static_cast<int>(keys);
}

__global__ void __launch_bounds__(kPlanThreads) k_shared_plan(SharedArgs a, SharedWs w, int ctas) {
  __shared__ int part[33];
  __shared__ int64_t part64[33];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int G = a.H / a.KV, per_tile = kTileRows / G;
  bool bad = false;
  for (int t = tid; t < a.n; t += kPlanThreads) w.tok_pre[t] = -1;
  // prefix tiles
  int n_tiles = 0;
  for (int g0 = 0; g0 < a.n_groups; g0 += kPlanThreads) {
    const int g = g0 + tid;
    int lo = 0, hi = 0, base = 0, len = 0;
    if (g < a.n_groups) {
      lo = a.group_off[g];
      hi = a.group_off[g + 1];
      base = a.prefix_base[g];
      len = a.prefix_len[g];
      if (lo < 0 || hi < lo || hi > a.n || base < 0 || len < 0 || static_cast<int64_t>(base) + len > a.n_rows) {
        bad = true;
        lo = hi = len = 0;
      }
    }
    const int tiles = len > 0 ? (hi - lo + per_tile - 1) / per_tile : 0;
    int total;
    const int first = n_tiles + block_scan_sum(tiles, part, total) - tiles;
    if (g < a.n_groups) {
      w.group_tile[g] = tiles > 0 ? first : -1;
      for (int i = 0; i < tiles && first + i < w.prefix_tiles; ++i) {
        Tile& x = w.tile[first + i];
        x.t0 = lo + i * per_tile;
        x.nt = min(per_tile, hi - x.t0);
        x.base = base;
        x.len = len;
        x.own = 0;
      }
    }
    n_tiles += total;
  }
  if (n_tiles > w.prefix_tiles) {  // groups that overlap one another: no result
    for (int t = tid; t < a.n; t += kPlanThreads) w.tok_own[t] = -1;
    if (tid == 0) {
      *w.head = PlanHead{0, 1, 0};
      if (a.status) atomicCAS(a.status, 0, kStatusBadIndex);
    }
    return;
  }
  __syncthreads();
  for (int g = warp; g < a.n_groups; g += kPlanThreads / 32) {
    const int first = w.group_tile[g];
    if (first < 0) continue;
    const int lo = a.group_off[g], hi = a.group_off[g + 1];
    for (int t = lo + lane; t < hi; t += 32) w.tok_pre[t] = first + (t - lo) / per_tile;
  }
  // own tiles: runs of tokens with the same first row, cut every per_tile tokens
  const int own0 = n_tiles;
  int run = 0;
  for (int t0 = 0; t0 < a.n; t0 += kPlanThreads) {
    const int t = t0 + tid;
    const bool in = t < a.n;
    const bool start = in && (t == 0 || a.kv_base[t] != a.kv_base[t - 1]);
    const int from = max(run, block_scan_max(start ? t : 0, part));
    const int cut = in && (t - from) % per_tile == 0 ? 1 : 0;
    int total;
    const int idx = n_tiles + block_scan_sum(cut, part, total) - 1;
    if (in) w.tok_own[t] = idx;
    if (cut) {
      Tile& x = w.tile[idx];
      x.t0 = t;
      x.base = a.kv_base[t];
      x.len = 0;
      x.own = 1;
    }
    n_tiles += total;
    // the last token's run goes on in the next round
    if (tid == kPlanThreads - 1) part[32] = from;
    __syncthreads();
    run = part[32];
    __syncthreads();
  }
  if (tid == 0) w.tile[n_tiles].t0 = a.n;
  __syncthreads();
  for (int t = tid; t < a.n; t += kPlanThreads) {
    const int keys = own_keys(a, t, &bad);
    if (keys > 0) atomicMax(&w.tile[w.tok_own[t]].len, keys);
  }
  __syncthreads();
  // blocks before each tile, then the pieces' length, then partial rows before each tile
  int64_t blocks = 0;
  for (int i0 = 0; i0 < n_tiles; i0 += kPlanThreads) {
    const int i = i0 + tid;
    int64_t mine = 0;
    if (i < n_tiles) {
      Tile& x = w.tile[i];
      if (i >= own0) x.nt = w.tile[i + 1].t0 - x.t0;
      x.blocks = (x.len + kBlock - 1) / kBlock;
      mine = static_cast<int64_t>(x.blocks) * a.KV;
    }
    int64_t total;
    const int64_t incl = block_scan_sum(mine, part64, total);
    if (i < n_tiles) w.tile[i].first = blocks + incl - mine;
    blocks += total;
  }
  const int per = static_cast<int>(max(static_cast<int64_t>(kMinBlocks), (blocks + ctas - 1) / ctas));
  int64_t rows = 0;
  for (int i0 = 0; i0 < n_tiles; i0 += kPlanThreads) {
    const int i = i0 + tid;
    int64_t mine = 0;
    if (i < n_tiles && w.tile[i].blocks > 0)
      mine = pieces_bound(w.tile[i].blocks, per) * a.KV * w.tile[i].nt * G;
    int64_t total;
    const int64_t incl = block_scan_sum(mine, part64, total);
    if (i < n_tiles) w.tile[i].row = rows + incl - mine;
    rows += total;
  }
  if (tid == 0) *w.head = PlanHead{n_tiles, per, rows <= w.rows ? blocks : 0};
  if (bad && a.status) atomicCAS(a.status, 0, kStatusBadIndex);
}

// ---------------- walk over a CTA's piece ----------------
struct Walk {
  int64_t at, end;  // blocks of the line
  int tile, kv, per;
  Tile x;
  // the current part: blocks b0 .. b1 - 1 of (tile, kv), its partial rows from `row`
  int b0, b1;
  int64_t row;

  __device__ __forceinline__ void part(const SharedArgs& a, int G) {
    const int64_t first = x.first + static_cast<int64_t>(kv) * x.blocks;
    b0 = static_cast<int>(at - first);
    b1 = static_cast<int>(min(static_cast<int64_t>(x.blocks), static_cast<int64_t>(b0) + (end - at)));
    const int64_t p = at / per - first / per;
    row = x.row + (kv * pieces_bound(x.blocks, per) + p) * x.nt * G;
  }
  // One whole warp calls it.
  __device__ __forceinline__ bool begin(const SharedArgs& a, const SharedWs& w, int cta, int G, int lane) {
    const PlanHead h = *w.head;
    per = h.per;
    at = static_cast<int64_t>(cta) * per;
    end = min(h.total, at + per);
    if (at >= end) return false;
    // the last tile that begins at or before `at`: 32 probes a round
    int lo = 0, hi = h.tiles;
    while (hi - lo > 1) {
      const int step = (hi - lo + 31) / 32;
      const int i = lo + lane * step;
      const bool before = i < hi && w.tile[i].first <= at;
      const int k = 31 - __clz(__ballot_sync(0xffffffffu, before));
      lo = lo + k * step;
      hi = min(hi, lo + step);
    }
    tile = lo;
    x = w.tile[tile];
    kv = static_cast<int>((at - x.first) / x.blocks);
    part(a, G);
    return true;
  }
  __device__ __forceinline__ bool next(const SharedArgs& a, const SharedWs& w, int G) {
    at += b1 - b0;
    if (at >= end) return false;
    if (++kv == a.KV) {
      kv = 0;
      do x = w.tile[++tile];
      while (x.blocks == 0);
    }
    part(a, G);
    return true;
  }
};

// ---------------- int8 to 16-bit ----------------
// 4 int8 values -> two words of two 16-bit values, exact.
template <typename T>
__device__ __forceinline__ uint2 widen4(uint32_t w);
template <>
__device__ __forceinline__ uint2 widen4<__half>(uint32_t w) {
  // x + 128 in the low byte of 0x6400 = 1024: the half 1024 + (x + 128), less 1152
  w ^= 0x80808080u;
  const __half2 off = __half2half2(__ushort_as_half(0x6480));
  uint2 r;
  uint32_t lo = __byte_perm(w, 0x64646464u, 0x4140), hi = __byte_perm(w, 0x64646464u, 0x4342);
  __half2 a = __hsub2(*reinterpret_cast<__half2*>(&lo), off), b = __hsub2(*reinterpret_cast<__half2*>(&hi), off);
  r.x = *reinterpret_cast<uint32_t*>(&a);
  r.y = *reinterpret_cast<uint32_t*>(&b);
  return r;
}
template <>
__device__ __forceinline__ uint2 widen4<__nv_bfloat16>(uint32_t w) {
  // 0x4300 = 128 with a step of 1: 128 + (x & 127), less 128 or, with the sign bit (0x4380 = 256), 256
  uint2 r;
  const uint32_t lo = __byte_perm(w, 0, 0x4140), hi = __byte_perm(w, 0, 0x4342);
  uint32_t a = (lo & 0x007F007Fu) | 0x43004300u, b = (lo & 0x00800080u) | 0x43004300u;
  uint32_t c = (hi & 0x007F007Fu) | 0x43004300u, d = (hi & 0x00800080u) | 0x43004300u;
  __nv_bfloat162 x = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
  __nv_bfloat162 y = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&c), *reinterpret_cast<__nv_bfloat162*>(&d));
  r.x = *reinterpret_cast<uint32_t*>(&x);
  r.y = *reinterpret_cast<uint32_t*>(&y);
  return r;
}

template <int D>
struct SharedShape {
  static constexpr int kHalves = D / 64;
  static constexpr int kQHalf = kTileRows * 128;      // bytes of 64 columns of the Q tile
  static constexpr int kKvHalf = kBlock * 128;        // of a K or V tile
  static constexpr int kQ = kHalves * kQHalf, kKv = kHalves * kKvHalf;
  static constexpr int kStages = 2;
  static constexpr int kRing = kQ, kSmall = kQ + kStages * 2 * kKv;
  static constexpr int kTmem = 256;  // columns: S | S | O
};
struct SharedSmall {
  uint64_t q_full, q_empty, full[2], empty[2], s_full[2], p_full[2], pv_done, o_free;
  float ks[2][kBlock];  // K scale x scale x log2 e
  float vs[2][kBlock];
  float vmax[2][2];         // largest finite |V scale| of each half of the block
  uint32_t tmem;
};
template <int D>
constexpr int shared_smem() {
  return SharedShape<D>::kSmall + static_cast<int>(sizeof(SharedSmall));
}

template <typename T, int D>
__global__ void __launch_bounds__(kAttendThreads, kCtasPerSm) k_shared_attend(SharedArgs a, SharedWs w) {
  using S = SharedShape<D>;
  extern __shared__ __align__(1024) uint8_t smem[];
  SharedSmall* sm = reinterpret_cast<SharedSmall*>(smem + S::kSmall);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, G = a.H / a.KV;
  Walk walk;
  if (!walk.begin(a, w, blockIdx.x, G, lane)) return;  // the same for every warp of the block
  if (warp == 8) tmem_alloc(&sm->tmem, S::kTmem);
  if (threadIdx.x == 0) {
    mbar_init(&sm->q_full, 128);
    mbar_init(&sm->q_empty, 1);
    mbar_init(&sm->pv_done, 1);
    mbar_init(&sm->o_free, 4);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sm->full[i], 128);
      mbar_init(&sm->empty[i], 1);
      mbar_init(&sm->s_full[i], 1);
      mbar_init(&sm->p_full[i], 4);
    }
    mbar_fence_init();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm->tmem, tmem_o = tmem + 2 * kBlock;
  int* const st = a.status;
  auto k_tile = [&](int s) { return smem + S::kRing + s * 2 * S::kKv; };
  auto v_tile = [&](int s) { return smem + S::kRing + s * 2 * S::kKv + S::kKv; };

  if (warp < 4) {
    // ---------------- softmax, rescaling, partial results ----------------
    regs_up<kRegsSoftmax>();
    const int row = warp * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>(warp * 32) << 16;
    uint32_t gb = 0;  // blocks of this CTA so far
    bool ok = true;
    do {
      const int rows = walk.x.nt * G;
      const bool on = warp * 32 < rows;
      int limit = 0;  // keys this row sees
      if (row < rows) limit = walk.x.own ? own_keys(a, walk.x.t0 + row / G, nullptr) : walk.x.len;
      float m = -INFINITY, l = 0.0f;
      for (int b = walk.b0; b < walk.b1 && ok; ++b, ++gb) {
        const int s = gb & 1;
        ok = mbar_wait_warp(&sm->s_full[s], (gb >> 1) & 1, st, kStatusTimeout);
        if (!ok) break;
        if (on) {
          tc_fence_after();
          const uint32_t ts = tmem + s * kBlock + lanes;
          float x[kBlock];
          tmem_ld32(ts, *reinterpret_cast<uint32_t(*)[32]>(x));
          tmem_ld32(ts + 32, *reinterpret_cast<uint32_t(*)[32]>(x + 32));
          tmem_wait_ld();
          const float4* ks = reinterpret_cast<const float4*>(sm->ks[s]);
          const float4* vs = reinterpret_cast<const float4*>(sm->vs[s]);
#pragma unroll
          for (int i = 0; i < kBlock / 4; ++i) {
            const float4 k4 = ks[i];
            x[4 * i] *= k4.x, x[4 * i + 1] *= k4.y, x[4 * i + 2] *= k4.z, x[4 * i + 3] *= k4.w;
          }
          const int left = limit - b * kBlock;
          const bool cut = __any_sync(0xffffffffu, left < kBlock);
          if (cut) {
#pragma unroll
            for (int i = 0; i < kBlock; ++i)
              if (i >= left) x[i] = -INFINITY;
          }
          float mx[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
          for (int i = 4; i < kBlock; i += 4) {
#pragma unroll
            for (int e = 0; e < 4; ++e) mx[e] = fmaxf(mx[e], x[i + e]);
          }
          const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
          const float big = fmaxf(sm->vmax[s][0], sm->vmax[s][1]);
          const int e = max(static_cast<int>(__float_as_uint(big) >> 23) - 127, kLeastExp);
          const float want = top + (static_cast<float>(e) - kHeadroom);
          float scale = 1.0f;
          if (want > m && (m == -INFINITY || want - m > kRaiseMax)) {
            scale = ex2_approx(m - want);
            m = want;
          }
          if (b > walk.b0 && __any_sync(0xffffffffu, scale != 1.0f)) {
            ok = mbar_wait_warp(&sm->pv_done, (gb - 1) & 1, st, kStatusTimeout);
            if (!ok) break;
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
              uint32_t v[32];
              tmem_ld32(tmem_o + 32 * c + lanes, v);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * scale);
              tmem_st32(tmem_o + 32 * c + lanes, v);
            }
          }
          const float ref = m == -INFINITY ? 0.0f : m;
          const f2 m2 = f2_make(-ref, -ref);
          f2 sum2 = f2_make(0.0f, 0.0f);
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t p[16];
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
              const float4 v4 = vs[8 * c + i / 2];
              const int j = 32 * c + 2 * i;
              const f2 y0 = f2_add(f2_make(x[j], x[j + 1]), m2), y1 = f2_add(f2_make(x[j + 2], x[j + 3]), m2);
              const f2 e0 = f2_make(ex2_approx(f2_lo(y0)), ex2_approx(f2_hi(y0)));
              const f2 e1 = f2_make(ex2_approx(f2_lo(y1)), ex2_approx(f2_hi(y1)));
              sum2 = f2_add(sum2, f2_add(e0, e1));
              f2 w0 = f2_mul(e0, f2_make(v4.x, v4.y)), w1 = f2_mul(e1, f2_make(v4.z, v4.w));
              if (cut) {  // a masked key's scale may be anything
                w0 = f2_make(j < left ? f2_lo(w0) : 0.0f, j + 1 < left ? f2_hi(w0) : 0.0f);
                w1 = f2_make(j + 2 < left ? f2_lo(w1) : 0.0f, j + 3 < left ? f2_hi(w1) : 0.0f);
              }
              p[i] = pack2<__half>(f2_lo(w0), f2_hi(w0));
              p[i + 1] = pack2<__half>(f2_lo(w1), f2_hi(w1));
            }
            tmem_st16(ts + 16 * c, p);
          }
          l = l * scale + (f2_lo(sum2) + f2_hi(sum2));
          tmem_wait_st();
          tc_fence_before();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm->p_full[s]);
      }
      if (!ok) break;
      ok = mbar_wait_warp(&sm->pv_done, (gb - 1) & 1, st, kStatusTimeout);
      if (!ok) break;
      if (on) {
        tc_fence_after();
        if (row < rows) w.ml[walk.row + row] = make_float2(m, l);
        float* o = w.o + (walk.row + row) * D;
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          uint32_t v[32];
          tmem_ld32(tmem_o + 32 * c + lanes, v);
          tmem_wait_ld();
          if (row < rows) {
#pragma unroll
            for (int i = 0; i < 32; i += 4)
              *reinterpret_cast<uint4*>(o + 32 * c + i) = make_uint4(v[i], v[i + 1], v[i + 2], v[i + 3]);
          }
          __syncwarp();
        }
        tc_fence_before();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm->o_free);
    } while (walk.next(a, w, G));
  } else if (warp < 8) {
    // ---------------- Q, and the cache rows as 16-bit tiles ----------------
    // thread: 16 int8 values (one load) at column block c4 of rows r, r + 32, in both halves of 64 columns. The eight
    // threads of a store phase hold two rows x four blocks, which the swizzle spreads over all banks.
    regs_up<kRegsConvert>();
    const int t = threadIdx.x - 128, c4 = t & 3, r0 = t >> 2;
    constexpr int L = 2 * S::kHalves;  // loads of each of K and V
    const float kscale = a.scale * 1.44269504088896341f;
    uint4 kreg[L], vreg[L];
    float sreg = 0.0f;
    uint32_t gb = 0, part = 0;
    bool ok = true;
    // key rows of a part: the first one's index in the cache planes, and how many there are
    auto first_row = [&]() { return static_cast<int64_t>(walk.kv) * a.n_rows + walk.x.base; };
    auto load_row = [&](const int8_t* p, int64_t row0, int len, int b, int i) {
      const int key = b * kBlock + r0 + 32 * (i & 1);
      if (key >= len) return make_uint4(0, 0, 0, 0);
      return ld_stream16(p + (row0 + key) * D + 64 * (i >> 1) + 16 * c4);
    };
    auto load_scale = [&](int64_t row0, int len, int b) {  // threads 0..63: K, 64..127: V
      const int key = b * kBlock + (t & 63);
      if (key >= len) return 0.0f;
      return t < 64 ? a.ks[row0 + key] * kscale : a.vs[row0 + key];
    };
    auto store_row = [&](uint8_t* tile, int i, uint4 v, auto tag) {
      using E = decltype(tag);
      const int r = r0 + 32 * (i & 1);
      uint8_t* base = tile + (i >> 1) * S::kKvHalf + r * 128;
      const uint2 a0 = widen4<E>(v.x), a1 = widen4<E>(v.y), a2 = widen4<E>(v.z), a3 = widen4<E>(v.w);
      *reinterpret_cast<uint4*>(base + (((2 * c4) ^ (r & 7)) * 16)) = make_uint4(a0.x, a0.y, a1.x, a1.y);
      *reinterpret_cast<uint4*>(base + (((2 * c4 + 1) ^ (r & 7)) * 16)) = make_uint4(a2.x, a2.y, a3.x, a3.y);
    };
    int64_t row0 = first_row();
    int len = walk.x.len;
#pragma unroll
    for (int i = 0; i < L; ++i) {
      kreg[i] = load_row(a.k, row0, len, walk.b0, i);
      vreg[i] = load_row(a.v, row0, len, walk.b0, i);
    }
    sreg = load_scale(row0, len, walk.b0);
    bool more = true;
    while (more && ok) {
      // Q of this part: 128 rows, those without a token are 0
      if (part > 0) ok = mbar_wait_warp(&sm->q_empty, (part - 1) & 1, st, kStatusTimeout);
      if (!ok) break;
      const int rows = walk.x.nt * G;
#pragma unroll 4
      for (int i = t; i < kTileRows * (D / 8); i += 128) {
        const int r = i / (D / 8), c = i % (D / 8);
        uint4 v = make_uint4(0, 0, 0, 0);
        if (r < rows)
          v = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + static_cast<int64_t>(walk.x.t0 + r / G) * a.q_ld +
                                              static_cast<int64_t>(walk.kv * G + r % G) * D + 8 * c);
        *reinterpret_cast<uint4*>(smem + (c / 8) * S::kQHalf + r * 128 + (((c % 8) ^ (r & 7)) * 16)) = v;
      }
      fence_async_smem();
      mbar_arrive(&sm->q_full);
      ++part;
      const int b0 = walk.b0, b1 = walk.b1;
      more = walk.next(a, w, G);
      for (int b = b0; b < b1 && ok; ++b, ++gb) {
        const int s = gb & 1;
        if (gb >= 2) ok = mbar_wait_warp(&sm->empty[s], ((gb >> 1) - 1) & 1, st, kStatusTimeout);
        if (!ok) break;
        int nb = b + 1;  // the next block, whose rows are loaded while this one is stored
        if (nb == b1) {
          nb = walk.b0;
          row0 = first_row();
          len = more ? walk.x.len : 0;
        }
        (t < 64 ? sm->ks[s] : sm->vs[s])[t & 63] = sreg;
        if (t >= 64) {
          const float big = warp_max(fabsf(sreg) < INFINITY ? fabsf(sreg) : 0.0f);
          if (lane == 0) sm->vmax[s][(t - 64) >> 5] = big;
        }
#pragma unroll
        for (int i = 0; i < L; ++i) {
          store_row(k_tile(s), i, kreg[i], T());
          kreg[i] = load_row(a.k, row0, len, nb, i);
        }
#pragma unroll
        for (int i = 0; i < L; ++i) {
          store_row(v_tile(s), i, vreg[i], __half());
          vreg[i] = load_row(a.v, row0, len, nb, i);
        }
        sreg = load_scale(row0, len, nb);
        fence_async_smem();
        mbar_arrive(&sm->full[s]);
      }
    }
  } else {
    regs_down<kRegsMma>();
    if (warp == 8 && lane == 0) {
      // ---------------- MMA ----------------
      constexpr int fmt = std::is_same<T, __half>::value ? 0 : 1;
      constexpr uint32_t id_s = umma_idesc_16(fmt, false, kTileRows, kBlock), id_o = umma_idesc_16(0, true, kTileRows, D);
      auto wait = [&](uint64_t* bar, uint32_t parity) { return mbar_wait(bar, parity & 1, st, kStatusTimeout); };
      auto scores = [&](int s) {
        const uint32_t q = smem_addr(smem), k = smem_addr(k_tile(s));
  #pragma unroll
        for (int d = 0; d < D / 16; ++d)
          tc_mma_f16_ss(tmem + s * kBlock, umma_desc_sw128(q + (d / 4) * S::kQHalf + (d % 4) * 32, 16, 1024),
                        umma_desc_sw128(k + (d / 4) * S::kKvHalf + (d % 4) * 32, 16, 1024), id_s, d > 0);
        tc_commit(&sm->s_full[s]);
      };
      auto values = [&](int s, bool acc) {
        const uint32_t v = smem_addr(v_tile(s));
  #pragma unroll
        for (int k = 0; k < kBlock / 16; ++k)
          tc_mma_f16_ts(tmem_o, tmem + s * kBlock + 8 * k, umma_desc_sw128(v + 2048 * k, S::kKvHalf, 1024), id_o,
                        acc || k > 0);
        tc_commit(&sm->pv_done);
        tc_commit(&sm->empty[s]);
      };
      uint32_t gb = 0, part = 0;
      bool ok = true;
      bool more = true;
      while (more && ok) {
        ok = wait(&sm->q_full, part) && wait(&sm->full[gb & 1], gb >> 1);
        if (!ok) break;
        tc_fence_after();
        scores(gb & 1);
        const int nb = walk.b1 - walk.b0;
        if (nb == 1) tc_commit(&sm->q_empty);
        for (int b = 0; b < nb && ok; ++b, ++gb) {
          if (b + 1 < nb) {
            ok = wait(&sm->full[(gb + 1) & 1], (gb + 1) >> 1);
            if (!ok) break;
            tc_fence_after();
            scores((gb + 1) & 1);
            if (b + 2 == nb) tc_commit(&sm->q_empty);
          }
          if (b == 0 && part > 0) ok = wait(&sm->o_free, part - 1);
          ok = ok && wait(&sm->p_full[gb & 1], gb >> 1);
          if (!ok) break;
          tc_fence_after();
          values(gb & 1, b > 0);
        }
        ++part;
        more = walk.next(a, w, G);
      }
      if (!ok) {  // let what was issued end before TMEM and shared memory go
        tc_commit(&sm->q_empty);
        mbar_wait(&sm->q_empty, 0, nullptr, 0);
        mbar_wait(&sm->q_empty, 1, nullptr, 0);
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 8) tmem_dealloc(tmem, S::kTmem);
}

// ---------------- join ----------------
template <typename T, int D>
__global__ void __launch_bounds__(256) k_shared_join(SharedArgs a, SharedWs w) {
  constexpr int N = D / 32;  // values of a lane
  const int64_t id = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (id >= static_cast<int64_t>(a.n) * a.H) return;
  const int t = static_cast<int>(id / a.H), h = static_cast<int>(id % a.H), G = a.H / a.KV, kv = h / G;
  const PlanHead head = *w.head;
  float m = -INFINITY, l = 0.0f, o[N] = {};
  if (head.total > 0) {
    for (int which = 0; which < 2; ++which) {
      const int i = which ? w.tok_own[t] : w.tok_pre[t];
      if (i < 0) continue;
      const Tile x = w.tile[i];
      if (x.blocks == 0) continue;
      const int64_t first = x.first + static_cast<int64_t>(kv) * x.blocks;
      const int pieces = static_cast<int>((first + x.blocks - 1) / head.per - first / head.per) + 1;
      const int64_t rows = static_cast<int64_t>(x.nt) * G;
      const int64_t r0 = x.row + kv * pieces_bound(x.blocks, head.per) * rows + (t - x.t0) * G + h % G;
      for (int p = 0; p < pieces; ++p) {
        const int64_t r = r0 + p * rows;
        const float2 ml = w.ml[r];
        if (ml.x == -INFINITY && ml.y == 0.0f) continue;
        const float top = fmaxf(m, ml.x);
        const float f = ex2_approx(m - top), g = ex2_approx(ml.x - top);
        m = top;
        l = l * f + ml.y * g;
#pragma unroll
        for (int e = 0; e < N; ++e) o[e] = o[e] * f + w.o[r * D + N * lane + e] * g;
      }
    }
  }
  // ancestors
  if (a.anc_off) {
    const int lo = a.anc_off[t], hi = a.anc_off[t + 1];
    const int64_t base = a.kv_base[t];
    bool bad = lo < 0 || hi < lo || hi > a.n_anc;
    const T* q = static_cast<const T*>(a.q) + static_cast<int64_t>(t) * a.q_ld + static_cast<int64_t>(h) * D + N * lane;
    float qv[N];
#pragma unroll
    for (int e = 0; e < N; ++e) qv[e] = to_float(q[e]);
    for (int i = lo; i < hi && !bad; ++i) {
      const int64_t r = base + a.anc[i];
      if (a.anc[i] < 0 || base < 0 || r >= a.n_rows) {
        bad = true;
        break;
      }
      const int64_t at = static_cast<int64_t>(kv) * a.n_rows + r;
      const int8_t* k = a.k + at * D + N * lane;
      const int8_t* v = a.v + at * D + N * lane;
      float s = 0.0f;
#pragma unroll
      for (int e = 0; e < N; ++e) s += qv[e] * static_cast<float>(k[e]);
      s = warp_sum(s) * (a.ks[at] * (a.scale * 1.44269504088896341f));
      const float top = fmaxf(m, s);
      const float f = m == -INFINITY ? 0.0f : ex2_approx(m - top), g = ex2_approx(s - top);
      m = top;
      l = l * f + g;
      const float gv = g * a.vs[at];
#pragma unroll
      for (int e = 0; e < N; ++e) o[e] = o[e] * f + gv * static_cast<float>(v[e]);
    }
    if (bad && lane == 0 && a.status) atomicCAS(a.status, 0, kStatusBadIndex);
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // no key at all: zeros
  T* out = static_cast<T*>(a.out) + static_cast<int64_t>(t) * a.out_ld + static_cast<int64_t>(h) * D + N * lane;
#pragma unroll
  for (int e = 0; e < N; e += 2) *reinterpret_cast<uint32_t*>(out + e) = pack2<T>(o[e] * inv, o[e + 1] * inv);
}

template <typename T, int D>
int run_shared(const SharedArgs& a, void* ws, int sms, cudaStream_t s) {
  static bool set[kMaxDevices] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= kMaxDevices) return cudaErrorInvalidDevice;
  if (!set[dev]) {
    e = cudaFuncSetAttribute(k_shared_attend<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, shared_smem<D>());
    if (e != cudaSuccess) return e;
    // the warpgroups' register shares come out of the launch's
    cudaFuncAttributes at;
    e = cudaFuncGetAttributes(&at, k_shared_attend<T, D>);
    if (e != cudaSuccess) return e;
    if (at.numRegs * 3 < kRegsSoftmax + kRegsConvert + kRegsMma) return cudaErrorInvalidConfiguration;
    set[dev] = true;
  }
  const int ctas = kCtasPerSm * sms;
  const WsLayout y = ws_layout(a.n, a.H, a.KV, D, a.n_groups, ctas);
  uint8_t* p = static_cast<uint8_t*>(ws);
  SharedWs w{reinterpret_cast<PlanHead*>(p + y.head), reinterpret_cast<Tile*>(p + y.tile),
             reinterpret_cast<int32_t*>(p + y.pre),   reinterpret_cast<int32_t*>(p + y.own),
             reinterpret_cast<int32_t*>(p + y.group), reinterpret_cast<float2*>(p + y.ml),
             reinterpret_cast<float*>(p + y.o),       y.rows,
             static_cast<int>(y.prefix_tiles)};
  k_shared_plan<<<1, kPlanThreads, 0, s>>>(a, w, ctas);
  k_shared_attend<T, D><<<ctas, kAttendThreads, shared_smem<D>(), s>>>(a, w);
  const int64_t warps = static_cast<int64_t>(a.n) * a.H;
  k_shared_join<T, D><<<static_cast<unsigned>((warps + 7) / 8), 256, 0, s>>>(a, w);
  return cudaGetLastError();
}

}  // namespace

int64_t attention_shared_workspace(int n, int H, int KV, int D, int n_groups, int sms) {
  return ws_layout(n, H, KV, D, n_groups, kCtasPerSm * sms).bytes;
}

int launch_attention_shared(const SharedArgs& a, ActType type, int D, void* ws, int sms, cudaStream_t s) {
  if (a.n <= 0) return cudaSuccess;
  if (type == ActType::f16) return D == 64 ? run_shared<__half, 64>(a, ws, sms, s) : run_shared<__half, 128>(a, ws, sms, s);
  return D == 64 ? run_shared<__nv_bfloat16, 64>(a, ws, sms, s) : run_shared<__nv_bfloat16, 128>(a, ws, sms, s);
}

}  // namespace mkb
