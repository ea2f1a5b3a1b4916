// Attention of a decoding batch whose requests share prefixes, over the int8 cache (mk_attention_shared).
//
// A token's keys are the prefix rows of its group, the first n_keys rows of its own sequence, and its ancestors' rows in
// a draft tree. The prefix part is computed once per group for the rows (tokens x query heads of one KV head) of all its
// requests, so its K and V are read once for up to 256 rows; the own part once per run of tokens with the same sequence.
// Softmax parts are joined from (maximum, sum, unnormalised output) triples in fp32.
//
//   k_shared_plan     one CTA: tiles of up to 256 rows over (group, prefix) and (run, own rows); the blocks of 96 keys of
//                     all (tile, KV head) units form one line that is cut into equal pieces, one per CTA of the next kernel
//   k_shared_attend   one CTA per SM walks its piece: int8 rows to fp16 / bf16 tiles in shared memory, S = Q K^T and
//                     O += P V on tcgen05, a partial triple per (unit, piece). Two streams of 128 rows share each converted
//                     block where a tile has more than 128 rows; otherwise they take the blocks in turn
//   k_shared_join     a warp per (token, head): joins its partial triples and the ancestors' few keys
//
// int8 values are exact in both 16-bit types. Row scales of K (with scale and log2 e) multiply the scores, those of V the
// weights. P V is in fp16 whatever q's type: a weight x scale is rounded by 2^-11 of itself (bf16 would lose 2^-8, which is
// what an fp16 output would then be off by). To stay in fp16's range a row's reference exponent is not its largest score but the
// largest sum of a score and the exponent of that key's V scale, over the keys the row sees, less 6: products are at most 2^15,
// and full precision reaches down to 2^-20 of the row's largest. Sums and outputs carry the same reference, so it cancels. Where
// the scales of a block lie within 2^4 of each other, as they do as a rule, the largest stands for each of them: that costs at
// most 4 of those 20 bits and spares the sums (two prefixes of 32768 rows: 257 us, with the sums in every block 263; the block's
// largest scale alone, seen by the row or not, 246, and wrong where scales lie far apart).
// Bound: HBM for one tile of rows a group (128 rows: 65.5 kFLOP against 264 bytes a key and head, the machine's balance),
// the tensor pipe and the conversion above that. What holds it: a block of 96 keys took 3700 cycles for 128 rows and 3900
// for 256 (now some 4 % more), 2500 of them the widening (K to bf16 1700, V to fp16 800); the plan takes 7 us, finding a
// piece's place 2, the join 4 to 5. Measured, with queries of 32 / 8 heads of 128: two prefixes of up to 32768 rows with 32
// requests of 4 rows each, bf16: 257 us; 8 trees of 17 rows behind 2048 rows, fp16: 45; 4 single rows behind 1000, 16 / 8
// heads, bf16: 27. Two CTAs an SM with blocks of 64 keys took 497 us at the first.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <climits>
#include <cstddef>
#include <type_traits>

#include "common.cuh"
#include "kernels.hpp"
#include "pdl.cuh"
#include "tcgen05.cuh"
#include "tensor_map.hpp"
#include "types16.cuh"

namespace mkb {

namespace {

constexpr int kTileRows = 128;     // of a stream
constexpr int kBlock = 96;         // keys: five 16-bit K / V tiles, three int8 ones and both Q tiles fill the shared memory
constexpr int kPlanThreads = 1024;
constexpr int kAttendThreads = 512;  // warpgroups: softmax of stream 0, of stream 1, conversion, MMA and Q
constexpr int kRegsSoftmax = 176, kRegsConvert = 80, kRegsMma = 80;  // 2 x 176 + 80 + 80 = 4 x the 128 of the launch
constexpr float kRaiseMax = 8.0f;   // a row's reference is raised when it is to grow by more (exponents of 2)
constexpr float kHeadroom = 6.0f;   // of it below the largest weight x scale
constexpr int kLeastExp = -40;      // of a V scale: rows of zeros must not push the sums out of range
constexpr int kSpread = 4;          // of a block's exponents, to be taken for one

// Tokens and keys of a unit (with a KV head). Its places on the line: one for each block (a block takes about as long for
// 256 rows as for 128: 3900 and 3700 cycles), after `open` for what a part costs before its first block and after its last.
// Batches of fewer than kFewBlocks blocks a CTA are cut into single blocks instead (open 0).
constexpr int kOpen = 2, kFewBlocks = 4;
struct Tile {
  int32_t t0, nt;      // tokens
  int32_t base, len;   // key rows
  int32_t blocks, places;
  int32_t own;         // 1: each token sees its own n_keys of them
  int32_t dual;        // 1: the streams have different rows
  int64_t first;       // places of all KV heads before this tile
  int64_t row;         // first partial row
};
struct PlanHead {
  int32_t tiles;
  int32_t per;       // places of a piece, more than open
  int64_t total;     // places of all units
  int32_t open;
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

__host__ __device__ inline int64_t pieces_bound(int places, int per) { return (places + per - 1) / per + 1; }

struct WsLayout {
  int64_t prefix_tiles, tiles, rows, head, tile, pre, own, group, ml, o, bytes;
};
WsLayout ws_layout(int n, int H, int KV, int D, int n_groups, int ctas) {
  const int per_tile = 2 * (kTileRows / (H / KV));  // tokens
  WsLayout w;
  w.prefix_tiles = n / per_tile + n_groups;  // a group of x tokens has at most x / per_tile + 1
  w.tiles = w.prefix_tiles + n;
  // whole pieces (at most one per CTA and one more) of at most 256 rows, and two part pieces per unit and segment
  w.rows = static_cast<int64_t>(ctas + 1) * 2 * kTileRows + 4 * static_cast<int64_t>(n) * H;
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

// Inclusive, of values from 0 on; left: without the thread's own.
__device__ __forceinline__ int block_scan_max(int v, int* part, int& left) {
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
  const int before = warp ? part[warp - 1] : 0;
  left = __shfl_up_sync(0xffffffffu, v, 1);
  left = lane ? max(left, before) : before;
  return max(v, before);
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
  pdl_launch();
  __shared__ int part[33];
  __shared__ int64_t part64[33];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int G = a.H / a.KV, half = kTileRows / G, per_tile = 2 * half;
  bool bad = false;
  for (int t = tid; t < a.n; t += kPlanThreads) w.tok_pre[t] = -1;
  // prefix tiles. A group that begins before the end of an earlier one is refused, so that a token is in one group at most and
  // the tiles are no more than there is room for. Offsets that nowhere descend put no token into two groups: only where one is
  // seen to, or there are several rounds of groups, the ends before each are looked at (`careful`, a second time around).
  int n_tiles;
  for (bool careful = a.n_groups > kPlanThreads;; careful = true) {
    bool falls = false;
    int grouped = 0;  // end of the groups before the round
    n_tiles = 0;
    for (int g0 = 0; g0 < a.n_groups; g0 += kPlanThreads) {
      const int g = g0 + tid;
      int lo = 0, hi = 0, base = 0, len = 0;
      if (g < a.n_groups) {
        lo = a.group_off[g];
        hi = a.group_off[g + 1];
        base = a.prefix_base[g];
        len = a.prefix_len[g];
        falls = hi < lo;
        if (lo < 0 || hi < lo || hi > a.n || base < 0 || len < 0 || static_cast<int64_t>(base) + len > a.n_rows) {
          bad = true;
          lo = hi = len = 0;
        }
      }
      if (careful) {
        int before;
        block_scan_max(hi > lo ? hi : 0, part, before);
        if (hi > lo && lo < max(before, grouped)) {
          bad = true;
          hi = lo;
        }
        grouped = max(grouped, part[31]);
      }
      const int tiles = len > 0 ? (hi - lo + per_tile - 1) / per_tile : 0;
      int total;
      const int first = n_tiles + block_scan_sum(tiles, part, total) - tiles;
      if (g < a.n_groups) {
        w.group_tile[g] = tiles > 0 ? first : -1;
        for (int i = 0; i < tiles && first + i < w.prefix_tiles; ++i) {  // all of them, once no token is in two groups
          Tile& x = w.tile[first + i];
          x.t0 = lo + i * per_tile;
          x.nt = min(per_tile, hi - x.t0);
          x.base = base;
          x.len = len;
          x.own = 0;
        }
      }
      n_tiles += total;  // at most 2^29 in a round that is not careful, which is the only one
    }
    if (!__syncthreads_or(falls && !careful)) break;
  }
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
    int left;
    const int from = max(run, block_scan_max(start ? t : 0, part, left));
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
  // places before each tile, then the pieces' length, then partial rows before each tile
  int64_t places = 0, n_units = 0;
  for (int i0 = 0; i0 < n_tiles; i0 += kPlanThreads) {
    const int i = i0 + tid;
    int64_t mine = 0, units = 0;
    if (i < n_tiles) {
      Tile& x = w.tile[i];
      if (i >= own0) x.nt = w.tile[i + 1].t0 - x.t0;
      x.blocks = (x.len + kBlock - 1) / kBlock;
      x.dual = x.nt > half;
      mine = static_cast<int64_t>(x.blocks) * a.KV;
      units = x.blocks > 0 ? a.KV : 0;
    }
    int64_t total;
    const int64_t incl = block_scan_sum(mine, part64, total);
    int64_t opened;
    const int64_t before = block_scan_sum(units, part64, opened);
    if (i < n_tiles) {
      w.tile[i].first = places + incl - mine;
      w.tile[i].row = n_units + before - units;
    }
    places += total;
    n_units += opened;
  }
  const int open = places < static_cast<int64_t>(kFewBlocks) * ctas ? 0 : kOpen;
  places += open * n_units;
  const int64_t longest = max(static_cast<int64_t>(open + 1), (places + ctas - 1) / ctas);
  const bool too_long = longest > INT_MAX;  // hours of work; a piece's places are counted in 32 bits
  const int per = too_long ? 1 : static_cast<int>(longest);
  bad |= too_long;
  int64_t rows = 0;
  for (int i0 = 0; i0 < n_tiles; i0 += kPlanThreads) {
    const int i = i0 + tid;
    int64_t mine = 0;
    if (i < n_tiles) {
      Tile& x = w.tile[i];
      x.first += open * x.row;
      x.places = x.blocks > 0 ? open + x.blocks : 0;
      if (x.blocks > 0) mine = pieces_bound(x.places, per) * a.KV * x.nt * G;
    }
    int64_t total;
    const int64_t incl = block_scan_sum(mine, part64, total);
    if (i < n_tiles) w.tile[i].row = rows + incl - mine;
    rows += total;
  }
  if (tid == 0) *w.head = PlanHead{n_tiles, per, rows <= w.rows && !too_long ? places : 0, open};
  if (bad && a.status) atomicCAS(a.status, 0, kStatusBadIndex);
}

// ---------------- a CTA's piece of the line, part by part ----------------
// One (tile, KV head) unit's share of the piece. One warp walks the plan and hands the parts to the others through a ring in
// shared memory, so that nobody else keeps the walk's state in registers.
struct Part {
  int b0, nb;      // blocks; nb 0: the piece has ended
  int t0, nt;      // tokens
  int len, kv;
  bool own, dual;
  int64_t key0;    // the first key's row in the cache planes
  int64_t row;     // first partial row
};

struct Walk {
  PlanHead h;
  Tile x;                    // the current tile
  int done, tile, kv, span;  // places before the current part, its unit and its places

  // The first part with blocks at or behind `done` (nb 0: none).
  __device__ __forceinline__ Part part(const SharedArgs& a, const SharedWs& w, int cta, int G) {
    Part p{};
    const int64_t from = static_cast<int64_t>(cta) * h.per, end = min(h.total, from + h.per);
    while (from + done < end && tile < h.tiles) {
      const int64_t at = from + done;
      const int64_t first = x.first + static_cast<int64_t>(kv) * x.places;
      const int p0 = static_cast<int>(at - first);
      const int p1 = static_cast<int>(min(static_cast<int64_t>(x.places), p0 + (end - at)));
      span = p1 - p0;
      p.b0 = max(0, p0 - h.open);
      p.nb = max(0, p1 - h.open) - p.b0;
      if (p.nb > 0) {
        p.t0 = x.t0, p.nt = x.nt, p.len = x.len, p.kv = kv;
        p.own = x.own != 0, p.dual = x.dual != 0;
        p.key0 = static_cast<int64_t>(kv) * a.n_rows + x.base;
        p.row = x.row + (kv * pieces_bound(x.places, h.per) + (at / h.per - first / h.per)) * x.nt * G;
        return p;
      }
      step(a, w);
    }
    p.nb = 0;
    return p;
  }
  __device__ __forceinline__ void step(const SharedArgs& a, const SharedWs& w) {
    done += span;
    if (++kv == a.KV) {
      kv = 0;
      while (++tile < h.tiles) {
        x = w.tile[tile];
        if (x.blocks > 0) break;
      }
    }
  }
  // One whole warp calls it.
  __device__ __forceinline__ Part begin(const SharedArgs& a, const SharedWs& w, int cta, int G, int lane) {
    h = *w.head;
    const int64_t at = static_cast<int64_t>(cta) * h.per;
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
    done = 0;
    tile = lo;
    x = w.tile[lo];
    kv = static_cast<int>((at - x.first) / x.places);
    return part(a, w, cta, G);
  }
  __device__ __forceinline__ Part next(const SharedArgs& a, const SharedWs& w, int cta, int G) {
    step(a, w);
    return part(a, w, cta, G);
  }
};

// Exponent of a V scale.
__device__ __forceinline__ float exponent(float v) {
  return static_cast<float>(max(static_cast<int>(__float_as_uint(fabsf(v)) >> 23) - 127, kLeastExp));
}

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
  static constexpr int kQHalf = kTileRows * 128;  // bytes of 64 columns of a Q tile
  static constexpr int kKvHalf = kBlock * 128;    // of a K or V tile
  static constexpr int kQ = kHalves * kQHalf, kKv = kHalves * kKvHalf;
  static constexpr int kRing = 2 * kQ, kSlots = 5;
  static constexpr int kRaws = 3, kRawTile = kBlock * D, kRaw = kRing + kSlots * kKv;  // int8 tiles as they come in
  static constexpr int kSmall = kRaw + kRaws * kRawTile;
};
constexpr int kScaleSlots = 4;  // a block's scales are overwritten four blocks later, after the P V of the block after it
constexpr int kParts = 4;       // parts known ahead
struct SharedSmall {
  uint64_t part_full[kParts], part_empty[kParts];
  uint64_t q_full[2], q_empty[2], full[5], empty[5], raw_full[3], raw_empty[3], s_full[2], p_full[2], pv_done[2], o_free[2], b_fin;
  alignas(16) float ks[kScaleSlots][kBlock];  // K scale x scale x log2 e
  alignas(16) float vs[kScaleSlots][kBlock];
  alignas(16) int hi[kScaleSlots][4], lo[kScaleSlots][4];  // exponent fields of each 32 keys' V scales: largest, least above 0
  uint32_t odd[kScaleSlots][4];   // those whose V scale is not finite, a bit each (the scale is kept as 0)
  Part part[kParts];
  float2 ml[kTileRows];           // stream 1's reference and sum, for stream 0 where they share the rows
  uint32_t tmem;
};
static_assert(offsetof(SharedSmall, ks) % 16 == 0 && offsetof(SharedSmall, vs) % 16 == 0 &&
                  offsetof(SharedSmall, hi) % 16 == 0 && offsetof(SharedSmall, lo) % 16 == 0 && sizeof(float) * kBlock % 16 == 0,
              "scales are read as 16-byte words");
template <int D>
constexpr int shared_smem() {
  static_assert(SharedShape<D>::kSmall % 1024 == 0, "tiles of whole swizzle atoms");
  return SharedShape<D>::kSmall + static_cast<int>(sizeof(SharedSmall));
}
constexpr uint32_t kTmemS = 128, kTmemO = 256;  // columns: S0 | S1 at 0 and 128, O0 | O1 from 256

// A lane's 32 bytes as one whole sector (p 32-byte aligned): a lane has a row of its own, so halves would be two requests each.
__device__ __forceinline__ void store_sector(float* p, const uint32_t* v) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]),
               "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

template <typename T, int D>
__global__ void __launch_bounds__(kAttendThreads, 1) k_shared_attend(const __grid_constant__ CUtensorMap mq,
                                                                     SharedArgs a, SharedWs w) {
  using S = SharedShape<D>;
  extern __shared__ __align__(1024) uint8_t smem[];
  SharedSmall* sm = reinterpret_cast<SharedSmall*>(smem + S::kSmall);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, G = a.H / a.KV, half = kTileRows / G;
  pdl_launch();
  pdl_wait();
  {
    const PlanHead h = *w.head;
    if (static_cast<int64_t>(blockIdx.x) * h.per >= h.total) return;
  }
  if (warp == 12) tmem_alloc(&sm->tmem, 512);
  if (threadIdx.x == 0) {
    for (int i = 0; i < kParts; ++i) {
      mbar_init(&sm->part_full[i], 1);
      mbar_init(&sm->part_empty[i], 14);  // 8 softmax and 4 conversion warps, the MMA and the Q warp
    }
    mbar_init(&sm->b_fin, 4);
    for (int i = 0; i < S::kSlots; ++i) {
      mbar_init(&sm->full[i], 128);
      mbar_init(&sm->empty[i], 1);
    }
    for (int i = 0; i < S::kRaws; ++i) {
      mbar_init(&sm->raw_full[i], 1);
      mbar_init(&sm->raw_empty[i], 4);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sm->q_full[i], 1);
      mbar_init(&sm->q_empty[i], 1);
      mbar_init(&sm->s_full[i], 1);
      mbar_init(&sm->p_full[i], 4);
      mbar_init(&sm->pv_done[i], 1);
      mbar_init(&sm->o_free[i], 4);
    }
    mbar_fence_init();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm->tmem;
  int* const st = a.status;
  // part i of the piece, once it is known; nb 0 (or a wait that ran out: ok false) ends the role's loop
  auto take = [&](uint32_t i, bool& ok) -> const Part& {
    ok = mbar_wait_warp(&sm->part_full[i % kParts], (i / kParts) & 1, st, kStatusTimeout);
    return sm->part[i % kParts];
  };
  auto give_back = [&](uint32_t i) { mbar_arrive(&sm->part_empty[i % kParts]); };
  auto slot = [&](uint32_t i) { return smem + S::kRing + (i % S::kSlots) * S::kKv; };

  if (warp < 8) {
    // ---------------- softmax, rescaling, partial results ----------------
    regs_up<kRegsSoftmax>();
    const int s = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + s * kTmemS + lanes, to = tmem + kTmemO + s * D + lanes;
    uint32_t gb = 0;              // blocks of this CTA before the part
    uint32_t mine = 0, other = 0; // blocks of this stream and of the other one so far
    uint32_t splits = 0;          // parts whose rows the streams shared
    bool ok = true;
    for (uint32_t part = 0;; ++part) {
      const Part& pt = take(part, ok);
      if (!ok || pt.nb == 0) break;
      const bool dual = pt.dual;
      const int rows = (dual ? (s ? pt.nt - half : half) : pt.nt) * G;
      const bool on = (warp & 3) * 32 < rows;
      int limit = pt.len;  // keys this row sees (a row without a token may see all: what comes of it is not looked at)
      if (row < rows) limit = pt.own ? own_keys(a, pt.t0 + (dual && s ? half : 0) + row / G, nullptr) : pt.len;
      limit -= pt.b0 * kBlock;
      float m = -INFINITY, l = 0.0f;
      bool spoilt = false;  // this row sees a key whose V scale is not finite
      const int nb = pt.nb, step = dual ? 1 : 2, j0 = dual ? 0 : s;
      for (int j = j0; j < nb; j += step, ++mine) {
        const int sl = (gb + j) & (kScaleSlots - 1);
        ok = mbar_wait_warp(&sm->s_full[s], mine & 1, st, kStatusTimeout);
        if (!ok) break;
        if (on) {
          tc_fence_after();
          float x[kBlock];
#pragma unroll
          for (int c = 0; c < kBlock / 32; ++c) tmem_ld32(ts + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(x + 32 * c));
          tmem_wait_ld();
          const float4* ks = reinterpret_cast<const float4*>(sm->ks[sl]);
          const float4* vs = reinterpret_cast<const float4*>(sm->vs[sl]);
          const int left = limit - j * kBlock;
          const bool cut = __any_sync(0xffffffffu, left < kBlock);
          float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int i = 0; i < kBlock / 4; ++i) {
            const float4 k4 = ks[i];
            const f2 y0 = f2_mul(f2_make(x[4 * i], x[4 * i + 1]), f2_make(k4.x, k4.y));
            const f2 y1 = f2_mul(f2_make(x[4 * i + 2], x[4 * i + 3]), f2_make(k4.z, k4.w));
            x[4 * i] = f2_lo(y0), x[4 * i + 1] = f2_hi(y0), x[4 * i + 2] = f2_lo(y1), x[4 * i + 3] = f2_hi(y1);
          }
          if (cut) {  // a branch of its own: selects on every score would cost as much as their exponentials
#pragma unroll
            for (int i = 0; i < kBlock; ++i)
              if (i >= left) x[i] = -INFINITY;
          }
#pragma unroll
          for (int i = 0; i < kBlock; i += 8) {
#pragma unroll
            for (int e = 0; e < 4; ++e) mx[e] = max3(mx[e], x[i + e], x[i + 4 + e]);
          }
          const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
          const int4 hi = *reinterpret_cast<const int4*>(sm->hi[sl]), lo = *reinterpret_cast<const int4*>(sm->lo[sl]);
          const int most = max(max(hi.x, hi.y), hi.z), least = min(min(lo.x, lo.y), lo.z);
          float want = top + static_cast<float>(max(most - 127, kLeastExp));
          const uint32_t* odd = sm->odd[sl];
          if (odd[0] | odd[1] | odd[2] | static_cast<uint32_t>(most - least > kSpread)) {  // one branch for what is rare
#pragma unroll 1
            for (int i = 0; i < 3; ++i) {
              const int v = left - 32 * i;
              spoilt |= (odd[i] & (v >= 32 ? 0xFFFFFFFFu : v <= 0 ? 0u : (1u << v) - 1)) != 0;
            }
            // exponents shuffled from a lane's three keys (loaded one by one: 46 us for 44, 8 trees)
            const float e0 = exponent(sm->vs[sl][lane]), e1 = exponent(sm->vs[sl][32 + lane]), e2 = exponent(sm->vs[sl][64 + lane]);
            want = -INFINITY;
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              want = max3(want, x[i] + __shfl_sync(0xffffffffu, e0, i), x[32 + i] + __shfl_sync(0xffffffffu, e1, i));
              want = fmaxf(want, x[64 + i] + __shfl_sync(0xffffffffu, e2, i));
            }
          }
          want -= kHeadroom;
          float scale = 1.0f;
          if (want > m && (m == -INFINITY || want - m > kRaiseMax)) {
            scale = ex2_approx(m - want);
            m = want;
          }
          if (j > j0 && __any_sync(0xffffffffu, scale != 1.0f)) {
            ok = mbar_wait_warp(&sm->pv_done[s], (mine - 1) & 1, st, kStatusTimeout);
            if (!ok) break;
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
              uint32_t v[32];
              tmem_ld32(to + 32 * c, v);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * scale);
              tmem_st32(to + 32 * c, v);
            }
          }
          const float ref = m == -INFINITY ? 0.0f : m;
          const f2 m2 = f2_make(-ref, -ref);
          f2 sum2 = f2_make(0.0f, 0.0f);
#pragma unroll
          for (int c = 0; c < kBlock / 32; ++c) {
            uint32_t p[16];
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
              const float4 v4 = vs[8 * c + i / 2];
              const int k = 32 * c + 2 * i;
              const f2 y0 = f2_add(f2_make(x[k], x[k + 1]), m2), y1 = f2_add(f2_make(x[k + 2], x[k + 3]), m2);
              const f2 e0 = f2_make(ex2_approx(f2_lo(y0)), ex2_approx(f2_hi(y0)));
              const f2 e1 = f2_make(ex2_approx(f2_lo(y1)), ex2_approx(f2_hi(y1)));
              sum2 = f2_add(sum2, f2_add(e0, e1));
              f2 w0 = f2_mul(e0, f2_make(v4.x, v4.y)), w1 = f2_mul(e1, f2_make(v4.z, v4.w));
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
      if (spoilt) l = __int_as_float(0x7FFFFFFF);  // its output is NaN
      const int n_mine = dual ? nb : (nb + 1 - s) / 2, n_other = dual ? nb : nb - n_mine;
      other += n_other;
      if (n_mine > 0) ok = mbar_wait_warp(&sm->pv_done[s], (mine - 1) & 1, st, kStatusTimeout);
      if (!ok) break;
      tc_fence_after();
      if (!dual && s == 1) {
        // stream 0 has taken the last part's: with no block in this part, nothing else holds this stream back
        if (part > 0) ok = mbar_wait_warp(&sm->o_free[1], (part - 1) & 1, st, kStatusTimeout);
        if (!ok) break;
        sm->ml[row] = make_float2(m, l);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm->b_fin);
      } else {
        float f0 = 1.0f, f1 = 0.0f;
        const bool join = !dual && n_other > 0;
        if (!dual) {
          ok = mbar_wait_warp(&sm->b_fin, splits & 1, st, kStatusTimeout) &&
               (n_other == 0 || mbar_wait_warp(&sm->pv_done[1], (other - 1) & 1, st, kStatusTimeout));
          if (!ok) break;
          tc_fence_after();
          const float2 o = sm->ml[row];
          if (join && !(o.x == -INFINITY && o.y == 0.0f)) {
            const float top = fmaxf(m, o.x);
            f0 = m == -INFINITY ? 0.0f : ex2_approx(m - top);
            f1 = ex2_approx(o.x - top);
            m = top;
            l = l * f0 + o.y * f1;
          }
        }
        if (on) {
          const int64_t r = pt.row + (dual && s ? half * G : 0) + row;
          if (row < rows) w.ml[r] = make_float2(m, l);
          float* o = w.o + r * D;
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            uint32_t v[32];
            tmem_ld32(to + 32 * c, v);
            tmem_wait_ld();
            if (join) {
              uint32_t u[32];
              tmem_ld32(to + D + 32 * c, u);
              tmem_wait_ld();
              // a row that sees none of a stream's keys has weights 0 there, and an output of 0
#pragma unroll
              for (int i = 0; i < 32; ++i)
                v[i] = __float_as_uint(__uint_as_float(v[i]) * f0 + __uint_as_float(u[i]) * f1);
            }
            if (row < rows) {
#pragma unroll
              for (int i = 0; i < 32; i += 8) store_sector(o + 32 * c + i, v + i);
            }
            __syncwarp();
          }
          tc_fence_before();
        }
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&sm->o_free[s]);
          if (!dual) mbar_arrive(&sm->o_free[1]);
        }
      }
      if (!dual) ++splits;
      gb += nb;
      __syncwarp();
      if (lane == 0) give_back(part);
    }
  } else if (warp < 12) {
    // ---------------- cache rows as 16-bit tiles ----------------
    // thread: 16 int8 values at column block c4 of rows r, r + 32, r + 64, in each half of 64 columns. The eight threads of a
    // store phase hold two rows x four blocks, which the swizzle spreads over all banks.
    regs_down<kRegsConvert>();
    const int t = threadIdx.x - 256, c4 = t & 3, r0 = t >> 2;
    const float kscale = a.scale * 1.44269504088896341f;
    uint32_t gb = 0, part = 0;
    bool ok = true, more = true;
    int64_t row0 = 0;
    int len = 0, b = 0, end = 0;  // the block whose scales are loaded next
    float ks = 0.0f, vs = 0.0f;   // scales of the block that is stored next
    auto open = [&]() {
      const Part& pt = take(part, ok);
      more = ok && pt.nb > 0;
      row0 = pt.key0;
      len = pt.len;
      b = pt.b0;
      end = pt.b0 + pt.nb;
      __syncwarp();
      if (more && lane == 0) give_back(part);
      ++part;
    };
    auto load_scales = [&]() {
      const int key = b * kBlock + t;
      const bool in = t < kBlock && key < len;
      ks = in ? a.ks[row0 + key] : 0.0f;
      vs = in ? a.vs[row0 + key] : 0.0f;
    };
    // tile i of the ring from the raw tile i
    auto convert = [&](uint32_t i, auto tag) {
      using E = decltype(tag);
      uint8_t* tile = slot(i);
      const uint8_t* raw = smem + S::kRaw + (i % S::kRaws) * S::kRawTile + 16 * c4;
#pragma unroll 1
      for (int h = 0; h < S::kHalves; ++h) {
        uint4 v[3];
#pragma unroll
        for (int u = 0; u < 3; ++u) v[u] = *reinterpret_cast<const uint4*>(raw + (r0 + 32 * u) * D + 64 * h);
#pragma unroll
        for (int u = 0; u < 3; ++u) {
          const int r = r0 + 32 * u;
          uint8_t* base = tile + h * S::kKvHalf + r * 128;
          const uint2 a0 = widen4<E>(v[u].x), a1 = widen4<E>(v[u].y), a2 = widen4<E>(v[u].z), a3 = widen4<E>(v[u].w);
          *reinterpret_cast<uint4*>(base + (((2 * c4) ^ (r & 7)) * 16)) = make_uint4(a0.x, a0.y, a1.x, a1.y);
          *reinterpret_cast<uint4*>(base + (((2 * c4 + 1) ^ (r & 7)) * 16)) = make_uint4(a2.x, a2.y, a3.x, a3.y);
        }
      }
      fence_async_smem();
      mbar_arrive(&sm->full[i % S::kSlots]);
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm->raw_empty[i % S::kRaws]);
    };
    auto ready = [&](uint32_t i) {  // the raw tile is there and the ring's slot is free
      ok = mbar_wait_warp(&sm->raw_full[i % S::kRaws], (i / S::kRaws) & 1, st, kStatusTimeout) &&
           (i < S::kSlots ||
            mbar_wait_warp_sleep(&sm->empty[i % S::kSlots], (i / S::kSlots - 1) & 1, st, kStatusTimeout, 40));
      return ok;
    };
    open();
    if (more) load_scales();
    while (more) {
      const int sl = gb & (kScaleSlots - 1);
      if (!ready(2 * gb)) break;
      if (t < kBlock) {
        const bool fine = fabsf(vs) < INFINITY;
        const int e = fine ? static_cast<int>(__float_as_uint(fabsf(vs)) >> 23) : 0;
        const int hi = __reduce_max_sync(0xffffffffu, e), lo = __reduce_min_sync(0xffffffffu, e ? e : 255);
        const uint32_t odd = __ballot_sync(0xffffffffu, !fine);
        sm->ks[sl][t] = ks * kscale;
        sm->vs[sl][t] = fine ? vs : 0.0f;
        if (lane == 0) sm->hi[sl][t >> 5] = hi, sm->lo[sl][t >> 5] = lo, sm->odd[sl][t >> 5] = odd;
      }
      if (++b == end) open();
      if (!ok) break;
      if (more) load_scales();
      convert(2 * gb, T());
      if (!ready(2 * gb + 1)) break;
      convert(2 * gb + 1, __half());
      ++gb;
    }
  } else {
    regs_down<kRegsMma>();
    if (warp == 12) {
      // ---------------- MMA ----------------
      constexpr int fmt = std::is_same<T, __half>::value ? 0 : 1;
      constexpr uint32_t id_s = umma_idesc_16(fmt, false, kTileRows, kBlock), id_o = umma_idesc_16(0, true, kTileRows, D);
      auto wait = [&](uint64_t* bar, uint32_t phase) { return mbar_wait_warp(bar, phase & 1, st, kStatusTimeout); };
      auto filled = [&](uint32_t i) { return wait(&sm->full[i % S::kSlots], i / S::kSlots); };
      // descriptors advance by their address field (in 16 bytes), which never carries out of it
      const uint64_t q_desc = umma_desc_sw128(smem_addr(smem), 16, 1024);
      const uint64_t k_desc = umma_desc_sw128(smem_addr(smem + S::kRing), 16, 1024);
      const uint64_t v_desc = umma_desc_sw128(smem_addr(smem + S::kRing), S::kKvHalf, 1024);
      auto scores = [&](int s, int q_tile, uint32_t i) {
        tc_fence_after();
        if (elect_one()) {
          const uint64_t q = q_desc + q_tile * (S::kQ >> 4), k = k_desc + (i % S::kSlots) * (S::kKv >> 4);
#pragma unroll
          for (int d = 0; d < D / 16; ++d)
            tc_mma_f16_ss(tmem + s * kTmemS, q + (d / 4) * (S::kQHalf >> 4) + (d % 4) * 2,
                          k + (d / 4) * (S::kKvHalf >> 4) + (d % 4) * 2, id_s, d > 0);
          tc_commit(&sm->s_full[s]);
        }
        __syncwarp();
      };
      auto values = [&](int s, uint32_t i, bool acc) {
        tc_fence_after();
        if (elect_one()) {
          const uint64_t v = v_desc + (i % S::kSlots) * (S::kKv >> 4);
#pragma unroll
          for (int k = 0; k < kBlock / 16; ++k)
            tc_mma_f16_ts(tmem + kTmemO + s * D, tmem + s * kTmemS + 8 * k, v + 128 * k, id_o, acc || k > 0);
          tc_commit(&sm->pv_done[s]);
        }
        __syncwarp();
      };
      auto commit = [&](uint64_t* bar) {
        if (elect_one()) tc_commit(bar);
        __syncwarp();
      };
      auto release = [&](uint32_t i) { commit(&sm->empty[i % S::kSlots]); };
      uint32_t gb = 0, done[2] = {0, 0};
      bool ok = true;
      for (uint32_t part = 0;; ++part) {
        ok = wait(&sm->part_full[part % kParts], part / kParts);
        if (!ok) break;
        const int nb = sm->part[part % kParts].nb;
        const bool dual = sm->part[part % kParts].dual;
        if (nb == 0) break;
        __syncwarp();
        if (lane == 0) give_back(part);
        const uint32_t i0 = 2 * gb;  // ring index of block j's K: i0 + 2 j, of its V: one more
        // a part whose streams share their rows has them in one of the two Q tiles, in turn, so that the next part's can come in
        const int qt = part & 1;
        auto q_done = [&]() {
          if (dual || qt == 0) commit(&sm->q_empty[0]);
          if (dual || qt == 1) commit(&sm->q_empty[1]);
        };
        ok = wait(&sm->q_full[part & 1], part >> 1) && filled(i0);
        if (!ok) break;
        if (dual) {
          scores(0, 0, i0);
          scores(1, 1, i0);
          release(i0);
          if (nb == 1) q_done();
          for (int j = 0; j < nb && ok; ++j) {
            const uint32_t vi = i0 + 2 * j + 1, kn = vi + 1;
            const bool again = j + 1 < nb;
            ok = filled(vi) && (!again || filled(kn));
            for (int s = 0; s < 2 && ok; ++s) {
              ok = (j > 0 || part == 0 || wait(&sm->o_free[s], part - 1)) && wait(&sm->p_full[s], done[s]);
              if (!ok) break;
              values(s, vi, j > 0);
              ++done[s];
              if (again) scores(s, s, kn);
            }
            if (!ok) break;
            release(vi);
            if (again) release(kn);
            if (j + 2 == nb) q_done();
          }
        } else {
          scores(0, qt, i0);
          release(i0);
          if (nb > 1) {
            ok = filled(i0 + 2);
            if (!ok) break;
            scores(1, qt, i0 + 2);
            release(i0 + 2);
          }
          if (nb <= 2) q_done();
          for (int j = 0; j < nb && ok; ++j) {
            const int s = j & 1;
            const uint32_t vi = i0 + 2 * j + 1, kn = vi + 3;
            ok = filled(vi) && (j > 1 || part == 0 || wait(&sm->o_free[s], part - 1)) && wait(&sm->p_full[s], done[s]);
            if (!ok) break;
            values(s, vi, j > 1);
            ++done[s];
            release(vi);
            if (j + 2 < nb) {
              ok = filled(kn);
              if (!ok) break;
              scores(s, qt, kn);
              release(kn);
              if (j + 3 == nb) q_done();
            }
          }
        }
        if (!ok) break;
        gb += nb;
      }
      if (!ok) {  // let what was issued end before TMEM and shared memory go
        commit(&sm->q_empty[0]);
        mbar_wait(&sm->q_empty[0], 0, nullptr, 0);
        mbar_wait(&sm->q_empty[0], 1, nullptr, 0);
      }
    } else if (warp == 13) {
      // ---------------- parts ----------------
      // and the loads of their K and V rows: a block's rows of a head are one piece of memory
      Walk walk;
      Part p = walk.begin(a, w, blockIdx.x, G, lane);
      uint32_t tile = 0;
      bool ok = true;
      for (uint32_t i = 0; ok; ++i) {
        if (i >= kParts)
          ok = mbar_wait_warp_sleep(&sm->part_empty[i % kParts], (i / kParts - 1) & 1, st, kStatusTimeout, 100);
        if (!ok) break;
        if (lane == 0) {
          sm->part[i % kParts] = p;
          mbar_arrive(&sm->part_full[i % kParts]);
        }
        __syncwarp();
        if (p.nb == 0) break;
        for (int b = p.b0; b < p.b0 + p.nb && ok; ++b) {
          const uint32_t bytes = static_cast<uint32_t>(min(kBlock, p.len - b * kBlock)) * D;
          const int64_t at = (p.key0 + static_cast<int64_t>(b) * kBlock) * D;
          for (int v = 0; v < 2 && ok; ++v, ++tile) {
            const uint32_t r = tile % S::kRaws;
            if (tile >= S::kRaws)
              ok = mbar_wait_warp_sleep(&sm->raw_empty[r], (tile / S::kRaws - 1) & 1, st, kStatusTimeout, 40);
            if (ok && lane == 0) {
              mbar_arrive_expect_tx(&sm->raw_full[r], bytes);
              bulk_g2s(smem + S::kRaw + r * S::kRawTile, (v ? a.v : a.k) + at, bytes, &sm->raw_full[r]);
            }
            __syncwarp();
          }
        }
        p = walk.next(a, w, blockIdx.x, G);
      }
      // every copy has landed before the block's shared memory goes
      for (uint32_t i = tile > S::kRaws ? tile - S::kRaws : 0; i < tile; ++i)
        mbar_wait_warp(&sm->raw_full[i % S::kRaws], (i / S::kRaws) & 1, st, kStatusTimeout);
    } else if (warp == 14) {
      // ---------------- Q ----------------
      // rows are (token, query head of the KV head), so 64 columns of a tile are one box of the tensor; behind a part's last
      // token it holds others', and what comes of those is not looked at
      bool ok = true;
      uint32_t uses[2] = {0, 0};  // parts that used each of the two tiles
      uint32_t issued = 0;
      for (uint32_t part = 0;; ++part) {
        const Part& pt = take(part, ok);
        if (!ok || pt.nb == 0) break;
        const bool dual = pt.dual;
#pragma unroll
        for (uint32_t q = 0; q < 2; ++q) {
          if (!ok || !(dual || (part & 1) == q)) continue;
          if (uses[q] > 0) ok = mbar_wait_warp_sleep(&sm->q_empty[q], (uses[q] - 1) & 1, st, kStatusTimeout, 40);
          ++uses[q];
        }
        if (!ok) break;
        if (lane == 0) {
          uint64_t* bar = &sm->q_full[part & 1];
          const int tiles = dual ? 2 : 1;
          mbar_arrive_expect_tx(bar, static_cast<uint32_t>(tiles * S::kHalves * half * G * 128));
          for (int q = 0; q < tiles; ++q)
#pragma unroll
            for (int x = 0; x < S::kHalves; ++x)
              tma_load_3d(smem + (dual ? q : static_cast<int>(part & 1)) * S::kQ + x * S::kQHalf, &mq, 64 * x, pt.kv * G,
                          pt.t0 + q * half, bar);
          issued = part + 1;
        }
        __syncwarp();
        if (lane == 0) give_back(part);
      }
      // every copy has landed before the block's shared memory goes
      if (lane == 0)
        for (uint32_t i = issued > 2 ? issued - 2 : 0; i < issued; ++i)
          mbar_wait(&sm->q_full[i & 1], (i >> 1) & 1, st, kStatusTimeout);
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 12) tmem_dealloc(tmem, 512);
}

// ---------------- join ----------------
template <typename T, int D>
__global__ void __launch_bounds__(256) k_shared_join(SharedArgs a, SharedWs w) {
  constexpr int N = D / 32;  // values of a lane
  const int64_t id = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  pdl_wait();
  if (id >= static_cast<int64_t>(a.n) * a.H) return;
  const int t = static_cast<int>(id / a.H), h = static_cast<int>(id % a.H), G = a.H / a.KV, kv = h / G;
  const PlanHead head = *w.head;
  const int pre = head.total > 0 ? w.tok_pre[t] : -1, own = head.total > 0 ? w.tok_own[t] : -1;
  const Tile tiles[2] = {w.tile[max(pre, 0)], w.tile[max(own, 0)]};
  float m = -INFINITY, l = 0.0f, o[N] = {};
  auto values = [&](const float* p, float (&v)[N]) {
    if constexpr (N == 4) {
      const float4 q = *reinterpret_cast<const float4*>(p);
      v[0] = q.x, v[1] = q.y, v[2] = q.z, v[3] = q.w;
    } else {
      const float2 q = *reinterpret_cast<const float2*>(p);
      v[0] = q.x, v[1] = q.y;
    }
  };
  if (head.total > 0) {
    // first partial row, distance of the next one and count, of the prefix's and of the own tile
    int64_t r0[2] = {0, 0}, dist[2] = {0, 0};
    int n[2] = {0, 0};
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      const Tile& x = tiles[which];
      if ((which ? own : pre) < 0 || x.blocks == 0) continue;
      const int64_t first = x.first + static_cast<int64_t>(kv) * x.places;
      n[which] = static_cast<int>((first + x.places - 1) / head.per - first / head.per) + 1;
      dist[which] = static_cast<int64_t>(x.nt) * G;
      r0[which] = x.row + kv * pieces_bound(x.places, head.per) * dist[which] + (t - x.t0) * G + h % G;
      if ((first / head.per + 1) * head.per - first <= head.open) --n[which], r0[which] += dist[which];  // cut before its blocks
    }
    for (int p0 = 0; p0 < n[0] + n[1]; p0 += 32) {  // a lane per piece, then the pieces' rows, four at a time
      const int p = p0 + lane, all = min(32, n[0] + n[1] - p0);
      int64_t r = 0;
      float2 ml = make_float2(-INFINITY, 0.0f);
      if (p < n[0] + n[1]) {
        r = p < n[0] ? r0[0] + p * dist[0] : r0[1] + (p - n[0]) * dist[1];
        ml = w.ml[r];
      }
      const float top = fmaxf(m, warp_max(ml.x));
      const float old = m == -INFINITY ? 0.0f : ex2_approx(m - top);
      const float f = ml.x == -INFINITY && ml.y == 0.0f ? 0.0f : ex2_approx(ml.x - top);
      l = l * old + warp_sum(f == 0.0f && ml.y == ml.y ? 0.0f : f * ml.y);
      m = top;
#pragma unroll
      for (int e = 0; e < N; ++e) o[e] *= old;
      for (int q = 0; q < all; q += 4) {
        float v[4][N], g[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int src = min(q + u, all - 1);
          const int64_t rr = __shfl_sync(0xffffffffu, r, src);
          g[u] = q + u < all ? __shfl_sync(0xffffffffu, f, src) : 0.0f;
          values(w.o + rr * D + N * lane, v[u]);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int e = 0; e < N; ++e) o[e] += g[u] * v[u][e];
      }
    }
  }
  // ancestors, four at a time
  if (a.anc_off) {
    const int lo = a.anc_off[t], hi = a.anc_off[t + 1];
    const int64_t base = a.kv_base[t];
    bool bad = lo < 0 || hi < lo || hi > a.n_anc;
    if (!bad && lo < hi) {
      const T* q = static_cast<const T*>(a.q) + static_cast<int64_t>(t) * a.q_ld + static_cast<int64_t>(h) * D + N * lane;
      float qv[N];
#pragma unroll
      for (int e = 0; e < N; ++e) qv[e] = to_float(q[e]) * (a.scale * 1.44269504088896341f);
      for (int i = lo; i < hi && !bad; i += 4) {
        int64_t at[4];
        int some = 0;  // of the four that are in the cache, up to the first that is not
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int64_t r = i + u < hi ? base + a.anc[i + u] : -1;
          const bool in = i + u < hi && a.anc[i + u] >= 0 && base >= 0 && r < a.n_rows;
          bad |= i + u < hi && !in;
          if (in && !bad) ++some;
          at[u] = static_cast<int64_t>(kv) * a.n_rows + (in ? r : 0);
        }
        float s[4], vs[4], v[4][N];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          s[u] = 0.0f;
#pragma unroll
          for (int e = 0; e < N; ++e) {
            s[u] += qv[e] * static_cast<float>(a.k[at[u] * D + N * lane + e]);
            v[u][e] = static_cast<float>(a.v[at[u] * D + N * lane + e]);
          }
          vs[u] = a.vs[at[u]];
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) s[u] = u < some ? warp_sum(s[u]) * a.ks[at[u]] : -INFINITY;
        const float top = fmaxf(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])), m);
        const float old = m == -INFINITY ? 0.0f : ex2_approx(m - top);
        m = top;
        l *= old;
#pragma unroll
        for (int e = 0; e < N; ++e) o[e] *= old;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          if (u < some) {
            const float g = ex2_approx(s[u] - top);
            // a V scale that is not finite: the output is NaN, as where the row is a prefix or own one
            l += fabsf(vs[u]) < INFINITY ? g : __int_as_float(0x7FFFFFFF);
#pragma unroll
            for (int e = 0; e < N; ++e) o[e] += g * vs[u] * v[u][e];
          }
        }
      }
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
  static std::atomic<bool> set[kMaxDevices] = {};  // several host threads may set the attributes at once
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
    if (at.numRegs * 4 < 2 * kRegsSoftmax + kRegsConvert + kRegsMma) return cudaErrorInvalidConfiguration;
    set[dev] = true;
  }
  CUtensorMap mq;
  const int G = a.H / a.KV;
  const int rc = make_map3(&mq, std::is_same<T, __nv_bfloat16>::value, a.q, D, a.H, a.n, a.q_ld, 64, kTileRows / G, G);
  if (rc != 0) return rc;
  const int ctas = sms;
  const WsLayout y = ws_layout(a.n, a.H, a.KV, D, a.n_groups, ctas);
  uint8_t* p = static_cast<uint8_t*>(ws);
  SharedWs w{reinterpret_cast<PlanHead*>(p + y.head), reinterpret_cast<Tile*>(p + y.tile),
             reinterpret_cast<int32_t*>(p + y.pre),   reinterpret_cast<int32_t*>(p + y.own),
             reinterpret_cast<int32_t*>(p + y.group), reinterpret_cast<float2*>(p + y.ml),
             reinterpret_cast<float*>(p + y.o),       y.rows,
             static_cast<int>(y.prefix_tiles)};
  k_shared_plan<<<1, kPlanThreads, 0, s>>>(a, w, ctas);
  e = cudaGetLastError();
  if (e == cudaSuccess)
    e = launch_pdl(k_shared_attend<T, D>, dim3(static_cast<unsigned>(ctas)), dim3(kAttendThreads), shared_smem<D>(), s,
                   mq, a, w);
  const int64_t warps = static_cast<int64_t>(a.n) * a.H;
  if (e == cudaSuccess)
    e = launch_pdl(k_shared_join<T, D>, dim3(static_cast<unsigned>((warps + 7) / 8)), dim3(256), 0, s, a, w);
  return e;
}

}  // namespace

int64_t attention_shared_workspace(int n, int H, int KV, int D, int n_groups, int sms) {
  return ws_layout(n, H, KV, D, n_groups, sms).bytes;
}

int launch_attention_shared(const SharedArgs& a, ActType type, int D, void* ws, int sms, cudaStream_t s) {
  if (a.n <= 0) return cudaSuccess;
  if (type == ActType::f16) return D == 64 ? run_shared<__half, 64>(a, ws, sms, s) : run_shared<__half, 128>(a, ws, sms, s);
  return D == 64 ? run_shared<__nv_bfloat16, 64>(a, ws, sms, s) : run_shared<__nv_bfloat16, 128>(a, ws, sms, s);
}

}  // namespace mkb
