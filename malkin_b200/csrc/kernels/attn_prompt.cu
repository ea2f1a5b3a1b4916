// Causal grouped-query attention over packed prompts, fp16 / bf16 (mk_attention_prompt).
//
// Row i of a sequence: out_i = sum_{j <= i} p_j v_j / sum p_j, p_j = exp(scale q_i k_j - m). One pass over the keys with
// the running maximum and sum of the softmax per row (fp32), S = Q K^T and O += P V on tcgen05 with both accumulators in
// TMEM. P is rounded to the operands' type (half a step of it, 2^-8 or 2^-11, of each weight; the sum of the weights is
// taken before that rounding): tcgen05 has no wider A operand at this rate, and the errors of a row's weights average out. fp16
// has no such steps below 2^-14, and its weights are kept 2^7 larger: those below 2^-21 of the largest are held to 2^-32 of it.
//
// A CTA takes 256 rows of one head as two tiles of 128, so each K / V tile read from L2 feeds two tiles, and one tile's
// MMAs run while the other's softmax does:
//   warps 0-3, 4-7   softmax of tile 0 / 1: a thread per row; S from TMEM, P back over S (16-bit, half the columns),
//                    O *= exp(m_old - m_new) when a row's maximum grew, the epilogue
//   warp 8           issues every MMA      warp 9  TMA loads     warps 10, 11  check the V tiles of the diagonal
// TMEM (512 columns): S0 | S1 | O0 | O1. Shared memory: both Q tiles and a ring of K and V tiles of 128 keys.
//
// The maximum used for a row is only raised when it grew by more than 8 in the exponent of 2 (weights stay below 2^8, in fp16
// 2^15, which both types hold), so that O is rarely rescaled.
//
// Bound: the tensor pipe from some 300 tokens on (4 D H operations a pair of a row and a key). What holds it: a pair of blocks
// of 128 keys (one for each tile) takes 3670 cycles at D 128; the tensor pipe works 2050 of them (four products of 512 each), a
// tile's softmax takes 2200. A tile's softmax, its P V and its next Q K follow one another, and with two tiles in turn both the
// tensor and the XU pipe idle for almost half of the time. TMEM has room to break that chain, which is not done: P leaves half
// of its S's columns free, and at D 64 128 columns are not used at all. Measured: 8192 tokens, 40 / 8 heads of 128, fp16: 628 us
// (1.1 PFLOP/s) in bursts, 716 to 720 in a loop of seconds, under the power limit (with weights not kept larger 621 and 712);
// eight prompts of up to 2048 tokens, 32 / 8 heads, bf16: 211 to 220 us. Not kept, at the long prompt: two threads a row 692 us;
// 64-key blocks with S in two buffers 777; 2^x by a polynomial on the FMA pipe for 1/4 of the weights 626 against 632 in the
// same run, for 3/8 664.
//
// Masked keys: scores above the diagonal are replaced by -inf, whatever K holds there. Their weight 0 would still make a
// NaN of an infinity or NaN in V, so the tiles on the diagonal, whose keys some rows must not see (later tokens, or the
// next sequence's), are checked: entries that are not finite are set to 0 in shared memory, and the epilogue adds them
// back to the rows that do see them.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "common.cuh"
#include "kernels.hpp"
#include "tcgen05.cuh"
#include "tensor_map.hpp"
#include "types16.cuh"

namespace mkb {

namespace {

constexpr int kRows = 128;   // rows of a tile
constexpr int kPair = 256;   // rows of a CTA
constexpr int kKeys = 128;   // keys of a block
constexpr int kPromptThreads = 384;
constexpr int kPromptSoftmaxRegs = 208, kPromptOtherRegs = 88;  // 2 x 208 + 88 = 3 x the 168 of the launch
constexpr float kRaise = 8.0f;
constexpr float kHalfHeadroom = 7.0f;  // exponent of what fp16 weights are multiplied by; their sum carries it too

template <int D>
struct PromptShape {
  static constexpr int kTile = kKeys * D * 2;  // bytes of a Q, K or V tile
  static constexpr int kHalf = kKeys * 128;    // bytes of 64 columns of it (128-byte swizzled rows)
  static constexpr int kStages = D == 128 ? 5 : 8;
  static constexpr int kQ = 0, kRing = 2 * kTile, kSmall = kRing + kStages * kTile;
};

struct PromptSmall {  // behind the tiles
  uint64_t q_full[2], full[8], empty[8], s_full[2], p_full[2], pv_done[2], go[2], clean[2];
  uint32_t tmem;
  int seq_lo, seq_hi, tile;
  int odd_v;  // a diagonal V tile held an entry that is not finite
};

template <int D>
constexpr int prompt_smem() {
  return PromptShape<D>::kSmall + static_cast<int>(sizeof(PromptSmall));
}

// The sequence and the 256-row tile that CTA `want` of a head takes: of each 32 sequences the tiles with the most keys first,
// so that what runs last is short (eight prompts of up to 2048 tokens, 32 heads of 128: 225 us for 229 in sequence order). A
// tile's place is found from the number of tiles at or above a depth, by bisection. A sequence that begins before the end of an
// earlier one is left out, which takes a look at those ends from the first offset on that descends.
__device__ __forceinline__ void find_tile(const int32_t* off, int n_seq, int n, int want, int lane, int* status,
                                          PromptSmall* sm) {
  int lo_f = 0, hi_f = 0, tile_f = -1, until = 0;  // until: end of the sequences before the 32
  bool falls = false;
  for (int s0 = 0; s0 < n_seq; s0 += 32) {
    const int s = s0 + lane;
    int lo = 0, hi = 0;
    if (s < n_seq) {
      lo = off[s];
      hi = off[s + 1];
    }
    falls = __any_sync(0xffffffffu, hi < lo) || falls;
    bool bad = lo < 0 || hi < lo || hi > n;
    int end = !bad && hi > lo ? hi : 0;  // with the scan: of the sequences up to the lane's
    if (falls) {
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, end, o);
        if (lane >= o) end = max(end, y);
      }
      const int before = max(until, __shfl_up_sync(0xffffffffu, end, 1) * (lane > 0));
      bad |= hi > lo && lo < before;
    }
    until = max(until, __reduce_max_sync(0xffffffffu, end));
    if (bad) {
      if (status) atomicCAS(status, 0, kStatusBadIndex);
      lo = hi = 0;
    }
    const int tiles = (hi - lo + kPair - 1) / kPair;
    const int all = warp_isum(tiles);
    if (want >= all) {
      want -= all;
      continue;
    }
    int d = 0, above = 0;  // the deepest level with more than `want` tiles at or below it in the order; tiles deeper still
    for (int top = __reduce_max_sync(0xffffffffu, tiles); top - d > 1;) {
      const int mid = (d + top) / 2, at = warp_isum(max(0, tiles - mid));
      if (at > want)
        d = mid;
      else
        top = mid;
    }
    above = warp_isum(max(0, tiles - d - 1));
    const int src = static_cast<int>(__fns(__ballot_sync(0xffffffffu, tiles > d), 0, want - above + 1));
    lo_f = __shfl_sync(0xffffffffu, lo, src);
    hi_f = __shfl_sync(0xffffffffu, hi, src);
    tile_f = d;
    break;
  }
  if (lane == 0) {
    sm->seq_lo = lo_f;
    sm->seq_hi = hi_f;
    sm->tile = tile_f;
  }
}

// acc + 0 x each of the two values of w: NaN once a value that is not finite has been seen.
template <typename T>
__device__ __forceinline__ uint32_t add_zero_times(uint32_t acc, uint32_t w);
template <>
__device__ __forceinline__ uint32_t add_zero_times<__half>(uint32_t acc, uint32_t w) {
  __half2 r = __hfma2(*reinterpret_cast<__half2*>(&w), __float2half2_rn(0.0f), *reinterpret_cast<__half2*>(&acc));
  return *reinterpret_cast<uint32_t*>(&r);
}
template <>
__device__ __forceinline__ uint32_t add_zero_times<__nv_bfloat16>(uint32_t acc, uint32_t w) {
  __nv_bfloat162 r = __hfma2(*reinterpret_cast<__nv_bfloat162*>(&w), __float2bfloat162_rn(0.0f),
                             *reinterpret_cast<__nv_bfloat162*>(&acc));
  return *reinterpret_cast<uint32_t*>(&r);
}

template <typename T, int D>
__global__ void __launch_bounds__(kPromptThreads, 1)
    k_attn_prompt(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                  const __grid_constant__ CUtensorMap mv, PromptArgs a) {
  using S = PromptShape<D>;
  extern __shared__ __align__(1024) uint8_t smem[];
  PromptSmall* sm = reinterpret_cast<PromptSmall*>(smem + S::kSmall);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int head = static_cast<int>(blockIdx.x % a.H), want = static_cast<int>(blockIdx.x / a.H);
  if (warp == 0) find_tile(a.off, a.n_seq, a.n, want, lane, a.status, sm);
  if (warp == 8) tmem_alloc(&sm->tmem, 512);
  if (threadIdx.x == 32) {
    for (int t = 0; t < 2; ++t) {
      mbar_init(&sm->q_full[t], 1);
      mbar_init(&sm->s_full[t], 1);
      mbar_init(&sm->p_full[t], 4);
      mbar_init(&sm->pv_done[t], 1);
      mbar_init(&sm->go[t], 1);
      mbar_init(&sm->clean[t], 2);
    }
    for (int s = 0; s < S::kStages; ++s) {
      mbar_init(&sm->full[s], 1);
      mbar_init(&sm->empty[s], 1);
    }
    sm->odd_v = 0;
    mbar_fence_init();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm->tmem;
  const int lo = sm->seq_lo, len = sm->seq_hi - lo, tile = sm->tile;
  // blocks of keys each tile reads; tile 1 is empty where the sequence ends in tile 0
  const int q0 = tile * kPair;
  const int nb0 = tile < 0 ? 0 : 2 * tile + 1;
  const int nb1 = tile >= 0 && q0 + kRows < len ? nb0 + 1 : 0;
  const int nb = max(nb0, nb1);
  const int kv = head / (a.H / a.KV);
  auto ring = [&](int i) { return smem + S::kRing + i * S::kTile; };
  int* const st = a.status;

  if (warp < 8) {
    // ---------------- softmax ----------------
    regs_up<kPromptSoftmaxRegs>();
    const int t = warp >> 2, row = (warp & 3) * 32 + lane;
    const int blocks = t == 0 ? nb0 : nb1;
    const uint32_t ts = tmem + static_cast<uint32_t>(t * kKeys) + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t to = tmem + static_cast<uint32_t>(2 * kKeys + t * D) + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const float c = a.scale * 1.44269504088896341f;  // exp(scale x) = 2^(c x)
    float m = -INFINITY, l = 0.0f;                   // maximum in use (of the raw scores), sum of the weights
    bool ok = true;
    for (int j = 0; j < blocks; ++j) {
      ok = mbar_wait_warp(&sm->s_full[t], j & 1, st, kStatusTimeout);
      if (!ok) break;
      tc_fence_after();
      float s[kKeys];
#pragma unroll
      for (int b = 0; b < 4; ++b) tmem_ld32(ts + 32 * b, *reinterpret_cast<uint32_t(*)[32]>(s + 32 * b));
      tmem_wait_ld();
      if (j == blocks - 1) {  // the diagonal
#pragma unroll
        for (int i = 0; i < kKeys; ++i)
          if (i > row) s[i] = -INFINITY;
      }
      float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
      for (int i = 4; i + 8 <= kKeys; i += 8) {
#pragma unroll
        for (int e = 0; e < 4; ++e) mx[e] = max3(mx[e], s[i + e], s[i + 4 + e]);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) mx[e] = fmaxf(mx[e], s[kKeys - 4 + e]);
      // scale is positive: the largest score is the largest exponent
      const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
      float scale = 1.0f;
      if (top > m && (j == 0 || (top - m) * c > kRaise)) {
        scale = j == 0 ? 0.0f : ex2_approx((m - top) * c);
        m = top;
      }
      if (j > 0 && __any_sync(0xffffffffu, scale != 1.0f)) {
        ok = mbar_wait_warp(&sm->pv_done[t], (j - 1) & 1, st, kStatusTimeout);
        if (!ok) break;
        tc_fence_after();
#pragma unroll 1
        for (int b = 0; b < D / 32; ++b) {
          uint32_t v[32];
          tmem_ld32(to + 32 * b, v);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * scale);
          tmem_st32(to + 32 * b, v);
        }
      }
      const float mc = (m == -INFINITY ? 0.0f : m * c) - (std::is_same<T, __half>::value ? kHalfHeadroom : 0.0f);
      const f2 c2 = f2_make(c, c), m2 = f2_make(-mc, -mc);
      f2 sum2 = f2_make(0.0f, 0.0f), sum3 = sum2;
#pragma unroll
      for (int i = 0; i < kKeys; i += 2) {
        const f2 x = f2_fma(f2_make(s[i], s[i + 1]), c2, m2);
        s[i] = f2_lo(x);
        s[i + 1] = f2_hi(x);
      }
      constexpr int kLag = 8;  // exponentials ahead of their sums and packing
      uint32_t p[16];
#pragma unroll
      for (int i = 0; i < kKeys + kLag; i += 2) {
        if (i < kKeys) {
          s[i] = ex2_approx(s[i]);
          s[i + 1] = ex2_approx(s[i + 1]);
        }
        const int k = i - kLag;
        if (k >= 0) {
          if (k & 2)
            sum3 = f2_add(sum3, f2_make(s[k], s[k + 1]));
          else
            sum2 = f2_add(sum2, f2_make(s[k], s[k + 1]));
          p[(k / 2) & 15] = pack2<T>(s[k], s[k + 1]);
          if ((k & 31) == 30) tmem_st16(ts + k / 32 * 16, p);
        }
      }
      sum2 = f2_add(sum2, sum3);
      l = l * scale + (f2_lo(sum2) + f2_hi(sum2));
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm->p_full[t]);
    }
    if (ok && blocks > 0) ok = mbar_wait_warp(&sm->pv_done[t], (blocks - 1) & 1, st, kStatusTimeout);
    if (ok && blocks > 0) {
      tc_fence_after();
      const float inv = 1.0f / l;
      const int i = q0 + t * kRows + row;  // row in the sequence
      const bool odd = sm->odd_v != 0;     // written before the MMAs that pv_done stands for
      T* out = static_cast<T*>(a.out) + static_cast<int64_t>(lo + i) * a.out_ld + static_cast<int64_t>(head) * D;
#pragma unroll 1
      for (int b = 0; b < D / 32; ++b) {
        uint32_t v[32];
        tmem_ld32(to + 32 * b, v);
        tmem_wait_ld();
        if (i < len) {
          float o[32];
  #pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = __uint_as_float(v[e]) * inv;
          if (odd) {  // entries of the checked tiles that this row sees and that are not finite: the row becomes them
            for (int j = (nb0 - 1) * kKeys; j <= i; ++j) {
              const T* vr = static_cast<const T*>(a.v) + static_cast<int64_t>(lo + j) * a.v_ld + kv * D + 32 * b;
  #pragma unroll
              for (int e = 0; e < 32; ++e) {
                const float x = to_float(vr[e]);
                if (!(fabsf(x) < INFINITY)) o[e] += x;
              }
            }
          }
  #pragma unroll
          for (int w = 0; w < 4; ++w) {
            uint4 q;
            q.x = pack2<T>(o[8 * w], o[8 * w + 1]);
            q.y = pack2<T>(o[8 * w + 2], o[8 * w + 3]);
            q.z = pack2<T>(o[8 * w + 4], o[8 * w + 5]);
            q.w = pack2<T>(o[8 * w + 6], o[8 * w + 7]);
            *reinterpret_cast<uint4*>(out + 32 * b + 8 * w) = q;
          }
        }
        __syncwarp();
      }
    }
  } else {
    regs_down<kPromptOtherRegs>();
    if (warp == 8) {
      // ---------------- MMA ----------------
      constexpr int fmt = std::is_same<T, __half>::value ? 0 : 1;
      constexpr uint32_t id_s = umma_idesc_16(fmt, false, kRows, kKeys), id_o = umma_idesc_16(fmt, true, kRows, D);
      auto wait = [&](uint64_t* bar, int parity) { return mbar_wait_warp(bar, parity & 1, st, kStatusTimeout); };
      // descriptors advance by their address field (in 16 bytes), which never carries out of it
      const uint64_t q_desc = umma_desc_sw128(smem_addr(smem + S::kQ), 16, 1024);
      const uint64_t k_desc = umma_desc_sw128(smem_addr(smem + S::kRing), 16, 1024);
      const uint64_t v_desc = umma_desc_sw128(smem_addr(smem + S::kRing), S::kHalf, 1024);
      auto scores = [&](int t, int stage) {
        tc_fence_after();
        if (elect_one()) {
          const uint64_t q = q_desc + t * (S::kTile >> 4), k = k_desc + stage * (S::kTile >> 4);
#pragma unroll
          for (int d = 0; d < D / 16; ++d) {
            const int o = ((d / 4) * S::kHalf + (d % 4) * 32) >> 4;
            tc_mma_f16_ss(tmem + t * kKeys, q + o, k + o, id_s, d > 0);
          }
          tc_commit(&sm->s_full[t]);
        }
        __syncwarp();
      };
      auto values = [&](int t, int stage, bool acc) {
        tc_fence_after();
        if (elect_one()) {
          const uint64_t v = v_desc + stage * (S::kTile >> 4);
#pragma unroll
          for (int k = 0; k < kKeys / 16; ++k)
            tc_mma_f16_ts(tmem + 2 * kKeys + t * D, tmem + t * kKeys + 8 * k, v + 128 * k, id_o, acc || k > 0);
          tc_commit(&sm->pv_done[t]);
        }
        __syncwarp();
      };
      auto release = [&](int stage) {
        if (elect_one()) tc_commit(&sm->empty[stage]);
        __syncwarp();
      };
      bool ok = nb > 0;
      if (ok) {
        ok = wait(&sm->full[0], 0) && wait(&sm->q_full[0], 0);
        if (ok) scores(0, 0);
        if (ok && nb1 > 0) {
          ok = wait(&sm->q_full[1], 0);
          if (ok) scores(1, 0);
        }
        if (ok) release(0);
      }
      int vs = 1, vp = 0, ks = 2, kp = 0;  // ring slots and phases of the block's V and of the next one's K
      auto step = [&](int& slot, int& phase) {
        slot += 2;
        if (slot >= S::kStages) slot -= S::kStages, phase ^= 1;
      };
      for (int j = 0; j < nb && ok; ++j) {
        ok = wait(&sm->full[vs], vp);
        if (ok && j >= nb0 - 1) ok = wait(&sm->clean[j - (nb0 - 1)], 0);
        if (ok && j + 1 < nb) ok = wait(&sm->full[ks], kp);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const int blocks = t == 0 ? nb0 : nb1;
          if (j >= blocks || !ok) continue;
          ok = wait(&sm->p_full[t], j);
          if (!ok) continue;
          values(t, vs, j > 0);
          if (j + 1 < blocks) scores(t, ks);
        }
        if (ok) {
          release(vs);
          if (j + 1 < nb) release(ks);
        }
        step(vs, vp);
        step(ks, kp);
      }
      if (!ok && nb > 0) {  // let what was issued end before TMEM and shared memory go
        if (elect_one()) tc_commit(&sm->pv_done[0]);
        __syncwarp();
        mbar_wait(&sm->pv_done[0], 0, nullptr, 0);
        mbar_wait(&sm->pv_done[0], 1, nullptr, 0);
        __syncwarp();
      }
    } else if (warp == 9 && lane == 0) {
      // ---------------- loads ----------------
      auto load = [&](const CUtensorMap* map, uint8_t* dst, int h, int at, uint64_t* bar) {
        mbar_arrive_expect_tx(bar, S::kTile);
#pragma unroll
        for (int x = 0; x < D / 64; ++x) tma_load_3d(dst + x * S::kHalf, map, 64 * x, h, at, bar);
      };
      int issued = 0;
      bool ok = true;
      if (nb0) load(&mq, smem + S::kQ, head, lo + q0, &sm->q_full[0]);
      for (int i = 0; i < 2 * nb && ok; ++i) {
        const int s = i % S::kStages, round = i / S::kStages;
        if (round > 0) ok = mbar_wait(&sm->empty[s], (round - 1) & 1, st, kStatusTimeout);
        if (!ok) break;
        load(i & 1 ? &mv : &mk, ring(s), kv, lo + (i / 2) * kKeys, &sm->full[s]);
        issued = i + 1;
        if ((i & 1) && i / 2 >= nb0 - 1) mbar_arrive(&sm->go[i / 2 - (nb0 - 1)]);
        if (i == 0 && nb1) load(&mq, smem + S::kQ + S::kTile, head, lo + q0 + kRows, &sm->q_full[1]);
      }
      // every copy has landed before the block's shared memory goes
      for (int i = max(0, issued - S::kStages); i < issued; ++i)
        mbar_wait(&sm->full[i % S::kStages], (i / S::kStages) & 1, st, kStatusTimeout);
      if (nb0) mbar_wait(&sm->q_full[0], 0, st, kStatusTimeout);
      if (nb1 && issued) mbar_wait(&sm->q_full[1], 0, st, kStatusTimeout);
    } else if (warp >= 10 && nb > 0) {
      // ---------------- V tiles whose keys some rows must not see ----------------
      for (int j = nb0 - 1; j < nb; ++j) {
        const int i = 2 * j + 1;
        // the load has been issued, so the stage's phase is this tile's; it is not reused before the tile is checked
        if (!mbar_wait_warp_sleep(&sm->go[j - (nb0 - 1)], 0, st, kStatusTimeout, 100) ||
            !mbar_wait_warp(&sm->full[i % S::kStages], (i / S::kStages) & 1, st, kStatusTimeout))
          break;
        uint4* v = reinterpret_cast<uint4*>(ring(i % S::kStages));
        const int x0 = (warp - 10) * 32 + lane;
        uint32_t acc[4] = {0, 0, 0, 0};
#pragma unroll 8
        for (int x = x0; x < S::kTile / 16; x += 64) {
          const uint4 q = v[x];
          acc[0] = add_zero_times<T>(acc[0], q.x);
          acc[1] = add_zero_times<T>(acc[1], q.y);
          acc[2] = add_zero_times<T>(acc[2], q.z);
          acc[3] = add_zero_times<T>(acc[3], q.w);
        }
        bool seen = false;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 f = unpack2<T>(acc[e]);
          seen |= f.x != f.x || f.y != f.y;
        }
        if (seen) {
          for (int x = x0; x < S::kTile / 16; x += 64) {
            alignas(16) T e[8];
            *reinterpret_cast<uint4*>(e) = v[x];
#pragma unroll
            for (int y = 0; y < 8; ++y)
              if (!(fabsf(to_float(e[y])) < INFINITY)) e[y] = from_float<T>(0.0f);
            v[x] = *reinterpret_cast<const uint4*>(e);
          }
        }
        if (seen) sm->odd_v = 1;
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm->clean[j - (nb0 - 1)]);
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 8) tmem_dealloc(tmem, 512);
}

template <typename T, int D>
int run_prompt(const PromptArgs& a, bool bf16, cudaStream_t s) {
  CUtensorMap mq, mk, mv;
  int rc = make_map3(&mq, bf16, a.q, D, a.H, a.n, a.q_ld, 64, kRows);
  if (rc == 0) rc = make_map3(&mk, bf16, a.k, D, a.KV, a.n, a.k_ld, 64, kKeys);
  if (rc == 0) rc = make_map3(&mv, bf16, a.v, D, a.KV, a.n, a.v_ld, 64, kKeys);
  if (rc != 0) return rc;
  static std::atomic<bool> set[kMaxDevices] = {};  // several host threads may set the attributes at once
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= kMaxDevices) return cudaErrorInvalidDevice;
  if (!set[dev]) {
    e = cudaFuncSetAttribute(k_attn_prompt<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, prompt_smem<D>());
    if (e != cudaSuccess) return e;
    // the warpgroups' register shares come out of the launch's
    cudaFuncAttributes at;
    e = cudaFuncGetAttributes(&at, k_attn_prompt<T, D>);
    if (e != cudaSuccess) return e;
    if (at.numRegs * 3 < 2 * kPromptSoftmaxRegs + kPromptOtherRegs) return cudaErrorInvalidConfiguration;
    set[dev] = true;
  }
  // a sequence of L rows has at most L / 256 + 1 tiles; one that is bad has none, so the last tile's search passes over all
  // offsets then, and finds each that is
  const int64_t tiles = a.n / kPair + std::min<int64_t>(a.n_seq, static_cast<int64_t>(a.n) + 1);
  const int64_t grid = tiles * a.H;
  if (grid > INT32_MAX) return cudaErrorInvalidValue;
  k_attn_prompt<T, D><<<static_cast<unsigned>(grid), kPromptThreads, prompt_smem<D>(), s>>>(mq, mk, mv, a);
  return cudaGetLastError();
}

}  // namespace

int launch_attention_prompt(const PromptArgs& a, ActType type, int D, cudaStream_t s) {
  if (a.n <= 0 || a.n_seq <= 0) return cudaSuccess;
  if (type == ActType::f16)
    return D == 64 ? run_prompt<__half, 64>(a, false, s) : run_prompt<__half, 128>(a, false, s);
  return D == 64 ? run_prompt<__nv_bfloat16, 64>(a, true, s) : run_prompt<__nv_bfloat16, 128>(a, true, s);
}

}  // namespace mkb
