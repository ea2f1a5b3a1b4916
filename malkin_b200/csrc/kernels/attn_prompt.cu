// Causal grouped-query attention over packed prompts, fp16 / bf16 (mk_attention_prompt).
//
// Row i of a sequence: out_i = sum_{j <= i} p_j v_j / sum p_j, p_j = exp(scale q_i k_j - m). One pass over the keys with
// the running maximum and sum of the softmax per row (fp32), S = Q K^T and O += P V on tcgen05 with both accumulators in
// TMEM. P is rounded to the operands' type (half a step of it, 2^-8 or 2^-11, of each weight; the sum of the weights is
// taken before that rounding): tcgen05 has no wider A operand at this rate, and the errors of a row's weights average out.
//
// A CTA takes 256 rows of one head as two tiles of 128, so each K / V tile read from L2 feeds two tiles, and one tile's
// MMAs run while the other's softmax does:
//   warps 0-3, 4-7   softmax of tile 0 / 1: a thread per row; S from TMEM, P back over S (16-bit, half the columns)
//   warps 8-11       O *= exp(m_old - m_new) when a row's maximum grew, then the epilogue of both tiles
//   warp 12          issues every MMA      warp 13  TMA loads     warps 14, 15  check the V tiles of the diagonal
// TMEM (512 columns): S0 | S1 | O0 | O1. Shared memory: both Q tiles and a ring of K and V tiles of 128 keys.
//
// The maximum used for a row is only raised when it grew by more than 8 in the exponent of 2 (weights stay below 2^8,
// which both types hold), so that O is rarely rescaled.
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
constexpr int kPromptThreads = 512;
constexpr float kRaise = 8.0f;

template <int D>
struct PromptShape {
  static constexpr int kTile = kKeys * D * 2;  // bytes of a Q, K or V tile
  static constexpr int kHalf = kKeys * 128;    // bytes of 64 columns of it (128-byte swizzled rows)
  static constexpr int kStages = D == 128 ? 5 : 8;
  static constexpr int kQ = 0, kRing = 2 * kTile, kSmall = kRing + kStages * kTile;
};

struct PromptSmall {  // behind the tiles
  uint64_t q_full[2], full[8], empty[8], s_full[2], p_full[2], sc_full[2], o_ready[2], pv_done[2], fin[2], go[2], clean[2];
  float scale[2][kRows];
  float sum[2][kRows];
  uint32_t tmem;
  int seq_lo, seq_hi, tile;
  int odd_v;  // a diagonal V tile held an entry that is not finite
};

template <int D>
constexpr int prompt_smem() {
  return PromptShape<D>::kSmall + static_cast<int>(sizeof(PromptSmall));
}

// The sequence and the 256-row tile `want` (counted sequence after sequence, a sequence's longest tile first) belongs to.
__device__ __forceinline__ void find_tile(const int32_t* off, int n_seq, int n, int want, int lane, int* status,
                                          PromptSmall* sm) {
  int base = 0, lo_f = 0, hi_f = 0, tile_f = -1;
  for (int s0 = 0; s0 < n_seq; s0 += 32) {
    const int s = s0 + lane;
    int lo = 0, hi = 0;
    if (s < n_seq) {
      lo = off[s];
      hi = off[s + 1];
      if (lo < 0 || hi < lo || hi > n) {
        if (status) atomicCAS(status, 0, kStatusBadIndex);
        lo = hi = 0;
      }
    }
    const int tiles = (hi - lo + kPair - 1) / kPair;
    int incl = tiles;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += y;
    }
    const int first = base + incl - tiles;
    const unsigned hit = __ballot_sync(0xffffffffu, want >= first && want < first + tiles);
    if (hit) {
      const int src = __ffs(hit) - 1;
      lo_f = __shfl_sync(0xffffffffu, lo, src);
      hi_f = __shfl_sync(0xffffffffu, hi, src);
      tile_f = __shfl_sync(0xffffffffu, first + tiles - 1, src) - want;
      break;
    }
    base += __shfl_sync(0xffffffffu, incl, 31);
  }
  if (lane == 0) {
    sm->seq_lo = lo_f;
    sm->seq_hi = hi_f;
    sm->tile = tile_f;
  }
}

template <typename T>
__device__ __forceinline__ bool odd16(uint32_t w) {  // either half not finite
  constexpr uint32_t E = sizeof(T) == 2 && std::is_same<T, __half>::value ? 0x7C00u : 0x7F80u;
  return (w & E) == E || ((w >> 16) & E) == E;
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
  if (warp == 12) tmem_alloc(&sm->tmem, 512);
  if (threadIdx.x == 32) {
    for (int t = 0; t < 2; ++t) {
      mbar_init(&sm->q_full[t], 1);
      mbar_init(&sm->s_full[t], 1);
      mbar_init(&sm->p_full[t], 4);
      mbar_init(&sm->sc_full[t], 4);
      mbar_init(&sm->o_ready[t], 4);
      mbar_init(&sm->pv_done[t], 1);
      mbar_init(&sm->fin[t], 4);
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
    regs_up<192>();
    const int t = warp >> 2, row = (warp & 3) * 32 + lane;
    const int blocks = t == 0 ? nb0 : nb1;
    const uint32_t ts = tmem + static_cast<uint32_t>(t * kKeys) + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const float c = a.scale * 1.44269504088896341f;  // exp(scale x) = 2^(c x)
    float m = -INFINITY, l = 0.0f;                   // maximum in use (of the raw scores), sum of the weights
    bool ok = true;
    for (int j = 0; j < blocks; ++j) {
      ok = mbar_park_warp(&sm->s_full[t], j & 1, st, kStatusTimeout);
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
      if (j > 0) {
        sm->scale[t][row] = scale;
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm->sc_full[t]);
      }
      const float mc = m == -INFINITY ? 0.0f : m * c;
      const f2 c2 = f2_make(c, c), m2 = f2_make(-mc, -mc);
      f2 sum2 = f2_make(0.0f, 0.0f), sum3 = sum2;
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        uint32_t p[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const f2 x = f2_fma(f2_make(s[32 * b + 2 * i], s[32 * b + 2 * i + 1]), c2, m2);
          const float e0 = ex2_approx(f2_lo(x)), e1 = ex2_approx(f2_hi(x));
          if (i & 1)
            sum3 = f2_add(sum3, f2_make(e0, e1));
          else
            sum2 = f2_add(sum2, f2_make(e0, e1));
          p[i] = pack2<T>(e0, e1);
        }
        tmem_st16(ts + 16 * b, p);
      }
      sum2 = f2_add(sum2, sum3);
      l = l * scale + (f2_lo(sum2) + f2_hi(sum2));
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm->p_full[t]);
    }
    if (ok && blocks > 0) {
      sm->sum[t][row] = l;
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm->fin[t]);
    }
  } else if (warp < 12) {
    // ---------------- rescaling of O, epilogue ----------------
    regs_down<80>();
    const int row = (warp & 3) * 32 + lane;
    const uint32_t to = tmem + 2 * kKeys + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    bool ok = true;
    for (int j = 1; j < nb && ok; ++j) {
      for (int t = 0; t < 2 && ok; ++t) {
        if (j >= (t == 0 ? nb0 : nb1)) continue;
        ok = mbar_park_warp(&sm->sc_full[t], (j - 1) & 1, st, kStatusTimeout);
        if (!ok) break;
        const float f = sm->scale[t][row];
        if (__any_sync(0xffffffffu, f != 1.0f)) {
          ok = mbar_park_warp(&sm->pv_done[t], (j - 1) & 1, st, kStatusTimeout);
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int b = 0; b < D / 32; ++b) {
            uint32_t v[32];
            tmem_ld32(to + t * D + 32 * b, v);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * f);
            tmem_st32(to + t * D + 32 * b, v);
          }
          tmem_wait_st();
          tc_fence_before();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm->o_ready[t]);
      }
    }
    for (int t = 0; t < 2 && ok; ++t) {
      const int blocks = t == 0 ? nb0 : nb1;
      if (blocks == 0) continue;
      ok = mbar_park_warp(&sm->fin[t], 0, st, kStatusTimeout) &&
           mbar_park_warp(&sm->pv_done[t], (blocks - 1) & 1, st, kStatusTimeout);
      if (!ok) break;
      tc_fence_after();
      const float inv = 1.0f / sm->sum[t][row];
      const int i = q0 + t * kRows + row;  // row in the sequence
      const bool odd = sm->odd_v != 0;     // written before the MMAs that pv_done stands for
      T* out = static_cast<T*>(a.out) + static_cast<int64_t>(lo + i) * a.out_ld + static_cast<int64_t>(head) * D;
#pragma unroll 1
      for (int b = 0; b < D / 32; ++b) {
        uint32_t v[32];
        tmem_ld32(to + t * D + 32 * b, v);
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
    regs_down<48>();
    if (warp == 12 && lane == 0) {
      // ---------------- MMA ----------------
      constexpr int fmt = std::is_same<T, __half>::value ? 0 : 1;
      constexpr uint32_t id_s = umma_idesc_16(fmt, false, kRows, kKeys), id_o = umma_idesc_16(fmt, true, kRows, D);
      auto wait = [&](uint64_t* bar, int parity) { return mbar_park(bar, parity & 1, st, kStatusTimeout); };
      auto scores = [&](int t, int stage) {
        const uint32_t q = smem_addr(smem + S::kQ + t * S::kTile), k = smem_addr(ring(stage));
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
          const uint32_t o = static_cast<uint32_t>((d / 4) * S::kHalf + (d % 4) * 32);
          tc_mma_f16_ss(tmem + t * kKeys, umma_desc_sw128(q + o, 16, 1024), umma_desc_sw128(k + o, 16, 1024), id_s, d > 0);
        }
        tc_commit(&sm->s_full[t]);
      };
      auto values = [&](int t, int stage, bool acc) {
        const uint32_t v = smem_addr(ring(stage));
#pragma unroll
        for (int k = 0; k < kKeys / 16; ++k)
          tc_mma_f16_ts(tmem + 2 * kKeys + t * D, tmem + t * kKeys + 8 * k, umma_desc_sw128(v + 2048 * k, S::kHalf, 1024),
                        id_o, acc || k > 0);
        tc_commit(&sm->pv_done[t]);
      };
      auto stage = [&](int i) { return i % S::kStages; };
      auto phase = [&](int i) { return i / S::kStages; };
      bool ok = nb > 0;
      if (ok) {
        ok = wait(&sm->full[0], 0);
        for (int t = 0; t < 2 && ok; ++t) {
          if ((t == 0 ? nb0 : nb1) == 0) continue;
          ok = wait(&sm->q_full[t], 0);
          if (ok) {
            tc_fence_after();
            scores(t, 0);
          }
        }
        if (ok) tc_commit(&sm->empty[0]);
      }
      for (int j = 0; j < nb && ok; ++j) {
        const int vi = 2 * j + 1, ki = 2 * j + 2;
        ok = wait(&sm->full[stage(vi)], phase(vi));
        if (ok && j >= nb0 - 1) ok = wait(&sm->clean[j - (nb0 - 1)], 0);
        if (ok && j + 1 < nb) ok = wait(&sm->full[stage(ki)], phase(ki));
        for (int t = 0; t < 2 && ok; ++t) {
          const int blocks = t == 0 ? nb0 : nb1;
          if (j >= blocks) continue;
          ok = wait(&sm->p_full[t], j) && (j == 0 || wait(&sm->o_ready[t], j - 1));
          if (!ok) break;
          tc_fence_after();
          values(t, stage(vi), j > 0);
          if (j + 1 < blocks) scores(t, stage(ki));
        }
        if (ok) {
          tc_commit(&sm->empty[stage(vi)]);
          if (j + 1 < nb) tc_commit(&sm->empty[stage(ki)]);
        }
      }
      if (!ok && nb > 0) {  // let what was issued end before TMEM and shared memory go
        tc_commit(&sm->pv_done[0]);
        mbar_park(&sm->pv_done[0], 0, nullptr, 0);
        mbar_park(&sm->pv_done[0], 1, nullptr, 0);
      }
    } else if (warp == 13 && lane == 0) {
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
        if (round > 0) ok = mbar_park(&sm->empty[s], (round - 1) & 1, st, kStatusTimeout);
        if (!ok) break;
        load(i & 1 ? &mv : &mk, ring(s), kv, lo + (i / 2) * kKeys, &sm->full[s]);
        issued = i + 1;
        if ((i & 1) && i / 2 >= nb0 - 1) mbar_arrive(&sm->go[i / 2 - (nb0 - 1)]);
        if (i == 0 && nb1) load(&mq, smem + S::kQ + S::kTile, head, lo + q0 + kRows, &sm->q_full[1]);
      }
      // every copy has landed before the block's shared memory goes
      for (int i = max(0, issued - S::kStages); i < issued; ++i)
        mbar_park(&sm->full[i % S::kStages], (i / S::kStages) & 1, st, kStatusTimeout);
      if (nb0) mbar_park(&sm->q_full[0], 0, st, kStatusTimeout);
      if (nb1 && issued) mbar_park(&sm->q_full[1], 0, st, kStatusTimeout);
    } else if (warp >= 14 && nb > 0) {
      // ---------------- V tiles whose keys some rows must not see ----------------
      for (int j = nb0 - 1; j < nb; ++j) {
        const int i = 2 * j + 1;
        // the load has been issued, so the stage's phase is this tile's; it is not reused before the tile is checked
        if (!mbar_park_warp(&sm->go[j - (nb0 - 1)], 0, st, kStatusTimeout) ||
            !mbar_park_warp(&sm->full[i % S::kStages], (i / S::kStages) & 1, st, kStatusTimeout))
          break;
        uint4* v = reinterpret_cast<uint4*>(ring(i % S::kStages));
        bool seen = false;
#pragma unroll 8
        for (int x = (warp - 14) * 32 + lane; x < S::kTile / 16; x += 64) {
          const uint4 q = v[x];
          if (odd16<T>(q.x) || odd16<T>(q.y) || odd16<T>(q.z) || odd16<T>(q.w)) {
            alignas(16) T e[8];
            *reinterpret_cast<uint4*>(e) = q;
#pragma unroll
            for (int y = 0; y < 8; ++y)
              if (!(fabsf(to_float(e[y])) < INFINITY)) e[y] = from_float<T>(0.0f);
            v[x] = *reinterpret_cast<const uint4*>(e);
            seen = true;
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
  if (warp == 12) tmem_dealloc(tmem, 512);
}

template <typename T, int D>
int run_prompt(const PromptArgs& a, bool bf16, cudaStream_t s) {
  CUtensorMap mq, mk, mv;
  int rc = make_map3(&mq, bf16, a.q, D, a.H, a.n, a.q_ld, 64, kRows);
  if (rc == 0) rc = make_map3(&mk, bf16, a.k, D, a.KV, a.n, a.k_ld, 64, kKeys);
  if (rc == 0) rc = make_map3(&mv, bf16, a.v, D, a.KV, a.n, a.v_ld, 64, kKeys);
  if (rc != 0) return rc;
  static bool set[kMaxDevices] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= kMaxDevices) return cudaErrorInvalidDevice;
  if (!set[dev]) {
    e = cudaFuncSetAttribute(k_attn_prompt<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, prompt_smem<D>());
    if (e != cudaSuccess) return e;
    // the warpgroups' register shares (2 x 192 + 80 + 48 for 128 threads each) come out of the launch's
    cudaFuncAttributes at;
    e = cudaFuncGetAttributes(&at, k_attn_prompt<T, D>);
    if (e != cudaSuccess) return e;
    if (at.numRegs * kPromptThreads < (2 * 192 + 80 + 48) * 128) return cudaErrorInvalidConfiguration;
    set[dev] = true;
  }
  // a sequence of L rows has at most L / 256 + 1 tiles
  const int64_t tiles = a.n / kPair + std::min<int64_t>(a.n_seq, a.n);
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
