// Per-head RMSNorm of queries and keys with the position rotation in the same pass, for float, fp16 and bf16 rows, and
// the int8 cache rows of the same tokens (mk_qk_norm_rope).
//
// Per head x of D values: y = x * w / sqrt(mean(x^2) + eps), then each pair (a, b) = (y[i], y[i + D/2]) becomes
// (a c - b s, a s + b c) with the token's row [cos D/2 | sin D/2] of the table. All of it in fp32 from the loaded values
// to the one rounding of the store. Cache rows follow quantize_i8 (quant.cpp:134-140): d = amax / 127,
// q = round(y / d), taken from the fp32 values, not from the rounded 16-bit ones.
//
// Bound: memory. A group of D / 8 lanes owns one head, each lane four values of the first half and the four they pair
// with, so the rotation needs no exchange and both halves are loaded and stored as whole 8- or 16-byte words.
//
//   k_qk_norm_rope       a group a head, a block per (token, heads): all loads asked for before the first is used. Short
//                        blocks whose bytes are in flight only a part of their life, so large batches stop at half of HBM:
//                        16384 tokens of 32 + 8 + 8 heads of 128, bf16 with cache rows: 115 us (3.5 TB/s)
//   k_qk_norm_rope_ring  large batches of wide rows: whole rows by bulk copies ahead of eight warps: 90 us (4.5 TB/s); with
//                        40 + 8 + 8 heads of 256 160 us (5.9 TB/s) against 270. What holds it is issue (70 % of the slots)
//                        and the latency of a head's chain in the 24 warps that fit beside the rows
// The rule: rows of at least 4 KB (rows of 3 KB: 41 us against 32, of 6 KB: 60 against 70, 16384 tokens) and at least eight
// of them for each CTA (2048 tokens of 12 KB: 15.5 us against 14.2, 4096: 26.4 against 28.5).
// Not kept: eight values a lane (16-byte words of 16-bit types; 109 us for 104 without the ring, 103 for 90 with it), two,
// three and four heads a lane one after the other (125, 104 and 123 us for 104).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "common.cuh"
#include "kernels.hpp"
#include "pipeline.cuh"
#include "types16.cuh"

namespace mkb {

namespace {

constexpr int kNrThreads = 256;

constexpr int kVals = 4;  // values of a lane in each half of a head

// kVals values at p, as one word where VEC.
template <typename T, bool VEC>
__device__ __forceinline__ void load(const T* p, float (&v)[kVals]) {
  if constexpr (!VEC) {
#pragma unroll
    for (int i = 0; i < kVals; ++i) v[i] = to_float(p[i]);
  } else if constexpr (sizeof(T) == 4) {
    const float4 q = *reinterpret_cast<const float4*>(p);
    v[0] = q.x, v[1] = q.y, v[2] = q.z, v[3] = q.w;
  } else {
    const uint2 q = *reinterpret_cast<const uint2*>(p);
    const float2 a = unpack2<T>(q.x), b = unpack2<T>(q.y);
    v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
  }
}

template <typename T, bool VEC>
__device__ __forceinline__ void store(T* p, const float (&v)[kVals]) {
  if constexpr (!VEC) {
#pragma unroll
    for (int i = 0; i < kVals; ++i) p[i] = from_float<T>(v[i]);
  } else if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]));
  }
}

template <int LANES>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
template <int LANES>
__device__ __forceinline__ float group_max(float v) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// Four int8 values of a cache row (4-byte aligned cache, D a multiple of 64: the word is aligned).
__device__ __forceinline__ void store_i8(int8_t* p, const float (&v)[kVals], float id) {
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < kVals; ++i) w |= (static_cast<uint32_t>(__float2int_rn(__fmul_rn(v[i], id))) & 0xFFu) << (8 * i);
  *reinterpret_cast<uint32_t*>(p) = w;
}

// A group's head h of token t from its values, weights and angles: the outputs, and the cache row at `at` (at least 0). Whole
// warps call it, with on false in lanes without a head; `cache` is the same for all of a warp.
template <typename T, int D, bool VEC>
__device__ __forceinline__ void finish_head(const NormRopeArgs& a, int t, int h, int lane, bool on, bool cache, int64_t at,
                                            float (&x0)[kVals], float (&x1)[kVals], const float (&w0)[kVals],
                                            const float (&w1)[kVals], const float (&c)[kVals], const float (&s)[kVals]) {
  constexpr int LANES = D / (2 * kVals), HALF = D / 2;
  const int i0 = kVals * lane;
  const bool rotated = h < a.H + a.KV;
  f2 p0[kVals / 2], p1[kVals / 2];
#pragma unroll
  for (int i = 0; i < kVals / 2; ++i)
    p0[i] = f2_make(x0[2 * i], x0[2 * i + 1]), p1[i] = f2_make(x1[2 * i], x1[2 * i + 1]);
  const f2 sq = f2_add(f2_fma(p0[1], p0[1], f2_mul(p0[0], p0[0])), f2_fma(p1[1], p1[1], f2_mul(p1[0], p1[0])));
  const float ss = group_sum<LANES>(f2_lo(sq) + f2_hi(sq));
  if (on && rotated) {
    const float r = rsqrtf(ss * (1.0f / D) + a.eps);
    const f2 r2 = f2_make(r, r);
#pragma unroll
    for (int i = 0; i < kVals / 2; ++i) {
      const f2 y0 = f2_mul(f2_mul(p0[i], r2), f2_make(w0[2 * i], w0[2 * i + 1]));
      const f2 y1 = f2_mul(f2_mul(p1[i], r2), f2_make(w1[2 * i], w1[2 * i + 1]));
      const f2 c2 = f2_make(c[2 * i], c[2 * i + 1]);
      const f2 a0 = f2_fma(y1, f2_make(-s[2 * i], -s[2 * i + 1]), f2_mul(y0, c2));
      const f2 a1 = f2_fma(y0, f2_make(s[2 * i], s[2 * i + 1]), f2_mul(y1, c2));
      x0[2 * i] = f2_lo(a0), x0[2 * i + 1] = f2_hi(a0);
      x1[2 * i] = f2_lo(a1), x1[2 * i + 1] = f2_hi(a1);
    }
    T* out = h < a.H ? static_cast<T*>(a.q) + static_cast<int64_t>(t) * a.q_ld + static_cast<int64_t>(h) * D
                     : static_cast<T*>(a.k) + static_cast<int64_t>(t) * a.k_ld + static_cast<int64_t>(h - a.H) * D;
    if (h < a.H || a.k) {
      store<T, VEC>(out + i0, x0);
      store<T, VEC>(out + HALF + i0, x1);
    }
  }
  if (!cache) return;
  float amax = 0.0f;
#pragma unroll
  for (int i = 0; i < kVals; ++i) amax = fmaxf(amax, fmaxf(fabsf(x0[i]), fabsf(x1[i])));
  amax = group_max<LANES>(amax);
  if (!on || h < a.H) return;
  const int kvh = rotated ? h - a.H : h - a.H - a.KV;
  const int64_t r = static_cast<int64_t>(kvh) * a.n_rows + at;
  const float d = __fdiv_rn(amax, 127.0f), id = d != 0.0f ? __fdiv_rn(1.0f, d) : 0.0f;
  int8_t* q8 = (rotated ? a.kc : a.vc) + r * D;
  store_i8(q8 + i0, x0, id);
  store_i8(q8 + HALF + i0, x1, id);
  if (lane == 0) (rotated ? a.ks : a.vs)[r] = d;
}

// Position and cache row of token t; -1: nothing is written, no cache row is written. Indexes past their tables are recorded
// where `report`.
__device__ __forceinline__ void token_places(const NormRopeArgs& a, int t, bool report, int& pos, int64_t& at) {
  pos = a.pos[t];
  at = a.kc ? a.kv_at[t] : -1;
  if ((pos >= a.n_pos || at >= a.n_rows) && report && a.status) atomicCAS(a.status, 0, kStatusBadIndex);
  if (pos >= a.n_pos) pos = -1;
  if (at >= a.n_rows) at = -1;
}

// Grid: (token, its heads by the block's groups).
template <typename T, int D, bool VEC>
__global__ void __launch_bounds__(kNrThreads) k_qk_norm_rope(NormRopeArgs a) {
  constexpr int LANES = D / (2 * kVals), GROUPS = kNrThreads / LANES, HALF = D / 2;
  const int t = blockIdx.x, lane = threadIdx.x % LANES, i0 = kVals * lane;
  const int h = blockIdx.y * GROUPS + threadIdx.x / LANES;
  const bool on = h < a.H + a.KV + (a.kc ? a.KV : 0);
  float x0[kVals] = {}, x1[kVals] = {}, w0[kVals] = {}, w1[kVals] = {}, c[kVals], s[kVals];
  if (on) {
    const T* x = static_cast<const T*>(a.qkv) + static_cast<int64_t>(t) * a.ld + static_cast<int64_t>(h) * D + i0;
    load<T, VEC>(x, x0);
    load<T, VEC>(x + HALF, x1);
  }
  if (h < a.H + a.KV) {
    const float* w = (h < a.H ? a.q_norm : a.k_norm) + i0;
    load<float, VEC>(w, w0);
    load<float, VEC>(w + HALF, w1);
  }
  int pos;
  int64_t at;
  token_places(a, t, threadIdx.x == 0 && blockIdx.y == 0, pos, at);
  if (pos < 0) return;
  const float* cs = a.rope + static_cast<int64_t>(pos) * D + i0;
  load<float, VEC>(cs, c);
  load<float, VEC>(cs + HALF, s);
  const bool cache = at >= 0 && static_cast<int>(blockIdx.y + 1) * GROUPS > a.H;  // the block has key or value heads
  finish_head<T, D, VEC>(a, t, h, lane, on, cache, at, x0, x1, w0, w1, c, s);
}

// The same for large batches: a CTA walks its tokens, one warp keeps a ring of whole rows (with their angles) filled by bulk
// copies, eight warps take the heads of a row from shared memory in rounds.
constexpr int kRingThreads = kNrThreads + 32, kRingCtas = 3, kRingMax = 8;
constexpr int kRingSmem = 72 * 1024;  // of a CTA
constexpr int kRingTokens = 8;        // of a CTA, at least
constexpr int kRingRow = 4096;        // bytes, at least

struct RingSmall {
  uint64_t full[kRingMax], empty[kRingMax];
  int64_t at[kRingMax], at32[32];
  int pos[kRingMax], pos32[32];
  alignas(16) float norm[2][256];  // weights of queries and keys: beside this much shared memory L1 holds little
};

template <typename T, int D>
__global__ void __launch_bounds__(kRingThreads, kRingCtas) k_qk_norm_rope_ring(NormRopeArgs a, int stages) {
  constexpr int LANES = D / (2 * kVals), GROUPS = kNrThreads / LANES, HALF = D / 2;
  extern __shared__ __align__(128) unsigned char smem[];
  const int heads = a.H + a.KV + (a.kc ? a.KV : 0), row = heads * D * static_cast<int>(sizeof(T)), stage = row + D * 4;
  RingSmall* sm = reinterpret_cast<RingSmall*>(smem + stages * stage);
  const int tid = threadIdx.x, warp = tid >> 5, step = gridDim.x;
  if (tid == 0) {
    for (int i = 0; i < stages; ++i) {
      mbar_init(&sm->full[i], 1);
      mbar_init(&sm->empty[i], kNrThreads / 32);
    }
    mbar_fence_init();
  }
  for (int i = tid; i < D; i += kRingThreads) {
    sm->norm[0][i] = a.q_norm[i];
    sm->norm[1][i] = a.k_norm[i];
  }
  __syncthreads();
  if (warp == kNrThreads / 32) {
    // a lane per token reads the places of 32 tokens ahead; lane 0 waits and issues
    const int me = tid % 32;
    int next_pos = -1, i = 0;
    int64_t next_at = -1;
    auto places = [&](int64_t first) {
      const int64_t t = first + static_cast<int64_t>(me) * step;
      if (t < a.n) token_places(a, static_cast<int>(t), true, next_pos, next_at);
    };
    places(blockIdx.x);
    bool ok = true;
    for (int64_t t = blockIdx.x; t < a.n && ok; t += step, ++i) {
      if (i % 32 == 0) {
        sm->pos32[me] = next_pos;
        sm->at32[me] = next_at;
        __syncwarp();
        places(t + 32 * static_cast<int64_t>(step));
      }
      const int slot = i % stages;
      if (me == 0) {
        if (i >= stages) ok = mbar_wait(&sm->empty[slot], (i / stages - 1) & 1, a.status, kStatusTimeout);
        if (ok) {
          const int pos = sm->pos32[i % 32];
          sm->pos[slot] = pos;
          sm->at[slot] = sm->at32[i % 32];
          if (pos < 0) {
            mbar_arrive(&sm->full[slot]);
          } else {
            unsigned char* to = smem + slot * stage;
            mbar_arrive_expect_tx(&sm->full[slot], static_cast<uint32_t>(stage));
            bulk_g2s(to, static_cast<const T*>(a.qkv) + t * a.ld, row, &sm->full[slot]);
            bulk_g2s(to + row, a.rope + static_cast<int64_t>(pos) * D, D * 4, &sm->full[slot]);
          }
        }
      }
      ok = __shfl_sync(0xffffffffu, ok, 0);
    }
    if (me == 0)  // no copy is in flight when the CTA ends
      for (int j = max(0, i - (ok ? 0 : 1) - stages); j < i - (ok ? 0 : 1); ++j)
        mbar_wait(&sm->full[j % stages], (j / stages) & 1, a.status, kStatusTimeout);
    return;
  }
  const int lane = tid % LANES, group = tid / LANES, i0 = kVals * lane;
  int slot = 0;
  uint32_t phase = 0;
  for (int64_t t = blockIdx.x; t < a.n; t += step) {
    if (!mbar_wait_warp(&sm->full[slot], phase, a.status, kStatusTimeout)) return;
    const int pos = sm->pos[slot];
    const int64_t at = sm->at[slot];
    if (pos >= 0) {
      const T* x = reinterpret_cast<const T*>(smem + slot * stage);
      const float* cs = reinterpret_cast<const float*>(smem + slot * stage + row) + i0;
      float c[kVals], s[kVals];
      load<float, true>(cs, c);
      load<float, true>(cs + HALF, s);
      // rounds of the warp's groups, as long as it has a head in them
      for (int h0 = 0; h0 + warp * (32 / LANES) < heads; h0 += GROUPS) {
        const int h = h0 + group;
        const bool on = h < heads;
        float x0[kVals] = {}, x1[kVals] = {}, w0[kVals] = {}, w1[kVals] = {};
        if (on) {
          load<T, true>(x + h * D + i0, x0);
          load<T, true>(x + h * D + HALF + i0, x1);
        }
        if (h < a.H + a.KV) {
          const float* w = sm->norm[h < a.H ? 0 : 1] + i0;
          load<float, true>(w, w0);
          load<float, true>(w + HALF, w1);
        }
        const bool cache = at >= 0 && h0 + (warp + 1) * (32 / LANES) > a.H;  // the warp has key or value heads
        finish_head<T, D, true>(a, static_cast<int>(t), h, lane, on, cache, at, x0, x1, w0, w1, c, s);
      }
    }
    __syncwarp();
    if (tid % 32 == 0) mbar_arrive(&sm->empty[slot]);
    if (++slot == stages) slot = 0, phase ^= 1;
  }
}

template <typename T, int D>
cudaError_t run_norm_rope(const NormRopeArgs& a, bool vec, bool bulk, int sms, cudaStream_t s) {
  constexpr int GROUPS = kNrThreads / (D / (2 * kVals));
  const int heads = a.H + a.KV + (a.kc ? a.KV : 0);
  const int64_t stage = static_cast<int64_t>(heads) * D * static_cast<int64_t>(sizeof(T)) + D * 4;
  const int room = kRingSmem - static_cast<int>(sizeof(RingSmall));
  const int ctas = kRingCtas * sms;
  if (bulk && stage - D * 4 >= kRingRow && 2 * stage <= room && a.n >= kRingTokens * ctas) {
    const int stages = static_cast<int>(std::min<int64_t>(kRingMax, room / stage));
    const cudaError_t e =
        cudaFuncSetAttribute(k_qk_norm_rope_ring<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingSmem);
    if (e != cudaSuccess) return e;
    k_qk_norm_rope_ring<T, D><<<ctas, kRingThreads, stages * stage + sizeof(RingSmall), s>>>(a, stages);
    return cudaGetLastError();
  }
  const dim3 grid(static_cast<unsigned>(a.n), static_cast<unsigned>((heads + GROUPS - 1) / GROUPS));
  if (vec)
    k_qk_norm_rope<T, D, true><<<grid, kNrThreads, 0, s>>>(a);
  else
    k_qk_norm_rope<T, D, false><<<grid, kNrThreads, 0, s>>>(a);
  return cudaGetLastError();
}

template <typename T>
cudaError_t run_norm_rope_d(const NormRopeArgs& a, int D, bool vec, bool bulk, int sms, cudaStream_t s) {
  if (D == 64) return run_norm_rope<T, 64>(a, vec, bulk, sms, s);
  if (D == 128) return run_norm_rope<T, 128>(a, vec, bulk, sms, s);
  return run_norm_rope<T, 256>(a, vec, bulk, sms, s);
}

}  // namespace

int launch_qk_norm_rope(const NormRopeArgs& a, ActType type, int D, int sms, cudaStream_t s) {
  if (a.n <= 0) return cudaSuccess;
  // whole words when every row of every buffer starts on one (heads are D apart inside a token, tokens ld)
  auto whole = [](const void* p, int64_t ld, int word, int vals) {
    return !p || (reinterpret_cast<uintptr_t>(p) % word == 0 && ld % vals == 0);
  };
  const int word = type == ActType::f32 ? 16 : 8;
  const bool vec = whole(a.qkv, a.ld, word, 4) && whole(a.q, a.q_ld, word, 4) && whole(a.k, a.k_ld, word, 4) &&
                   whole(a.rope, 0, 16, 4) && whole(a.q_norm, 0, 16, 4) && whole(a.k_norm, 0, 16, 4);
  const bool bulk = vec && whole(a.qkv, a.ld, 16, type == ActType::f32 ? 4 : 8);  // bulk copies take 16-byte words
  if (type == ActType::f32) return run_norm_rope_d<float>(a, D, vec, bulk, sms, s);
  if (type == ActType::f16) return run_norm_rope_d<__half>(a, D, vec, bulk, sms, s);
  return run_norm_rope_d<__nv_bfloat16>(a, D, vec, bulk, sms, s);
}

}  // namespace mkb
