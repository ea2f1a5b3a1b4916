// Per-head RMSNorm of queries and keys with the position rotation in the same pass, for float, fp16 and bf16 rows, and
// the int8 cache rows of the same tokens (mk_qk_norm_rope).
//
// Per head x of D values: y = x * w / sqrt(mean(x^2) + eps), then each pair (a, b) = (y[i], y[i + D/2]) becomes
// (a c - b s, a s + b c) with the token's row [cos D/2 | sin D/2] of the table. All of it in fp32 from the loaded values
// to the one rounding of the store. Cache rows follow quantize_i8 (quant.cpp:134-140): d = amax / 127,
// q = round(y / d), taken from the fp32 values, not from the rounded 16-bit ones.
//
// Bound: memory. A group of D / 8 lanes owns one head, each lane four values of the first half and the four they pair
// with, so the rotation needs no exchange and both halves are loaded and stored as whole 8- or 16-byte words. The head's
// values and the weights are asked for before the first of them is used. At 16384 tokens of 32 + 8 + 8 heads of 128 in bf16
// with their cache rows it takes 104 to 115 us (3.5 to 3.9 TB/s), on fp32 rows without a cache (8192 tokens, 40 heads) 56 to
// 65 (5.2 to 6.0 TB/s). Eight values a lane (16-byte words of 16-bit types) take 109 there and 61; two, three and four heads a
// lane one after the other 125, 104 and 123; a token's heads in rounds, angles and weights kept in registers, 112.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "common.cuh"
#include "kernels.hpp"
#include "types16.cuh"

namespace mkb {

namespace {

constexpr int kNrThreads = 256;

template <typename T, bool VEC>
__device__ __forceinline__ void load4(const T* p, float (&v)[4]) {
  if constexpr (!VEC) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = to_float(p[i]);
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
__device__ __forceinline__ void store4(T* p, const float (&v)[4]) {
  if constexpr (!VEC) {
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = from_float<T>(v[i]);
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

// Four int8 values of a cache row (16-byte aligned cache, D % 8 == 0: the word is aligned).
__device__ __forceinline__ void store_i8x4(int8_t* p, const float (&v)[4], float id) {
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) w |= (static_cast<uint32_t>(__float2int_rn(__fmul_rn(v[i], id))) & 0xFFu) << (8 * i);
  *reinterpret_cast<uint32_t*>(p) = w;
}

// Grid: (token, its heads by the block's groups). A block past the last head's group has lanes without a head; they run
// along, so that the shuffles see whole warps.
template <typename T, int D, bool VEC>
__global__ void __launch_bounds__(kNrThreads) k_qk_norm_rope(NormRopeArgs a) {
  constexpr int LANES = D / 8, GROUPS = kNrThreads / LANES, HALF = D / 2;
  const int t = blockIdx.x, lane = threadIdx.x % LANES, i0 = 4 * lane;
  const int h = blockIdx.y * GROUPS + threadIdx.x / LANES;
  const bool on = h < a.H + a.KV + (a.kc ? a.KV : 0), rotated = h < a.H + a.KV;
  const int pos = a.pos[t];
  float x0[4] = {}, x1[4] = {}, w0[4] = {}, w1[4] = {};
  if (on) {
    const T* x = static_cast<const T*>(a.qkv) + static_cast<int64_t>(t) * a.ld + static_cast<int64_t>(h) * D + i0;
    load4<T, VEC>(x, x0);
    load4<T, VEC>(x + HALF, x1);
  }
  if (rotated) {
    const float* w = (h < a.H ? a.q_norm : a.k_norm) + i0;
    load4<float, VEC>(w, w0);
    load4<float, VEC>(w + HALF, w1);
  }
  int64_t at = -1;
  bool bad = pos >= a.n_pos;
  if (a.kc) {
    at = a.kv_at[t];
    bad |= at >= a.n_rows;
    if (at >= a.n_rows) at = -1;
  }
  if (bad && threadIdx.x == 0 && blockIdx.y == 0 && a.status) atomicCAS(a.status, 0, kStatusBadIndex);
  if (pos < 0 || pos >= a.n_pos) return;  // padding or refused: nothing of this token is written
  float ss = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) ss += x0[i] * x0[i] + x1[i] * x1[i];
  ss = group_sum<LANES>(ss);
  if (rotated) {
    const float* cs = a.rope + static_cast<int64_t>(pos) * D + i0;
    float c[4], s[4];
    load4<float, VEC>(cs, c);
    load4<float, VEC>(cs + HALF, s);
    const float r = rsqrtf(ss * (1.0f / D) + a.eps);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float y0 = x0[i] * r * w0[i], y1 = x1[i] * r * w1[i];
      x0[i] = y0 * c[i] - y1 * s[i];
      x1[i] = y0 * s[i] + y1 * c[i];
    }
    T* out = h < a.H ? static_cast<T*>(a.q) + static_cast<int64_t>(t) * a.q_ld + static_cast<int64_t>(h) * D
                     : static_cast<T*>(a.k) + static_cast<int64_t>(t) * a.k_ld + static_cast<int64_t>(h - a.H) * D;
    if (h < a.H || a.k) {
      store4<T, VEC>(out + i0, x0);
      store4<T, VEC>(out + HALF + i0, x1);
    }
  }
  if (at < 0) return;  // the whole block: no cache row for this token
  float amax = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) amax = fmaxf(amax, fmaxf(fabsf(x0[i]), fabsf(x1[i])));
  amax = group_max<LANES>(amax);
  if (!on || h < a.H) return;
  const int kvh = rotated ? h - a.H : h - a.H - a.KV;
  const int64_t r = static_cast<int64_t>(kvh) * a.n_rows + at;
  const float d = __fdiv_rn(amax, 127.0f), id = d != 0.0f ? __fdiv_rn(1.0f, d) : 0.0f;
  int8_t* q8 = (rotated ? a.kc : a.vc) + r * D;
  store_i8x4(q8 + i0, x0, id);
  store_i8x4(q8 + HALF + i0, x1, id);
  if (lane == 0) (rotated ? a.ks : a.vs)[r] = d;
}

template <typename T, int D>
void run_norm_rope(const NormRopeArgs& a, bool vec, cudaStream_t s) {
  constexpr int GROUPS = kNrThreads / (D / 8);
  const int heads = a.H + a.KV + (a.kc ? a.KV : 0);
  const dim3 grid(static_cast<unsigned>(a.n), static_cast<unsigned>((heads + GROUPS - 1) / GROUPS));
  if (vec)
    k_qk_norm_rope<T, D, true><<<grid, kNrThreads, 0, s>>>(a);
  else
    k_qk_norm_rope<T, D, false><<<grid, kNrThreads, 0, s>>>(a);
}

template <typename T>
void run_norm_rope_d(const NormRopeArgs& a, int D, bool vec, cudaStream_t s) {
  if (D == 64) return run_norm_rope<T, 64>(a, vec, s);
  if (D == 128) return run_norm_rope<T, 128>(a, vec, s);
  run_norm_rope<T, 256>(a, vec, s);
}

}  // namespace

void launch_qk_norm_rope(const NormRopeArgs& a, ActType type, int D, cudaStream_t s) {
  if (a.n <= 0) return;
  // whole words when every row of every buffer starts on one (heads are D apart inside a token, tokens ld)
  auto whole = [](const void* p, int64_t ld, int word) {
    return !p || (reinterpret_cast<uintptr_t>(p) % word == 0 && ld % 4 == 0);
  };
  const int word = type == ActType::f32 ? 16 : 8;
  const bool vec = whole(a.qkv, a.ld, word) && whole(a.q, a.q_ld, word) && whole(a.k, a.k_ld, word) &&
                   whole(a.rope, 0, 16) && whole(a.q_norm, 0, 16) && whole(a.k_norm, 0, 16);
  if (type == ActType::f32) return run_norm_rope_d<float>(a, D, vec, s);
  if (type == ActType::f16) return run_norm_rope_d<__half>(a, D, vec, s);
  run_norm_rope_d<__nv_bfloat16>(a, D, vec, s);
}

}  // namespace mkb
