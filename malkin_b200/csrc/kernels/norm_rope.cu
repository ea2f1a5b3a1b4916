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

// Grid: (token, head slice). A group takes heads g, g + groups, ... of its slice.
template <typename T, int D, bool VEC>
__global__ void __launch_bounds__(kNrThreads)
    k_qk_norm_rope(NormRopeArgs a) {
  constexpr int LANES = D / 8, GROUPS = kNrThreads / LANES, HALF = D / 2;
  const int t = blockIdx.x, lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
  const int heads = a.H + a.KV + (a.kc ? a.KV : 0);
  const int pos = a.pos[t];
  const bool in_table = pos >= 0 && pos < a.n_pos;
  int64_t at = -1;
  bool bad = pos >= a.n_pos;
  if (a.kc) {
    at = a.kv_at[t];
    bad |= at >= a.n_rows;
    if (at >= a.n_rows) at = -1;
  }
  if (bad && threadIdx.x == 0 && blockIdx.y == 0 && a.status) atomicCAS(a.status, 0, kStatusBadIndex);
  if (!in_table) return;  // padding (pos < 0) or refused: nothing of this token is written
  const T* row = static_cast<const T*>(a.qkv) + static_cast<int64_t>(t) * a.ld;
  const int i0 = 4 * lane;
  float c[4], s[4];
  {
    const float* cs = a.rope + static_cast<int64_t>(pos) * D;
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = cs[i0 + i], s[i] = cs[HALF + i0 + i];
  }
  // every lane of a warp runs every round, so the shuffles see whole warps
  for (int h0 = blockIdx.y * GROUPS; h0 < heads; h0 += gridDim.y * GROUPS) {
    const int h = h0 + group;
    const bool on = h < heads;
    float x0[4] = {}, x1[4] = {};
    if (on) {
      const T* x = row + static_cast<int64_t>(h) * D;
      load4<T, VEC>(x + i0, x0);
      load4<T, VEC>(x + HALF + i0, x1);
    }
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) ss += x0[i] * x0[i] + x1[i] * x1[i];
    ss = group_sum<LANES>(ss);
    if (h < a.H + a.KV) {
      const float* w = h < a.H ? a.q_norm : a.k_norm;
      const float r = rsqrtf(ss * (1.0f / D) + a.eps);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float y0 = x0[i] * r * w[i0 + i], y1 = x1[i] * r * w[HALF + i0 + i];
        x0[i] = y0 * c[i] - y1 * s[i];
        x1[i] = y0 * s[i] + y1 * c[i];
      }
    }
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) amax = fmaxf(amax, fmaxf(fabsf(x0[i]), fabsf(x1[i])));
    amax = group_max<LANES>(amax);
    if (!on) continue;
    if (h < a.H + a.KV) {
      T* out = h < a.H ? static_cast<T*>(a.q) + static_cast<int64_t>(t) * a.q_ld + static_cast<int64_t>(h) * D
                       : static_cast<T*>(a.k) + static_cast<int64_t>(t) * a.k_ld + static_cast<int64_t>(h - a.H) * D;
      if (h < a.H || a.k) {
        store4<T, VEC>(out + i0, x0);
        store4<T, VEC>(out + HALF + i0, x1);
      }
    }
    if (a.kc && h >= a.H && at >= 0) {
      const bool is_k = h < a.H + a.KV;
      const int kvh = is_k ? h - a.H : h - a.H - a.KV;
      const int64_t r = static_cast<int64_t>(kvh) * a.n_rows + at;
      const float d = __fdiv_rn(amax, 127.0f), id = d != 0.0f ? __fdiv_rn(1.0f, d) : 0.0f;
      int8_t* q8 = (is_k ? a.kc : a.vc) + r * D;
      store_i8x4(q8 + i0, x0, id);
      store_i8x4(q8 + HALF + i0, x1, id);
      if (lane == 0) (is_k ? a.ks : a.vs)[r] = d;
    }
  }
}

template <typename T, int D>
void run_norm_rope(const NormRopeArgs& a, bool vec, int sms, cudaStream_t s) {
  constexpr int GROUPS = kNrThreads / (D / 8);
  const int heads = a.H + a.KV + (a.kc ? a.KV : 0);
  const int slices = (heads + GROUPS - 1) / GROUPS;
  const dim3 grid(static_cast<unsigned>(a.n), static_cast<unsigned>(slices));
  (void)sms;
  if (vec)
    k_qk_norm_rope<T, D, true><<<grid, kNrThreads, 0, s>>>(a);
  else
    k_qk_norm_rope<T, D, false><<<grid, kNrThreads, 0, s>>>(a);
}

template <typename T>
void run_norm_rope_d(const NormRopeArgs& a, int D, bool vec, int sms, cudaStream_t s) {
  if (D == 64) return run_norm_rope<T, 64>(a, vec, sms, s);
  if (D == 128) return run_norm_rope<T, 128>(a, vec, sms, s);
  run_norm_rope<T, 256>(a, vec, sms, s);
}

}  // namespace

void launch_qk_norm_rope(const NormRopeArgs& a, ActType type, int D, int sms, cudaStream_t s) {
  if (a.n <= 0) return;
  // whole words when every row of every buffer starts on one (rows are D apart inside a token, ld apart between them)
  const int word = type == ActType::f32 ? 16 : 8;
  auto whole = [&](const void* p, int64_t ld) {
    return !p || (reinterpret_cast<uintptr_t>(p) % word == 0 && ld % 4 == 0);
  };
  const bool vec = whole(a.qkv, a.ld) && whole(a.q, a.q_ld) && whole(a.k, a.k_ld);
  if (type == ActType::f32) return run_norm_rope_d<float>(a, D, vec, sms, s);
  if (type == ActType::f16) return run_norm_rope_d<__half>(a, D, vec, sms, s);
  run_norm_rope_d<__nv_bfloat16>(a, D, vec, sms, s);
}

}  // namespace mkb
