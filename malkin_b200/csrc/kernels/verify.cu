// Verification of drafted tokens over the whole vocabulary (mk_verify_draft): the exact rejection rule of
// Engine::accept_sampled (engine.cpp:482-507) and Sampler::verify / draw (sampler.cpp:64-97) with p = softmax(l / T) of a
// row's V logits in place of a candidate list.
//
// Draft i of a request is kept while u_i q(d_i) < p(d_i); at the first that is not, the next token is drawn from
// max(p - q, 0) (from p where that leaves nothing), after the last from p of the last row: the lowest index j whose
// running sum reaches u * total among entries above 0. T <= 0: kept while d_i is the row's argmax, next = argmax.
//
//   k_verify_rows  one CTA per (row, vocabulary chunk): maximum, its lowest index, and sum of exp((l - max) / T).
//                  Bound: HBM, every row is read once.
//   k_verify_draw  one cluster of 16 CTAs per request: joins the chunks of each row, walks the drafts, then works on the
//                  one row that the draw needs. A running sum over 151936 entries that is compared with a border has to
//                  be the same for whoever forms it, so this row's exponentials and sums are in 64 bits: with 32 the
//                  drawn index would differ from the exact one about once in 10^4 draws.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cfloat>

#include "common.cuh"
#include "kernels.hpp"
#include "pdl.cuh"
#include "types16.cuh"

namespace cg = cooperative_groups;

namespace mkb {

namespace {

constexpr int kRowThreads = 256;
constexpr int kRowVals = 16;                        // logits a thread holds at a time
constexpr int kRowTile = kRowThreads * kRowVals;    // 4096
constexpr int kDrawThreads = 512, kDrawWarps = kDrawThreads / 32, kDrawCtas = 16;
constexpr int kDrawCache = 12800;                   // 64-bit weights a CTA of the draw keeps in shared memory (two per SM)

struct RowPart {  // of one chunk of a row
  float mx;
  int idx;
  double sum;
};

__host__ __device__ inline int verify_chunk_tiles(int n_rows, int V, int sms) {
  // one tile per CTA while that gives fewer than 8 CTAs per SM, else up to four tiles (fewer, longer CTAs)
  const int64_t tiles = (static_cast<int64_t>(V) + kRowTile - 1) / kRowTile;
  const int64_t per = tiles * n_rows / (8 * static_cast<int64_t>(sms));
  return static_cast<int>(per < 1 ? 1 : per > 4 ? 4 : per);
}

__device__ __forceinline__ bool above(float v, int i, float bv, int bi) { return v > bv || (v == bv && i < bi); }

// One 16-byte word of logits as floats.
template <typename T>
__device__ __forceinline__ void load16b(const T* p, float* v) {
  const uint4 q = ld_stream16(p);
  if constexpr (sizeof(T) == 4) {
    v[0] = __uint_as_float(q.x), v[1] = __uint_as_float(q.y), v[2] = __uint_as_float(q.z), v[3] = __uint_as_float(q.w);
  } else {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = unpack2<T>(w[i]);
      v[2 * i] = f.x, v[2 * i + 1] = f.y;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kRowThreads) k_verify_rows(VerifyArgs a, int tiles, int n_chunks, RowPart* parts) {
  constexpr int W = 16 / sizeof(T);  // values per word
  __shared__ float s_mx[kRowThreads / 32];
  __shared__ int s_idx[kRowThreads / 32];
  __shared__ double s_sum[kRowThreads / 32];
  const int row = blockIdx.x, chunk = blockIdx.y, tid = threadIdx.x;
  const T* l = static_cast<const T*>(a.logits) + static_cast<int64_t>(row) * a.ld;
  const int64_t begin = static_cast<int64_t>(chunk) * tiles * kRowTile;
  const int64_t end = min(begin + static_cast<int64_t>(tiles) * kRowTile, static_cast<int64_t>(a.V));
  // rows whose address is not a multiple of 16 are read value by value
  const bool vec = (reinterpret_cast<uintptr_t>(l) & 15) == 0;
  pdl_launch();
  float v[kRowVals];
  auto load = [&](int64_t at) {  // tile `at`: W-value words, kRowThreads apart; absent values are -inf
#pragma unroll
    for (int b = 0; b < kRowVals / W; ++b) {
      const int64_t i = at + static_cast<int64_t>(b * kRowThreads + tid) * W;
      if (vec && i + W <= end) {
        load16b<T>(l + i, v + b * W);
      } else {
#pragma unroll
        for (int e = 0; e < W; ++e) v[b * W + e] = i + e < end ? to_float(l[i + e]) : -INFINITY;
      }
    }
  };
  load(begin);
  // the row's request: offsets ascend, so it is the number of requests that end at or before the row
  int before = 0;
  for (int r0 = 0; r0 < a.n_req; r0 += kRowThreads)
    before += __syncthreads_count(r0 + tid < a.n_req && a.row_off[r0 + tid + 1] <= row);
  const float T0 = before < a.n_req ? a.temperature[before] : 0.0f;
  const bool sums = T0 > 0.0f;                                      // greedy rows need no sum
  const float c = sums ? fminf(1.44269504088896341f / T0, FLT_MAX) : 0.0f;  // exp(x / T) = 2^(x c)
  float mx = -INFINITY, sum = 0.0f;
  int idx = INT32_MAX;
  for (int64_t at = begin;;) {
    float m = -INFINITY;
#pragma unroll
    for (int e = 0; e < kRowVals; ++e) {
      v[e] = fmaxf(v[e], -INFINITY);  // NaN reads as -inf
      m = fmaxf(m, v[e]);
    }
    if (m > mx) {
      sum = mx > -INFINITY ? sum * exp2f((mx - m) * c) : 0.0f;
      mx = m;
#pragma unroll
      for (int e = kRowVals - 1; e >= 0; --e)
        if (v[e] == m) idx = static_cast<int>(at + static_cast<int64_t>((e / W) * kRowThreads + tid) * W + e % W);
    }
    if (mx > -INFINITY && sums) {
#pragma unroll
      for (int e = 0; e < kRowVals; ++e) sum += exp2f((v[e] - mx) * c);
    }
    at += kRowTile;
    if (at >= end) break;
    load(at);
  }
  // join the block: maximum and index first, then the sums at that maximum
  float bm = mx;
  int bi = idx;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float om = __shfl_xor_sync(0xffffffffu, bm, o);
    const int oi = __shfl_xor_sync(0xffffffffu, bi, o);
    if (above(om, oi, bm, bi)) bm = om, bi = oi;
  }
  double s = mx > -INFINITY ? static_cast<double>(sum * exp2f((mx - bm) * c)) : 0.0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((tid & 31) == 0) s_mx[tid >> 5] = bm, s_idx[tid >> 5] = bi, s_sum[tid >> 5] = s;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < kRowThreads / 32; ++w)
      if (above(s_mx[w], s_idx[w], bm, bi)) bm = s_mx[w], bi = s_idx[w];
    double total = 0.0;
    for (int w = 0; w < kRowThreads / 32; ++w)
      if (s_mx[w] > -INFINITY) total += s_sum[w] * static_cast<double>(exp2f((s_mx[w] - bm) * c));
    parts[static_cast<int64_t>(row) * n_chunks + chunk] = RowPart{bm, bi, total};
  }
}

// 2^t for t <= 0 in 64 bits: t = n + f, |f| <= 1/2, the Taylor series of 2^f to degree 9 (remainder
// (ln 2 / 2)^10 / 10! = 7e-12), n into the exponent. 0 below the normal numbers.
__device__ __forceinline__ double exp2_64(double t) {
  if (!(t > -1000.0)) return 0.0;
  constexpr double kRound = 6755399441055744.0;  // 1.5 * 2^52: adding it leaves round(t) in the low word
  const double m = t + kRound;
  const double f = t - (m - kRound);
  constexpr double L = 0.693147180559945309417;
  constexpr double c1 = L, c2 = c1 * L / 2, c3 = c2 * L / 3, c4 = c3 * L / 4, c5 = c4 * L / 5, c6 = c5 * L / 6,
                   c7 = c6 * L / 7, c8 = c7 * L / 8, c9 = c8 * L / 9;
  double p = c9;
  p = fma(p, f, c8);
  p = fma(p, f, c7);
  p = fma(p, f, c6);
  p = fma(p, f, c5);
  p = fma(p, f, c4);
  p = fma(p, f, c3);
  p = fma(p, f, c2);
  p = fma(p, f, c1);
  p = fma(p, f, 1.0);
  return __hiloint2double(__double2hiint(p) + (__double2loint(m) << 20), __double2loint(p));
}

// Maximum, lowest index and sum of a row from its chunks, by one warp; every lane gets them.
__device__ __forceinline__ void join_row(const RowPart* parts, int n_chunks, double c, int lane, float& mx, int& idx,
                                         double& sum) {
  mx = -INFINITY;
  idx = INT32_MAX;
  for (int i = lane; i < n_chunks; i += 32)
    if (above(parts[i].mx, parts[i].idx, mx, idx)) mx = parts[i].mx, idx = parts[i].idx;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float om = __shfl_xor_sync(0xffffffffu, mx, o);
    const int oi = __shfl_xor_sync(0xffffffffu, idx, o);
    if (above(om, oi, mx, idx)) mx = om, idx = oi;
  }
  sum = 0.0;
  for (int i = lane; i < n_chunks; i += 32)
    if (parts[i].mx > -INFINITY)
      sum += parts[i].sum * exp2_64((static_cast<double>(parts[i].mx) - static_cast<double>(mx)) * c);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
}

constexpr int kDrawRows = 64;  // rows of a request whose maximum is kept from the walk over its drafts

struct DrawShared {
  int first;                 // first draft that was not kept
  float mx[kDrawRows];
  int idx[kDrawRows];
  double warp[kDrawWarps];   // sums of the warps' segments
  double sum[2];             // of this CTA: normalisation, weights
};

template <typename T>
__global__ void __launch_bounds__(kDrawThreads, 2)
    k_verify_draw(VerifyArgs a, int n_chunks, const RowPart* parts, int seg, bool kept) {
  extern __shared__ double cache[];
  __shared__ DrawShared sh;
  cg::cluster_group cluster = cg::this_cluster();
  const int r = blockIdx.x / kDrawCtas, rank = static_cast<int>(cluster.block_rank());
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int lo = a.row_off[r], hi = a.row_off[r + 1];
  const bool valid = lo >= r && hi > lo && hi <= a.n_rows && hi - 1 - r <= a.n_rows - a.n_req;
  const float temp = a.temperature[r];
  pdl_wait();
  if (!valid) {  // the same for all CTAs of the cluster
    if (rank == 0 && tid == 0) {
      a.n_acc[r] = 0;
      a.next[r] = -1;
      if (a.status) atomicCAS(a.status, 0, kStatusBadIndex);
    }
    return;
  }
  const int k = hi - lo - 1, j0 = lo - r;  // drafts and their first index
  const bool greedy = !(temp > 0.0f);
  const double c = greedy ? 0.0 : 1.4426950408889634074 / static_cast<double>(temp);
  const T* logits = static_cast<const T*>(a.logits);
  if (tid == 0) sh.first = k;
  __syncthreads();
  for (int i = warp; i <= k; i += kDrawWarps) {
    const int d = i < k ? a.draft[j0 + i] : -1;
    const bool in = d >= 0 && d < a.V;
    float l = -INFINITY, qd = 0.0f;
    if (in && !greedy) {  // issued before the chunks are joined
      l = to_float(logits[static_cast<int64_t>(lo + i) * a.ld + d]);
      qd = a.q ? a.q[static_cast<int64_t>(j0 + i) * a.q_ld + d] : 1.0f;
    }
    const double ui = a.u[lo + i];
    float mx;
    int idx;
    double sum;
    join_row(parts + static_cast<int64_t>(lo + i) * n_chunks, n_chunks, c, lane, mx, idx, sum);
    if (lane == 0) {
      if (i < kDrawRows) sh.mx[i] = mx, sh.idx[i] = idx;
      if (i < k) {
        const bool some = mx > -INFINITY && mx < INFINITY;
        double p = 0.0;
        bool keep;
        if (greedy) {
          p = some && d == idx ? 1.0 : 0.0;
          keep = p > 0.0;
        } else {
          if (some) p = exp2_64((static_cast<double>(fmaxf(l, -INFINITY)) - static_cast<double>(mx)) * c) / sum;
          keep = qd > 0.0f && ui * static_cast<double>(qd) < p;
        }
        if (!keep) atomicMin(&sh.first, i);
        if (rank == 0 && a.p) a.p[j0 + i] = static_cast<float>(p);
      }
    }
  }
  __syncthreads();
  const int stop = sh.first;
  if (rank == 0) {
    if (a.p)
      for (int i = stop + 1 + tid; i < k; i += kDrawThreads) a.p[j0 + i] = 0.0f;  // never looked at
    if (tid == 0) a.n_acc[r] = stop;
  }
  const int row = lo + stop;
  float mx;
  int idx;
  if (stop < kDrawRows) {
    mx = sh.mx[stop];
    idx = sh.idx[stop];
  } else {
    double unused;
    join_row(parts + static_cast<int64_t>(row) * n_chunks, n_chunks, c, lane, mx, idx, unused);
  }
  if (greedy || !(mx > -INFINITY && mx < INFINITY)) {
    if (rank == 0 && tid == 0) a.next[r] = mx > -INFINITY && mx < INFINITY ? idx : -1;
    return;
  }
  const T* l = logits + static_cast<int64_t>(row) * a.ld;
  const bool reject = stop < k;
  const int d = reject ? a.draft[j0 + stop] : -1;
  const float* q = reject && a.q ? a.q + static_cast<int64_t>(j0 + stop) * a.q_ld : nullptr;
  const double u = a.u[row + (reject ? 1 : 0)];
  // this CTA's slice of the vocabulary: a contiguous segment of seg values for each warp, a value per lane and step (the
  // 64-bit weights of a step then lie in consecutive banks; four values a lane took 8 wavefronts a store where this takes 2)
  const int s0 = rank * kDrawWarps * seg;
  const int w0 = min(a.V, s0 + warp * seg), w1 = min(a.V, w0 + seg);
  auto weigh = [&](float x) {
    return exp2_64((static_cast<double>(fmaxf(x, -INFINITY)) - static_cast<double>(mx)) * c);
  };
  // sums of the CTAs, in rank order
  auto cluster_sum = [&](int which, double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (lane == 0) sh.warp[warp] = v;
    __syncthreads();
    if (tid == 0) {
      double t = 0.0;
      for (int w = 0; w < kDrawWarps; ++w) t += sh.warp[w];
      sh.sum[which] = t;
    }
    cluster.sync();
    double t = 0.0;
    for (int o = 0; o < kDrawCtas; ++o) t += cluster.map_shared_rank(&sh, o)->sum[which];
    return t;
  };
  // kU steps' loads are issued before the first is used, those of the draft probabilities before the clusters meet over the
  // normalisation. The weights stay in shared memory (kept) unless a slice is too long for it; those are formed again.
  constexpr int kU = 10;
  float x[kU];
  auto load = [&](auto* from, int j, float fill) {
#pragma unroll
    for (int g = 0; g < kU; ++g) x[g] = j + 32 * g < w1 ? to_float(from[j + 32 * g]) : fill;
  };
  double v = 0.0;
  for (int j = w0 + lane; j < w1; j += 32 * kU) {
    load(l, j, -INFINITY);
#pragma unroll
    for (int g = 0; g < kU; ++g) {
      const double e = weigh(x[g]);  // 0 past the segment
      if (kept && j + 32 * g < w1) cache[j + 32 * g - s0] = e;
      v += e;
    }
  }
  if (q) load(q, w0 + lane, 0.0f);
  const double Z = cluster_sum(0, v);
  bool residual = reject;
  double total = Z;
  auto rest = [&](int j, double e, float qj) {
    if (q) {
      const double left = e - static_cast<double>(qj) * Z;
      return left > 0.0 ? left : 0.0;
    }
    return j == d ? 0.0 : e;  // a draft without probabilities is certain of itself
  };
  if (residual) {
    v = 0.0;
    if (kept) {
      for (int j = w0 + lane; j < w1; j += 32 * kU) {
        if (q && j != w0 + lane) load(q, j, 0.0f);
#pragma unroll
        for (int g = 0; g < kU; ++g) {
          const int at = j + 32 * g;
          if (at < w1) {
            const double e = rest(at, cache[at - s0], x[g]);
            cache[at - s0] = e;
            v += e;
          }
        }
      }
    } else {
#pragma unroll 1
      for (int j = w0 + lane; j < w1; j += 32) v += rest(j, weigh(to_float(l[j])), q ? q[j] : 0.0f);
    }
    total = cluster_sum(1, v);
    if (!(total > 0.0)) {  // p <= q everywhere: draw from p
      residual = false;
      total = Z;
      v = 0.0;
      for (int j = w0 + lane; j < w1; j += 32) {
        const double e = weigh(to_float(l[j]));
        if (kept) cache[j - s0] = e;
        v += e;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
      __syncthreads();
      if (lane == 0) sh.warp[warp] = v;
    }
  }
  __syncthreads();
  const int which = residual ? 1 : 0;
  const double target = u * total;
  // the CTA, the warp, the lane and the entry that the running sum reaches the target in; where rounding leaves a part
  // short of its own sum, its last entry above 0
  double before = 0.0;
  int owner = -1;
  double owner_before = 0.0;
  for (int o = 0; o < kDrawCtas; ++o) {
    const double t = cluster.map_shared_rank(&sh, o)->sum[which];
    if (t > 0.0) {
      owner = o;
      owner_before = before;
      if (before + t >= target) break;
    }
    before += t;
  }
  cluster.sync();  // every CTA has read the sums
  if (owner != rank) return;
  before = owner_before;
  int ow = -1;
  double warp_before = before;
  for (int w = 0; w < kDrawWarps; ++w) {
    const double t = sh.warp[w];
    if (t > 0.0) {
      ow = w;
      warp_before = before;
      if (before + t >= target) break;
    }
    before += t;
  }
  if (warp != ow) return;
  auto value = [&](int j) {
    if (kept) return cache[j - s0];
    const double e = weigh(to_float(l[j]));
    return residual ? rest(j, e, q ? q[j] : 0.0f) : e;
  };
  const int part = ((w1 - w0 + 31) / 32) | 1;  // odd: the lanes' values lie in different banks
  const int p0 = min(w1, w0 + lane * part), p1 = min(w1, p0 + part);
  double mine = 0.0;
#pragma unroll 1
  for (int j = p0; j < p1; ++j) mine += value(j);
  double incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double y = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += y;
  }
  const unsigned reach = __ballot_sync(0xffffffffu, mine > 0.0 && warp_before + incl >= target);
  const unsigned some = __ballot_sync(0xffffffffu, mine > 0.0);
  const int pick = reach ? __ffs(reach) - 1 : 31 - __clz(some);
  // the picked lane's values by the whole warp, 32 at a time, in order
  const int c0 = __shfl_sync(0xffffffffu, p0, pick), c1 = __shfl_sync(0xffffffffu, p1, pick);
  double run = warp_before + __shfl_sync(0xffffffffu, incl - mine, pick);
  int found = -1;
  for (int j = c0; j < c1; j += 32) {
    double e = j + lane < c1 ? value(j + lane) : 0.0;
    double s = e;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double y = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += y;
    }
    const unsigned pos = __ballot_sync(0xffffffffu, e > 0.0);
    const unsigned hit = __ballot_sync(0xffffffffu, e > 0.0 && run + s >= target);
    if (hit) {
      found = j + __ffs(hit) - 1;
      break;
    }
    if (pos) found = j + 31 - __clz(pos);
    run += __shfl_sync(0xffffffffu, s, 31);
  }
  if (lane == 0) a.next[r] = found;
}

template <typename T>
int run_verify(const VerifyArgs& a, int sms, cudaStream_t s) {
  const int tiles = verify_chunk_tiles(a.n_rows, a.V, sms);
  const int n_chunks = static_cast<int>((static_cast<int64_t>(a.V) + static_cast<int64_t>(tiles) * kRowTile - 1) /
                                        (static_cast<int64_t>(tiles) * kRowTile));
  RowPart* parts = static_cast<RowPart*>(a.ws);
  k_verify_rows<T><<<dim3(static_cast<unsigned>(a.n_rows), static_cast<unsigned>(n_chunks)), kRowThreads, 0, s>>>(
      a, tiles, n_chunks, parts);
  const int seg = (a.V + kDrawCtas * kDrawWarps * 32 - 1) / (kDrawCtas * kDrawWarps * 32) * 32;
  const bool kept = seg * kDrawWarps <= kDrawCache;
  const size_t smem = kept ? static_cast<size_t>(seg) * kDrawWarps * sizeof(double) : 0;
  static bool set[kMaxDevices] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= kMaxDevices) return cudaErrorInvalidDevice;
  if (!set[dev]) {
    e = cudaFuncSetAttribute(k_verify_draw<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             kDrawCache * static_cast<int>(sizeof(double)));
    if (e == cudaSuccess) e = cudaFuncSetAttribute(k_verify_draw<T>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
    set[dev] = true;
  }
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  return launch_pdl(k_verify_draw<T>, dim3(static_cast<unsigned>(a.n_req) * kDrawCtas), dim3(kDrawThreads), smem, s, kDrawCtas, a,
                    n_chunks, static_cast<const RowPart*>(parts), seg, kept);
}

}  // namespace

int64_t verify_workspace(int n_rows, int V) {
  // chunks of one tile are the most a row can have
  const int64_t chunks = (static_cast<int64_t>(V) + kRowTile - 1) / kRowTile;
  return std::max<int64_t>(256, chunks * n_rows * static_cast<int64_t>(sizeof(RowPart)));
}

int launch_verify_draft(const VerifyArgs& a, ActType type, int sms, cudaStream_t s) {
  if (a.n_req <= 0) return cudaSuccess;
  if (type == ActType::f32) return run_verify<float>(a, sms, s);
  if (type == ActType::f16) return run_verify<__half>(a, sms, s);
  return run_verify<__nv_bfloat16>(a, sms, s);
}

}  // namespace mkb
