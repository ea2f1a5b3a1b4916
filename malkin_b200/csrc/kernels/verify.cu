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
//   k_verify_norm  CTAs (request, chunk): each joins the chunks of the request's rows and walks its drafts (a warp a row;
//                  cheaper than a kernel of its own), then the chunk's share of the normalisation of the one row that the
//                  draw needs
//   k_verify_rest  CTAs (request, chunk): the chunk's share of the draw's total
//   k_verify_pick  one CTA per request: the chunk, the segment and the token the running sum reaches its target in
// A running sum over 151936 entries that is compared with a border has to be the same for whoever forms it, so the drawn
// row's exponentials and sums are in 64 bits: with 32 the drawn index would differ from the exact one about once in 10^4
// draws. An acceptance compares with one probability: its exponential is in 64 bits, its row's sum is k_verify_rows' of
// 32-bit exponentials (4e-7 of itself at most over the measured rows), and where that could decide, the row is summed again
// in 64 bits. All sums are taken in a fixed order. (Clusters of 4, 8 or 16 CTAs a request that kept the row in shared
// memory were slower: 93, 85 and 96 us against 75 us at 64 requests of 5 rows; a cluster barrier waits for its slowest SM
// three times.)
// Measured, V = 151936: 64 requests of 5 fp32 rows with probabilities 79 us, of which k_verify_rows 35 (5.6 TB/s, 0.85 of a
// copy's rate); one request of 9 fp32 rows 19 us, 8 requests of up to 9 bf16 rows 24, both held by four dependent launches.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cfloat>

#include "common.cuh"
#include "kernels.hpp"
#include "pdl.cuh"
#include "tcgen05.cuh"
#include "types16.cuh"

namespace mkb {

namespace {

constexpr int kRowThreads = 256;
constexpr int kRowVals = 16;                        // logits a thread holds at a time
constexpr int kRowTile = kRowThreads * kRowVals;    // 4096
constexpr int kRowTilesMax = 8;                     // of a CTA
constexpr int kDrawThreads = 256, kDrawVals = 16;   // of the normalisation and the rest
constexpr int kDrawChunk = kDrawThreads * kDrawVals;
constexpr int kPickThreads = 512, kPickWarps = kPickThreads / 32;

struct RowPart {  // of one chunk of a row
  float mx;
  int idx;
  double sum;
};

struct Decision {  // of a request
  int32_t draw;    // 1: the token is drawn from `row`; 0: it is written already
  int32_t row;     // logits row
  int32_t draft;   // index of the draft refused there, -1: none
  int32_t token;   // that draft
  float mx, pad;
  double c, u;     // log2 e / T, the draw's uniform
};

int verify_chunk_tiles(int n_rows, int V, int sms) {
  // as many tiles a CTA as give four CTAs per SM, one wave, in which the next tile's loads run under this one's work
  const int64_t tiles = (static_cast<int64_t>(V) + kRowTile - 1) / kRowTile;
  const int64_t per = (tiles * n_rows + 4 * sms - 1) / (4 * sms);
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(per, kRowTilesMax)));
}

// The rows of request r lie in the buffers, and so do its drafts (row x of it has draft x - r).
__device__ __forceinline__ bool rows_fit(const VerifyArgs& a, int r, int lo, int hi) {
  return lo >= r && hi > lo && hi <= a.n_rows && hi - 1 - r <= a.n_rows - a.n_req;
}

__device__ __forceinline__ bool above(float v, int i, float bv, int bi) { return v > bv || (v == bv && i < bi); }

template <typename T>
__device__ __forceinline__ void unpack16b(uint4 q, float* v) {
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
__global__ void __launch_bounds__(kRowThreads, 4) k_verify_rows(VerifyArgs a, int tiles, int n_chunks, RowPart* parts) {
  constexpr int W = 16 / sizeof(T), N = kRowVals / W;  // values of a word, words of a thread
  __shared__ float s_mx[kRowThreads / 32];
  __shared__ int s_idx[kRowThreads / 32];
  __shared__ double s_sum[kRowThreads / 32];
  __shared__ int s_req;
  const int row = blockIdx.x, chunk = blockIdx.y, tid = threadIdx.x;
  const T* l = static_cast<const T*>(a.logits) + static_cast<int64_t>(row) * a.ld;
  const int64_t begin = static_cast<int64_t>(chunk) * tiles * kRowTile;
  const int64_t end = min(begin + static_cast<int64_t>(tiles) * kRowTile, static_cast<int64_t>(a.V));
  // rows whose address is not a multiple of 16 are read value by value
  const bool vec = (reinterpret_cast<uintptr_t>(l) & 15) == 0;
  pdl_launch();
  uint4 raw[N];
  auto load = [&](int64_t at) {  // tile `at`: words kRowThreads apart; absent values are -inf
#pragma unroll
    for (int b = 0; b < N; ++b) {
      const int64_t i = at + static_cast<int64_t>(b * kRowThreads + tid) * W;
      if (vec && i + W <= end) {
        raw[b] = ld_stream16(l + i);
      } else {
        alignas(16) T one[W];
#pragma unroll
        for (int e = 0; e < W; ++e) one[e] = i + e < end ? l[i + e] : from_float<T>(-INFINITY);
        raw[b] = *reinterpret_cast<const uint4*>(one);
      }
    }
  };
  load(begin);
  // the row's request: the first one whose own offsets hold it. A request that is not refused has no row of an earlier one
  // that fits, so offsets that are wrong elsewhere do not change it.
  if (tid == 0) s_req = a.n_req;
  __syncthreads();
  for (int r = tid; r < a.n_req; r += kRowThreads) {
    const int lo = a.row_off[r], hi = a.row_off[r + 1];
    if (row >= lo && row < hi && rows_fit(a, r, lo, hi)) atomicMin(&s_req, r);
  }
  __syncthreads();
  const float T0 = s_req < a.n_req ? a.temperature[s_req] : 0.0f;
  const bool sums = T0 > 0.0f;  // rows of a greedy request need the index of the maximum, the others the sum
  // exp(x / T) = 2^(x c); above 0, so that -infinity keeps its weight 0 where T is infinite
  const float c = sums ? fmaxf(fminf(1.44269504088896341f / T0, FLT_MAX), FLT_MIN) : 0.0f;
  float mx = -INFINITY, sum = 0.0f;
  int idx = INT32_MAX;
  for (int64_t at = begin; at < end; at += kRowTile) {
    float v[kRowVals];
#pragma unroll
    for (int b = 0; b < N; ++b) unpack16b<T>(raw[b], v + b * W);
    if (at + kRowTile < end) load(at + kRowTile);
    float m = -INFINITY;  // fmaxf passes over NaN
#pragma unroll
    for (int e = 0; e < kRowVals; ++e) m = fmaxf(m, v[e]);
    if (m > mx) {
      sum = mx > -INFINITY ? sum * ex2_approx((mx - m) * c) : 0.0f;
      mx = m;
      if (!sums) {
#pragma unroll
        for (int e = kRowVals - 1; e >= 0; --e)
          if (v[e] == m) idx = static_cast<int>(at + static_cast<int64_t>((e / W) * kRowThreads + tid) * W + e % W);
      }
    }
    if (mx > -INFINITY && sums) {
#pragma unroll
      for (int e = 0; e < kRowVals; ++e) sum += ex2_approx((fmaxf(v[e], -INFINITY) - mx) * c);
    }
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
  double s = mx > -INFINITY ? static_cast<double>(sum * ex2_approx((mx - bm) * c)) : 0.0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((tid & 31) == 0) s_mx[tid >> 5] = bm, s_idx[tid >> 5] = bi, s_sum[tid >> 5] = s;
  __syncthreads();
  if (tid < 32) {
    constexpr int kW = kRowThreads / 32;
    const bool in = tid < kW;
    const float wm = in ? s_mx[tid] : -INFINITY;
    bm = wm;
    bi = in ? s_idx[tid] : INT32_MAX;
#pragma unroll
    for (int o = kW / 2; o > 0; o >>= 1) {
      const float om = __shfl_xor_sync(0xffffffffu, bm, o);
      const int oi = __shfl_xor_sync(0xffffffffu, bi, o);
      if (above(om, oi, bm, bi)) bm = om, bi = oi;
    }
    double total = in && wm > -INFINITY ? s_sum[tid] * static_cast<double>(ex2_approx((wm - bm) * c)) : 0.0;
#pragma unroll
    for (int o = kW / 2; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    if (tid == 0) parts[static_cast<int64_t>(row) * n_chunks + chunk] = RowPart{bm, bi, total};
  }
}

// 2^t, t = x c, for -1000 < t <= 0 in 64 bits: t = n + k / 16 + f with |f| <= 1/32, 2^(k/16) from a table of 16 (one row of
// shared memory's banks), the Taylor series of 2^f to degree 5 (remainder (ln 2 / 32)^6 / 6! = 1.4e-13), n into the exponent.
// The product is fused into its two uses by name: every kernel that forms a weight has to round it alike.
__device__ __forceinline__ double exp2_64(double x, double c, const double* tab) {
  constexpr double kRound = 6755399441055744.0 / 16;  // 1.5 * 2^48: adding it leaves round(16 t) in the low word
  const double m = fma(x, c, kRound);
  const double f = fma(x, c, kRound - m);
  const int q = __double2loint(m);
  constexpr double L = 0.693147180559945309417;
  constexpr double c1 = L, c2 = c1 * L / 2, c3 = c2 * L / 3, c4 = c3 * L / 4, c5 = c4 * L / 5;
  double p = c5;
  p = fma(p, f, c4);
  p = fma(p, f, c3);
  p = fma(p, f, c2);
  p = fma(p, f, c1);
  p = fma(p, f, 1.0) * tab[q & 15];
  return __hiloint2double(__double2hiint(p) + ((q >> 4) << 20), __double2loint(p));
}
// exp((x - mx) / T) in 64 bits with c = log2 e / T: 0 for -infinity, NaN and what is below 2^-1000.
__device__ __forceinline__ double weigh64(float x, float mx, double c, const double* tab) {
  const double d = static_cast<double>(fmaxf(x, -INFINITY)) - static_cast<double>(mx);
  return d * c > -1000.0 ? exp2_64(d, c, tab) : 0.0;
}
__constant__ double kSixteenths[16] = {  // 2^(k/16)
    1.0, 1.0442737824274138403, 1.0905077326652576592, 1.1387886347566916537, 1.1892071150027210667,
    1.2418578120734840486, 1.2968395546510096659, 1.3542555469368927283, 1.4142135623730950488, 1.4768261459394993114,
    1.5422108254079408236, 1.6104903319492543082, 1.6817928305074290861, 1.7562521603732994831, 1.8340080864093424635,
    1.9152065613971472939};

// Maximum, lowest index and sum of a row from its chunks, by one warp; every lane gets them.
__device__ __forceinline__ void join_row(const RowPart* parts, int n_chunks, double c, const double* tab, int lane,
                                         float& mx, int& idx, double& sum) {
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
    if (parts[i].mx > -INFINITY) sum += parts[i].sum * weigh64(parts[i].mx, mx, c, tab);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
}

__device__ __forceinline__ double block_sum(double v, double* part) {  // the same on every thread; part: a value a warp
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  double t = 0.0;
  for (unsigned w = 0; w < blockDim.x / 32; ++w) t += part[w];
  return t;
}

// Weight of a draw before normalisation: exp((l - mx) / T), and where a draft was refused what is left of it beside the
// draft's probabilities (Z: the row's sum).
struct Weigh {
  float mx, cf;
  double mx64, c, Z;
  const double* tab;
  bool dense;   // a draft with probabilities was refused
  int token;    // a certain draft that was refused, -1
  __device__ __forceinline__ Weigh(const Decision& d, const double* t, bool with_q)
      : mx(d.mx), cf(fminf(static_cast<float>(d.c), FLT_MAX)), mx64(static_cast<double>(d.mx)), c(d.c), Z(0.0), tab(t),
        dense(d.draft >= 0 && with_q), token(d.draft >= 0 && !with_q ? d.token : -1) {}
  __device__ __forceinline__ double whole(float x) const {
    const bool some = (x - mx) * cf > -1000.0f;  // selected, not branched on: the chains of several calls interleave
    const double y = exp2_64(static_cast<double>(some ? x : mx) - mx64, c, tab);
    return some ? y : 0.0;
  }
  __device__ __forceinline__ double rest(int j, float x, float q) const {
    const double e = whole(x);
    if (!dense) return j == token ? 0.0 : e;
    const double left = fma(-static_cast<double>(fminf(q, INFINITY)), Z, e);  // a NaN probability leaves nothing
    return __double2hiint(left) < 0 ? 0.0 : left;
  }
};

// A thread's values of one of the draw's chunks, kDrawThreads apart; `fill` past the row's end.
template <typename T>
__device__ __forceinline__ void load_chunk(const T* row, int chunk, int V, T fill, T (&v)[kDrawVals]) {
  const int j0 = chunk * kDrawChunk + static_cast<int>(threadIdx.x);  // V is at most 2^27
  const T* p = row + j0;
  if ((chunk + 1) * static_cast<int64_t>(kDrawChunk) <= V) {
#pragma unroll
    for (int g = 0; g < kDrawVals; ++g) v[g] = p[g * kDrawThreads];
  } else {
#pragma unroll
    for (int g = 0; g < kDrawVals; ++g) v[g] = j0 + g * kDrawThreads < V ? p[g * kDrawThreads] : fill;
  }
}

// Where u q(d) lies this near p(d), relative to it, the row's sum is formed again in 64 bits. The sum behind p is of 32-bit
// exponentials 2^t and off by less than 120 x 2^-23 < 2^-16 of itself for rows of up to 2^27 tokens: t carries three roundings,
// 1.5 x 2^-23 |t| ln 2 of a weight, and the mean of |t| under the weights is at most log2 V = 27 (28); 2^x is good to 2^-22 (2);
// a thread adds at most 128 weights (64) and brings them to a larger maximum at most 8 times, its block and warp once (25).
constexpr double kClose = 1.0 / (1 << 15);

// Grid: (CTAs of a request, request); each takes `per` of the draw's chunks.
template <typename T>
__global__ void __launch_bounds__(kDrawThreads, 4) k_verify_norm(VerifyArgs a, int n_chunks, const RowPart* parts,
                                                              Decision* decide, double* zpart, int chunks, int per) {
  __shared__ double tab[16], part[kDrawThreads / 32];
  __shared__ int first, close;  // draft that is not kept, that is too close to tell; `last`: none
  __shared__ int from, last;    // drafts before `from` are kept, that at `last` is not (k: none)
  const int r = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int lo = a.row_off[r], hi = a.row_off[r + 1];
  const float temp = a.temperature[r];
  // refused too: a request with drafts (which implies: or rows) that an earlier one has
  bool over = !rows_fit(a, r, lo, hi);
  for (int e = tid; e < r && !over; e += kDrawThreads) {
    const int lo_e = a.row_off[e], hi_e = a.row_off[e + 1];
    over = rows_fit(a, e, lo_e, hi_e) && hi_e - 1 - e > lo - r;
  }
  const bool valid = !__syncthreads_or(over);
  if (tid < 16) tab[tid] = kSixteenths[tid];
  const bool writer = blockIdx.x == 0;
  pdl_launch();
  if (!valid) {
    if (writer && tid == 0) {
      a.n_acc[r] = 0;
      a.next[r] = -1;
      decide[r].draw = 0;
      if (a.status) atomicCAS(a.status, 0, kStatusBadIndex);
    }
    pdl_wait();
    return;
  }
  const int k = hi - lo - 1, j0 = lo - r;  // drafts and their first index
  const bool greedy = !(temp > 0.0f);
  const double c = greedy ? 0.0 : 1.4426950408889634074 / static_cast<double>(temp);
  const T* logits = static_cast<const T*>(a.logits);
  const int c0 = blockIdx.x * per, c1 = min(chunks, c0 + per);
  // Once around as a rule. A draft that is too close to tell takes a turn of its own, in which every CTA forms the whole sum of
  // its row by the code that forms the chunks' shares (a second copy of that code costs 0.7 us a call without being reached, this
  // 0.3 to 0.9).
  if (tid == 0) from = 0, first = close = last = k;
  __syncthreads();
  pdl_wait();
  for (;;) {
    for (int i = from + warp; i < last; i += kDrawThreads / 32) {
      const int d = a.draft[j0 + i];
      const bool in = d >= 0 && d < a.V;
      float l = -INFINITY, qd = 0.0f;
      if (in && !greedy) {
        l = to_float(logits[static_cast<int64_t>(lo + i) * a.ld + d]);
        qd = a.q ? a.q[static_cast<int64_t>(j0 + i) * a.q_ld + d] : 1.0f;
      }
      const double ui = a.u[lo + i];
      float mx;
      int idx;
      double sum;
      join_row(parts + static_cast<int64_t>(lo + i) * n_chunks, n_chunks, c, tab, lane, mx, idx, sum);
      if (lane == 0) {
        const bool some = mx > -INFINITY && mx < INFINITY;
        double p = 0.0;
        bool keep, near = false;
        if (greedy) {
          p = some && d == idx ? 1.0 : 0.0;
          keep = p > 0.0;
        } else {
          if (some) p = weigh64(l, mx, c, tab) / sum;
          const double uq = ui * static_cast<double>(qd);
          keep = qd > 0.0f && uq < p;
          near = qd > 0.0f && p > 0.0 && fabs(uq - p) <= kClose * p;
        }
        if (near)
          atomicMin(&close, i);
        else if (!keep)
          atomicMin(&first, i);
        if (writer && a.p) a.p[j0 + i] = static_cast<float>(p);
      }
    }
    __syncthreads();
    const int stop = min(first, close), row = lo + stop;
    const bool settle = close < first;
    Decision d;
    int idx;
    double unused;
    join_row(parts + static_cast<int64_t>(row) * n_chunks, n_chunks, c, tab, lane, d.mx, idx, unused);
    const bool some = d.mx > -INFINITY && d.mx < INFINITY;
    d.draw = some && !greedy;
    d.row = row;
    d.draft = stop < k ? j0 + stop : -1;
    d.token = stop < k ? a.draft[j0 + stop] : -1;
    d.c = c;
    d.u = a.u[row + (stop < k ? 1 : 0)];
    d.pad = 0.0f;
    if (writer && !settle) {
      if (a.p)
        for (int i = stop + 1 + tid; i < k; i += kDrawThreads) a.p[j0 + i] = 0.0f;  // never looked at
      if (tid == 0) {
        a.n_acc[r] = stop;
        decide[r] = d;
        if (!d.draw) a.next[r] = some ? idx : -1;
      }
    }
    if (!d.draw) return;
    const T* l = logits + static_cast<int64_t>(row) * a.ld;
    const Weigh w(d, tab, a.q != nullptr);
    T next[kDrawVals];
    auto load = [&](int chunk) { load_chunk(l, chunk, a.V, from_float<T>(-INFINITY), next); };
    const int end = settle ? chunks : c1;
    double v = 0.0;
    load(settle ? 0 : c0);
    for (int chunk = settle ? 0 : c0; chunk < end; ++chunk) {
      float x[kDrawVals];
#pragma unroll
      for (int g = 0; g < kDrawVals; ++g) x[g] = to_float(next[g]);
      if (chunk + 1 < end) load(chunk + 1);
#pragma unroll
      for (int g = 0; g < kDrawVals; ++g) v += w.whole(x[g]);
      if (settle) continue;
      v = block_sum(v, part);
      if (tid == 0) zpart[static_cast<int64_t>(r) * chunks + chunk] = v;
      v = 0.0;
    }
    if (!settle) return;
    // a draft that is too close has a token and a q above 0
    const double p = w.whole(to_float(l[d.token])) / block_sum(v, part);
    const double uq = a.u[row] * static_cast<double>(a.q ? a.q[static_cast<int64_t>(d.draft) * a.q_ld + d.token] : 1.0f);
    if (writer && a.p && tid == 0) a.p[d.draft] = static_cast<float>(p);
    if (tid == 0) {  // block_sum's barriers lie behind the last use of these
      from = uq < p ? stop + 1 : stop;
      if (!(uq < p)) last = stop;
      first = close = last;
    }
    __syncthreads();
  }
}

template <typename T>
__global__ void __launch_bounds__(kDrawThreads, 4) k_verify_rest(VerifyArgs a, const Decision* decide, const double* zpart,
                                                              double* rpart, double* zsum) {
  __shared__ double tab[16], part[kDrawThreads / 32];
  const int r = blockIdx.y, chunk = blockIdx.x, tid = threadIdx.x;
  if (tid < 16) tab[tid] = kSixteenths[tid];
  __syncthreads();
  pdl_launch();
  pdl_wait();
  const Decision d = decide[r];
  if (!d.draw || d.draft < 0) return;  // drawn from p itself: the shares are the normalisation's
  const T* l = static_cast<const T*>(a.logits) + static_cast<int64_t>(d.row) * a.ld;
  const float* q = a.q ? a.q + static_cast<int64_t>(d.draft) * a.q_ld : nullptr;
  T x[kDrawVals];
  float y[kDrawVals] = {};
  load_chunk(l, chunk, a.V, from_float<T>(-INFINITY), x);
  if (q) load_chunk(q, chunk, a.V, 0.0f, y);
  Weigh w(d, tab, q != nullptr);
  double z = 0.0;
  for (unsigned i = tid; i < gridDim.x; i += kDrawThreads) z += zpart[static_cast<int64_t>(r) * gridDim.x + i];
  w.Z = block_sum(z, part);
  if (chunk == 0 && tid == 0) zsum[r] = w.Z;  // the pick takes this one: a sum in another order could move a residual's sign
  double v = 0.0;
#pragma unroll
  for (int g = 0; g < kDrawVals; ++g) v += w.rest(chunk * kDrawChunk + g * kDrawThreads + tid, to_float(x[g]), y[g]);
  v = block_sum(v, part);
  if (tid == 0) rpart[static_cast<int64_t>(r) * gridDim.x + chunk] = v;
}

// Where a running sum over parts reaches the target: the first part above 0 at or past it, else the last above 0 (where
// rounding leaves the parts short of their total). One warp; before: the sum ahead of that part.
__device__ __forceinline__ int reach(const double* p, int n, double target, int lane, double& before) {
  double run = before;
  int found = -1;
  for (int i0 = 0; i0 < n; i0 += 32) {
    const double t = i0 + lane < n ? p[i0 + lane] : 0.0;
    double s = t;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double y = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += y;
    }
    const unsigned some = __ballot_sync(0xffffffffu, t > 0.0);
    const unsigned hit = __ballot_sync(0xffffffffu, t > 0.0 && run + s >= target);
    const unsigned at = hit ? hit & (0u - hit) : some ? 0x80000000u >> __clz(some) : 0u;
    if (at) {
      const int src = __ffs(at) - 1;
      found = i0 + src;
      before = run + __shfl_sync(0xffffffffu, s - t, src);
    }
    if (hit) break;
    run += __shfl_sync(0xffffffffu, s, 31);
  }
  return found;
}

template <typename T>
__global__ void __launch_bounds__(kPickThreads) k_verify_pick(VerifyArgs a, const Decision* decide, const double* zpart,
                                                              const double* rpart, const double* zsum, int chunks) {
  __shared__ double tab[16], part[2][kPickWarps], seg[kPickWarps];
  const int r = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid < 16) tab[tid] = kSixteenths[tid];
  pdl_wait();
  Decision d = decide[r];
  if (!d.draw) return;
  const T* l = static_cast<const T*>(a.logits) + static_cast<int64_t>(d.row) * a.ld;
  const double* zp = zpart + static_cast<int64_t>(r) * chunks;
  const double* rp = rpart + static_cast<int64_t>(r) * chunks;
  const double zs = d.draft >= 0 ? zsum[r] : 0.0;
  double z = 0.0, t = 0.0;
  for (int i = tid; i < chunks; i += kPickThreads) {
    z += zp[i];
    if (d.draft >= 0) t += rp[i];
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    z += __shfl_xor_sync(0xffffffffu, z, o);
    t += __shfl_xor_sync(0xffffffffu, t, o);
  }
  if (lane == 0) part[0][warp] = z, part[1][warp] = t;
  __syncthreads();
  z = t = 0.0;
  for (int w = 0; w < kPickWarps; ++w) z += part[0][w], t += part[1][w];
  if (d.draft >= 0 && !(t > 0.0)) d.draft = -1;  // p <= q everywhere: draw from p
  const float* q = d.draft >= 0 && a.q ? a.q + static_cast<int64_t>(d.draft) * a.q_ld : nullptr;
  Weigh w(d, tab, q != nullptr);
  w.Z = zs;
  const double target = d.u * (d.draft >= 0 ? t : z);
  // every warp finds the chunk; then the chunk's segments, one a warp, the segment's lanes and the lane's values
  double before = 0.0;
  const int chunk = reach(d.draft >= 0 ? rp : zp, chunks, target, lane, before);
  constexpr int kOwn = kDrawChunk / kPickThreads;  // consecutive values of a lane
  const int64_t j0 = static_cast<int64_t>(max(chunk, 0)) * kDrawChunk + static_cast<int64_t>(tid) * kOwn;
  float x[kOwn], y[kOwn];
#pragma unroll
  for (int g = 0; g < kOwn; ++g) {
    const bool in = j0 + g < a.V;
    x[g] = in ? to_float(l[j0 + g]) : -INFINITY;
    y[g] = in && q ? q[j0 + g] : 0.0f;
  }
  double e[kOwn], v = 0.0;
#pragma unroll
  for (int g = 0; g < kOwn; ++g) {
    e[g] = w.rest(static_cast<int>(j0 + g), x[g], y[g]);
    v += e[g];
  }
  double incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double s = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += s;
  }
  if (lane == 31) seg[warp] = incl;
  __syncthreads();
  if (warp != reach(seg, kPickWarps, target, lane, before)) return;
  const unsigned some = __ballot_sync(0xffffffffu, v > 0.0);
  const unsigned hit = __ballot_sync(0xffffffffu, v > 0.0 && before + incl >= target);
  if (lane != (hit ? __ffs(hit) - 1 : 31 - __clz(some))) return;
  double run = before + (incl - v);
  int64_t found = -1;
#pragma unroll
  for (int g = 0; g < kOwn; ++g) {
    if (e[g] > 0.0 && (found < 0 || run < target)) found = j0 + g;
    run += e[g];
  }
  a.next[r] = static_cast<int32_t>(found);
}

struct VerifyWs {
  int64_t chunks;  // of the draw
  int64_t parts, decide, zpart, rpart, zsum, bytes;
};
VerifyWs verify_ws(int n_rows, int n_req, int V) {
  VerifyWs w;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t p = at;
    at = (at + bytes + 255) / 256 * 256;
    return p;
  };
  // chunks of one tile are the most a row can have
  w.parts = take((static_cast<int64_t>(V) + kRowTile - 1) / kRowTile * n_rows * static_cast<int64_t>(sizeof(RowPart)));
  w.chunks = (static_cast<int64_t>(V) + kDrawChunk - 1) / kDrawChunk;
  w.decide = take(n_req * static_cast<int64_t>(sizeof(Decision)));
  w.zpart = take(n_req * w.chunks * 8);
  w.rpart = take(n_req * w.chunks * 8);
  w.zsum = take(n_req * static_cast<int64_t>(8));
  w.bytes = std::max<int64_t>(at, 256);
  return w;
}

template <typename T>
int run_verify(const VerifyArgs& a, int sms, cudaStream_t s) {
  const int tiles = verify_chunk_tiles(a.n_rows, a.V, sms);
  const int n_chunks = static_cast<int>((static_cast<int64_t>(a.V) + static_cast<int64_t>(tiles) * kRowTile - 1) /
                                        (static_cast<int64_t>(tiles) * kRowTile));
  const VerifyWs y = verify_ws(a.n_rows, a.n_req, a.V);
  uint8_t* p = static_cast<uint8_t*>(a.ws);
  RowPart* parts = reinterpret_cast<RowPart*>(p + y.parts);
  Decision* decide = reinterpret_cast<Decision*>(p + y.decide);
  double* zpart = reinterpret_cast<double*>(p + y.zpart);
  double* rpart = reinterpret_cast<double*>(p + y.rpart);
  double* zsum = reinterpret_cast<double*>(p + y.zsum);
  k_verify_rows<T><<<dim3(static_cast<unsigned>(a.n_rows), static_cast<unsigned>(n_chunks)), kRowThreads, 0, s>>>(
      a, tiles, n_chunks, parts);
  cudaError_t e = cudaGetLastError();
  const dim3 grid(static_cast<unsigned>(y.chunks), static_cast<unsigned>(a.n_req));
  // every CTA of a request walks its drafts again, so requests get no more CTAs than the SMs hold at once
  const int most = std::max(1, 4 * sms / a.n_req), per = static_cast<int>((y.chunks + most - 1) / most);
  const dim3 walk(static_cast<unsigned>((y.chunks + per - 1) / per), static_cast<unsigned>(a.n_req));
  if (e == cudaSuccess)
    e = launch_pdl(k_verify_norm<T>, walk, dim3(kDrawThreads), 0, s, a, n_chunks, static_cast<const RowPart*>(parts),
                   decide, zpart, static_cast<int>(y.chunks), per);
  if (e == cudaSuccess)
    e = launch_pdl(k_verify_rest<T>, grid, dim3(kDrawThreads), 0, s, a, static_cast<const Decision*>(decide),
                   static_cast<const double*>(zpart), rpart, zsum);
  if (e == cudaSuccess)
    e = launch_pdl(k_verify_pick<T>, dim3(static_cast<unsigned>(a.n_req)), dim3(kPickThreads), 0, s, a,
                   static_cast<const Decision*>(decide), static_cast<const double*>(zpart),
                   static_cast<const double*>(rpart), static_cast<const double*>(zsum), static_cast<int>(y.chunks));
  return e;
}

}  // namespace

int64_t verify_workspace(int n_rows, int n_req, int V) { return verify_ws(n_rows, n_req, V).bytes; }

int launch_verify_draft(const VerifyArgs& a, ActType type, int sms, cudaStream_t s) {
  if (a.n_req <= 0) return cudaSuccess;
  if (type == ActType::f32) return run_verify<float>(a, sms, s);
  if (type == ActType::f16) return run_verify<__half>(a, sms, s);
  return run_verify<__nv_bfloat16>(a, sms, s);
}

}  // namespace mkb
