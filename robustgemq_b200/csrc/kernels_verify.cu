// Verification of drafted tokens against the target's probabilities from given random
// numbers.
//
// Sequence b has len <= n drafted tokens x_0.., the target's logits at n + 1 positions
// and, where the draft sampled, its probabilities q_i. With p_i = softmax(logits_i / T)
// (T = 0: all of it on the first maximum), x_i is taken while u_i q_i(x_i) < p_i(x_i)
// (q_i(x_i) = 1 without probabilities). At the first position r that is not taken (or
// r = len) one token comes from w = max(p_r - q_r, 0) (w = p_r at r = len, or where that
// leaves nothing) as the winner of a race, argmax_j w_j / e_j with exponential e_j: that
// samples from w / sum(w) without its sum, and a maximum does not hang on the order in
// which the vocabulary is split, as a running sum would. Ties go to the lowest index.
// A row with a NaN, a +inf or nothing finite, or a temperature that is negative or not
// finite, has no distribution: its draft is not taken and its token is -1.
//
// Two launches: every row's maximum and sum over parts of the vocabulary (one pass over
// the logits, the traffic's bulk), then the decisions and the race over parts of one row
// of each sequence, whose last part writes the answer. The second is bound by the first
// only where it needs the sums; drafts, their logits and the race's random numbers are on
// their way while the first ends. (One launch, a cluster of blocks a sequence that
// exchange the sums in shared memory, took 10.7, 58.7 and 13.0 us at its best cluster
// sizes, 16, 4 and 4, where this takes 8.3, 54.2 and 12.8, in the order below.)
//
// Measured on a B200, with the bytes that must move against the copy bandwidth: 1
// sequence of 4 drafts, vocabulary 50,304, fp16: 8.3 us, latency (two launches, four
// dependent reads); 64 of 7, 151,936, bf16 with fp32 probabilities: 54.2 us, 35.5 of
// bytes: the statistics use the exponentials' pipe to 65% and the DRAM to half, the pick
// waits for its loads, a step at a time (30% of the issue slots); 24 of up to 5, 32,001
// fp32 (rows off 16-byte boundaries, so single loads): 12.5 us, latency.
#include <algorithm>
#include <cfloat>

#include "paged.cuh"

namespace gemq {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxParts = 32;   // one lane a part where the parts are joined
constexpr int kMaxRaces = 128;
constexpr int kMaxRows = 64;    // drafts + 1
constexpr int kStatBlocks = 5;  // of the first kernel, resident on an SM
constexpr int kPickBlocks = 4;  // of the second

struct VerifyArgs {
  const void* logits;          // [B][n + 1][V]
  int64_t logits_seq, logits_row;  // strides in elements
  const int64_t* drafts;       // [B][n]
  const void* probs;           // [B][n][V] or null
  int64_t probs_seq, probs_row;
  const int32_t* draft_lens;   // [B] or null
  const float* uniforms;       // [B][n]
  const float* noise;          // [B][V]
  const float* temperature;    // [B] or null
  int B, n, V, parts, part_len, race_len;
  float4* stats;               // [B][n + 1][parts]: maximum, sum, the maximum's index
  unsigned long long* best;    // [B][2]: race of the rest, race of p
  uint32_t* done;              // [B]
  int64_t* tokens;             // [B][n + 1]
  int32_t* accepted;           // [B]
  float* logprobs;             // [B][n + 1]
};

__device__ __forceinline__ int draft_len(const VerifyArgs& a, int b) {
  return a.draft_lens == nullptr ? a.n : min(max(a.draft_lens[b], 0), a.n);
}
__device__ __forceinline__ float temperature(const VerifyArgs& a, int b) {
  return a.temperature == nullptr ? 1.f : a.temperature[b];
}

// Maximum (first index) and sum of exp((l - maximum) / T), as powers of two with
// f = log2(e) / T. A NaN or +inf among the values makes the sum a NaN.
struct Stat {
  float m, s;
  int at;
};
__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.f : m; }
__device__ __forceinline__ Stat join(const Stat& x, const Stat& y, float f) {
  const bool first = x.m > y.m || (x.m == y.m && x.at <= y.at);
  Stat r;
  r.m = first ? x.m : y.m;
  r.at = first ? x.at : y.at;
  const float ref = base_of(r.m);
  r.s = x.s * ex2((x.m - ref) * f) + y.s * ex2((y.m - ref) * f);
  return r;
}
__device__ __forceinline__ Stat warp_join(Stat x, float f) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Stat y;
    y.m = __shfl_xor_sync(0xffffffffu, x.m, o);
    y.s = __shfl_xor_sync(0xffffffffu, x.s, o);
    y.at = __shfl_xor_sync(0xffffffffu, x.at, o);
    x = join(x, y, f);
  }
  return x;
}

// A warp's step is 256 values of a row from j on, eight a lane: neighbours by 16-byte
// loads where the rows are aligned (VEC), else one of every 32, which is as coalesced.
// A step that is not FULL ends at `end`; past it comes `fill`.
constexpr int kStep = 256;
template <bool VEC>
__device__ __forceinline__ int at(int j, int e) {
  const int lane = static_cast<int>(threadIdx.x) & 31;
  return VEC ? j + lane * 8 + e : j + e * 32 + lane;
}
template <typename V>
struct Raw {
  uint4 r[sizeof(V) / 2];
  __device__ __forceinline__ void load(const V* p) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(V) / 2); ++i) r[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
  }
  __device__ __forceinline__ void unpack(float (&x)[8]) const {
    if constexpr (sizeof(V) == 4) {
      const uint32_t w[8] = {r[0].x, r[0].y, r[0].z, r[0].w, r[1].x, r[1].y, r[1].z, r[1].w};
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = __uint_as_float(w[e]);
    } else {
      const uint32_t w[4] = {r[0].x, r[0].y, r[0].z, r[0].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 g = unpack2<V>(w[e]);
        x[2 * e] = g.x;
        x[2 * e + 1] = g.y;
      }
    }
  }
};
template <bool VEC, bool FULL, typename V>
__device__ __forceinline__ void load8(const V* row, int j, int end, float fill, float (&x)[8]) {
  if (VEC && (FULL || at<VEC>(j, 8) <= end)) {
    Raw<V> raw;
    raw.load(row + at<VEC>(j, 0));
    raw.unpack(x);
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = FULL || at<VEC>(j, e) < end ? to_f32(row[at<VEC>(j, e)]) : fill;
}
__device__ __forceinline__ bool vec_ok(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// ex2((v - ref) * f) of eight values.
__device__ __forceinline__ void exps(const float (&v)[8], float ref, float f, F2 (&p)[4]) {
  const F2 minus = f2(-ref, -ref), ff = f2(f, f);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float x, y;
    split(mul2(add2(f2(v[2 * e], v[2 * e + 1]), minus), ff), x, y);
    p[e] = f2(ex2(x), ex2(y));
  }
}

// The statistics of a warp's steps j, j + stride, .. below j1, its lanes' apart. The index
// of the maximum costs as much as all the rest, and only the greedy form asks for it.
template <bool FIRST>
__device__ __forceinline__ void stat_step(const float (&v)[8], float f, Stat& x, int j, bool vec) {
  float top = fmaxf(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])), fmaxf(fmaxf(v[4], v[5]), fmaxf(v[6], v[7])));
  if (FIRST && top > x.m) {
    x.at = 0x7fffffff;
#pragma unroll
    for (int e = 7; e >= 0; --e)
      if (v[e] == top) x.at = vec ? at<true>(j, e) : at<false>(j, e);
  }
  top = fmaxf(top, x.m);
  const float ref = base_of(top);
  F2 p[4];
  exps(v, ref, f, p);
  float lo, hi;
  split(add2(add2(p[0], p[1]), add2(p[2], p[3])), lo, hi);
  x.s = x.s * ex2((x.m - ref) * f) + (lo + hi);
  x.m = top;
}
template <bool VEC, bool FIRST, typename L>
__device__ __forceinline__ Stat row_stat(const L* row, int j, int j1, int stride, float f) {
  constexpr int kAhead = sizeof(L) == 4 ? 3 : 4;  // steps whose loads are on their way together
  Stat x{-INFINITY, 0.f, 0x7fffffff};
  float v[8];
  if (VEC) {
#pragma unroll 1
    for (; j + (kAhead - 1) * stride + kStep <= j1; j += kAhead * stride) {
      Raw<L> raw[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) raw[u].load(row + at<true>(j + u * stride, 0));
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        raw[u].unpack(v);
        stat_step<FIRST>(v, f, x, j + u * stride, true);
      }
    }
  }
#pragma unroll 1
  for (; j + kStep <= j1; j += stride) {
    load8<VEC, true>(row, j, j1, 0.f, v);
    stat_step<FIRST>(v, f, x, j, VEC);
  }
  if (j < j1) {
    load8<VEC, false>(row, j, j1, -INFINITY, v);
    stat_step<FIRST>(v, f, x, j, VEC);
  }
  return x;
}
template <typename L>
__device__ __forceinline__ Stat row_stat(const L* row, int j, int j1, int stride, float f, bool greedy) {
  if (vec_ok(row)) return greedy ? row_stat<true, true>(row, j, j1, stride, f) : row_stat<true, false>(row, j, j1, stride, f);
  return greedy ? row_stat<false, true>(row, j, j1, stride, f) : row_stat<false, false>(row, j, j1, stride, f);
}

// log2(e) / T; the greedy form keeps T = 1 for its log probabilities. Of a subnormal T the
// quotient is infinite, and times the maximum's distance from itself it would be a NaN.
__device__ __forceinline__ float slope(float t) { return fminf(kLog2e / (t == 0.f ? 1.f : t), FLT_MAX); }

template <typename L>
__global__ void __launch_bounds__(kThreads, kStatBlocks) k_verify_stats(const VerifyArgs a) {
  __shared__ Stat s_warp[kWarps];
  grid_dep_wait();
  grid_dep_launch();  // the pick's blocks may come up in the tail of this kernel
  const int part = blockIdx.x, i = blockIdx.y, b = blockIdx.z;
  if (part == 0 && i == 0 && threadIdx.x == 0) {
    a.best[2 * b] = a.best[2 * b + 1] = 0ull;
    a.done[b] = 0u;
  }
  if (i > draft_len(a, b)) return;
  const float t = temperature(a, b), f = slope(t);
  const L* row = static_cast<const L*>(a.logits) + b * a.logits_seq + i * a.logits_row;
  const int j0 = part * a.part_len, j1 = min(a.V, j0 + a.part_len);
  Stat x = row_stat(row, j0 + static_cast<int>(threadIdx.x >> 5) * kStep, j1, kWarps * kStep, f, t == 0.f);
  x = warp_join(x, f);
  if ((threadIdx.x & 31) == 0) s_warp[threadIdx.x >> 5] = x;
  __syncthreads();
  if (threadIdx.x < 32) {
    x = threadIdx.x < kWarps ? s_warp[threadIdx.x] : Stat{-INFINITY, 0.f, 0x7fffffff};
    x = warp_join(x, f);
    if (threadIdx.x == 0)
      a.stats[(static_cast<int64_t>(b) * (a.n + 1) + i) * a.parts + part] =
          make_float4(x.m, x.s, __int_as_float(x.at), 0.f);
  }
}

__device__ __forceinline__ unsigned long long race_key(float score, int j) {
  return static_cast<unsigned long long>(__float_as_uint(score)) << 32 | (0xffffffffu - static_cast<uint32_t>(j));
}

// One row's part of the race: the best of (p - q)+ / e, and of p / e, which counts only
// where no part finds anything in the rest.
struct Race {
  unsigned long long rest, all;
};
// A warp's steps. Quick quotients say which few values can win: those that come within
// 2e-5 of the best that the warp has seen (a quick quotient is good to 1e-6) get the
// rounded one. Where the best is too small, or infinite, to tell, all of them do.
template <bool VEC, bool DRAFT, bool FULL, typename L, typename Q>
__device__ __forceinline__ void race_step(const L* lr, const Q* qr, int x_r, const float* noise, const Stat& row, float f,
                                          float inv_s, int j, int j1, float& top, float& best, int& best_at) {
  float l[8], q[8], e[8], w[8], quick[8];
  load8<VEC, FULL>(lr, j, j1, -INFINITY, l);
  load8<VEC, FULL>(noise, j, j1, 1.f, e);
  if (DRAFT) load8<VEC, FULL>(qr, j, j1, 0.f, q);
  F2 p[4];
  exps(l, row.m, f, p);
  const F2 inv = f2(inv_s, inv_s), neg = f2(-1.f, -1.f);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    F2 x = mul2(p[i], inv);
    if (DRAFT) x = fma2(f2(q[2 * i], q[2 * i + 1]), neg, x);
    split(x, w[2 * i], w[2 * i + 1]);
  }
  if (!DRAFT) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (at<VEC>(j, i) == x_r) w[i] -= 1.f;
  }
  float most = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(quick[i]) : "f"(e[i]));
    quick[i] *= w[i];
    most = fmaxf(most, quick[i]);
  }
  top = fmaxf(top, __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(most))));
  const float floor = top > 0x1p-100f && top < INFINITY ? top * (1.f - 2e-5f) : 0.f;
  if (most >= floor) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (w[i] > 0.f && !(quick[i] < floor)) {
        const float s = __fdiv_rn(w[i], e[i]);
        if (s > best) {
          best = s;
          best_at = at<VEC>(j, i);
        }
      }
  }
}
template <bool VEC, bool DRAFT, typename L, typename Q>
__device__ __forceinline__ unsigned long long race(const L* lr, const Q* qr, int x_r, const float* noise, const Stat& row,
                                                   float f, int j, int j1, int stride) {
  const float inv_s = 1.f / row.s;
  float top = 0.f, best = 0.f;
  int best_at = -1;
#pragma unroll 1
  for (; j + kStep <= j1; j += stride)
    race_step<VEC, DRAFT, true>(lr, qr, x_r, noise, row, f, inv_s, j, j1, top, best, best_at);
  if (j < j1) race_step<VEC, DRAFT, false>(lr, qr, x_r, noise, row, f, inv_s, j, j1, top, best, best_at);
  return best_at >= 0 ? race_key(best, best_at) : 0ull;
}
template <bool VEC, typename L, typename Q>
__device__ __forceinline__ Race race(const L* lr, const Q* qr, int x_r, const float* noise, const Stat& row, bool greedy,
                                     float f, int j, int j1, int stride) {
  Race r{0, 0};
  if (greedy) {  // p is 1 at one place and 0 elsewhere: its warp's first lane runs the race
    const int k = row.at;
    const bool mine = k >= j && k < j1 && (k - j) % stride < kStep;
    if (mine && (threadIdx.x & 31) == 0) {
      const float w = 1.f - (qr != nullptr ? to_f32(qr[k]) : (k == x_r ? 1.f : 0.f));
      const float s = __fdiv_rn(w, noise[k]), s_all = __fdiv_rn(1.f, noise[k]);
      if (w > 0.f && s > 0.f) r.rest = race_key(s, k);
      if (s_all > 0.f) r.all = race_key(s_all, k);
    }
    return r;
  }
  r.rest = qr != nullptr ? race<VEC, true>(lr, qr, x_r, noise, row, f, j, j1, stride)
                         : race<VEC, false>(lr, qr, x_r, noise, row, f, j, j1, stride);
  if ((qr != nullptr || x_r >= 0) && __ballot_sync(0xffffffffu, r.rest != 0) == 0)
    r.all = race<VEC, false>(lr, qr, -1, noise, row, f, j, j1, stride);
  return r;
}
template <typename L, typename Q>
__device__ __forceinline__ Race race_part(const L* lr, const Q* qr, int x_r, const float* noise, const Stat& row,
                                          bool greedy, float f, int j, int j1, int stride) {
  return vec_ok(lr) && vec_ok(noise) && vec_ok(qr)
             ? race<true>(lr, qr, x_r, noise, row, greedy, f, j, j1, stride)
             : race<false>(lr, qr, x_r, noise, row, greedy, f, j, j1, stride);
}

template <typename L, typename Q>
__global__ void __launch_bounds__(kThreads, kPickBlocks) k_verify_pick(const VerifyArgs a) {
  __shared__ Stat s_row[kMaxRows];
  __shared__ float s_logit[kMaxRows], s_q[kMaxRows], s_u[kMaxRows];  // of the drafts
  __shared__ int s_x[kMaxRows];                                      // -1: no token
  __shared__ unsigned long long s_best[2][kWarps];
  __shared__ bool s_last;
  // What does not come from the statistics kernel is read before it has ended: that
  // kernel let this one up only after it had itself waited for all that came before.
  const int part = blockIdx.x, b = blockIdx.y;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int j0 = min(a.V, part * a.race_len), j1 = min(a.V, j0 + a.race_len);
  const float* const noise = a.noise + static_cast<int64_t>(b) * a.V;
  for (int j = j0 + static_cast<int>(threadIdx.x) * 32; j < j1; j += kThreads * 32)
    asm volatile("prefetch.global.L2 [%0];" ::"l"(noise + j));
  const int len = draft_len(a, b);
  const float t = temperature(a, b);
  const bool greedy = t == 0.f;
  const float f = slope(t);
  const L* const logits = static_cast<const L*>(a.logits) + b * a.logits_seq;
  const Q* const probs = a.probs != nullptr ? static_cast<const Q*>(a.probs) + b * a.probs_seq : nullptr;
  if (static_cast<int>(threadIdx.x) < len) {
    const int i = threadIdx.x;
    const int64_t x = a.drafts[static_cast<int64_t>(b) * a.n + i];
    const bool is_token = x >= 0 && x < a.V;
    s_x[i] = is_token ? static_cast<int>(x) : -1;
    s_u[i] = a.uniforms[static_cast<int64_t>(b) * a.n + i];
    s_logit[i] = is_token ? to_f32(logits[i * a.logits_row + x]) : 0.f;
    s_q[i] = is_token && probs != nullptr ? to_f32(probs[i * a.probs_row + x]) : 1.f;
  }
  grid_dep_wait();
  for (int i = warp; i <= len; i += kWarps) {
    Stat x{-INFINITY, 0.f, 0x7fffffff};
    if (lane < a.parts) {
      const float4 g = __ldcg(a.stats + (static_cast<int64_t>(b) * (a.n + 1) + i) * a.parts + lane);
      x = Stat{g.x, g.y, __float_as_int(g.z)};
    }
    x = warp_join(x, f);
    // no distribution: nothing finite, a NaN or +inf (a NaN sum), or no temperature
    if (x.m == -INFINITY || !(x.m < INFINITY) || !(t >= 0.f && t < INFINITY)) x.s = NAN;
    if (lane == 0) s_row[i] = x;
  }
  __syncthreads();
  // whether draft i is taken, one lane each; every warp comes to the same answer
  int r = 0;
  for (int i0 = 0; i0 < len; i0 += 32) {
    const int i = i0 + lane;
    bool ok = false;
    if (i < len && s_x[i] >= 0) {
      const Stat row = s_row[i];
      float p = greedy ? (s_x[i] == row.at ? 1.f : 0.f) : __fdiv_rn(ex2((s_logit[i] - row.m) * f), row.s);
      if (isnan(row.s)) p = 0.f;
      ok = s_u[i] * s_q[i] < p;
    }
    const uint32_t yes = __ballot_sync(0xffffffffu, ok);
    if (yes == 0xffffffffu) {
      r += 32;
      continue;
    }
    r += __ffs(~yes) - 1;
    break;
  }
  r = min(r, len);
  const Stat row = s_row[r];
  Race best{0, 0};
  if (!isnan(row.s)) {
    const L* lr = logits + r * a.logits_row;
    const Q* qr = r < len && probs != nullptr ? probs + r * a.probs_row : nullptr;
    const int x_r = r < len && probs == nullptr ? s_x[r] : -1;
    best = race_part(lr, qr, x_r, noise, row, greedy, f, j0 + warp * kStep, j1, kWarps * kStep);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    best.rest = max(best.rest, __shfl_xor_sync(0xffffffffu, best.rest, o));
    best.all = max(best.all, __shfl_xor_sync(0xffffffffu, best.all, o));
  }
  if (lane == 0) {
    s_best[0][warp] = best.rest;
    s_best[1][warp] = best.all;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kWarps; ++w) {
      best.rest = max(best.rest, s_best[0][w]);
      best.all = max(best.all, s_best[1][w]);
    }
    atomicMax(&a.best[2 * b], best.rest);
    atomicMax(&a.best[2 * b + 1], best.all);
    __threadfence();
    s_last = atomicAdd(&a.done[b], 1u) == static_cast<uint32_t>(gridDim.x) - 1u;
  }
  __syncthreads();
  if (!s_last || warp != 0) return;
  __threadfence();
  const unsigned long long k0 = __ldcg(&a.best[2 * b]), k1 = __ldcg(&a.best[2 * b + 1]);
  const unsigned long long key = k0 != 0 ? k0 : k1;
  const int last = key == 0 ? -1 : static_cast<int>(0xffffffffu - static_cast<uint32_t>(key));
  for (int i = lane; i <= a.n; i += 32) {
    const int tok = i < r ? s_x[i] : (i == r ? last : -1);
    const int64_t to = static_cast<int64_t>(b) * (a.n + 1) + i;
    a.tokens[to] = tok;
    const float l = tok < 0 ? 0.f : i < r ? s_logit[i] : to_f32(logits[i * a.logits_row + tok]);
    a.logprobs[to] = tok < 0 ? 0.f : ((l - s_row[i].m) * f - log2f(s_row[i].s)) * kLn2;
  }
  if (lane == 0) a.accepted[b] = r;
}

// ------------------------------------------------------------------ host
// Parts of each of `rows` rows, at least one step of the block's warps each: the count
// that makes the rounds of `resident` blocks times a block's steps the least, a block's
// fixed work counting as kFixed steps. (Sixteen blocks an SM whatever the rows took
// 14.7 us where this takes 12.8, 24 sequences of up to five drafts at 32,001.)
constexpr int kFixed = 1;
int parts_of(int64_t rows, int V, int64_t resident, int most) {
  const int64_t steps = (V + kWarps * kStep - 1) / (kWarps * kStep);
  int64_t best = 1, least = INT64_MAX;
  for (int64_t p = 1; p <= std::min<int64_t>(steps, most); ++p) {
    const int64_t cost = (rows * p + resident - 1) / resident * ((steps + p - 1) / p + kFixed);
    if (cost < least) {
      least = cost;
      best = p;
    }
  }
  return static_cast<int>(best);
}
int stat_parts(int B, int n, int V) {
  return parts_of(static_cast<int64_t>(B) * (n + 1), V, kStatBlocks * device_sm_count(), kMaxParts);
}
// Values of a part: a multiple of 8, so that parts of an aligned row are aligned.
int part_length(int V, int parts) { return ((V + parts - 1) / parts + 7) / 8 * 8; }

size_t align256(size_t v) { return (v + 255) & ~static_cast<size_t>(255); }

}  // namespace

size_t verify_workspace(int B, int n, int V) {
  return align256(sizeof(float4) * static_cast<size_t>(B) * (n + 1) * stat_parts(B, n, V)) +
         align256(16 * static_cast<size_t>(B)) + align256(4 * static_cast<size_t>(B));
}

cudaError_t launch_verify(const gemq_verify_t& v, int B, int n, int V, void* workspace, cudaStream_t s) {
  VerifyArgs a{};
  a.logits = v.logits;
  a.logits_seq = v.logits_seq_stride;
  a.logits_row = v.logits_row_stride;
  a.drafts = v.draft_tokens;
  a.probs = v.draft_probs;
  a.probs_seq = v.probs_seq_stride;
  a.probs_row = v.probs_row_stride;
  a.draft_lens = v.draft_lens;
  a.uniforms = v.uniforms;
  a.noise = v.noise;
  a.temperature = v.temperature;
  a.B = B;
  a.n = n;
  a.V = V;
  a.parts = stat_parts(B, n, V);
  a.part_len = part_length(V, a.parts);
  const int races = parts_of(B, V, kPickBlocks * device_sm_count(), kMaxRaces);
  a.race_len = part_length(V, races);
  char* w = static_cast<char*>(workspace);
  a.stats = reinterpret_cast<float4*>(w);
  w += align256(sizeof(float4) * static_cast<size_t>(B) * (n + 1) * a.parts);
  a.best = reinterpret_cast<unsigned long long*>(w);
  a.done = reinterpret_cast<uint32_t*>(w + align256(16 * static_cast<size_t>(B)));
  a.tokens = v.tokens;
  a.accepted = v.num_accepted;
  a.logprobs = v.logprobs;
  const dim3 g1(static_cast<unsigned>(a.parts), static_cast<unsigned>(n + 1), static_cast<unsigned>(B));
  const dim3 g2(static_cast<unsigned>(races), static_cast<unsigned>(B));
  auto pick = [&](auto l) -> cudaError_t {
    using L = decltype(l);
    const cudaError_t e = launch_dep(k_verify_stats<L>, g1, dim3(kThreads), 0, s, a);
    if (e != cudaSuccess) return e;
    if (v.probs_dtype == GEMQ_FP32) return launch_dep(k_verify_pick<L, float>, g2, dim3(kThreads), 0, s, a);
    if (v.probs_dtype == GEMQ_BF16) return launch_dep(k_verify_pick<L, __nv_bfloat16>, g2, dim3(kThreads), 0, s, a);
    return launch_dep(k_verify_pick<L, __half>, g2, dim3(kThreads), 0, s, a);
  };
  if (v.logits_dtype == GEMQ_FP32) return pick(0.f);
  if (v.logits_dtype == GEMQ_BF16) return pick(__nv_bfloat16());
  return pick(__half());
}

}  // namespace gemq
