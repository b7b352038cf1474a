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
// A row with a NaN, a +inf or nothing finite, or a temperature that is negative or not finite, has
// no distribution: its draft is not taken and its token is -1.
//
// Two launches: every row's maximum and sum over parts of the vocabulary (one pass over
// the logits, the traffic's bulk), then the decisions and the race over parts of one row
// of each sequence, whose last part writes the answer.
#include <algorithm>

#include "paged.cuh"

namespace gemq {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxParts = 32;   // one lane a part where the parts are joined
constexpr int kMaxRows = 64;    // drafts + 1
constexpr int kPickBlocks = 4;  // of the second kernel, resident on an SM

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

// Eight values of a row for this thread: neighbours by 16-byte loads where the row is
// aligned, else one of every kThreads, which is as coalesced. Element e of the step at j
// is at(j, e); steps are 8 * kThreads apart. Past `end` comes `fill`.
template <bool VEC>
__device__ __forceinline__ int at(int j, int e) {
  return VEC ? j + static_cast<int>(threadIdx.x) * 8 + e : j + e * kThreads + static_cast<int>(threadIdx.x);
}
template <bool VEC, typename V>
__device__ __forceinline__ void load8(const V* row, int j, int end, float fill, float (&x)[8]) {
  if (VEC && at<VEC>(j, 8) <= end) {
    const uint4* p = reinterpret_cast<const uint4*>(row + at<VEC>(j, 0));
    if constexpr (sizeof(V) == 4) {
      const uint4 a = __ldg(p), b = __ldg(p + 1);
      const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = __uint_as_float(w[e]);
    } else {
      const uint4 a = __ldg(p);
      const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 g = unpack2<V>(w[e]);
        x[2 * e] = g.x;
        x[2 * e + 1] = g.y;
      }
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = at<VEC>(j, e) < end ? to_f32(row[at<VEC>(j, e)]) : fill;
}
__device__ __forceinline__ bool vec_ok(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <bool VEC, typename L>
__device__ __forceinline__ Stat row_stat(const L* row, int j0, int j1, float f) {
  Stat x{-INFINITY, 0.f, 0x7fffffff};
#pragma unroll 2
  for (int j = j0; j < j1; j += 8 * kThreads) {
    float v[8];
    load8<VEC>(row, j, j1, -INFINITY, v);
    float top = v[0];
#pragma unroll
    for (int e = 1; e < 8; ++e) top = fmaxf(top, v[e]);
    if (top > x.m) {
      x.s *= ex2((x.m - top) * f);
      x.m = top;
      x.at = 0x7fffffff;
#pragma unroll
      for (int e = 7; e >= 0; --e)
        if (v[e] == top) x.at = at<VEC>(j, e);
    }
    const float ref = base_of(x.m);
#pragma unroll
    for (int e = 0; e < 8; ++e) x.s += ex2((v[e] - ref) * f);
  }
  return x;
}

// log2(e) / T; the greedy form keeps T = 1 for its log probabilities.
__device__ __forceinline__ float slope(float t) { return kLog2e / (t == 0.f ? 1.f : t); }

template <typename L>
__global__ void __launch_bounds__(kThreads, 5) k_verify_stats(const VerifyArgs a) {
  __shared__ Stat s_warp[kWarps];
  grid_dep_wait();
  grid_dep_launch();  // the pick's blocks may come up in the tail of this kernel
  const int part = blockIdx.x, i = blockIdx.y, b = blockIdx.z;
  if (part == 0 && i == 0 && threadIdx.x == 0) {
    a.best[2 * b] = a.best[2 * b + 1] = 0ull;
    a.done[b] = 0u;
  }
  if (i > draft_len(a, b)) return;
  const float f = slope(temperature(a, b));
  const L* row = static_cast<const L*>(a.logits) + b * a.logits_seq + i * a.logits_row;
  const int j0 = part * a.part_len, j1 = min(a.V, j0 + a.part_len);
  Stat x = vec_ok(row) ? row_stat<true>(row, j0, j1, f) : row_stat<false>(row, j0, j1, f);
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

// One row's part of the race: the best of (p - q)+ / e and of p / e.
struct Race {
  unsigned long long rest, all;
};
template <bool VEC, typename L, typename Q>
__device__ __forceinline__ Race run_race(const L* lr, const Q* qr, int x_r, const float* noise, const Stat& row,
                                         bool greedy, float f, int j0, int j1) {
  // the scores stay floats (no NaN comes up: a score must exceed the best so far), with
  // the first index that reached the best
  // (the race of p counts only where no thread finds anything in the rest)
  float best0 = 0.f, best1 = 0.f;
  int at0 = -1, at1 = -1;
  const float inv_s = 1.f / row.s;
  for (int j = j0; j < j1; j += 8 * kThreads) {
    float l[8], q[8], e[8];
    load8<VEC>(lr, j, j1, -INFINITY, l);
    load8<VEC>(noise, j, j1, 1.f, e);
    if (qr != nullptr) load8<VEC>(qr, j, j1, 0.f, q);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int k = at<VEC>(j, i);
      const float p = greedy ? (k == row.at ? 1.f : 0.f) : ex2((l[i] - row.m) * f) * inv_s;
      const float w = p - (qr != nullptr ? q[i] : (k == x_r ? 1.f : 0.f));
      // a quick quotient (good to 2 ulp) says which few values need the rounded one
      if (w > 0.f && __fdividef(w, e[i]) * 1.00001f >= best0) {
        const float s = __fdiv_rn(w, e[i]);
        if (s > best0) {
          best0 = s;
          at0 = k;
        }
      }
      if (best0 == 0.f && p > 0.f && __fdividef(p, e[i]) * 1.00001f >= best1) {
        const float s = __fdiv_rn(p, e[i]);
        if (s > best1) {
          best1 = s;
          at1 = k;
        }
      }
    }
  }
  return Race{at0 >= 0 ? race_key(best0, at0) : 0ull, at1 >= 0 ? race_key(best1, at1) : 0ull};
}

template <typename L, typename Q>
__global__ void __launch_bounds__(kThreads, kPickBlocks) k_verify_pick(const VerifyArgs a) {
  __shared__ Stat s_row[kMaxRows];
  __shared__ unsigned long long s_best[2][kWarps];
  __shared__ bool s_last;
  grid_dep_wait();
  const int part = blockIdx.x, b = blockIdx.y;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int len = draft_len(a, b);
  const float t = temperature(a, b);
  const bool greedy = t == 0.f;
  const float f = slope(t);
  for (int i = warp; i <= len; i += kWarps) {
    Stat x{-INFINITY, 0.f, 0x7fffffff};
    if (lane < a.parts) {
      const float4 g = a.stats[(static_cast<int64_t>(b) * (a.n + 1) + i) * a.parts + lane];
      x = Stat{g.x, g.y, __float_as_int(g.z)};
    }
    x = warp_join(x, f);
    // no distribution: nothing finite, a NaN or +inf (a NaN sum), or no temperature
    if (x.m == -INFINITY || !(x.m < INFINITY) || !(t >= 0.f && t < INFINITY)) x.s = NAN;
    if (lane == 0) s_row[i] = x;
  }
  __syncthreads();
  const L* logits = static_cast<const L*>(a.logits) + b * a.logits_seq;
  const int64_t* drafts = a.drafts + static_cast<int64_t>(b) * a.n;
  // whether draft i is taken, one lane each; every warp comes to the same answer
  int r = 0;
  for (int i0 = 0; i0 < len; i0 += 32) {
    const int i = i0 + lane;
    bool ok = false;
    if (i < len) {
      const int64_t x = drafts[i];
      if (x >= 0 && x < a.V) {
        const Stat row = s_row[i];
        const float l = to_f32(logits[i * a.logits_row + x]);
        float p = greedy ? (x == row.at ? 1.f : 0.f) : __fdiv_rn(ex2((l - row.m) * f), row.s);
        if (isnan(row.s)) p = 0.f;
        const float q = a.probs == nullptr ? 1.f : to_f32(static_cast<const Q*>(a.probs)[b * a.probs_seq + i * a.probs_row + x]);
        ok = a.uniforms[static_cast<int64_t>(b) * a.n + i] * q < p;
      }
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
    const Q* qr = r < len && a.probs != nullptr ? static_cast<const Q*>(a.probs) + b * a.probs_seq + r * a.probs_row : nullptr;
    const int x_r = r < len && a.probs == nullptr ? static_cast<int>(min(max(drafts[r], int64_t(-1)), int64_t(a.V))) : -1;
    const float* noise = a.noise + static_cast<int64_t>(b) * a.V;
    const int j0 = part * a.race_len, j1 = min(a.V, j0 + a.race_len);
    best = vec_ok(lr) && vec_ok(noise) && vec_ok(qr)
               ? run_race<true>(lr, qr, x_r, noise, row, greedy, f, j0, j1)
               : run_race<false>(lr, qr, x_r, noise, row, greedy, f, j0, j1);
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
    const int tok = i < r ? static_cast<int>(drafts[i]) : (i == r ? last : -1);
    const int64_t to = static_cast<int64_t>(b) * (a.n + 1) + i;
    a.tokens[to] = tok;
    a.logprobs[to] = tok < 0 ? 0.f : ((to_f32(logits[i * a.logits_row + tok]) - s_row[i].m) * f - log2f(s_row[i].s)) * kLn2;
  }
  if (lane == 0) a.accepted[b] = r;
}

// Parts of a row for `rows` of them: at least one step of 8 * kThreads values each.
// Statistics: sixteen blocks an SM, so that the last round of them is a small share. The
// race: one round of resident blocks, since every block first repeats the decisions.
int parts_of(int64_t rows, int V, int64_t blocks, int most) {
  const int64_t want = std::max<int64_t>(1, blocks / rows);
  const int64_t steps = (V + 8 * kThreads - 1) / (8 * kThreads);
  return static_cast<int>(std::min<int64_t>({want, steps, most}));
}
int stat_parts(int B, int n, int V) {
  return parts_of(static_cast<int64_t>(B) * (n + 1), V, 16 * device_sm_count(), kMaxParts);
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
  const int races = parts_of(B, V, kPickBlocks * device_sm_count(), 1024);
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
