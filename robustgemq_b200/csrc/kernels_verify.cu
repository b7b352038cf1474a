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
// A row with a NaN, a +inf or nothing finite, or a temperature below zero or NaN, has no
// distribution: its draft is not taken and its token is -1.
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
  int B, n, V, parts, part_len;
  float4* stats;               // [B][n + 1][parts]: maximum, sum, its index, bad
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

// Maximum (first index), sum of exp((l - maximum) / T) and whether a value is no number.
struct Stat {
  float m, s;
  int at;
  bool bad;
};
__device__ __forceinline__ Stat join(const Stat& x, const Stat& y, float inv_t) {
  Stat r;
  r.bad = x.bad || y.bad;
  const bool first = x.m > y.m || (x.m == y.m && x.at <= y.at);
  r.m = first ? x.m : y.m;
  r.at = first ? x.at : y.at;
  r.s = r.m == -INFINITY ? 0.f : x.s * __expf((x.m - r.m) * inv_t) + y.s * __expf((y.m - r.m) * inv_t);
  return r;
}
__device__ __forceinline__ Stat shfl(const Stat& x, int o) {
  Stat r;
  r.m = __shfl_xor_sync(0xffffffffu, x.m, o);
  r.s = __shfl_xor_sync(0xffffffffu, x.s, o);
  r.at = __shfl_xor_sync(0xffffffffu, x.at, o);
  r.bad = __shfl_xor_sync(0xffffffffu, static_cast<int>(x.bad), o) != 0;
  return r;
}
__device__ __forceinline__ Stat warp_join(Stat x, float inv_t) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x = join(x, shfl(x, o), inv_t);
  return x;
}

template <typename L>
__global__ void __launch_bounds__(kThreads) k_verify_stats(const VerifyArgs a) {
  __shared__ Stat s_warp[kWarps];
  grid_dep_wait();
  const int part = blockIdx.x, i = blockIdx.y, b = blockIdx.z;
  if (part == 0 && i == 0 && threadIdx.x == 0) {
    a.best[2 * b] = a.best[2 * b + 1] = 0ull;
    a.done[b] = 0u;
  }
  if (i > draft_len(a, b)) return;
  const float t = temperature(a, b);
  const float inv_t = t == 0.f ? 1.f : 1.f / t;
  const L* row = static_cast<const L*>(a.logits) + b * a.logits_seq + i * a.logits_row;
  const int j0 = part * a.part_len, j1 = min(a.V, j0 + a.part_len);
  Stat x{-INFINITY, 0.f, 0x7fffffff, false};
  for (int j = j0 + static_cast<int>(threadIdx.x); j < j1; j += kThreads) {
    const float l = to_f32(row[j]);
    x.bad |= !(l < INFINITY);
    if (l > x.m) {
      x.s = x.s * __expf((x.m - l) * inv_t) + 1.f;
      x.m = l;
      x.at = j;
    } else if (l > -INFINITY) {
      x.s += __expf((l - x.m) * inv_t);
    }
  }
  x = warp_join(x, inv_t);
  if ((threadIdx.x & 31) == 0) s_warp[threadIdx.x >> 5] = x;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kWarps; ++w) x = join(x, s_warp[w], inv_t);
    a.stats[(static_cast<int64_t>(b) * (a.n + 1) + i) * a.parts + part] =
        make_float4(x.m, x.s, __int_as_float(x.at), x.bad ? 1.f : 0.f);
  }
}

__device__ __forceinline__ unsigned long long race_key(float score, int j) {
  return static_cast<unsigned long long>(__float_as_uint(score)) << 32 | (0xffffffffu - static_cast<uint32_t>(j));
}

template <typename L, typename Q>
__global__ void __launch_bounds__(kThreads) k_verify_pick(const VerifyArgs a) {
  __shared__ Stat s_row[kMaxRows];
  __shared__ unsigned long long s_best[2][kWarps];
  __shared__ bool s_last;
  grid_dep_wait();
  const int part = blockIdx.x, b = blockIdx.y;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int len = draft_len(a, b);
  const float t = temperature(a, b);
  const bool greedy = t == 0.f;
  const float inv_t = greedy ? 1.f : 1.f / t;
  for (int i = warp; i <= len; i += kWarps) {
    Stat x{-INFINITY, 0.f, 0x7fffffff, false};
    if (lane < a.parts) {
      const float4 f = a.stats[(static_cast<int64_t>(b) * (a.n + 1) + i) * a.parts + lane];
      x = Stat{f.x, f.y, __float_as_int(f.z), f.w != 0.f};
    }
    x = warp_join(x, inv_t);
    x.bad |= x.m == -INFINITY || !(t >= 0.f);
    if (lane == 0) s_row[i] = x;
  }
  __syncthreads();
  // p of one value of row i, given its logit
  auto prob = [&](const Stat& x, float l, int j) {
    return greedy ? (j == x.at ? 1.f : 0.f) : __fdiv_rn(__expf((l - x.m) * inv_t), x.s);
  };
  const L* logits = static_cast<const L*>(a.logits) + b * a.logits_seq;
  const int64_t* drafts = a.drafts + static_cast<int64_t>(b) * a.n;
  // whether draft i is taken, one lane each; every warp comes to the same answer
  int r = 0;
  for (int i0 = 0; i0 < len; i0 += 32) {
    const int i = i0 + lane;
    bool ok = false;
    if (i < len) {
      const int64_t x = drafts[i];
      if (x >= 0 && x < a.V && !s_row[i].bad) {
        const float p = prob(s_row[i], to_f32(logits[i * a.logits_row + x]), static_cast<int>(x));
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
  const L* lr = logits + r * a.logits_row;
  const Q* qr = r < len && a.probs != nullptr ? static_cast<const Q*>(a.probs) + b * a.probs_seq + r * a.probs_row : nullptr;
  const int x_r = r < len && a.probs == nullptr ? static_cast<int>(min(max(drafts[r], int64_t(-1)), int64_t(a.V))) : -1;
  unsigned long long best0 = 0, best1 = 0;
  if (!row.bad) {
    const float* noise = a.noise + static_cast<int64_t>(b) * a.V;
    const int j0 = part * a.part_len, j1 = min(a.V, j0 + a.part_len);
    for (int j = j0 + static_cast<int>(threadIdx.x); j < j1; j += kThreads) {
      const float p = prob(row, to_f32(lr[j]), j);
      const float q = qr != nullptr ? to_f32(qr[j]) : (j == x_r ? 1.f : 0.f);
      const float e = noise[j];
      const float w = fmaxf(p - q, 0.f);
      if (w > 0.f) {
        const float s = __fdiv_rn(w, e);
        if (s >= 0.f) best0 = max(best0, race_key(s, j));
      }
      if (p > 0.f) {
        const float s = __fdiv_rn(p, e);
        if (s >= 0.f) best1 = max(best1, race_key(s, j));
      }
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    best0 = max(best0, __shfl_xor_sync(0xffffffffu, best0, o));
    best1 = max(best1, __shfl_xor_sync(0xffffffffu, best1, o));
  }
  if (lane == 0) {
    s_best[0][warp] = best0;
    s_best[1][warp] = best1;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kWarps; ++w) {
      best0 = max(best0, s_best[0][w]);
      best1 = max(best1, s_best[1][w]);
    }
    atomicMax(&a.best[2 * b], best0);
    atomicMax(&a.best[2 * b + 1], best1);
    __threadfence();
    s_last = atomicAdd(&a.done[b], 1u) == static_cast<uint32_t>(gridDim.x) - 1u;
  }
  __syncthreads();
  if (!s_last || warp != 0) return;
  __threadfence();
  const unsigned long long k0 = __ldcg(&a.best[2 * b]), k1 = __ldcg(&a.best[2 * b + 1]);
  const unsigned long long key = k0 != 0 ? k0 : k1;
  const int last = row.bad || key == 0 ? -1 : static_cast<int>(0xffffffffu - static_cast<uint32_t>(key));
  for (int i = lane; i <= a.n; i += 32) {
    const int tok = i < r ? static_cast<int>(drafts[i]) : (i == r ? last : -1);
    const int64_t at = static_cast<int64_t>(b) * (a.n + 1) + i;
    a.tokens[at] = tok;
    a.logprobs[at] = tok < 0 ? 0.f : (to_f32(logits[i * a.logits_row + tok]) - s_row[i].m) * inv_t - logf(s_row[i].s);
  }
  if (lane == 0) a.accepted[b] = r;
}

int verify_parts(int B, int n, int V) {
  // enough blocks for four on each SM, parts of at least 2048 values
  const int64_t rows = static_cast<int64_t>(B) * (n + 1);
  const int64_t want = (4 * device_sm_count() + rows - 1) / rows;
  const int64_t most = (V + 2047) / 2048;
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({want, most, kMaxParts})));
}

size_t align256(size_t v) { return (v + 255) & ~static_cast<size_t>(255); }

}  // namespace

size_t verify_workspace(int B, int n, int V) {
  return align256(sizeof(float4) * static_cast<size_t>(B) * (n + 1) * verify_parts(B, n, V)) +
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
  a.parts = verify_parts(B, n, V);
  a.part_len = ((V + a.parts - 1) / a.parts + 7) / 8 * 8;
  char* w = static_cast<char*>(workspace);
  a.stats = reinterpret_cast<float4*>(w);
  w += align256(sizeof(float4) * static_cast<size_t>(B) * (n + 1) * a.parts);
  a.best = reinterpret_cast<unsigned long long*>(w);
  a.done = reinterpret_cast<uint32_t*>(w + align256(16 * static_cast<size_t>(B)));
  a.tokens = v.tokens;
  a.accepted = v.num_accepted;
  a.logprobs = v.logprobs;
  const dim3 g1(static_cast<unsigned>(a.parts), static_cast<unsigned>(n + 1), static_cast<unsigned>(B));
  const dim3 g2(static_cast<unsigned>(a.parts), static_cast<unsigned>(B));
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
