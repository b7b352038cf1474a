// Attention of a chunk of new tokens over a paged KV cache.
//
// Row (token i of the n new ones of a sequence of length L with them, query head h) has
// position p = L - n + i and sees the keys j <= p (j > p - window where there is one):
//   o = sum_j w_j v_j / sum_j w_j,  w_j = 2^(x_j - m),  x_j = scale log2(e) q.k_j,
//   lse = (m + log2 sum_j w_j) ln(2)
// A row that sees nothing gives o = 0 and lse = -inf. What a row does not see does not
// reach it whatever it holds.
//
// Quantised rows k_j = s_j c_j + z_j and v_j = t_j d_j + y_j go to the tensor cores as
// their codes, which are exact in fp16:
//   q.k_j = s_j (q.c_j) + z_j sum(q)
//   o = sum_j w'_j (d_j + y_j / t_j) / sum_j w'_j / t_j,  w'_j = 2^(x_j + log2 t_j - m)
// so the value's step acts as a shift of the score, w' stays in [0, 1], and the only
// rounding below 32 bits is that of w' to 16 bits, as without quantisation. An unsigned
// code in the low bits of a half with zero exponent is the subnormal code 2^-24, exactly,
// and costs one mask; keys take that form at both widths (8 bits as c + 128, with z_j =
// -128 s_j). Values become signed halves (4 bits: c - 8, y_j the value of code 8): a bias
// would stand in the sums as a multiple of sum w' that cancels, at 8 bits against long
// contexts' small averages, at 4 bits where a value is near zero.
//
// This file: few rows a KV head (decode steps, drafted tokens), where the cache's bytes
// are the time. mma.sync with the 16 rows of one KV head (tokens x query heads that share
// it) as M: at most 1/8 of the legacy tensor rate is needed to keep up with HBM, so the
// tensor-memory form would only add its round trips. Every warp streams its own tiles of
// 16 or 32 keys through its own cp.async ring, without block barriers; the keys of all
// sequences and heads form one axis of 64- or 128-key units that is cut evenly over all
// blocks (so uneven lengths do not matter), and k_attn_join adds up heads that were cut.
#include <algorithm>

#include "attn_rows.cuh"
#include "paged.cuh"

namespace gemq {

namespace {

// ------------------------------------------------------------------ small pieces
__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp8(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp4(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void ldsm4(uint32_t a, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t a, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a)
               : "memory");
}
// D (16x8 fp32) += A (16x16) B (16x8), fragments as the PTX ISA lays them out.
template <typename C>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Codes of a pair of words with bits 4 S..4 S + 3 in each half (S = 0, 1), minus 8.
template <int S>
__device__ __forceinline__ uint32_t signed4(uint32_t w) {
  // under the exponents of 2^10 and 2^6 the code reads as 1024 + c, 64 + c
  constexpr uint32_t kMask = S ? 0x00f000f0u : 0x000f000fu, kExp = S ? 0x54005400u : 0x64006400u;
  constexpr uint32_t kOff = S ? 0x54805480u : 0x64086408u;  // 64 + 8, 1024 + 8
  return h2_as_u32(__hsub2(u32_as_h2((w & kMask) | kExp), u32_as_h2(kOff)));
}
// Bytes c + 128 in places 0 and 2 of a word, 0x64 in 1 and 3 (1024 + c + 128), to c.
__device__ __forceinline__ uint32_t signed8(uint32_t pair) {
  const __half2 off = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
  return h2_as_u32(__hsub2(u32_as_h2(pair), off));
}

// ------------------------------------------------------------------ geometry
constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kM = 16;

template <typename T, int BITS, int DP>
struct Cfg {
  static constexpr int kKeys = BITS == 16 ? 16 : 32;  // keys of one warp's tile
  static constexpr int kUnit = kKeys * kWarps;        // keys of one unit of the axis
  static constexpr int kRow = DP * BITS / 8;          // bytes of a staged row
  static constexpr int kChunks = kRow / 16;
  static constexpr int kBlocks = DP == 256 ? 1 : 3;   // resident on an SM
  static constexpr int kStages = DP * BITS >= 4096 ? 3 : DP * BITS >= 1024 ? 2 : 3;
  static constexpr int kScale = BITS == 16 ? 0 : BITS == 8 ? 4 : 8;  // bytes of a row's scale
  static constexpr int kVOff = kKeys * kRow;
  static constexpr int kScOff = 2 * kKeys * kRow;
  static constexpr int kStage = kScOff + 2 * kKeys * kScale;
  // a tile's scales as the scores take them: [keys] each of a, log2 step, 1 / step, z, y / step
  static constexpr int kPrep = BITS == 16 ? 0 : 5 * kKeys * 4;
  static constexpr int kWarpBytes = kStages * kStage + kPrep;
  static constexpr int kSmem = kWarps * kWarpBytes;
  static_assert(kWarpBytes >= kM * DP * 4, "a warp's ring holds its output tile at the end");
  using C = std::conditional_t<BITS == 16, T, __half>;
  static constexpr bool kRowFactor = BITS != 16 && std::is_same_v<T, __nv_bfloat16>;
};

// Where chunk c (16 bytes) of a staged row lies, so that the fragment loads below meet
// no bank twice: 16-bit rows as ldmatrix wants them; quantised keys are read as whole
// 16-byte pieces of two neighbouring rows at a time, quantised values as words of rows
// 2t, t = 0..3, 32 bytes each.
template <int BITS, int CHUNKS, bool IS_V>
__device__ __forceinline__ uint32_t chunk_at(int row, int c) {
  if constexpr (BITS == 16) {
    return static_cast<uint32_t>(row * CHUNKS + (c ^ (row & 7))) * 16u;
  } else if constexpr (!IS_V) {
    return static_cast<uint32_t>(row * CHUNKS + (CHUNKS >= 8 ? c ^ (row & 1) : c)) * 16u;
  } else {
    const int l = row * CHUNKS + c;
    return static_cast<uint32_t>(l ^ (((row >> 1) & 3) << 1)) * 16u;
  }
}

// What the units of one sequence are: row tiles x KV heads x `units` each, the first at
// unit t0 of the key axis. Every item has at least one, so that rows that see nothing are
// written too.
struct SeqPlan {
  SeqRange r;
  int row_tiles, t0, units;
  __device__ __forceinline__ int64_t total(int kv_heads) const {
    return static_cast<int64_t>(row_tiles) * kv_heads * units;
  }
};
__device__ __forceinline__ SeqPlan plan_seq(const AttnArgs& a, int b, int unit) {
  SeqPlan p;
  p.r = seq_range(a, b);
  p.row_tiles = (p.r.q_len * a.group + kM - 1) / kM;
  const int lo = a.window > 0 ? max(0, p.r.kv_len - p.r.q_len - a.window + 1) : 0;
  p.t0 = lo / unit;
  p.units = max(1, (p.r.kv_len + unit - 1) / unit - p.t0);
  return p;
}

__device__ __forceinline__ int64_t warp_scan(int64_t v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t w = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += w;
  }
  return v;
}
// All units of the call (by a whole warp).
__device__ __forceinline__ int64_t all_units(const AttnArgs& a, int unit, int lane) {
  int64_t sum = 0;
  for (int b = lane; b < a.num_seqs; b += 32) sum += plan_seq(a, b, unit).total(a.kv.kv_heads);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  return sum;
}
// The sequence that unit u lies in and its first unit; `rows`: the same for row tiles.
template <typename F>
__device__ __forceinline__ bool find_seq(const AttnArgs& a, int64_t u, int lane, int& b, int64_t& first, F&& size) {
  int64_t base = 0;
  for (int b0 = 0; b0 < a.num_seqs; b0 += 32) {
    const int64_t n = b0 + lane < a.num_seqs ? size(b0 + lane) : 0;
    const int64_t incl = base + warp_scan(n, lane);
    const uint32_t past = __ballot_sync(0xffffffffu, incl > u);
    if (past != 0) {
      const int src = __ffs(past) - 1;
      b = b0 + src;
      first = __shfl_sync(0xffffffffu, incl - n, src);
      return true;
    }
    base = __shfl_sync(0xffffffffu, incl, 31);
  }
  return false;
}

// Blocks that share the units (each has at least one), unit range of block w of n, and the block that unit u falls to.
__device__ __forceinline__ int sharing(int64_t units, int blocks) {
  return static_cast<int>(min(units, static_cast<int64_t>(blocks)));
}
__device__ __forceinline__ int64_t first_unit(int64_t units, int w, int n) { return units * w / n; }
__device__ __forceinline__ int owner(int64_t units, int64_t u, int n) {
  return static_cast<int>(((u + 1) * n - 1) / units);
}

// Unnormalised parts of heads that several blocks share: block w's first piece in slot
// 2 w, a last piece that another block goes on with in 2 w + 1.
struct Parts {
  float* o;    // [slots][kM][DP]
  float2* ml;  // [slots][kM]: reference m, sum l
};

// ------------------------------------------------------------------ the kernel
template <typename T, int BITS, int DP>
__global__ void __launch_bounds__(kThreads, Cfg<T, BITS, DP>::kBlocks) k_attn_few(const AttnArgs a, const Parts parts) {
  using K = Cfg<T, BITS, DP>;
  using C = typename K::C;
  constexpr int kKeys = K::kKeys, kChunks = K::kChunks, kStages = K::kStages;
  constexpr int kNt = kKeys / 8;    // score tiles of 8 keys
  constexpr int kKs = DP / 16;      // k steps of q.k
  constexpr int kDt = DP / 8;       // output tiles of 8 columns
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float s_m[kWarps][kM], s_l[kWarps][kM];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int gid = lane >> 2, tig = lane & 3;
  const uint32_t ring = smem_u32(smem) + static_cast<uint32_t>(warp * K::kWarpBytes);
  float* const my_out = reinterpret_cast<float*>(smem + warp * K::kWarpBytes);
  float* const prep = reinterpret_cast<float*>(smem + warp * K::kWarpBytes + kStages * K::kStage);
  const int D = a.kv.head_dim;
  const int row_bytes = D * BITS / 8;
  const int mask = (1 << a.kv.page_shift) - 1;
  const float cs = a.scale * kLog2e;

  grid_dep_wait();
  // every block of this grid is resident, so the join's may be placed beside them now
  grid_dep_launch();
  const int64_t units = all_units(a, K::kUnit, lane);
  const int blocks = sharing(units, gridDim.x);
  if (static_cast<int>(blockIdx.x) >= blocks) return;
  int64_t u = first_unit(units, blockIdx.x, blocks);
  const int64_t u_end = first_unit(units, blockIdx.x + 1, blocks);
  bool first_piece = true;
  int64_t seq_first = 0, seq_end = 0;
  int b = 0;
  SeqPlan p{};
  while (u < u_end) {
    if (u >= seq_end) {
      if (!find_seq(a, u, lane, b, seq_first, [&](int s) { return plan_seq(a, s, K::kUnit).total(a.kv.kv_heads); })) break;
      p = plan_seq(a, b, K::kUnit);
      seq_end = seq_first + p.total(a.kv.kv_heads);
    }
    // the piece: units [tile, tile + cnt) of KV head h, row tile rt
    const int64_t local = u - seq_first;
    const int item = static_cast<int>(local / p.units), tile = static_cast<int>(local % p.units);
    const int rt = item / a.kv.kv_heads, h = item % a.kv.kv_heads;
    const int cnt = static_cast<int>(min(static_cast<int64_t>(p.units - tile), u_end - u));
    const int rows = min(kM, p.r.q_len * a.group - rt * kM);
    const int pos0 = p.r.kv_len - p.r.q_len;  // position of the first new token
    // this thread's rows, gid and gid + 8: last and first position they see
    int last[2], from[2];
    const T* q_row[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = gid + 8 * i;
      const int tok = (rt * kM + r) / a.group, hh = (rt * kM + r) % a.group;
      last[i] = r < rows ? pos0 + tok : -1;
      from[i] = a.window > 0 ? max(0, last[i] - a.window + 1) : 0;
      q_row[i] = r < rows ? static_cast<const T*>(a.q) + (p.r.start + tok) * a.q_token_stride +
                                static_cast<int64_t>(h * a.group + hh) * D
                          : nullptr;
    }
    const int tile_min = pos0 + rt * kM / a.group;  // positions of the row tile's first and last row
    const int tile_max = pos0 + (rt * kM + rows - 1) / a.group;

    // ---------------------------------------------------------- loads
    // Stages this warp's keys of the piece's unit t. Where a page holds whole tiles, one
    // page id serves a tile (and the next one's is asked for a tile ahead).
    const bool one_page = (1 << a.kv.page_shift) >= kKeys;
    const int tile_key = (p.t0 + tile) * K::kUnit + warp * kKeys;
    const int32_t* const table = a.page_table + b * a.page_table_stride;
    auto page_at = [&](int t) {
      const int j = tile_key + t * K::kUnit;
      return t < cnt && j < p.r.kv_len ? __ldg(table + (j >> a.kv.page_shift)) : -1;
    };
    int next_page = one_page ? page_at(0) : -1;
    constexpr int kRowsIt = 32 / kChunks;  // rows of one step of a warp's copies
    auto load = [&](int t) {
      if (t < cnt) {
        const uint32_t st = ring + static_cast<uint32_t>(t % kStages) * K::kStage;
        const int j0 = tile_key + t * K::kUnit;
        const bool wide = BITS != 4 || row_bytes % 16 == 0;
        int64_t soff = 0;
        int live;
        if (one_page) {
          const int page = next_page;
          next_page = page_at(t + 1);
          live = p.r.kv_len - j0;
          if (static_cast<uint32_t>(page) >= static_cast<uint32_t>(a.kv.num_pages)) {
            if (live > 0) set_device_error(kDevBadCachePos);
            live = 0;
          }
          const int off = j0 & mask;
          const int row0 = lane / kChunks, c = lane % kChunks;
          int64_t src = live > 0 ? a.kv.row(page, h, off + row0) + c * 16 : 0;
          const int64_t step = live > 0 ? static_cast<int64_t>(a.kv.token_stride) * (8 * kRowsIt) : 0;
          if constexpr (BITS != 16) soff = live > 0 ? a.kv.scale_row(page, h, off + lane) : 0;
          if (c * 16 < row_bytes) {
#pragma unroll
            for (int it = 0; it < kKeys / kRowsIt; ++it) {
              const int row = it * kRowsIt + row0;
              const uint32_t kd = st + chunk_at<BITS, kChunks, false>(row, c);
              const uint32_t vd = st + K::kVOff + chunk_at<BITS, kChunks, true>(row, c);
              if (wide) {
                const uint32_t n = row < live ? 16u : 0u;
                cp16(kd, a.kv.k + src, n);
                cp16(vd, a.kv.v + src, n);
              } else {  // rows of 8-byte alignment (4 bits, head_dim not a multiple of 32)
                const uint32_t n = row < live ? 8u : 0u;
                cp8(kd, a.kv.k + src, n);
                cp8(vd, a.kv.v + src, n);
                if (c * 16 + 8 < row_bytes) {
                  cp8(kd + 8, a.kv.k + src + 8, n);
                  cp8(vd + 8, a.kv.v + src + 8, n);
                }
              }
              src += step;
            }
          }
          live -= lane;
        } else {
          const int j = j0 + lane;
          int64_t off = -1;
          if (lane < kKeys && j < p.r.kv_len) {
            const int page = page_of(a, b, j >> a.kv.page_shift);
            if (page >= 0) {
              off = a.kv.row(page, h, j & mask);
              if constexpr (BITS != 16) soff = a.kv.scale_row(page, h, j & mask);
            }
          }
          live = off >= 0;
          for (int it = 0; it < kKeys / kRowsIt; ++it) {
            const int row = it * kRowsIt + lane / kChunks, c = lane % kChunks;
            const int64_t ro = __shfl_sync(0xffffffffu, off, row);
            if (c * 16 < row_bytes) {
              const int64_t src = ro < 0 ? 0 : ro + c * 16;
              const uint32_t kd = st + chunk_at<BITS, kChunks, false>(row, c);
              const uint32_t vd = st + K::kVOff + chunk_at<BITS, kChunks, true>(row, c);
              const uint32_t n = ro < 0 ? 0u : 8u;
              if (wide) {
                cp16(kd, a.kv.k + src, 2 * n);
                cp16(vd, a.kv.v + src, 2 * n);
              } else {
                cp8(kd, a.kv.k + src, n);
                cp8(vd, a.kv.v + src, n);
                if (c * 16 + 8 < row_bytes) {
                  cp8(kd + 8, a.kv.k + src + n, n);
                  cp8(vd + 8, a.kv.v + src + n, n);
                }
              }
            }
          }
        }
        if constexpr (BITS != 16) {
          const uint32_t sd = st + K::kScOff + static_cast<uint32_t>(lane) * K::kScale;
          constexpr uint32_t kV = kKeys * K::kScale;
          if constexpr (BITS == 8) {
            cp4(sd, a.kv.k_scale + soff, live > 0 ? 4u : 0u);
            cp4(sd + kV, a.kv.v_scale + soff, live > 0 ? 4u : 0u);
          } else {
            cp8(sd, a.kv.k_scale + soff, live > 0 ? 8u : 0u);
            cp8(sd + kV, a.kv.v_scale + soff, live > 0 ? 8u : 0u);
          }
        }
      }
      cp_commit();
    };
    if (BITS == 16 && D < DP) {
      // columns past head_dim meet zero queries; they must not hold a NaN
      for (int i = lane; i < kStages * kKeys * (kChunks - row_bytes / 16); i += 32) {
        const int n = kChunks - row_bytes / 16;
        const int row = i / n % kKeys, c = row_bytes / 16 + i % n;
        const uint32_t at = static_cast<uint32_t>(i / n / kKeys) * K::kStage + chunk_at<BITS, kChunks, false>(row, c);
        *reinterpret_cast<uint4*>(smem + warp * K::kWarpBytes + at) = make_uint4(0, 0, 0, 0);
      }
    }
#pragma unroll
    for (int t = 0; t < kStages - 1; ++t) load(t);

    // ---------------------------------------------------------- queries
    // Fragment k index <-> element: in order for 16 bits; for codes the order in which a
    // thread's contiguous quarter row unpacks (a dot product takes any).
    uint32_t qa[kKs][4];
    float rf[2] = {1.f, 1.f}, qsum[2] = {0.f, 0.f};
    if constexpr (K::kRowFactor) {
      // bf16 queries against fp16 codes: each row scaled by a power of two to at most 2,
      // which costs only what lies 2^-24 below its largest element
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float most = 0.f;
        if (q_row[i] != nullptr)
          for (int d = tig * 8; d < D; d += 32) {
            const uint4 w = *reinterpret_cast<const uint4*>(q_row[i] + d);
            const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float2 f = unpack2<T>(ws[e]);
              most = fmaxf(most, fmaxf(fabsf(f.x), fabsf(f.y)));
            }
          }
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
        const int e = most > 0.f && most < INFINITY ? min(max(ilogbf(most), -100), 100) : 0;
        rf[i] = exp2f(static_cast<float>(e));
      }
    }
    auto q2 = [&](int i, int d0, int d1) -> uint32_t {  // elements d0, d1 of row i
      if (q_row[i] == nullptr) return 0u;
      if constexpr (!K::kRowFactor) {
        const uint16_t* x = reinterpret_cast<const uint16_t*>(q_row[i]);
        const uint32_t lo = d0 < D ? x[d0] : 0u, hi = d1 < D ? x[d1] : 0u;
        return lo | hi << 16;
      } else {
        const float inv = 1.f / rf[i];
        return pack2<__half>(d0 < D ? to_f32(q_row[i][d0]) * inv : 0.f, d1 < D ? to_f32(q_row[i][d1]) * inv : 0.f);
      }
    };
#pragma unroll
    for (int ks = 0; ks < kKs; ++ks) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if constexpr (BITS == 16) {
          qa[ks][i] = q2(i, ks * 16 + 2 * tig, ks * 16 + 2 * tig + 1);
          qa[ks][i + 2] = q2(i, ks * 16 + 2 * tig + 8, ks * 16 + 2 * tig + 9);
        } else if constexpr (BITS == 8) {
          const int d = tig * (DP / 4) + 4 * ks;
          qa[ks][i] = q2(i, d, d + 1);
          qa[ks][i + 2] = q2(i, d + 2, d + 3);
        } else {
          const int d = tig * (DP / 4) + 8 * (ks >> 1) + 2 * (ks & 1);
          qa[ks][i] = q2(i, d, d + 4);
          qa[ks][i + 2] = q2(i, d + 1, d + 5);
        }
        if constexpr (BITS != 16) {
          const float2 f = __half22float2(u32_as_h2(qa[ks][i])), g = __half22float2(u32_as_h2(qa[ks][i + 2]));
          qsum[i] += f.x + f.y + g.x + g.y;
        }
      }
    }
    if constexpr (BITS != 16) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if constexpr (K::kRowFactor) rf[i] *= 16777216.f;  // undoes the subnormal codes' 2^-24
        qsum[i] += __shfl_xor_sync(0xffffffffu, qsum[i], 1);
        qsum[i] += __shfl_xor_sync(0xffffffffu, qsum[i], 2);
      }
    }

    // ---------------------------------------------------------- the keys
    float o[kDt][4];
#pragma unroll
    for (int i = 0; i < kDt; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, zacc[2] = {0.f, 0.f};
    for (int t = 0; t < cnt; ++t) {
      cp_wait<kStages - 2>();
      __syncwarp();
      load(t + kStages - 1);
      const uint32_t st = ring + static_cast<uint32_t>(t % kStages) * K::kStage;
      const int j0 = (p.t0 + tile + t) * K::kUnit + warp * kKeys;
      if (j0 > tile_max) continue;  // nothing here for any row
      const uint8_t* const stp = smem + (st - smem_u32(smem));
      if constexpr (BITS != 16) {
        // lane = key: a = 2^24 s c and z c, with c = scale log2(e); log2 t, 1 / t, y / t.
        // (bf16: the 2^24 goes with the row factors, whose range takes it)
        constexpr float kUp = K::kRowFactor ? 1.f : 16777216.f, kDown = K::kRowFactor ? 5.9604644775390625e-8f : 1.f;
        const float* ksc = reinterpret_cast<const float*>(stp + K::kScOff);
        const float* vsc = ksc + kKeys * K::kScale / 4;
        float step, base, vstep, vbase = 0.f;
        if constexpr (BITS == 8) {
          step = ksc[lane];
          base = -128.f * step;
          vstep = vsc[lane];
        } else {
          const float2 kk = reinterpret_cast<const float2*>(ksc)[lane], vv = reinterpret_cast<const float2*>(vsc)[lane];
          step = kk.x;
          base = kk.y;
          vstep = vv.x;
          vbase = fmaf(8.f, vv.x, vv.y);
        }
        vstep = vstep < kMinScale ? kMinScale : vstep;  // a step of zero; a NaN stays
        const float lv = lg2(vstep), inv = ex2(-lv);
        prep[lane] = step * cs * kUp;
        prep[kKeys + lane] = lv;
        prep[2 * kKeys + lane] = inv;
        prep[3 * kKeys + lane] = base * cs * kDown;
        // (the rounded quotient: codes and base nearly cancel where a value is near zero)
        if constexpr (BITS == 4) prep[4 * kKeys + lane] = vbase / vstep;
      }
      float s[kNt][4];
#pragma unroll
      for (int i = 0; i < kNt; ++i) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
      if constexpr (BITS == 16) {
#pragma unroll
        for (int ks = 0; ks < kKs; ++ks) {
          uint32_t f[4];
          ldsm4(st + chunk_at<BITS, kChunks, false>((lane & 7) + ((lane >> 4) << 3), 2 * ks + ((lane >> 3) & 1)), f);
          mma<C>(s[0], qa[ks], f[0], f[1]);
          mma<C>(s[1], qa[ks], f[2], f[3]);
        }
      } else {
        constexpr int kBytes = DP * BITS / 32;          // of a row, a thread
        constexpr int kWords = kBytes >= 16 ? 4 : 2;    // a load
        using Words = std::conditional_t<kWords == 4, uint4, uint2>;
#pragma unroll
        for (int i = 0; i < kNt; ++i) {
#pragma unroll
          for (int n = 0; n < kBytes / (4 * kWords); ++n) {
            const int byte = tig * kBytes + n * 4 * kWords;
            const Words ww = *reinterpret_cast<const Words*>(stp + chunk_at<BITS, kChunks, false>(8 * i + gid, byte >> 4) + (byte & 15));
            uint32_t w[4];
            w[0] = ww.x;
            w[1] = ww.y;
            if constexpr (kWords == 4) {
              w[2] = ww.z;
              w[3] = ww.w;
            }
#pragma unroll
            for (int e = 0; e < kWords; ++e) {
              const int ks = n * kWords + e;
              if constexpr (BITS == 8) {
                const uint32_t x = w[e] ^ 0x80808080u;
                mma<C>(s[i], qa[ks], __byte_perm(x, 0u, 0x4140), __byte_perm(x, 0u, 0x4342));
              } else {
                constexpr uint32_t kLow = 0x000f000fu;
                mma<C>(s[i], qa[2 * ks], w[e] & kLow, (w[e] >> 4) & kLow);
                mma<C>(s[i], qa[2 * ks + 1], (w[e] >> 8) & kLow, (w[e] >> 12) & kLow);
              }
            }
          }
        }
      }
      // scores, in powers of two
      float2 inv[kNt], zr[kNt];
      if constexpr (BITS == 16) {
#pragma unroll
        for (int i = 0; i < kNt; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[i][e] *= cs;
      } else {
        __syncwarp();
#pragma unroll
        for (int i = 0; i < kNt; ++i) {
          const int j = 8 * i + 2 * tig;
          const float2 aj = *reinterpret_cast<const float2*>(prep + j);
          const float2 lv = *reinterpret_cast<const float2*>(prep + kKeys + j);
          const float2 zj = *reinterpret_cast<const float2*>(prep + 3 * kKeys + j);
          inv[i] = *reinterpret_cast<const float2*>(prep + 2 * kKeys + j);
          if constexpr (BITS == 4) zr[i] = *reinterpret_cast<const float2*>(prep + 4 * kKeys + j);
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            if constexpr (K::kRowFactor) {
              s[i][2 * r] = fmaf(fmaf(qsum[r], zj.x, s[i][2 * r] * aj.x), rf[r], lv.x);
              s[i][2 * r + 1] = fmaf(fmaf(qsum[r], zj.y, s[i][2 * r + 1] * aj.y), rf[r], lv.y);
            } else {
              s[i][2 * r] = fmaf(s[i][2 * r], aj.x, fmaf(qsum[r], zj.x, lv.x));
              s[i][2 * r + 1] = fmaf(s[i][2 * r + 1], aj.y, fmaf(qsum[r], zj.y, lv.y));
            }
          }
        }
      }
      const bool full = j0 + kKeys - 1 <= tile_min && (a.window <= 0 || j0 > tile_max - a.window);
      if (!full) {
#pragma unroll
        for (int i = 0; i < kNt; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int j = j0 + 8 * i + 2 * tig + (e & 1);
            if (j > last[e >> 1] || j < from[e >> 1]) s[i][e] = -INFINITY;
          }
      }
      float ref[2], now[2];
      bool moved = false;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float top = m[r];
#pragma unroll
        for (int i = 0; i < kNt; ++i) top = fmaxf(top, fmaxf(s[i][2 * r], s[i][2 * r + 1]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        ref[r] = top == -INFINITY ? 0.f : top;
        now[r] = top;
        moved |= top != m[r];
      }
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float keep = ex2(m[r] - ref[r]);
          l[r] *= keep;
          zacc[r] *= keep;
#pragma unroll
          for (int i = 0; i < kDt; ++i) {
            o[i][2 * r] *= keep;
            o[i][2 * r + 1] *= keep;
          }
          m[r] = now[r];
        }
      }
      uint32_t pa[kKeys / 16][4];
#pragma unroll
      for (int i = 0; i < kNt; ++i) {
        float w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = e >> 1;
          w[e] = ex2(s[i][e] - ref[r]);
          if constexpr (BITS == 16) {
            l[r] += w[e];
          } else {
            // what a row does not see may have any step: it stays out of the sums
            const bool in = full || s[i][e] != -INFINITY;
            l[r] += in ? w[e] * (e & 1 ? inv[i].y : inv[i].x) : 0.f;
          }
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const uint32_t pair = pack2<C>(w[2 * r], w[2 * r + 1]);
          pa[i >> 1][(i & 1) * 2 + r] = pair;
          if constexpr (BITS == 4) {
            // the rounded weights, so that their rounding scales with the value and not
            // with the code's distance from 8
            const float2 f = unpack2<C>(pair);
            zacc[r] += full || s[i][2 * r] != -INFINITY ? f.x * zr[i].x : 0.f;
            zacc[r] += full || s[i][2 * r + 1] != -INFINITY ? f.y * zr[i].y : 0.f;
          }
        }
      }
      if constexpr (BITS == 16) {
        bool odd = false;  // a value that is no number, in a tile that not every row sees whole
        if (!full) {
          for (int i = lane; i < kKeys * kChunks; i += 32) {
            if (i % kChunks * 16 >= row_bytes) continue;
            const uint4 v = *reinterpret_cast<const uint4*>(stp + K::kVOff +
                                                            chunk_at<BITS, kChunks, true>(i / kChunks, i % kChunks));
            const uint32_t ws[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float2 f = unpack2<T>(ws[e]);
              odd |= !isfinite(f.x) || !isfinite(f.y);
            }
          }
          odd = __any_sync(0xffffffffu, odd);
        }
        if (!odd) {
#pragma unroll
          for (int kk = 0; kk < kKeys / 16; ++kk)
#pragma unroll
            for (int d = 0; d < DP / 16; ++d) {
              uint32_t f[4];
              ldsm4_t(st + K::kVOff + chunk_at<BITS, kChunks, true>(kk * 16 + (lane & 15), 2 * d + (lane >> 4)), f);
              mma<C>(o[2 * d], pa[kk], f[0], f[1]);
              mma<C>(o[2 * d + 1], pa[kk], f[2], f[3]);
            }
        } else {
          // zero times such a value is no number: only rows that see a key may touch it
          for (int j = 0; j < kKeys; ++j) {
            const int src = gid * 4 + (j % 8) / 2;
            float w[2];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              const uint32_t pair = __shfl_sync(0xffffffffu, j < 8 ? pa[0][r] : pa[0][2 + r], src);
              const float2 f = unpack2<C>(pair);
              w[r] = j % 2 ? f.y : f.x;
            }
            const bool sees[2] = {j0 + j <= last[0] && j0 + j >= from[0], j0 + j <= last[1] && j0 + j >= from[1]};
#pragma unroll
            for (int i = 0; i < kDt; ++i)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const int d = 8 * i + 2 * tig + e;
                if (d >= D) continue;
                const float v = to_f32(*reinterpret_cast<const T*>(stp + K::kVOff +
                                                                   chunk_at<BITS, kChunks, true>(j, d >> 3) + (d & 7) * 2));
                if (sees[0]) o[i][e] = fmaf(w[0], v, o[i][e]);
                if (sees[1]) o[i][2 + e] = fmaf(w[1], v, o[i][2 + e]);
              }
          }
        }
      } else {
#pragma unroll
        for (int kk = 0; kk < kKeys / 16; ++kk)
#pragma unroll
          for (int n = 0; n < K::kRow / 32; ++n) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int row = kk * 16 + 2 * tig + (e & 1) + (e >> 1) * 8;
              w[e] = *reinterpret_cast<const uint32_t*>(stp + K::kVOff +
                                                        chunk_at<BITS, kChunks, true>(row, 2 * n + (gid >> 2)) + (gid & 3) * 4);
            }
            if constexpr (BITS == 8) {
#pragma unroll
              for (int e = 0; e < 4; ++e) w[e] ^= 0x80808080u;
              // bytes 0 and 1, then 2 and 3, of two rows side by side
              const uint32_t g[2][2] = {{__byte_perm(w[0], w[1], 0x5140), __byte_perm(w[2], w[3], 0x5140)},
                                        {__byte_perm(w[0], w[1], 0x7362), __byte_perm(w[2], w[3], 0x7362)}};
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const uint32_t sel = j & 1 ? 0x4342u : 0x4140u;
                mma<C>(o[4 * n + j], pa[kk], signed8(__byte_perm(g[j >> 1][0], 0x64646464u, sel)),
                       signed8(__byte_perm(g[j >> 1][1], 0x64646464u, sel)));
              }
            } else {
              // codes 0..3, then 4..7, of two rows
              const uint32_t g[2][2] = {{__byte_perm(w[0], w[1], 0x5410), __byte_perm(w[2], w[3], 0x5410)},
                                        {__byte_perm(w[0], w[1], 0x7632), __byte_perm(w[2], w[3], 0x7632)}};
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const uint32_t x = g[j >> 1][0] >> (j & 1 ? 8 : 0), y = g[j >> 1][1] >> (j & 1 ? 8 : 0);
                mma<C>(o[8 * n + 2 * j], pa[kk], signed4<0>(x), signed4<0>(y));
                mma<C>(o[8 * n + 2 * j + 1], pa[kk], signed4<1>(x), signed4<1>(y));
              }
            }
          }
      }
    }
    cp_wait<0>();

    // ---------------------------------------------------------- join the warps, write
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
      if constexpr (BITS == 4) {
        zacc[r] += __shfl_xor_sync(0xffffffffu, zacc[r], 1);
        zacc[r] += __shfl_xor_sync(0xffffffffu, zacc[r], 2);
      }
      if (tig == 0) {
        s_m[warp][gid + 8 * r] = m[r];
        s_l[warp][gid + 8 * r] = l[r];
      }
    }
    __syncthreads();  // also: every warp has read its last stage
    float top[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      top[r] = s_m[0][gid + 8 * r];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) top[r] = fmaxf(top[r], s_m[w][gid + 8 * r]);
      const float keep = ex2(m[r] - (top[r] == -INFINITY ? 0.f : top[r]));
#pragma unroll
      for (int i = 0; i < kDt; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          int d;  // the column this fragment element stands for
          if constexpr (BITS == 16) d = 8 * i + 2 * tig + e;
          else if constexpr (BITS == 8) d = 32 * (i / 4) + 4 * (2 * tig + e) + i % 4;
          else d = 64 * (i / 8) + 8 * (2 * tig + e) + i % 8;
          my_out[(gid + 8 * r) * DP + d] = (o[i][2 * r + e] + zacc[r]) * keep;
        }
    }
    __syncthreads();
    const bool whole = tile == 0 && cnt == p.units;
    const int64_t slot = 2 * static_cast<int64_t>(blockIdx.x) + (first_piece ? 0 : 1);
    for (int i = threadIdx.x; i < rows * (DP / 2); i += kThreads) {
      const int row = i / (DP / 2), d = i % (DP / 2) * 2;
      if (d >= D) continue;
      float mm = s_m[0][row];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) mm = fmaxf(mm, s_m[w][row]);
      const float rr = mm == -INFINITY ? 0.f : mm;
      float sum = 0.f, x = 0.f, y = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        sum += s_l[w][row] * ex2(s_m[w][row] - rr);
        const float2 f = *reinterpret_cast<const float2*>(smem + w * K::kWarpBytes + (row * DP + d) * 4);
        x += f.x;
        y += f.y;
      }
      if (whole) {
        const int tok = (rt * kM + row) / a.group, hh = (rt * kM + row) % a.group;
        const int64_t at = static_cast<int64_t>(p.r.start + tok) * a.q_heads + h * a.group + hh;
        const float n = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);
        *reinterpret_cast<uint32_t*>(static_cast<T*>(a.out) + at * D + d) = pack2<T>(x * n, y * n);
        if (d == 0 && a.lse != nullptr) a.lse[at] = sum == 0.f ? -INFINITY : (mm + log2f(sum)) * kLn2;
      } else {
        *reinterpret_cast<float2*>(parts.o + (slot * kM + row) * DP + d) = make_float2(x, y);
        if (d == 0) parts.ml[slot * kM + row] = make_float2(mm, sum);
      }
    }
    __syncthreads();  // the rings are free again
    u += cnt;
    first_piece = false;
  }
}

// Adds up the parts of heads that were cut: block (row tile and KV head, row of the
// tile). 8 groups of threads take every eighth part; the order of the sums is fixed.
constexpr int kJoinThreads = 256;
template <typename T, int BITS, int DP>
__global__ void __launch_bounds__(kJoinThreads) k_attn_join(const AttnArgs a, const Parts parts, int launched) {
  using K = Cfg<T, BITS, DP>;
  constexpr int kCols = DP / 4, kGroups = kJoinThreads / kCols;
  __shared__ float4 s_o[kGroups][kCols];
  __shared__ float s_l[kGroups], s_m[kJoinThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  grid_dep_wait();
  const int h = blockIdx.x % a.kv.kv_heads, row = blockIdx.y;
  const int64_t which = blockIdx.x / a.kv.kv_heads;
  // (sequence, row tile) number `which`, and the first unit of its sequence
  int b = 0;
  int64_t tile_first = 0, unit_base = 0;
  if (!find_seq(a, which, lane, b, tile_first, [&](int s) { return static_cast<int64_t>(plan_seq(a, s, K::kUnit).row_tiles); }))
    return;
  for (int s = lane; s < b; s += 32) unit_base += plan_seq(a, s, K::kUnit).total(a.kv.kv_heads);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) unit_base += __shfl_xor_sync(0xffffffffu, unit_base, o);
  const int64_t units = all_units(a, K::kUnit, lane);
  const int blocks = sharing(units, launched);
  const SeqPlan p = plan_seq(a, b, K::kUnit);
  const int rt = static_cast<int>(which - tile_first);
  if (row >= min(kM, p.r.q_len * a.group - rt * kM)) return;
  const int64_t u0 = unit_base + (static_cast<int64_t>(rt) * a.kv.kv_heads + h) * p.units;
  const int w0 = owner(units, u0, blocks), w1 = owner(units, u0 + p.units - 1, blocks);
  if (w0 == w1) return;  // one block had it whole
  auto slot = [&](int w) -> int64_t {
    return 2 * static_cast<int64_t>(w) + (w == w0 && first_unit(units, w, blocks) < u0 ? 1 : 0);
  };
  float top = -INFINITY;
  for (int w = w0 + static_cast<int>(threadIdx.x); w <= w1; w += kJoinThreads)
    top = fmaxf(top, parts.ml[slot(w) * kM + row].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane == 0) s_m[warp] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kJoinThreads / 32; ++i) top = fmaxf(top, s_m[i]);
  const float ref = top == -INFINITY ? 0.f : top;
  const int col = threadIdx.x % kCols, grp = threadIdx.x / kCols;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float l = 0.f;
#pragma unroll 4
  for (int w = w0 + grp; w <= w1; w += kGroups) {
    const int64_t s = slot(w) * kM + row;
    const float2 ml = parts.ml[s];
    const float4 v = *reinterpret_cast<const float4*>(parts.o + s * DP + col * 4);
    const float f = ex2(ml.x - ref);
    l = fmaf(ml.y, f, l);
    acc.x = fmaf(v.x, f, acc.x);
    acc.y = fmaf(v.y, f, acc.y);
    acc.z = fmaf(v.z, f, acc.z);
    acc.w = fmaf(v.w, f, acc.w);
  }
  s_o[grp][col] = acc;
  if (col == 0) s_l[grp] = l;
  __syncthreads();
  if (grp != 0 || col * 4 >= a.kv.head_dim) return;
  for (int g = 1; g < kGroups; ++g) {
    const float4 v = s_o[g][col];
    acc.x += v.x;
    acc.y += v.y;
    acc.z += v.z;
    acc.w += v.w;
    l += s_l[g];
  }
  const int tok = (rt * kM + row) / a.group, hh = (rt * kM + row) % a.group;
  const int64_t at = static_cast<int64_t>(p.r.start + tok) * a.q_heads + h * a.group + hh;
  const float n = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
  uint2 out;
  out.x = pack2<T>(acc.x * n, acc.y * n);
  out.y = pack2<T>(acc.z * n, acc.w * n);
  *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + at * a.kv.head_dim + col * 4) = out;
  if (col == 0 && a.lse != nullptr) a.lse[at] = l == 0.f ? -INFINITY : (top + log2f(l)) * kLn2;
}

// ------------------------------------------------------------------ host
template <typename T, int BITS, int DP>
struct Few {
  using K = Cfg<T, BITS, DP>;
  static std::atomic<size_t> raised[kMaxDevices];
  static std::atomic<int> resident;

  // Blocks of the axis: all that are resident at once.
  static int blocks(cudaError_t* err) {
    *err = raise_smem_limit(k_attn_few<T, BITS, DP>, K::kSmem, raised);
    int n = resident.load();
    if (n == 0 && *err == cudaSuccess) {
      *err = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, k_attn_few<T, BITS, DP>, kThreads, K::kSmem);
      n = std::max(1, n);
      if (*err == cudaSuccess) resident.store(n);
    }
    return device_sm_count() * std::max(1, n);
  }
  static size_t workspace(cudaError_t* err) {
    const size_t slots = 2 * static_cast<size_t>(blocks(err));
    return slots * kM * (DP * sizeof(float) + sizeof(float2));
  }
  static cudaError_t launch(const AttnArgs& a, void* ws, cudaStream_t s) {
    cudaError_t e;
    const int n = blocks(&e);
    if (e != cudaSuccess) return e;
    Parts parts;
    parts.o = static_cast<float*>(ws);
    parts.ml = reinterpret_cast<float2*>(parts.o + 2 * static_cast<size_t>(n) * kM * DP);
    e = launch_dep(k_attn_few<T, BITS, DP>, dim3(static_cast<unsigned>(n)), dim3(kThreads), K::kSmem, s, a, parts);
    if (e != cudaSuccess) return e;
    // at most this many row tiles: each sequence may end in a partial one
    const int64_t rows = static_cast<int64_t>(a.num_tokens) * a.group;
    const int64_t tiles = std::min<int64_t>(rows, rows / kM + a.num_seqs);
    return launch_dep(k_attn_join<T, BITS, DP>, dim3(static_cast<unsigned>(tiles * a.kv.kv_heads), static_cast<unsigned>(std::min<int64_t>(kM, rows))),
                      dim3(kJoinThreads), 0, s, a, parts, n);
  }
};
template <typename T, int BITS, int DP>
std::atomic<size_t> Few<T, BITS, DP>::raised[kMaxDevices];
template <typename T, int BITS, int DP>
std::atomic<int> Few<T, BITS, DP>::resident{0};

template <typename F>
auto with_few(int bits, bool bf16, int head_dim, F&& f) {
  auto dim = [&](auto t, auto b) {
    if (head_dim <= 64) return f(Few<decltype(t), decltype(b)::value, 64>());
    if (head_dim <= 128) return f(Few<decltype(t), decltype(b)::value, 128>());
    return f(Few<decltype(t), decltype(b)::value, 256>());
  };
  auto form = [&](auto t) {
    if (bits == 16) return dim(t, std::integral_constant<int, 16>());
    if (bits == 8) return dim(t, std::integral_constant<int, 8>());
    return dim(t, std::integral_constant<int, 4>());
  };
  return bf16 ? form(__nv_bfloat16()) : form(__half());
}

}  // namespace

size_t attention_workspace(const AttnArgs& a, int bits, bool bf16, int, int) {
  cudaError_t e = cudaSuccess;
  return with_few(bits, bf16, a.kv.head_dim, [&](auto k) { return decltype(k)::workspace(&e); });
}

cudaError_t launch_attention(const AttnArgs& a, int bits, bool bf16, int, int, void* workspace, cudaStream_t s) {
  return with_few(bits, bf16, a.kv.head_dim, [&](auto k) { return decltype(k)::launch(a, workspace, s); });
}

}  // namespace gemq
