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
// are the time. Rows (tokens x query heads that share the KV head) are the N of
// mma.sync: S^T = K Q^T and O^T = V^T P^T with 16 keys, or 16 columns of v, as M, so a
// step of 8 rows wastes nothing and every unpacked key or value serves all rows of the
// tile (8, 16 or 32). That takes a fraction of the legacy tensor rate even at 4 bits, so
// tensor memory would only add its round trips. Every warp streams its own tiles of 16 or
// 32 keys through its own cp.async ring, without block barriers; the keys of all
// sequences and heads form one axis of 64- or 128-key units that is cut evenly over all
// resident blocks (so uneven lengths do not matter), and k_attn_join adds up heads that
// were cut.
//
// Measured on a B200: 2 sequences of 131,072, 32 query and 8 KV heads x 128, bf16: 164 us,
// 6.5 TB/s, bytes. 64 uneven ones up to 8,192, 32 on 4 heads, 8 bits: 62 us, 4.6 TB/s, and
// 16 up to 4,096, 5 tokens each, 16 heads, 4 bits: 39.5 us, 2.2 TB/s: neither bytes (57% and
// 28% of the DRAM's time) nor issue slots (58% and 55%) are used up; a scheduler has two or
// three warps, each a chain of unpacking, product, maximum, exponentials and product, and
// the second spends a third of its time on pieces' set-up and join. 1 of 2,048, 16 heads,
// fp16: 9.8 us, 1.7 TB/s, latency (page table, keys, join in turn).
#include <algorithm>

#include "paged.cuh"

namespace gemq {

namespace {

// ------------------------------------------------------------------ small pieces
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
// Transposes the 8x8 16-bit matrix that a warp holds two neighbours of a row a lane.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
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

// NR: tiles of 8 rows that a warp holds.
template <typename T, int BITS, int DP, int NR>
struct Cfg {
  static constexpr int kM = 8 * NR;
  static constexpr int kKeys = BITS == 16 ? 16 : 32;  // keys of one warp's tile
  static constexpr int kUnit = kKeys * kWarps;        // keys of one unit of the axis
  static constexpr int kRow = DP * BITS / 8;          // bytes of a staged row
  static constexpr int kChunks = kRow / 16;
  static constexpr int kBlocks = DP == 256 ? (NR == 1 ? 2 : 1) : NR * DP >= 256 ? 2 : 3;  // resident on an SM
  static constexpr int kStages = DP * BITS >= 4096 ? 3 : DP * BITS >= 1024 ? 2 : 3;
  static constexpr int kScale = BITS == 16 ? 0 : BITS == 8 ? 4 : 8;  // bytes of a row's scale
  static constexpr int kVOff = kKeys * kRow;
  static constexpr int kScOff = 2 * kKeys * kRow;
  static constexpr int kStage = kScOff + 2 * kKeys * kScale;
  // a tile's scales as the scores take them: [keys] each of a, log2 step, 1 / step, z, y / step
  static constexpr int kPrep = BITS == 16 ? 0 : 5 * kKeys * 4;
  static constexpr int kWarpBytes = kStages * kStage + kPrep;
  static constexpr int kSmem = kWarps * kWarpBytes;
  static constexpr int kOutFloats = kM * DP;             // of a warp's output tile
  // the output tile takes the ring's place at the end, in row slices where it is larger
  static constexpr int kSlices = (kOutFloats * 4 + kWarpBytes - 1) / kWarpBytes;
  static constexpr int kSliceRows = kSlices == 1 ? kM : 8;
  static_assert(kSliceRows * DP * 4 <= kWarpBytes, "a slice must fit the ring");
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
template <int M>
__device__ __forceinline__ SeqPlan plan_seq(const AttnArgs& a, int b, int unit) {
  SeqPlan p;
  p.r = seq_range(a, b);
  p.row_tiles = (p.r.q_len * a.group + M - 1) / M;
  p.t0 = first_seen(p.r.kv_len - p.r.q_len, a.window) / unit;
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
template <int M>
__device__ __forceinline__ int64_t all_units(const AttnArgs& a, int unit, int lane) {
  int64_t sum = 0;
  for (int b = lane; b < a.num_seqs; b += 32) sum += plan_seq<M>(a, b, unit).total(a.kv.kv_heads);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  return sum;
}
// The sequence that unit u lies in and its first unit.
template <int M>
__device__ __forceinline__ bool find_seq(const AttnArgs& a, int64_t u, int unit, int lane, int& b, int64_t& first) {
  int64_t base = 0;
  for (int b0 = 0; b0 < a.num_seqs; b0 += 32) {
    const int64_t n = b0 + lane < a.num_seqs ? plan_seq<M>(a, b0 + lane, unit).total(a.kv.kv_heads) : 0;
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

// Blocks that share the units (each has at least one), the first unit of block w of n,
// and the block that unit u falls to.
__device__ __forceinline__ int sharing(int64_t units, int blocks) {
  return static_cast<int>(min(units, static_cast<int64_t>(blocks)));
}
__device__ __forceinline__ int64_t first_unit(int64_t units, int w, int n) { return units * w / n; }
__device__ __forceinline__ int owner(int64_t units, int64_t u, int n) {
  return static_cast<int>(((u + 1) * n - 1) / units);
}

// Unnormalised parts of heads that several blocks share: block w's first piece in slot
// 2 w, a last piece that another block goes on with in 2 w + 1. The block that ends such
// a head leaves a note of it.
struct Note {
  int first, odd;  // the block that began the head, and whether in its odd slot
  int rows;        // 0: this block ends no shared head
  int start;       // first token of the sequence
  int row0, head;  // first row of the tile in the sequence, KV head
  int pad[2];
};
struct Parts {
  float* o;    // [slots][kM][DP]
  float2* ml;  // [slots][kM]: reference m, sum l
  Note* note;  // [blocks]
};

// ------------------------------------------------------------------ the kernel
template <typename T, int BITS, int DP, int NR>
__global__ void __launch_bounds__(kThreads, Cfg<T, BITS, DP, NR>::kBlocks) k_attn_few(const AttnArgs a, const Parts parts) {
  using K = Cfg<T, BITS, DP, NR>;
  using C = typename K::C;
  constexpr int kKeys = K::kKeys, kChunks = K::kChunks, kStages = K::kStages, kM = K::kM;
  constexpr int kMt = kKeys / 16;   // score tiles of 16 keys
  constexpr int kKs = DP / 16;      // k steps of q.k, and output tiles of 16 columns
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
  const int64_t units = all_units<kM>(a, K::kUnit, lane);
  const int blocks = sharing(units, gridDim.x);
  Note note{};
  int64_t u = 0, u_end = 0;
  if (static_cast<int>(blockIdx.x) < blocks) {
    u = first_unit(units, blockIdx.x, blocks);
    u_end = first_unit(units, blockIdx.x + 1, blocks);
  }
  bool first_piece = true;
  int64_t seq_first = 0, seq_end = 0;
  int b = 0;
  SeqPlan p{};
  while (u < u_end) {
    if (u >= seq_end) {
      if (!find_seq<kM>(a, u, K::kUnit, lane, b, seq_first)) break;
      p = plan_seq<kM>(a, b, K::kUnit);
      seq_end = seq_first + p.total(a.kv.kv_heads);
    }
    // the piece: units [tile, tile + cnt) of KV head h, row tile rt
    const int64_t local = u - seq_first;
    const int item = static_cast<int>(local / p.units), tile = static_cast<int>(local % p.units);
    const int rt = item / a.kv.kv_heads, h = item % a.kv.kv_heads;
    const int cnt = static_cast<int>(min(static_cast<int64_t>(p.units - tile), u_end - u));
    const int rows = min(kM, p.r.q_len * a.group - rt * kM);
    const int pos0 = p.r.kv_len - p.r.q_len;  // position of the first new token
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
    // As the B operand: row gid of each tile, two k pairs a step. k index <-> element: in
    // order for 16 bits; for codes the order in which a thread's contiguous quarter of a
    // key unpacks (a dot product takes any).
    uint32_t qb[NR][kKs][2];
    // of the rows this thread has scores of, 2 tig + e of each tile: the last and first
    // position they see; row factor and sum of the queries
    int last[NR][2], from[NR][2];
    float rf[NR][2], qsum[NR][2];
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      const int r = 8 * i + gid;
      const int tok = (rt * kM + r) / a.group, hh = (rt * kM + r) % a.group;
      const bool in = r < rows;
      const T* q = static_cast<const T*>(a.q) + (in ? (p.r.start + tok) * a.q_token_stride +
                                                          static_cast<int64_t>(h * a.group + hh) * D
                                                    : 0);
      float factor = 1.f, sum = 0.f;
      if constexpr (K::kRowFactor) {
        // bf16 queries against fp16 codes: each row scaled by a power of two to at most 2,
        // which costs only what lies 2^-24 below its largest element
        float most = 0.f;
        for (int d = tig * 8; in && d < D; d += 32) {
          const uint4 w = *reinterpret_cast<const uint4*>(q + d);
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
        factor = exp2f(static_cast<float>(e));
      }
      const float inv_factor = 1.f / factor;
      auto conv = [&](uint32_t pair) -> uint32_t {
        if constexpr (!K::kRowFactor) return pair;
        const float2 f = unpack2<T>(pair);
        return pack2<__half>(f.x * inv_factor, f.y * inv_factor);
      };
      if constexpr (BITS == 16) {
#pragma unroll
        for (int ks = 0; ks < kKs; ++ks)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int d = ks * 16 + 8 * e + 2 * tig;
            qb[i][ks][e] = in && d < D ? *reinterpret_cast<const uint32_t*>(q + d) : 0u;
          }
      } else if constexpr (BITS == 8) {
#pragma unroll
        for (int ks = 0; ks < kKs; ++ks) {
          const int d = tig * (DP / 4) + 4 * ks;
          const uint2 w = in && d < D ? *reinterpret_cast<const uint2*>(q + d) : make_uint2(0u, 0u);
          qb[i][ks][0] = conv(w.x);
          qb[i][ks][1] = conv(w.y);
        }
      } else {
#pragma unroll
        for (int k2 = 0; k2 < kKs / 2; ++k2) {
          const int d = tig * (DP / 4) + 8 * k2;
          const uint4 w = in && d < D ? *reinterpret_cast<const uint4*>(q + d) : make_uint4(0u, 0u, 0u, 0u);
          // elements (0, 4), (1, 5), (2, 6), (3, 7): a word's nibbles and those 16 bits up
          qb[i][2 * k2][0] = conv(__byte_perm(w.x, w.z, 0x5410));
          qb[i][2 * k2][1] = conv(__byte_perm(w.x, w.z, 0x7632));
          qb[i][2 * k2 + 1][0] = conv(__byte_perm(w.y, w.w, 0x5410));
          qb[i][2 * k2 + 1][1] = conv(__byte_perm(w.y, w.w, 0x7632));
        }
      }
      if constexpr (BITS != 16) {
#pragma unroll
        for (int ks = 0; ks < kKs; ++ks)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float2 f = __half22float2(u32_as_h2(qb[i][ks][e]));
            sum += f.x + f.y;
          }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        if constexpr (K::kRowFactor) factor *= 16777216.f;  // undoes the subnormal codes' 2^-24
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int c = 8 * i + 2 * tig + e;
        last[i][e] = c < rows ? pos0 + (rt * kM + c) / a.group : -1;
        from[i][e] = first_seen(last[i][e], a.window);
        if constexpr (BITS != 16) {
          rf[i][e] = __shfl_sync(0xffffffffu, factor, (2 * tig + e) * 4);
          qsum[i][e] = __shfl_sync(0xffffffffu, sum, (2 * tig + e) * 4);
        }
      }
    }

    // ---------------------------------------------------------- the keys
    float o[kKs][NR][4];
#pragma unroll
    for (int i = 0; i < kKs; ++i)
#pragma unroll
      for (int r = 0; r < NR; ++r) o[i][r][0] = o[i][r][1] = o[i][r][2] = o[i][r][3] = 0.f;
    float m[NR][2], l[NR][2], zacc[NR][2];
#pragma unroll
    for (int r = 0; r < NR; ++r)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        m[r][e] = -INFINITY;
        l[r][e] = zacc[r][e] = 0.f;
      }
    for (int t = 0; t < cnt; ++t) {
      cp_wait<kStages - 2>();
      __syncwarp();
      load(t + kStages - 1);
      const uint32_t st = ring + static_cast<uint32_t>(t % kStages) * K::kStage;
      const uint8_t* const stp = smem + (st - smem_u32(smem));
      const int j0 = tile_key + t * K::kUnit;
      if (j0 > tile_max) continue;  // nothing here for any row
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
        vstep = value_step(vstep, vbase);
        const float lv = lg2(vstep);
        prep[lane] = step * cs * kUp;
        prep[kKeys + lane] = lv;
        prep[2 * kKeys + lane] = ex2(-lv);
        prep[3 * kKeys + lane] = base * cs * kDown;
        // (the rounded quotient: codes and base nearly cancel where a value is near zero)
        if constexpr (BITS == 4) prep[4 * kKeys + lane] = vbase / vstep;
      }
      // s[i][r]: keys 16 i + gid (elements 0, 1) and + 8 (2, 3), rows 8 r + 2 tig + e
      float s[kMt][NR][4];
#pragma unroll
      for (int i = 0; i < kMt; ++i)
#pragma unroll
        for (int r = 0; r < NR; ++r) s[i][r][0] = s[i][r][1] = s[i][r][2] = s[i][r][3] = 0.f;
      if constexpr (BITS == 16) {
#pragma unroll
        for (int ks = 0; ks < kKs; ++ks) {
          uint32_t f[4];
          ldsm4(st + chunk_at<BITS, kChunks, false>(lane & 15, 2 * ks + (lane >> 4)), f);
#pragma unroll
          for (int r = 0; r < NR; ++r) mma<C>(s[0][r], f, qb[r][ks][0], qb[r][ks][1]);
        }
      } else {
        constexpr int kBytes = DP * BITS / 32;          // of a row, a thread
        constexpr int kWords = kBytes >= 16 ? 4 : 2;    // a load
        using Words = std::conditional_t<kWords == 4, uint4, uint2>;
#pragma unroll
        for (int n = 0; n < kBytes / (4 * kWords); ++n) {
          uint32_t w[kMt][2][4];  // keys gid, gid + 8 of each tile
#pragma unroll
          for (int i = 0; i < kMt; ++i)
#pragma unroll
            for (int hi = 0; hi < 2; ++hi) {
              const int byte = tig * kBytes + n * 4 * kWords;
              const Words ww = *reinterpret_cast<const Words*>(
                  stp + chunk_at<BITS, kChunks, false>(16 * i + 8 * hi + gid, byte >> 4) + (byte & 15));
              w[i][hi][0] = ww.x;
              w[i][hi][1] = ww.y;
              if constexpr (kWords == 4) {
                w[i][hi][2] = ww.z;
                w[i][hi][3] = ww.w;
              }
            }
#pragma unroll
          for (int e = 0; e < kWords; ++e) {
            const int ks = n * kWords + e;
#pragma unroll
            for (int i = 0; i < kMt; ++i) {
              const uint32_t x = w[i][0][e], y = w[i][1][e];
              if constexpr (BITS == 8) {
                const uint32_t xb = x ^ 0x80808080u, yb = y ^ 0x80808080u;
                const uint32_t f[4] = {__byte_perm(xb, 0u, 0x4140), __byte_perm(yb, 0u, 0x4140),
                                       __byte_perm(xb, 0u, 0x4342), __byte_perm(yb, 0u, 0x4342)};
#pragma unroll
                for (int r = 0; r < NR; ++r) mma<C>(s[i][r], f, qb[r][ks][0], qb[r][ks][1]);
              } else {
                constexpr uint32_t kLow = 0x000f000fu;
                const uint32_t f[4] = {x & kLow, y & kLow, (x >> 4) & kLow, (y >> 4) & kLow};
                const uint32_t g[4] = {(x >> 8) & kLow, (y >> 8) & kLow, (x >> 12) & kLow, (y >> 12) & kLow};
#pragma unroll
                for (int r = 0; r < NR; ++r) {
                  mma<C>(s[i][r], f, qb[r][2 * ks][0], qb[r][2 * ks][1]);
                  mma<C>(s[i][r], g, qb[r][2 * ks + 1][0], qb[r][2 * ks + 1][1]);
                }
              }
            }
          }
        }
      }
      // scores, in powers of two
      float inv[kMt][2], zr[kMt][2];
      if constexpr (BITS == 16) {
#pragma unroll
        for (int r = 0; r < NR; ++r)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[0][r][e] *= cs;
      } else {
        __syncwarp();
#pragma unroll
        for (int i = 0; i < kMt; ++i)
#pragma unroll
          for (int hi = 0; hi < 2; ++hi) {
            const int j = 16 * i + 8 * hi + gid;
            const float aj = prep[j], lv = prep[kKeys + j], zj = prep[3 * kKeys + j];
            inv[i][hi] = prep[2 * kKeys + j];
            if constexpr (BITS == 4) zr[i][hi] = prep[4 * kKeys + j];
#pragma unroll
            for (int r = 0; r < NR; ++r)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                float& x = s[i][r][2 * hi + e];
                if constexpr (K::kRowFactor) x = fmaf(fmaf(qsum[r][e], zj, x * aj), rf[r][e], lv);
                else x = fmaf(x, aj, fmaf(qsum[r][e], zj, lv));
              }
          }
      }
      const bool full = j0 + kKeys - 1 <= tile_min && (a.window <= 0 || tile_max - j0 < a.window);
      if (!full) {
#pragma unroll
        for (int i = 0; i < kMt; ++i)
#pragma unroll
          for (int r = 0; r < NR; ++r)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int j = j0 + 16 * i + 8 * (e >> 1) + gid;
              if (j > last[r][e & 1] || j < from[r][e & 1]) s[i][r][e] = -INFINITY;
            }
        if constexpr (BITS != 16) {
          // what no row sees may have any step: a key's factors count only where it is seen
#pragma unroll
          for (int i = 0; i < kMt; ++i)
#pragma unroll
            for (int hi = 0; hi < 2; ++hi) {
              const bool odd = !(inv[i][hi] < INFINITY) || (BITS == 4 && !(fabsf(zr[i][hi]) < INFINITY));
              const int j = j0 + 16 * i + 8 * hi + gid;
              if (odd && j > tile_min) inv[i][hi] = zr[i][hi] = 0.f;
              if (odd && a.window > 0 && tile_max - j >= a.window) inv[i][hi] = zr[i][hi] = 0.f;
            }
        }
      }
      float ref[NR][2], now[NR][2];
      bool moved = false;
#pragma unroll
      for (int r = 0; r < NR; ++r)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float top = m[r][e];
#pragma unroll
          for (int i = 0; i < kMt; ++i) top = fmaxf(top, fmaxf(s[i][r][e], s[i][r][2 + e]));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
          ref[r][e] = top == -INFINITY ? 0.f : top;
          now[r][e] = top;
          moved |= top != m[r][e];
        }
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int r = 0; r < NR; ++r)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float keep = ex2(m[r][e] - ref[r][e]);
            l[r][e] *= keep;
            zacc[r][e] *= keep;
#pragma unroll
            for (int i = 0; i < kKs; ++i) {
              o[i][r][e] *= keep;
              o[i][r][2 + e] *= keep;
            }
            m[r][e] = now[r][e];
          }
      }
      // weights; pairs of rows, then (transposed) pairs of keys as the B operand
      uint32_t pw[kMt][NR][2], pb[kMt][NR][2];
#pragma unroll
      for (int i = 0; i < kMt; ++i)
#pragma unroll
        for (int r = 0; r < NR; ++r)
#pragma unroll
          for (int hi = 0; hi < 2; ++hi) {
            const float w0 = ex2(s[i][r][2 * hi] - ref[r][0]), w1 = ex2(s[i][r][2 * hi + 1] - ref[r][1]);
            const uint32_t pair = pack2<C>(w0, w1);
            pw[i][r][hi] = pair;
            pb[i][r][hi] = transpose8(pair);
            if constexpr (BITS == 16) {
              l[r][0] += w0;
              l[r][1] += w1;
            } else {
              l[r][0] = fmaf(w0, inv[i][hi], l[r][0]);
              l[r][1] = fmaf(w1, inv[i][hi], l[r][1]);
              if constexpr (BITS == 4) {
                // the rounded weights, so that their rounding scales with the value and
                // not with the code's distance from 8 (but below fp16's normal range,
                // where a row of equal values comes with its tiny step, the weight itself)
                const float2 f = unpack2<C>(pair);
                zacc[r][0] = fmaf(w0 < kHalfMin ? w0 : f.x, zr[i][hi], zacc[r][0]);
                zacc[r][1] = fmaf(w1 < kHalfMin ? w1 : f.y, zr[i][hi], zacc[r][1]);
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
          for (int d = 0; d < kKs; ++d) {
            uint32_t f[4];
            ldsm4_t(st + K::kVOff + chunk_at<BITS, kChunks, true>((lane & 7) + ((lane >> 4) << 3), 2 * d + ((lane >> 3) & 1)), f);
#pragma unroll
            for (int r = 0; r < NR; ++r) mma<C>(o[d][r], f, pb[0][r][0], pb[0][r][1]);
          }
        } else {
          // zero times such a value is no number: only rows that see a key may touch it
          for (int j = 0; j < kKeys; ++j) {
#pragma unroll
            for (int r = 0; r < NR; ++r) {
              const float2 w = unpack2<C>(__shfl_sync(0xffffffffu, j < 8 ? pw[0][r][0] : pw[0][r][1], (j % 8) * 4 + tig));
              const bool see0 = j0 + j <= last[r][0] && j0 + j >= from[r][0];
              const bool see1 = j0 + j <= last[r][1] && j0 + j >= from[r][1];
#pragma unroll
              for (int i = 0; i < kKs; ++i)
#pragma unroll
                for (int hi = 0; hi < 2; ++hi) {
                  const int d = 16 * i + 8 * hi + gid;
                  if (d >= D) continue;
                  const float v = to_f32(*reinterpret_cast<const T*>(stp + K::kVOff + chunk_at<BITS, kChunks, true>(j, d >> 3) + (d & 7) * 2));
                  if (see0) o[i][r][2 * hi] = fmaf(w.x, v, o[i][r][2 * hi]);
                  if (see1) o[i][r][2 * hi + 1] = fmaf(w.y, v, o[i][r][2 * hi + 1]);
                }
            }
          }
        }
      } else {
#pragma unroll
        for (int kk = 0; kk < kMt; ++kk)
#pragma unroll
          for (int n = 0; n < K::kRow / 32; ++n) {
            uint32_t w[4];  // the same columns of keys 2 tig, + 1, + 8, + 9
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int row = kk * 16 + 2 * tig + (e & 1) + (e >> 1) * 8;
              w[e] = *reinterpret_cast<const uint32_t*>(stp + K::kVOff +
                                                        chunk_at<BITS, kChunks, true>(row, 2 * n + (gid >> 2)) + (gid & 3) * 4);
            }
            if constexpr (BITS == 8) {
#pragma unroll
              for (int e = 0; e < 4; ++e) w[e] ^= 0x80808080u;
              // bytes 0 and 1, then 2 and 3, of two keys side by side
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                const uint32_t sel = j ? 0x7362u : 0x5140u;
                const uint32_t x = __byte_perm(w[0], w[1], sel), y = __byte_perm(w[2], w[3], sel);
                const uint32_t f[4] = {signed8(__byte_perm(x, 0x64646464u, 0x4140)), signed8(__byte_perm(x, 0x64646464u, 0x4342)),
                                       signed8(__byte_perm(y, 0x64646464u, 0x4140)), signed8(__byte_perm(y, 0x64646464u, 0x4342))};
#pragma unroll
                for (int r = 0; r < NR; ++r) mma<C>(o[2 * n + j][r], f, pb[kk][r][0], pb[kk][r][1]);
              }
            } else {
              // codes 0..3, then 4..7, of two keys
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const uint32_t sel = j & 2 ? 0x7632u : 0x5410u;
                const uint32_t x = __byte_perm(w[0], w[1], sel) >> (j & 1 ? 8 : 0);
                const uint32_t y = __byte_perm(w[2], w[3], sel) >> (j & 1 ? 8 : 0);
                const uint32_t f[4] = {signed4<0>(x), signed4<1>(x), signed4<0>(y), signed4<1>(y)};
#pragma unroll
                for (int r = 0; r < NR; ++r) mma<C>(o[4 * n + j][r], f, pb[kk][r][0], pb[kk][r][1]);
              }
            }
          }
      }
    }
    cp_wait<0>();

    // ---------------------------------------------------------- join the warps, write
#pragma unroll
    for (int r = 0; r < NR; ++r)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) {
          l[r][e] += __shfl_xor_sync(0xffffffffu, l[r][e], x);
          if constexpr (BITS == 4) zacc[r][e] += __shfl_xor_sync(0xffffffffu, zacc[r][e], x);
        }
        if (gid == 0) {
          s_m[warp][8 * r + 2 * tig + e] = m[r][e];
          s_l[warp][8 * r + 2 * tig + e] = l[r][e];
        }
      }
    __syncthreads();  // also: every warp has read its last stage
    const bool whole = tile == 0 && cnt == p.units;
    const int64_t slot = 2 * static_cast<int64_t>(blockIdx.x) + (first_piece ? 0 : 1);
    constexpr int kSliceRows = K::kSliceRows;
#pragma unroll
    for (int r0 = 0; r0 < kM; r0 += kSliceRows) {
      if (r0 > 0) __syncthreads();  // the slice before has been read
#pragma unroll
      for (int r = r0 / 8; r < (r0 + kSliceRows) / 8; ++r)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int row = 8 * r + 2 * tig + e;
          float top = s_m[0][row];
#pragma unroll
          for (int w = 1; w < kWarps; ++w) top = fmaxf(top, s_m[w][row]);
          const float keep = ex2(m[r][e] - (top == -INFINITY ? 0.f : top));
          if (row < rows) {
#pragma unroll
            for (int i = 0; i < kKs; ++i)
#pragma unroll
              for (int hi = 0; hi < 2; ++hi) {
                int d;  // the column this fragment element stands for
                if constexpr (BITS == 16) d = 16 * i + 8 * hi + gid;
                else if constexpr (BITS == 8) d = 32 * (i / 2) + 4 * gid + 2 * (i % 2) + hi;
                else d = 64 * (i / 4) + 8 * gid + 2 * (i % 4) + hi;
                my_out[(row - r0) * DP + d] = (o[i][r][2 * hi + e] + zacc[r][e]) * keep;
              }
          }
        }
      __syncthreads();
      const int here = min(rows - r0, kSliceRows);
      for (int i = threadIdx.x; i < here * (DP / 2); i += kThreads) {
        const int at_row = i / (DP / 2), row = r0 + at_row, d = i % (DP / 2) * 2;
        if (d >= D) continue;
        float mm = s_m[0][row];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) mm = fmaxf(mm, s_m[w][row]);
        const float rr = mm == -INFINITY ? 0.f : mm;
        float sum = 0.f, x = 0.f, y = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          sum += s_l[w][row] * ex2(s_m[w][row] - rr);
          const float2 f = *reinterpret_cast<const float2*>(smem + w * K::kWarpBytes + (at_row * DP + d) * 4);
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
    }
    if (!whole && tile + cnt == p.units) {  // (tile > 0: this block's first piece)
      const int64_t u0 = u - tile;
      note.first = owner(units, u0, blocks);
      note.odd = first_unit(units, note.first, blocks) < u0;
      note.rows = rows;
      note.start = p.r.start;
      note.row0 = rt * kM;
      note.head = h;
    }
    __syncthreads();  // the rings are free again
    u += cnt;
    first_piece = false;
  }
  if (threadIdx.x == 0) parts.note[blockIdx.x] = note;
}

// Adds up the parts of a head that was cut, as the block that ended it noted: 8 groups of
// threads (4 for 256 columns), a row each where the parts are few, else every 8th part of
// one row. The order of the sums is fixed.
constexpr int kJoinThreads = 256;
template <typename T, int DP, int M>
__global__ void __launch_bounds__(kJoinThreads) k_attn_join(const AttnArgs a, const Parts parts) {
  constexpr int kCols = DP / 4, kGroups = kJoinThreads / kCols;
  __shared__ float4 s_o[kGroups][kCols];
  __shared__ float s_l[kGroups], s_m[kJoinThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int col = threadIdx.x % kCols, grp = threadIdx.x / kCols;
  grid_dep_wait();
  const int w1 = blockIdx.x;
  const Note note = parts.note[w1];
  auto slot = [&](int w) -> int64_t { return 2 * static_cast<int64_t>(w) + (w == note.first ? note.odd : 0); };
  auto write = [&](int row, float4 acc, float l, float top) {
    const int r = note.row0 + row;
    const int64_t at = static_cast<int64_t>(note.start + r / a.group) * a.q_heads + note.head * a.group + r % a.group;
    const float n = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
    if (col * 4 < a.kv.head_dim) {
      uint2 out;
      out.x = pack2<T>(acc.x * n, acc.y * n);
      out.y = pack2<T>(acc.z * n, acc.w * n);
      *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + at * a.kv.head_dim + col * 4) = out;
    }
    if (col == 0 && a.lse != nullptr) a.lse[at] = l == 0.f ? -INFINITY : (top + log2f(l)) * kLn2;
  };
  auto add = [&](int row, int w, float ref, float4& acc, float& l) {
    const int64_t s = slot(w) * M + row;
    const float2 ml = parts.ml[s];
    const float4 v = *reinterpret_cast<const float4*>(parts.o + s * DP + col * 4);
    const float f = ex2(ml.x - ref);
    l = fmaf(ml.y, f, l);
    acc.x = fmaf(v.x, f, acc.x);
    acc.y = fmaf(v.y, f, acc.y);
    acc.z = fmaf(v.z, f, acc.z);
    acc.w = fmaf(v.w, f, acc.w);
  };
  if (w1 - note.first < 2 * kGroups) {
    for (int row = blockIdx.y * kGroups + grp; row < note.rows; row += gridDim.y * kGroups) {
      float top = -INFINITY;
      for (int w = note.first; w <= w1; ++w) top = fmaxf(top, parts.ml[slot(w) * M + row].x);
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      float l = 0.f;
#pragma unroll 4
      for (int w = note.first; w <= w1; ++w) add(row, w, top == -INFINITY ? 0.f : top, acc, l);
      write(row, acc, l, top);
    }
    return;
  }
  for (int row = blockIdx.y; row < note.rows; row += gridDim.y) {
    float top = -INFINITY;
    for (int w = note.first + static_cast<int>(threadIdx.x); w <= w1; w += kJoinThreads)
      top = fmaxf(top, parts.ml[slot(w) * M + row].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    __syncthreads();  // the row before has been read
    if (lane == 0) s_m[warp] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kJoinThreads / 32; ++i) top = fmaxf(top, s_m[i]);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = 0.f;
#pragma unroll 4
    for (int w = note.first + grp; w <= w1; w += kGroups) add(row, w, top == -INFINITY ? 0.f : top, acc, l);
    s_o[grp][col] = acc;
    if (col == 0) s_l[grp] = l;
    __syncthreads();
    if (grp == 0) {
      for (int g = 1; g < kGroups; ++g) {
        const float4 v = s_o[g][col];
        acc.x += v.x;
        acc.y += v.y;
        acc.z += v.z;
        acc.w += v.w;
        l += s_l[g];
      }
      write(row, acc, l, top);
    }
  }
}

// ------------------------------------------------------------------ host
template <typename T, int BITS, int DP, int NR>
struct Few {
  using K = Cfg<T, BITS, DP, NR>;
  static std::atomic<size_t> raised[kMaxDevices];
  static std::atomic<int> resident;

  // Blocks of the axis: all that are resident at once.
  static int blocks(cudaError_t* err) {
    *err = raise_smem_limit(k_attn_few<T, BITS, DP, NR>, K::kSmem, raised);
    int n = resident.load();
    if (n == 0 && *err == cudaSuccess) {
      *err = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, k_attn_few<T, BITS, DP, NR>, kThreads, K::kSmem);
      n = std::max(1, n);
      if (*err == cudaSuccess) resident.store(n);
    }
    return device_sm_count() * std::max(1, n);
  }
  static size_t workspace() {
    cudaError_t e;
    const size_t n = static_cast<size_t>(blocks(&e));
    return n * (2 * K::kM * (DP * sizeof(float) + sizeof(float2)) + sizeof(Note));
  }
  static cudaError_t launch(const AttnArgs& a, int rows, void* ws, cudaStream_t s) {
    cudaError_t e;
    const int n = blocks(&e);
    if (e != cudaSuccess) return e;
    Parts parts;
    parts.o = static_cast<float*>(ws);
    parts.note = reinterpret_cast<Note*>(parts.o + 2 * static_cast<size_t>(n) * K::kM * DP);
    parts.ml = reinterpret_cast<float2*>(parts.note + n);
    e = launch_dep(k_attn_few<T, BITS, DP, NR>, dim3(static_cast<unsigned>(n)), dim3(kThreads), K::kSmem, s, a, parts);
    if (e != cudaSuccess) return e;
    return launch_dep(k_attn_join<T, DP, K::kM>, dim3(static_cast<unsigned>(n), static_cast<unsigned>(std::min(K::kM, rows))),
                      dim3(kJoinThreads), 0, s, a, parts);
  }
};
template <typename T, int BITS, int DP, int NR>
std::atomic<size_t> Few<T, BITS, DP, NR>::raised[kMaxDevices];
template <typename T, int BITS, int DP, int NR>
std::atomic<int> Few<T, BITS, DP, NR>::resident{0};

// `rows`: the most rows a sequence brings to a KV head. Tiles of 8, 16 or 32: the smallest
// that takes them at once (256 columns: 16 at most, by registers).
template <typename F>
auto with_few(int bits, bool bf16, int head_dim, int rows, F&& f) {
  auto tile = [&](auto t, auto b, auto d) {
    using Tt = decltype(t);
    constexpr int kB = decltype(b)::value, kD = decltype(d)::value;
    if (rows <= 8) return f(Few<Tt, kB, kD, 1>());
    if constexpr (kD < 256) {
      if (rows > 16) return f(Few<Tt, kB, kD, 4>());
    }
    return f(Few<Tt, kB, kD, 2>());
  };
  auto dim = [&](auto t, auto b) {
    if (head_dim <= 64) return tile(t, b, std::integral_constant<int, 64>());
    if (head_dim <= 128) return tile(t, b, std::integral_constant<int, 128>());
    return tile(t, b, std::integral_constant<int, 256>());
  };
  auto form = [&](auto t) {
    if (bits == 16) return dim(t, std::integral_constant<int, 16>());
    if (bits == 8) return dim(t, std::integral_constant<int, 8>());
    return dim(t, std::integral_constant<int, 4>());
  };
  return bf16 ? form(__nv_bfloat16()) : form(__half());
}

int most_rows(const AttnArgs& a, int max_q_len) {
  return static_cast<int>(std::min<int64_t>(static_cast<int64_t>(max_q_len) * a.group, 1 << 20));
}

// More rows a KV head than this go to the tensor-memory kernel. Above 128 columns its
// loaders' unpacking serves 128 rows only, so that codes take more rows to pay (16
// sequences of 3,000, 36 rows a KV head x 256: 16 bits 68 us there against 141 here, 8 bits
// 161 against 133).
bool takes_many(const AttnArgs& a, int bits, int max_q_len) {
  return most_rows(a, max_q_len) > (bits != 16 && a.kv.head_dim > 128 ? 64 : 32);
}

}  // namespace

size_t attention_workspace(const AttnArgs& a, int bits, bool bf16, int max_q_len, int max_kv_len) {
  if (takes_many(a, bits, max_q_len)) return many_workspace(a, bits, bf16, max_q_len, max_kv_len);
  return with_few(bits, bf16, a.kv.head_dim, most_rows(a, max_q_len), [&](auto k) { return decltype(k)::workspace(); });
}

cudaError_t launch_attention(const AttnArgs& a, int bits, bool bf16, int max_q_len, int max_kv_len, void* workspace,
                             cudaStream_t s) {
  if (takes_many(a, bits, max_q_len)) return launch_many(a, bits, bf16, max_q_len, max_kv_len, workspace, s);
  const int rows = most_rows(a, max_q_len);
  return with_few(bits, bf16, a.kv.head_dim, rows, [&](auto k) { return decltype(k)::launch(a, rows, workspace, s); });
}

}  // namespace gemq
