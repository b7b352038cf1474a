// Attention of a chunk of new tokens over a paged KV cache, many rows a KV head: a
// prompt's chunk, where the products are the time. The mathematics is kernels_attn.cu's.
//
// One block takes 256 rows (tokens x query heads that share a KV head) as two tiles of
// 128, each a chain of its own, over all the keys they see (or one of several spans of
// them), 128 at a time:
//   S = Q K^T   tcgen05.mma, Q and K from shared memory, S fp32 in tensor memory
//   P = 2^(S - ref) in 16 bits, back into S's columns
//   O += P V    tcgen05.mma, P from tensor memory, V from shared memory as it is stored
//               ([key][column]: the N-major form of the B operand)
// 512 columns of tensor memory hold both chains (2 x 128 for S and P, 2 x up to 128 for
// O); while one chain's threads take exponentials the tensor cores work for the other.
// Warps: 0-3 and 4-7 the two chains' softmax (a thread a row, the row's 128 scores in its
// registers: these warps take 184 each and the others 72), 8 and 9 their MMA issue (a
// chain's next S overwrites P, so each waits for its own last product; the other warp's go
// on meanwhile), 12-15 load: 16-bit rows by cp.async, codes by way of registers, unpacked
// to exact fp16 as they are stored. Pages may have any size: a row's address is looked up
// per key, a tile ahead.
//
// The reference of the exponentials moves only when a row's scores pass it by more than
// 2^8 (in 16 bits 2^8 is as exact as 1), so that the sums in tensor memory are rarely
// touched between products.
//
// Where few tiles there are to fill the machine, each takes part of the keys and
// k_attn_tiles adds the parts up; with at most 128 rows a KV head both chains take the
// same rows and every second tile of keys each.
#define GEMQ_OWN_ERROR_WORDS  // compiled without relocatable device code, for setmaxnreg
#include <algorithm>

#include "attn_rows.cuh"
#include "paged.cuh"

namespace gemq {

namespace {

constexpr int kKeys = 128;        // of a tile
constexpr int kRows = 128;        // of a chain
constexpr int kSoftWarps = 8;
constexpr int kMmaWarp = 8;       // and 9
constexpr int kLoadWarp = 12;
constexpr int kLoaders = 128;
constexpr int kThreads = 32 * (kLoadWarp + 4);
// Registers after the split: 256 x 184 + 256 x 72 = 512 x 128, what the block starts with.
constexpr int kSoftRegs = 184, kOtherRegs = 72;
static_assert(256 * (kSoftRegs + kOtherRegs) <= kThreads * 128, "more registers than the block was launched with");
constexpr float kSlack = 8.f;     // how far a score may pass the reference, in powers of two

template <typename T, int BITS, int DP>
struct Tc {
  static constexpr int kPanels = DP / 64;          // of 64 columns (128 bytes) each
  static constexpr int kPanel = kKeys * 128;       // bytes
  static constexpr int kTile = kPanels * kPanel;   // Q tile, K tile, V tile
  static constexpr int kStages = 4;                // K and V in turn
  static constexpr int kQOff = 0;
  static constexpr int kRingOff = 2 * kTile;
  static constexpr int kOffOff = kRingOff + kStages * kTile;    // int64 row offsets, two tiles
  static constexpr int kPrepOff = kOffOff + 2 * kKeys * 8;      // per key factors, two tiles
  static constexpr int kPrepTile = BITS == 16 ? 0 : 5 * kKeys * 4;
  static constexpr int kBarOff = kPrepOff + 2 * kPrepTile;
  static constexpr int kBars = 2 * kStages + 14;
  static constexpr int kSmem = kBarOff + kBars * 8 + 64 + 1024;  // + alignment
  static_assert(kSmem <= 227 * 1024, "shared memory");
  using C = std::conditional_t<BITS == 16, T, __half>;
  static constexpr bool kRowFactor = BITS != 16 && std::is_same_v<T, __nv_bfloat16>;
  static constexpr uint32_t kType = std::is_same_v<C, __nv_bfloat16> ? 1u : 0u;
  // two chains: S (and P) in columns 0 and 128, O in 256 and 256 + DP
  static constexpr int kCols = 512;
};

// Instruction descriptor: A and B of one 16-bit type, fp32 sums, M = 128; `v`: B is
// N-major.
__device__ __forceinline__ uint32_t idesc(uint32_t type, int n, bool v) {
  return 1u << 4 | type << 7 | type << 10 | (v ? 1u << 16 : 0u) | static_cast<uint32_t>(n >> 3) << 17 | (128u >> 4) << 24;
}
// V as B: 64-column panels kKeys * 128 bytes apart (leading), 8 keys 1024 bytes (stride),
// 128-byte swizzle.
__device__ __forceinline__ uint64_t sdesc_v(uint32_t saddr, uint32_t panel) {
  uint64_t d = static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4);
  d |= static_cast<uint64_t>(panel >> 4) << 16;
  d |= static_cast<uint64_t>(1024u >> 4) << 32;
  d |= static_cast<uint64_t>(1u) << 46;
  d |= static_cast<uint64_t>(2u) << 61;
  return d;
}

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <int N>
__device__ __forceinline__ void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// Pairs of fp32.
struct F2 {
  uint64_t v;
};
__device__ __forceinline__ F2 f2(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void split(F2 x, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x.v)); }
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}

// The eight K = 16 steps of O += P V, issued from one asm block (their operands are then
// formed back to back): P 8 columns a step, V 16 keys of 128 bytes.
__device__ __forceinline__ void umma_pv(uint32_t d, uint32_t p, uint64_t v, uint32_t id, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      ".reg .b32 a1, a2, a3, a4, a5, a6, a7;\n\t"
      ".reg .b64 b1, b2, b3, b4, b5, b6, b7;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.eq.u32 q, 0, 0;\n\t"
      "add.u32 a1, %1, 8;\n\tadd.u32 a2, %1, 16;\n\tadd.u32 a3, %1, 24;\n\tadd.u32 a4, %1, 32;\n\t"
      "add.u32 a5, %1, 40;\n\tadd.u32 a6, %1, 48;\n\tadd.u32 a7, %1, 56;\n\t"
      "add.u64 b1, %2, 128;\n\tadd.u64 b2, %2, 256;\n\tadd.u64 b3, %2, 384;\n\tadd.u64 b4, %2, 512;\n\t"
      "add.u64 b5, %2, 640;\n\tadd.u64 b6, %2, 768;\n\tadd.u64 b7, %2, 896;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [a1], b1, %3, q;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [a2], b2, %3, q;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [a3], b3, %3, q;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [a4], b4, %3, q;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [a5], b5, %3, q;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [a6], b6, %3, q;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [a7], b7, %3, q;\n\t}" ::"r"(d),
      "r"(p), "l"(v), "r"(id), "r"(accumulate)
      : "memory");
}

// One arrival for a warp whose lanes have done their part.
__device__ __forceinline__ void warp_arrive(uint64_t* bar) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}

// Codes minus their middle as fp16 pairs, exactly (a code under the exponent of 1024, or
// of 64 four bits up, reads as that plus the code).
__device__ __forceinline__ uint32_t less(uint32_t pair, uint32_t off) {
  return h2_as_u32(__hsub2(u32_as_h2(pair), u32_as_h2(off)));
}
__device__ __forceinline__ void unpack8(uint32_t w, uint32_t (&o)[2]) {  // four codes in order
  const uint32_t x = w ^ 0x80808080u;
  o[0] = less(__byte_perm(x, 0x64646464u, 0x4140), 0x64806480u);
  o[1] = less(__byte_perm(x, 0x64646464u, 0x4342), 0x64806480u);
}
__device__ __forceinline__ void unpack4(uint32_t w, uint32_t (&o)[4]) {  // eight: (0, 4), (1, 5), (2, 6), (3, 7)
  o[0] = less((w & 0x000f000fu) | 0x64006400u, 0x64086408u);
  o[1] = less((w & 0x00f000f0u) | 0x54005400u, 0x54805480u);
  o[2] = less(((w >> 8) & 0x000f000fu) | 0x64006400u, 0x64086408u);
  o[3] = less(((w >> 8) & 0x00f000f0u) | 0x54005400u, 0x54805480u);
}
// Which element of its eight stands at place p of a 4-bit row's columns.
__host__ __device__ constexpr int place4(int p) { return (p >> 1) + 4 * (p & 1); }

struct TileNote {
  int start, row0, rows, head, seq;
  int odd;  // a value that is no number lay in a tile that not every row sees whole
};

struct TileArgs {
  TileNote* note;  // [tiles][kv_heads][spans]
  float* o;        // [tiles][kv_heads][parts][tile rows][DP], with parts only
  float2* ml;      // [tiles][kv_heads][parts][tile rows]
  int spans;       // key spans of a tile
  int parts;       // 0: rows are written whole; else parts of a row (spans, or 2 spans)
  int tile_rows;   // 256; 128 where both chains take the same rows
};

template <typename T, int BITS, int DP>
__global__ void __launch_bounds__(kThreads, 1) k_attn_many(const AttnArgs a, const TileArgs ta) {
  using K = Tc<T, BITS, DP>;
  using C = typename K::C;
  constexpr int kStages = K::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* const smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  int64_t* const s_off = reinterpret_cast<int64_t*>(smem + K::kOffOff);
  float* const s_prep = reinterpret_cast<float*>(smem + K::kPrepOff);
  uint64_t* const bars = reinterpret_cast<uint64_t*>(smem + K::kBarOff);
  uint64_t* const full = bars;                  // [stages] rows landed
  uint64_t* const empty = bars + kStages;       // [stages] products done with them
  uint64_t* const s_full = bars + 2 * kStages;  // [2] S written
  uint64_t* const p_full = s_full + 2;          // [2] P written (and O moved, where it was)
  uint64_t* const o_done = s_full + 4;          // [2] P V done
  uint64_t* const prep_full = s_full + 6;       // [2]
  uint64_t* const prep_empty = s_full + 8;      // [2]
  uint64_t* const offs_full = s_full + 10;      // [2] row offsets written
  uint64_t* const drain = s_full + 12;          // [2]
  uint32_t* const s_tmem = reinterpret_cast<uint32_t*>(bars + K::kBars);
  int* const s_odd = reinterpret_cast<int*>(s_tmem + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int D = a.kv.head_dim;
  const bool same_rows = ta.tile_rows == kRows;

  if (warp == kMmaWarp) {
    tmem_alloc(s_tmem, K::kCols);
    tmem_relinquish();
  }
  grid_dep_wait();

  // ------------------------------------------------------------ this block's rows and keys
  // Tiles in descending order of their position: of a causal sequence's tiles the last
  // ones are the longest, and the short ones fill the machine's end.
  const int span = static_cast<int>(blockIdx.x) % ta.spans;
  const int h = static_cast<int>(blockIdx.x) / ta.spans % a.kv.kv_heads;
  const int tile_back = static_cast<int>(blockIdx.x) / ta.spans / a.kv.kv_heads;
  auto tiles_of = [&](int b) { return (seq_range(a, b).q_len * a.group + ta.tile_rows - 1) / ta.tile_rows; };
  int total = 0;
  for (int b = lane; b < a.num_seqs; b += 32) total += tiles_of(b);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  const int tile = total - 1 - tile_back;
  bool work = tile >= 0;
  int b = 0, first_tile = 0;
  if (work) {
    int base = 0;
    for (int b0 = 0; b0 < a.num_seqs; b0 += 32) {
      const int n = b0 + lane < a.num_seqs ? tiles_of(b0 + lane) : 0;
      int incl = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int w = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += w;
      }
      incl += base;
      const uint32_t past = __ballot_sync(0xffffffffu, incl > tile);
      if (past != 0) {
        const int src = __ffs(past) - 1;
        b = b0 + src;
        first_tile = __shfl_sync(0xffffffffu, incl - n, src);
        break;
      }
      base = __shfl_sync(0xffffffffu, incl, 31);
    }
  }
  const SeqRange r = work ? seq_range(a, b) : SeqRange{0, 0, 0};
  const int row0 = (tile - first_tile) * ta.tile_rows;
  const int rows = work ? min(ta.tile_rows, r.q_len * a.group - row0) : 0;
  const int pos0 = r.kv_len - r.q_len;
  const int tile_min = pos0 + row0 / a.group;
  const int tile_max = pos0 + (row0 + max(rows, 1) - 1) / a.group;
  // key tiles [k0, k1) of this span, the first key of key tile 0 is 0
  int k0 = 0, k1 = 0;
  if (work) {
    const int lo = a.window > 0 ? max(0, tile_min - a.window + 1) : 0;
    const int t0 = lo / kKeys, n = max(0, (tile_max + 1 + kKeys - 1) / kKeys - t0);
    k0 = t0 + static_cast<int>(static_cast<int64_t>(n) * span / ta.spans);
    k1 = t0 + static_cast<int>(static_cast<int64_t>(n) * (span + 1) / ta.spans);
  }
  const int n_tiles = k1 - k0;
  const float cs = fabsf(a.scale) * kLog2e;

  // which tiles chain i takes: all, or every second one
  const int step = same_rows ? 2 : 1;
  auto chain_first = [&](int i) { return same_rows ? i : 0; };
  // a chain without rows is left out
  const bool chain_b = same_rows || rows > kRows;

  if (threadIdx.x == 0) {
    const int chains = chain_b && !same_rows ? 2 : 1;  // that take each tile
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 4);  // one arrival a warp
      mbar_init(&empty[s], chains);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&o_done[i], 1);
      mbar_init(&prep_full[i], 4);
      mbar_init(&prep_empty[i], 4 * chains);  // softmax warps
      mbar_init(&offs_full[i], 4);
      mbar_init(&drain[i], 1);
    }
    fence_barrier_init();
    *s_odd = 0;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *s_tmem;
  // ------------------------------------------------------------ queries, by the row's thread
  const int chain = warp >> 2;  // of a softmax warp
  const int tid = static_cast<int>(threadIdx.x) & 127;
  const int my_row = (same_rows ? 0 : chain * kRows) + tid;  // in the block's rows
  float rf = 1.f, qsum = 0.f;
  int last = -1, from = 0;
  if (warp < kSoftWarps) {
    const bool in = my_row < rows;
    const int tok = (row0 + my_row) / a.group, hh = (row0 + my_row) % a.group;
    if (in) {
      last = pos0 + tok;
      from = a.window > 0 ? max(0, last - a.window + 1) : 0;
    }
    const T* q = static_cast<const T*>(a.q) +
                 (in ? (r.start + tok) * a.q_token_stride + static_cast<int64_t>(h * a.group + hh) * D : 0);
    float inv_factor = 1.f;
    if constexpr (K::kRowFactor) {
      // bf16 queries against fp16 codes: the row scaled by a power of two to at most 2
      float most = 0.f;
      for (int c = 0; in && c < D / 8; ++c) {
        const uint4 w = *reinterpret_cast<const uint4*>(q + 8 * c);
        const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 f = unpack2<T>(ws[e]);
          most = fmaxf(most, fmaxf(fabsf(f.x), fabsf(f.y)));
        }
      }
      const int e = most > 0.f && most < INFINITY ? min(max(ilogbf(most), -100), 100) : 0;
      rf = exp2f(static_cast<float>(e));
      inv_factor = 1.f / rf;
    }
    uint8_t* const dst = smem + K::kQOff + chain * K::kTile + tid * 128;
#pragma unroll 4
    for (int c = 0; c < D / 8; ++c) {
      uint4 w = make_uint4(0u, 0u, 0u, 0u);
      if (in) w = *reinterpret_cast<const uint4*>(q + 8 * c);
      if constexpr (BITS == 4)
        w = make_uint4(__byte_perm(w.x, w.z, 0x5410), __byte_perm(w.x, w.z, 0x7632), __byte_perm(w.y, w.w, 0x5410),
                       __byte_perm(w.y, w.w, 0x7632));
      if constexpr (K::kRowFactor) {
        uint32_t* ws = &w.x;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 f = unpack2<T>(ws[e]);
          ws[e] = pack2<__half>(f.x * inv_factor, f.y * inv_factor);
        }
      }
      if (a.scale < 0.f) {  // (the scores' factor is its magnitude)
        w.x ^= 0x80008000u;
        w.y ^= 0x80008000u;
        w.z ^= 0x80008000u;
        w.w ^= 0x80008000u;
      }
      if constexpr (BITS == 4) {
        const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 f = __half22float2(u32_as_h2(ws[e]));
          qsum += f.x + f.y;
        }
      }
      *reinterpret_cast<uint4*>(dst + (c >> 3) * K::kPanel + (((c & 7) ^ (tid & 7)) << 4)) = w;
    }
    fence_proxy_async_smem();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();

  bool ok = true;  // no wait of this thread ran out
  if (warp >= kLoadWarp) {
    regs_down<kOtherRegs>();
    // ---------------------------------------------------------- loads
    const int me = static_cast<int>(threadIdx.x) - kLoadWarp * 32;
    const int mask = (1 << a.kv.page_shift) - 1;
    const int row_bytes = D * BITS / 8;
    constexpr int kChunks = DP * BITS / 128;     // 16-byte pieces of a stored row
    constexpr int kRowsIt = kLoaders / kChunks;  // rows of one step of the loaders
    constexpr int kIts = kKeys / kRowsIt;
    const int32_t* const table = a.page_table + b * a.page_table_stride;
    auto page_at = [&](int t) {
      const int j = (k0 + t) * kKeys + me;
      return t < n_tiles && j < r.kv_len ? __ldg(table + (j >> a.kv.page_shift)) : -1;
    };
    int next_page = page_at(0);
    // tile t, K then V: stage 2 t + v of the ring
    const int c = me % kChunks, crow = me / kChunks;
    const bool wide = BITS != 4 || row_bytes % 16 == 0;
    int done = 0;  // stages whose rows this thread has handed over
    bool odd = false;
    auto hand_over = [&]() {  // 16 bits: the oldest stage's copies of this thread have landed
      const int s = done % kStages;
      if (done & 1) {
        // a value tile: look for what is no number where not every row sees every key
        const int j0 = (k0 + done / 2) * kKeys;
        if (j0 + kKeys - 1 > tile_min || (a.window > 0 && j0 <= tile_max - a.window)) {
          if (c * 16 < row_bytes) {
            for (int it = 0; it < kIts; ++it) {
              const int row = it * kRowsIt + crow;
              const uint4 w = *reinterpret_cast<const uint4*>(smem + K::kRingOff + s * K::kTile + (c >> 3) * K::kPanel +
                                                              row * 128 + (((c & 7) ^ (row & 7)) << 4));
              const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float2 f = unpack2<T>(ws[e]);
                odd |= !isfinite(f.x) || !isfinite(f.y);
              }
            }
          }
        }
      }
      fence_proxy_async_smem();
      warp_arrive(&full[s]);
      ++done;
    };
    for (int t = 0; t < n_tiles && ok; ++t) {
      // where the tile's rows lie, one a loader
      const int j = (k0 + t) * kKeys + me;
      int64_t off = -1, soff = 0;
      if (j < r.kv_len) {
        const int page = next_page;
        if (page >= 0 && page < a.kv.num_pages) {
          off = a.kv.row(page, h, j & mask);
          if constexpr (BITS != 16) soff = a.kv.scale_row(page, h, j & mask);
        } else {
          set_device_error(kDevBadCachePos);
        }
      }
      next_page = page_at(t + 1);
      int64_t* const offs = s_off + (t & 1) * kKeys;
      offs[me] = off;
      float2 ksc = make_float2(0.f, 0.f), vsc = ksc;
      if constexpr (BITS != 16) {
        if (off >= 0) {
          if constexpr (BITS == 8) {
            ksc.x = __ldg(a.kv.k_scale + soff);
            vsc.x = __ldg(a.kv.v_scale + soff);
          } else {
            ksc = __ldg(reinterpret_cast<const float2*>(a.kv.k_scale + soff));
            vsc = __ldg(reinterpret_cast<const float2*>(a.kv.v_scale + soff));
          }
        }
      }
      warp_arrive(&offs_full[t & 1]);
      ok = warp_wait(&offs_full[t & 1], (t >> 1) & 1, kDevTimeoutAFull);
#pragma unroll 1
      for (int v = 0; v < 2 && ok; ++v) {
        const int g = 2 * t + v, s = g % kStages;
        const uint8_t* const src = v ? a.kv.v : a.kv.k;
        uint8_t* const dst = smem + K::kRingOff + s * K::kTile;
        uint4 raw[BITS == 16 ? 1 : kIts];
        if constexpr (BITS != 16) {
          // codes first: their way from memory overlaps the wait
#pragma unroll
          for (int it = 0; it < kIts; ++it) {
            const int64_t ro = offs[it * kRowsIt + crow];
            raw[it] = make_uint4(0u, 0u, 0u, 0u);
            if (ro >= 0 && c * 16 < row_bytes) {
              if (wide) {
                raw[it] = __ldg(reinterpret_cast<const uint4*>(src + ro + c * 16));
              } else {
                const uint2 x = __ldg(reinterpret_cast<const uint2*>(src + ro + c * 16));
                raw[it].x = x.x;
                raw[it].y = x.y;
                if (c * 16 + 8 < row_bytes) {
                  const uint2 y = __ldg(reinterpret_cast<const uint2*>(src + ro + c * 16 + 8));
                  raw[it].z = y.x;
                  raw[it].w = y.y;
                }
              }
            }
          }
        }
        if (!__all_sync(0xffffffffu, mbar_try_wait(smem_u32(&empty[s]), ((g / kStages) & 1) ^ 1u))) {
          if constexpr (BITS == 16) {
            // nothing to issue: hand over what is on its way
            if (done < g) {
              cp_wait<0>();
              hand_over();
            }
          }
          ok = warp_wait(&empty[s], ((g / kStages) & 1) ^ 1u, kDevTimeoutAEmpty);
          if (!ok) break;
        }
        if constexpr (BITS == 16) {
          if (c * 16 < row_bytes) {
#pragma unroll
            for (int it = 0; it < kIts; ++it) {
              const int row = it * kRowsIt + crow;
              const int64_t ro = offs[row];
              cp16(smem_u32(dst + (c >> 3) * K::kPanel + row * 128 + (((c & 7) ^ (row & 7)) << 4)),
                   src + (ro < 0 ? 0 : ro + c * 16), ro < 0 ? 0u : 16u);
            }
          }
          cp_commit();
          if (done < g) {
            cp_wait<1>();
            hand_over();
          }
        } else {
          if (v == 0) {
            // the key's factors: a = s c, log2 t, 1 / t, z c, y / t, with c = scale log2(e)
            ok = warp_wait(&prep_empty[t & 1], ((t >> 1) & 1) ^ 1u, kDevTimeoutAEmpty);
            if (!ok) break;
            float* const prep = s_prep + (t & 1) * 5 * kKeys;
            const float vstep = vsc.x < kMinScale ? kMinScale : vsc.x;  // a step of zero; a NaN stays
            const float lv = lg2(vstep), inv = ex2(-lv);
            prep[me] = ksc.x * cs;
            prep[kKeys + me] = lv;
            // a row that sees a poisoned key has a NaN weight; one that does not has weight
            // zero, which must meet a number here
            prep[2 * kKeys + me] = inv < INFINITY ? inv : 0.f;
            if constexpr (BITS == 4) {
              const float zr = fmaf(8.f, vsc.x, vsc.y) / vstep;
              prep[3 * kKeys + me] = fmaf(8.f, ksc.x, ksc.y) * cs;
              prep[4 * kKeys + me] = fabsf(zr) < INFINITY ? zr : 0.f;
            }
            warp_arrive(&prep_full[t & 1]);
          }
          if (c * 16 < row_bytes) {
#pragma unroll
            for (int it = 0; it < kIts; ++it) {
              const int row = it * kRowsIt + crow;
              const uint32_t ws[4] = {raw[it].x, raw[it].y, raw[it].z, raw[it].w};
              constexpr int kOut = 16 / BITS;  // 16-byte pieces that a piece of codes becomes
#pragma unroll
              for (int o = 0; o < kOut; ++o) {
                uint4 w;
                if constexpr (BITS == 8) {
                  uint32_t x[2], y[2];
                  unpack8(ws[2 * o], x);
                  unpack8(ws[2 * o + 1], y);
                  w = make_uint4(x[0], x[1], y[0], y[1]);
                } else {
                  uint32_t x[4];
                  unpack4(ws[o], x);
                  w = make_uint4(x[0], x[1], x[2], x[3]);
                }
                const int cc = c * kOut + o;
                *reinterpret_cast<uint4*>(dst + (cc >> 3) * K::kPanel + row * 128 + (((cc & 7) ^ (row & 7)) << 4)) = w;
              }
            }
          }
          fence_proxy_async_smem();
          warp_arrive(&full[s]);
        }
      }
    }
    if constexpr (BITS == 16) {
      cp_wait<0>();
      if (ok && done < 2 * n_tiles) hand_over();
      if (odd) *s_odd = 1;
    }
  } else if (warp >= kMmaWarp) {
    // ---------------------------------------------------------- products of one chain
    regs_down<kOtherRegs>();
    const int i = warp - kMmaWarp;
    if (i == 0 || (i == 1 && chain_b)) {
      const uint32_t s_col = tmem + i * 128, o_col = tmem + 256 + i * DP;
      const uint32_t id_s = idesc(K::kType, kKeys, false), id_o = idesc(K::kType, D, true);
      const uint32_t q_addr = smem_u32(smem + K::kQOff + i * K::kTile);
      const int ks = D / 16;
      int n = 0;  // tiles of this chain so far
      for (int t = chain_first(i); t < n_tiles && ok; t += step, ++n) {
        const int gk = 2 * t, gv = gk + 1;
        ok = warp_wait(&full[gk % kStages], (gk / kStages) & 1, kDevTimeoutAFull);
        // S overwrites P: the last product with it must have ended
        if (ok && n > 0) ok = warp_wait(&o_done[i], (n - 1) & 1, kDevTimeoutAccFull);
        if (!ok) break;
        tc_fence_after();
        const uint32_t k_addr = smem_u32(smem + K::kRingOff + (gk % kStages) * K::kTile);
        if (elect_one()) {
          int k = 0;
          for (; k + 4 <= ks; k += 4)
            umma_f16_k64(s_col, sdesc_sw128(q_addr + (k >> 2) * K::kPanel), sdesc_sw128(k_addr + (k >> 2) * K::kPanel), id_s, k > 0);
          for (; k < ks; ++k) {
            const uint32_t at = (k >> 2) * K::kPanel + (k & 3) * 32;
            umma_f16(s_col, sdesc_sw128(q_addr + at), sdesc_sw128(k_addr + at), id_s, k > 0);
          }
          umma_commit(&s_full[i]);
          umma_commit(&empty[gk % kStages]);
        }
        __syncwarp();
        ok = warp_wait(&full[gv % kStages], (gv / kStages) & 1, kDevTimeoutAFull) &&
             warp_wait(&p_full[i], n & 1, kDevTimeoutAccEmpty);
        if (!ok) break;
        tc_fence_after();
        const uint32_t v_addr = smem_u32(smem + K::kRingOff + (gv % kStages) * K::kTile);
        if (elect_one()) {
          umma_pv(o_col, s_col, sdesc_v(v_addr, K::kPanel), id_o, n > 0);
          umma_commit(&o_done[i]);
          umma_commit(&empty[gv % kStages]);
        }
        __syncwarp();
      }
      if (elect_one()) umma_commit(&drain[i]);
      __syncwarp();
      mbar_wait_drain(&drain[i], 0);
    }
  } else {
    regs_up<kSoftRegs>();
    if (chain == 0 || chain_b) {
    // ---------------------------------------------------------- softmax: a thread a row
    const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;  // 32 lanes a warp
    const uint32_t s_col = tmem + lanes + chain * 128, o_col = tmem + lanes + 256 + chain * DP;
    // positions of this warp's first and last row
    const int w_row = my_row - lane;
    const int w_min = pos0 + (row0 + w_row) / a.group;
    const int w_max = pos0 + (row0 + min(w_row + 31, max(rows, 1) - 1)) / a.group;
    float ref = -INFINITY, l = 0.f, zacc = 0.f;
    int n = 0;
    for (int t = chain_first(chain); t < n_tiles && ok; t += step, ++n) {
      const int j0 = (k0 + t) * kKeys;
      const bool whole = j0 + kKeys - 1 <= w_min && (a.window <= 0 || j0 > w_max - a.window);
      const float* const prep = s_prep + (t & 1) * 5 * kKeys;
      if constexpr (BITS != 16) ok = warp_wait(&prep_full[t & 1], (t >> 1) & 1, kDevTimeoutAFull);
      ok = ok && warp_wait(&s_full[chain], n & 1, kDevTimeoutAccFull);
      if (!ok) break;
      tc_fence_after();
      uint32_t s[kKeys];
#pragma unroll
      for (int c = 0; c < kKeys / 32; ++c) tmem_ld32(s_col + 32 * c, reinterpret_cast<uint32_t(&)[32]>(s[32 * c]));
      tmem_ld_wait();
      auto sf = [&](int j) { return __uint_as_float(s[j]); };
      if constexpr (BITS != 16) {
        // scores of codes, with the values' steps in them
        const F2 qs2 = f2(qsum, qsum), rf2 = f2(rf, rf);
#pragma unroll
        for (int j = 0; j < kKeys; j += 4) {
          const float4 aj = *reinterpret_cast<const float4*>(prep + j);
          const float4 lv = *reinterpret_cast<const float4*>(prep + kKeys + j);
          float4 zj = make_float4(0.f, 0.f, 0.f, 0.f);
          if constexpr (BITS == 4) zj = *reinterpret_cast<const float4*>(prep + 3 * kKeys + j);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const F2 a2 = e ? f2(aj.z, aj.w) : f2(aj.x, aj.y), l2 = e ? f2(lv.z, lv.w) : f2(lv.x, lv.y);
            const F2 z2 = e ? f2(zj.z, zj.w) : f2(zj.x, zj.y), s2 = f2(sf(j + 2 * e), sf(j + 2 * e + 1));
            F2 x;
            if constexpr (K::kRowFactor) x = fma2(BITS == 4 ? fma2(s2, a2, mul2(qs2, z2)) : mul2(s2, a2), rf2, l2);
            else x = fma2(s2, a2, BITS == 4 ? fma2(qs2, z2, l2) : l2);
            float x0, x1;
            split(x, x0, x1);
            s[j + 2 * e] = __float_as_uint(x0);
            s[j + 2 * e + 1] = __float_as_uint(x1);
          }
        }
      }
      if (!whole) {
#pragma unroll
        for (int j = 0; j < kKeys; ++j)
          if (j0 + j > last || j0 + j < from) s[j] = 0xff800000u;  // -inf
      }
      float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int j = 0; j < kKeys; j += 8)
#pragma unroll
        for (int e = 0; e < 4; ++e) tops[e] = fmaxf(fmaxf(tops[e], sf(j + 2 * e)), sf(j + 2 * e + 1));
      // (cs is not negative: the queries carry its sign)
      const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])) * (BITS == 16 ? cs : 1.f);
      // a row whose reference is not set yet, or is left behind, takes its maximum
      const bool behind = ref == -INFINITY ? top > -INFINITY : top > ref + kSlack;
      if (__any_sync(0xffffffffu, behind)) {
        const float now = behind ? top : ref;
        const float keep = now == -INFINITY ? 1.f : ex2(ref - now);  // ref = -inf: 0
        l *= keep;
        zacc *= keep;
        ref = now;
        if (n > 0) {
          ok = warp_wait(&o_done[chain], (n - 1) & 1, kDevTimeoutAccFull);
          if (!ok) break;
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < D; c += 16) {
            uint32_t o[16];
            tmem_ld16(o_col + c, o);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
            tmem_st16(o_col + c, o);
          }
        }
      }
      const float base = ref == -INFINITY ? 0.f : ref;
      const F2 base2 = f2(-base, -base), cs2 = f2(cs, cs);
      F2 lt[2] = {f2(l, 0.f), f2(0.f, 0.f)}, zt = f2(zacc, 0.f);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t p[32];
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
          const int j = 64 * half + 2 * i;
          float4 iv, zr;
          if constexpr (BITS != 16) iv = *reinterpret_cast<const float4*>(prep + 2 * kKeys + j);
          if constexpr (BITS == 4) zr = *reinterpret_cast<const float4*>(prep + 4 * kKeys + j);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const F2 s2 = f2(sf(j + 2 * e), sf(j + 2 * e + 1));
            float y0, y1;
            split(BITS == 16 ? fma2(s2, cs2, base2) : add2(s2, base2), y0, y1);
            const float w0 = ex2(y0), w1 = ex2(y1);
            p[i + e] = pack2<C>(w0, w1);
            if constexpr (BITS == 16) {
              lt[e] = add2(lt[e], f2(w0, w1));
            } else {
              lt[e] = fma2(f2(w0, w1), e ? f2(iv.z, iv.w) : f2(iv.x, iv.y), lt[e]);
              if constexpr (BITS == 4) {
                // the rounded weights, so that their rounding scales with the value and
                // not with the code's distance from 8
                const float2 f = unpack2<C>(p[i + e]);
                zt = fma2(f2(f.x, f.y), e ? f2(zr.z, zr.w) : f2(zr.x, zr.y), zt);
              }
            }
          }
        }
        tmem_st32(s_col + 32 * half, p);
      }
      {
        float x0, x1, y0, y1;
        split(lt[0], x0, x1);
        split(lt[1], y0, y1);
        l = (x0 + x1) + (y0 + y1);
        split(zt, x0, x1);
        zacc = x0 + x1;
      }
      if constexpr (BITS != 16) warp_arrive(&prep_empty[t & 1]);
      tmem_st_wait();
      tc_fence_before();
      warp_arrive(&p_full[chain]);
    }
    // ---------------------------------------------------------- rows out
    if (ok && n > 0) ok = warp_wait(&o_done[chain], (n - 1) & 1, kDevTimeoutAccFull);
    tc_fence_after();
    if (ok && work) {
      const bool in = my_row < rows;
      const int tok = (row0 + my_row) / a.group, hh = (row0 + my_row) % a.group;
      const int64_t at = static_cast<int64_t>(r.start + tok) * a.q_heads + h * a.group + hh;
      const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
      const int part = same_rows ? 2 * span + chain : span;
      const int64_t slot = ((static_cast<int64_t>(tile) * a.kv.kv_heads + h) * max(ta.parts, 1) + part) * ta.tile_rows + my_row;
      if (in && ta.parts > 0) ta.ml[slot] = make_float2(ref, l);
      if (in && ta.parts == 0 && a.lse != nullptr) a.lse[at] = l == 0.f ? -INFINITY : (ref + log2f(l)) * kLn2;
#pragma unroll 1
      for (int c = 0; c < D; c += 16) {
        float x[16];
        if (n > 0) {
          uint32_t o[16];
          tmem_ld16(o_col + c, o);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            // a 4-bit row's columns stand in the order its codes unpack
            const int d = BITS == 4 ? (e & 8) + place4(e & 7) : e;
            x[d] = __uint_as_float(o[e]) + zacc;
          }
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e) x[e] = 0.f;
        }
        if (!in) continue;
        if (ta.parts > 0) {
          float4* const dst = reinterpret_cast<float4*>(ta.o + slot * DP + c);
#pragma unroll
          for (int e = 0; e < 4; ++e) dst[e] = make_float4(x[4 * e], x[4 * e + 1], x[4 * e + 2], x[4 * e + 3]);
        } else {
          uint4* const dst = reinterpret_cast<uint4*>(static_cast<T*>(a.out) + at * D + c);
#pragma unroll
          for (int e = 0; e < 2; ++e)
            dst[e] = make_uint4(pack2<T>(x[8 * e] * inv, x[8 * e + 1] * inv), pack2<T>(x[8 * e + 2] * inv, x[8 * e + 3] * inv),
                                pack2<T>(x[8 * e + 4] * inv, x[8 * e + 5] * inv), pack2<T>(x[8 * e + 6] * inv, x[8 * e + 7] * inv));
        }
      }
    }
  }
  }
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0) {
    const int64_t at = (work ? (static_cast<int64_t>(tile) * a.kv.kv_heads + h) * ta.spans + span : blockIdx.x);
    ta.note[at] = TileNote{r.start, row0, rows, h, b, *s_odd};
  }
  if (warp == kMmaWarp) tmem_dealloc(tmem, K::kCols);
}

// Adds up a tile's parts, eight rows (four of 256 columns) a step; and, where a value that
// is no number met rows that do not see it, takes the tile's rows one by one.
constexpr int kJoinThreads = 128;
template <typename T, int BITS, int DP>
__global__ void __launch_bounds__(kJoinThreads) k_attn_tiles(const AttnArgs a, const TileArgs ta) {
  __shared__ AttnRowSmem sm;
  constexpr int kCols = DP / 4, kGroups = kJoinThreads / kCols;
  grid_dep_wait();
  const int64_t which = blockIdx.x;
  const TileNote note = ta.note[which * ta.spans];
  if (note.rows <= 0) return;
  if constexpr (BITS == 16) {
    bool odd = false;
    for (int s = 0; s < ta.spans; ++s) odd |= ta.note[which * ta.spans + s].odd != 0;
    if (odd) {
      const SeqRange r = seq_range(a, note.seq);
      for (int row = blockIdx.y; row < note.rows; row += gridDim.y)
        attn_one_row<T, BITS>(a, note.seq, r, (note.row0 + row) / a.group, note.head * a.group + (note.row0 + row) % a.group, sm);
      return;
    }
  }
  if (ta.parts == 0) return;
  const int col = threadIdx.x % kCols, grp = threadIdx.x / kCols;
  for (int row = blockIdx.y * kGroups + grp; row < note.rows; row += gridDim.y * kGroups) {
    const int64_t s0 = which * ta.parts * ta.tile_rows + row;
    float top = -INFINITY;
    for (int p = 0; p < ta.parts; ++p) top = fmaxf(top, ta.ml[s0 + static_cast<int64_t>(p) * ta.tile_rows].x);
    const float ref = top == -INFINITY ? 0.f : top;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = 0.f;
#pragma unroll 4
    for (int p = 0; p < ta.parts; ++p) {
      const int64_t s = s0 + static_cast<int64_t>(p) * ta.tile_rows;
      const float2 ml = ta.ml[s];
      const float4 v = *reinterpret_cast<const float4*>(ta.o + s * DP + col * 4);
      const float f = ex2(ml.x - ref);
      l = fmaf(ml.y, f, l);
      acc.x = fmaf(v.x, f, acc.x);
      acc.y = fmaf(v.y, f, acc.y);
      acc.z = fmaf(v.z, f, acc.z);
      acc.w = fmaf(v.w, f, acc.w);
    }
    const int rr = note.row0 + row;
    const int64_t at = static_cast<int64_t>(note.start + rr / a.group) * a.q_heads + note.head * a.group + rr % a.group;
    const float n = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
    if (col * 4 < a.kv.head_dim) {
      uint2 out;
      out.x = pack2<T>(acc.x * n, acc.y * n);
      out.y = pack2<T>(acc.z * n, acc.w * n);
      *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + at * a.kv.head_dim + col * 4) = out;
    }
    if (col == 0 && a.lse != nullptr) a.lse[at] = l == 0.f ? -INFINITY : (top + log2f(l)) * kLn2;
  }
}

// ------------------------------------------------------------------ host
struct Plan {
  int tile_rows, spans, parts;
  int64_t tiles;  // at most
};
Plan plan(const AttnArgs& a, int max_q_len, int max_kv_len) {
  Plan p;
  const int64_t rows = static_cast<int64_t>(a.num_tokens) * a.group;
  p.tile_rows = static_cast<int64_t>(max_q_len) * a.group <= kRows ? kRows : 2 * kRows;
  p.tiles = std::min<int64_t>(rows, rows / p.tile_rows + a.num_seqs);  // a partial one each
  const int64_t blocks = p.tiles * a.kv.kv_heads;
  // spans until the blocks fill the machine, none shorter than four tiles of keys
  const int64_t most = std::max<int64_t>(1, max_kv_len / (4 * kKeys));
  p.spans = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(device_sm_count() / std::max<int64_t>(1, blocks), most)));
  p.parts = p.tile_rows == kRows ? 2 * p.spans : p.spans > 1 ? p.spans : 0;
  return p;
}
size_t round256(size_t v) { return (v + 255) & ~static_cast<size_t>(255); }

template <typename T, int BITS, int DP>
struct Many {
  static std::atomic<size_t> raised[kMaxDevices];
  static size_t workspace(const AttnArgs& a, const Plan& p) {
    const size_t heads = static_cast<size_t>(p.tiles) * a.kv.kv_heads;
    return round256(heads * p.spans * sizeof(TileNote)) +
           heads * p.parts * p.tile_rows * (DP * sizeof(float) + sizeof(float2));
  }
  static cudaError_t launch(const AttnArgs& a, const Plan& p, void* ws, cudaStream_t s) {
    using K = Tc<T, BITS, DP>;
    cudaError_t e = raise_smem_limit(k_attn_many<T, BITS, DP>, K::kSmem, raised);
    if (e != cudaSuccess) return e;
    const size_t heads = static_cast<size_t>(p.tiles) * a.kv.kv_heads;
    TileArgs ta;
    ta.note = static_cast<TileNote*>(ws);
    ta.o = reinterpret_cast<float*>(static_cast<char*>(ws) + round256(heads * p.spans * sizeof(TileNote)));
    ta.ml = reinterpret_cast<float2*>(ta.o + heads * p.parts * p.tile_rows * DP);
    ta.spans = p.spans;
    ta.parts = p.parts;
    ta.tile_rows = p.tile_rows;
    e = launch_dep(k_attn_many<T, BITS, DP>, dim3(static_cast<unsigned>(heads * p.spans)), dim3(kThreads), K::kSmem, s, a, ta);
    if (e != cudaSuccess || (BITS != 16 && p.parts == 0)) return e;
    return launch_dep(k_attn_tiles<T, BITS, DP>, dim3(static_cast<unsigned>(heads), p.parts > 0 ? 32u : 1u), dim3(kJoinThreads), 0,
                      s, a, ta);
  }
};
template <typename T, int BITS, int DP>
std::atomic<size_t> Many<T, BITS, DP>::raised[kMaxDevices];

template <typename F>
auto with_many(int bits, bool bf16, int head_dim, F&& f) {
  auto dim = [&](auto t, auto b) {
    if (head_dim <= 64) return f(Many<decltype(t), decltype(b)::value, 64>());
    return f(Many<decltype(t), decltype(b)::value, 128>());
  };
  auto form = [&](auto t) {
    if (bits == 16) return dim(t, std::integral_constant<int, 16>());
    if (bits == 8) return dim(t, std::integral_constant<int, 8>());
    return dim(t, std::integral_constant<int, 4>());
  };
  return bf16 ? form(__nv_bfloat16()) : form(__half());
}

}  // namespace

cudaError_t take_many_error(uint32_t* code) {
  cudaError_t e = cudaMemcpyFromSymbol(code, g_device_error, sizeof(*code));
  const uint32_t zero = 0;
  if (e == cudaSuccess) e = cudaMemcpyToSymbol(g_device_error, &zero, sizeof(zero));
  if (e == cudaSuccess) e = cudaMemcpyToSymbol(g_device_abort, &zero, sizeof(zero));
  return e;
}

size_t many_workspace(const AttnArgs& a, int bits, bool bf16, int max_q_len, int max_kv_len) {
  const Plan p = plan(a, max_q_len, max_kv_len);
  return with_many(bits, bf16, a.kv.head_dim, [&](auto k) { return decltype(k)::workspace(a, p); });
}
cudaError_t launch_many(const AttnArgs& a, int bits, bool bf16, int max_q_len, int max_kv_len, void* workspace,
                        cudaStream_t s) {
  const Plan p = plan(a, max_q_len, max_kv_len);
  return with_many(bits, bf16, a.kv.head_dim, [&](auto k) { return decltype(k)::launch(a, p, workspace, s); });
}

}  // namespace gemq
