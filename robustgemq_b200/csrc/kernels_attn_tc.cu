// Attention of a chunk of new tokens over a paged KV cache, many rows a KV head: a
// prompt's chunk, where the products are the time. The mathematics is kernels_attn.cu's.
//
// One block takes 256 rows (tokens x query heads that share a KV head) as two tiles of
// 128, each a chain of its own, over all the keys they see (or one of several spans of
// them), 80 at a time (128 with at most 64 columns):
//   S = Q K^T   tcgen05.mma, Q and K from shared memory, S fp32 in tensor memory
//   P = 2^(S - ref) in 16 bits, in tensor memory
//   O += P V    tcgen05.mma, P from tensor memory, V from shared memory as it is stored
//               ([key][column]: the N-major form of the B operand)
// The tile is what lets S, P and O of both chains stand side by side in the 512 columns
// (2 x (80 + 40 + 128)): a chain's next S is formed as soon as its threads have the last
// one in registers, and both products run under the exponentials. (With 128 keys P had to
// overwrite S, and each tile's exponentials waited for two products in a row: 4750 cycles
// a tile with the chains left to themselves, 4250 with the exponentials in turns.)
// Warps: 0-3 and 4-7 the two chains' softmax (a thread a row, the row's scores in its
// registers: these warps take 184 each and the others 72), 8 and 9 their MMA issue, 12-15
// load: 16-bit rows by TMA, codes by way of registers, unpacked to exact fp16 as they are
// stored.
//
// Codes: a key's factors (its step and the value's as a shift, 1 / t; at 4 bits also z and
// y / t) are prepared once by the loaders, and its 256 rows read them from shared memory.
// The value's step shifts the score, as in kernels_attn.cu, so that a row's reference
// follows the largest w_j t_j among the keys that it sees: with one exponent for all keys
// of a block in its place a large step that a row does not see, or gives no weight, pushed
// its own weights out of fp16's range.
//
// The reference of the exponentials moves only when a row's scores pass it by more than
// 2^8 (in 16 bits 2^8 is as exact as 1), so that the sums in tensor memory are rarely
// touched between products.
//
// Row tiles that do not fill a last round of the machine (all of them, where they are few)
// are cut along their keys until they do, and k_attn_tiles adds the parts up; with at most
// 128 rows a KV head both chains take the same rows and every second tile of keys each.
// Above 128 columns the sums of 256 rows would fill tensor memory: both chains take the
// same 128 rows and all keys, 64 at a time, and half of V's columns each. S and P are formed
// twice, so two of six products are repeated, but Q and the keys stand in shared memory
// once, and all else stays as it is. (2,048 tokens at the end of 8,192, 16 query and 4 KV
// heads x 256: 334 us, 720 TFLOP/s, at 16 bits, where 16-row tiles took 3,141; 711 to 759
// and 730 to 745 at 8 and 4 bits, the loaders' unpacking, against 2,810 and 1,683.)
//
// Measured on a B200: 4,096 tokens at the end of 16,384, 32 query and 8 KV heads x 128,
// bf16: 900 us (1,070 TFLOP/s of the visible pairs; 1,030 us in long runs under the power
// limit), with the exponentials' pipe and the tensor cores half used each and 47% of the
// issue slots: two softmax warps a scheduler do not cover each other's waits. At 8 and 4
// bits 2,090 and 2,440 us, the loaders' unpacking and the factors. 12 uneven chunks up to
// 1,000 of 9,000, 24 on 8 heads x 64, window 4,096, 8 bits: 477 us (330 TFLOP/s), issue 42%,
// shared memory 38%, the exponentials' pipe 36% used: the softmax warps' chain of waits,
// factors, maximum and exponentials.
#define GEMQ_OWN_ERROR_WORDS  // compiled without relocatable device code, for setmaxnreg
#include <cudaTypedefs.h>

#include <algorithm>

#include "attn_rows.cuh"
#include "paged.cuh"

namespace gemq {

namespace {

constexpr int kRows = 128;        // of a chain
constexpr int kSoftWarps = 8;
constexpr int kMmaWarp = 8;       // and 9
constexpr int kLoadWarp = 12;
constexpr int kLoaders = 128;
constexpr int kThreads = 32 * (kLoadWarp + 4);
constexpr float kSlack = 8.f;     // how far a score may pass the reference, in powers of two

template <typename T, int BITS, int DP>
struct Tc {
  static constexpr bool kWide = DP == 256;           // each chain half of the columns of V
  static constexpr int kKeys = DP == 64 ? 128 : DP == 128 ? 80 : 64;  // of a tile
  static constexpr int kPanels = DP / 64;            // of 64 columns (128 bytes) each
  static constexpr int kPanel = kKeys * 128;         // bytes
  static constexpr int kTile = kPanels * kPanel;     // K tile, V tile
  static constexpr int kQPanel = kRows * 128;
  static constexpr int kQTile = kPanels * kQPanel;
  static constexpr int kStages = kWide ? 4 : 6;      // K and V in turn
  static constexpr int kQOff = 0;
  static constexpr int kRingOff = (kWide ? 1 : 2) * kQTile;
  static constexpr int kPrepOff = kRingOff + kStages * kTile;   // per key factors, two tiles
  static constexpr int kPrepTile = BITS == 16 ? 0 : (BITS == 8 ? 3 : 5) * kKeys * 4;
  static constexpr int kBarOff = kPrepOff + 2 * kPrepTile;
  static constexpr int kBars = 2 * kStages + 14;
  static constexpr int kSmem = kBarOff + kBars * 8 + 128 + 1024;  // + alignment
  static_assert(kSmem <= 227 * 1024, "shared memory");
  // Registers after the split: 256 x (184 + 72) = 512 x 128, what the block starts with (a
  // tile of 64 keys is less to hold, and its rows of 256 columns more to have on the way).
  static constexpr int kSoftRegs = kWide ? 160 : 184, kOtherRegs = kWide ? 96 : 72;
  static_assert(256 * (kSoftRegs + kOtherRegs) <= kThreads * 128, "more registers than the block was launched with");
  using C = std::conditional_t<BITS == 16, T, __half>;
  static constexpr bool kRowFactor = BITS != 16 && std::is_same_v<T, __nv_bfloat16>;
  static constexpr uint32_t kType = std::is_same_v<C, __nv_bfloat16> ? 1u : 0u;
  // columns of tensor memory: S, P and O of chain i
  static constexpr int kCols = 512;
  static constexpr int kOCol = DP == 64 ? 384 : 256;
  __device__ static constexpr uint32_t s_at(int i) { return i * 128; }
  __device__ static constexpr uint32_t p_at(int i) { return DP == 64 ? 256 + i * 64 : i * 128 + kKeys; }
  __device__ static constexpr uint32_t o_at(int i) { return kOCol + i * (kWide ? 128 : DP); }
  // the columns of V, and of the output, that are chain i's: a number of them from the first
  __device__ static constexpr int first_col(int i) { return kWide ? i * 128 : 0; }
  __device__ static constexpr int num_cols(int i, int head_dim) { return !kWide ? head_dim : i == 0 ? 128 : head_dim - 128; }
  static_assert(DP == 64 || kKeys + kKeys / 2 <= 128, "S and P of a chain in 128 columns");
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

template <int N>
__device__ __forceinline__ void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// 64 columns x 16 tokens of one page and head (no multicast).
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z, int w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
      "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}
// Shared memory is read by its 32-bit address: the compiler does not see through the
// aligned base and would read generically.
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void sts128(uint32_t addr, uint4 v) {
  asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void lds_pairs(uint32_t addr, F2 (&v)[2]) {
  asm volatile("ld.shared.v2.b64 {%0, %1}, [%2];" : "=l"(v[0].v), "=l"(v[1].v) : "r"(addr) : "memory");
}

// Four K = 16 steps of O += P V, issued from one asm block (their operands are then formed
// back to back): P 8 columns a step, V 16 keys of 128 bytes.
__device__ __forceinline__ void umma_pv(uint32_t d, uint32_t p, uint64_t v, uint32_t id, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      ".reg .b32 a1, a2, a3;\n\t"
      ".reg .b64 b1, b2, b3;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.eq.u32 q, 0, 0;\n\t"
      "add.u32 a1, %1, 8;\n\tadd.u32 a2, %1, 16;\n\tadd.u32 a3, %1, 24;\n\t"
      "add.u64 b1, %2, 128;\n\tadd.u64 b2, %2, 256;\n\tadd.u64 b3, %2, 384;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [a1], b1, %3, q;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [a2], b2, %3, q;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [a3], b3, %3, q;\n\t}" ::"r"(d),
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

// What a block did, for k_attn_tiles.
struct TileNote {
  int start, row0, rows, head, seq;
  int odd;  // a value that is no number lay in a tile that not every row sees whole
};
// How the items (row tiles x KV heads) fall to the blocks: the first `whole` to one each,
// the rest to `spans` each.
struct Shares {
  int items, whole, spans;
};

struct TileArgs {
  TileNote* note;  // [blocks]
  Shares* shares;
  float* o;        // [slots][tile rows][DP]: parts of rows
  float2* ml;      // [slots][tile rows]
  int sms;
  int most_tiles;  // row tiles that the grid and the buffers are planned for
  int most_spans;  // of an item
  int tile_rows;   // 256; 128 where both chains take the same rows
  bool alternate;  // they take every second tile of keys each
  bool tma;        // the maps of the cache are valid (16 bits, pages of 16 tokens and more)

  __device__ __forceinline__ Shares share(int items) const {
    Shares s;
    s.items = items;
    s.whole = items / sms * sms;
    s.spans = items > s.whole ? min(most_spans, max(1, sms / (items - s.whole))) : 1;
    return s;
  }
  // the first slot of block i's parts (one, or a chain each)
  __device__ __forceinline__ int slot(const Shares& s, int i) const {
    return alternate ? 2 * i : i - s.whole;
  }
  __device__ __forceinline__ bool cut(const Shares& s, int i) const {
    return alternate || (i >= s.whole && s.spans > 1);
  }
};

template <typename T, int BITS, int DP>
__global__ void __launch_bounds__(kThreads, 1) k_attn_many(const AttnArgs a, const TileArgs ta,
                                                        const __grid_constant__ CUtensorMap map_k,
                                                        const __grid_constant__ CUtensorMap map_v) {
  using K = Tc<T, BITS, DP>;
  using C = typename K::C;
  constexpr int kStages = K::kStages, kKeys = K::kKeys;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* const smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* const s_prep = reinterpret_cast<float*>(smem + K::kPrepOff);
  uint64_t* const bars = reinterpret_cast<uint64_t*>(smem + K::kBarOff);
  uint64_t* const full = bars;                  // [stages] rows landed
  uint64_t* const empty = bars + kStages;       // [stages] products done with them
  uint64_t* const s_full = bars + 2 * kStages;  // [2] S written
  uint64_t* const p_full = s_full + 2;          // [2] P written (and O moved, where it was)
  uint64_t* const o_done = s_full + 4;          // [2] P V done
  uint64_t* const prep_full = s_full + 6;       // [2]
  uint64_t* const prep_empty = s_full + 8;      // [2]
  uint64_t* const drain = s_full + 10;          // [2]
  uint64_t* const s_free = s_full + 12;         // [2] S in registers
  uint32_t* const s_tmem = reinterpret_cast<uint32_t*>(bars + K::kBars);
  int* const s_odd = reinterpret_cast<int*>(s_tmem + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int D = a.kv.head_dim;
  const bool alternate = !K::kWide && ta.alternate, same_rows = K::kWide || alternate;

  if (warp == kMmaWarp) {
    tmem_alloc(s_tmem, K::kCols);
    tmem_relinquish();
  }
  grid_dep_wait();

  // ------------------------------------------------------------ this block's rows and keys
  // Tiles in descending order of their position: of a causal sequence's tiles the last
  // ones are the longest, and the short ones fill the machine's end.
  auto tiles_of = [&](int b) { return (seq_range(a, b).q_len * a.group + ta.tile_rows - 1) / ta.tile_rows; };
  int64_t tiles = 0;
  for (int b = lane; b < a.num_seqs; b += 32) tiles += tiles_of(b);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) tiles += __shfl_xor_sync(0xffffffffu, tiles, o);
  // Starts that go back give several sequences the same tokens, and more tiles than the
  // call's tokens have: those past the plan are left out.
  if (tiles > ta.most_tiles) set_device_error(kDevBadCachePos);
  const int total = static_cast<int>(min(tiles, static_cast<int64_t>(ta.most_tiles)));
  const int block = static_cast<int>(blockIdx.x);
  const Shares shares = ta.share(total * a.kv.kv_heads);
  if (block == 0 && threadIdx.x == 0) *ta.shares = shares;
  const bool own_item = block < shares.whole;
  const int spans = own_item ? 1 : shares.spans;
  const int span = own_item ? 0 : (block - shares.whole) % spans;
  const int item = own_item ? block : shares.whole + (block - shares.whole) / spans;
  const int h = item % a.kv.kv_heads;
  const int tile = total - 1 - item / a.kv.kv_heads;
  const bool work = item < shares.items;
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
    const int t0 = first_seen(tile_min, a.window) / kKeys, n = max(0, (tile_max + 1 + kKeys - 1) / kKeys - t0);
    k0 = t0 + static_cast<int>(static_cast<int64_t>(n) * span / spans);
    k1 = t0 + static_cast<int>(static_cast<int64_t>(n) * (span + 1) / spans);
  }
  const int n_tiles = k1 - k0;
  // (not zero: a score that is masked by -inf stays so times it)
  const float cs = fmaxf(fabsf(a.scale) * kLog2e, 1.17549435e-38f);

  // which tiles chain i takes: all, or every second one
  const int step = alternate ? 2 : 1;
  auto chain_first = [&](int i) { return alternate ? i : 0; };
  // a chain without rows is left out
  const bool chain_b = same_rows || rows > kRows;

  if (threadIdx.x == 0) {
    const int chains = chain_b && !alternate ? 2 : 1;  // that take each tile
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 4);  // one arrival a loader warp
      mbar_init(&empty[s], chains);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&o_done[i], 1);
      mbar_init(&prep_full[i], 4);
      mbar_init(&prep_empty[i], 4 * chains);  // softmax warps
      mbar_init(&drain[i], 1);
      mbar_init(&s_free[i], 4);
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
      from = first_seen(last, a.window);
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
    uint8_t* const dst = smem + K::kQOff + (K::kWide ? 0 : chain * K::kQTile) + tid * 128;
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
      if (!K::kWide || chain == 0)
        *reinterpret_cast<uint4*>(dst + (c >> 3) * K::kQPanel + (((c & 7) ^ (tid & 7)) << 4)) = w;
    }
    fence_proxy_async_smem();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();

  bool ok = true;  // no wait of this thread ran out
  if (warp >= kLoadWarp) {
    regs_down<K::kOtherRegs>();
    // ---------------------------------------------------------- loads
    const int me = static_cast<int>(threadIdx.x) - kLoadWarp * 32;
    const int mask = (1 << a.kv.page_shift) - 1;
    const int row_bytes = D * BITS / 8;
    constexpr int kChunks = DP * BITS / 128;     // 16-byte pieces of a stored row
    constexpr int kRowsIt = kLoaders / kChunks;  // rows of one step of the loaders
    constexpr int kIts = (kKeys + kRowsIt - 1) / kRowsIt;
    const int32_t* const table = a.page_table + b * a.page_table_stride;
    const int c = me % kChunks, crow = me / kChunks;
    const bool mine = c * 16 < row_bytes;
    const uint32_t ring = smem_u32(smem + K::kRingOff);
    // This thread's rows of a tile: kIts neighbours from `row0`, so that pages of 16 tokens
    // and more give it two pages at most. Their ids are asked for a tile ahead.
    const int row0 = crow * kIts;
    const int n_rows = mine ? min(kIts, max(0, kKeys - row0)) : 0;
    const bool two_pages = mask >= 15;
    int ids[2] = {-1, -1};
    auto ask_pages = [&](int t) {
      const int j = (k0 + t) * kKeys + row0, end = min(r.kv_len, j + n_rows);
      ids[0] = t < n_tiles && j < end ? __ldg(table + (j >> a.kv.page_shift)) : -1;
      ids[1] = t < n_tiles && j < end ? __ldg(table + ((end - 1) >> a.kv.page_shift)) : -1;
    };
    struct Rows {
      int64_t at[2];  // of the first row, and of the first in its last page
      int turn;       // rows in the first page
      int live[2];    // rows below this (from the start, from the turn) have data
    };
    auto good_page = [&](int id) {
      const bool good = static_cast<uint32_t>(id) < static_cast<uint32_t>(a.kv.num_pages);
      if (!good) set_device_error(kDevBadCachePos);
      return good;
    };
    auto rows_of = [&](int t) {
      Rows x{{0, 0}, kIts, {0, 0}};
      const int j = (k0 + t) * kKeys + row0, n = min(r.kv_len - j, n_rows);
      if (n <= 0 || t >= n_tiles) return x;
      const int off = j & mask;
      x.turn = min(kIts, mask + 1 - off);
      if (two_pages) {
        if (good_page(ids[0])) {
          x.at[0] = a.kv.row(ids[0], h, off);
          x.live[0] = min(n, x.turn);
        }
        if (n > x.turn && good_page(ids[1])) {
          x.at[1] = a.kv.row(ids[1], h, 0);
          x.live[1] = n - x.turn;
        }
      }
      return x;
    };
    const int64_t row_step = static_cast<int64_t>(a.kv.token_stride) * 8;
    // byte offset of row `it` of this thread in tile t, -1 without data
    auto row_at = [&](const Rows& x, int t, int it) -> int64_t {
      if (two_pages) {
        if (it < x.turn) return it < x.live[0] ? x.at[0] + it * row_step : -1;
        return it - x.turn < x.live[1] ? x.at[1] + (it - x.turn) * row_step : -1;
      }
      const int j = (k0 + t) * kKeys + row0 + it;
      if (it >= n_rows || j >= r.kv_len) return -1;
      const int id = __ldg(table + (j >> a.kv.page_shift));
      return good_page(id) ? a.kv.row(id, h, j & mask) : -1;
    };
    // 16-byte piece cc of this thread's row `it` in stage g
    auto place = [&](int g, int cc, int it) {
      const int row = row0 + it;
      return ring + g % kStages * K::kTile + (cc >> 3) * K::kPanel + row * 128 + (((cc & 7) ^ (row & 7)) << 4);
    };
    // K then V of each tile: stages g = 2 t + v of the ring
    if constexpr (BITS == 16) {
      // Tiles that every row sees whole come by TMA, 16 tokens (of one page) and 64 columns
      // a box, their boxes spread over the loader warps. The others, a few a block, are
      // copied row by row, which leaves out what lies past the sequence; their values are
      // then searched for what is no number.
      const int lw = warp - kLoadWarp;
      constexpr int kGroups = kKeys / 16;
      const int panels = (D + 63) / 64;
      int box_ids[2] = {-1, -1};  // pages of 16-token groups lw and lw + 4 of the next tile
      auto ask_boxes = [&](int t) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int j = (k0 + t) * kKeys + (lw + 4 * i) * 16;
          if (t < n_tiles && lw + 4 * i < kGroups && j < r.kv_len) box_ids[i] = __ldg(table + (j >> a.kv.page_shift));
        }
      };
      ask_boxes(0);
      bool odd = false;
      int armed = 0;  // stages filled so far
      for (int t = 0; t < n_tiles && ok; ++t) {
        const int j0 = (k0 + t) * kKeys;
        const bool mixed = j0 + kKeys - 1 > tile_min || (a.window > 0 && tile_max - j0 >= a.window);
        if (!mixed && ta.tma) {  // (no row sees past the sequence: the tile is inside it)
          int ids[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            ids[i] = box_ids[i];
            if (lw + 4 * i < kGroups && static_cast<uint32_t>(ids[i]) >= static_cast<uint32_t>(a.kv.num_pages)) {
              set_device_error(kDevBadCachePos);
              ids[i] = a.kv.num_pages;  // outside the map: zeros
            }
          }
          ask_boxes(t + 1);
          const uint32_t bytes = static_cast<uint32_t>(kGroups - lw > 4 ? 2 : 1) * panels * 2048u;
#pragma unroll
          for (int v = 0; v < 2; ++v) {
            const int g = 2 * t + v, s = g % kStages;
            ok = warp_wait(&empty[s], ((g / kStages) & 1) ^ 1u, kDevTimeoutAEmpty);
            if (!ok) break;
            if (elect_one()) {
              mbar_arrive_expect_tx(&full[s], bytes);
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                const int row = (lw + 4 * i) * 16;
                if (row >= kKeys) break;
                for (int q = 0; q < panels; ++q)
                  tma_load_4d(ring + s * K::kTile + q * K::kPanel + row * 128, v ? &map_v : &map_k, &full[s], 64 * q,
                              (j0 + row) & mask, h, ids[i]);
              }
            }
            __syncwarp();
            armed = g + 1;
          }
          continue;
        }
        ask_pages(t);
        const Rows x = rows_of(t);
        ask_boxes(t + 1);
#pragma unroll 1
        for (int v = 0; v < 2; ++v) {
          const int g = 2 * t + v, s = g % kStages;
          ok = warp_wait(&empty[s], ((g / kStages) & 1) ^ 1u, kDevTimeoutAEmpty);
          if (!ok) break;
          const uint8_t* const src = (v ? a.kv.v : a.kv.k) + c * 16;
#pragma unroll 1
          for (int it = 0; it < n_rows; ++it) {
            const int64_t ro = row_at(x, t, it);
            cp16(place(g, c, it), src + max(ro, int64_t{0}), ro < 0 ? 0u : 16u);
          }
          cp_commit();
          cp_wait<0>();
          if (v == 1 && mixed) {
            for (int it = 0; it < n_rows; ++it) {
              const uint4 w = lds128(place(g, c, it));
              const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float2 f = unpack2<T>(ws[e]);
                odd |= !isfinite(f.x) || !isfinite(f.y);
              }
            }
          }
          fence_proxy_async_smem();
          warp_arrive(&full[s]);
          armed = g + 1;
        }
      }
      if (odd) *s_odd = 1;
      // copies by TMA that no product has waited for (a wait ran out) must land before the
      // block leaves its shared memory
      if (!ok) {
        for (int s = 0; s < kStages && s < armed; ++s) mbar_wait_drain(&full[s], ((armed - 1 - s) / kStages) & 1);
      }
    } else {
      const bool wide = BITS == 8 || row_bytes % 16 == 0;
      // Steps of the tile's keys, one a loader, asked for a tile ahead.
      float2 ksc = make_float2(0.f, 0.f), vsc = ksc;
      auto ask_steps = [&](int t) {
        ksc = vsc = make_float2(0.f, 0.f);
        const int j = (k0 + t) * kKeys + me;
        if (me >= kKeys || t >= n_tiles || j >= r.kv_len) return;
        const int page = __ldg(table + (j >> a.kv.page_shift));
        if (static_cast<uint32_t>(page) >= static_cast<uint32_t>(a.kv.num_pages)) return;
        const int64_t at = a.kv.scale_row(page, h, j & mask);
        if constexpr (BITS == 8) {
          ksc.x = __ldg(a.kv.k_scale + at);
          vsc.x = __ldg(a.kv.v_scale + at);
        } else {
          ksc = __ldg(reinterpret_cast<const float2*>(a.kv.k_scale + at));
          vsc = __ldg(reinterpret_cast<const float2*>(a.kv.v_scale + at));
        }
      };
      auto fetch_codes = [&](const Rows& x, int t, const uint8_t* base, uint4 (&raw)[kIts]) {
        if (x.live[0] == kIts && wide) {  // all in one page, as nearly always
          const uint8_t* src = base + x.at[0] + c * 16;
#pragma unroll
          for (int it = 0; it < kIts; ++it, src += row_step) raw[it] = __ldg(reinterpret_cast<const uint4*>(src));
          return;
        }
#pragma unroll
        for (int it = 0; it < kIts; ++it) {
          raw[it] = make_uint4(0u, 0u, 0u, 0u);
          const int64_t ro = row_at(x, t, it);
          if (ro < 0) continue;
          const uint8_t* const src = base + ro + c * 16;
          if (wide) {
            raw[it] = __ldg(reinterpret_cast<const uint4*>(src));
          } else {
            const uint2 x = __ldg(reinterpret_cast<const uint2*>(src));
            raw[it].x = x.x;
            raw[it].y = x.y;
            if (c * 16 + 8 < row_bytes) {
              const uint2 y = __ldg(reinterpret_cast<const uint2*>(src + 8));
              raw[it].z = y.x;
              raw[it].w = y.y;
            }
          }
        }
      };
      auto store_codes = [&](int g, const uint4 (&raw)[kIts]) {
        ok = warp_wait(&empty[g % kStages], ((g / kStages) & 1) ^ 1u, kDevTimeoutAEmpty);
        if (!ok) return;
        {
#pragma unroll
          for (int it = 0; it < kIts; ++it) {
            if (it >= n_rows) break;
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
              sts128(place(g, c * kOut + o, it), w);
            }
          }
        }
        fence_proxy_async_smem();
        warp_arrive(&full[g % kStages]);
      };
      auto factors = [&](int t, float2 kstep, float2 vstep) {
        ok = warp_wait(&prep_empty[t & 1], ((t >> 1) & 1) ^ 1u, kDevTimeoutAEmpty);
        if (!ok) return;
        // the key's factors: a = s c, log2 t, 1 / t (and z c, y / t), with c = scale log2(e).
        // A poisoned step of either makes a NaN in a, which reaches the weights of the rows
        // that see the key and no others; the rest must then be numbers.
        if (me < kKeys) {
          float* const prep = s_prep + (t & 1) * (K::kPrepTile / 4);
          const float vbase = BITS == 4 ? fmaf(8.f, vstep.x, vstep.y) : 0.f;
          const float vs = value_step(vstep.x, vbase);
          const float lv = lg2(vs);
          bool bad = !(vs < INFINITY);
          if constexpr (BITS == 4) {
            const float zr = vbase / vs;
            bad = bad || !(fabsf(zr) < INFINITY);
            prep[3 * kKeys + me] = fmaf(8.f, kstep.x, kstep.y) * cs;
            prep[4 * kKeys + me] = bad ? 0.f : zr;
          }
          prep[me] = bad ? NAN : kstep.x * cs;
          prep[kKeys + me] = bad ? 0.f : lv;
          prep[2 * kKeys + me] = bad ? 0.f : ex2(-lv);
        }
        warp_arrive(&prep_full[t & 1]);
      };
      // each stage's codes are asked for a stage ahead
      uint4 raw_k[kIts], raw_v[kIts];
      ask_steps(0);
      ask_pages(0);
      Rows x = rows_of(0);
      ask_pages(1);
      if (n_tiles > 0) {
        fetch_codes(x, 0, a.kv.k, raw_k);
      }
      for (int t = 0; t < n_tiles && ok; ++t) {
        fetch_codes(x, t, a.kv.v, raw_v);
        const float2 kstep = ksc, vstep = vsc;
        ask_steps(t + 1);
        factors(t, kstep, vstep);
        if (ok) store_codes(2 * t, raw_k);
        if (!ok) break;
        if (t + 1 < n_tiles) {
          x = rows_of(t + 1);
          ask_pages(t + 2);
          fetch_codes(x, t + 1, a.kv.k, raw_k);
        }
        store_codes(2 * t + 1, raw_v);
      }
    }
  } else if (warp >= kMmaWarp) {
    // ---------------------------------------------------------- products of one chain
    regs_down<K::kOtherRegs>();
    const int i = warp - kMmaWarp;
    if (i == 0 || (i == 1 && chain_b)) {
      const uint32_t s_col = tmem + K::s_at(i), p_col = tmem + K::p_at(i), o_col = tmem + K::o_at(i);
      const uint32_t id_s = idesc(K::kType, kKeys, false), id_o = idesc(K::kType, K::num_cols(i, D), true);
      const uint32_t q_addr = smem_u32(smem + K::kQOff + (K::kWide ? 0 : i * K::kQTile));
      const int ks = D / 16;
      // S of tile t, once its keys are there
      auto product_s = [&](int t) {
        const int g = 2 * t, s = g % kStages;
        ok = warp_wait(&full[s], (g / kStages) & 1, kDevTimeoutAFull);
        if (!ok) return;
        tc_fence_after();
        if (elect_one()) {
          const uint32_t k_addr = smem_u32(smem + K::kRingOff + s * K::kTile);
          int k = 0;
          for (; k + 4 <= ks; k += 4)
            umma_f16_k64(s_col, sdesc_sw128(q_addr + (k >> 2) * K::kQPanel), sdesc_sw128(k_addr + (k >> 2) * K::kPanel), id_s, k > 0);
          for (; k < ks; ++k)
            umma_f16(s_col, sdesc_sw128(q_addr + (k >> 2) * K::kQPanel + (k & 3) * 32),
                     sdesc_sw128(k_addr + (k >> 2) * K::kPanel + (k & 3) * 32), id_s, k > 0);
          umma_commit(&s_full[i]);
          umma_commit(&empty[s]);
        }
        __syncwarp();
      };
      int t = chain_first(i);
      if (t < n_tiles) product_s(t);
      for (int n = 0; t < n_tiles && ok; t += step, ++n) {
        if (t + step < n_tiles) {
          // the next tile's S, once this one's is in registers: under the exponentials
          ok = warp_wait(&s_free[i], n & 1, kDevTimeoutAccEmpty);
          if (ok) product_s(t + step);
        }
        const int g = 2 * t + 1, s = g % kStages;
        ok = ok && warp_wait(&full[s], (g / kStages) & 1, kDevTimeoutAFull) && warp_wait(&p_full[i], n & 1, kDevTimeoutAccEmpty);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          const uint64_t v = sdesc_v(smem_u32(smem + K::kRingOff + s * K::kTile + K::first_col(i) / 64 * K::kPanel), K::kPanel);
          umma_pv(o_col, p_col, v, id_o, n > 0);
          if constexpr (kKeys == 128) umma_pv(o_col, p_col + 32, v + 512, id_o, 1);
          if constexpr (kKeys == 80) umma_f16_ts(o_col, p_col + 32, v + 512, id_o, 1);
          umma_commit(&o_done[i]);
          umma_commit(&empty[s]);
        }
        __syncwarp();
      }
      if (elect_one()) umma_commit(&drain[i]);
      __syncwarp();
      mbar_wait_drain(&drain[i], 0);
    }
  } else {
    regs_up<K::kSoftRegs>();
    if (chain == 0 || chain_b) {
    // ---------------------------------------------------------- softmax: a thread a row
    const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;  // 32 lanes a warp
    const uint32_t s_col = tmem + lanes + K::s_at(chain), p_col = tmem + lanes + K::p_at(chain),
                   o_col = tmem + lanes + K::o_at(chain);
    // positions of this warp's first and last row
    const int w_row = my_row - lane;
    const int w_min = pos0 + (row0 + w_row) / a.group;
    const int w_max = pos0 + (row0 + min(w_row + 31, max(rows, 1) - 1)) / a.group;
    const int cols = K::num_cols(chain, D);
    float ref = -INFINITY, l = 0.f, zacc = 0.f;
    int n = 0;
    for (int t = chain_first(chain); t < n_tiles && ok; t += step, ++n) {
      const int j0 = (k0 + t) * kKeys;
      const bool whole = j0 + kKeys - 1 <= w_min && (a.window <= 0 || w_max - j0 < a.window);
      const uint32_t prep = smem_u32(s_prep + (t & 1) * (K::kPrepTile / 4));
      if constexpr (BITS != 16) ok = warp_wait(&prep_full[t & 1], (t >> 1) & 1, kDevTimeoutAFull);
      ok = ok && warp_wait(&s_full[chain], n & 1, kDevTimeoutAccFull);
      if (!ok) break;
      tc_fence_after();
      uint32_t s[kKeys];
#pragma unroll
      for (int c = 0; c < kKeys / 32; ++c) tmem_ld32(s_col + 32 * c, reinterpret_cast<uint32_t(&)[32]>(s[32 * c]));
      if constexpr (kKeys % 32 != 0) tmem_ld16(s_col + kKeys - 16, reinterpret_cast<uint32_t(&)[16]>(s[kKeys - 16]));
      tmem_ld_wait();
      tc_fence_before();
      warp_arrive(&s_free[chain]);
      auto sf = [&](int j) { return __uint_as_float(s[j]); };
      if constexpr (BITS != 16) {
        // scores of codes, the value's step as a shift
        const F2 qs2 = f2(qsum, qsum), rf2 = f2(rf, rf);
#pragma unroll
        for (int j = 0; j < kKeys; j += 4) {
          F2 a2[2], lv2[2], z2[2];
          lds_pairs(prep + 4 * j, a2);
          lds_pairs(prep + 4 * (kKeys + j), lv2);
          if constexpr (BITS == 4) lds_pairs(prep + 4 * (3 * kKeys + j), z2);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const F2 s2 = f2(sf(j + 2 * e), sf(j + 2 * e + 1));
            F2 x;
            if constexpr (K::kRowFactor) {
              x = mul2(s2, a2[e]);
              if constexpr (BITS == 4) x = fma2(qs2, z2[e], x);
              x = fma2(x, rf2, lv2[e]);
            } else {
              if constexpr (BITS == 4) lv2[e] = fma2(qs2, z2[e], lv2[e]);
              x = fma2(s2, a2[e], lv2[e]);
            }
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
          for (int c = 0; c < cols; c += 16) {
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
      uint32_t p[kKeys / 2];
      auto weights = [&](int from_i, int to_i) {  // pairs of keys
#pragma unroll
        for (int i = from_i; i < to_i; i += 2) {
          const int j = 2 * i;
          F2 inv[2], zr[2];
          if constexpr (BITS != 16) lds_pairs(prep + 4 * (2 * kKeys + j), inv);
          if constexpr (BITS == 4) lds_pairs(prep + 4 * (4 * kKeys + j), zr);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const F2 s2 = f2(sf(j + 2 * e), sf(j + 2 * e + 1));
            float y0, y1;
            split(BITS == 16 ? fma2(s2, cs2, base2) : add2(s2, base2), y0, y1);
            const float w0 = ex2(y0), w1 = ex2(y1);
            const F2 w = f2(w0, w1);
            if constexpr (BITS == 16) lt[e] = add2(lt[e], w);
            else lt[e] = fma2(w, inv[e], lt[e]);
            p[i + e] = pack2<C>(w0, w1);
            if constexpr (BITS == 4) {
              // the rounded weights, so that their rounding scales with the value and not
              // with the code's distance from 8 (but below fp16's normal range, where a
              // row of equal values comes with its tiny step, the weight itself)
              const float2 f = unpack2<C>(p[i + e]);
              zt = fma2(f2(w0 < kHalfMin ? w0 : f.x, w1 < kHalfMin ? w1 : f.y), zr[e], zt);
            }
          }
        }
      };
      // (asked now, so that the answer is there when P goes out)
      const bool p_free = n == 0 || mbar_test_wait(smem_u32(&o_done[chain]), (n - 1) & 1);
      weights(0, 32);
      if (!__all_sync(0xffffffffu, p_free)) {
        ok = warp_wait(&o_done[chain], (n - 1) & 1, kDevTimeoutAccFull);
        if (!ok) break;
      }
      tc_fence_after();
      tmem_st32(p_col, reinterpret_cast<uint32_t(&)[32]>(p[0]));
      weights(32, kKeys / 2);
      if constexpr (kKeys == 128) tmem_st32(p_col + 32, reinterpret_cast<uint32_t(&)[32]>(p[32]));
      if constexpr (kKeys == 80) tmem_st8(p_col + 32, reinterpret_cast<uint32_t(&)[8]>(p[32]));
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
      const bool cut = ta.cut(shares, block);
      const int64_t slot = cut ? static_cast<int64_t>(ta.slot(shares, block) + (alternate ? chain : 0)) * ta.tile_rows + my_row : 0;
      const bool tells = in && (!K::kWide || chain == 0);  // the row's sums, which both have
      if (tells && cut) ta.ml[slot] = make_float2(ref, l);
      if (tells && !cut && a.lse != nullptr) a.lse[at] = l == 0.f ? -INFINITY : (ref + log2f(l)) * kLn2;
#pragma unroll 1
      for (int c = 0; c < cols; c += 16) {
        float x[16];
        if (n > 0) {
          uint32_t o[16];
          tmem_ld16(o_col + c, o);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            // a 4-bit row's columns stand in the order its codes unpack
            const int d = BITS == 4 ? (e & 8) + place4(e & 7) : e;
            x[d] = BITS == 16 ? __uint_as_float(o[e]) : __uint_as_float(o[e]) + zacc;
          }
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e) x[e] = 0.f;
        }
        if (!in) continue;
        if (cut) {
          float4* const dst = reinterpret_cast<float4*>(ta.o + slot * DP + K::first_col(chain) + c);
#pragma unroll
          for (int e = 0; e < 4; ++e) dst[e] = make_float4(x[4 * e], x[4 * e + 1], x[4 * e + 2], x[4 * e + 3]);
        } else {
          uint4* const dst = reinterpret_cast<uint4*>(static_cast<T*>(a.out) + at * D + K::first_col(chain) + c);
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
  if (threadIdx.x == 0) ta.note[block] = TileNote{r.start, row0, rows, h, b, *s_odd};
  if (warp == kMmaWarp) tmem_dealloc(tmem, K::kCols);
}

// Adds up the parts of items that were cut, a few rows of one at a time; and, where a
// value that is no number met rows that do not see it, takes an item's rows one by one.
constexpr int kJoinThreads = 128;
template <typename T, int BITS, int DP>
__global__ void __launch_bounds__(kJoinThreads) k_attn_tiles(const AttnArgs a, const TileArgs ta) {
  __shared__ AttnRowSmem sm;
  constexpr int kCols = DP / 4, kGroups = kJoinThreads / kCols;
  grid_dep_wait();
  const Shares shares = *ta.shares;
  const int chains = ta.alternate ? 2 : 1;
  auto first_block = [&](int item) {
    return item < shares.whole ? item : shares.whole + (item - shares.whole) * shares.spans;
  };
  auto is_odd = [&](int item) {
    bool odd = false;
    if constexpr (BITS == 16) {
      const int i = first_block(item);
      for (int s = 0; s < (item < shares.whole ? 1 : shares.spans); ++s) odd |= ta.note[i + s].odd != 0;
    }
    return odd;
  };
  const int steps = ta.tile_rows / kGroups;  // of kGroups rows an item
  const int first = chains == 2 ? 0 : shares.spans > 1 ? shares.whole : shares.items;
  const int col = threadIdx.x % kCols, grp = threadIdx.x / kCols;
  for (int64_t u = blockIdx.x; u < static_cast<int64_t>(shares.items - first) * steps; u += gridDim.x) {
    const int item = first + static_cast<int>(u / steps);
    const int i = first_block(item), parts = chains * (item < shares.whole ? 1 : shares.spans);
    const TileNote note = ta.note[i];
    const int row = static_cast<int>(u % steps) * kGroups + grp;
    if (row >= note.rows || is_odd(item)) continue;
    const int64_t s0 = static_cast<int64_t>(ta.slot(shares, i)) * ta.tile_rows + row;
    float top = -INFINITY;
    for (int p = 0; p < parts; ++p) top = fmaxf(top, ta.ml[s0 + static_cast<int64_t>(p) * ta.tile_rows].x);
    const float ref = top == -INFINITY ? 0.f : top;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = 0.f;
#pragma unroll 4
    for (int p = 0; p < parts; ++p) {
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
  if constexpr (BITS == 16) {
    for (int item = blockIdx.x; item < shares.items; item += gridDim.x) {
      if (!is_odd(item)) continue;
      const TileNote note = ta.note[first_block(item)];
      const SeqRange r = seq_range(a, note.seq);
      for (int row = 0; row < note.rows; ++row)
        attn_one_row<T>(a, note.seq, r, (note.row0 + row) / a.group, note.head * a.group + (note.row0 + row) % a.group, sm);
    }
  }
}

// ------------------------------------------------------------------ host
struct Plan {
  int tile_rows, tiles, most_spans, blocks, slots;
  bool alternate;
};
Plan plan(const AttnArgs& a, int max_q_len, int max_kv_len) {
  Plan p;
  const int sms = device_sm_count();
  const int64_t rows = static_cast<int64_t>(a.num_tokens) * a.group;
  const bool wide = a.kv.head_dim > 128;
  p.alternate = !wide && static_cast<int64_t>(max_q_len) * a.group <= kRows;
  p.tile_rows = wide || p.alternate ? kRows : 2 * kRows;
  p.tiles = static_cast<int>(std::min<int64_t>(rows, rows / p.tile_rows + a.num_seqs));  // a partial one each
  // an item may be cut until a part has 512 keys
  p.most_spans = std::max(1, max_kv_len / 512);
  // whole rounds of items, and a round of parts
  p.blocks = static_cast<int>(static_cast<int64_t>(p.tiles) * a.kv.kv_heads / sms * sms + sms);
  p.slots = p.alternate ? 2 * p.blocks : sms;
  return p;
}
size_t round256(size_t v) { return (v + 255) & ~static_cast<size_t>(255); }

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static const PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
    return static_cast<PFN_cuTensorMapEncodeTiled_v12000>(nullptr);
  }();
  return fn;
}

// Keys or values of a 16-bit cache as [page][head][token][column], 16 tokens x 64 columns
// a box. False where the map cannot be made; the rows are then copied one by one.
bool cache_map(CUtensorMap* m, const KvDev& kv, const void* base, bool bf16) {
  const auto fn = encode_fn();
  if (fn == nullptr || kv.page_shift < 4) return false;
  cuuint64_t dims[4] = {static_cast<cuuint64_t>(kv.head_dim), cuuint64_t{1} << kv.page_shift,
                        static_cast<cuuint64_t>(kv.kv_heads), static_cast<cuuint64_t>(kv.num_pages)};
  cuuint64_t strides[3] = {cuuint64_t{kv.token_stride} * 8, cuuint64_t{kv.head_stride} * 8, cuuint64_t{kv.page_stride} * 8};
  cuuint32_t box[4] = {64, 16, 1, 1};
  cuuint32_t ones[4] = {1, 1, 1, 1};
  return fn(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(base), dims,
            strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int BITS, int DP>
struct Many {
  static std::atomic<size_t> raised[kMaxDevices];
  static size_t workspace(const Plan& p) {
    return round256(sizeof(Shares)) + round256(p.blocks * sizeof(TileNote)) +
           static_cast<size_t>(p.slots) * p.tile_rows * (DP * sizeof(float) + sizeof(float2));
  }
  static cudaError_t launch(const AttnArgs& a, const Plan& p, void* ws, cudaStream_t s) {
    using K = Tc<T, BITS, DP>;
    cudaError_t e = raise_smem_limit(k_attn_many<T, BITS, DP>, K::kSmem, raised);
    if (e != cudaSuccess) return e;
    TileArgs ta;
    char* w = static_cast<char*>(ws);
    ta.shares = reinterpret_cast<Shares*>(w);
    w += round256(sizeof(Shares));
    ta.note = reinterpret_cast<TileNote*>(w);
    w += round256(p.blocks * sizeof(TileNote));
    ta.o = reinterpret_cast<float*>(w);
    ta.ml = reinterpret_cast<float2*>(ta.o + static_cast<size_t>(p.slots) * p.tile_rows * DP);
    ta.sms = device_sm_count();
    ta.most_tiles = p.tiles;
    ta.most_spans = p.most_spans;
    ta.tile_rows = p.tile_rows;
    ta.alternate = p.alternate;
    CUtensorMap maps[2] = {};
    ta.tma = BITS == 16 && cache_map(&maps[0], a.kv, a.kv.k, std::is_same_v<T, __nv_bfloat16>) &&
             cache_map(&maps[1], a.kv, a.kv.v, std::is_same_v<T, __nv_bfloat16>);
    e = launch_dep(k_attn_many<T, BITS, DP>, dim3(static_cast<unsigned>(p.blocks)), dim3(kThreads), K::kSmem, s, a, ta, maps[0],
                   maps[1]);
    if (e != cudaSuccess) return e;
    return launch_dep(k_attn_tiles<T, BITS, DP>, dim3(static_cast<unsigned>(8 * ta.sms)), dim3(kJoinThreads), 0, s, a, ta);
  }
};
template <typename T, int BITS, int DP>
std::atomic<size_t> Many<T, BITS, DP>::raised[kMaxDevices];

template <typename F>
auto with_many(int bits, bool bf16, int head_dim, F&& f) {
  auto dim = [&](auto t, auto b) {
    if (head_dim <= 64) return f(Many<decltype(t), decltype(b)::value, 64>());
    if (head_dim <= 128) return f(Many<decltype(t), decltype(b)::value, 128>());
    return f(Many<decltype(t), decltype(b)::value, 256>());
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
  return with_many(bits, bf16, a.kv.head_dim, [&](auto k) { return decltype(k)::workspace(p); });
}
cudaError_t launch_many(const AttnArgs& a, int bits, bool bf16, int max_q_len, int max_kv_len, void* workspace,
                        cudaStream_t s) {
  const Plan p = plan(a, max_q_len, max_kv_len);
  return with_many(bits, bf16, a.kv.head_dim, [&](auto k) { return decltype(k)::launch(a, p, workspace, s); });
}

}  // namespace gemq
