// Attention of a few new tokens over a paged key/value cache, on sm_100a tensor cores (TMA, tcgen05
// MMA, TMEM accumulators): a tree of drafted tokens, or causal with a sliding window and a few first
// tokens that stay visible.
//
// For query row (sequence b, token t, head h), over the keys j it sees:
//   s_j = scale * q . k_j ; m = max s ; o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m)
// scores, m, sums and o in fp32; the exponentials are rounded to the cache's type for the product
// with V (the tensor core multiplies 16-bit operands), o once at the end.  A row that sees nothing
// gives 0.
//
// Work.  A unit is (sequence, key head, block of tokens): its rows are the block's tokens times the
// G query heads of the key head, packed token-major into one or two 128-row tiles, so each key and value
// row is read once for all of them.  A unit's key axis is cut into tiles; all units' tiles form one
// line (ordered by sequence, token block, key head) that is cut into equal pieces, one per CTA.  A CTA
// runs its piece as one stream of tiles; a unit inside one piece is finished there, a unit cut between
// pieces leaves (o, m, l) parts in the workspace that cache_attn_join adds up in order.  So ragged
// lengths balance by themselves, from lengths that only the device knows.
// Where the sizes say that units are short (few_tiles), pieces begin at units and none is cut.
//
// Two shapes of CTA (one per SM), chosen by the rows a unit has (see launch()).  Both run two softmax
// streams of four warps, so that one stream's tensor work overlaps the other's exponentials:
//   NT = 1: one 128-row tile; the streams take alternate key tiles of the same rows, each with its own
//           (o, m, l), and merge at the unit's end.  For up to 128 rows: decode and small trees, bound by
//           HBM.  Up to 16 rows (KS = 4 key groups) are copied to the four quarters of a 64-row MMA, and
//           each softmax warp takes a quarter of the key tile: a quarter of the exponentials per
//           warp, half of the tensor work.
//           Tiles are 64 keys with four S buffers at head_dim 128 (3 to 6% faster than 128 keys, whose ring is
//           only 2 + 3 tiles deep) and 128 keys with three at head_dim 64 (64 keys: 13% slower, each
//           Q K^T reads all of Q from shared memory, however few keys it covers).
//   NT = 2: two 128-row tiles that share every K and V tile of 128 keys; a stream is a row tile.  For
//           wide trees and prompt chunks, bound by the tensor cores and the exponentials.
// Warps: 8 softmax (one thread per row = TMEM lane; the same thread rescales and writes out the row),
// one for K loads, one for V loads, and two that issue MMAs and load Q: NT = 1 has Q and Q K^T in one, P V in the
// other (one thread for both products waited for P while K had landed: 5% slower decode); NT = 2 all MMAs in
// one, Q in the other.
// A value row that no token of the unit sees (past the sequence's end, between the sinks and the window, a draft that
// no mask names) must not be multiplied as it is: it may never have been written, and 0 * NaN is not 0.
// Whole pages of such rows are loaded from outside the tensor map, which reads as zeros.  Of a page seen in part,
//   with key groups: the softmax warps clear them in shared memory before they hand over P;
//   without: V comes in boxes of 8 rows, and of single rows where 8 are seen in part, each from its page or from outside.
// (Boxes with key groups: 64 x 1 token, window 4096: 175 -> 180 us, 59 x 1 token, window 86: 9.5 -> 11.6.  Clearing
// without: 16 x 27 drafts 55.1 -> 57.1, 1 x 9 drafts x 3 heads over 348 keys 10.6 -> 11.4.  Clearing by the warp that issues
// P V: 1 to 8% slower than either.)
// Every wait is bounded: one that gives up records a status code, and the CTA drains its copies
// and MMAs, frees TMEM and returns.
#include <atomic>
#include <climits>
#include <cuda_bf16.h>
#include <mutex>
#include <type_traits>

#include "ntl_common.cuh"

namespace {

__device__ uint32_t g_cache_attn_status;

constexpr int BM = 128;                // rows per tile
constexpr int kOutRow = 80;            // bytes from one staged output row to the next: 64 and a gap against bank conflicts
// O is rescaled only when a row's maximum rose by more than 2^15 since it was taken: exponentials stay below
// fp16's 2^16, and their rounding is relative.  (2^8: 2% slower where a row first sees a few sinks, 4096 tokens x 32
// heads, window 2048: 172 against 169 us.)
constexpr float kRescaleLog2 = 15.0f;

struct AttnBase {
  uint16_t* o;
  const int32_t* table;
  const int32_t* lens;
  const int32_t* q_lens;  // null: every sequence has `tokens`
  const uint32_t* tree;   // null: window
  float* part;            // workspace: [2 * ctas][rows][D] values, then [2 * ctas][rows] (m, l)
  float2* part_ml;
  int4* head;             // [ctas] the unit a CTA begins and does not end: {item, key head, last CTA, new tokens}
  int64_t table_stride, tree_stride;
  int seqs, tokens, heads, kv_heads, group, page_size, max_pages, words, window, sinks;
  int tile_tokens;   // tokens per 128-row tile
  int blocks;        // token blocks per sequence (units of NT tiles)
  int tile_keys;     // keys per tile: whole pages, or a part of a page
  int tile_pages;    // pages per tile (1 where a page holds several tiles)
  int page_tiles;    // tiles per page where the last is shorter, else 0
  int page_shift;    // log2 of page_size, -1 if it is no power of two
  int tile_shift;    // log2 of tile_keys, the same
  int rows;          // rows a workspace slot has
  int whole;         // no unit is cut: a CTA takes those that begin in its piece
  float c;           // softmax scale in log2 units
  int64_t wait_limit;
};

// SPLIT: a page holds several tiles and the last is shorter (page_tiles is set).  In the type, because the divisions
// cost the kernels that need none of them 1 to 17% (4096 tokens x 32 heads, window 2048: 159 against 186 us).
template <bool SPLIT>
struct AttnParams : AttnBase {
  static constexpr bool kSplit = SPLIT;
};

constexpr int SOFTMAX_WARPS = 8, MMA_WARP = 8, K_WARP = 9, V_WARP = 10, AUX_WARP = 11, THREADS = 384;
// Register split: the launch's registers per thread, what the softmax warps take, what the others keep.
constexpr int REGS_LAUNCH = 168, REGS_SOFTMAX = 200, REGS_OTHER = 104;
static_assert(8 * REGS_SOFTMAX + 4 * REGS_OTHER == 12 * REGS_LAUNCH, "register split must match the launch");
constexpr int kMaxStages = 6;
constexpr uint32_t TMEM_COLS = 512;

template <int D, int NT>
struct Shape {
  static constexpr int BN = NT == 1 && D == 128 ? 64 : 128;  // keys per tile
  static constexpr int BUFFERS = NT == 2 ? 2 : D == 128 ? 4 : 3;  // of S: of tile g in g % BUFFERS, or (NT = 2) by row tile
  static constexpr int K_STAGES = NT == 1 ? (D == 64 ? 4 : 5) : (D == 64 ? 4 : 2);
  static constexpr int V_STAGES = NT == 1 ? (D == 64 ? 6 : 5) : (D == 64 ? 4 : 2);
  static constexpr int Q_BYTES = BM * D * 2;
  static constexpr int KV_BYTES = BN * D * 2;
  static constexpr int K_OFF = NT * Q_BYTES;
  static constexpr int V_OFF = K_OFF + K_STAGES * KV_BYTES;
  static constexpr int OUT_OFF = V_OFF + V_STAGES * KV_BYTES;  // staging of the outputs, kOutRow * 32 bytes a warp
  static constexpr int CTL_OFF = OUT_OFF + SOFTMAX_WARPS * 32 * kOutRow;
  // S buffer b, O of stream i.
  __host__ __device__ static constexpr uint32_t S_COL(int i) { return static_cast<uint32_t>(i * BN); }
  __host__ __device__ static constexpr uint32_t O_COL(int i) { return static_cast<uint32_t>(BUFFERS * BN + i * D); }
  static_assert(BUFFERS * BN + 2 * D <= 512, "tensor memory columns");
};

struct Unit {
  int b, t0;        // sequence, first token
  int len, live;    // cached tokens; new tokens among them
  int tiles, sink_tiles, first;  // key tiles; those of the sinks; the window's first
};

// Beginning and ending a unit takes a CTA as long as several key tiles do, so each unit has that many
// places of the line after its tiles, and a CTA with many short units gets fewer tiles.
template <int NT>
constexpr int kUnitPlaces = NT == 1 ? 6 : 3;

struct __align__(16) Ctl {
  uint64_t q_full, q_empty;
  uint64_t k_full[kMaxStages], k_empty[kMaxStages], v_full[kMaxStages], v_empty[kMaxStages];
  uint64_t s_full[4];          // S buffer b holds scores
  uint64_t p_half[4];          // it holds the exponentials of the first half of the keys (4 warps; see HALVES)
  uint64_t p_ready[4];         // it holds all exponentials (4 warps)
  uint64_t pv_done[4];         // P V out of it is complete
  uint64_t o_free;             // NT = 1: a unit's O has been read out (8 warps)
  uint64_t streams;            // NT = 1: a unit's (m, l) are in `ml` and its P V are complete (8 warps)
  uint64_t groups[2];          // stream i's key groups: hand-offs among its four warps
  uint64_t drain[2];
  uint32_t tmem_base;
  int abort;
  int start[5];  // first unit's item, key head, tile; tiles of this CTA; total tiles
  Unit unit;     // the first unit
  int sums[32];
  float2 ml[2][2][BM];  // NT = 1: (m, l) of this and the next unit, by stream and TMEM lane
};

// A place in a ring of stages, and the phase its barriers are in there.
struct Ring {
  int s = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next(int stages) {
    if (++s == stages) s = 0, phase ^= 1;
  }
};

template <int D, int NT>
constexpr int smem_bytes() {
  const int used = Shape<D, NT>::CTL_OFF + static_cast<int>(sizeof(Ctl)) + 1024;
  static_assert(used <= 232448, "shared memory per CTA");
  // One CTA per SM needs >= 116 KB, so that its 512-column TMEM allocation never contends.
  return used < 118784 ? 118784 : used;
}

__device__ __forceinline__ void give_up(Ctl* ctl, uint32_t code) {
  if (!*reinterpret_cast<volatile int*>(&ctl->abort)) atomicCAS(&g_cache_attn_status, 0u, code);
  *reinterpret_cast<volatile int*>(&ctl->abort) = 1;
}

// mbar_wait_bounded with the clock read only once the wait is long (reading it first costs more than
// most of the waits here take).
__device__ __forceinline__ bool wait_bounded(uint64_t* bar, uint32_t parity, int64_t limit, volatile int* abort_flag) {
  if (mbar_test_wait(bar, parity)) return true;
  uint64_t t0 = 0;
  for (int64_t i = 1; i < limit; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((i & 63) == 63) {
      if (abort_flag != nullptr && *abort_flag) return false;
      const uint64_t now = global_ns();
      if (t0 == 0) t0 = now;
      if (now - t0 > kWaitCapNs) return false;
    }
  }
  return false;
}

// A wait of a whole warp, which gives up as one: no lane goes on without the others.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int64_t limit, volatile int* abort_flag) {
  return __all_sync(0xffffffffu, wait_bounded(bar, parity, limit, abort_flag));
}

// ------------------------------------------------------------------------------ units

template <class P>
__device__ __forceinline__ int tile_index(const P& p, int key) {
  if constexpr (P::kSplit) {
    const int page = key / p.page_size;
    return page * p.page_tiles + (key - page * p.page_size) / p.tile_keys;
  }
  return p.tile_shift >= 0 ? key >> p.tile_shift : key / p.tile_keys;
}

template <class P>
__device__ __forceinline__ Unit unit_of(const P& p, int item, int block_tokens) {
  Unit u;
  u.b = p.blocks == 1 ? item : item / p.blocks;
  u.t0 = (item - u.b * p.blocks) * block_tokens;
  u.len = min(max(p.lens[u.b], 0), p.max_pages * p.page_size);
  u.live = min(u.len, p.q_lens ? min(max(p.q_lens[u.b], 0), p.tokens) : p.tokens);
  u.tiles = 1;  // a unit without keys has one tile that nothing sees, and writes zeros
  u.sink_tiles = u.first = 0;
  if (u.t0 >= u.live) return u;
  if (p.tree) {
    u.tiles = tile_index(p, u.len - 1) + 1;
  } else {
    const int prefix = u.len - u.live;
    const int last = prefix + min(u.t0 + block_tokens, u.live) - 1;
    u.first = tile_index(p, max(0, prefix + u.t0 - p.window + 1));
    u.sink_tiles = p.sinks > 0 ? min(u.first, tile_index(p, p.sinks - 1) + 1) : 0;
    u.tiles = u.sink_tiles + tile_index(p, last) - u.first + 1;
  }
  return u;
}

template <class P>
__device__ __forceinline__ int tile_key(const P& p, const Unit& u, int a) {
  const int x = a < u.sink_tiles ? a : u.first + a - u.sink_tiles;
  if constexpr (P::kSplit) return x / p.page_tiles * p.page_size + x % p.page_tiles * p.tile_keys;
  return x * p.tile_keys;
}

// Keys of the tile that begins at key k0.  (Rows of a page's last tile past the page are zeros.)
template <class P>
__device__ __forceinline__ int tile_span(const P& p, int k0) {
  if constexpr (P::kSplit) return min(p.tile_keys, p.page_size - k0 % p.page_size);
  return p.tile_keys;
}

// The first key inside the window of the unit's first token.
template <class P>
__device__ __forceinline__ int window_from(const P& p, const Unit& u) {
  return max(0, u.len - u.live + u.t0 - p.window + 1);
}

// Whether the tile may hold rows that no token of the unit sees: rows past the sequence's end, rows between the sinks
// and the window, drafts.
template <class P>
__device__ __forceinline__ bool may_be_unseen(const P& p, const Unit& u, int a) {
  const int k0 = tile_key(p, u, a), end = k0 + tile_span(p, k0);
  if (p.tree) return end > u.len - u.live;
  return end > u.len || max(k0, p.sinks) < min(end, window_from(p, u));
}

// a / b for a >= 0, b > 0: the fast divide is within one of it below 2^22.
__device__ __forceinline__ int quotient(int a, int b) {
  if (a >> 22) return a / b;
  int q = static_cast<int>(__fdividef(static_cast<float>(a), static_cast<float>(b)));
  const int r = a - q * b;
  return r < 0 ? q - 1 : r >= b ? q + 1 : q;
}

// The pieces: `total` places of the line over `ctas` CTAs, CTA i from piece_start(i).
__device__ __forceinline__ int piece_start(int i, int total, int ctas) {  // floor(i * total / ctas)
  const int each = quotient(total, ctas);
  return i * each + quotient(i * (total - each * ctas), ctas);
}
__device__ __forceinline__ int piece_of(int place, int total, int ctas) {
  return static_cast<int>(((static_cast<int64_t>(place) + 1) * ctas - 1) / total);
}

__device__ __forceinline__ int block_exclusive(int x, int* sums, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  int s = x;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, s, d);
    if (lane >= d) s += y;
  }
  if (lane == 31) sums[warp] = s;
  __syncthreads();
  int before = 0;
  total = 0;
  for (int w = 0; w < warps; ++w) {
    const int n = sums[w];
    if (w < warp) before += n;
    total += n;
  }
  __syncthreads();
  return before + s - x;
}

// Finds this CTA's piece (ctl->start and its first unit); all threads.  `places`: of the line after each
// unit's tiles.  Returns the CTAs that have a piece.
template <class P>
__device__ __forceinline__ int find_piece(const P& p, Ctl* ctl, int block_tokens, int places) {
  const int items = p.seqs * p.blocks;
  int total = 0, at = 0;
  Unit u;
  u.tiles = -places;
  for (int e0 = 0; e0 < items; e0 += blockDim.x) {
    const int e = e0 + threadIdx.x;
    u.tiles = -places;
    if (e < items) u = unit_of(p, e, block_tokens);
    int sum;
    at = total + block_exclusive((u.tiles + places) * p.kv_heads, ctl->sums, sum);
    total += sum;
  }
  const int ctas = min(static_cast<int>(gridDim.x), total);
  if (static_cast<int>(blockIdx.x) >= ctas) return ctas;
  const int begin = piece_start(blockIdx.x, total, ctas);
  int seen = 0;
  for (int e0 = 0; e0 < items; e0 += blockDim.x) {
    const int e = e0 + threadIdx.x;
    if (items > static_cast<int>(blockDim.x)) {
      u.tiles = -places;
      if (e < items) u = unit_of(p, e, block_tokens);
      int sum;
      at = seen + block_exclusive((u.tiles + places) * p.kv_heads, ctl->sums, sum);
      seen += sum;
    }
    const int length = u.tiles + places;
    if (at <= begin && begin < at + length * p.kv_heads) {
      const int head = quotient(begin - at, length);
      ctl->unit = u;
      ctl->start[0] = e;
      ctl->start[1] = head;
      ctl->start[2] = begin - at - head * length;
      ctl->start[3] = piece_start(blockIdx.x + 1, total, ctas) - begin;
      ctl->start[4] = total;
    }
  }
  return ctas;
}

// The tiles of a CTA in order; every role walks its own copy.
struct Walk {
  int item, kv_head;
  int place, left;  // where the piece begins in this unit's stretch of the line; places left from there
  Unit u;
  int a0, a1;  // this unit's tiles in this CTA

  // The first unit of the piece with tiles in it; false when it has none.
  template <class P>
  __device__ __forceinline__ bool begin(const P& p, const Ctl* ctl, int block_tokens, int places) {
    item = ctl->start[0];
    kv_head = ctl->start[1];
    place = ctl->start[2];
    left = ctl->start[3];
    u = ctl->unit;
    a0 = place;
    a1 = p.whole ? (a0 > 0 ? a0 : u.tiles) : min(u.tiles, a0 + left);
    return a0 < a1 || next(p, block_tokens, places);
  }
  template <class P>
  __device__ __forceinline__ bool next(const P& p, int block_tokens, int places) {
    left -= u.tiles + places - place;
    if (left <= 0) return false;
    if (++kv_head == p.kv_heads) {
      kv_head = 0;
      u = unit_of(p, ++item, block_tokens);
    }
    place = a0 = 0;
    a1 = p.whole ? u.tiles : min(u.tiles, left);
    return true;
  }
};

// ------------------------------------------------------------------------------ PTX

__device__ __forceinline__ void tma_load_4d(void* smem_dst, const CUtensorMap* map, uint64_t* bar, int32_t x, int32_t y,
                                            int32_t z, int32_t w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::
          "r"(smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}

__device__ __forceinline__ void tmem_st(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void tmem_st(uint32_t taddr, const uint32_t (&r)[16]) { tmem_st_32x32b_x16(taddr, r); }

// kind::f16 instruction descriptor (see umma_idesc_f16_f32) with both operands fp16 or both bf16.
template <bool BF16>
__host__ __device__ constexpr uint32_t idesc(uint32_t m, uint32_t n, uint32_t b_mn_major) {
  return umma_idesc_f16_f32(m, n, 0, b_mn_major) | (BF16 ? (1u << 7) | (1u << 10) : 0u);
}

// umma_desc_sw128 as its low word and a constant high word: the descriptor of an operand `bytes` further on
// is one 32-bit add away (shared memory ends below 2^18 bytes, so the 14-bit address field does not
// overflow), which keeps the issuing thread ahead of the softmax.
__device__ __forceinline__ uint32_t desc_low(uint32_t smem_addr, uint32_t lbo_bytes) {
  return (smem_addr >> 4) | (lbo_bytes >> 4) << 16;
}
__device__ __forceinline__ uint64_t desc_at(uint32_t low, uint32_t bytes) {
  constexpr uint32_t high = (1024u >> 4) | 1u << 14 | 2u << 29;  // stride 1024 bytes, version 1, 128-byte swizzle
  return static_cast<uint64_t>(high) << 32 | (low + (bytes >> 4));
}

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (BF16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

// Three-operand max that returns NaN when an operand is NaN.
__device__ __forceinline__ float fmax3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// The x low bits of 64 (none for x <= 0, all for x >= 64).
__device__ __forceinline__ uint64_t low_bits(int x) {
  return x <= 0 ? 0ull : x >= 64 ? ~0ull : (1ull << x) - 1;
}

// Which of the 64 keys from k0 on the row sees.
template <class P>
__device__ __forceinline__ uint64_t visible(const P& p, const Unit& u, int t, int k0) {
  const int prefix = u.len - u.live;
  if (!p.tree) {
    const int pos = prefix + t;
    return low_bits(pos + 1 - k0) & (~low_bits(pos - p.window + 1 - k0) | low_bits(p.sinks - k0));
  }
  uint64_t bits = low_bits(prefix - k0);
  if (k0 + 64 > prefix) {
    const uint32_t* row = p.tree + u.b * p.tree_stride + static_cast<int64_t>(t) * p.words;
    const int s0 = k0 - prefix;  // draft at bit 0
    const int w0 = s0 >> 5;      // floor
    uint64_t lo = 0, hi = 0;     // words w0 .. w0 + 2
    if (w0 >= 0 && w0 < p.words) lo = row[w0];
    if (w0 + 1 >= 0 && w0 + 1 < p.words) lo |= static_cast<uint64_t>(row[w0 + 1]) << 32;
    if (w0 + 2 >= 0 && w0 + 2 < p.words) hi = row[w0 + 2];
    const int sh = s0 & 31;
    uint64_t drafts = lo >> sh;
    if (sh) drafts |= hi << (64 - sh);
    bits |= drafts & ~low_bits(prefix - k0);
  }
  return bits & low_bits(u.len - k0);
}

__device__ __forceinline__ uint64_t or_sync(uint64_t x) {  // of a whole warp
  return static_cast<uint64_t>(__reduce_or_sync(0xffffffffu, static_cast<uint32_t>(x >> 32))) << 32 |
         __reduce_or_sync(0xffffffffu, static_cast<uint32_t>(x));
}

// Which of the 64 keys from k0 on some token of the unit sees (window: all from its first token's first to the
// sequence's end).  One warp.
template <class P>
__device__ __forceinline__ uint64_t unit_sees(const P& p, const Unit& u, int block_tokens, int k0) {
  if (!p.tree) return low_bits(u.len - k0) & (~low_bits(window_from(p, u) - k0) | low_bits(p.sinks - k0));
  uint64_t bits = low_bits(u.len - u.live - k0);
  if (k0 + 64 > u.len - u.live) {
    for (int t = u.t0 + (threadIdx.x & 31); t < min(u.t0 + block_tokens, u.live); t += 32) bits |= visible(p, u, t, k0);
    bits = or_sync(bits);
  }
  return bits;
}

// ------------------------------------------------------------------------------ kernel

template <int D, int NT, int KS, bool BF16, bool SPLIT>
__global__ void __launch_bounds__(THREADS, 1)
    cache_attn_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                      const __grid_constant__ CUtensorMap tv, const __grid_constant__ CUtensorMap tv8,
                      const __grid_constant__ CUtensorMap tv1, const AttnParams<SPLIT> p) {
  using C = Shape<D, NT>;
  constexpr int BN = C::BN, NB = C::BUFFERS;
  // Hand P over in halves: with 128 keys and no key groups (which finish together).
  constexpr int HALVES = KS == 1 && BN == 128 ? 2 : 1;
  constexpr int M = KS == 1 ? BM : 64;  // rows of an MMA; 64 rows lie in the first half of each 32 TMEM lanes
  constexpr int KC = BN / KS;           // keys of a tile per key group
  constexpr int GROUP_ROWS = BM / KS;   // TMEM lanes per key group
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Ctl* ctl = reinterpret_cast<Ctl*>(smem + C::CTL_OFF);
  volatile int* abort_flag = &ctl->abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int block_tokens = NT * p.tile_tokens;

  pdl_trigger();
  if (threadIdx.x < (KS > 1 ? 3 : 5))
    prefetch_tensormap(threadIdx.x == 0   ? &tq
                       : threadIdx.x == 1 ? &tk
                       : threadIdx.x == 2 ? &tv
                       : threadIdx.x == 3 ? &tv8
                                          : &tv1);
  if (warp == MMA_WARP) {
    tmem_alloc(&ctl->tmem_base, TMEM_COLS);
    tmem_relinquish();
  } else if (threadIdx.x == 0) {
    mbar_init(&ctl->q_full, 1);
    mbar_init(&ctl->q_empty, 1);
    for (int s = 0; s < kMaxStages; ++s) {
      mbar_init(&ctl->k_full[s], 1);
      mbar_init(&ctl->k_empty[s], 1);
      mbar_init(&ctl->v_full[s], 1);
      mbar_init(&ctl->v_empty[s], 1);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&ctl->s_full[i], 1);
      mbar_init(&ctl->p_half[i], 4);
      mbar_init(&ctl->p_ready[i], 4);
      mbar_init(&ctl->pv_done[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&ctl->groups[i], 4);
      mbar_init(&ctl->drain[i], 1);
    }
    mbar_init(&ctl->o_free, 8);
    mbar_init(&ctl->streams, 8);
    ctl->abort = 0;
    fence_mbar_init();
  }
  if (p.tile_keys < BN) {
    // Rows of the V stages that no page reaches: zero once, no copy writes them.
    const int spare = (BN - p.tile_keys) * 8;  // 16-byte units per 64-column half
    for (int e = threadIdx.x; e < C::V_STAGES * (D / 64) * spare; e += blockDim.x) {
      const int half = e / spare, at = e % spare;
      *reinterpret_cast<uint4*>(smem + C::V_OFF + half * (BN * 128) + p.tile_keys * 128 + at * 16) =
          make_uint4(0, 0, 0, 0);
    }
    fence_proxy_async_smem();
  }
  pdl_wait();
  constexpr int PLACES = kUnitPlaces<NT>;
  const int ctas = find_piece(p, ctl, block_tokens, PLACES);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (static_cast<int>(blockIdx.x) >= ctas || !Walk().begin(p, ctl, block_tokens, PLACES)) {  // no tiles
    if (threadIdx.x == 0) p.head[blockIdx.x] = make_int4(0, 0, -1, 0);
    if (warp == MMA_WARP) tmem_dealloc(ctl->tmem_base, TMEM_COLS);
    return;
  }
  const uint32_t tmem = ctl->tmem_base;

  if (warp >= SOFTMAX_WARPS) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(REGS_OTHER) : "memory");
    // One thread: the unit's Q, as row tiles (NT = 2) or copies for the key groups.
    auto load_q = [&](const Walk& w) {
      mbar_arrive_expect_tx(&ctl->q_full, static_cast<uint32_t>(NT * KS * (D / 64) * p.tile_tokens * p.group * 128));
#pragma unroll
      for (int i = 0; i < NT * KS; ++i)
#pragma unroll
        for (int d = 0; d < D / 64; ++d)
          tma_load_4d(smem + (NT == 2 ? i * C::Q_BYTES : i * (M / KS) * 128) + d * (M * 128), &tq, &ctl->q_full, d * 64,
                      w.kv_head * p.group, w.u.t0 + (NT == 2 ? i * p.tile_tokens : 0), w.u.b);
    };
    if (warp == K_WARP || warp == V_WARP) {
      // ---------------------------------------------- K loads, V loads: one warp each, a lane per page
      // K frees its stages a softmax earlier than V does; one warp for both would hold K back.
      // Lane 0 waits for the whole warp, so that either every lane issues its boxes or none does.
      const bool is_v = warp == V_WARP;
      uint64_t* full = is_v ? ctl->v_full : ctl->k_full;
      uint64_t* empty = is_v ? ctl->v_empty : ctl->k_empty;
      const int count = is_v ? C::V_STAGES : C::K_STAGES;
      const CUtensorMap* map = is_v ? &tv : &tk;
      uint8_t* stages = smem + (is_v ? C::V_OFF : C::K_OFF);
      const int boxes = p.tile_pages;
      const int box_keys = p.tile_keys / boxes;
      const int box_bytes = box_keys * 128;  // one page's rows of one 64-column half
      const uint32_t tile_bytes = static_cast<uint32_t>(boxes * box_bytes * (D / 64));
      // The table is read for several tiles at once, a batch ahead: a lane per page.
      const int batch = quotient(32, boxes), lane_tile = quotient(lane, boxes), lane_box = lane - lane_tile * boxes;
      bool ok = true;
      Walk w;
      w.begin(p, ctl, block_tokens, PLACES);
      Ring ring;
      int issued = 0;
      do {
        const int lo = p.tree ? 0 : window_from(p, w.u);
        const int32_t* row = p.table + w.u.b * p.table_stride;
        // A page that the unit sees nothing of, or that is not there, reads as zeros (the tensor
        // map fills what lies outside it), so a page given back or never written is not touched.
        auto pages_from = [&](int a) -> int {  // of `batch` tiles from a on, one per lane
          const int k0 = tile_key(p, w.u, a + lane_tile) + lane_box * box_keys;
          const int j = p.page_shift >= 0 ? k0 >> p.page_shift : k0 / p.page_size;
          if (lane_tile >= batch || a + lane_tile >= w.a1 || j >= p.max_pages || k0 >= w.u.len ||
              (k0 + box_keys <= lo && k0 >= p.sinks))
            return -1;
          return row[j];
        };
        int pages = pages_from(w.a0), pages_next = pages_from(w.a0 + batch), at = 0;
        // Tiles that may be seen in part: from here on, and the sinks' last and the window's first.
        const int part_from = KS > 1 || !is_v ? INT_MAX : p.tree ? tile_index(p, w.u.len - w.u.live) : w.u.tiles - 1;
        const int part_at = KS > 1 || !is_v || p.tree ? INT_MIN : w.u.sink_tiles - 1;
        for (int a = w.a0; a < w.a1; ++a, ++at) {
          const int s = ring.s;
          if (at == batch) {
            at = 0;
            pages = pages_next;
            pages_next = pages_from(a + batch);
          }
          const int page = __shfl_sync(0xffffffffu, pages, (at * boxes + lane) & 31);
          int y = 0;  // row of the page
          if (p.page_size > p.tile_keys) {
            const int k0 = tile_key(p, w.u, a);
            y = p.page_shift >= 0 ? k0 & (p.page_size - 1) : k0 % p.page_size;
          }
          const bool in_part =
              KS == 1 && (a >= part_from || static_cast<unsigned>(a) - static_cast<unsigned>(part_at) < 2u) && may_be_unseen(p, w.u, a);
          uint64_t seen[BN / 64] = {};
          if (in_part) {
#pragma unroll
            for (int ch = 0; ch < BN / 64; ++ch) seen[ch] = unit_sees(p, w.u, block_tokens, tile_key(p, w.u, a) + ch * 64);
          }
          ok = lane != 0 || wait_bounded(&empty[s], ring.phase ^ 1, p.wait_limit, abort_flag);
          ok = __shfl_sync(0xffffffffu, ok, 0);
          if (!ok) break;
          if (lane == 0) mbar_arrive_expect_tx(&full[s], tile_bytes);
          __syncwarp();
          uint8_t* to = stages + s * C::KV_BYTES;
          uint32_t in_eights = 0;  // boxes that are loaded 8 rows at a time
          if (in_part) {
            // Lane l: rows 8 l to 8 l + 7, if the tile has them, of box `box`, their page's row y8.
            const int box = quotient(lane * 8, box_keys);
            const int page8 = __shfl_sync(0xffffffffu, pages, (at * boxes + box) & 31), y8 = y + lane * 8 - box * box_keys;
            const uint32_t rows = static_cast<uint32_t>((lane < 8 ? seen[0] : seen[BN / 64 - 1]) >> (lane & 7) * 8) & 0xff;
            const bool has = lane < p.tile_keys / 8 && page8 != -1;
            in_eights = __reduce_or_sync(0xffffffffu, has && rows != 0xff ? 1u << box : 0u);
            const bool mine = has && (in_eights >> box & 1);
            if (mine && (rows == 0 || rows == 0xff)) {
#pragma unroll
              for (int d = 0; d < D / 64; ++d)
                tma_load_4d(to + lane * 1024 + d * (BN * 128), &tv8, &full[s], d * 64, w.kv_head, y8, rows ? page8 : -1);
            }
#pragma unroll 1
            for (uint32_t left = __ballot_sync(0xffffffffu, mine && rows != 0 && rows != 0xff); left; left &= left - 1) {
              const int from = __ffs(left) - 1;
              const uint32_t which = __shfl_sync(0xffffffffu, rows, from);
              const int page1 = __shfl_sync(0xffffffffu, page8, from), y1 = __shfl_sync(0xffffffffu, y8, from) + lane;
              if (lane < 8) {
#pragma unroll
                for (int d = 0; d < D / 64; ++d)
                  tma_load_4d(to + (from * 8 + lane) * 128 + d * (BN * 128), &tv1, &full[s], d * 64, w.kv_head, y1,
                              which >> lane & 1 ? page1 : -1);
              }
            }
          }
          if (lane < boxes && !(in_eights >> lane & 1)) {
#pragma unroll
            for (int d = 0; d < D / 64; ++d)
              tma_load_4d(to + lane * box_bytes + d * (BN * 128), map, &full[s], d * 64, w.kv_head, y, page);
          }
          ++issued;
          ring.next(count);
        }
      } while (ok && w.next(p, block_tokens, PLACES));
      if (lane == 0) {
        if (!ok) give_up(ctl, NTL_STATUS_TMA_EMPTY_WAIT);
        // Every copy of this warp lands before the CTA exits.  (The MMA threads waited for all of them, unless one
        // gave up; that may be after this warp's last copy, so it waits whether or not its own waits held.)
        for (int j = max(0, issued - count); j < issued; ++j) {
          if (!wait_bounded(&full[j % count], (j / count) & 1, int64_t(1) << 24, nullptr))
            atomicCAS(&g_cache_attn_status, 0u, NTL_STATUS_DRAIN_WAIT);
        }
      }
    } else if (NT == 2 && warp == AUX_WARP) {
      // ---------------------------------------------- Q loads (one lane)
      if (lane == 0) {
        bool ok = true;
        Walk w;
        w.begin(p, ctl, block_tokens, PLACES);
        int n = 0;
        do {
          // The next unit's Q once the last Q K^T of the unit before retired.
          if (!(ok = n == 0 || wait_bounded(&ctl->q_empty, (n - 1) & 1, p.wait_limit, abort_flag))) break;
          load_q(w);
          ++n;
        } while (w.next(p, block_tokens, PLACES));
        if (!ok) give_up(ctl, NTL_STATUS_TMA_EMPTY_WAIT);
        // The MMA thread waits for each Q load; if it gave up, this thread does before the CTA exits.
        if (n > 0 && !wait_bounded(&ctl->q_full, (n - 1) & 1, int64_t(1) << 24, nullptr))
          atomicCAS(&g_cache_attn_status, 0u, NTL_STATUS_DRAIN_WAIT);
      }
    } else if (elect_one_lane()) {
      // ---------------------------------------------- MMA issue (one lane)
      constexpr uint32_t idesc_s = idesc<BF16>(M, BN, 0);  // B = K tile, K-major
      constexpr uint32_t idesc_o = idesc<BF16>(M, D, 1);   // B = V tile, N-major
      const uint32_t q_low = desc_low(smem_u32(smem), 16);
      const uint32_t k_low = desc_low(smem_u32(smem + C::K_OFF), 16);
      const uint32_t v_low = desc_low(smem_u32(smem + C::V_OFF), BN * 128);
      auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
        if (wait_bounded(bar, parity, p.wait_limit, abort_flag)) return true;
        give_up(ctl, NTL_STATUS_MMA_FULL_WAIT);
        return false;
      };
      bool ok = true;
      Walk w;
      w.begin(p, ctl, block_tokens, PLACES);
      Ring kr, vr;
      int g = 0;
      auto qk = [&](int i) {  // S buffer i = Q K^T
        const uint32_t q = q_low + (NT == 2 ? i : 0) * (C::Q_BYTES >> 4), k = k_low + kr.s * (C::KV_BYTES >> 4);
        tc_fence_after();
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
          tc_mma_f16_ss(tmem + C::S_COL(i), desc_at(q, (kk >> 2) * (M * 128) + (kk & 3) * 32),
                        desc_at(k, (kk >> 2) * (BN * 128) + (kk & 3) * 32), idesc_s, kk > 0 ? 1u : 0u);
        tc_commit(&ctl->s_full[i]);
      };
      // O_i += P V out of buffer `buf`, keys of one half (see HALVES); `add` 0 overwrites O.
      auto pv = [&](int i, int buf, int half, uint32_t add) {
        const uint32_t v = v_low + vr.s * (C::KV_BYTES >> 4);
        tc_fence_after();
#pragma unroll
        for (int kk = 0; kk < BN / 16 / HALVES; ++kk) {
          const uint32_t from = half * (BN / 16 / HALVES);
          tc_mma_f16_ts(tmem + C::O_COL(i), tmem + C::S_COL(buf) + (from + kk) * 8, desc_at(v, (from + kk) * 2048), idesc_o,
                        kk > 0 ? 1u : add);
        }
        if (half + 1 == HALVES) tc_commit(&ctl->pv_done[buf]);
      };
      if constexpr (NT == 1) {
        if (warp == MMA_WARP) {  // Q and Q K^T
          uint32_t q_phase = 0;
          load_q(w);
          do {
            if (!(ok = wait(&ctl->q_full, q_phase))) break;
            for (int a = w.a0; a < w.a1; ++a, ++g, kr.next(C::K_STAGES)) {
              // S buffer g % NB is free once P V of tile g - NB is complete.
              if (!(ok = (g < NB || wait(&ctl->pv_done[g % NB], (g / NB - 1) & 1)) && wait(&ctl->k_full[kr.s], kr.phase)))
                break;
              qk(g % NB);
              tc_commit(&ctl->k_empty[kr.s]);
            }
            if (!ok || !w.next(p, block_tokens, PLACES)) break;
            // The next unit's Q once this one's last Q K^T retired.
            tc_commit(&ctl->q_empty);
            if (!(ok = wait(&ctl->q_empty, q_phase))) break;
            load_q(w);
            q_phase ^= 1;
          } while (true);
          // Every Q load has landed before the CTA exits (this thread waited for it, unless it gave up).
          if (!ok && !wait_bounded(&ctl->q_full, q_phase, int64_t(1) << 24, nullptr))
            atomicCAS(&g_cache_attn_status, 0u, NTL_STATUS_DRAIN_WAIT);
        } else {  // P V
          int unit = 0;
          do {
            // O of the unit before has been read out, by both streams.
            if (unit > 0 && !(ok = wait(&ctl->o_free, (unit - 1) & 1))) break;
            for (int a = w.a0; a < w.a1; ++a, ++g, vr.next(C::V_STAGES)) {
              const int buf = g % NB;
              const uint32_t phase = (g / NB) & 1, add = a - w.a0 >= 2;  // each stream's first tile overwrites its O
              if (!(ok = wait(&ctl->v_full[vr.s], vr.phase))) break;
              if constexpr (HALVES == 2) {
                if (!(ok = wait(&ctl->p_half[buf], phase))) break;
                pv(g & 1, buf, 0, add);
              }
              if (!(ok = wait(&ctl->p_ready[buf], phase))) break;
              pv(g & 1, buf, HALVES - 1, HALVES == 2 ? 1u : add);
              tc_commit(&ctl->v_empty[vr.s]);
            }
            ++unit;
          } while (ok && w.next(p, block_tokens, PLACES));
        }
      } else {
        // Two cursors over the same tiles: Q K^T runs one tile ahead of P V, right after the P V that frees its
        // S, during the other row tile's softmax; a new unit's waits for loads that the end of this unit must
        // not wait for, and goes after it.
        Walk wq;
        wq.begin(p, ctl, block_tokens, PLACES);
        int aq = wq.a0;
        uint32_t q_phase = 0;
        bool more = true;
        auto qk_ready = [&]() -> bool {
          if (aq == wq.a0 && !wait(&ctl->q_full, q_phase)) return false;
          return wait(&ctl->k_full[kr.s], kr.phase);
        };
        auto qk_end = [&]() {  // after the second row tile's
          tc_commit(&ctl->k_empty[kr.s]);
          kr.next(C::K_STAGES);
          if (++aq == wq.a1) {
            tc_commit(&ctl->q_empty);
            more = wq.next(p, block_tokens, PLACES);
            aq = wq.a0;
            q_phase ^= 1;
          }
        };
        auto pv_both = [&](int i, uint32_t add) -> bool {
          if (!wait(&ctl->p_half[i], g & 1)) return false;
          pv(i, i, 0, add);
          if (!wait(&ctl->p_ready[i], g & 1)) return false;
          pv(i, i, 1, 1u);
          return true;
        };
        while ((ok = qk_ready())) {
          qk(0);
          qk(1);
          qk_end();
          for (int a = w.a0; a < w.a1; ++a, ++g, vr.next(C::V_STAGES)) {
            // V of this tile and K of the next have landed long before P is ready: only P is on the critical
            // path.
            const bool ahead = more && aq != wq.a0;
            const uint32_t add = a > w.a0;
            if (!(ok = wait(&ctl->v_full[vr.s], vr.phase) && (!ahead || qk_ready()) && pv_both(0, add))) break;
            if (ahead) qk(0);
            if (!(ok = pv_both(1, add))) break;
            tc_commit(&ctl->v_empty[vr.s]);
            if (ahead) {
              qk(1);
              qk_end();
            }
          }
          if (!ok || !w.next(p, block_tokens, PLACES)) break;
        }
      }
      // Every MMA retires before the CTA exits.  (The softmax waits for each, unless it gave up, which this thread may
      // not see.)
      uint64_t* drain = &ctl->drain[warp == MMA_WARP ? 0 : 1];
      tc_commit(drain);
      if (!wait_bounded(drain, 0, int64_t(1) << 24, nullptr))
        atomicCAS(&g_cache_attn_status, 0u, NTL_STATUS_DRAIN_WAIT);
    }
  } else {
    // ---------------------------------------------- softmax: one thread per row (and key group)
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(REGS_SOFTMAX) : "memory");
    const int i = warp >> 2;                       // stream
    const int row_lane = (warp & 3) * 32 + lane;   // TMEM lane
    const int group = row_lane / GROUP_ROWS;       // key group
    const int r = row_lane - group * GROUP_ROWS;   // row of the tile
    const int row_token = quotient(r, p.group), row_head = r - row_token * p.group;
    const int t_in_block = (NT == 2 ? i * p.tile_tokens : 0) + row_token;
    const bool in_tile = row_token < p.tile_tokens;
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t o_addr = tmem + lane_off + C::O_COL(i);
    const float c = p.c;
    int4 cut = make_int4(0, 0, -1, 0);
    bool ok = true;
    Walk w;
    w.begin(p, ctl, block_tokens, PLACES);
    int g0 = 0;  // tiles before this unit
    uint32_t units = 0, group_meets = 0, stream_meets = 0;
    // Several warps meet at a barrier: false when one of them gave up.
    auto meet = [&](uint64_t* bar, uint32_t& meets) -> bool {
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);
      return warp_wait(bar, meets++ & 1, p.wait_limit, abort_flag);
    };
    // Key groups: the stream's 128 threads write zeros over V rows of tile a that no row sees: past the sequence's end
    // and between the sinks and the window, 8 threads to a row; drafts, each warp those of its keys (`see`: of a lane's row).
    auto clear_unseen = [&](const Unit& u, int a, int g, uint64_t see) -> bool {
      if (!warp_wait(&ctl->v_full[g % C::V_STAGES], (g / C::V_STAGES) & 1, p.wait_limit, abort_flag)) return false;
      uint8_t* tile = smem + C::V_OFF + g % C::V_STAGES * C::KV_BYTES;
      const int k0 = tile_key(p, u, a);
      auto row_at = [&](int key) { return min(max(key - k0, 0), p.tile_keys); };
      int from = p.tree ? 0 : row_at(p.sinks), to = p.tree ? 0 : row_at(window_from(p, u));
#pragma unroll 1
      for (int k = 0; k < 2; ++k) {
#pragma unroll 2
        for (int e = from * 8 + row_lane; e < to * 8; e += 128)
#pragma unroll
          for (int half = 0; half < D / 64; ++half)
            *reinterpret_cast<uint4*>(tile + half * (BN * 128) + e * 16) = make_uint4(0, 0, 0, 0);
        from = row_at(u.len);
        to = p.tile_keys;
      }
      if (p.tree) {
        const int first = k0 + group * KC;
        const uint32_t drafts = static_cast<uint32_t>(low_bits(min(u.len - first, KC)) & ~low_bits(u.len - u.live - first));
        for (uint32_t left = drafts & ~__reduce_or_sync(0xffffffffu, static_cast<uint32_t>(see)); left; left &= left - 1) {
          const int row = group * KC + __ffs(left) - 1;
          if (row < p.tile_keys && lane < 8 * (D / 64))
            *reinterpret_cast<uint4*>(tile + (lane >> 3) * (BN * 128) + row * 128 + (lane & 7) * 16) = make_uint4(0, 0, 0, 0);
        }
      }
      fence_proxy_async_smem();
      return true;
    };
    do {
      const Unit& u = w.u;
      const int t = u.t0 + t_in_block;
      const bool live = in_tile && t < u.live;
      const bool any = KS > 1 ? u.t0 < u.live : __any_sync(0xffffffffu, live);
      // Tiles that every row of this row tile sees whole: [whole_from, whole_to).  (Tiles of sinks alone
      // are left to the masked path.)
      int whole_from = 0, whole_to = 0;
      if (!SPLIT && p.tile_keys == BN) {
        const int prefix = u.len - u.live;
        const int t_first = u.t0 + (NT == 2 ? i * p.tile_tokens : 0), t_last = min(t_first + p.tile_tokens, u.live) - 1;
        const int all_lo = p.tree ? 0 : max(prefix + t_last - p.window + 1, 0);
        const int all_hi = p.tree ? prefix : prefix + t_first + 1;
        whole_from = u.sink_tiles + max((all_lo + BN - 1) / BN - u.first, 0);
        whole_to = u.sink_tiles + all_hi / BN - u.first;
      }
      float m = -INFINITY, l = 0.0f;
      // This stream's tiles: every one, or (NT = 1) those of its parity.
      constexpr int STEP = NT == 1 ? 2 : 1;
      const int a_first = w.a0 + (NT == 1 ? (g0 ^ i) & 1 : 0);
      if (!any) {  // rows past the end: this warp only keeps step
        for (int a = a_first; a < w.a1; a += STEP) {
          const int g = g0 + a - w.a0, buf = NT == 2 ? i : g % NB;
          if (!(ok = warp_wait(&ctl->s_full[buf], (NT == 2 ? g : g / NB) & 1, p.wait_limit, abort_flag))) break;
          if (lane == 0) {
            if (HALVES == 2) mbar_arrive(&ctl->p_half[buf]);
            mbar_arrive(&ctl->p_ready[buf]);
          }
        }
      } else {
        for (int a = a_first; a < w.a1; a += STEP) {
          const int g = g0 + a - w.a0, buf = NT == 2 ? i : g % NB;
          const uint32_t s_addr = tmem + lane_off + C::S_COL(buf);
          // What the row sees, worked out while S is on its way.
          const bool masked = a < whole_from || a >= whole_to;
          uint64_t see[(KC + 63) / 64] = {};
          if (masked && live) {
            const int k0 = tile_key(p, u, a), from = group * KC, span = tile_span(p, k0) - from;
#pragma unroll
            for (int ch = 0; ch < (KC + 63) / 64; ++ch)
              see[ch] = visible(p, u, t, k0 + from + ch * 64) & low_bits(span - ch * 64);
          }
          if (!(ok = warp_wait(&ctl->s_full[buf], (NT == 2 ? g : g / NB) & 1, p.wait_limit, abort_flag))) break;
          if constexpr (KS > 1) {
            // Not before S is there: until then the barrier of V may be a lap behind.
            if (masked && may_be_unseen(p, u, a) && !(ok = clear_unseen(u, a, g, see[0]))) break;
          }
          tc_fence_after();
          uint32_t sv[KC];
          if constexpr (KC == 16) {
            tmem_ld_32x32b_x16(s_addr + group * KC, sv);
          } else {
#pragma unroll
            for (int ch = 0; ch < KC / 32; ++ch)
              tmem_ld_32x32b_x32(s_addr + group * KC + ch * 32, *reinterpret_cast<uint32_t(*)[32]>(sv + ch * 32));
          }
          tc_wait_ld();
          if (__builtin_expect(masked, 0)) {
#pragma unroll
            for (int e = 0; e < KC; ++e)
              if (!(see[e / 64] >> (e % 64) & 1)) sv[e] = __float_as_uint(-INFINITY);
          }
          float top;
          {
            float x[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int e = 0; e < KC; e += 8) {
              x[0] = fmax3_nan(x[0], __uint_as_float(sv[e]), __uint_as_float(sv[e + 1]));
              x[1] = fmax3_nan(x[1], __uint_as_float(sv[e + 2]), __uint_as_float(sv[e + 3]));
              x[2] = fmax3_nan(x[2], __uint_as_float(sv[e + 4]), __uint_as_float(sv[e + 5]));
              x[3] = fmax3_nan(x[3], __uint_as_float(sv[e + 6]), __uint_as_float(sv[e + 7]));
            }
            top = fmax3_nan(fmax3_nan(x[0], x[1], x[2]), x[3], x[3]);
          }
          float scale_old = 1.0f;
          bool moved = false;
          if (!(top < INFINITY)) {  // a NaN or +inf score: the row's softmax is NaN
            l = __uint_as_float(0x7fffffffu);
            top = m;
          }
          if (m == -INFINITY) {
            m = top;  // nothing seen so far: o and l are zero (or not begun)
          } else if (live && (top - m) * c > kRescaleLog2) {
            scale_old = ex2_approx((m - top) * c);
            m = top;
            moved = true;
          }
          const bool rescale = __any_sync(0xffffffffu, moved);
          if (__builtin_expect(rescale, 0)) {
            // O is stable once P V of the stream's tile before is complete.  (NT = 2 issued S after it.)
            if (NT == 1 && !(ok = warp_wait(&ctl->pv_done[(g - 2) % NB], ((g - 2) / NB) & 1, p.wait_limit, abort_flag))) break;
            tc_fence_after();
#pragma unroll 1
            for (int ch = 0; ch < D / 32; ++ch) {
              uint32_t o[32];
              tmem_ld_32x32b_x32(o_addr + ch * 32, o);
              tc_wait_ld();
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * scale_old);
              tmem_st_32x32b_x32(o_addr + ch * 32, o);
            }
          }
          const float shift = m == -INFINITY ? 0.0f : -m * c;
          const uint64_t c2 = f2_make(c, c), shift2 = f2_make(shift, shift);
          uint64_t acc[2] = {0ull, 0ull};
          // This group's exponentials over its own 16-bit columns of the tile; the others' are zero
          // in these lanes, so that P V adds up this group's keys alone.
          constexpr int PC = KC < 32 ? KC / 2 : 16;  // packed columns per store
#pragma unroll
          for (int ch = 0; ch < KC / (2 * PC); ++ch) {
            uint32_t packed[PC];
#pragma unroll
            for (int e = 0; e < PC; ++e) {
              const int k = ch * 2 * PC + 2 * e;
              float x0, x1;
              f2_split(f2_fma(f2_make(__uint_as_float(sv[k]), __uint_as_float(sv[k + 1])), c2, shift2), x0, x1);
              const float p0 = ex2_approx(x0), p1 = ex2_approx(x1);
              acc[e & 1] = f2_add(acc[e & 1], f2_make(p0, p1));
              packed[e] = pack2<BF16>(p0, p1);
            }
            tmem_st(s_addr + group * (KC / 2) + ch * PC, packed);
            if (HALVES == 2 && ch == KC / (4 * PC) - 1) {  // the first half of the keys may be multiplied
              tc_wait_st();
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(&ctl->p_half[buf]);
            }
          }
          if constexpr (KS > 1) {
            uint32_t zero[PC] = {};
#pragma unroll
            for (int j = 1; j < KS; ++j) tmem_st(s_addr + ((group + j) % KS) * (KC / 2), zero);
          }
          float s0, s1;
          f2_split(f2_add(acc[0], acc[1]), s0, s1);
          l = __fmaf_rn(l, scale_old, s0 + s1);
          tc_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&ctl->p_ready[buf]);
        }
      }
      if (!ok) break;
      const int n = w.a1 - w.a0;
      const int g_last = g0 + (NT == 1 ? ((n - 1 - ((g0 ^ i) & 1)) | 1) - 1 + ((g0 ^ i) & 1) : n - 1);  // of this stream
      g0 += n;
      // Rows that see nothing wait too: P V of the unit must not fall two units behind (it waits for o_free by parity).
      if (a_first < w.a1 &&
          !(ok = warp_wait(&ctl->pv_done[NT == 2 ? i : g_last % NB], (NT == 2 ? g_last : g_last / NB) & 1,
                           p.wait_limit, abort_flag)))
        break;
      tc_fence_after();
      const bool done = w.a0 == 0 && w.a1 == u.tiles;
      const bool here = in_tile && t < p.tokens;  // the output has this row
      const int64_t out_row =
          (static_cast<int64_t>(u.b) * p.tokens + t) * p.heads + w.kv_head * p.group + row_head;
      if (!done && w.a0 == 0 && threadIdx.x == 0) {
        const int total = ctl->start[4];
        const int unit_start = piece_start(blockIdx.x + 1, total, ctas) - w.left;
        cut = make_int4(w.item, w.kv_head, piece_of(unit_start + u.tiles - 1, total, ctas), u.live);
      }
      const int64_t slot_row = (2 * static_cast<int64_t>(blockIdx.x) + (w.a0 == 0 ? 1 : 0)) * p.rows + (NT == 2 ? i * BM : 0);
      // O leaves through shared memory, so that store instructions write whole sectors (a thread writing
      // its own row 16 bytes at a time took 5 to 9 us per 108 rows).  A unit that is cut leaves its sums
      // and (m, l) in the workspace.  NT = 1: both streams' O are in this warp's lanes; each stream writes
      // half of the columns of weight0 * O_0 + weight1 * O_1.
      float weight[2] = {1.0f, 0.0f};
      uint32_t o_from[2] = {o_addr, o_addr};
      float mc = m == -INFINITY ? m : m * c, sum = l;
      if constexpr (NT == 1) {
        // Units that nothing sees meet too: a stream that ran ahead would count twice in o_free.
        float2(*ml)[BM] = ctl->ml[units & 1];
        ml[i][row_lane] = make_float2(mc, l);
        tc_fence_before();
        if (!(ok = meet(&ctl->streams, stream_meets))) break;
        tc_fence_after();
        mc = -INFINITY;
        sum = 0.0f;
#pragma unroll
        for (int k = 0; k < KS; ++k)
          mc = fmaxf(mc, fmaxf(ml[0][k * GROUP_ROWS + r].x, ml[1][k * GROUP_ROWS + r].x));
        // 2^(m - max m), 0 for a part that saw nothing (m = -inf; l is 0, or NaN for NaN scores and stays it).
        const float top = mc == -INFINITY ? 0.0f : mc;
        auto weigh = [&](float2 x) { return ex2_approx(x.x - top); };
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float2 x = ml[j][k * GROUP_ROWS + r];
            sum += weigh(x) * x.y;
          }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          // A stream without a tile in this unit weighs nothing; the other's O stands in for what it has not.
          const bool has = n > (((g0 - n) ^ j) & 1);
          o_from[j] = tmem + lane_off + (has ? C::O_COL(j) : C::O_COL(1 - j));
          weight[j] = weigh(ml[j][row_lane]);
        }
      }
      ++units;
      if (done) {
        const float inv = sum > 0.0f ? __fdividef(1.0f, sum) : sum == sum ? 0.0f : sum;  // NaN stays
        weight[0] *= inv;
        weight[1] *= inv;
      } else if (live && group == 0 && (NT == 2 || i == 0)) {
        p.part_ml[slot_row + r] = make_float2(mc, sum);
      }
      if constexpr (KS > 1) {
        if (any) {
          // Each row's key groups add up.  (Code that runs once per unit costs ~8 cycles an instruction, so this part
          // divides nothing that it need not: 1024 x 1 token, window 128: 263 -> 250 us.)  16 columns of every live row and group are staged at a time, or
          // more where few rows leave room.
          const int rows = min(p.tile_tokens, u.live - u.t0) * p.group;
          const int at_once = D == 64 || rows <= 8 ? D / 32 : 2;
          const int shift = rows <= 4 ? 2 : rows <= 8 ? 3 : 4;  // rows rounded up
          uint8_t* stage = smem + C::OUT_OFF + i * (4 * 32 * kOutRow);
#pragma unroll 1
          for (int c0 = 0; c0 < D / 32 && ok; c0 += at_once) {
            const int chunks = min(at_once, D / 32 - c0);
            // The lines before have been read.  (Those of the unit before: the warps have met since.)
            if (c0 > 0 && !(ok = meet(&ctl->groups[i], group_meets))) break;
#pragma unroll 1
            for (int ch = 0; ch < chunks; ++ch) {
              const uint32_t column = i * (D / 2) + (c0 + ch) * 16;
              uint32_t o[2][16];
#pragma unroll
              for (int j = 0; j < 2; ++j) tmem_ld_32x32b_x16(o_from[j] + column, o[j]);
              tc_wait_ld();
              if (r < rows) {
                float4* to = reinterpret_cast<float4*>(stage + ((ch * KS + group) * rows + r) * kOutRow);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  float x[4];
#pragma unroll
                  for (int k = 0; k < 4; ++k)
                    x[k] = __uint_as_float(o[0][4 * e + k]) * weight[0] + __uint_as_float(o[1][4 * e + k]) * weight[1];
                  to[e] = make_float4(x[0], x[1], x[2], x[3]);
                }
              }
            }
            if (!(ok = meet(&ctl->groups[i], group_meets))) break;
            // 4 columns of a row per thread and round
#pragma unroll 1
            for (int e = row_lane; e < chunks << (shift + 2); e += 128) {
              const int ch = e >> (shift + 2), row = (e >> 2) - (ch << shift);
              if (row >= rows) continue;
              float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
              for (int k = 0; k < KS; ++k) {
                const float4 y =
                    *reinterpret_cast<const float4*>(stage + ((ch * KS + k) * rows + row) * kOutRow + (e & 3) * 16);
                x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w;
              }
              const int column = i * (D / 2) + (c0 + ch) * 16 + (e & 3) * 4;
              if (done) {
                const int token = row < p.group ? 0 : quotient(row, p.group);
                const int64_t to = (static_cast<int64_t>(u.b) * p.tokens + u.t0 + token) * p.heads +
                                   w.kv_head * p.group + row - token * p.group;
                *reinterpret_cast<uint2*>(p.o + to * D + column) = make_uint2(pack2<BF16>(x.x, x.y), pack2<BF16>(x.z, x.w));
              } else {
                *reinterpret_cast<float4*>(p.part + (slot_row + row) * D + column) = x;
              }
            }
          }
          if (!ok) break;
        }
      } else if (any) {
        // Quad n of a warp writes 64 bytes of row 8 e + n.
        constexpr int CHUNKS = NT == 1 ? D / 64 : D / 32;  // of 32 columns
        const int column0 = NT == 1 ? i * (D / 2) : 0;
        uint8_t* stage = smem + C::OUT_OFF + warp * 32 * kOutRow;
        uint8_t* to[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int row = 8 * e + (lane >> 2);
          const int64_t at = __shfl_sync(0xffffffffu, out_row, row);
          const bool row_live = __shfl_sync(0xffffffffu, static_cast<int>(live), row);
          to[e] = !row_live ? nullptr
                  : done    ? reinterpret_cast<uint8_t*>(p.o + at * D + column0)
                            : reinterpret_cast<uint8_t*>(p.part + (slot_row + (warp & 3) * 32 + row) * D + column0);
          if (to[e]) to[e] += (lane & 3) * 16;
        }
#pragma unroll 1
        for (int ch = 0; ch < CHUNKS; ++ch) {
          uint32_t o[32];
          if constexpr (NT == 2) {
            tmem_ld_32x32b_x32(o_addr + ch * 32, o);
            tc_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * weight[0]);
          } else {
#pragma unroll
            for (int part = 0; part < 2; ++part) {
              uint32_t x[2][16];
#pragma unroll
              for (int j = 0; j < 2; ++j) tmem_ld_32x32b_x16(o_from[j] + column0 + ch * 32 + part * 16, x[j]);
              tc_wait_ld();
#pragma unroll
              for (int e = 0; e < 16; ++e)
                o[part * 16 + e] =
                    __float_as_uint(__uint_as_float(x[0][e]) * weight[0] + __uint_as_float(x[1][e]) * weight[1]);
            }
          }
          if (done) {
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = pack2<BF16>(__uint_as_float(o[2 * e]), __uint_as_float(o[2 * e + 1]));
          }
#pragma unroll
          for (int half = 0; half < 2; ++half) {  // 16-bit: one half of 64 bytes; fp32: two
            if (half == 1 && done) break;
            __syncwarp();
#pragma unroll
            for (int e = 0; e < 4; ++e)
              *reinterpret_cast<uint4*>(stage + lane * kOutRow + e * 16) =
                  make_uint4(o[half * 16 + 4 * e], o[half * 16 + 4 * e + 1], o[half * 16 + 4 * e + 2], o[half * 16 + 4 * e + 3]);
            __syncwarp();
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (to[e]) {
                *reinterpret_cast<uint4*>(to[e]) =
                    *reinterpret_cast<const uint4*>(stage + (8 * e + (lane >> 2)) * kOutRow + (lane & 3) * 16);
                to[e] += 64;
              }
          }
        }
      }
      if constexpr (NT == 1) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctl->o_free);
      }
      if (done && here && !live && group == 0 && (NT == 2 || i == 0))
#pragma unroll 1
        for (int e = 0; e < D / 8; ++e) reinterpret_cast<uint4*>(p.o + out_row * D)[e] = make_uint4(0, 0, 0, 0);
      tc_fence_before();
    } while (w.next(p, block_tokens, PLACES));
    if (!ok) give_up(ctl, NTL_STATUS_SOFTMAX_WAIT);
    if (threadIdx.x == 0) p.head[blockIdx.x] = cut;
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == MMA_WARP) tmem_dealloc(tmem, TMEM_COLS);
}

// Adds up the parts of the unit that CTA blockIdx.x of the attention kernel began and did not end, in
// CTA order: weights 2^(m_s - max m), o = sum w_s o_s / sum w_s l_s.  A warp takes R rows: its lanes hold
// (m, l) of R rows x 32 / R parts, and 16 rows and parts of values are in flight at a time, so a warp
// costs a few memory latencies and not one per part and row.  R = 4 for units of over 64 rows (which
// few CTAs share: 27 -> 11 us for 147 cuts of 256 rows), 1 for the others (few rows, many parts).
constexpr int kJoinWarps = 4;

template <int D, int R, bool BF16>
__global__ void __launch_bounds__(kJoinWarps * 32) cache_attn_join(const AttnBase p, int row_tiles) {
  constexpr int kJoinRows = R, kJoinParts = 32 / R, kJoinAhead = 16 / R;
  constexpr int E = D / 32;
  using Vec = typename std::conditional<E == 4, float4, float2>::type;
  pdl_wait();
  const int4 cut = p.head[blockIdx.x];
  if (cut.z < 0) return;
  const int first = blockIdx.x, parts = cut.z - first + 1;
  const int row0 = (blockIdx.y * kJoinWarps + (threadIdx.x >> 5)) * kJoinRows, lane = threadIdx.x & 31;
  if (row0 >= p.rows) return;
  const int b = cut.x / p.blocks, t0 = (cut.x - b * p.blocks) * row_tiles * p.tile_tokens, live = cut.w;
  // Part s of the unit: CTA first's second slot, then the first slots of the CTAs after it.
  auto at = [&](int s, int row) { return (2ll * (first + s) + (s == 0)) * p.rows + row; };
  // Token of a row within the sequence, past every token if the tile has no such row.
  auto token_of = [&](int row) {
    const int r = row % BM, t = r / p.group;
    return t < p.tile_tokens && row < p.rows ? t0 + (row / BM) * p.tile_tokens + t : p.tokens;
  };
  int t[kJoinRows];
#pragma unroll
  for (int i = 0; i < kJoinRows; ++i) t[i] = token_of(row0 + i);
  float o[kJoinRows][E] = {}, m = -INFINITY, l = 0.0f;  // (m, l) of row lane / 8
  const int mine = row0 + lane / kJoinParts;
  for (int s0 = 0; s0 < parts; s0 += kJoinParts) {
    const int s = s0 + lane % kJoinParts;
    const float2 ml = s < parts && token_of(mine) < live ? p.part_ml[at(s, mine)] : make_float2(-INFINITY, 0.0f);
    float v[kJoinAhead][kJoinRows][E];
    auto fetch = [&](int j0) {
#pragma unroll
      for (int j = 0; j < kJoinAhead; ++j)
#pragma unroll
        for (int i = 0; i < kJoinRows; ++i)
          if (s0 + j0 + j < parts && t[i] < live)
            *reinterpret_cast<Vec*>(v[j][i]) =
                *reinterpret_cast<const Vec*>(p.part + at(s0 + j0 + j, row0 + i) * D + lane * E);
    };
    fetch(0);
    float top = fmaxf(m, ml.x);
#pragma unroll
    for (int d = kJoinParts / 2; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    const float old = m == -INFINITY ? 0.0f : ex2_approx(m - top);
    // A part that saw nothing has m = -inf and l = 0 (or NaN scores: l NaN).
    const float weight = ml.x == -INFINITY ? (ml.y == ml.y ? 0.0f : ml.y) : ex2_approx(ml.x - top);
    float sum = weight * ml.y;
#pragma unroll
    for (int d = kJoinParts / 2; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    l = l * old + sum;
    m = top;
#pragma unroll
    for (int i = 0; i < kJoinRows; ++i) {
      const float scale = __shfl_sync(0xffffffffu, old, i * kJoinParts);
#pragma unroll
      for (int e = 0; e < E; ++e) o[i][e] *= scale;
    }
    const int n = min(kJoinParts, parts - s0);
    for (int j0 = 0; j0 < n; j0 += kJoinAhead) {
      if (j0 > 0) fetch(j0);
#pragma unroll
      for (int j = 0; j < kJoinAhead; ++j)
#pragma unroll
        for (int i = 0; i < kJoinRows; ++i) {
          const float w = __shfl_sync(0xffffffffu, weight, i * kJoinParts + ((j0 + j) & (kJoinParts - 1)));
          if (j0 + j < n && t[i] < live)
#pragma unroll
            for (int e = 0; e < E; ++e) o[i][e] += w * v[j][i][e];
        }
    }
  }
  const float inv = l > 0.0f ? 1.0f / l : l == l ? 0.0f : l;
#pragma unroll
  for (int i = 0; i < kJoinRows; ++i) {
    const float scale = __shfl_sync(0xffffffffu, inv, i * kJoinParts);
    if (t[i] >= p.tokens) continue;
    uint32_t h[E / 2];
#pragma unroll
    for (int e = 0; e < E / 2; ++e) h[e] = pack2<BF16>(o[i][2 * e] * scale, o[i][2 * e + 1] * scale);
    const int head = cut.y * p.group + (row0 + i) % BM % p.group;
    uint16_t* out = p.o + ((static_cast<int64_t>(b) * p.tokens + t[i]) * p.heads + head) * D + lane * E;
    if constexpr (E == 4) {
      *reinterpret_cast<uint2*>(out) = make_uint2(h[0], h[1]);
    } else {
      *reinterpret_cast<uint32_t*>(out) = h[0];
    }
  }
}

// ------------------------------------------------------------------------------ host side

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(ptr);
  });
  return fn;
}

// A 4-D tensor of 16-bit values, strides in values (of dimensions 1 to 3), 128-byte swizzle.
int make_map(CUtensorMap* map, const char* what, const void* base, bool bf16, const int64_t (&dims)[4],
             const int64_t (&strides)[3], const int64_t (&box)[4]) {
  EncodeTiledFn fn = encode_fn();
  if (fn == nullptr) return ntl_fail(NTL_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable");
  cuuint64_t d[4], s[3];
  cuuint32_t b[4], one[4] = {1, 1, 1, 1};
  for (int i = 0; i < 4; ++i) {
    d[i] = static_cast<cuuint64_t>(dims[i]);
    b[i] = static_cast<cuuint32_t>(box[i]);
  }
  // The stride of a dimension of one is never used; any legal one will do.
  for (int i = 0; i < 3; ++i) s[i] = dims[i + 1] == 1 ? 16 : static_cast<cuuint64_t>(strides[i]) * 2;
  CUresult r = fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                  const_cast<void*>(base), d, s, b, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  dims[0] == 64 ? CU_TENSOR_MAP_L2_PROMOTION_L2_128B : CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return ntl_fail(NTL_ERR_CUDA, "%s: cuTensorMapEncodeTiled failed (%d)", what, int(r));
  return NTL_OK;
}

// Units of few tiles are not cut, which saves the join: its launch, and for two row tiles ~15 us where every CTA
// cuts one.  That many tiles in a row must not take longer: at most 8 of 64 keys (30 x 3 tokens, window 40: 13.4 ->
// 10.6 us; 18 x 1 token over 255 to 482 keys in pages of 8, 8 tiles: 12.8 -> 14.9), 6 of 128 keys; two row tiles as
// long as the CTA with the most units has at most 4 more tiles than the mean (4 x 512 tokens, window 512, 8 tiles,
// 1.7 units a CTA: 58.5 -> 41.4 us; 12 x 29 tokens over 351 to 672 keys, 6 tiles, 0.08 units: 20.4 -> 25.4).
bool few_tiles(int row_tiles, int tile_keys, int64_t tiles, int64_t units, int64_t sms) {
  if (tiles > (row_tiles == 1 && tile_keys > 64 ? 6 : 8)) return false;
  return row_tiles == 1 || ((units + sms - 1) / sms * sms - units) * tiles <= 4 * sms;
}

// What the sizes decide: the shape of CTA, the grid and the workspace.
struct Plan {
  int row_tiles, tile_tokens, blocks, tile_keys, tile_pages, page_tiles, rows, ctas;
  bool whole;
  uint64_t part_bytes, bytes;
};

// `sees`: keys that a token sees at most, besides the first `sinks`.
int make_plan(const char* what, const ntl_cache_t* c, const ntl_query_t* q, int64_t sees, int64_t sinks, Plan* plan) {
  const int64_t group = q->heads / c->kv_heads;
  Plan& n = *plan;
  n.row_tiles = q->tokens * group > BM ? 2 : 1;
  n.tile_tokens = static_cast<int>(BM / group < q->tokens ? BM / group : q->tokens);
  n.page_tiles = 0;
  const int64_t block_tokens = int64_t(n.row_tiles) * n.tile_tokens;
  const int64_t blocks = (q->tokens + block_tokens - 1) / block_tokens;
  const int most = n.row_tiles == 1 && c->head_dim == 128 ? Shape<128, 1>::BN : 128;
  if (c->page_size <= most) {
    n.tile_pages = static_cast<int>(most / c->page_size);
    n.tile_keys = static_cast<int>(n.tile_pages * c->page_size);
  } else {
    // As few tiles as possible, equal but for the last: pages of 136 are 3 tiles of 48, 48 and 40.  (Their largest
    // even part is 8 keys: 16 x 1 token over 4000 to 8000, 357 against 82 us.)
    const int64_t parts = (c->page_size + most - 1) / most;
    n.tile_pages = 1;
    n.tile_keys = static_cast<int>((c->page_size + parts * 8 - 1) / (parts * 8) * 8);
    if (parts * n.tile_keys != c->page_size) n.page_tiles = static_cast<int>(parts);
  }
  n.rows = n.row_tiles == 1 ? static_cast<int>(q->tokens * group) : 2 * BM;
  // Places of the line that one unit takes, at most.
  const int64_t tiles =
      (n.page_tiles ? q->max_pages * n.page_tiles : q->max_pages * c->page_size / n.tile_keys) + 2 + kUnitPlaces<1>;
  NTL_REQUIRE(q->seqs * blocks < (int64_t(1) << 31) / c->kv_heads / tiles, NTL_ERR_UNSUPPORTED,
              "%s: more than 2^31 tiles of keys", what);
  static_assert(kUnitPlaces<1> >= kUnitPlaces<2>, "the bound above");
  n.blocks = static_cast<int>(blocks);
  int sms = 0;
  if (int rc = ntl_num_sms(&sms)) return rc;
  const int64_t work = q->seqs * blocks * c->kv_heads * tiles;
  n.ctas = static_cast<int>(work < sms ? work : sms);
  const int64_t keys = q->max_pages * c->page_size, k = n.tile_keys;
  const int64_t span = sees + block_tokens - 1 < keys ? sees + block_tokens - 1 : keys;
  const int64_t all = (keys + k - 1) / k, seen = (span + k - 2) / k + 1 + (sinks < keys ? sinks + k - 1 : keys) / k;
  n.whole = few_tiles(n.row_tiles, n.tile_keys, seen < all ? seen : all, q->seqs * blocks * c->kv_heads, sms);
  n.part_bytes = static_cast<uint64_t>(2) * n.ctas * n.rows * c->head_dim * 4;
  n.bytes = n.part_bytes + static_cast<uint64_t>(2) * n.ctas * n.rows * 8 + static_cast<uint64_t>(n.ctas) * 16;
  n.bytes = (n.bytes + 15) / 16 * 16;
  return NTL_OK;
}

template <int D, int NT, int KS, bool BF16, bool SPLIT>
int launch_shape(const char* what, const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv,
                 const CUtensorMap& mv8, const CUtensorMap& mv1, const AttnBase& p, const Plan& n, cudaStream_t s) {
  static std::atomic<uint64_t> done_mask{0};
  auto kernel = cache_attn_kernel<D, NT, KS, BF16, SPLIT>;
  constexpr int smem = smem_bytes<D, NT>();
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return ntl_fail(NTL_ERR_CUDA, "cudaGetDevice failed");
  const uint64_t bit = dev < 64 ? uint64_t(1) << dev : 0;
  if (!(bit && (done_mask.load(std::memory_order_acquire) & bit))) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return ntl_fail(NTL_ERR_CUDA, "%s: cudaFuncSetAttribute: %s", what, cudaGetErrorString(e));
    // The register split must equal what the launch allocates, or the raising warps would wait for
    // registers forever: refuse a build whose register count differs.
    cudaFuncAttributes fa;
    if (cudaFuncGetAttributes(&fa, kernel) != cudaSuccess || fa.numRegs != REGS_LAUNCH)
      return ntl_fail(NTL_ERR_UNSUPPORTED, "%s: kernel compiled with %d registers, the split needs %d", what,
                      fa.numRegs, REGS_LAUNCH);
    done_mask.fetch_or(bit, std::memory_order_release);
  }
  cudaError_t e = ntl_launch_pdl(kernel, dim3(n.ctas), dim3(THREADS), smem, s, mq, mk, mv, mv8, mv1, AttnParams<SPLIT>{p});
  if (e != cudaSuccess) return ntl_fail(NTL_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
  ntl_note_launch();
  if (int rc = ntl_check_launch(what)) return rc;
  if (n.ctas == 1 || n.whole) return NTL_OK;  // no unit is cut
  const int join_rows = n.rows > 64 ? 4 : 1;
  const unsigned chunks = static_cast<unsigned>((n.rows + kJoinWarps * join_rows - 1) / (kJoinWarps * join_rows));
  e = ntl_launch_pdl(join_rows == 4 ? cache_attn_join<D, 4, BF16> : cache_attn_join<D, 1, BF16>,
                     dim3(n.ctas - 1, chunks), dim3(kJoinWarps * 32), 0, s, p, NT);
  if (e != cudaSuccess) return ntl_fail(NTL_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
  ntl_note_launch();
  return ntl_check_launch(what);
}

int launch(const char* what, const ntl_cache_t* c, const ntl_query_t* q, const uint32_t* tree, int64_t tree_stride,
           int64_t window, int64_t sinks, void* workspace, uint64_t workspace_bytes, cudaStream_t s) {
  Plan n;
  if (int rc = make_plan(what, c, q, tree ? int64_t(1) << 31 : window, tree ? 0 : sinks, &n)) return rc;
  NTL_REQUIRE(workspace && workspace_bytes >= n.bytes && ntl_aligned(workspace, 16), NTL_ERR_INVALID,
              "%s: workspace of %llu bytes, %llu needed (16-byte aligned)", what, (unsigned long long)workspace_bytes,
              (unsigned long long)n.bytes);
  const int64_t group = q->heads / c->kv_heads, dim = c->head_dim;
  const bool bf16 = c->dtype == NTL_BF16;
  CUtensorMap mq, mk, mv, mv8 = {}, mv1 = {};
  if (int rc = make_map(&mq, what, q->q, bf16, {dim, q->heads, q->tokens, q->seqs},
                        {q->head_stride, q->token_stride, q->seq_stride}, {64, group, n.tile_tokens, 1}))
    return rc;
  const int64_t dims[4] = {dim, c->kv_heads, c->page_size, c->pages};
  const int64_t strides[3] = {c->head_stride, c->row_stride, c->page_stride};
  const int64_t box[4] = {64, 1, n.tile_keys / n.tile_pages, 1};
  if (int rc = make_map(&mk, what, c->k, bf16, dims, strides, box)) return rc;
  if (int rc = make_map(&mv, what, c->v, bf16, dims, strides, box)) return rc;
  const bool key_groups = n.rows <= 16;
  if (!key_groups) {
    if (int rc = make_map(&mv8, what, c->v, bf16, dims, strides, {64, 1, 8, 1})) return rc;
    if (int rc = make_map(&mv1, what, c->v, bf16, dims, strides, {64, 1, 1, 1})) return rc;
  }
  AttnBase p = {};
  p.o = static_cast<uint16_t*>(q->o);
  p.table = q->table;
  p.lens = q->lens;
  p.q_lens = q->q_lens;
  p.tree = tree;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  p.part = reinterpret_cast<float*>(ws);
  p.part_ml = reinterpret_cast<float2*>(ws + n.part_bytes);
  p.head = reinterpret_cast<int4*>(ws + n.part_bytes + static_cast<uint64_t>(2) * n.ctas * n.rows * 8);
  p.table_stride = q->table_stride;
  p.tree_stride = tree_stride;
  p.seqs = static_cast<int>(q->seqs);
  p.tokens = static_cast<int>(q->tokens);
  p.heads = static_cast<int>(q->heads);
  p.kv_heads = static_cast<int>(c->kv_heads);
  p.group = static_cast<int>(group);
  p.page_size = static_cast<int>(c->page_size);
  p.max_pages = static_cast<int>(q->max_pages);
  p.words = static_cast<int>((q->tokens + 31) / 32);
  p.window = static_cast<int>(window);
  p.sinks = static_cast<int>(sinks);
  p.tile_tokens = n.tile_tokens;
  p.blocks = n.blocks;
  p.tile_keys = n.tile_keys;
  p.tile_pages = n.tile_pages;
  p.page_tiles = n.page_tiles;
  p.page_shift = p.tile_shift = -1;
  for (int i = 3; i <= 20; ++i) {
    if (p.page_size == 1 << i) p.page_shift = i;
    if (n.tile_keys == 1 << i) p.tile_shift = i;
  }
  p.rows = n.rows;
  p.whole = n.whole;
  p.c = static_cast<float>(q->scale * 1.4426950408889634);
  p.wait_limit = ntl_wait_limit();
  // Key groups for up to 16 rows: 64 sequences x 1 token x 4 heads per key head, window 4096: 175 us against
  // 197 us without (back to back, at the power cap).  Four groups of up to 32 rows need the 128-row MMA
  // and measured slower than none at head_dim 128 (32 x 8 drafts over 8192 tokens: 213 against 201 us).
#define NTL_CACHE_ATTN(D, NT, KS)                                                                       \
  return n.page_tiles ? bf16 ? launch_shape<D, NT, KS, true, true>(what, mq, mk, mv, mv8, mv1, p, n, s)           \
                             : launch_shape<D, NT, KS, false, true>(what, mq, mk, mv, mv8, mv1, p, n, s)          \
         : bf16       ? launch_shape<D, NT, KS, true, false>(what, mq, mk, mv, mv8, mv1, p, n, s)                 \
                      : launch_shape<D, NT, KS, false, false>(what, mq, mk, mv, mv8, mv1, p, n, s)
  if (dim == 64) {
    if (n.row_tiles == 2) NTL_CACHE_ATTN(64, 2, 1);
    if (key_groups) NTL_CACHE_ATTN(64, 1, 4);
    NTL_CACHE_ATTN(64, 1, 1);
  }
  if (n.row_tiles == 2) NTL_CACHE_ATTN(128, 2, 1);
  if (key_groups) NTL_CACHE_ATTN(128, 1, 4);
  NTL_CACHE_ATTN(128, 1, 1);
#undef NTL_CACHE_ATTN
}

int check(const char* what, const ntl_cache_t* c, const ntl_query_t* q) {
  NTL_REQUIRE(c && q, NTL_ERR_INVALID, "%s: NULL descriptor", what);
  NTL_REQUIRE(c->pages >= 0 && c->kv_heads >= 0 && q->seqs >= 0 && q->tokens >= 0 && q->heads >= 0 &&
                  q->max_pages >= 0 && q->table_stride >= 0,
              NTL_ERR_INVALID, "%s: negative size", what);
  NTL_REQUIRE(c->dtype == NTL_F16 || c->dtype == NTL_BF16, NTL_ERR_UNSUPPORTED, "%s: data type %lld", what,
              (long long)c->dtype);
  NTL_REQUIRE(c->head_dim == 64 || c->head_dim == 128, NTL_ERR_UNSUPPORTED,
              "%s: head_dim %lld is not supported (64 or 128)", what, (long long)c->head_dim);
  NTL_REQUIRE(c->page_size >= 8 && c->page_size % 8 == 0 && c->page_size <= (1 << 20), NTL_ERR_UNSUPPORTED,
              "%s: page_size %lld is not a multiple of 8", what, (long long)c->page_size);
  if (q->seqs == 0 || q->tokens == 0 || q->heads == 0) return NTL_OK;
  NTL_REQUIRE(c->kv_heads > 0 && q->heads % c->kv_heads == 0 && q->heads / c->kv_heads <= 128, NTL_ERR_UNSUPPORTED,
              "%s: %lld heads over %lld key heads (a whole number up to 128 each)", what, (long long)q->heads,
              (long long)c->kv_heads);
  NTL_REQUIRE(q->tokens < (1 << 24) && q->seqs < (1 << 24) && c->pages < (int64_t(1) << 31) &&
                  q->max_pages * c->page_size < (int64_t(1) << 31) - 1024,
              NTL_ERR_UNSUPPORTED, "%s: too large", what);
  NTL_REQUIRE(q->scale > 0 && q->scale < 1e30, NTL_ERR_INVALID, "%s: scale must be positive", what);
  NTL_REQUIRE(q->q && q->o && q->lens && c->k && c->v && (q->table || q->max_pages == 0), NTL_ERR_INVALID,
              "%s: NULL pointer", what);
  NTL_REQUIRE(ntl_aligned(q->q, 16) && ntl_aligned(q->o, 16) && ntl_aligned(c->k, 16) && ntl_aligned(c->v, 16) &&
                  q->seq_stride % 8 == 0 && q->token_stride % 8 == 0 && q->head_stride % 8 == 0 &&
                  c->page_stride % 8 == 0 && c->row_stride % 8 == 0 && c->head_stride % 8 == 0,
              NTL_ERR_ALIGNMENT, "%s: pointers must be 16-byte aligned and strides multiples of 8 values", what);
  return NTL_OK;
}

}  // namespace

uint32_t ntl_cache_attn_status_read(int clear) {
  uint32_t v = 0;
  if (cudaMemcpyFromSymbol(&v, g_cache_attn_status, sizeof(v)) != cudaSuccess) return 0;
  if (clear) {
    uint32_t z = 0;
    cudaMemcpyToSymbol(g_cache_attn_status, &z, sizeof(z));
  }
  return v;
}

extern "C" int ntl_cache_attention_workspace(const ntl_cache_t* cache, const ntl_query_t* query, uint64_t* bytes_out) {
  if (int rc = check("cache attention", cache, query)) return rc;
  NTL_REQUIRE(bytes_out, NTL_ERR_INVALID, "cache attention: NULL result");
  *bytes_out = 0;
  if (query->seqs == 0 || query->tokens == 0 || query->heads == 0) return NTL_OK;
  Plan n;
  if (int rc = make_plan("cache attention", cache, query, int64_t(1) << 31, 0, &n)) return rc;
  *bytes_out = n.bytes;
  return NTL_OK;
}

extern "C" int ntl_tree_attention(const ntl_cache_t* cache, const ntl_query_t* query, const uint32_t* tree,
                                  int64_t tree_stride, void* workspace, uint64_t workspace_bytes,
                                  ntl_stream_t stream) {
  if (int rc = check("tree attention", cache, query)) return rc;
  NTL_REQUIRE(tree_stride >= 0, NTL_ERR_INVALID, "tree attention: negative mask stride");
  if (query->seqs == 0 || query->tokens == 0 || query->heads == 0) return NTL_OK;
  NTL_REQUIRE(tree, NTL_ERR_INVALID, "tree attention: NULL mask");
  return launch("tree attention", cache, query, tree, tree_stride, 0, 0, workspace, workspace_bytes,
                static_cast<cudaStream_t>(stream));
}

extern "C" int ntl_window_attention(const ntl_cache_t* cache, const ntl_query_t* query, int64_t window, int64_t sinks,
                                    void* workspace, uint64_t workspace_bytes, ntl_stream_t stream) {
  if (int rc = check("window attention", cache, query)) return rc;
  NTL_REQUIRE(window >= 1 && sinks >= 0, NTL_ERR_INVALID, "window attention: window %lld, sinks %lld",
              (long long)window, (long long)sinks);
  if (query->seqs == 0 || query->tokens == 0 || query->heads == 0) return NTL_OK;
  const int64_t most = int64_t(1) << 30;
  return launch("window attention", cache, query, nullptr, 0, window < most ? window : most, sinks < most ? sinks : most,
                workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
}
