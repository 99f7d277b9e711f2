// Upkeep of a paged key/value cache: append, accept (close up a verified draft path), copy, fork,
// free, reserve and compact, and the ancestor masks of draft trees.
//
// A cache is [layers, pages, page_size, kv_heads, head_dim] 16-bit values, K and V with the same
// strides; a sequence is a row of `table` (page numbers, -1 = none) and its length.  `refs` counts
// the sequences that hold each page.  Every operator moves bits, so results do not depend on
// order, and pages are always handed out lowest number first, so they do not depend on timing.
//
// All data movement is rows of kv_heads * head_dim values, one warp per row, 16 bytes per lane and
// access, K and V of a row in flight together.  Bound: HBM, each moved byte read and written once.
// Page numbers, positions and sequence numbers come from device memory: each is checked against its
// range before it is used, and what is out of range is skipped.
#include <climits>

#include "ntl_common.cuh"

namespace {

constexpr int kRowWarps = 8;        // warps (rows in flight) per block of the row kernels
constexpr int kRowUnroll = 4;       // 16-byte accesses in flight per lane and tensor
constexpr int kPlanThreads = 1024;  // the one-CTA bookkeeping kernels
constexpr int kPlanPages = 8;       // pages per thread and pass of the free-page search

// Strides in 16-byte units.
struct View {
  uint4* k;
  uint4* v;
  int64_t layer, page, row, head;
  int layers, pages, page_size, heads, chunks;  // chunks: 16-byte units of one head's values
};

__device__ __forceinline__ int64_t row_offset(const View& c, int layer, int page, int row) {
  return layer * c.layer + page * c.page + row * c.row;
}

// One warp copies a row of K and V (`units` = heads * chunks 16-byte units each); the sides may
// have different head strides.
__device__ __forceinline__ void copy_row(const uint4* ks, const uint4* vs, int64_t src_head, uint4* kd, uint4* vd,
                                         int64_t dst_head, int units, int chunks, int lane) {
  for (int e0 = lane; e0 < units; e0 += 32 * kRowUnroll) {
    uint4 a[kRowUnroll], b[kRowUnroll];
#pragma unroll
    for (int u = 0; u < kRowUnroll; ++u) {
      const int e = e0 + 32 * u;
      if (e < units) {
        const int64_t at = (e / chunks) * src_head + e % chunks;
        a[u] = ks[at];
        b[u] = vs[at];
      }
    }
#pragma unroll
    for (int u = 0; u < kRowUnroll; ++u) {
      const int e = e0 + 32 * u;
      if (e < units) {
        const int64_t at = (e / chunks) * dst_head + e % chunks;
        kd[at] = a[u];
        vd[at] = b[u];
      }
    }
  }
}

// Page of `position` in a sequence's table row; -1 where the row or the pool has none.
__device__ __forceinline__ int page_of(const int32_t* row, int max_pages, int pages, int64_t position, int page_size) {
  if (position < 0) return -1;
  const int64_t j = position / page_size;
  if (j >= max_pages) return -1;
  const int p = row[j];
  return p >= 0 && p < pages ? p : -1;
}

// ------------------------------------------------------------------------------ append, accept

struct NewRows {
  const uint4* k;
  const uint4* v;
  int64_t layer, seq, token, head;  // strides in 16-byte units
};

__global__ void __launch_bounds__(kRowWarps * 32)
    append_kernel(const View c, const NewRows n, const int32_t* table, int64_t table_stride, int max_pages,
                  const int32_t* lens, const int32_t* counts, int32_t* lens_out, int seqs, int tokens) {
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t id = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  for (int64_t b = id; b < seqs; b += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int add = counts ? min(max(counts[b], 0), tokens) : tokens;
    const int64_t room = static_cast<int64_t>(max_pages) * c.page_size;
    lens_out[b] = static_cast<int32_t>(min(static_cast<int64_t>(max(lens[b], 0)) + add, room));
  }
  const int64_t rows = static_cast<int64_t>(c.layers) * seqs * tokens;
  const int64_t stride = static_cast<int64_t>(gridDim.x) * kRowWarps;
  for (int64_t r = id >> 5; r < rows; r += stride) {
    const int t = static_cast<int>(r % tokens);
    const int64_t lb = r / tokens;
    const int b = static_cast<int>(lb % seqs), l = static_cast<int>(lb / seqs);
    if (counts && t >= counts[b]) continue;
    const int64_t pos = static_cast<int64_t>(max(lens[b], 0)) + t;
    const int page = page_of(table + b * table_stride, max_pages, c.pages, pos, c.page_size);
    if (page < 0) continue;
    const int64_t src = l * n.layer + b * n.seq + t * n.token;
    const int64_t dst = row_offset(c, l, page, static_cast<int>(pos % c.page_size));
    copy_row(n.k + src, n.v + src, n.head, c.k + dst, c.v + dst, c.head, c.heads * c.chunks, c.chunks, lane);
  }
}

// Row prefix + path[i] moves to prefix + i, in place.  A block takes one layer of one sequence and up to
// kPathThreads 16-byte columns of its K and V rows; a thread owns one column and walks the path in order:
// path is increasing, so path[j] >= j > i for every later j and no row is overwritten before it has been
// read.  Where the rows lie is worked out once per block, a step per thread (every thread for itself
// costs two dependent loads per step: 12.4 us against 5.5 us for 16 x 27 drafts in 4 layers).
constexpr int kPathThreads = 256, kPathSteps = 128, kPathUnroll = 8;

__global__ void __launch_bounds__(kPathThreads)
    accept_kernel(const View c, const int32_t* table, int64_t table_stride, int max_pages, const int32_t* lens,
                  const int32_t* drafts_of, int drafts, const int32_t* path, int64_t path_stride, int path_len,
                  const int32_t* counts, int32_t* lens_out, int seqs) {
  __shared__ int64_t from[kPathSteps], to[kPathSteps];  // row offsets; from < 0: nothing to move
  pdl_wait();
  const int units = c.heads * c.chunks, columns = 2 * units;
  const int slices = max((columns + kPathThreads - 1) / kPathThreads, 1);
  const int64_t job = blockIdx.x / slices;
  const int b = static_cast<int>(job % seqs), l = static_cast<int>(job / seqs);
  const int column = (blockIdx.x % slices) * kPathThreads + threadIdx.x;
  const int len = max(lens[b], 0), t = drafts_of ? max(drafts_of[b], 0) : drafts;
  const int prefix = max(len - t, 0);
  const int n = min(max(counts[b], 0), min(path_len, t));
  if (l == 0 && column == 0) lens_out[b] = prefix + n;
  if (c.layers == 0 || units == 0) return;  // nothing to move
  const int32_t* row = table + b * table_stride;
  const int e = column < units ? column : column - units;
  uint4* base = (column < units ? c.k : c.v) + (e / c.chunks) * c.head + e % c.chunks;
  for (int i0 = 0; i0 < n; i0 += kPathSteps) {
    const int steps = min(kPathSteps, n - i0);
    __syncthreads();
    for (int i = threadIdx.x; i < steps; i += kPathThreads) {
      const int src = path[b * path_stride + i0 + i], dst = i0 + i;
      int64_t a = -1, z = 0;
      if (src >= 0 && src < t && src != dst) {
        const int64_t sp = static_cast<int64_t>(prefix) + src, dp = static_cast<int64_t>(prefix) + dst;
        const int s_page = page_of(row, max_pages, c.pages, sp, c.page_size);
        const int d_page = page_of(row, max_pages, c.pages, dp, c.page_size);
        if (s_page >= 0 && d_page >= 0) {
          a = row_offset(c, l, s_page, static_cast<int>(sp % c.page_size));
          z = row_offset(c, l, d_page, static_cast<int>(dp % c.page_size));
        }
      }
      from[i] = a;
      to[i] = z;
    }
    __syncthreads();
    if (column >= columns) continue;
    for (int j0 = 0; j0 < steps; j0 += kPathUnroll) {
      uint4 x[kPathUnroll];
#pragma unroll
      for (int u = 0; u < kPathUnroll; ++u)
        if (j0 + u < steps && from[j0 + u] >= 0) x[u] = base[from[j0 + u]];
#pragma unroll
      for (int u = 0; u < kPathUnroll; ++u)
        if (j0 + u < steps && from[j0 + u] >= 0) base[to[j0 + u]] = x[u];
    }
  }
}

// ------------------------------------------------------------------------------ whole pages

__global__ void __launch_bounds__(kRowWarps * 32)
    copy_pages_kernel(const View c, const int32_t* src, const int32_t* dst, int n) {
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t rows = static_cast<int64_t>(c.layers) * n * c.page_size;
  const int64_t stride = static_cast<int64_t>(gridDim.x) * kRowWarps;
  for (int64_t r = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5; r < rows; r += stride) {
    const int row = static_cast<int>(r % c.page_size);
    const int64_t li = r / c.page_size;
    const int i = static_cast<int>(li % n), l = static_cast<int>(li / n);
    const int from = src[i], to = dst[i];
    if (from < 0 || from >= c.pages || to < 0 || to >= c.pages || from == to) continue;
    const int64_t a = row_offset(c, l, from, row), b = row_offset(c, l, to, row);
    copy_row(c.k + a, c.v + a, c.head, c.k + b, c.v + b, c.head, c.heads * c.chunks, c.chunks, lane);
  }
}

// ------------------------------------------------------------------------------ allocation

// Exclusive prefix sum of one value per thread over the block, and the block's total.
template <class T>
__device__ __forceinline__ T block_scan(T x, T* warp_sums, T& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  T s = x;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const T y = __shfl_up_sync(0xffffffffu, s, d);
    if (lane >= d) s += y;
  }
  if (lane == 31) warp_sums[warp] = s;
  __syncthreads();
  if (warp == 0) {
    T w = lane < warps ? warp_sums[lane] : 0;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const T y = __shfl_up_sync(0xffffffffu, w, d);
      if (lane >= d) w += y;
    }
    if (lane < warps) warp_sums[lane] = w;
  }
  __syncthreads();
  total = warp_sums[warps - 1];
  const T before = warp ? warp_sums[warp - 1] : 0;
  __syncthreads();
  return before + s - x;
}

// Pages that a sequence lacks in reserve: the unmapped entries from the page of its next token up to its
// length + extra (entries before that may be pages a window left behind, and stay as they are).  -1 when the
// table is too narrow.
__device__ __forceinline__ int pages_needed(const int32_t* row, int len, int extra, int page_size, int max_pages) {
  const int64_t want = (static_cast<int64_t>(len) + extra + page_size - 1) / page_size;
  if (want > max_pages) return -1;
  int n = 0;
  for (int j = len / page_size; j < want; ++j) n += row[j] < 0;
  return n;
}

// Whether a child can be forked: both sequences there, and not the same.
__device__ __forceinline__ bool fork_pair(int from, int to, int seqs) {
  return from >= 0 && from < seqs && to >= 0 && to < seqs && from != to;
}

// A parent's length as fork sees it, and the page that holds the part of a page at its end (-1: none there).
struct ForkParent {
  int len, full, part, last;
  __device__ __forceinline__ ForkParent(const int32_t* row, int length, int max_pages, int pages, int page_size) {
    len = static_cast<int>(min(static_cast<int64_t>(max(length, 0)), static_cast<int64_t>(max_pages) * page_size));
    full = len / page_size;
    part = len % page_size;
    last = part ? row[full] : -1;
    if (last >= pages) last = -1;
  }
};

// One CTA.  Ranks the needs of n sequences in order (first[i] = pages needed before sequence i),
// lists the lowest free pages in order, and for reserve hands them out.  A sequence whose pages do not
// all exist gets none; those after it that need pages get none either.  For fork (`child` is not null) seq[i]
// is the parent and needs a page for the part at its end; pairs that are refused need none.  Needs are summed in 64
// bits (2^11 sequences with 2^20 unmapped entries each pass 2^31); first[] stops at pages + 1, which is not to be had.
// work: first[n + 1], list[pages].  fork reads first, list and found in the next kernel.
__global__ void __launch_bounds__(kPlanThreads)
    plan_kernel(int32_t* table, int64_t table_stride, int max_pages, const int32_t* lens, int32_t* refs, int pages,
                int page_size, const int32_t* seq, const int32_t* child, int n, int seqs, int extra,
                const int32_t* extra_of, int32_t* granted, int32_t* found_out, int32_t* first, int32_t* list) {
  __shared__ int warp_sums[32];
  __shared__ int64_t need_sums[32];
  const int64_t most = min(static_cast<int64_t>(pages) + 1, static_cast<int64_t>(INT_MAX));
  pdl_wait();
  pdl_trigger();
  int64_t need = 0;
  for (int i0 = 0; i0 < n; i0 += blockDim.x) {
    const int i = i0 + threadIdx.x;
    int64_t mine = 0;
    if (i < n) {
      const int b = seq[i];
      if (child) {
        if (fork_pair(b, child[i], seqs))
          mine = ForkParent(table + b * table_stride, lens[b], max_pages, pages, page_size).last >= 0;
      } else if (b >= 0 && b < seqs) {
        const int add = extra_of ? max(extra_of[i], 0) : extra;
        mine = max(pages_needed(table + b * table_stride, max(lens[b], 0), add, page_size, max_pages), 0);
      }
    }
    int64_t total;
    const int64_t at = need + block_scan(mine, need_sums, total);
    if (i < n) first[i] = static_cast<int32_t>(min(at, most));
    need += total;
  }
  need = min(need, most);
  if (threadIdx.x == 0) first[n] = static_cast<int32_t>(need);
  int found = 0;
  for (int p0 = 0; p0 < pages && found < need; p0 += blockDim.x * kPlanPages) {
    const int base = p0 + threadIdx.x * kPlanPages;
    unsigned unused = 0;
#pragma unroll
    for (int u = 0; u < kPlanPages; ++u)
      if (base + u < pages && refs[base + u] <= 0) unused |= 1u << u;
    int total;
    int at = found + block_scan(__popc(unused), warp_sums, total);
#pragma unroll
    for (int u = 0; u < kPlanPages; ++u)
      if (unused >> u & 1) {
        if (at < need) list[at] = base + u;
        ++at;
      }
    found = static_cast<int>(min(need, static_cast<int64_t>(found) + total));
  }
  if (threadIdx.x == 0) *found_out = found;
  if (child) return;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const int b = seq[i];
    bool ok = false;
    if (b >= 0 && b < seqs) {
      int32_t* row = table + b * table_stride;
      const int len = max(lens[b], 0), add = extra_of ? max(extra_of[i], 0) : extra;
      const int lacks = pages_needed(row, len, add, page_size, max_pages);
      ok = lacks == 0 || (lacks > 0 && first[i + 1] <= found);
      int at = first[i];
      for (int j = len / page_size; ok && lacks > 0 && j < max_pages && at < first[i + 1]; ++j)
        if (row[j] < 0) {
          refs[list[at]] = 1;
          row[j] = list[at++];
        }
    }
    granted[i] = ok;
  }
}

// blockIdx.y = child.  Block x = 0 writes the child's table row, counts the shared pages and sets its
// length; the others copy the rows of the page that the parent has only part of.
__global__ void __launch_bounds__(kRowWarps * 32)
    fork_kernel(const View c, int32_t* table, int64_t table_stride, int max_pages, int32_t* lens, int32_t* refs,
                const int32_t* src, const int32_t* dst, int seqs, const int32_t* first, const int32_t* list,
                const int32_t* found, int32_t* granted) {
  pdl_wait();
  const int i = blockIdx.y;
  const int from = src[i], to = dst[i];
  if (!fork_pair(from, to, seqs)) {
    if (blockIdx.x == 0 && threadIdx.x == 0) granted[i] = 0;
    return;
  }
  const int32_t* parent = table + from * table_stride;
  const ForkParent end(parent, lens[from], max_pages, c.pages, c.page_size);
  const int full = end.full, part = end.part;
  const bool ok = part == 0 || (end.last >= 0 && first[i] < *found);
  const int fresh = part && ok ? list[first[i]] : -1;
  if (blockIdx.x == 0) {
    int32_t* row = table + to * table_stride;
    for (int j = threadIdx.x; j < max_pages; j += blockDim.x) {
      int p = ok && j < full ? parent[j] : -1;
      if (p >= c.pages) p = -1;
      if (p >= 0) atomicAdd(refs + p, 1);
      if (j == full) p = fresh;
      row[j] = p;
    }
    if (threadIdx.x == 0) {
      lens[to] = ok ? end.len : 0;
      granted[i] = ok;
      if (fresh >= 0) refs[fresh] = 1;
    }
    return;
  }
  if (fresh < 0) return;
  const int old = end.last;
  const int lane = threadIdx.x & 31;
  const int64_t rows = static_cast<int64_t>(c.layers) * part;
  for (int64_t r = (blockIdx.x - 1) * kRowWarps + (threadIdx.x >> 5); r < rows; r += (gridDim.x - 1) * kRowWarps) {
    const int l = static_cast<int>(r / part), at = static_cast<int>(r % part);
    const int64_t a = row_offset(c, l, old, at), b = row_offset(c, l, fresh, at);
    copy_row(c.k + a, c.v + a, c.head, c.k + b, c.v + b, c.head, c.heads * c.chunks, c.chunks, lane);
  }
}

// Block = sequence.  A page is given back once for each entry that held it (the entry is taken by
// an exchange, so a sequence listed twice counts once).
__global__ void free_kernel(int32_t* table, int64_t table_stride, int max_pages, int32_t* lens, int32_t* refs,
                            int pages, const int32_t* seq, int seqs) {
  pdl_wait();
  const int b = seq[blockIdx.x];
  if (b < 0 || b >= seqs) return;
  int32_t* row = table + b * table_stride;
  for (int j = threadIdx.x; j < max_pages; j += blockDim.x) {
    if (row[j] < 0) continue;
    const int p = atomicExch(row + j, -1);
    if (p >= 0 && p < pages) atomicSub(refs + p, 1);
  }
  if (threadIdx.x == 0) lens[b] = 0;
}

// One CTA.  n live pages; the k-th live page at or past n moves into the k-th hole before n, so no
// page is both read and written.  work: moves (1), map[pages], hole[pages], mover[pages].
__global__ void __launch_bounds__(kPlanThreads)
    compact_plan_kernel(const int32_t* refs, int32_t* refs_out, int pages, int32_t* live_out, int32_t* moves,
                        int32_t* map, int32_t* hole, int32_t* mover) {
  __shared__ int warp_sums[32];
  pdl_wait();
  pdl_trigger();
  int mine = 0;
  for (int p = threadIdx.x; p < pages; p += blockDim.x) mine += refs[p] > 0;
  int live;
  block_scan(mine, warp_sums, live);
  int holes = 0, movers = 0;
  for (int p0 = 0; p0 < pages; p0 += blockDim.x * kPlanPages) {
    const int base = p0 + threadIdx.x * kPlanPages;
    unsigned h = 0, m = 0;
#pragma unroll
    for (int u = 0; u < kPlanPages; ++u) {
      const int p = base + u;
      if (p >= pages) break;
      map[p] = p;
      const bool is_live = refs[p] > 0;
      if (p < live && !is_live) h |= 1u << u;
      if (p >= live && is_live) m |= 1u << u;
    }
    int total;
    int at = holes + block_scan(__popc(h), warp_sums, total);
    holes += total;
#pragma unroll
    for (int u = 0; u < kPlanPages; ++u)
      if (h >> u & 1) hole[at++] = base + u;
    at = movers + block_scan(__popc(m), warp_sums, total);
    movers += total;
#pragma unroll
    for (int u = 0; u < kPlanPages; ++u)
      if (m >> u & 1) mover[at++] = base + u;
  }
  __syncthreads();
  for (int r = threadIdx.x; r < movers; r += blockDim.x) {
    map[mover[r]] = hole[r];
    refs_out[hole[r]] = refs[mover[r]];
  }
  __syncthreads();
  for (int p = threadIdx.x; p < pages; p += blockDim.x) {
    if (p >= live) {
      refs_out[p] = 0;
    } else if (refs[p] > 0) {
      refs_out[p] = refs[p];
    }
  }
  if (threadIdx.x == 0) {
    *live_out = live;
    *moves = movers;
  }
}

__global__ void __launch_bounds__(kRowWarps * 32)
    compact_kernel(const View c, const int32_t* table, int64_t table_stride, int32_t* table_out, int64_t out_stride,
                   int seqs, int max_pages, const int32_t* moves, const int32_t* map, const int32_t* hole,
                   const int32_t* mover) {
  pdl_wait();
  const int64_t id = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  const int64_t entries = static_cast<int64_t>(seqs) * max_pages;
  for (int64_t e = id; e < entries; e += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t b = e / max_pages, j = e % max_pages;
    const int p = table[b * table_stride + j];
    table_out[b * out_stride + j] = p >= 0 && p < c.pages ? map[p] : -1;
  }
  const int lane = threadIdx.x & 31, n = *moves;
  const int64_t rows = static_cast<int64_t>(c.layers) * n * c.page_size;
  const int64_t stride = static_cast<int64_t>(gridDim.x) * kRowWarps;
  for (int64_t r = id >> 5; r < rows; r += stride) {
    const int row = static_cast<int>(r % c.page_size);
    const int64_t li = r / c.page_size;
    const int i = static_cast<int>(li % n), l = static_cast<int>(li / n);
    const int64_t a = row_offset(c, l, mover[i], row), b = row_offset(c, l, hole[i], row);
    copy_row(c.k + a, c.v + a, c.head, c.k + b, c.v + b, c.head, c.heads * c.chunks, c.chunks, lane);
  }
}

// ------------------------------------------------------------------------------ tree masks

// Block = sequence.  Bit s of words[t] is set when s is t or an ancestor of t.  A parent that is not
// an earlier draft (negative, or not below its child) ends the walk, so every walk ends.
__global__ void tree_mask_kernel(const int32_t* parents, int64_t stride, int tokens, int words, uint32_t* out) {
  extern __shared__ int32_t parent[];
  pdl_wait();
  pdl_trigger();
  const int32_t* row = parents + blockIdx.x * stride;
  for (int t = threadIdx.x; t < tokens; t += blockDim.x) parent[t] = row[t];
  __syncthreads();
  for (int e = threadIdx.x; e < tokens * words; e += blockDim.x) {
    const int t = e / words, w = e % words;
    uint32_t bits = 0;
    for (int a = t; a >= 0;) {
      if (a >> 5 == w) bits |= 1u << (a & 31);
      const int up = parent[a];
      a = up < a ? up : -1;
    }
    out[(static_cast<int64_t>(blockIdx.x) * tokens + t) * words + w] = bits;
  }
}

// ------------------------------------------------------------------------------ host side

// The plans' passes over pages and sequences, kPlanThreads * kPlanPages at a time, count in 32 bits.
constexpr int64_t kMostPages = (int64_t(1) << 31) - 2 * kPlanThreads * kPlanPages;

int make_view(const char* what, const ntl_cache_t* c, View* view) {
  NTL_REQUIRE(c != nullptr, NTL_ERR_INVALID, "%s: NULL cache", what);
  NTL_REQUIRE(c->layers >= 0 && c->pages >= 0 && c->kv_heads >= 0, NTL_ERR_INVALID, "%s: negative cache size", what);
  NTL_REQUIRE(c->page_size >= 1 && c->head_dim >= 8 && c->head_dim % 8 == 0, NTL_ERR_UNSUPPORTED,
              "%s: page_size %lld must be positive and head_dim %lld a multiple of 8", what, (long long)c->page_size,
              (long long)c->head_dim);
  NTL_REQUIRE(c->layers < (1 << 20) && c->pages <= kMostPages && c->page_size <= (1 << 20) &&
                  c->kv_heads * c->head_dim < (int64_t(1) << 24),
              NTL_ERR_UNSUPPORTED, "%s: cache too large", what);
  NTL_REQUIRE(c->layer_stride % 8 == 0 && c->page_stride % 8 == 0 && c->row_stride % 8 == 0 && c->head_stride % 8 == 0,
              NTL_ERR_ALIGNMENT, "%s: cache strides must be multiples of 8 values", what);
  if (c->layers > 0 && c->pages > 0 && c->kv_heads > 0) {
    NTL_REQUIRE(c->k && c->v, NTL_ERR_INVALID, "%s: NULL cache pointer", what);
    NTL_REQUIRE(ntl_aligned(c->k, 16) && ntl_aligned(c->v, 16), NTL_ERR_ALIGNMENT,
                "%s: cache must be 16-byte aligned", what);
  }
  view->k = static_cast<uint4*>(c->k);
  view->v = static_cast<uint4*>(c->v);
  view->layer = c->layer_stride / 8;
  view->page = c->page_stride / 8;
  view->row = c->row_stride / 8;
  view->head = c->head_stride / 8;
  view->layers = static_cast<int>(c->layers);
  view->pages = static_cast<int>(c->pages);
  view->page_size = static_cast<int>(c->page_size);
  view->heads = static_cast<int>(c->kv_heads);
  view->chunks = static_cast<int>(c->head_dim / 8);
  return NTL_OK;
}

int check_table(const char* what, const int32_t* table, int64_t stride, int64_t seqs, int64_t max_pages, bool written) {
  NTL_REQUIRE(seqs >= 0 && max_pages >= 0 && stride >= 0, NTL_ERR_INVALID, "%s: negative table size", what);
  NTL_REQUIRE(seqs < (int64_t(1) << 31) && max_pages < (int64_t(1) << 31), NTL_ERR_UNSUPPORTED,
              "%s: table too large", what);
  NTL_REQUIRE(seqs == 0 || max_pages == 0 || table, NTL_ERR_INVALID, "%s: NULL table", what);
  NTL_REQUIRE(!written || seqs <= 1 || stride >= max_pages, NTL_ERR_INVALID,
              "%s: rows of a table that is written must not overlap", what);
  return NTL_OK;
}

// Blocks for `jobs` jobs of `per_block`: all at once up to 16 blocks per SM (each then loops).
int grid_for(int64_t jobs, int64_t per_block, unsigned* grid) {
  int sms = 0;
  if (int rc = ntl_num_sms(&sms)) return rc;
  const int64_t want = (jobs + per_block - 1) / per_block, most = int64_t(16) * sms;
  *grid = static_cast<unsigned>(want < 1 ? 1 : want < most ? want : most);
  return NTL_OK;
}

int launched(const char* what, cudaError_t err) {
  if (err != cudaSuccess) return ntl_fail(NTL_ERR_CUDA, "%s: %s", what, cudaGetErrorString(err));
  ntl_note_launch();
  return ntl_check_launch(what);
}

}  // namespace

extern "C" int ntl_cache_append(const ntl_cache_t* cache, const void* k_new, const void* v_new, int64_t layer_stride,
                                int64_t seq_stride, int64_t token_stride, int64_t head_stride, const int32_t* table,
                                int64_t table_stride, int64_t seqs, int64_t max_pages, const int32_t* lens,
                                const int32_t* counts, int64_t tokens, int32_t* lens_out, ntl_stream_t stream) {
  View c = {};
  if (int rc = make_view("cache append", cache, &c)) return rc;
  if (int rc = check_table("cache append", table, table_stride, seqs, max_pages, false)) return rc;
  NTL_REQUIRE(tokens >= 0 && tokens < (int64_t(1) << 31), NTL_ERR_INVALID, "cache append: bad token count %lld",
              (long long)tokens);
  if (seqs == 0) return NTL_OK;
  NTL_REQUIRE(lens && lens_out, NTL_ERR_INVALID, "cache append: NULL lengths");
  NTL_REQUIRE(lens != lens_out, NTL_ERR_INVALID, "cache append: lens_out must not be lens");
  NTL_REQUIRE(tokens == 0 || (k_new && v_new), NTL_ERR_INVALID, "cache append: NULL rows");
  NTL_REQUIRE(ntl_aligned(k_new, 16) && ntl_aligned(v_new, 16) && layer_stride % 8 == 0 && seq_stride % 8 == 0 &&
                  token_stride % 8 == 0 && head_stride % 8 == 0,
              NTL_ERR_ALIGNMENT, "cache append: new rows must be 16-byte aligned");
  const NewRows n = {static_cast<const uint4*>(k_new), static_cast<const uint4*>(v_new), layer_stride / 8,
                     seq_stride / 8, token_stride / 8, head_stride / 8};
  unsigned grid;
  if (int rc = grid_for(c.layers * seqs * tokens, kRowWarps, &grid)) return rc;
  return launched("cache append",
                  ntl_launch_pdl(append_kernel, dim3(grid), dim3(kRowWarps * 32), 0, static_cast<cudaStream_t>(stream),
                                 c, n, table, table_stride, static_cast<int>(max_pages), lens, counts, lens_out,
                                 static_cast<int>(seqs), static_cast<int>(tokens)));
}

extern "C" int ntl_cache_accept(const ntl_cache_t* cache, const int32_t* table, int64_t table_stride, int64_t seqs,
                                int64_t max_pages, const int32_t* lens, const int32_t* drafts_of, int64_t drafts,
                                const int32_t* path, int64_t path_stride, int64_t path_len, const int32_t* counts,
                                int32_t* lens_out, ntl_stream_t stream) {
  View c = {};
  if (int rc = make_view("cache accept", cache, &c)) return rc;
  if (int rc = check_table("cache accept", table, table_stride, seqs, max_pages, false)) return rc;
  NTL_REQUIRE(drafts >= 0 && drafts < (int64_t(1) << 31) && path_len >= 0 && path_len < (int64_t(1) << 31),
              NTL_ERR_INVALID, "cache accept: bad draft count or path length");
  if (seqs == 0) return NTL_OK;
  NTL_REQUIRE(lens && lens_out && counts, NTL_ERR_INVALID, "cache accept: NULL lengths or counts");
  NTL_REQUIRE(lens != lens_out, NTL_ERR_INVALID, "cache accept: lens_out must not be lens");
  NTL_REQUIRE(path_len == 0 || path, NTL_ERR_INVALID, "cache accept: NULL path");
  const int64_t slices = (2ll * c.heads * c.chunks + kPathThreads - 1) / kPathThreads;
  const int64_t blocks = (c.layers > 0 ? c.layers : 1) * seqs * (slices > 0 ? slices : 1);
  NTL_REQUIRE(blocks < (int64_t(1) << 31), NTL_ERR_UNSUPPORTED, "cache accept: too large");
  return launched("cache accept",
                  ntl_launch_pdl(accept_kernel, dim3(static_cast<unsigned>(blocks)), dim3(kPathThreads), 0,
                                 static_cast<cudaStream_t>(stream), c, table, table_stride, static_cast<int>(max_pages),
                                 lens, drafts_of, static_cast<int>(drafts), path, path_stride,
                                 static_cast<int>(path_len), counts, lens_out, static_cast<int>(seqs)));
}

extern "C" int ntl_cache_copy_pages(const ntl_cache_t* cache, const int32_t* src, const int32_t* dst, int64_t n,
                                    ntl_stream_t stream) {
  View c = {};
  if (int rc = make_view("cache copy", cache, &c)) return rc;
  NTL_REQUIRE(n >= 0 && n < (int64_t(1) << 31), NTL_ERR_INVALID, "cache copy: bad page count %lld", (long long)n);
  if (n == 0 || c.layers == 0) return NTL_OK;
  NTL_REQUIRE(src && dst, NTL_ERR_INVALID, "cache copy: NULL page list");
  unsigned grid;
  if (int rc = grid_for(static_cast<int64_t>(c.layers) * n * c.page_size, kRowWarps, &grid)) return rc;
  return launched("cache copy", ntl_launch_pdl(copy_pages_kernel, dim3(grid), dim3(kRowWarps * 32), 0,
                                               static_cast<cudaStream_t>(stream), c, src, dst, static_cast<int>(n)));
}

extern "C" int ntl_cache_workspace_size(int64_t pages, int64_t n, uint64_t* bytes_out) {
  NTL_REQUIRE(bytes_out, NTL_ERR_INVALID, "cache workspace: NULL result");
  NTL_REQUIRE(pages >= 0 && n >= 0, NTL_ERR_INVALID, "cache workspace: negative size");
  *bytes_out = static_cast<uint64_t>(3 * pages + n + 8) * 4;
  return NTL_OK;
}

extern "C" int ntl_cache_fork(const ntl_cache_t* cache, int32_t* table, int64_t table_stride, int64_t seqs,
                              int64_t max_pages, int32_t* lens, int32_t* refs, const int32_t* src, const int32_t* dst,
                              int64_t n, int32_t* granted, void* workspace, uint64_t workspace_bytes,
                              ntl_stream_t stream) {
  View c = {};
  if (int rc = make_view("cache fork", cache, &c)) return rc;
  if (int rc = check_table("cache fork", table, table_stride, seqs, max_pages, true)) return rc;
  NTL_REQUIRE(n >= 0 && n <= 65535, NTL_ERR_UNSUPPORTED, "cache fork: %lld children (at most 65535 per call)",
              (long long)n);
  if (n == 0) return NTL_OK;
  NTL_REQUIRE(lens && refs && src && dst && granted, NTL_ERR_INVALID, "cache fork: NULL pointer");
  uint64_t need = 0;
  if (int rc = ntl_cache_workspace_size(c.pages, n, &need)) return rc;
  NTL_REQUIRE(workspace && workspace_bytes >= need && ntl_aligned(workspace, 4), NTL_ERR_INVALID,
              "cache fork: workspace of %llu bytes, %llu needed", (unsigned long long)workspace_bytes,
              (unsigned long long)need);
  int32_t* found = static_cast<int32_t*>(workspace);
  int32_t* first = found + 1;
  int32_t* list = first + n + 1;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (int rc = launched("cache fork",
                        ntl_launch_pdl(plan_kernel, dim3(1), dim3(kPlanThreads), 0, s, table, table_stride,
                                       static_cast<int>(max_pages), lens, refs, c.pages, c.page_size, src, dst,
                                       static_cast<int>(n), static_cast<int>(seqs), 0, nullptr, granted, found, first,
                                       list)))
    return rc;
  const int64_t rows = static_cast<int64_t>(c.layers) * (c.page_size - 1);
  const unsigned copies = static_cast<unsigned>(rows == 0 ? 0 : (rows + kRowWarps - 1) / kRowWarps < 64
                                                                    ? (rows + kRowWarps - 1) / kRowWarps
                                                                    : 64);
  return launched("cache fork",
                  ntl_launch_pdl(fork_kernel, dim3(1 + copies, static_cast<unsigned>(n)), dim3(kRowWarps * 32), 0, s, c,
                                 table, table_stride, static_cast<int>(max_pages), lens, refs, src, dst,
                                 static_cast<int>(seqs), first, list, found, granted));
}

extern "C" int ntl_cache_reserve(int64_t pages, int64_t page_size, int32_t* table, int64_t table_stride, int64_t seqs,
                                 int64_t max_pages, const int32_t* lens, int32_t* refs, const int32_t* seq, int64_t n,
                                 int64_t extra, const int32_t* extra_of, int32_t* granted, void* workspace,
                                 uint64_t workspace_bytes, ntl_stream_t stream) {
  if (int rc = check_table("cache reserve", table, table_stride, seqs, max_pages, true)) return rc;
  NTL_REQUIRE(pages >= 0 && pages <= kMostPages && page_size >= 1 && page_size <= (1 << 20), NTL_ERR_INVALID,
              "cache reserve: bad pool size");
  NTL_REQUIRE(n >= 0 && n <= kMostPages && extra >= 0 && extra < (int64_t(1) << 31), NTL_ERR_INVALID,
              "cache reserve: bad count");
  if (n == 0) return NTL_OK;
  NTL_REQUIRE(lens && refs && seq && granted, NTL_ERR_INVALID, "cache reserve: NULL pointer");
  uint64_t need = 0;
  if (int rc = ntl_cache_workspace_size(pages, n, &need)) return rc;
  NTL_REQUIRE(workspace && workspace_bytes >= need && ntl_aligned(workspace, 4), NTL_ERR_INVALID,
              "cache reserve: workspace of %llu bytes, %llu needed", (unsigned long long)workspace_bytes,
              (unsigned long long)need);
  int32_t* found = static_cast<int32_t*>(workspace);
  int32_t* first = found + 1;
  int32_t* list = first + n + 1;
  return launched("cache reserve",
                  ntl_launch_pdl(plan_kernel, dim3(1), dim3(kPlanThreads), 0, static_cast<cudaStream_t>(stream), table,
                                 table_stride, static_cast<int>(max_pages), lens, refs, static_cast<int>(pages),
                                 static_cast<int>(page_size), seq, nullptr, static_cast<int>(n), static_cast<int>(seqs),
                                 static_cast<int>(extra), extra_of, granted, found, first, list));
}

extern "C" int ntl_cache_free(int64_t pages, int32_t* table, int64_t table_stride, int64_t seqs, int64_t max_pages,
                              int32_t* lens, int32_t* refs, const int32_t* seq, int64_t n, ntl_stream_t stream) {
  if (int rc = check_table("cache free", table, table_stride, seqs, max_pages, true)) return rc;
  NTL_REQUIRE(pages >= 0 && pages < (int64_t(1) << 31) && n >= 0 && n < (int64_t(1) << 31), NTL_ERR_INVALID,
              "cache free: bad size");
  if (n == 0) return NTL_OK;
  NTL_REQUIRE(lens && refs && seq, NTL_ERR_INVALID, "cache free: NULL pointer");
  return launched("cache free", ntl_launch_pdl(free_kernel, dim3(static_cast<unsigned>(n)), dim3(256), 0,
                                               static_cast<cudaStream_t>(stream), table, table_stride,
                                               static_cast<int>(max_pages), lens, refs, static_cast<int>(pages), seq,
                                               static_cast<int>(seqs)));
}

extern "C" int ntl_cache_compact(const ntl_cache_t* cache, const int32_t* table, int64_t table_stride,
                                 int32_t* table_out, int64_t out_stride, int64_t seqs, int64_t max_pages,
                                 const int32_t* refs, int32_t* refs_out, int32_t* live, void* workspace,
                                 uint64_t workspace_bytes, ntl_stream_t stream) {
  View c = {};
  if (int rc = make_view("cache compact", cache, &c)) return rc;
  if (int rc = check_table("cache compact", table, table_stride, seqs, max_pages, false)) return rc;
  if (int rc = check_table("cache compact", table_out, out_stride, seqs, max_pages, true)) return rc;
  NTL_REQUIRE(live, NTL_ERR_INVALID, "cache compact: NULL live count");
  NTL_REQUIRE(c.pages == 0 || (refs && refs_out), NTL_ERR_INVALID, "cache compact: NULL counts");
  uint64_t need = 0;
  if (int rc = ntl_cache_workspace_size(c.pages, 0, &need)) return rc;
  NTL_REQUIRE(workspace && workspace_bytes >= need && ntl_aligned(workspace, 4), NTL_ERR_INVALID,
              "cache compact: workspace of %llu bytes, %llu needed", (unsigned long long)workspace_bytes,
              (unsigned long long)need);
  int32_t* moves = static_cast<int32_t*>(workspace);
  int32_t* map = moves + 4;
  int32_t* hole = map + c.pages;
  int32_t* mover = hole + c.pages;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (int rc = launched("cache compact", ntl_launch_pdl(compact_plan_kernel, dim3(1), dim3(kPlanThreads), 0, s, refs,
                                                        refs_out, c.pages, live, moves, map, hole, mover)))
    return rc;
  // How many pages move is known on the device only: half the pool at most.
  int64_t jobs = static_cast<int64_t>(c.layers) * (c.pages / 2) * c.page_size;
  if (seqs * max_pages / 32 > jobs) jobs = seqs * max_pages / 32;
  unsigned grid;
  if (int rc = grid_for(jobs, kRowWarps, &grid)) return rc;
  return launched("cache compact", ntl_launch_pdl(compact_kernel, dim3(grid), dim3(kRowWarps * 32), 0, s, c, table,
                                                  table_stride, table_out, out_stride, static_cast<int>(seqs),
                                                  static_cast<int>(max_pages), moves, map, hole, mover));
}

extern "C" int ntl_tree_mask(const int32_t* parents, int64_t stride, int64_t seqs, int64_t tokens, uint32_t* words,
                             ntl_stream_t stream) {
  NTL_REQUIRE(seqs >= 0 && tokens >= 0 && stride >= 0, NTL_ERR_INVALID, "tree mask: negative size");
  NTL_REQUIRE(seqs < (int64_t(1) << 31) && tokens <= 8192, NTL_ERR_UNSUPPORTED,
              "tree mask: %lld drafts per sequence (at most 8192)", (long long)tokens);
  if (seqs == 0 || tokens == 0) return NTL_OK;
  NTL_REQUIRE(parents && words, NTL_ERR_INVALID, "tree mask: NULL pointer");
  const int n = static_cast<int>((tokens + 31) / 32);
  const int64_t jobs = tokens * n;
  const unsigned threads = jobs >= 512 ? 512 : static_cast<unsigned>((jobs + 31) / 32 * 32);
  return launched("tree mask", ntl_launch_pdl(tree_mask_kernel, dim3(static_cast<unsigned>(seqs)), dim3(threads),
                                              static_cast<size_t>(tokens) * 4, static_cast<cudaStream_t>(stream),
                                              parents, stride, static_cast<int>(tokens), n, words));
}
