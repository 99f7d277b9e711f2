// Attention of a few new tokens over a paged key/value cache: a tree of drafted tokens, or causal
// with a sliding window and a few first tokens that stay visible.
//
// For query row (sequence b, token t, head h), over the keys j it sees:
//   s_j = scale * q . k_j ; m = max s ; o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m)
// in 32 bits, rounded once; a row that sees nothing gives 0.
#include <cuda_bf16.h>

#include "ntl_common.cuh"

namespace {

struct AttnParams {
  const uint16_t* q;
  uint16_t* o;
  const uint16_t* k;
  const uint16_t* v;
  const int32_t* table;
  const int32_t* lens;
  const int32_t* q_lens;
  const uint32_t* tree;  // null: window
  int64_t table_stride, q_seq, q_token, q_head, page_stride, row_stride, head_stride, tree_stride;
  int seqs, tokens, heads, kv_heads, group, pages, page_size, max_pages, words, window, sinks;
  float scale_log2;
};

template <bool BF16>
__device__ __forceinline__ float to_float(uint16_t x) {
  if constexpr (BF16) return __uint_as_float(static_cast<uint32_t>(x) << 16);
  return __half2float(__ushort_as_half(x));
}
template <bool BF16>
__device__ __forceinline__ uint16_t from_float(float x) {
  if constexpr (BF16) return __bfloat16_as_ushort(__float2bfloat16_rn(x));
  return __half_as_ushort(__float2half_rn(x));
}

// One warp per query row.
template <int D, bool BF16>
__global__ void cache_attn_simple(const AttnParams p) {
  constexpr int E = D / 32;
  const int lane = threadIdx.x & 31;
  const int64_t w = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
  if (w >= static_cast<int64_t>(p.seqs) * p.tokens * p.heads) return;
  const int h = w % p.heads, t = (w / p.heads) % p.tokens, b = w / p.heads / p.tokens;
  const int len = min(static_cast<int64_t>(max(p.lens[b], 0)), static_cast<int64_t>(p.max_pages) * p.page_size);
  const int n = min(len, p.q_lens ? min(max(p.q_lens[b], 0), p.tokens) : p.tokens);
  const int prefix = len - n, pos = prefix + t;
  float q[E], o[E] = {}, m = -INFINITY, l = 0;
  for (int e = 0; e < E; ++e)
    q[e] = to_float<BF16>(p.q[b * p.q_seq + t * p.q_token + h * p.q_head + e * 32 + lane]);
  const int last = p.tree ? len : pos + 1;
  for (int j = 0; j < last && t < n; ++j) {
    if (p.tree) {
      const int s = j - prefix;
      if (s >= 0 && !(p.tree[b * p.tree_stride + static_cast<int64_t>(t) * p.words + (s >> 5)] >> (s & 31) & 1))
        continue;
    } else if (pos - j >= p.window && j >= p.sinks) {
      continue;
    }
    const int page = p.table[b * p.table_stride + j / p.page_size];
    if (page < 0 || page >= p.pages) continue;
    const int64_t at = page * p.page_stride + (j % p.page_size) * p.row_stride + (h / p.group) * p.head_stride + lane;
    float s = 0;
    for (int e = 0; e < E; ++e) s += q[e] * to_float<BF16>(p.k[at + e * 32]);
    for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    s *= p.scale_log2;
    const float top = fmaxf(m, s), old = m == -INFINITY ? 0.f : exp2f(m - top), x = exp2f(s - top);
    l = l * old + x;
    for (int e = 0; e < E; ++e) o[e] = o[e] * old + x * to_float<BF16>(p.v[at + e * 32]);
    m = top;
  }
  for (int e = 0; e < E; ++e) p.o[w * D + e * 32 + lane] = from_float<BF16>(l > 0 ? o[e] / l : (l == l ? 0.f : l));
}

int launch(const char* what, const ntl_cache_t* c, const ntl_query_t* q, const uint32_t* tree, int64_t tree_stride,
           int64_t window, int64_t sinks, cudaStream_t s) {
  AttnParams p = {};
  p.q = static_cast<const uint16_t*>(q->q);
  p.o = static_cast<uint16_t*>(q->o);
  p.k = static_cast<const uint16_t*>(c->k);
  p.v = static_cast<const uint16_t*>(c->v);
  p.table = q->table;
  p.lens = q->lens;
  p.q_lens = q->q_lens;
  p.tree = tree;
  p.tree_stride = tree_stride;
  p.table_stride = q->table_stride;
  p.q_seq = q->seq_stride;
  p.q_token = q->token_stride;
  p.q_head = q->head_stride;
  p.page_stride = c->page_stride;
  p.row_stride = c->row_stride;
  p.head_stride = c->head_stride;
  p.seqs = q->seqs;
  p.tokens = q->tokens;
  p.heads = q->heads;
  p.kv_heads = c->kv_heads;
  p.group = q->heads / c->kv_heads;
  p.pages = c->pages;
  p.page_size = c->page_size;
  p.max_pages = q->max_pages;
  p.words = (q->tokens + 31) / 32;
  p.window = window;
  p.sinks = sinks;
  p.scale_log2 = static_cast<float>(q->scale * 1.4426950408889634);
  const unsigned grid = (q->seqs * q->tokens * q->heads + 3) / 4;
  const bool bf = c->dtype == NTL_BF16;
  if (c->head_dim == 128) {
    if (bf) cache_attn_simple<128, true><<<grid, 128, 0, s>>>(p);
    else cache_attn_simple<128, false><<<grid, 128, 0, s>>>(p);
  } else {
    if (bf) cache_attn_simple<64, true><<<grid, 128, 0, s>>>(p);
    else cache_attn_simple<64, false><<<grid, 128, 0, s>>>(p);
  }
  ntl_note_launch();
  return ntl_check_launch(what);
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

extern "C" int ntl_cache_attention_workspace(const ntl_cache_t* cache, const ntl_query_t* query, uint64_t* bytes_out) {
  if (int rc = check("cache attention", cache, query)) return rc;
  *bytes_out = 0;
  return NTL_OK;
}

extern "C" int ntl_tree_attention(const ntl_cache_t* cache, const ntl_query_t* query, const uint32_t* tree,
                                  int64_t tree_stride, void* workspace, uint64_t workspace_bytes,
                                  ntl_stream_t stream) {
  if (int rc = check("tree attention", cache, query)) return rc;
  NTL_REQUIRE(tree_stride >= 0, NTL_ERR_INVALID, "tree attention: negative mask stride");
  if (query->seqs == 0 || query->tokens == 0 || query->heads == 0) return NTL_OK;
  NTL_REQUIRE(tree, NTL_ERR_INVALID, "tree attention: NULL mask");
  return launch("tree attention", cache, query, tree, tree_stride, 0, 0, static_cast<cudaStream_t>(stream));
}

extern "C" int ntl_window_attention(const ntl_cache_t* cache, const ntl_query_t* query, int64_t window, int64_t sinks,
                                    void* workspace, uint64_t workspace_bytes, ntl_stream_t stream) {
  if (int rc = check("window attention", cache, query)) return rc;
  NTL_REQUIRE(window >= 1 && sinks >= 0, NTL_ERR_INVALID, "window attention: window %lld, sinks %lld",
              (long long)window, (long long)sinks);
  if (query->seqs == 0 || query->tokens == 0 || query->heads == 0) return NTL_OK;
  const int64_t most = int64_t(1) << 30;
  return launch("window attention", cache, query, nullptr, 0, window < most ? window : most, sinks < most ? sinks : most,
                static_cast<cudaStream_t>(stream));
}
