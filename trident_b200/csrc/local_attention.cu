// Entry points of local attention (window and sinks), training and serving, and the cache write:
// validate, pick a kernel family, launch.
#include "local_attention_tc.cuh"

namespace tb200 {
namespace {

// New keys and values into their pages, one thread per 16 bytes (or per element where strides or
// alignment do not allow that). Bounded by HBM: reads and writes each element once (a prompt of 54 MB: 11 us,
// 5 TB/s); single tokens of a batch by the launch (3 us).
template <typename T, bool VECTOR>
__global__ void __launch_bounds__(256)
    cache_append(T* kc, T* vc, const T* k, const T* v, const LocalArgs a, const int64_t sk0, const int64_t sk1,
                 const int64_t sk2, const int64_t sv0, const int64_t sv1, const int64_t sv2) {
  constexpr int N = VECTOR ? Traits<T>::VEC : 1;
  const int s = blockIdx.z;
  const Sequence sq = load_sequence(a, s);
  const int per_row = a.D / N, per_token = a.KV * per_row;
  const int64_t total = (int64_t)sq.q_len * per_token;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int t = (int)(i / per_token), rest = (int)(i % per_token), h = rest / per_row, d = rest % per_row * N;
    const int pos = sq.base + t;
    if (pos < 0 || pos >= sq.kv_len) continue;  // (a context may go beyond the table)
    const int page = a.table[s * a.table_stride + pos / a.page];
    if (page < 0 || page >= a.pages) continue;
    const int64_t off = pos % a.page, tok = sq.q_begin + t;
    T* dk = kc + (int64_t)page * a.ks[0] + h * a.ks[1] + off * a.ks[2] + d * a.ks[3];
    T* dv = vc + (int64_t)page * a.vs[0] + h * a.vs[1] + off * a.vs[2] + d * a.vs[3];
    const T* pk = k + tok * sk0 + h * sk1 + d * sk2;
    const T* pv = v + tok * sv0 + h * sv1 + d * sv2;
    if constexpr (VECTOR) {
      const uint4 x = ld_stream(pk), y = ld_stream(pv);
      *reinterpret_cast<uint4*>(dk) = x;
      *reinterpret_cast<uint4*>(dv) = y;
    } else {
      *dk = *pk;
      *dv = *pv;
    }
  }
}

// Fills the list form's array. One CTA: a stretch of sequences a thread, then the stretches' sums.
__global__ void __launch_bounds__(1024) list_tiles(int* before, const LocalArgs a, const int tile_tokens) {
  __shared__ int64_t sums[1024];
  const int per = (a.n + 1023) / 1024, s0 = threadIdx.x * per, s1 = min(s0 + per, a.n);
  int64_t own = 0;
  for (int s = s0; s < s1; ++s) own += (load_sequence(a, s).q_len + tile_tokens - 1) / tile_tokens;
  sums[threadIdx.x] = own;
  __syncthreads();
  for (int d = 1; d < 1024; d <<= 1) {
    const int64_t left = (int)threadIdx.x >= d ? sums[threadIdx.x - d] : 0;
    __syncthreads();
    sums[threadIdx.x] += left;
    __syncthreads();
  }
  // (sequences that overlap, which no call should have, may add up to more: the rest is not computed)
  constexpr int64_t MOST = (1ll << 31) - (1 << 20);
  int64_t at = sums[threadIdx.x] - own;
  for (int s = s0; s < s1; ++s) {
    before[s] = (int)(at < MOST ? at : MOST);
    at += (load_sequence(a, s).q_len + tile_tokens - 1) / tile_tokens;
  }
  if (threadIdx.x == 1023) before[a.n] = (int)(sums[1023] < MOST ? sums[1023] : MOST);
}

int check_heads(const char* who, int64_t H, int64_t KV, int64_t D) {
  TB200_REQUIRE(H > 0 && KV > 0 && H % KV == 0, TB200_ERR_INVALID, "%s: %lld query heads are no multiple of %lld key heads",
                who, (long long)H, (long long)KV);
  TB200_REQUIRE(H / KV <= 64 && KV <= 65535, TB200_ERR_UNSUPPORTED, "%s: more than 64 query heads per key head", who);
  TB200_REQUIRE(D == 16 || D == 32 || D == 64 || D == 128, TB200_ERR_UNSUPPORTED, "%s: head size %lld not in {16,32,64,128}",
                who, (long long)D);
  return 0;
}

void copy4(int64_t* dst, const int64_t* src) {
  for (int i = 0; i < 4; ++i) dst[i] = src[i];
}

int fill_window(LocalArgs* a, const char* who, int64_t B, int64_t H, int64_t KV, int64_t S, int64_t D, const int64_t* qs,
                const int64_t* ks, const int64_t* vs, const int64_t* os, int64_t window, int64_t sinks, float scale) {
  if (int rc = check_heads(who, H, KV, D)) return rc;
  TB200_REQUIRE(B >= 0 && S >= 0, TB200_ERR_INVALID, "%s: negative size", who);
  TB200_REQUIRE(B <= 65535 && S < (1ll << 30), TB200_ERR_UNSUPPORTED, "%s: more than 65535 sequences or 2^30 tokens", who);
  TB200_REQUIRE(window >= 1 && sinks >= 0, TB200_ERR_INVALID, "%s: window %lld, sinks %lld", who, (long long)window,
                (long long)sinks);
  TB200_REQUIRE(qs && ks && vs && os, TB200_ERR_INVALID, "%s: null stride array", who);
  a->n = (int)B; a->H = (int)H; a->KV = (int)KV; a->G = (int)(H / KV); a->D = (int)D;
  a->tokens = (int)S;
  a->window = window >= S ? NO_WINDOW : (int)window;
  a->sinks = (int)(sinks < S ? sinks : S);
  a->scale = scale;
  copy4(a->qs, qs); copy4(a->ks, ks); copy4(a->vs, vs); copy4(a->os, os);
  return 0;
}

// Far pieces of the backward pass (see LocalBwdArgs), each about as long as a key tile's walk inside the window, and
// of all sequences, heads and sink tiles together no more than FAR_PER_SM an SM: beyond that they no longer even out
// the work, but each takes a tile of fp32 gradients of the workspace (backward pass of 32 heads on 8 key heads, 65536 x
// 128 bf16, window 1024, 8192 sinks: 2 pieces 26.8 ms and 0.2 GB, 56 pieces 31.5 ms and 4.1 GB; 8 heads x 32768, window
// 256, 2048 sinks: 9 pieces 1.28 ms, 64 pieces 2.04).
constexpr int64_t FAR_PER_SM = 8;
void plan_far(LocalBwdArgs* b, int key_tile) {
  const LocalArgs& a = b->f;
  b->sink_tiles = b->far = 0;
  if (a.window == NO_WINDOW || a.sinks == 0) return;
  const int st = (a.sinks + key_tile - 1) / key_tile;
  while (b->sink_tiles < st && near_end(a, b->sink_tiles, key_tile) < a.tokens) ++b->sink_tiles;
  if (b->sink_tiles == 0) return;
  const int64_t span = a.tokens - near_end(a, 0, key_tile), walk = (int64_t)a.window + key_tile;
  int64_t pieces = ceil_div(span, walk);
  if (pieces > 64) pieces = 64;
  const int64_t most = FAR_PER_SM * sm_count() / ((int64_t)a.n * a.KV * b->sink_tiles);
  if (pieces > most) pieces = most;
  b->far = pieces > 1 ? (int)pieces : 1;
}
size_t far_bytes(const LocalBwdArgs& b, int key_tile) {
  return (size_t)b.f.n * b.f.KV * b.sink_tiles * (b.far + 1) * 2 * key_tile * b.f.D * sizeof(float);
}
// delta of each score row (CUDA cores), or -lse and -delta by column tile (tensor cores)
size_t row_bytes(const LocalArgs& a, bool tc) {
  const int64_t floats = tc ? 2 * local_tc_rows(a) : (int64_t)a.n * a.H * a.tokens;
  return ((size_t)floats * sizeof(float) + 255) & ~(size_t)255;
}
size_t bwd_bytes(LocalBwdArgs b, bool tc) {
  const int key_tile = tc ? LOCAL_TC_TILE : local_simt_key_tile();
  plan_far(&b, key_tile);
  return row_bytes(b.f, tc) + far_bytes(b, key_tile);
}

// Parts of a split walk. One row tile of a sequence and key head is one CTA (or unit of work); where those
// are too few for the GPU the walk along the keys is cut into parts for `target` CTAs: with one row tile
// per sequence (few rows) that is several times what runs at once, so that sequences of unequal length even
// out (the parts' outputs are small next to the keys); with more, only as many as leave no SM without work.
// A part is at least 256 keys.
void plan_split(LocalArgs* a, int64_t max_q, int64_t max_ctx, int row_tile, int key_tile, int64_t target) {
  a->splits = 1;
  a->split_tiles = 0;
  const int64_t row_tiles = ceil_div(max_q, row_tile / a->G), units = (int64_t)a->n * a->KV * row_tiles;
  if (row_tiles > 1) target = sm_count();
  int64_t keys = max_ctx;
  if (a->window != NO_WINDOW) {
    const int64_t seen = (int64_t)a->window + row_tile / a->G + 2 * key_tile + (a->sinks > 0 ? a->sinks + key_tile : 0);
    if (seen < keys) keys = seen;
  }
  const int64_t tiles = ceil_div(keys, key_tile), least = 256 / key_tile;
  if (units >= target || tiles < 2 * least) return;
  int64_t splits = ceil_div(target, units);
  if (splits > tiles / least) splits = tiles / least;
  if (splits * a->n > 65535) splits = 65535 / a->n;
  if (splits < 2) return;
  a->split_tiles = (int)ceil_div(tiles, splits);
  a->splits = (int)ceil_div(tiles, a->split_tiles);
}
// The kernel family of a serving call and its tiles.
struct PagedPlan {
  bool tc = false;
  bool few = false;  // the kernel for few rows
  int row_tile = 0, key_tile = 0, row_tokens = 0;
  bool list = false;  // row tiles are listed on the device first
};
// As many row tiles are planned for each sequence as the longest announced one has. Where most of them would be empty
// (no length announced, or one long chunk among many sequences) they are listed first: a launch of 2 us, and a search
// for each tile. n sequences of 64 tokens, not announced, 8 x 4 heads, D = 128, bf16: 8 sequences (3 empty tiles an SM)
// 31 us listed and 29 not, 16 (13 an SM) 33 and 35, 64 (218) 101 and 198, 128 (880) 169 and 609.
constexpr int64_t LIST_FROM = 8;  // empty tiles an SM
PagedPlan plan_paged(LocalArgs* a, int64_t max_q, int64_t max_ctx, bool tc) {
  PagedPlan p;
  p.tc = tc;
  p.few = tc && local_few_rows(*a, (int)max_q);
  p.row_tile = p.few ? LOCAL_FEW_ROWS : (tc ? 2 * LOCAL_TC_TILE : local_simt_row_tile(*a, (int)max_q));
  p.key_tile = tc ? LOCAL_TC_TILE : local_simt_key_tile();
  p.row_tokens = p.few || !tc ? p.row_tile / a->G : local_tc_row_tokens(*a);
  plan_split(a, max_q, max_ctx, p.row_tile, p.key_tile, (int64_t)sm_count() * (p.few ? 8 : 4));
  if (a->starts && !p.few && a->split_tiles == 0) {
    const int64_t planned = a->n * ceil_div(max_q, p.row_tokens), most = a->tokens / p.row_tokens + a->n;  // (per key head)
    p.list = (planned - most) * a->KV > LIST_FROM * sm_count();
  }
  return p;
}
size_t paged_bytes(const LocalArgs& a, const PagedPlan& p) {
  if (p.list) return (size_t)(a.n + 1) * sizeof(int);
  return a.split_tiles == 0 ? 0 : (size_t)a.splits * a.tokens * a.H * (a.D + 1) * sizeof(float);
}

int fill_paged(LocalArgs* a, const char* who, int64_t T, int64_t n, int64_t H, int64_t KV, int64_t D, const void* table,
               const int32_t* context, const int32_t* starts, int64_t table_cols, int64_t table_stride, int64_t page,
               int64_t pages, const int64_t* ks, const int64_t* vs) {
  if (int rc = check_heads(who, H, KV, D)) return rc;
  TB200_REQUIRE(T >= 0 && n >= 0 && page > 0 && pages >= 0 && table_cols >= 0, TB200_ERR_INVALID, "%s: bad size", who);
  TB200_REQUIRE(n <= 65535 && T < (1ll << 30) && pages < (1ll << 31) && page < (1ll << 30) && table_cols < (1ll << 31),
                TB200_ERR_UNSUPPORTED, "%s: more than 65535 sequences, 2^30 tokens or keys per page, or 2^31 pages", who);
  TB200_REQUIRE(starts || T == n || n == 0, TB200_ERR_INVALID, "%s: %lld tokens for %lld sequences without starts", who,
                (long long)T, (long long)n);
  TB200_REQUIRE((table && context) || n == 0 || T == 0, TB200_ERR_INVALID, "%s: null pointer", who);
  TB200_REQUIRE(ks && vs, TB200_ERR_INVALID, "%s: null stride array", who);
  a->n = (int)n; a->H = (int)H; a->KV = (int)KV; a->G = (int)(H / KV); a->D = (int)D;
  a->tokens = (int)T;
  a->table = (const int*)table; a->context = context; a->starts = starts;
  a->table_cols = (int)table_cols; a->table_stride = table_stride;
  a->page = (int)page; a->pages = (int)pages;
  const int to[4] = {0, 2, 1, 3};  // [pages, page, KV, D] -> (page, head, position, feature)
  for (int i = 0; i < 4; ++i) {
    a->ks[to[i]] = ks[i];
    a->vs[to[i]] = vs[i];
  }
  return 0;
}

void set_window(LocalArgs* a, int64_t window, int64_t sinks) {
  a->window = window <= 0 || window >= NO_WINDOW ? NO_WINDOW : (int)window;
  a->sinks = a->window == NO_WINDOW ? 0 : (int)(sinks < (1 << 30) ? sinks : (1 << 30));
}

}  // namespace
}  // namespace tb200

using namespace tb200;

extern "C" int tb200_window_attention_fwd(void* out, float* lse, const void* q, const void* k, const void* v, int64_t B,
                                          int64_t H, int64_t KV, int64_t S, int64_t D, const int64_t* q_strides,
                                          const int64_t* k_strides, const int64_t* v_strides, const int64_t* out_strides,
                                          int64_t window, int64_t sinks, float softmax_scale, int dtype, void* stream) {
  return tb200_window_attention_fwd_low(out, nullptr, lse, q, k, v, B, H, KV, S, D, q_strides, k_strides, v_strides, out_strides,
                                        window, sinks, softmax_scale, dtype, stream);
}

extern "C" int tb200_window_attention_fwd_low(void* out, void* out_low, float* lse, const void* q, const void* k, const void* v,
                                              int64_t B, int64_t H, int64_t KV, int64_t S, int64_t D,
                                              const int64_t* q_strides, const int64_t* k_strides, const int64_t* v_strides,
                                              const int64_t* out_strides, int64_t window, int64_t sinks, float softmax_scale,
                                              int dtype, void* stream) {
  LocalArgs a;
  if (int rc = fill_window(&a, "window_attention_fwd", B, H, KV, S, D, q_strides, k_strides, v_strides, out_strides, window,
                           sinks, softmax_scale))
    return rc;
  if (B == 0 || S == 0) return 0;
  TB200_REQUIRE(out && q && k && v, TB200_ERR_INVALID, "window_attention_fwd: null pointer");
  a.low = dtype == TB200_F32 ? nullptr : out_low;
  const bool tc = local_tc_supported(a, dtype, q, k, v, out) && (!a.low || aligned16(a.low));
  int rc = tc ? launch_local_fwd_tc(out, lse, q, k, v, a, (int)S, dtype, (cudaStream_t)stream)
              : launch_local_fwd_simt(out, lse, q, k, v, a, (int)S, dtype, (cudaStream_t)stream);
  if (rc == 0) note_kernel(tc ? "local_tcgen05" : "local_simt", 1);
  return rc;
}

extern "C" size_t tb200_window_attention_bwd_workspace(int64_t B, int64_t H, int64_t KV, int64_t S, int64_t D,
                                                       int64_t window, int64_t sinks, int dtype) {
  (void)dtype;
  const int64_t st[4] = {0, 0, 0, 0};
  LocalBwdArgs b;
  if (fill_window(&b.f, "window_attention_bwd", B, H, KV, S, D, st, st, st, st, window, sinks, 1.f)) return 0;
  // (which kernel family takes the call depends on strides and alignment: enough for either)
  const size_t simt = bwd_bytes(b, false), tc = bwd_bytes(b, true);
  return simt > tc ? simt : tc;
}

extern "C" int tb200_window_attention_bwd(void* dq, void* dk, void* dv, const void* dout, const void* q, const void* k,
                                          const void* v, const void* out, const float* lse, void* workspace,
                                          size_t workspace_bytes, int64_t B, int64_t H, int64_t KV, int64_t S, int64_t D,
                                          const int64_t* q_strides, const int64_t* k_strides, const int64_t* v_strides,
                                          const int64_t* out_strides, const int64_t* dout_strides,
                                          const int64_t* dq_strides, const int64_t* dk_strides,
                                          const int64_t* dv_strides, int64_t window, int64_t sinks, float softmax_scale,
                                          int dtype, void* stream) {
  return tb200_window_attention_bwd_low(dq, dk, dv, dout, q, k, v, out, nullptr, lse, workspace, workspace_bytes, B, H, KV, S, D,
                                        q_strides, k_strides, v_strides, out_strides, dout_strides, dq_strides, dk_strides,
                                        dv_strides, window, sinks, softmax_scale, dtype, stream);
}

extern "C" int tb200_window_attention_bwd_low(void* dq, void* dk, void* dv, const void* dout, const void* q, const void* k,
                                              const void* v, const void* out, const void* out_low, const float* lse,
                                              void* workspace, size_t workspace_bytes, int64_t B, int64_t H, int64_t KV,
                                              int64_t S, int64_t D, const int64_t* q_strides, const int64_t* k_strides,
                                              const int64_t* v_strides, const int64_t* out_strides,
                                              const int64_t* dout_strides, const int64_t* dq_strides,
                                              const int64_t* dk_strides, const int64_t* dv_strides, int64_t window,
                                              int64_t sinks, float softmax_scale, int dtype, void* stream) {
  LocalBwdArgs b;
  if (int rc = fill_window(&b.f, "window_attention_bwd", B, H, KV, S, D, q_strides, k_strides, v_strides, out_strides, window,
                           sinks, softmax_scale))
    return rc;
  TB200_REQUIRE(dout_strides && dq_strides && dk_strides && dv_strides, TB200_ERR_INVALID,
                "window_attention_bwd: null stride array");
  if (B == 0 || S == 0) return 0;
  TB200_REQUIRE(dq && dk && dv && dout && q && k && v && out && lse && workspace, TB200_ERR_INVALID,
                "window_attention_bwd: null pointer");
  copy4(b.dos, dout_strides); copy4(b.dqs, dq_strides); copy4(b.dks, dk_strides); copy4(b.dvs, dv_strides);
  cudaStream_t st = (cudaStream_t)stream;
  b.f.low = dtype == TB200_F32 ? nullptr : const_cast<void*>(out_low);
  const bool tc = local_bwd_tc_supported(b, dtype, q, k, v, out, dout, dq, dk, dv) && (!b.f.low || aligned16(b.f.low));
  const int key_tile = tc ? LOCAL_TC_TILE : local_simt_key_tile();
  const size_t need = bwd_bytes(b, tc);
  plan_far(&b, key_tile);
  TB200_REQUIRE(workspace_bytes >= need, TB200_ERR_WORKSPACE, "window_attention_bwd: workspace of %zu bytes, %zu needed",
                workspace_bytes, need);
  TB200_REQUIRE(aligned16(workspace), TB200_ERR_INVALID, "window_attention_bwd: workspace must be 16-byte aligned");
  float* row_scratch = (float*)workspace;
  b.part = (float*)((char*)workspace + row_bytes(b.f, tc));
  if (tc) {
    if (int rc = launch_local_bwd_tc(dq, dk, dv, dout, q, k, v, out, lse, row_scratch, b, dtype, st)) return rc;
  } else {
    if (int rc = launch_local_delta(row_scratch, out, dout, b.dos, b.f, dtype, st)) return rc;
    if (int rc = launch_local_bwd_simt(dq, dk, dv, dout, q, k, v, lse, row_scratch, b, dtype, st)) return rc;
  }
  int launches = 3;
  if (b.sink_tiles > 0) {
    if (int rc = launch_local_far_sum(dk, dv, b, key_tile, dtype, st)) return rc;
    ++launches;
  }
  note_kernel(tc ? "local_tcgen05" : "local_simt", launches);
  return 0;
}

extern "C" size_t tb200_paged_attention_workspace(int64_t T, int64_t n, int64_t H, int64_t KV, int64_t D,
                                                  int64_t max_query_length, int64_t max_context_length, int64_t window,
                                                  int64_t sinks, int dtype) {
  (void)dtype;
  const int64_t st[4] = {0, 0, 0, 0};
  LocalArgs a;
  if (T <= 0 || n <= 0) return 0;
  const int32_t some = 0;
  if (fill_paged(&a, "paged_attention", T, n, H, KV, D, &some, &some, &some, 1, 1, 1, 1, st, st)) return 0;
  set_window(&a, window, sinks);
  const int max_q = (int)(max_query_length < T ? max_query_length : T);
  if (max_q <= 0) return 0;
  // (which kernel family takes the call depends on strides and alignment: enough for either)
  LocalArgs b = a;
  const PagedPlan simt = plan_paged(&a, max_q, max_context_length, false), tc = plan_paged(&b, max_q, max_context_length, true);
  return paged_bytes(a, simt) > paged_bytes(b, tc) ? paged_bytes(a, simt) : paged_bytes(b, tc);
}

extern "C" int tb200_paged_attention(void* out, const void* q, const void* key_cache, const void* value_cache,
                                     const int32_t* table, const int32_t* context, const int32_t* starts, void* workspace,
                                     size_t workspace_bytes, int64_t T, int64_t n, int64_t H, int64_t KV, int64_t D,
                                     int64_t page, int64_t pages, int64_t table_cols, int64_t table_stride,
                                     const int64_t* q_strides, const int64_t* k_strides, const int64_t* v_strides,
                                     const int64_t* out_strides, int64_t max_query_length, int64_t max_context_length,
                                     int64_t window, int64_t sinks, float softmax_scale, int zero_rest, int dtype,
                                     void* stream) {
  LocalArgs a;
  if (int rc = fill_paged(&a, "paged_attention", T, n, H, KV, D, table, context, starts, table_cols, table_stride, page,
                          pages, k_strides, v_strides))
    return rc;
  TB200_REQUIRE(q_strides && out_strides, TB200_ERR_INVALID, "paged_attention: null stride array");
  TB200_REQUIRE(sinks >= 0, TB200_ERR_INVALID, "paged_attention: %lld sinks", (long long)sinks);
  TB200_REQUIRE(max_query_length > 0 && max_query_length < (1ll << 30) && max_context_length >= 0 &&
                max_context_length < (1ll << 31), TB200_ERR_INVALID, "paged_attention: bad longest query or context");
  if (T == 0 || n == 0) return 0;
  TB200_REQUIRE(out && q && key_cache && value_cache, TB200_ERR_INVALID, "paged_attention: null pointer");
  for (int i = 0; i < 3; ++i) {  // (head, token, feature) of q and out come as (token, head, feature)
    const int to[3] = {2, 1, 3};
    a.qs[to[i]] = q_strides[i];
    a.os[to[i]] = out_strides[i];
  }
  set_window(&a, window, sinks);
  a.scale = softmax_scale;
  a.zero_rest = zero_rest;
  cudaStream_t st = (cudaStream_t)stream;
  const int max_q = (int)(max_query_length < T ? max_query_length : T);
  a.max_q = max_q;
  const PagedPlan plan = plan_paged(&a, max_q, max_context_length, local_tc_supported(a, dtype, q, key_cache, value_cache, out));
  const size_t need = paged_bytes(a, plan);
  TB200_REQUIRE(workspace_bytes >= need && (workspace || need == 0), TB200_ERR_WORKSPACE,
                "paged_attention: workspace of %zu bytes, %zu needed", workspace_bytes, need);
  if (plan.list) {
    list_tiles<<<1, 1024, 0, st>>>((int*)workspace, a, plan.row_tokens);
    if (int rc = launch_status("list_tiles")) return rc;
    a.before = (const int*)workspace;
  }
  a.part_out = (float*)workspace;
  a.part_lse = a.part_out + (size_t)a.splits * a.tokens * a.H * a.D;
  int rc = plan.few ? launch_local_few_tc(out, q, key_cache, value_cache, a, dtype, st)
           : plan.tc ? launch_local_fwd_tc(out, nullptr, q, key_cache, value_cache, a, max_q, dtype, st)
                     : launch_local_fwd_simt(out, nullptr, q, key_cache, value_cache, a, max_q, dtype, st);
  if (rc) return rc;
  if (a.split_tiles > 0)
    if ((rc = launch_local_combine(out, a, max_q, plan.row_tokens, plan.key_tile, dtype, st))) return rc;
  note_kernel(plan.tc ? "local_tcgen05" : "local_simt", a.split_tiles > 0 || plan.list ? 2 : 1);
  return 0;
}

extern "C" int tb200_paged_cache_append(void* key_cache, void* value_cache, const void* k, const void* v,
                                        const int32_t* table, const int32_t* context, const int32_t* starts, int64_t T,
                                        int64_t n, int64_t KV, int64_t D, int64_t page, int64_t pages, int64_t table_cols,
                                        int64_t table_stride, const int64_t* kc_strides, const int64_t* vc_strides,
                                        const int64_t* k_strides, const int64_t* v_strides, int dtype, void* stream) {
  LocalArgs a;
  if (int rc = fill_paged(&a, "paged_cache_append", T, n, KV, KV, D, table, context, starts, table_cols, table_stride, page,
                          pages, kc_strides, vc_strides))
    return rc;
  TB200_REQUIRE(k_strides && v_strides, TB200_ERR_INVALID, "paged_cache_append: null stride array");
  if (T == 0 || n == 0) return 0;
  TB200_REQUIRE(key_cache && value_cache && k && v, TB200_ERR_INVALID, "paged_cache_append: null pointer");
  return dispatch_dtype(dtype, [&](auto tag) -> int {
    using T_ = decltype(tag);
    constexpr int VEC = Traits<T_>::VEC;
    auto fits = [](const void* p, const int64_t* s, int last) {
      bool ok = aligned16(p) && s[last] == 1;
      for (int i = 0; i < last; ++i) ok = ok && s[i] % VEC == 0;
      return ok;
    };
    const bool vec = fits(key_cache, a.ks, 3) && fits(value_cache, a.vs, 3) && fits(k, k_strides, 2) && fits(v, v_strides, 2);
    // enough CTAs for all tokens in one sequence, at most 8 an SM over all sequences
    const int64_t work = ceil_div(T * KV * D / (vec ? VEC : 1), 256), cap = ceil_div((int64_t)sm_count() * 8, n);
    const dim3 grid((unsigned)(work < cap ? (work > 0 ? work : 1) : cap), 1, (unsigned)n);
    auto kern = vec ? cache_append<T_, true> : cache_append<T_, false>;
    kern<<<grid, 256, 0, (cudaStream_t)stream>>>((T_*)key_cache, (T_*)value_cache, (const T_*)k, (const T_*)v, a, k_strides[0],
                                                 k_strides[1], k_strides[2], v_strides[0], v_strides[1], v_strides[2]);
    const int rc = launch_status("cache_append");
    if (rc == 0) note_kernel("cache_append", 1);
    return rc;
  });
}
