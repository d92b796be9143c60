// Local attention: causal attention in which a query at position p sees the key at position j when
// j <= p and (p - j < window or j < sinks), with groups of query heads sharing a key/value head.
// Shared by the training form (equal lengths, contiguous keys) and the serving form (each sequence's
// newest tokens over keys in the pages of a cache).
//
// Rows. The G query heads of a key/value head are packed with the tokens: packed row = token * G + g.
// A tile of packed rows then shares its keys among all heads of the group, and a sequence's single new
// token is G rows of one tile instead of G tiles.
//
// Keys. A tile of rows walks the key tiles that any of its rows can see: first the tiles that hold
// sinks, then those of the window (KeyRange).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"

namespace tb200 {

constexpr int NO_WINDOW = 0x7fffffff;

struct LocalArgs {
  int n = 0;            // sequences (batch)
  int H = 0, KV = 0, G = 0, D = 0;
  int tokens = 0;       // rows of q along its token dimension: S, or all new tokens
  int window = NO_WINDOW, sinks = 0;
  float scale = 1.f;
  int64_t qs[4] = {0, 0, 0, 0};  // strides (sequence, head, token, feature); sequence 0 in the serving form
  int64_t os[4] = {0, 0, 0, 0};
  int64_t ks[4] = {0, 0, 0, 0};  // strides (sequence or page, head, position, feature)
  int64_t vs[4] = {0, 0, 0, 0};
  // serving form (table != nullptr)
  const int* table = nullptr;    // [n, table_cols]: page of each block of a sequence
  const int* context = nullptr;  // [n]: keys of a sequence, new tokens included
  const int* starts = nullptr;   // [n + 1] first new token of each sequence; null: one token each
  int max_q = 0x7fffffff;        // new tokens of a sequence beyond these are not computed
  int table_cols = 0;
  int64_t table_stride = 0;
  int page = 0, pages = 0;       // keys per page, pages in the pool
  // split form: key tiles per CTA (0: all), and where the parts go
  int split_tiles = 0, splits = 1;
  float* part_out = nullptr;     // [splits][tokens * H][D]
  float* part_lse = nullptr;     // [splits][tokens * H]
  // list form: row tiles (units of work) of the sequences before s, [n + 1]; null: as many for each as for the longest
  const int* before = nullptr;
  int zero_rest = 0;             // rows that are not computed (of no sequence, beyond max_q) are set to zero
  int* status = nullptr;
  // training form, 16-bit operands: what the rounding of out leaves, in the same type and layout; null: not kept
  void* low = nullptr;
};

// New tokens [q_begin, q_begin + q_len) of a sequence that are computed, the end of all that it has, the position of
// the first of them and the number of keys that the table has room for. Offsets out of range are cut to the rows that there are; a context beyond the table
// moves no token: its positions are counted from the context's own end, and the keys behind the table do not exist.
struct Sequence {
  int q_begin, q_len, q_end, base, kv_len;
};
constexpr int MOST_KEYS = 0x7ffff000;  // (positions and a tile's columns behind them stay within 32 bits)
__device__ inline Sequence load_sequence(const LocalArgs& a, int s) {
  Sequence r;
  if (a.table == nullptr) {
    r.q_begin = r.base = 0;
    r.q_len = r.q_end = r.kv_len = a.tokens;
    return r;
  }
  if (a.starts) {
    const int b = a.starts[s], e = a.starts[s + 1];
    r.q_begin = b < 0 ? 0 : (b > a.tokens ? a.tokens : b);
    const int end = e > a.tokens ? a.tokens : e;
    r.q_end = end > r.q_begin ? end : r.q_begin;
  } else {
    r.q_begin = s;
    r.q_end = s < a.tokens ? s + 1 : s;
  }
  const int count = r.q_end - r.q_begin;
  r.q_len = count < a.max_q ? count : a.max_q;
  const int64_t room = (int64_t)a.table_cols * a.page;
  int context = a.context[s];
  context = context < 0 ? 0 : (context > MOST_KEYS ? MOST_KEYS : context);
  r.base = context - count;
  r.kv_len = context > room ? (int)room : context;
  return r;
}

// The key tiles (of `tile` keys) that rows at positions pmin..pmax can see, in walking order.
struct KeyRange {
  int sink_tiles, lo, count;
  __device__ int tile(int m) const { return m < sink_tiles ? m : lo + (m - sink_tiles); }
};
__device__ inline KeyRange key_range(const LocalArgs& a, int pmin, int pmax, int kv_len, int tile) {
  KeyRange r{0, 0, 0};
  const int last = pmax < kv_len - 1 ? pmax : kv_len - 1;  // last visible position
  if (last < 0) return r;
  if (pmin < 0) pmin = 0;
  const int first = a.window > pmin ? 0 : pmin - a.window + 1;
  r.lo = first / tile;
  const int hi = last / tile + 1;
  if (a.window != NO_WINDOW && a.sinks > 0) {
    const int st = (a.sinks + tile - 1) / tile;
    r.sink_tiles = st < r.lo ? st : r.lo;
    if (r.sink_tiles > hi) r.sink_tiles = hi;  // (a window that lies behind the table's end)
  }
  r.count = r.sink_tiles + (hi > r.lo ? hi - r.lo : 0);
  return r;
}
__device__ inline bool visible(const LocalArgs& a, int p, int j) {
  return j <= p && (p - j < a.window || j < a.sinks);
}
// First key of the window of a row tile whose first row is at position pmin (rows below it, sinks
// excepted, are seen by no row of the tile: their pages may have been given away).
__device__ inline int first_key(const LocalArgs& a, int pmin) { return a.window > pmin ? 0 : pmin - a.window + 1; }

// Sets rows [begin, end) of the output to zero: every `parts`-th of them from `part` on, by `threads` threads.
template <typename T>
__device__ inline void zero_rows(T* out, const LocalArgs& a, int64_t begin, int64_t end, int part, int parts, int thread, int threads) {
  for (int64_t t = begin + part; t < end; t += parts)
    for (int i = thread; i < a.H * a.D; i += threads)
      out[t * a.os[2] + (int64_t)(i / a.D) * a.os[1] + (int64_t)(i % a.D) * a.os[3]] = Traits<T>::from_f(0.f);
}
// Rows that no sequence computes, by the CTAs (part of parts) of sequence s: those of s beyond max_q, and before the
// first and behind the last sequence.
template <typename T>
__device__ inline void zero_rest_of(T* out, const LocalArgs& a, int s, const Sequence& seq, int part, int parts) {
  if (s == 0) zero_rows(out, a, 0, seq.q_begin, part, parts, threadIdx.x, blockDim.x);
  zero_rows(out, a, (int64_t)seq.q_begin + seq.q_len, s == a.n - 1 ? a.tokens : seq.q_end, part, parts, threadIdx.x, blockDim.x);
}

// Sequence and row tile of number `tile` (below before[n]) of the list form.
__device__ inline void listed_tile(const LocalArgs& a, int tile, int* s, int* t) {
  int lo = 0, hi = a.n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.before[mid] <= tile) lo = mid;
    else hi = mid;
  }
  *s = lo;
  *t = tile - a.before[lo];
}

// Key tiles of the walk that split `s` of a row tile takes.
__device__ inline void split_range(const LocalArgs& a, int count, int s, int* begin, int* end) {
  if (a.split_tiles == 0) {
    *begin = 0;
    *end = count;
    return;
  }
  const int64_t b = (int64_t)s * a.split_tiles;
  *begin = b < count ? (int)b : count;
  // (the last part takes what a context beyond the announced longest one leaves)
  *end = s < a.splits - 1 && b + a.split_tiles < count ? (int)(b + a.split_tiles) : count;
}

// ---- CUDA-core kernels (local_attention_simt.cu): any strides, head sizes 16, 32, 64, 128
int launch_local_fwd_simt(void* out, float* lse, const void* q, const void* k, const void* v, const LocalArgs& a,
                          int max_q, int dtype, cudaStream_t st);
int local_simt_key_tile();
// packed rows of a tile of the forward kernel
static inline int local_simt_row_tile(const LocalArgs& a, int max_q) { return (int64_t)max_q * a.G <= 16 ? 16 : 64; }
// adds the parts of a split forward: rows of sequences whose walk has more than one part
int launch_local_combine(void* out, const LocalArgs& a, int max_q, int row_tokens, int key_tile, int dtype, cudaStream_t st);
// delta[b,h,s] = sum_d out * dout
int launch_local_delta(float* delta, const void* out, const void* dout, const int64_t* dos, const LocalArgs& a, int dtype,
                       cudaStream_t st);

struct LocalBwdArgs {
  LocalArgs f;
  int64_t dos[4] = {0, 0, 0, 0};                                   // dout
  int64_t dqs[4] = {0, 0, 0, 0}, dks[4] = {0, 0, 0, 0}, dvs[4] = {0, 0, 0, 0};
  // Sinks: the queries beyond the window of a key tile that holds sinks ("far" queries) are cut into
  // `far` pieces, each handled by a CTA of its own; pieces and the window part go to
  // part[n * KV][sink_tiles][far + 1][2][key tile][D] in fp32 and are added in that order.
  int sink_tiles = 0, far = 0;
  float* part = nullptr;
};
int launch_local_bwd_simt(void* dq, void* dk, void* dv, const void* dout, const void* q, const void* k, const void* v,
                          const float* lse, const float* delta, const LocalBwdArgs& b, int dtype, cudaStream_t st);
int launch_local_far_sum(void* dk, void* dv, const LocalBwdArgs& b, int key_tile, int dtype, cudaStream_t st);
// first token beyond the window of all keys of a key tile
__host__ __device__ inline int near_end(const LocalArgs& a, int tile_index, int tile) {
  const int64_t e = (int64_t)(tile_index + 1) * tile - 1 + a.window;
  return e < a.tokens ? (int)e : a.tokens;
}

}  // namespace tb200
