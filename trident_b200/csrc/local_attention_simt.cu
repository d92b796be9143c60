// Local attention on the CUDA cores: fp32 operands (products and sums in full fp32), 16-bit operands
// with head sizes or strides that the tensor-core kernels do not take.
//
// All three kernels have one shape: RM "resident" rows in shared memory, RS "streamed" rows per
// step, both converted to fp32 on the way in, 16 (or 32) x RM / 4 threads; a thread owns 4 resident
// rows and RS / TX streamed ones of the score tile, and 4 rows x D / TX features of the result. Row
// strides are padded by 4 floats so that the 16-byte reads of a quarter-warp fall into different banks.
//   forward   resident: 64 (or 16) packed query rows, streamed: 64 keys; running maximum and sum.
//             16 rows serve single tokens, where 64 would mostly be empty.
//   dQ        resident: 64 packed query rows (Q, dO), streamed: 64 keys (K, V)
//   dK, dV    resident: 64 keys (K, V), streamed: 64 packed query rows (Q, dO): the sum over the
//             heads of a group is part of the walk, in a fixed order
// A thread issues 8 16-byte reads for 64 multiply-adds of a score tile's 4 features. At 8 heads, 1024 tokens,
// window 256, D = 64 (128 CTAs, 8 warps an SM) the kernels wait for those reads and the tiles' loads: dK/dV
// 77 us, dQ 52, forward 40, the multiply-adds 30 % and the issue slots 42 % busy in each. In the backward kernels a
// warp covers 4 x 8 threads of the tile (2 x 16 and 32 streamed rows: 92 and 57 us); 8 columns a thread need
// a quarter fewer reads, but leave 4 warps an SM (110, 71 and 57 us).
#include <type_traits>

#include "local_attention.cuh"
#include "row_common.cuh"

namespace tb200 {
namespace {

constexpr int KEY_TILE = 64;

// RM x RS score tile over RD features: TX threads walk the streamed rows, TY = RM / 4 the resident.
template <int D, int RM, int RS, int TX>
struct Shape {
  static constexpr int TY = RM / 4, THREADS = TX * TY, LD = D + 4;
  static constexpr int SC = RS / TX;                     // streamed rows of a thread
  static constexpr int W = D / TX < 4 ? D / TX : 4;      // features per access of the result
  static constexpr int DC = D / (TX * W);                // accesses
  static_assert(RS % TX == 0 && W >= 1, "tile shape");
};

template <int W>
__device__ inline void load_w(float (&f)[W], const float* p) {
  if constexpr (W == 4) {
    const float4 v = *reinterpret_cast<const float4*>(p);
    f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
  } else if constexpr (W == 2) {
    const float2 v = *reinterpret_cast<const float2*>(p);
    f[0] = v.x; f[1] = v.y;
  } else {
    f[0] = *p;
  }
}

// s[i][j] += sum_d a[row i][d] b[row j][d]; rows ty * 4 + i of a, tx + TX * j of b
template <int D, int RM, int RS, int TX>
__device__ inline void dot_tile(float (&s)[4][Shape<D, RM, RS, TX>::SC], const float* a, const float* b, int ty, int tx) {
  using Sh = Shape<D, RM, RS, TX>;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < Sh::SC; ++j) s[i][j] = 0.f;
#pragma unroll 4
  for (int d = 0; d < D; d += 4) {
    float av[4][4], bv[Sh::SC][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) load_w<4>(av[i], a + (ty * 4 + i) * Sh::LD + d);
#pragma unroll
    for (int j = 0; j < Sh::SC; ++j) load_w<4>(bv[j], b + (tx + TX * j) * Sh::LD + d);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < Sh::SC; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[i][j] = fmaf(av[i][e], bv[j][e], s[i][j]);
  }
}

// acc[i][..] += sum_k p[row i][k] b[k][..]; p has RS + 4 floats a row
template <int D, int RM, int RS, int TX>
__device__ inline void accumulate(float (&acc)[4][Shape<D, RM, RS, TX>::DC][Shape<D, RM, RS, TX>::W], const float* p,
                                  const float* b, int ty, int tx) {
  using Sh = Shape<D, RM, RS, TX>;
#pragma unroll 2
  for (int k = 0; k < RS; k += 4) {
    float pv[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) load_w<4>(pv[i], p + (ty * 4 + i) * (RS + 4) + k);
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int c = 0; c < Sh::DC; ++c) {
        float bv[Sh::W];
        load_w<Sh::W>(bv, b + (k + e) * Sh::LD + (c * TX + tx) * Sh::W);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int w = 0; w < Sh::W; ++w) acc[i][c][w] = fmaf(pv[i][e], bv[w], acc[i][c][w]);
      }
  }
}

// The same with a sum of its own for the step, added at its end: one running sum over the rows of 64 heads and 600
// tokens was off by 4e-6 of the result, 10 times a matrix product's error, one over 65536 keys of a forward walk by 3.6e-6
// in the mean (now 0.5e-6).
template <int D, int RM, int RS, int TX>
__device__ inline void accumulate_step(float (&acc)[4][Shape<D, RM, RS, TX>::DC][Shape<D, RM, RS, TX>::W], const float* p,
                                       const float* b, int ty, int tx) {
  using Sh = Shape<D, RM, RS, TX>;
  float sum[4][Sh::DC][Sh::W];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int c = 0; c < Sh::DC; ++c)
#pragma unroll
      for (int w = 0; w < Sh::W; ++w) sum[i][c][w] = 0.f;
  accumulate<D, RM, RS, TX>(sum, p, b, ty, tx);
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int c = 0; c < Sh::DC; ++c)
#pragma unroll
      for (int w = 0; w < Sh::W; ++w) acc[i][c][w] += sum[i][c][w];
}

// Rows [0, rows) of a tile into shared memory as fp32; row_ptr(r) is null for rows that do not exist.
template <typename T, int D, int THREADS, typename RowPtr>
__device__ inline void load_rows(float* dst, int rows, int64_t feature_stride, bool vec, RowPtr row_ptr) {
  constexpr int LD = D + 4, VEC = Traits<T>::VEC;
  if (vec) {
    for (int i = threadIdx.x; i < rows * (D / VEC); i += THREADS) {
      const int r = i / (D / VEC), c = (i % (D / VEC)) * VEC;
      const T* p = row_ptr(r);
      float f[VEC];
      if (p) {
        unpack<T>(__ldg(reinterpret_cast<const uint4*>(p + c)), f);
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) f[e] = 0.f;
      }
#pragma unroll
      for (int e = 0; e < VEC; e += 4)
        *reinterpret_cast<float4*>(dst + r * LD + c + e) = make_float4(f[e], f[e + 1], f[e + 2], f[e + 3]);
    }
  } else {
    for (int i = threadIdx.x; i < rows * D; i += THREADS) {
      const int r = i / D, c = i % D;
      const T* p = row_ptr(r);
      dst[r * LD + c] = p ? Traits<T>::to_f(p[c * feature_stride]) : 0.f;
    }
  }
}

// Row of the key (or value) at position j of sequence s, head h; null where there is none.
template <typename T>
__device__ inline const T* key_row(const LocalArgs& a, const T* base, const int64_t* st, int s, int h, int j, int kv_len) {
  if (j < 0 || j >= kv_len) return nullptr;
  if (a.table == nullptr) return base + (int64_t)s * st[0] + h * st[1] + (int64_t)j * st[2];
  const int page = a.table[s * a.table_stride + j / a.page];
  if (page < 0 || page >= a.pages) return nullptr;
  return base + (int64_t)page * st[0] + h * st[1] + (int64_t)(j % a.page) * st[2];
}

template <typename T>
bool rows_vectorised(const void* p, const int64_t* st) {
  constexpr int VEC = Traits<T>::VEC;
  return aligned16(p) && st[3] == 1 && st[0] % VEC == 0 && st[1] % VEC == 0 && st[2] % VEC == 0;
}

// max or sum over the TX threads of a row (lanes of one warp)
template <int TX, bool MAX>
__device__ inline float row_fold(float v) {
#pragma unroll
  for (int o = TX / 2; o > 0; o >>= 1) {
    const float w = __shfl_xor_sync(0xffffffffu, v, o);
    v = MAX ? fmaxf(v, w) : v + w;
  }
  return v;
}

// ------------------------------------------------------------------ forward
template <typename T, int D, int RM, int TX>
__global__ void __launch_bounds__(Shape<D, RM, KEY_TILE, TX>::THREADS)
    local_fwd_simt(T* out, float* lse, const T* q, const T* k, const T* v, const LocalArgs a, int qvec, int kvec) {
  using Sh = Shape<D, RM, KEY_TILE, TX>;
  constexpr int THREADS = Sh::THREADS, LD = Sh::LD, SC = Sh::SC;
  extern __shared__ __align__(16) float sm[];
  float* sq = sm;                    // [RM][LD]
  float* sk = sq + RM * LD;          // [64][LD], and the probabilities [RM][68] once the scores are out
  float* sv = sk + KEY_TILE * LD;    // [64][LD]
  constexpr int PLD = KEY_TILE + 4;
  static_assert(RM * PLD <= (RM > KEY_TILE ? RM : KEY_TILE) * LD || D < 64, "probabilities fit over the keys");
  float* sp = D >= 64 ? sk : sv + KEY_TILE * LD;

  const int tx = threadIdx.x % TX, ty = threadIdx.x / TX;
  int s = blockIdx.z / a.splits, tile = blockIdx.x;
  const int split = blockIdx.z % a.splits, hk = blockIdx.y;
  if (a.before == nullptr) {
    if (a.zero_rest && hk == 0 && split == 0) zero_rest_of(out, a, s, load_sequence(a, s), blockIdx.x, gridDim.x);
  } else {
    const bool zero = a.zero_rest && hk == 0;
    if (zero) {
      zero_rows(out, a, 0, load_sequence(a, 0).q_begin, blockIdx.x, gridDim.x, threadIdx.x, THREADS);
      zero_rows(out, a, load_sequence(a, a.n - 1).q_end, a.tokens, blockIdx.x, gridDim.x, threadIdx.x, THREADS);
    }
    if (tile >= a.before[a.n]) return;
    listed_tile(a, tile, &s, &tile);
    if (zero) {  // (a sequence with rows beyond max_q has tiles)
      const Sequence seq = load_sequence(a, s);
      zero_rows(out, a, (int64_t)seq.q_begin + seq.q_len, seq.q_end, tile, a.before[s + 1] - a.before[s], threadIdx.x, THREADS);
    }
  }
  const Sequence sq_ = load_sequence(a, s);
  // the packed rows of this tile: row r is token r / G of the tile, head r % G of the group
  const int tile_tokens = RM / a.G, t0 = tile * tile_tokens;
  const int ntok = min(tile_tokens, sq_.q_len - t0);
  if (ntok <= 0) return;
  const int base = sq_.base;
  const KeyRange kr = key_range(a, base + t0, base + t0 + ntok - 1, sq_.kv_len, KEY_TILE);
  int m0, m1;
  split_range(a, kr.count, split, &m0, &m1);
  if (split > 0 && m0 >= m1) return;
  const bool whole = a.split_tiles == 0 || kr.count <= a.split_tiles;
  const int rows = ntok * a.G, from = first_key(a, base + t0);
  auto key_at = [&](const T* p, const int64_t* st, int j) -> const T* {
    return j >= from || j < a.sinks ? key_row(a, p, st, s, hk, j, sq_.kv_len) : nullptr;
  };
  const T* qb = q + s * a.qs[0] + (int64_t)(hk * a.G) * a.qs[1] + (int64_t)(sq_.q_begin + t0) * a.qs[2];
  load_rows<T, D, THREADS>(sq, RM, a.qs[3], qvec, [&](int r) -> const T* {
    return r < rows ? qb + (int64_t)(r % a.G) * a.qs[1] + (int64_t)(r / a.G) * a.qs[2] : nullptr;
  });
  float acc[4][Sh::DC][Sh::W], m[4], l[4];
  int pos[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
    const int r = ty * 4 + i;
    pos[i] = r < rows ? base + t0 + r / a.G : -1;
#pragma unroll
    for (int c = 0; c < Sh::DC; ++c)
#pragma unroll
      for (int w = 0; w < Sh::W; ++w) acc[i][c][w] = 0.f;
  }
  for (int step = m0; step < m1; ++step) {
    const int j0 = kr.tile(step) * KEY_TILE;
    __syncthreads();  // (the previous step's values have been read)
    load_rows<T, D, THREADS>(sk, KEY_TILE, a.ks[3], kvec,
                             [&](int r) { return key_at(k, a.ks, j0 + r); });
    load_rows<T, D, THREADS>(sv, KEY_TILE, a.vs[3], kvec,
                             [&](int r) { return key_at(v, a.vs, j0 + r); });
    __syncthreads();
    float sc[4][SC];
    dot_tile<D, RM, KEY_TILE, TX>(sc, sq, sk, ty, tx);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float mx = -INFINITY;
#pragma unroll
      for (int j = 0; j < SC; ++j) {
        const int key = j0 + tx + TX * j;
        sc[i][j] = key < sq_.kv_len && visible(a, pos[i], key) ? sc[i][j] * a.scale : -INFINITY;
        mx = fmaxf(mx, sc[i][j]);
      }
      mx = fmaxf(m[i], row_fold<TX, true>(mx));
      const float safe = mx == -INFINITY ? 0.f : mx;  // a row that has seen no key yet
      const float shrink = expf(m[i] - safe);
      m[i] = mx;
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < SC; ++j) {
        const float p = expf(sc[i][j] - safe);
        sum += p;
        sp[(ty * 4 + i) * PLD + tx + TX * j] = p;
      }
      l[i] = l[i] * shrink + row_fold<TX, false>(sum);
#pragma unroll
      for (int c = 0; c < Sh::DC; ++c)
#pragma unroll
        for (int w = 0; w < Sh::W; ++w) acc[i][c][w] *= shrink;
    }
    __syncthreads();
    accumulate_step<D, RM, KEY_TILE, TX>(acc, sp, sv, ty, tx);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = ty * 4 + i;
    if (r >= rows) continue;
    const float inv = l[i] > 0.f ? 1.f / l[i] : 0.f;  // a row without keys: zeros
    const float ls = l[i] > 0.f ? m[i] + logf(l[i]) : -INFINITY;
    const int head = hk * a.G + r % a.G, token = sq_.q_begin + t0 + r / a.G;
    if (whole) {
      T* o = out + s * a.os[0] + head * a.os[1] + token * a.os[2];
#pragma unroll
      for (int c = 0; c < Sh::DC; ++c)
#pragma unroll
        for (int w = 0; w < Sh::W; ++w) o[((c * TX + tx) * Sh::W + w) * a.os[3]] = Traits<T>::from_f(acc[i][c][w] * inv);
      if (a.low) {
        T* low = reinterpret_cast<T*>(a.low) + (o - out);
#pragma unroll
        for (int c = 0; c < Sh::DC; ++c)
#pragma unroll
          for (int w = 0; w < Sh::W; ++w) {
            const float x = acc[i][c][w] * inv;
            low[((c * TX + tx) * Sh::W + w) * a.os[3]] = Traits<T>::from_f(x - Traits<T>::to_f(Traits<T>::from_f(x)));
          }
      }
      if (lse && tx == 0) lse[((int64_t)s * a.H + head) * a.tokens + token] = ls;
    } else {
      const int64_t row = ((int64_t)split * a.tokens + token) * a.H + head;
#pragma unroll
      for (int c = 0; c < Sh::DC; ++c)
#pragma unroll
        for (int w = 0; w < Sh::W; ++w) a.part_out[row * D + (c * TX + tx) * Sh::W + w] = acc[i][c][w] * inv;
      if (tx == 0) a.part_lse[row] = ls;
    }
  }
}

// ------------------------------------------------------------------ joining the parts of a split walk
// One warp per (token, head): the parts' outputs weighted by exp(lse_part - max), in the parts' order.
template <typename T, int D>
__global__ void __launch_bounds__(256)
    local_combine(T* out, const LocalArgs a, int row_tokens, int key_tile) {
  const int lane = threadIdx.x & 31;
  const int s = blockIdx.z;
  pdl_wait();
  const Sequence sq = load_sequence(a, s);
  const int item = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const int t = item / a.H, head = item % a.H;
  if (t >= sq.q_len) return;
  const int base = sq.base, t0 = t / row_tokens * row_tokens;
  const int t1 = min(t0 + row_tokens, sq.q_len) - 1;
  const KeyRange kr = key_range(a, base + t0, base + t1, sq.kv_len, key_tile);
  if (kr.count <= a.split_tiles) return;  // written whole
  const int parts = min((kr.count + a.split_tiles - 1) / a.split_tiles, a.splits);
  const int token = sq.q_begin + t;
  const int64_t row = (int64_t)token * a.H + head, step = (int64_t)a.tokens * a.H;
  float mx = -INFINITY;
  for (int p = lane; p < parts; p += 32) mx = fmaxf(mx, a.part_lse[row + p * step]);
  mx = warp_max(mx);
  const float safe = mx == -INFINITY ? 0.f : mx;
  constexpr int PER = D >= 32 ? D / 32 : 1;
  float acc[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) acc[i] = 0.f;
  float total = 0.f;
  const bool live = lane * PER < D;
  for (int p = 0; p < parts; ++p) {
    const float w = expf(a.part_lse[row + p * step] - safe);
    total += w;
    if (live && w > 0.f) {  // (a part without keys has no output)
      const float* src = a.part_out + (row + p * step) * D + lane * PER;
      float f[PER];
      load_w<PER>(f, src);
#pragma unroll
      for (int i = 0; i < PER; ++i) acc[i] = fmaf(w, f[i], acc[i]);
    }
  }
  const float inv = total > 0.f ? 1.f / total : 0.f;
  if (live) {
    T* o = out + head * a.os[1] + token * a.os[2];
#pragma unroll
    for (int i = 0; i < PER; ++i) o[(lane * PER + i) * a.os[3]] = Traits<T>::from_f(acc[i] * inv);
  }
}

// ------------------------------------------------------------------ delta = sum_d out * dout
// (out with what its rounding left, where that was kept)
template <typename T>
__global__ void __launch_bounds__(256)
    local_delta(float* delta, const T* out, const T* dout, const LocalArgs a, const LocalBwdArgs strides) {
  const int lane = threadIdx.x & 31;
  const int64_t rows = (int64_t)a.n * a.H * a.tokens;
  const int64_t row = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (row >= rows) return;
  const int64_t t = row % a.tokens, h = row / a.tokens % a.H, b = row / a.tokens / a.H;
  const T* o = out + b * a.os[0] + h * a.os[1] + t * a.os[2];
  const T* g = dout + b * strides.dos[0] + h * strides.dos[1] + t * strides.dos[2];
  float acc = 0.f;
  const T* low = a.low ? reinterpret_cast<const T*>(a.low) + (o - out) : nullptr;
  for (int d = lane; d < a.D; d += 32) {
    const float x = Traits<T>::to_f(o[d * a.os[3]]) + (low ? Traits<T>::to_f(low[d * a.os[3]]) : 0.f);
    acc = fmaf(x, Traits<T>::to_f(g[d * strides.dos[3]]), acc);
  }
  acc = warp_sum(acc);
  if (lane == 0) delta[row] = acc;
}

// ------------------------------------------------------------------ backward
constexpr int BRM = 64, BRS = 64, BTX = 16;
// place of a thread in the 16 x 16 threads of a tile, 4 x 8 a warp
__device__ inline int bwd_tx() { return (threadIdx.x & 7) | ((threadIdx.x >> 2) & 8); }
__device__ inline int bwd_ty() { return ((threadIdx.x >> 3) & 3) | ((threadIdx.x >> 4) & 12); }

// dQ of 64 packed rows.
template <typename T, int D>
__global__ void __launch_bounds__(256)
    local_dq_simt(T* dq, const T* dout, const T* q, const T* k, const T* v, const float* lse, const float* delta,
                  const LocalBwdArgs b, int qvec, int kvec) {
  using Sh = Shape<D, BRM, BRS, BTX>;
  constexpr int THREADS = Sh::THREADS, LD = Sh::LD, SC = Sh::SC, PLD = BRS + 4;
  const LocalArgs& a = b.f;
  extern __shared__ __align__(16) float sm[];
  float* sq = sm;
  float* sd = sq + BRM * LD;
  float* sk = sd + BRM * LD;
  float* sv = sk + BRS * LD;
  float* sp = sv + BRS * LD;  // [64][68]
  const int tx = bwd_tx(), ty = bwd_ty();
  const int s = blockIdx.z, hk = blockIdx.y;
  const int tile_tokens = BRM / a.G, t0 = blockIdx.x * tile_tokens;
  const int ntok = min(tile_tokens, a.tokens - t0), rows = ntok * a.G;
  auto rows_of = [&](const T* p, const int64_t* st) {
    const T* tile = p + s * st[0] + (int64_t)(hk * a.G) * st[1] + (int64_t)t0 * st[2];
    return [=, &a](int r) -> const T* { return r < rows ? tile + (int64_t)(r % a.G) * st[1] + (int64_t)(r / a.G) * st[2] : nullptr; };
  };
  load_rows<T, D, THREADS>(sq, BRM, a.qs[3], qvec, rows_of(q, a.qs));
  load_rows<T, D, THREADS>(sd, BRM, b.dos[3], qvec, rows_of(dout, b.dos));
  float acc[4][Sh::DC][Sh::W], ls[4], de[4];
  int pos[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = ty * 4 + i;
    pos[i] = r < rows ? t0 + r / a.G : -1;
    const int64_t row = ((int64_t)s * a.H + hk * a.G + r % a.G) * a.tokens + t0 + r / a.G;
    ls[i] = r < rows ? lse[row] : 0.f;
    de[i] = r < rows ? delta[row] : 0.f;
#pragma unroll
    for (int c = 0; c < Sh::DC; ++c)
#pragma unroll
      for (int w = 0; w < Sh::W; ++w) acc[i][c][w] = 0.f;
  }
  const KeyRange kr = key_range(a, t0, t0 + ntok - 1, a.tokens, BRS);
  for (int step = 0; step < kr.count; ++step) {
    const int j0 = kr.tile(step) * BRS;
    __syncthreads();
    load_rows<T, D, THREADS>(sk, BRS, a.ks[3], kvec, [&](int r) { return key_row(a, k, a.ks, s, hk, j0 + r, a.tokens); });
    load_rows<T, D, THREADS>(sv, BRS, a.vs[3], kvec, [&](int r) { return key_row(a, v, a.vs, s, hk, j0 + r, a.tokens); });
    __syncthreads();
    float sc[4][SC], dp[4][SC];
    dot_tile<D, BRM, BRS, BTX>(sc, sq, sk, ty, tx);
    dot_tile<D, BRM, BRS, BTX>(dp, sd, sv, ty, tx);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < SC; ++j) {
        const int key = j0 + tx + BTX * j;
        const bool seen = key < a.tokens && visible(a, pos[i], key);
        const float p = seen ? expf(sc[i][j] * a.scale - ls[i]) : 0.f;
        sp[(ty * 4 + i) * PLD + tx + BTX * j] = p * (dp[i][j] - de[i]);
      }
    __syncthreads();
    accumulate_step<D, BRM, BRS, BTX>(acc, sp, sk, ty, tx);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = ty * 4 + i;
    if (r >= rows) continue;
    T* o = dq + s * b.dqs[0] + (int64_t)(hk * a.G + r % a.G) * b.dqs[1] + (int64_t)(t0 + r / a.G) * b.dqs[2];
#pragma unroll
    for (int c = 0; c < Sh::DC; ++c)
#pragma unroll
      for (int w = 0; w < Sh::W; ++w)
        o[((c * BTX + tx) * Sh::W + w) * b.dqs[3]] = Traits<T>::from_f(acc[i][c][w] * a.scale);
  }
}

// dK and dV of 64 keys; blockIdx.x below the number of key tiles: the queries inside the window of
// the tile, above: one far piece of a tile that holds sinks.
template <typename T, int D>
__global__ void __launch_bounds__(256)
    local_dkv_simt(T* dk, T* dv, const T* dout, const T* q, const T* k, const T* v, const float* lse, const float* delta,
                   const LocalBwdArgs b, int qvec, int kvec) {
  using Sh = Shape<D, BRM, BRS, BTX>;
  constexpr int THREADS = Sh::THREADS, LD = Sh::LD, SC = Sh::SC, PLD = BRS + 4;
  const LocalArgs& a = b.f;
  extern __shared__ __align__(16) float sm[];
  float* sk = sm;
  float* sv = sk + BRM * LD;
  float* sq = sv + BRM * LD;
  float* sd = sq + BRS * LD;
  float* sp = sd + BRS * LD;      // [64][68] probabilities
  float* sg = sp + BRM * PLD;     // [64][68] score gradients
  float* srow = sg + BRM * PLD;   // [2][64] lse, delta of the streamed rows
  const int tx = bwd_tx(), ty = bwd_ty();
  const int s = blockIdx.z, hk = blockIdx.y;
  const int tiles = (a.tokens + BRM - 1) / BRM;
  int kt = blockIdx.x, piece = -1, first, last;  // tokens [first, last)
  if (kt < tiles) {
    first = kt * BRM;
    last = near_end(a, kt, BRM);
  } else {
    kt = (blockIdx.x - tiles) / b.far;
    piece = (blockIdx.x - tiles) % b.far;
    const int from = near_end(a, kt, BRM);
    const int64_t span = a.tokens - from;
    first = from + (int)(span * piece / b.far);
    last = from + (int)(span * (piece + 1) / b.far);
  }
  const int j0 = kt * BRM;
  load_rows<T, D, THREADS>(sk, BRM, a.ks[3], kvec, [&](int r) { return key_row(a, k, a.ks, s, hk, j0 + r, a.tokens); });
  load_rows<T, D, THREADS>(sv, BRM, a.vs[3], kvec, [&](int r) { return key_row(a, v, a.vs, s, hk, j0 + r, a.tokens); });
  float ak[4][Sh::DC][Sh::W], av[4][Sh::DC][Sh::W];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int c = 0; c < Sh::DC; ++c)
#pragma unroll
      for (int w = 0; w < Sh::W; ++w) ak[i][c][w] = av[i][c][w] = 0.f;
  // streamed rows: packed rows [first * G, last * G)
  for (int64_t r0 = (int64_t)first * a.G; r0 < (int64_t)last * a.G; r0 += BRS) {
    const int rows = (int)min((int64_t)BRS, (int64_t)last * a.G - r0);
    auto rows_of = [&](const T* p, const int64_t* st) {
      return [=, &a](int r) -> const T* {
        if (r >= rows) return nullptr;
        const int t = (int)((r0 + r) / a.G), g = (int)((r0 + r) % a.G);
        return p + s * st[0] + (int64_t)(hk * a.G + g) * st[1] + (int64_t)t * st[2];
      };
    };
    __syncthreads();
    load_rows<T, D, THREADS>(sq, BRS, a.qs[3], qvec, rows_of(q, a.qs));
    load_rows<T, D, THREADS>(sd, BRS, b.dos[3], qvec, rows_of(dout, b.dos));
    if (threadIdx.x < BRS) {
      const int r = threadIdx.x;
      const int t = (int)((r0 + r) / a.G), g = (int)((r0 + r) % a.G);
      const int64_t row = ((int64_t)s * a.H + hk * a.G + g) * a.tokens + t;
      srow[r] = r < rows ? lse[row] : 0.f;
      srow[BRS + r] = r < rows ? delta[row] : 0.f;
    }
    __syncthreads();
    float sc[4][SC], dp[4][SC];
    dot_tile<D, BRM, BRS, BTX>(sc, sk, sq, ty, tx);
    dot_tile<D, BRM, BRS, BTX>(dp, sv, sd, ty, tx);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < SC; ++j) {
        const int r = tx + BTX * j, key = j0 + ty * 4 + i;
        const bool seen = r < rows && key < a.tokens && visible(a, (int)((r0 + r) / a.G), key);
        const float p = seen ? expf(sc[i][j] * a.scale - srow[r]) : 0.f;
        sp[(ty * 4 + i) * PLD + r] = p;
        sg[(ty * 4 + i) * PLD + r] = p * (dp[i][j] - srow[BRS + r]);
      }
    __syncthreads();
    accumulate_step<D, BRM, BRS, BTX>(av, sp, sd, ty, tx);
    accumulate_step<D, BRM, BRS, BTX>(ak, sg, sq, ty, tx);
  }
  const bool parted = kt < b.sink_tiles;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = ty * 4 + i, key = j0 + r;
    if (parted) {
      float* pk = b.part + (((((int64_t)s * a.KV + hk) * b.sink_tiles + kt) * (b.far + 1) + piece + 1) * 2) * BRM * D + r * D;
      float* pv = pk + BRM * D;
#pragma unroll
      for (int c = 0; c < Sh::DC; ++c)
#pragma unroll
        for (int w = 0; w < Sh::W; ++w) {
          const int d = (c * BTX + tx) * Sh::W + w;
          pk[d] = ak[i][c][w] * a.scale;
          pv[d] = av[i][c][w];
        }
    } else if (key < a.tokens) {
      T* ok = dk + s * b.dks[0] + hk * b.dks[1] + (int64_t)key * b.dks[2];
      T* ov = dv + s * b.dvs[0] + hk * b.dvs[1] + (int64_t)key * b.dvs[2];
#pragma unroll
      for (int c = 0; c < Sh::DC; ++c)
#pragma unroll
        for (int w = 0; w < Sh::W; ++w) {
          const int d = (c * BTX + tx) * Sh::W + w;
          ok[d * b.dks[3]] = Traits<T>::from_f(ak[i][c][w] * a.scale);
          ov[d * b.dvs[3]] = Traits<T>::from_f(av[i][c][w]);
        }
    }
  }
}

// dK and dV of the keys of sink tiles: window part and far pieces added in order.
template <typename T>
__global__ void __launch_bounds__(256) local_far_sum(T* dk, T* dv, const LocalBwdArgs b, int key_tile) {
  const LocalArgs& a = b.f;
  const int s = blockIdx.z, hk = blockIdx.y;
  const int per_row = a.D, idx = blockIdx.x * blockDim.x + threadIdx.x;
  const int key = idx / per_row, d = idx % per_row;
  pdl_wait();
  if (key >= b.sink_tiles * key_tile || key >= a.tokens) return;
  const int64_t tile = ((int64_t)s * a.KV + hk) * b.sink_tiles + key / key_tile;
  const float* p = b.part + tile * (b.far + 1) * 2 * key_tile * a.D + (int64_t)(key % key_tile) * a.D + d;
  float sk = 0.f, sv = 0.f;
  for (int f = 0; f <= b.far; ++f, p += 2 * (int64_t)key_tile * a.D) {
    sk += p[0];
    sv += p[(int64_t)key_tile * a.D];
  }
  dk[s * b.dks[0] + hk * b.dks[1] + (int64_t)key * b.dks[2] + d * b.dks[3]] = Traits<T>::from_f(sk);
  dv[s * b.dvs[0] + hk * b.dvs[1] + (int64_t)key * b.dvs[2] + d * b.dvs[3]] = Traits<T>::from_f(sv);
}

template <typename Fn>
int dispatch_head(int D, Fn&& fn) {
  switch (D) {
    case 16: return fn(std::integral_constant<int, 16>{});
    case 32: return fn(std::integral_constant<int, 32>{});
    case 64: return fn(std::integral_constant<int, 64>{});
    case 128: return fn(std::integral_constant<int, 128>{});
  }
  set_error("local attention: head size %d not in {16,32,64,128}", D);
  return TB200_ERR_UNSUPPORTED;
}

template <typename Kernel>
int optin(Kernel kern, int bytes, std::atomic<unsigned long long>& done, const char* who) {
  const cudaError_t e = smem_optin_per_device(done, reinterpret_cast<const void*>(kern), bytes);
  if (e == cudaSuccess) return 0;
  set_error("%s: cudaFuncSetAttribute failed: %s", who, cudaGetErrorString(e));
  return (int)e;
}

template <typename T, int D, int RM, int TX>
int launch_fwd(T* out, float* lse, const T* q, const T* k, const T* v, const LocalArgs& a, int max_q, cudaStream_t st) {
  using Sh = Shape<D, RM, KEY_TILE, TX>;
  constexpr int SMEM = ((RM + 2 * KEY_TILE) * Sh::LD + (D >= 64 ? 0 : RM * (KEY_TILE + 4))) * 4;
  auto kern = local_fwd_simt<T, D, RM, TX>;
  static std::atomic<unsigned long long> done{0};
  if (int rc = optin(kern, SMEM, done, "local_fwd_simt")) return rc;
  const int qvec = rows_vectorised<T>(q, a.qs), kvec = rows_vectorised<T>(k, a.ks) && rows_vectorised<T>(v, a.vs);
  // (list form: no sequence has more tiles than its tokens fill, and one that is not full)
  const int64_t tiles = a.before ? a.tokens / (RM / a.G) + a.n : ceil_div(max_q, RM / a.G);
  const dim3 grid((unsigned)tiles, (unsigned)a.KV, (unsigned)(a.before ? 1 : a.n * a.splits));
  kern<<<grid, Sh::THREADS, SMEM, st>>>(out, lse, q, k, v, a, qvec, kvec);
  return launch_status("local_fwd_simt");
}

}  // namespace

int local_simt_key_tile() { return KEY_TILE; }

int launch_local_fwd_simt(void* out, float* lse, const void* q, const void* k, const void* v, const LocalArgs& a,
                          int max_q, int dtype, cudaStream_t st) {
  return dispatch_dtype(dtype, [&](auto tag) -> int {
    using T = decltype(tag);
    return dispatch_head(a.D, [&](auto d) -> int {
      constexpr int D = decltype(d)::value;
      // few rows: tiles of 16 rows (32 threads along the keys where the head size allows)
      if (local_simt_row_tile(a, max_q) == 16)
        return launch_fwd<T, D, 16, (D >= 32 ? 32 : 16)>((T*)out, lse, (const T*)q, (const T*)k, (const T*)v, a, max_q, st);
      return launch_fwd<T, D, 64, 16>((T*)out, lse, (const T*)q, (const T*)k, (const T*)v, a, max_q, st);
    });
  });
}

int launch_local_combine(void* out, const LocalArgs& a, int max_q, int row_tokens, int key_tile, int dtype, cudaStream_t st) {
  return dispatch_dtype(dtype, [&](auto tag) -> int {
    using T = decltype(tag);
    return dispatch_head(a.D, [&](auto d) -> int {
      constexpr int D = decltype(d)::value;
      const dim3 grid((unsigned)ceil_div((int64_t)max_q * a.H, 8), 1, (unsigned)a.n);
      (void)launch_pdl(local_combine<T, D>, grid, dim3(256), 0, st, false, (T*)out, a, row_tokens, key_tile);
      return launch_status("local_combine");
    });
  });
}

int launch_local_delta(float* delta, const void* out, const void* dout, const int64_t* dos, const LocalArgs& a, int dtype,
                       cudaStream_t st) {
  return dispatch_dtype(dtype, [&](auto tag) -> int {
    using T = decltype(tag);
    LocalBwdArgs b;
    for (int i = 0; i < 4; ++i) b.dos[i] = dos[i];
    local_delta<T><<<(unsigned)ceil_div((int64_t)a.n * a.H * a.tokens, 8), 256, 0, st>>>(delta, (const T*)out, (const T*)dout, a, b);
    return launch_status("local_delta");
  });
}

int launch_local_bwd_simt(void* dq, void* dk, void* dv, const void* dout, const void* q, const void* k, const void* v,
                          const float* lse, const float* delta, const LocalBwdArgs& b, int dtype, cudaStream_t st) {
  const LocalArgs& a = b.f;
  return dispatch_dtype(dtype, [&](auto tag) -> int {
    using T = decltype(tag);
    return dispatch_head(a.D, [&](auto d) -> int {
      constexpr int D = decltype(d)::value;
      constexpr int DQ_SMEM = ((2 * BRM + 2 * BRS) * (D + 4) + BRM * (BRS + 4)) * 4;
      constexpr int DKV_SMEM = DQ_SMEM + (BRM * (BRS + 4) + 2 * BRS) * 4;
      const int qvec = rows_vectorised<T>(q, a.qs) && rows_vectorised<T>(dout, b.dos);
      const int kvec = rows_vectorised<T>(k, a.ks) && rows_vectorised<T>(v, a.vs);
      auto kq = local_dq_simt<T, D>;
      auto kkv = local_dkv_simt<T, D>;
      static std::atomic<unsigned long long> done_q{0}, done_kv{0};
      if (int rc = optin(kq, DQ_SMEM, done_q, "local_dq_simt")) return rc;
      if (int rc = optin(kkv, DKV_SMEM, done_kv, "local_dkv_simt")) return rc;
      kq<<<dim3((unsigned)ceil_div(a.tokens, BRM / a.G), (unsigned)a.KV, (unsigned)a.n), 256, DQ_SMEM, st>>>(
          (T*)dq, (const T*)dout, (const T*)q, (const T*)k, (const T*)v, lse, delta, b, qvec, kvec);
      if (int rc = launch_status("local_dq_simt")) return rc;
      const int tiles = (a.tokens + BRM - 1) / BRM;
      kkv<<<dim3((unsigned)(tiles + b.sink_tiles * b.far), (unsigned)a.KV, (unsigned)a.n), 256, DKV_SMEM, st>>>(
          (T*)dk, (T*)dv, (const T*)dout, (const T*)q, (const T*)k, (const T*)v, lse, delta, b, qvec, kvec);
      return launch_status("local_dkv_simt");
    });
  });
}

int launch_local_far_sum(void* dk, void* dv, const LocalBwdArgs& b, int key_tile, int dtype, cudaStream_t st) {
  return dispatch_dtype(dtype, [&](auto tag) -> int {
    using T = decltype(tag);
    const dim3 grid((unsigned)ceil_div((int64_t)b.sink_tiles * key_tile * b.f.D, 256), (unsigned)b.f.KV, (unsigned)b.f.n);
    (void)launch_pdl(local_far_sum<T>, grid, dim3(256), 0, st, false, (T*)dk, (T*)dv, b, key_tile);
    return launch_status("local_far_sum");
  });
}

}  // namespace tb200
