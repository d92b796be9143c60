// What stands between two blocks of a transformer, in one pass: the norm after a block, its gate,
// the scaled residual and the norm before the next block, forward and backward.
//
//   n = x / (rms(x) + eps) * w1        (w1 null: n = x, no norm after the block)
//   y = a * r + g * n                  (g null: 1)
//   h = y / (rms(y) + eps) * w2        rms(v) = sqrt(mean(v^2)), eps outside the root as in RMSNorm
//
// Backward, with i1 = 1 / (rms(x) + eps), i2 = 1 / (rms(y) + eps), N = cols:
//   dY = dy + dh w2 i2 - y k2          k2 = sum(dh w2 y) i2^2 / (N rms(y))
//   dr = a dY
//   t  = dY g w1;  dx = t i1 - x k1    k1 = sum(t x) i1^2 / (N rms(x))
//   dw2 = sum_rows dh y i2;  with A = sum_rows dY x i1 over the rows that share a gate vector:
//   dg = w1 A,  dw1 = sum over the gate vectors g A
// (a row of zeros has rms 0: its k is 0, the limit of the first-order term). y is recomputed from x
// and r in fp32, so h and every gradient follow the unrounded y and no copy of it is kept.
//
// The gate is absent, one vector for all rows, one per `rows_per_gate` rows (a sequence), or one per
// row. Statistics, sums and column sums are fp32; every output is rounded once.
//
// The column sums are deterministic: part c of n takes the rows [c rows / n, (c+1) rows / n) and adds
// them in order; where its rows belong to several gate vectors, each stretch of one vector gets a
// partial row of its own, numbered c + (index of the vector), which no other stretch shares; a last
// kernel adds the partial rows in that order.
//
// Bounded by HBM: forward reads x, r and writes y, h (4 e bytes an element of e bytes); backward
// reads x, r, dy, dh and writes dx, dr (6 e).
#include <type_traits>

#include "ptx.cuh"
#include "row_common.cuh"

namespace tb200 {
namespace {

struct ResNormArgs {
  int64_t rows = 0;
  int64_t cols = 0;
  int64_t rows_per_gate = 0;  // 0: one vector for all rows (or no gate)
  float scale = 1.f, eps = 0.f;
};

__device__ inline int64_t gate_index(const ResNormArgs& a, int64_t row) {
  return a.rows_per_gate > 0 ? row / a.rows_per_gate : 0;
}
__host__ __device__ inline int64_t part_begin(int64_t c, int64_t n, int64_t rows) { return c * rows / n; }
// the part that row belongs to
__host__ __device__ inline int64_t part_of(int64_t row, int64_t n, int64_t rows) { return ((row + 1) * n - 1) / rows; }

__device__ inline float block_sum(float v, float* slot) {
  v = warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) slot[threadIdx.x >> 5] = v;
  __syncthreads();
  const int nwarps = (blockDim.x + 31) >> 5;
  float r = (threadIdx.x & 31) < nwarps ? slot[threadIdx.x & 31] : 0.f;
  return warp_sum(r);
}

// ------------------------------------------------------------------ any width and alignment, from 4097 columns on
// One CTA per row; the row is read again (from L1 or L2) for every pass.
template <typename T>
__global__ void __launch_bounds__(256)
    resnorm_fwd_generic(T* h, T* y, float* rms1, float* rms2, const T* x, const T* r, const T* w1, const T* w2,
                        const T* gate, ResNormArgs a) {
  using Tr = Traits<T>;
  __shared__ float slot[32];
  const int64_t row = blockIdx.x, off = row * a.cols;
  const T* g = gate ? gate + gate_index(a, row) * a.cols : nullptr;
  float i1 = 1.f;
  if (w1) {
    float s = 0.f;
    for (int64_t c = threadIdx.x; c < a.cols; c += blockDim.x) {
      const float v = Tr::to_f(x[off + c]);
      s = fmaf(v, v, s);
    }
    const float rms = sqrtf(block_sum(s, slot) / (float)a.cols);
    i1 = 1.f / (rms + a.eps);
    if (rms1 && threadIdx.x == 0) rms1[row] = rms;
  }
  auto y_at = [&](int64_t c) {
    float n = Tr::to_f(x[off + c]);
    if (w1) n = n * i1 * Tr::to_f(w1[c]);
    if (g) n *= Tr::to_f(g[c]);
    return fmaf(a.scale, Tr::to_f(r[off + c]), n);
  };
  float s = 0.f;
  for (int64_t c = threadIdx.x; c < a.cols; c += blockDim.x) {
    const float v = y_at(c);
    s = fmaf(v, v, s);
    y[off + c] = Tr::from_f(v);
  }
  const float rms = sqrtf(block_sum(s, slot) / (float)a.cols);
  const float i2 = 1.f / (rms + a.eps);
  if (rms2 && threadIdx.x == 0) rms2[row] = rms;
  for (int64_t c = threadIdx.x; c < a.cols; c += blockDim.x) h[off + c] = Tr::from_f(y_at(c) * i2 * Tr::to_f(w2[c]));
}

// Part c of the rows; the column sums accumulate in the part's own partial rows.
template <typename T>
__global__ void __launch_bounds__(256)
    resnorm_bwd_generic(T* dx, T* dr, T* dgate_rows, float* part_a, float* part_b, const T* dh, const T* dy, const T* x,
                        const T* r, const T* w1, const T* w2, const T* gate, const float* rms1, const float* rms2,
                        ResNormArgs a, int per_row) {
  using Tr = Traits<T>;
  __shared__ float slot[32];
  const int64_t n = gridDim.x, begin = part_begin(blockIdx.x, n, a.rows), end = part_begin(blockIdx.x + 1, n, a.rows);
  float* pb = part_b ? part_b + (int64_t)blockIdx.x * a.cols : nullptr;
  int64_t current = -1;
  float* pa = nullptr;
  for (int64_t row = begin; row < end; ++row) {
    const int64_t off = row * a.cols, gi = gate_index(a, row);
    const T* g = gate ? gate + gi * a.cols : nullptr;
    if (part_a && (row == begin || (!per_row && gi != current))) {
      current = gi;
      pa = part_a + ((int64_t)blockIdx.x + (per_row ? 0 : gi)) * a.cols;
      for (int64_t c = threadIdx.x; c < a.cols; c += blockDim.x) pa[c] = 0.f;
    }
    if (pb && row == begin)
      for (int64_t c = threadIdx.x; c < a.cols; c += blockDim.x) pb[c] = 0.f;
    const float m1 = w1 ? rms1[row] : 1.f, m2 = rms2[row];
    const float i1 = w1 ? 1.f / (m1 + a.eps) : 1.f, i2 = 1.f / (m2 + a.eps);
    auto y_at = [&](int64_t c, float xv) {
      float v = w1 ? xv * i1 * Tr::to_f(w1[c]) : xv;
      if (g) v *= Tr::to_f(g[c]);
      return fmaf(a.scale, Tr::to_f(r[off + c]), v);
    };
    float s = 0.f;
    if (dh)
      for (int64_t c = threadIdx.x; c < a.cols; c += blockDim.x)
        s = fmaf(Tr::to_f(dh[off + c]) * Tr::to_f(w2[c]), y_at(c, Tr::to_f(x[off + c])), s);
    const float s2 = block_sum(s, slot);
    const float k2 = m2 > 0.f ? s2 * i2 * i2 / ((float)a.cols * m2) : 0.f;
    auto dY_at = [&](int64_t c, float yv) {
      float v = dy ? Tr::to_f(dy[off + c]) : 0.f;
      if (dh) v += Tr::to_f(dh[off + c]) * Tr::to_f(w2[c]) * i2 - yv * k2;
      return v;
    };
    float k1 = 0.f;
    if (w1) {
      s = 0.f;
      for (int64_t c = threadIdx.x; c < a.cols; c += blockDim.x) {
        const float xv = Tr::to_f(x[off + c]);
        float t = dY_at(c, y_at(c, xv)) * Tr::to_f(w1[c]);
        if (g) t *= Tr::to_f(g[c]);
        s = fmaf(t, xv, s);
      }
      const float s1 = block_sum(s, slot);
      k1 = m1 > 0.f ? s1 * i1 * i1 / ((float)a.cols * m1) : 0.f;
    }
    for (int64_t c = threadIdx.x; c < a.cols; c += blockDim.x) {
      const float xv = Tr::to_f(x[off + c]), yv = y_at(c, xv), d = dY_at(c, yv);
      const float wv = w1 ? Tr::to_f(w1[c]) : 1.f, gv = g ? Tr::to_f(g[c]) : 1.f;
      dr[off + c] = Tr::from_f(a.scale * d);
      dx[off + c] = Tr::from_f(d * gv * wv * i1 - xv * k1);
      const float ax = d * xv * i1;
      if (dgate_rows) dgate_rows[off + c] = Tr::from_f(ax * wv);
      if (pa) pa[c] += per_row ? ax * gv : ax;
      if (pb && dh) pb[c] = fmaf(Tr::to_f(dh[off + c]), yv * i2, pb[c]);
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------------ rows of up to 4096 columns, any alignment
// Widths that are no multiple of 16 bytes, unaligned views: a CTA holds a row in registers, C columns a thread,
// a block apart, and reads and writes each element once, one element at a time. At 1665 rows of 1021 fp32 columns
// (27 MB forward, 41 backward) forward and backward take 9 and 17 us; the kernels above, which read a row again for
// every pass and keep the column sums in memory, take 15 and 54.
template <typename T, int C>
__global__ void __launch_bounds__(512)
    resnorm_fwd_cols(T* __restrict__ h, T* __restrict__ y, float* __restrict__ rms1, float* __restrict__ rms2,
                     const T* __restrict__ x, const T* __restrict__ r, const T* __restrict__ w1, const T* __restrict__ w2,
                     const T* __restrict__ gate, const ResNormArgs a) {
  using Tr = Traits<T>;
  __shared__ float slot[32];
  const int64_t row = blockIdx.x, off = row * a.cols;
  const T* g = gate ? gate + gate_index(a, row) * a.cols : nullptr;
  float v[C], rv[C], w[C];
#pragma unroll
  for (int k = 0; k < C; ++k) {
    const int c = threadIdx.x + k * blockDim.x;
    const bool live = c < a.cols;
    v[k] = live ? Tr::to_f(x[off + c]) : 0.f;
    rv[k] = live ? Tr::to_f(r[off + c]) : 0.f;
    w[k] = live ? (w1 ? Tr::to_f(w1[c]) : 1.f) * (g ? Tr::to_f(g[c]) : 1.f) : 0.f;
  }
  float i1 = 1.f;
  if (w1) {
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < C; ++k) s = fmaf(v[k], v[k], s);
    const float rms = sqrtf(block_sum(s, slot) / (float)a.cols);
    i1 = 1.f / (rms + a.eps);
    if (rms1 && threadIdx.x == 0) rms1[row] = rms;
  }
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < C; ++k) {
    v[k] = fmaf(a.scale, rv[k], v[k] * i1 * w[k]);
    s = fmaf(v[k], v[k], s);
  }
#pragma unroll
  for (int k = 0; k < C; ++k) w[k] = threadIdx.x + k * blockDim.x < a.cols ? Tr::to_f(w2[threadIdx.x + k * blockDim.x]) : 0.f;
  const float rms = sqrtf(block_sum(s, slot) / (float)a.cols), i2 = 1.f / (rms + a.eps);
  if (rms2 && threadIdx.x == 0) rms2[row] = rms;
#pragma unroll
  for (int k = 0; k < C; ++k) {
    const int c = threadIdx.x + k * blockDim.x;
    if (c < a.cols) {
      y[off + c] = Tr::from_f(v[k]);
      h[off + c] = Tr::from_f(v[k] * i2 * w[k]);
    }
  }
}

// A part of the rows; the next row is read while the sums of this one are formed.
template <typename T, int C>
__global__ void __launch_bounds__(512)
    resnorm_bwd_cols(T* __restrict__ dx, T* __restrict__ dr, T* __restrict__ dgate_rows, float* __restrict__ part_a,
                     float* __restrict__ part_b, const T* __restrict__ dh, const T* __restrict__ dy, const T* __restrict__ x,
                     const T* __restrict__ r, const T* __restrict__ w1, const T* __restrict__ w2, const T* __restrict__ gate,
                     const float* __restrict__ rms1, const float* __restrict__ rms2, const ResNormArgs a, int per_row) {
  using Tr = Traits<T>;
  __shared__ float slot[32];
  const int64_t n = gridDim.x, begin = part_begin(blockIdx.x, n, a.rows), end = part_begin(blockIdx.x + 1, n, a.rows);
  float W1[C], W2[C], G[C], acc_a[C], acc_b[C], nx[C], nr[C], nh[C], ny[C], nm1 = 1.f, nm2 = 1.f;
  auto load = [&](int64_t row) {
    const int64_t off = row * a.cols;
#pragma unroll
    for (int k = 0; k < C; ++k) {
      const int c = threadIdx.x + k * blockDim.x;
      const bool live = c < a.cols;
      nx[k] = live ? Tr::to_f(x[off + c]) : 0.f;
      nr[k] = live ? Tr::to_f(r[off + c]) : 0.f;
      nh[k] = live && dh ? Tr::to_f(dh[off + c]) : 0.f;
      ny[k] = live && dy ? Tr::to_f(dy[off + c]) : 0.f;
    }
    if (w1) nm1 = rms1[row];
    nm2 = rms2[row];
  };
  auto flush = [&](float* part, const float (&acc)[C]) {
#pragma unroll
    for (int k = 0; k < C; ++k) {
      const int c = threadIdx.x + k * blockDim.x;
      if (c < a.cols) part[c] = acc[k];
    }
  };
#pragma unroll
  for (int k = 0; k < C; ++k) {
    const int c = threadIdx.x + k * blockDim.x;
    const bool live = c < a.cols;
    W1[k] = live && w1 ? Tr::to_f(w1[c]) : 1.f;
    W2[k] = live ? Tr::to_f(w2[c]) : 0.f;
    G[k] = 1.f;
    acc_a[k] = acc_b[k] = 0.f;
  }
  int64_t current = -1;
  if (begin < end) load(begin);
  for (int64_t row = begin; row < end; ++row) {
    const int64_t gi = gate_index(a, row);
    if (gate && gi != current) {
      if (part_a && !per_row && current >= 0) {
        flush(part_a + ((int64_t)blockIdx.x + current) * a.cols, acc_a);
#pragma unroll
        for (int k = 0; k < C; ++k) acc_a[k] = 0.f;
      }
#pragma unroll
      for (int k = 0; k < C; ++k) {
        const int c = threadIdx.x + k * blockDim.x;
        if (c < a.cols) G[k] = Tr::to_f(gate[gi * a.cols + c]);
      }
    }
    current = gi;
    const float m1 = nm1, m2 = nm2, i1 = w1 ? 1.f / (m1 + a.eps) : 1.f, i2 = 1.f / (m2 + a.eps);
    float xv[C], yv[C], hv[C], d[C], s = 0.f;
#pragma unroll
    for (int k = 0; k < C; ++k) {
      xv[k] = nx[k];
      hv[k] = nh[k];
      d[k] = ny[k];
      yv[k] = fmaf(a.scale, nr[k], xv[k] * i1 * W1[k] * G[k]);
      s = fmaf(hv[k] * W2[k], yv[k], s);
    }
    if (row + 1 < end) load(row + 1);
    float k2 = 0.f;
    if (dh) {
      const float s2 = block_sum(s, slot);
      k2 = m2 > 0.f ? s2 * i2 * i2 / ((float)a.cols * m2) : 0.f;
    }
    s = 0.f;
#pragma unroll
    for (int k = 0; k < C; ++k) {
      d[k] += hv[k] * W2[k] * i2 - yv[k] * k2;
      s = fmaf(d[k] * W1[k] * G[k], xv[k], s);
    }
    float k1 = 0.f;
    if (w1) {
      const float s1 = block_sum(s, slot);
      k1 = m1 > 0.f ? s1 * i1 * i1 / ((float)a.cols * m1) : 0.f;
    }
    const int64_t off = row * a.cols;
#pragma unroll
    for (int k = 0; k < C; ++k) {
      const int c = threadIdx.x + k * blockDim.x;
      const float ax = d[k] * xv[k] * i1;
      acc_a[k] += per_row ? ax * G[k] : ax;
      acc_b[k] = fmaf(hv[k], yv[k] * i2, acc_b[k]);
      if (c < a.cols) {
        dr[off + c] = Tr::from_f(a.scale * d[k]);
        dx[off + c] = Tr::from_f(d[k] * G[k] * W1[k] * i1 - xv[k] * k1);
        if (dgate_rows) dgate_rows[off + c] = Tr::from_f(ax * W1[k]);
      }
    }
  }
  if (part_a) flush(part_a + ((int64_t)blockIdx.x + (per_row ? 0 : current)) * a.cols, acc_a);
  if (part_b) flush(part_b + (int64_t)blockIdx.x * a.cols, acc_b);
}

// ------------------------------------------------------------------ rows of 16-byte vectors
// Forward: a row stays in registers (a warp or a CTA owns it, RowPlan); x, r, the weights and the gate
// are requested together before the first reduction. 8192 x 4096 bf16: 48 us, 5.6 TB/s.
template <typename T, int CHUNKS, bool CTA_ROW>
__global__ void __launch_bounds__(CTA_ROW ? 512 : 256, CTA_ROW ? 2 : 4)
    resnorm_fwd_vec(T* __restrict__ h, T* __restrict__ y, float* __restrict__ rms1, float* __restrict__ rms2,
                    const T* __restrict__ x, const T* __restrict__ r, const T* __restrict__ w1, const T* __restrict__ w2,
                    const T* __restrict__ gate, const ResNormArgs a) {
  constexpr int VEC = Traits<T>::VEC, PAIRS = VEC / 2;
  __shared__ float slot[64];
  int phase = 0;
  RowThread<CTA_ROW> rt;
  const int cols = (int)a.cols;
  const float inv_n = 1.f / (float)cols;
  pdl_wait();
  pdl_release();
  for (int64_t row = rt.first_row(); row < a.rows; row += rt.row_step()) {
    const int64_t off = row * a.cols;
    const T* g = gate ? gate + gate_index(a, row) * a.cols : nullptr;
    uint4 xr[CHUNKS], rr[CHUNKS];
    uint64_t v[CHUNKS][PAIRS];
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      const int col = rt.template col<VEC>(c);
      const bool in = col < cols;
      xr[c] = in ? ld_stream(x + off + col) : make_uint4(0, 0, 0, 0);
      rr[c] = in ? ld_stream(r + off + col) : make_uint4(0, 0, 0, 0);
    }
    float i1 = 1.f;
    if (w1) {
      uint64_t s2 = 0ull;
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) {
        unpack2<T>(xr[c], v[c]);
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) s2 = am::fma2(v[c][i], v[c][i], s2);
      }
      const float rms = sqrtf(row_reduce<CTA_ROW, false>(hsum2(s2), slot, phase) * inv_n);
      i1 = 1.f / (rms + a.eps);
      if (rms1 && rt.tid == 0) rms1[row] = rms;
    }
    const uint64_t i1_2 = splat2(i1), scale2 = splat2(a.scale);
    uint64_t s2 = 0ull;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      const int col = rt.template col<VEC>(c);
      unpack2<T>(xr[c], v[c]);
      if (col < cols) {
        uint64_t t[PAIRS];
        if (w1) {
          unpack2<T>(ld_cached(w1 + col), t);
#pragma unroll
          for (int i = 0; i < PAIRS; ++i) v[c][i] = am::mul2(am::mul2(v[c][i], i1_2), t[i]);
        }
        if (g) {
          unpack2<T>(ld_cached(g + col), t);
#pragma unroll
          for (int i = 0; i < PAIRS; ++i) v[c][i] = am::mul2(v[c][i], t[i]);
        }
        unpack2<T>(rr[c], t);
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) {
          v[c][i] = am::fma2(scale2, t[i], v[c][i]);
          s2 = am::fma2(v[c][i], v[c][i], s2);
        }
        st_stream(y + off + col, pack2<T>(v[c]));
      }
    }
    const float rms = sqrtf(row_reduce<CTA_ROW, false>(hsum2(s2), slot, phase) * inv_n);
    const uint64_t i2_2 = splat2(1.f / (rms + a.eps));
    if (rms2 && rt.tid == 0) rms2[row] = rms;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      const int col = rt.template col<VEC>(c);
      if (col < cols) {
        uint64_t t[PAIRS];
        unpack2<T>(ld_cached(w2 + col), t);
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) v[c][i] = am::mul2(am::mul2(v[c][i], i2_2), t[i]);
        st_stream(h + off + col, pack2<T>(v[c]));
      }
    }
  }
}

// Backward: a CTA walks its part of the rows. x, r, dy and dh of a row arrive in a ring of shared-memory
// stages by bulk copies (one thread issues them stages ahead, so loads stay in flight across the two
// reductions of a row). A thread keeps its columns' w2 and gate * w1 (as long as the gate vector stays the
// same) and their column sums in registers as fp32 pairs; per element of the four inputs that leaves a
// conversion and about eight two-lane operations, where weights unpacked anew for every row and divisions
// per thread bounded the kernel at 2.8 TB/s. 8192 x 4096 bf16: 93 us, 4.3 TB/s, with half of the issue slots
// used and two block-wide sums a row in between; joining the parts another 9.
__device__ inline float reciprocal(float v) {  // (one unit in the last place)
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(v));
  return y;
}
template <typename T, int CHUNKS, int THREADS>
__global__ void __launch_bounds__(THREADS, CHUNKS <= 2 ? 2 : 1)
    resnorm_bwd_vec(T* __restrict__ dx, T* __restrict__ dr, T* __restrict__ dgate_rows, float* __restrict__ part_a,
                    float* __restrict__ part_b, const T* __restrict__ dh, const T* __restrict__ dy, const T* __restrict__ x,
                    const T* __restrict__ r, const T* __restrict__ w1, const T* __restrict__ w2, const T* __restrict__ gate,
                    const float* __restrict__ rms1, const float* __restrict__ rms2, const ResNormArgs a, int per_row,
                    int stages, int* status, const WaitTest test) {
  constexpr int VEC = Traits<T>::VEC, PAIRS = VEC / 2;
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ float slot[64];
  __shared__ uint64_t full[4];
  __shared__ uint32_t abort_words[3];  // abort flag, wait limit (ptx::mbar_wait), rows requested
  volatile uint32_t* abort_flag = abort_words;
  const int cols = (int)a.cols;
  const int bytes = cols * (int)sizeof(T);
  const int64_t n = gridDim.x, begin = part_begin(blockIdx.x, n, a.rows), end = part_begin(blockIdx.x + 1, n, a.rows);
  const int count = (int)(end - begin);
  const float inv_n = 1.f / (float)cols;
  int phase = 0;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 4; ++i) ptx::mbar_init(&full[i], 1);
    abort_flag[0] = abort_flag[2] = 0;
    abort_flag[1] = test.units;
    ptx::fence_barrier_init();
  }
  __syncthreads();
  pdl_wait();
  pdl_release();
  const int tensors = 2 + (dh ? 1 : 0) + (dy ? 1 : 0);
  auto request = [&](int i, int st) {  // (thread 0) row begin + i into stage st
    abort_flag[2] = i + 1;
    if (i == test.skip && blockIdx.x == 0) return;  // (test hook)
    uint8_t* dst = ring + (size_t)st * 4 * bytes;
    const int64_t off = (begin + i) * a.cols;
    ptx::mbar_expect_tx(&full[st], (uint32_t)(tensors * bytes));
    auto copy = [&](const T* src, int k) {
      asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                       ptx::smem_u32(dst + (size_t)k * bytes)),
                   "l"(src + off), "r"(bytes), "r"(ptx::smem_u32(&full[st]))
                   : "memory");
    };
    copy(x, 0);
    copy(r, 1);
    if (dh) copy(dh, 2);
    if (dy) copy(dy, 3);
  };
  if (threadIdx.x == 0)
    for (int i = 0; i < stages && i < count; ++i) request(i, i);

  uint64_t acc_a[CHUNKS][PAIRS], acc_b[CHUNKS][PAIRS], gw[CHUNKS][PAIRS], wv[CHUNKS][PAIRS];
  auto col_of = [&](int c) { return (c * (int)blockDim.x + (int)threadIdx.x) * VEC; };
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) acc_a[c][i] = acc_b[c][i] = gw[c][i] = wv[c][i] = 0ull;
    if (col_of(c) < cols) unpack2<T>(ld_cached(w2 + col_of(c)), wv[c]);
  }
  auto flush = [&](float* dst, uint64_t (&acc)[CHUNKS][PAIRS]) {
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      const int col = col_of(c);
      if (col < cols)
#pragma unroll
        for (int i = 0; i < PAIRS; i += 2) {
          float f0, f1, f2, f3;
          am::unpack2f(acc[c][i], f0, f1);
          am::unpack2f(acc[c][i + 1], f2, f3);
          *reinterpret_cast<float4*>(dst + col + i * 2) = make_float4(f0, f1, f2, f3);
          acc[c][i] = acc[c][i + 1] = 0ull;
        }
    }
  };
  int64_t current = -1;  // gate vector whose product with w1 is in gw
  int st = 0;
  uint32_t ring_phase = 0;
  float next1 = w1 ? rms1[begin] : 1.f, next2 = rms2[begin];
  for (int i = 0; i < count; ++i) {
    const int64_t row = begin + i, off = row * a.cols, gi = gate_index(a, row);
    if (gi != current) {
      if (part_a && !per_row && current >= 0) flush(part_a + ((int64_t)blockIdx.x + current) * a.cols, acc_a);
      current = gi;
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) {
        const int col = col_of(c);
        if (col >= cols) continue;
        uint64_t w[PAIRS];
        if (w1) unpack2<T>(ld_cached(w1 + col), gw[c]);
        if (gate) unpack2<T>(ld_cached(gate + gi * a.cols + col), w);
#pragma unroll
        for (int k = 0; k < PAIRS; ++k) {
          if (!w1) gw[c][k] = gate ? w[k] : splat2(1.f);
          else if (gate) gw[c][k] = am::mul2(gw[c][k], w[k]);
        }
      }
    }
    const float m1 = next1, m2 = next2;
    if (i + 1 < count) {  // (a row ahead)
      if (w1) next1 = rms1[row + 1];
      next2 = rms2[row + 1];
    }
    const float i1 = w1 ? reciprocal(m1 + a.eps) : 1.f, i2 = reciprocal(m2 + a.eps);
    const uint64_t i1_2 = splat2(i1), i2_2 = splat2(i2), scale2 = splat2(a.scale);
    const uint8_t* src = ring + (size_t)st * 4 * bytes;
    ptx::mbar_wait(&full[st], ring_phase, abort_flag, status, 161);
    // u = x i1, v = y, t = dh w2 i2 (then dY, then dY gate w1)
    uint64_t t[CHUNKS][PAIRS], u[CHUNKS][PAIRS], v[CHUNKS][PAIRS];
    uint4 dyr[CHUNKS];
    uint64_t s2 = 0ull;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      const int col = col_of(c);
      const bool in = col < cols;
      const uint8_t* at = src + col * (int)sizeof(T);
      const uint4 none = make_uint4(0, 0, 0, 0);
      unpack2<T>(in ? *reinterpret_cast<const uint4*>(at) : none, u[c]);
      unpack2<T>(in ? *reinterpret_cast<const uint4*>(at + bytes) : none, v[c]);
      dyr[c] = dy && in ? *reinterpret_cast<const uint4*>(at + 3 * (size_t)bytes) : none;
      unpack2<T>(dh && in ? *reinterpret_cast<const uint4*>(at + 2 * (size_t)bytes) : none, t[c]);
#pragma unroll
      for (int k = 0; k < PAIRS; ++k) {
        u[c][k] = am::mul2(u[c][k], i1_2);
        v[c][k] = am::fma2(u[c][k], gw[c][k], am::mul2(scale2, v[c][k]));
        t[c][k] = am::mul2(t[c][k], i2_2);
        acc_b[c][k] = am::fma2(t[c][k], v[c][k], acc_b[c][k]);
        t[c][k] = am::mul2(t[c][k], wv[c][k]);
        s2 = am::fma2(t[c][k], v[c][k], s2);
      }
    }
    // (the reduction's barrier also says that every thread has taken its part of the stage)
    const float sum2 = row_reduce<true, false>(hsum2(s2), slot, phase);
    if (threadIdx.x == 0 && i + stages < count && !abort_flag[0]) request(i + stages, st);  // (not after an expired wait)
    if (++st == stages) {
      st = 0;
      ring_phase ^= 1u;
    }
    // k2 = sum(dh w2 y) i2^2 / (N rms2); one factor i2 is in the sum
    const uint64_t nk2 = splat2(m2 > 0.f ? -(sum2 * i2 * inv_n * reciprocal(m2)) : 0.f);
    uint64_t s1 = 0ull;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      const int col = col_of(c);
      uint64_t w[PAIRS];
      unpack2<T>(dyr[c], w);
#pragma unroll
      for (int k = 0; k < PAIRS; ++k) {
        t[c][k] = am::fma2(v[c][k], nk2, am::add2(t[c][k], w[k]));
        v[c][k] = am::mul2(scale2, t[c][k]);
      }
      if (col < cols) st_stream(dr + off + col, pack2<T>(v[c]));
      if (per_row && col < cols) {  // a gate of its own: its gradient, and the sum A with the gate in it
        uint64_t g[PAIRS];
        unpack2<T>(ld_cached(gate + gi * a.cols + col), g);
        if (w1) unpack2<T>(ld_cached(w1 + col), w);
#pragma unroll
        for (int k = 0; k < PAIRS; ++k) {
          const uint64_t ax = am::mul2(t[c][k], u[c][k]);
          v[c][k] = w1 ? am::mul2(ax, w[k]) : ax;
          acc_a[c][k] = am::fma2(ax, g[k], acc_a[c][k]);
        }
        if (dgate_rows) st_stream(dgate_rows + off + col, pack2<T>(v[c]));
      }
#pragma unroll
      for (int k = 0; k < PAIRS; ++k) {
        if (!per_row) acc_a[c][k] = am::fma2(t[c][k], u[c][k], acc_a[c][k]);
        t[c][k] = am::mul2(t[c][k], gw[c][k]);
        s1 = am::fma2(t[c][k], u[c][k], s1);
      }
    }
    // dx = i1 (t - u k1'), k1' = sum(t x) i1 / (N rms1): sum(t u) / (N rms1) (w1 null: dx = t)
    uint64_t nk1 = 0ull;
    if (w1) {
      const float sum1 = row_reduce<true, false>(hsum2(s1), slot, phase);
      nk1 = splat2(m1 > 0.f ? -(sum1 * inv_n * reciprocal(m1) * (m1 + a.eps)) : 0.f);
    }
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      const int col = col_of(c);
#pragma unroll
      for (int k = 0; k < PAIRS; ++k) t[c][k] = am::mul2(i1_2, am::fma2(u[c][k], nk1, t[c][k]));
      if (col < cols) st_stream(dx + off + col, pack2<T>(t[c]));
    }
  }
  if (part_a) flush(part_a + ((int64_t)blockIdx.x + (per_row ? 0 : current)) * a.cols, acc_a);
  if (part_b) flush(part_b + (int64_t)blockIdx.x * a.cols, acc_b);
  // Every copy has landed before the CTA gives up its shared memory (without an expired wait all have been waited for).
  if (threadIdx.x == 0 && abort_flag[0])
    for (int requested = abort_flag[2], i = requested > stages ? requested - stages : 0; i < requested; ++i)
      ptx::mbar_wait_drain(&full[i % stages], (i / stages) & 1, abort_flag, status, 162);
}

// blockIdx.y 0: dw1 (and dgate where one vector serves all rows), 1: dw2, 2..: dgate of one vector each.
// Block (32, 32): threadIdx.x walks columns, threadIdx.y splits the partial rows.
template <typename T>
__global__ void __launch_bounds__(1024)
    resnorm_finalize(T* dw1, T* dw2, T* dgate, const float* part_a, const float* part_b, const T* w1, const T* gate,
                     int64_t n, ResNormArgs a, int gate_rows_done) {
  using Tr = Traits<T>;
  __shared__ float tile[32][33];
  pdl_wait();
  pdl_release();
  const int64_t col = (int64_t)blockIdx.x * 32 + threadIdx.x;
  const bool live = col < a.cols;
  const bool shared_gate = a.rows_per_gate == 0;  // one vector (or none) for all rows
  auto fold = [&](float acc) {
    tile[threadIdx.y][threadIdx.x] = acc;
    __syncthreads();
    float s = 0.f;
    if (threadIdx.y == 0)
#pragma unroll
      for (int i = 0; i < 32; ++i) s += tile[i][threadIdx.x];
    __syncthreads();
    return s;
  };
  if (blockIdx.y == 0) {
    if (!part_a) return;
    float acc = 0.f;
    if (live) {
      if (shared_gate || gate_rows_done) {
        for (int64_t p0 = threadIdx.y; p0 < n; p0 += 32 * 8) {
          float v[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = p0 + 32 * j < n ? part_a[(p0 + 32 * j) * a.cols + col] : 0.f;
#pragma unroll
          for (int j = 0; j < 8; ++j) acc += v[j];
        }
      } else {
        // by gate vectors (the parts of one take two divisions to find): all threads of a column on one vector's
        // parts, or, of 32 vectors and more, on one vector each
        const int64_t vectors = a.rows / a.rows_per_gate;
        const bool apart = vectors >= 32;
        for (int64_t g = apart ? threadIdx.y : 0; g < vectors; g += apart ? 32 : 1) {
          const int64_t c0 = part_of(g * a.rows_per_gate, n, a.rows), c1 = part_of((g + 1) * a.rows_per_gate - 1, n, a.rows);
          float sum = 0.f;
          for (int64_t c = apart ? c0 : c0 + threadIdx.y; c <= c1; c += apart ? 1 : 32) sum += part_a[(c + g) * a.cols + col];
          acc = fmaf(Tr::to_f(gate[g * a.cols + col]), sum, acc);
        }
      }
    }
    const float s = fold(acc);
    if (threadIdx.y == 0 && live) {
      if (shared_gate && !gate_rows_done) {
        if (dw1) dw1[col] = Tr::from_f(gate ? s * Tr::to_f(gate[col]) : s);
        if (dgate) dgate[col] = Tr::from_f(w1 ? s * Tr::to_f(w1[col]) : s);
      } else if (dw1) {
        dw1[col] = Tr::from_f(s);
      }
    }
  } else if (blockIdx.y == 1) {
    if (!part_b || !dw2) return;
    float acc = 0.f;
    if (live)
      for (int64_t p0 = threadIdx.y; p0 < n; p0 += 32 * 8) {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = p0 + 32 * j < n ? part_b[(p0 + 32 * j) * a.cols + col] : 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) acc += v[j];
      }
    const float s = fold(acc);
    if (threadIdx.y == 0 && live) dw2[col] = Tr::from_f(s);
  } else {
    const int64_t vectors = a.rows / a.rows_per_gate;
    for (int64_t g = blockIdx.y - 2; g < vectors; g += gridDim.y - 2) {
      const int64_t c0 = part_of(g * a.rows_per_gate, n, a.rows), c1 = part_of((g + 1) * a.rows_per_gate - 1, n, a.rows);
      float acc = 0.f;
      if (live)
        for (int64_t c = c0 + threadIdx.y; c <= c1; c += 32) acc += part_a[(c + g) * a.cols + col];
      const float s = fold(acc);
      if (threadIdx.y == 0 && live) dgate[g * a.cols + col] = Tr::from_f(w1 ? s * Tr::to_f(w1[col]) : s);
    }
  }
}

// Parts of the backward pass: enough CTAs to fill the GPU, at least eight rows each unless that
// leaves SMs without one (a part costs two partial rows of fp32 to write and read again).
int64_t backward_parts(int64_t rows, int64_t per_sm) {
  const int64_t sms = sm_count(), most = sms * per_sm;
  int64_t n = rows / 8;
  if (n < sms) n = sms;
  if (n > most) n = most;
  return n < rows ? n : rows;
}
constexpr int64_t MAX_PARTS_PER_SM = 16;

// Shape of the vector kernel of the backward pass (chunks 0: the generic one). Up to three rows of
// the four tensors are in flight per CTA; CTAs per SM by shared memory and 1024 threads.
struct BackwardPlan {
  int chunks = 0, threads = 0, stages = 0, per_sm = 0;
};
constexpr int RING_BYTES = 200 * 1024;
template <typename T>
BackwardPlan plan_backward(int64_t cols, bool ptrs_ok) {
  BackwardPlan p;
  constexpr int VEC = Traits<T>::VEC;
  if (!ptrs_ok || cols % VEC != 0 || cols > 2048 * VEC) return p;
  const int64_t vecs = cols / VEC, stage = 4 * cols * (int64_t)sizeof(T);
  // Two vectors a thread where the row has them: with one, half of a thread's instructions were the row's
  // two reductions, barriers and addresses.
  p.chunks = vecs <= 128 ? 1 : (vecs <= 512 ? 2 : 4);
  p.threads = (int)(ceil_div(ceil_div(vecs, p.chunks), 32) * 32);
  p.stages = (int)(RING_BYTES / stage < 3 ? RING_BYTES / stage : 3);
  int64_t per_sm = 220 * 1024 / (p.stages * stage + 2048);
  if (per_sm > 1024 / p.threads) per_sm = 1024 / p.threads;
  p.per_sm = (int)(per_sm < 1 ? 1 : (per_sm > MAX_PARTS_PER_SM ? MAX_PARTS_PER_SM : per_sm));
  return p;
}

// threads of the kernels for any alignment: 4 columns each up to 1024, then 8
int cols_threads(int64_t cols) { return cols > 2048 && cols <= 4096 ? 512 : 256; }

int check(const char* who, const ResNormArgs& a, const void* gate) {
  TB200_REQUIRE(a.rows >= 0 && a.cols > 0, TB200_ERR_INVALID, "%s: bad shape", who);
  TB200_REQUIRE(a.rows < (1ll << 31) && a.cols < (1ll << 30), TB200_ERR_UNSUPPORTED, "%s: more than 2^31 rows or 2^30 columns", who);
  TB200_REQUIRE(a.rows_per_gate >= 0 && (!gate || a.rows_per_gate == 0 || a.rows % a.rows_per_gate == 0), TB200_ERR_INVALID,
                "%s: rows_per_gate %lld does not divide %lld rows", who, (long long)a.rows_per_gate, (long long)a.rows);
  return 0;
}

}  // namespace
}  // namespace tb200

using namespace tb200;

extern "C" int tb200_gated_residual_rms_norm_fwd(void* h, void* y, float* rms1, float* rms2, const void* x, const void* r,
                                                 const void* w1, const void* w2, const void* gate, int64_t rows,
                                                 int64_t cols, int64_t rows_per_gate, float residual_scale, float eps,
                                                 int dtype, void* stream) {
  ResNormArgs a;
  a.rows = rows; a.cols = cols; a.rows_per_gate = gate ? rows_per_gate : 0;
  a.scale = residual_scale; a.eps = eps;
  if (int rc = check("gated_residual_rms_norm_fwd", a, gate)) return rc;
  if (rows == 0) return 0;
  TB200_REQUIRE(h && y && x && r && w2, TB200_ERR_INVALID, "gated_residual_rms_norm_fwd: null pointer");
  cudaStream_t st = (cudaStream_t)stream;
  return dispatch_dtype(dtype, [&](auto tag) -> int {
    using T = decltype(tag);
    const bool ok = aligned16(h) && aligned16(y) && aligned16(x) && aligned16(r) && aligned16(w2) && (!w1 || aligned16(w1)) &&
                    (!gate || aligned16(gate));
    const RowPlan plan = plan_rows<T>(cols, ok);
    if (plan.vec) {
      const int rc = dispatch_plan<T>(plan, [&](auto c, auto cta) -> int {
        (void)launch_pdl(resnorm_fwd_vec<T, decltype(c)::value, decltype(cta)::value>,
                         dim3((unsigned)ceil_div(rows, plan.rows_per_cta)), dim3(plan.threads), 0, st, false, (T*)h, (T*)y, rms1,
                         rms2, (const T*)x, (const T*)r, (const T*)w1, (const T*)w2, (const T*)gate, a);
        return launch_status("resnorm_fwd_vec");
      });
      if (rc == 0) note_kernel("row_vec", 1);
      return rc;
    }
    auto kern = cols > 4096 ? resnorm_fwd_generic<T> : (cols <= 1024 ? resnorm_fwd_cols<T, 4> : resnorm_fwd_cols<T, 8>);
    kern<<<(unsigned)rows, cols_threads(cols), 0, st>>>((T*)h, (T*)y, rms1, rms2, (const T*)x, (const T*)r, (const T*)w1,
                                                        (const T*)w2, (const T*)gate, a);
    const int rc = launch_status("resnorm_fwd_cols");
    if (rc == 0) note_kernel("row_generic", 1);
    return rc;
  });
}

extern "C" size_t tb200_gated_residual_rms_norm_bwd_workspace(int64_t rows, int64_t cols, int64_t rows_per_gate) {
  if (rows <= 0 || cols <= 0) return 0;
  const int64_t n = backward_parts(rows, MAX_PARTS_PER_SM);
  const int64_t vectors = rows_per_gate > 1 ? rows / rows_per_gate : 1;
  return (size_t)(2 * n + vectors) * (size_t)cols * sizeof(float);
}

extern "C" int tb200_gated_residual_rms_norm_bwd(void* dx, void* dr, void* dw1, void* dw2, void* dgate, const void* dh,
                                                 const void* dy, const void* x, const void* r, const void* w1,
                                                 const void* w2, const void* gate, const float* rms1, const float* rms2,
                                                 void* workspace, size_t workspace_bytes, int64_t rows, int64_t cols,
                                                 int64_t rows_per_gate, float residual_scale, float eps, int dtype,
                                                 void* stream) {
  ResNormArgs a;
  a.rows = rows; a.cols = cols; a.rows_per_gate = gate ? rows_per_gate : 0;
  a.scale = residual_scale; a.eps = eps;
  if (int rc = check("gated_residual_rms_norm_bwd", a, gate)) return rc;
  TB200_REQUIRE(!dgate || gate, TB200_ERR_INVALID, "gated_residual_rms_norm_bwd: dgate without gate");
  TB200_REQUIRE(!dw1 || w1, TB200_ERR_INVALID, "gated_residual_rms_norm_bwd: dw1 without w1");
  cudaStream_t st = (cudaStream_t)stream;
  if (rows == 0) {  // sums over no rows
    const size_t bytes = (size_t)cols * dtype_size(dtype);
    if (int rc = zero_fill(dw1, bytes, st, "gated_residual_rms_norm_bwd")) return rc;
    if (int rc = zero_fill(dw2, bytes, st, "gated_residual_rms_norm_bwd")) return rc;
    return a.rows_per_gate ? 0 : zero_fill(dgate, bytes, st, "gated_residual_rms_norm_bwd");
  }
  TB200_REQUIRE(dx && dr && (dh || dy) && x && r && w2 && rms2 && (!w1 || rms1), TB200_ERR_INVALID,
                "gated_residual_rms_norm_bwd: null pointer");
  const bool per_row = gate && rows_per_gate == 1;
  const bool want_a = dw1 || (dgate && !per_row), want_b = dw2 != nullptr;
  if (want_a || want_b)
    TB200_REQUIRE(workspace && workspace_bytes >= tb200_gated_residual_rms_norm_bwd_workspace(rows, cols, gate ? rows_per_gate : 0),
                  TB200_ERR_WORKSPACE, "gated_residual_rms_norm_bwd: workspace missing or too small");
  return dispatch_dtype(dtype, [&](auto tag) -> int {
    using T = decltype(tag);
    const int64_t vectors = a.rows_per_gate > 1 ? rows / a.rows_per_gate : 1;
    const bool ok = aligned16(dx) && aligned16(dr) && aligned16(x) && aligned16(r) && aligned16(w2) && (!dh || aligned16(dh)) &&
                    (!dy || aligned16(dy)) && (!w1 || aligned16(w1)) && (!gate || aligned16(gate)) && (!dgate || aligned16(dgate)) &&
                    (!workspace || aligned16(workspace));
    const BackwardPlan plan = plan_backward<T>(cols, ok);
    const int64_t n = backward_parts(rows, plan.chunks ? plan.per_sm : 4);
    float* part_a = want_a ? (float*)workspace : nullptr;
    float* part_b = want_b ? (float*)workspace + (n + vectors) * cols : nullptr;
    int rc = 0;
    if (plan.chunks) {
      auto go = [&](auto c, auto most) -> int {
        auto kern = resnorm_bwd_vec<T, decltype(c)::value, decltype(most)::value>;
        static std::atomic<unsigned long long> done{0};
        const cudaError_t e = smem_optin_per_device(done, reinterpret_cast<const void*>(kern), RING_BYTES);
        if (e != cudaSuccess) {
          set_error("gated_residual_rms_norm_bwd: cudaFuncSetAttribute failed: %s", cudaGetErrorString(e));
          return (int)e;
        }
        (void)launch_pdl(kern, dim3((unsigned)n), dim3(plan.threads), (size_t)plan.stages * 4 * cols * sizeof(T), st, false,
                         (T*)dx, (T*)dr, per_row ? (T*)dgate : nullptr, part_a, part_b, (const T*)dh, (const T*)dy, (const T*)x,
                         (const T*)r, (const T*)w1, (const T*)w2, (const T*)gate, rms1, rms2, a, per_row ? 1 : 0, plan.stages,
                         device_status_ptr(), WaitTest::of_this_thread(1, 1));
        return launch_status("resnorm_bwd_vec");
      };
      rc = plan.chunks == 1   ? go(IntC<1>{}, IntC<128>{})
           : plan.chunks == 2 ? go(IntC<2>{}, IntC<256>{})
           : plan.threads <= 256 ? go(IntC<4>{}, IntC<256>{})
                                 : go(IntC<4>{}, IntC<512>{});
    } else {
      auto kern = cols > 4096 ? resnorm_bwd_generic<T> : (cols <= 1024 ? resnorm_bwd_cols<T, 4> : resnorm_bwd_cols<T, 8>);
      kern<<<(unsigned)n, cols_threads(cols), 0, st>>>(
          (T*)dx, (T*)dr, per_row ? (T*)dgate : nullptr, part_a, part_b, (const T*)dh, (const T*)dy, (const T*)x, (const T*)r,
          (const T*)w1, (const T*)w2, (const T*)gate, rms1, rms2, a, per_row ? 1 : 0);
      rc = launch_status("resnorm_bwd_cols");
    }
    if (rc) return rc;
    int launches = 1;
    if (want_a || want_b) {
      const bool groups = dgate && !per_row && a.rows_per_gate > 0;
      const int64_t gy = groups ? 2 + (vectors < 4096 ? vectors : 4096) : 2;
      (void)launch_pdl(resnorm_finalize<T>, dim3((unsigned)ceil_div(cols, 32), (unsigned)gy), dim3(32, 32), 0, st, false, (T*)dw1,
                       (T*)dw2, per_row ? (T*)nullptr : (T*)dgate, part_a, part_b, (const T*)w1, (const T*)gate, n, a,
                       per_row ? 1 : 0);
      rc = launch_status("resnorm_finalize");
      if (rc) return rc;
      ++launches;
    }
    note_kernel(plan.chunks ? "row_vec" : "row_generic", launches);
    return 0;
  });
}
