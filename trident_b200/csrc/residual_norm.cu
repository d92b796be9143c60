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

// ------------------------------------------------------------------ any width and alignment
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
    if (threadIdx.x == 0) rms1[row] = rms;
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
  if (threadIdx.x == 0) rms2[row] = rms;
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
        for (int64_t c = threadIdx.y; c < n; c += 32) {
          const int64_t g0 = part_begin(c, n, a.rows) / a.rows_per_gate;
          const int64_t g1 = (part_begin(c + 1, n, a.rows) - 1) / a.rows_per_gate;
          for (int64_t g = g0; g <= g1; ++g) acc = fmaf(Tr::to_f(gate[g * a.cols + col]), part_a[(c + g) * a.cols + col], acc);
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
  TB200_REQUIRE(h && y && rms2 && x && r && w2 && (!w1 || rms1), TB200_ERR_INVALID,
                "gated_residual_rms_norm_fwd: null pointer");
  cudaStream_t st = (cudaStream_t)stream;
  return dispatch_dtype(dtype, [&](auto tag) -> int {
    using T = decltype(tag);
    resnorm_fwd_generic<T><<<(unsigned)rows, 256, 0, st>>>((T*)h, (T*)y, rms1, rms2, (const T*)x, (const T*)r,
                                                           (const T*)w1, (const T*)w2, (const T*)gate, a);
    const int rc = launch_status("resnorm_fwd_generic");
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
    const int64_t n = backward_parts(rows, 4);
    float* part_a = want_a ? (float*)workspace : nullptr;
    float* part_b = want_b ? (float*)workspace + (n + vectors) * cols : nullptr;
    resnorm_bwd_generic<T><<<(unsigned)n, 256, 0, st>>>(
        (T*)dx, (T*)dr, per_row ? (T*)dgate : nullptr, part_a, part_b, (const T*)dh, (const T*)dy, (const T*)x, (const T*)r,
        (const T*)w1, (const T*)w2, (const T*)gate, rms1, rms2, a, per_row ? 1 : 0);
    int rc = launch_status("resnorm_bwd_generic");
    if (rc) return rc;
    int launches = 1;
    if (want_a || want_b) {
      const bool groups = dgate && !per_row && a.rows_per_gate > 0;
      const int64_t gy = groups ? 2 + (vectors < 4096 ? vectors : 4096) : 2;
      resnorm_finalize<T><<<dim3((unsigned)ceil_div(cols, 32), (unsigned)gy), dim3(32, 32), 0, st>>>(
          (T*)dw1, (T*)dw2, per_row ? nullptr : (T*)dgate, part_a, part_b, (const T*)w1, (const T*)gate, n, a, per_row ? 1 : 0);
      rc = launch_status("resnorm_finalize");
      if (rc) return rc;
      ++launches;
    }
    note_kernel("row_generic", launches);
    return 0;
  });
}
