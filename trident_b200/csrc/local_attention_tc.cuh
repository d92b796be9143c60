// Tensor maps and launch entry points of the tcgen05 kernels of local attention.
#pragma once
#include <cuda.h>

#include "local_attention.cuh"

namespace tb200 {

constexpr int LOCAL_TC_TILE = 128;  // packed query rows and keys of a tile
constexpr int LOCAL_TC_COLS = 96;   // packed query rows of a step of the dK, dV kernel

// Division of 0 <= n < 2^31 by a number that is known at launch: a product, an addition and a shift (the
// roles of the persistent kernels look up their units of work between one tile and the next, where the five
// divisions by variables took over 1000 cycles). With 2^(l-1) < d <= 2^l and m = floor(2^32 (2^l - d) / d) + 1
// the quotient is (floor(m n / 2^32) + n) / 2^l rounded down (Granlund and Montgomery, 1994).
struct Divisor {
  uint32_t d = 1, m = 1, l = 0;
  Divisor() = default;
  explicit Divisor(int divisor) : d((uint32_t)divisor) {
    while ((1ull << l) < d) ++l;
    m = (uint32_t)((((1ull << l) - d) << 32) / d + 1);
  }
  __device__ int quotient(int n) const { return (int)((__umulhi(m, (uint32_t)n) + (uint32_t)n) >> l); }
};

// What the tensor-core kernels take: 16-bit operands, head size 64 or 128, unit feature strides, other
// strides multiples of 16 bytes, and (serving form) a page size that shares a factor of at least 8 with 128.
bool local_tc_supported(const LocalArgs& a, int dtype, const void* q, const void* k, const void* v, const void* out);
int launch_local_fwd_tc(void* out, float* lse, const void* q, const void* k, const void* v, const LocalArgs& a, int max_q,
                        int dtype, cudaStream_t st);
// Serving form with few rows: keys on the tensor-memory lanes, LOCAL_FEW_ROWS columns. 64 contexts of 4096 bf16
// keys, 8 key heads: 4, 8, 16 rows take 149, 157, 175 us at D = 64 and 220, 230, 253 at D = 128, the forward
// kernel 204 to 212 and 247 to 253; 4 contexts of 16384: 68, 73, 83 against 74 to 76, and 87, 93, 103 against 85.
// The rule sees rows and head size alone (the lengths lie on the device, and the announced longest says little of the
// others): where a few long contexts are all there is, it costs up to 12 %.
// (Of 32 and 64 columns the per-row work of every thread outweighs the loads: 304 and 1177 us against 219 and 229.)
constexpr int LOCAL_FEW_ROWS = 16;
static inline bool local_few_rows(const LocalArgs& a, int max_q) {
  return a.table && (int64_t)max_q * a.G <= (a.D == 64 ? LOCAL_FEW_ROWS : 8);
}
int launch_local_few_tc(void* out, const void* q, const void* k, const void* v, const LocalArgs& a, int dtype,
                        cudaStream_t st);

// Tensor maps (false with the error text set when the driver refuses one; the caller has bound the primary
// context) and what they take.
// (rows: boxes of `tokens` tokens with the heads of a group)
bool local_map_rows(CUtensorMap* map, const void* q, const int64_t* st, const LocalArgs& a, int tokens, const char* what);
bool local_map_keys(CUtensorMap* map, const void* k, const int64_t* st, const LocalArgs& a, int piece, const char* what);
int local_piece(const LocalArgs& a);  // rows of one copy of keys
bool local_rows_ok(const void* p, const int64_t* st, const LocalArgs& a);
bool local_keys_ok(const void* p, const int64_t* st, const LocalArgs& a);

// Backward pass of the training form. row_scratch: two float arrays of local_tc_rows(a) elements.
bool local_bwd_tc_supported(const LocalBwdArgs& b, int dtype, const void* q, const void* k, const void* v, const void* out,
                            const void* dout, const void* dq, const void* dk, const void* dv);
int launch_local_bwd_tc(void* dq, void* dk, void* dv, const void* dout, const void* q, const void* k, const void* v,
                        const void* out, const float* lse, float* row_scratch, const LocalBwdArgs& b, int dtype,
                        cudaStream_t st);
// packed rows of all column tiles, unused ones included
static inline int64_t local_tc_rows(const LocalArgs& a) {
  return (int64_t)a.n * a.KV * ceil_div(a.tokens, LOCAL_TC_COLS / a.G) * LOCAL_TC_COLS;
}
// tokens of the two query tiles of a CTA
static inline int local_tc_row_tokens(const LocalArgs& a) { return 2 * (LOCAL_TC_TILE / a.G); }

}  // namespace tb200
