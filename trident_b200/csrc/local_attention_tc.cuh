// Tensor maps and launch entry points of the tcgen05 kernels of local attention.
#pragma once
#include "local_attention.cuh"

namespace tb200 {

constexpr int LOCAL_TC_TILE = 128;  // packed query rows and keys of a tile

// What the tensor-core kernels take: 16-bit operands, head size 64 or 128, unit feature strides, other
// strides multiples of 16 bytes, and (serving form) a page size that shares a factor of at least 8 with 128.
bool local_tc_supported(const LocalArgs& a, int dtype, const void* q, const void* k, const void* v, const void* out);
int launch_local_fwd_tc(void* out, float* lse, const void* q, const void* k, const void* v, const LocalArgs& a, int max_q,
                        int dtype, cudaStream_t st);
// tokens of the two query tiles of a CTA
static inline int local_tc_row_tokens(const LocalArgs& a) { return 2 * (LOCAL_TC_TILE / a.G); }

}  // namespace tb200
