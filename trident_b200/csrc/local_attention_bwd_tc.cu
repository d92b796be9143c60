// tcgen05 backward of window attention with sinks, for 16-bit operands with head size 64 or 128.
//
// Two kernels, each of which owns what it sums, so that nothing is added with atomics and the same inputs
// give the same bits (one kernel for all three gradients would need 5 products a tile pair instead of 7,
// but has to add dQ across CTAs), behind one over the rows (local_rows_tc_kernel):
//
//   dQ      tiles of 128 packed query rows (token * G + head); a persistent CTA takes every gridDim-th of
//           them. Q and dO of the tile are put into tensor memory as operands (their products then read only
//           K or V from shared memory: with both operands there, the four 4 KB reads of an instruction pair
//           took the pipe 120 cycles an instruction instead of 64); along the keys of the tile's walk
//             S = Q K^T, dP = dO V^T, P = exp2(S scale log2e - lse log2e), dS = P (dP - delta), dQ += dS K
//           (dS 16-bit in tensor memory over dP). S(i+1) is computed as soon as S(i) is in registers, dP(i+1)
//           after dQ(i), so that exponentials and score gradients follow each other without a pause.
//   dK, dV  a CTA owns 128 keys (K_j, V_j resident in shared memory) and walks the tiles of 96 packed query
//           rows that see any of them; the sum over the heads of a group is part of the walk. All
//           transposed, keys on the tensor-memory lanes:
//             S^T = K_j Q^T, dP^T = V_j dO^T, dV += P^T dO, dK += dS^T Q
//           96 rows because dV, dK, S^T, dP^T and a P^T of its own then fit into the 512 columns: with P^T
//           over S^T (128 rows) the chain exponentials -> dV -> S^T -> exponentials bounded a step at 4100
//           cycles.
//
// The queries beyond the window of a key tile that holds sinks ("far", LocalBwdArgs) are cut into pieces
// about as long as a walk inside the window, each a CTA of its own: a single CTA would walk all queries.
//
// P and dS are rounded to 16 bits as operands of their products, as the tensor cores take them: half a step each
// (2-norm of the error of dq against 64 bits 0.0025 in bf16, 0.00031 in fp16 at any window, of which the final rounding
// alone is 0.0017 and 0.00021; with delta of the rounded output it was 0.0026 at a window of 1024 and 0.0038 at 2).
// fp16 score gradients below 2^-14 are multiples of 2^-24. Statistics, delta and all sums are fp32.
//
// Bounds, at 2 x 32 heads x 4096 x 128 bf16, window 1024, 8 key heads. dK, dV: 252 us (957 TFLOP/s); a step takes
// 2350 cycles, of which the products alone, two of them with both operands in shared memory, take about 2200 (dS^T
// over P^T instead of dP^T, so that the next dP^T need not wait for dK: 302 us, one chain of all four products). dQ:
// 180 us (1008 TFLOP/s); a step takes 2050 cycles, the chain dQ -> dP -> score gradients (1536 of products).
#include <type_traits>

#include "attn_math.cuh"
#include "local_attention_tc.cuh"
#include "ptx.cuh"

namespace tb200 {
namespace {

constexpr int TILE = LOCAL_TC_TILE;
constexpr int COLS = LOCAL_TC_COLS;  // packed query rows of a step of the dK, dV kernel
constexpr int THREADS = 384;  // 4 service warps, 8 compute warps: two threads per row, 64 columns each
constexpr float LOG2E = 1.4426950408889634f;

struct BwdParams {
  LocalBwdArgs b;
  void *dk, *dv;
  const float* lse;
  float* nlse2;         // [n * KV][column tiles][96]  -lse * log2(e), written by the kernel of the rows
  float* ndelta;        // [n * KV][column tiles][96]  -delta
  float scale_log2;
  int tile_tokens;      // tokens of a row tile (dQ)
  int row_tiles;
  int col_tokens;       // tokens of a column tile (dK, dV)
  int col_tiles, key_tiles;
  Divisor heads, kv;    // n * KV, KV
  int* status;
  WaitTest test_dq, test_dkv;
};

__device__ inline void tma_load_4d(void* dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z, int w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
      ::"r"(ptx::smem_u32(dst)), "l"(map), "r"(ptx::smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}
__device__ inline void tma_load_5d(void* dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z, int w, int u) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6, %7}], [%2];"
      ::"r"(ptx::smem_u32(dst)), "l"(map), "r"(ptx::smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(u)
      : "memory");
}
__device__ inline void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   ptx::smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(ptx::smem_u32(bar))
               : "memory");
}
// the lowest n bits
__device__ inline uint32_t low_bits(int n) { return n <= 0 ? 0u : (n >= 32 ? 0xffffffffu : (1u << n) - 1u); }
__device__ inline int saturate(int64_t v) { return v < -(1 << 20) ? -(1 << 20) : (v > (1 << 20) ? (1 << 20) : (int)v); }
// Rows [rows, 96) of `boxes` swizzled boxes set to zero (rows that no copy writes, but products read).
__device__ inline void zero_rows(uint8_t* smem, int boxes, int rows) {
  const int per_box = (COLS - rows) * 8;  // 16-byte chunks
  for (int i = threadIdx.x; i < boxes * per_box; i += THREADS)
    *reinterpret_cast<uint4*>(smem + (i / per_box) * (COLS * 128) + rows * 128 + (i % per_box) * 16) = make_uint4(0, 0, 0, 0);
}

// ------------------------------------------------------------------ -lse log2e, -delta
// Of all packed rows, in the order in which the other kernels read them (entries of column tiles that belong to no row:
// zeros; the products that meet them see rows of zeros). delta = sum_d out dout in fp32, of the output before its
// rounding where what that left was kept (LocalArgs::low): the score gradients of a row sum to zero, and an error of delta
// goes to dq as a common part of them times sum p k, which does not average out over a short window. Bounded by HBM:
// reads out, low and dout once (2 x 32 heads x 4096 x 128: 201 MB, 36 us, 5.5 TB/s; two warps of the dQ
// kernel, which did this before for out alone, were 85 us slower with low: a row's loads there are not under way together).
template <typename T, int D>
__global__ void __launch_bounds__(256) local_rows_tc_kernel(const T* out, const T* dout, const BwdParams p) {
  constexpr int LANES = D / 8, ROWS = 32 / LANES, AHEAD = 4, EACH = 16;  // lanes and rows of a load; rows of a warp
  const LocalArgs& a = p.b.f;
  const T* low = reinterpret_cast<const T*>(a.low);
  const int lane = threadIdx.x & 31, sub = lane / LANES, at = lane % LANES * 8;
  const int64_t warp = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5), row0 = warp * EACH;
  static_assert(COLS % EACH == 0 && EACH % (ROWS * AHEAD) == 0, "a column tile is a whole number of warps");
  const int64_t tile = row0 / COLS;
  if (tile >= (int64_t)a.n * a.KV * p.col_tiles) return;
  const int it = (int)(tile % p.col_tiles), sh = (int)(tile / p.col_tiles), hk = sh % a.KV, s = sh / a.KV;
#pragma unroll
  for (int b = 0; b < EACH; b += ROWS * AHEAD) {
    uint4 o[AHEAD], l[AHEAD], g[AHEAD];
    float lse[AHEAD];
    bool live[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int c = (int)(row0 % COLS) + b + k * ROWS + sub, t = it * p.col_tokens + c / a.G, h = hk * a.G + c % a.G;
      live[k] = c < p.col_tokens * a.G && t < a.tokens;
      o[k] = l[k] = g[k] = make_uint4(0, 0, 0, 0);
      lse[k] = 0.f;
      if (live[k]) {
        const int64_t from = (int64_t)s * a.os[0] + (int64_t)h * a.os[1] + (int64_t)t * a.os[2] + at;
        o[k] = ld_stream(out + from);
        if (low) l[k] = ld_stream(low + from);
        g[k] = *reinterpret_cast<const uint4*>(dout + (int64_t)s * p.b.dos[0] + (int64_t)h * p.b.dos[1] + (int64_t)t * p.b.dos[2] + at);
        lse[k] = p.lse[((int64_t)s * a.H + h) * a.tokens + t];
      }
    }
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      float x[8], y[8], z[8], sum = 0.f;
      unpack<T>(o[k], x);
      unpack<T>(l[k], y);
      unpack<T>(g[k], z);
#pragma unroll
      for (int e = 0; e < 8; ++e) sum = fmaf(x[e] + y[e], z[e], sum);
#pragma unroll
      for (int d = LANES / 2; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      if (at == 0) {
        const int64_t row = row0 + b + k * ROWS + sub;
        p.nlse2[row] = live[k] ? -lse[k] * LOG2E : 0.f;
        p.ndelta[row] = live[k] ? -sum : 0.f;
      }
    }
  }
}

// ------------------------------------------------------------------ dK, dV
template <typename T, int D>
__global__ void __launch_bounds__(THREADS, 1)
    local_dkv_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_do,
                        const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                        const BwdParams p) {
  constexpr int STAGES = 3;
  constexpr int KEY_BYTES = TILE * D * 2, COL_BYTES = COLS * D * 2, NBOX = D / 64;
  constexpr int KEY_BOX = TILE * 128, COL_BOX = COLS * 128;
  constexpr int HALF = COLS / 2;  // columns of a compute thread
  constexpr bool IS_BF16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr uint32_t IDESC_S = ptx::make_idesc(IS_BF16, false, false, TILE, COLS);
  constexpr uint32_t IDESC_D = ptx::make_idesc(IS_BF16, false, true, TILE, D);
  constexpr uint32_t TMEM_COLS = 512, COL_S = 0, COL_DP = COLS, COL_P = 2 * COLS, COL_DV = 256, COL_DK = 256 + D;
  static_assert(COL_P + COLS / 2 <= COL_DV, "tensor memory");

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* k_smem = smem;
  uint8_t* v_smem = smem + KEY_BYTES;
  uint8_t* q_smem = smem + 2 * KEY_BYTES;           // [STAGES]
  uint8_t* do_smem = q_smem + STAGES * COL_BYTES;   // [STAGES]
  float* nlse_smem = reinterpret_cast<float*>(do_smem + STAGES * COL_BYTES);  // [STAGES][96]
  float* ndelta_smem = nlse_smem + STAGES * COLS;                             // [STAGES][96]
  uint64_t* bars = reinterpret_cast<uint64_t*>(ndelta_smem + STAGES * COLS);
  uint64_t* kv_full = bars;
  uint64_t* qdo_full = bars + 1;             // [STAGES]
  uint64_t* qdo_empty = bars + 1 + STAGES;   // [STAGES]
  uint64_t* s_ready = bars + 1 + 2 * STAGES; // S^T(i) computed
  uint64_t* dp_ready = s_ready + 1;          // dP^T(i) computed
  uint64_t* dv_done = s_ready + 2;           // dV(i) has read P^T(i)
  uint64_t* all_done = s_ready + 3;
  uint64_t* s_free = s_ready + 4;            // S^T(i) read          (256 arrivals)
  uint64_t* p_ready = s_ready + 5;           // P^T(i) written       (256 arrivals)
  uint64_t* ds_ready = s_ready + 6;          // dS^T(i) over dP^T(i) (256 arrivals)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(s_ready + 7);
  volatile uint32_t* abort_flag = tmem_slot + 1;

  const LocalArgs& a = p.b.f;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // The longest walks of all sequences and heads first (far pieces, then the key tiles in order, whose walks end
  // with the sequence): the short ones even out the last CTAs of the SMs. By sequence and head SMs stood idle 15 %
  // of the time at 512 key tiles and 48 far pieces (262 us, so 252; the dQ kernel's tiles likewise: 189 and 184).
  const int rank = p.heads.quotient(blockIdx.x), sh = blockIdx.x - rank * (int)p.heads.d;
  const int s = p.kv.quotient(sh), hk = sh - s * a.KV;
  // the walk: column tiles [i0, i0 + steps)
  const int far_pieces = p.b.sink_tiles * p.b.far;
  int jt = rank - far_pieces, piece = -1, i0, i1;
  const bool far = jt < 0;
  if (far) {
    piece = rank % p.b.far;
    jt = rank / p.b.far;
  }
  const int beyond = (near_end(a, jt, TILE) + p.col_tokens - 1) / p.col_tokens;  // first column tile beyond the window
  if (far) {
    const int64_t span = p.col_tiles - beyond;
    i0 = beyond + (int)(span * piece / p.b.far);
    i1 = beyond + (int)(span * (piece + 1) / p.b.far);
  } else {
    i0 = jt * TILE / p.col_tokens;
    i1 = beyond;
  }
  const int steps = i1 - i0;
  const int rows = p.col_tokens * a.G;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 1 + 2 * STAGES + 4; ++i) ptx::mbar_init(&bars[i], 1);
    for (int i = 0; i < 3; ++i) ptx::mbar_init(s_free + i, 256);
    abort_flag[0] = 0;
    abort_flag[1] = p.test_dkv.units;
    ptx::fence_barrier_init();
    ptx::prefetch_tensormap(&map_q);
    ptx::prefetch_tensormap(&map_do);
    ptx::prefetch_tensormap(&map_k);
    ptx::prefetch_tensormap(&map_v);
  }
  if (warp == 2) {
    ptx::tmem_alloc(tmem_slot, TMEM_COLS);
    ptx::tmem_relinquish();
  }
  if (rows < COLS) {
    zero_rows(q_smem, 2 * STAGES * NBOX, rows);
    ptx::fence_proxy_async_smem();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    if (lane == 0 && steps > 0) {
      ptx::mbar_expect_tx(kv_full, 2 * KEY_BYTES);
#pragma unroll
      for (int c = 0; c < NBOX; ++c) {
        tma_load_4d(k_smem + c * KEY_BOX, &map_k, kv_full, c * 64, jt * TILE, hk, s);
        tma_load_4d(v_smem + c * KEY_BOX, &map_v, kv_full, c * 64, jt * TILE, hk, s);
      }
      int brought = 0;
      for (int i = 0; i < steps; ++i) {
        const int st = i % STAGES, it = i0 + i;
        ptx::mbar_wait(&qdo_empty[st], ((i / STAGES) & 1) ^ 1, abort_flag, p.status, 101);
        if (abort_flag[0]) break;  // a wait has run out: nothing more is brought
        brought = i + 1;
        if (i == p.test_dkv.skip && blockIdx.x == 0) continue;  // (test hook)
        ptx::mbar_expect_tx(&qdo_full[st], 2 * NBOX * rows * 128 + 2 * COLS * 4);
#pragma unroll
        for (int c = 0; c < NBOX; ++c) {
          tma_load_5d(q_smem + st * COL_BYTES + c * COL_BOX, &map_q, &qdo_full[st], c * 64, 0, it * p.col_tokens, hk, s);
          tma_load_5d(do_smem + st * COL_BYTES + c * COL_BOX, &map_do, &qdo_full[st], c * 64, 0, it * p.col_tokens, hk, s);
        }
        const int64_t row0 = (((int64_t)s * a.KV + hk) * p.col_tiles + it) * COLS;
        bulk_load(nlse_smem + st * COLS, p.nlse2 + row0, COLS * 4, &qdo_full[st]);
        bulk_load(ndelta_smem + st * COLS, p.ndelta + row0, COLS * 4, &qdo_full[st]);
      }
      // every copy has landed before the CTA gives up its shared memory
      ptx::mbar_wait_drain(kv_full, 0, abort_flag, p.status, 102);
      for (int i = brought > STAGES ? brought - STAGES : 0; i < brought; ++i)
        ptx::mbar_wait_drain(&qdo_full[i % STAGES], (i / STAGES) & 1, abort_flag, p.status, 102);
    }
    __syncwarp();
  } else if (warp == 1) {
    // The whole warp walks the loop and waits; one elected lane issues. (With the waits in the elected lane
    // alone, a commit was seen to take effect only after that lane's next wait had given up.)
    const bool elected = ptx::elect_one();
    auto wait_ = [&](uint64_t* bar, uint32_t parity, int code) {
      ptx::mbar_wait(bar, parity, abort_flag, p.status, code);
      __syncwarp();
    };
    auto commit_ = [&](uint64_t* bar) {
      if (elected) ptx::umma_commit(bar);
    };
    const uint64_t dk = ptx::make_smem_desc(ptx::smem_u32(k_smem), 16, 1024), dv = ptx::make_smem_desc(ptx::smem_u32(v_smem), 16, 1024);
    const uint64_t dq = ptx::make_smem_desc(ptx::smem_u32(q_smem), 16, 1024), dd = ptx::make_smem_desc(ptx::smem_u32(do_smem), 16, 1024);
    const uint64_t dq_t = ptx::make_smem_desc(ptx::smem_u32(q_smem), COL_BOX, 1024);  // read along the rows
    const uint64_t dd_t = ptx::make_smem_desc(ptx::smem_u32(do_smem), COL_BOX, 1024);
    constexpr uint64_t STAGE = static_cast<uint64_t>(COL_BYTES >> 4);
    auto score = [&](uint32_t col, uint64_t ad, uint64_t bd) {  // [keys][rows] = A B^T over the features
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        const uint64_t oa = static_cast<uint64_t>(((ks >> 2) * KEY_BOX + (ks & 3) * 32) >> 4);
        const uint64_t ob = static_cast<uint64_t>(((ks >> 2) * COL_BOX + (ks & 3) * 32) >> 4);
        if (elected) ptx::umma_ss(tmem_base + col, ad + oa, bd + ob, IDESC_S, ks != 0);
      }
    };
    if (steps > 0) {
      wait_(kv_full, 0, 103);
      wait_(&qdo_full[0], 0, 104);
      ptx::tc_fence_after();
      score(COL_S, dk, dq);
      commit_(s_ready);
      score(COL_DP, dv, dd);
      commit_(dp_ready);
      for (int i = 0; i < steps; ++i) {
        const uint32_t ph = i & 1;
        const uint64_t cur = (i % STAGES) * STAGE, nxt = ((i + 1) % STAGES) * STAGE;
        if (i + 1 < steps) {
          // (waiting for what arrived long ago costs 150 cycles: not between the softmax threads and the product)
          wait_(&qdo_full[(i + 1) % STAGES], ((i + 1) / STAGES) & 1, 106);
          wait_(s_free, ph, 105);
          ptx::tc_fence_after();
          score(COL_S, dk, dq + nxt);
          commit_(s_ready);
        }
        wait_(p_ready, ph, 107);
        ptx::tc_fence_after();
#pragma unroll
        for (int ks = 0; ks < COLS / 16; ++ks)
          if (elected)
            ptx::umma_ts(tmem_base + COL_DV, tmem_base + COL_P + ks * 8, dd_t + cur + static_cast<uint64_t>((ks * 2048) >> 4),
                         IDESC_D, (i | ks) != 0);
        commit_(dv_done);
        wait_(ds_ready, ph, 108);
        ptx::tc_fence_after();
#pragma unroll
        for (int ks = 0; ks < COLS / 16; ++ks)  // (a thread packs dS^T into the first half of its own columns)
          if (elected)
            ptx::umma_ts(tmem_base + COL_DK, tmem_base + COL_DP + (ks / (HALF / 16)) * HALF + (ks % (HALF / 16)) * 8,
                         dq_t + cur + static_cast<uint64_t>((ks * 2048) >> 4), IDESC_D, (i | ks) != 0);
        commit_(&qdo_empty[i % STAGES]);
        if (i + 1 < steps) {
          score(COL_DP, dv, dd + nxt);  // over dS^T(i), which dK(i) reads first on the in-order pipe
          commit_(dp_ready);
        }
      }
    }
    commit_(all_done);
    ptx::mbar_wait_drain(all_done, 0, abort_flag, p.status, 109);
    __syncwarp();
  } else if (warp >= 4) {
    const int quarter = warp & 3, half = (warp - 4) >> 2;
    const int r = quarter * 32 + lane, key = jt * TILE + r;
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t s_addr = tmem_base + lane_off + COL_S + half * HALF, dp_addr = tmem_base + lane_off + COL_DP + half * HALF;
    const uint32_t p_addr = tmem_base + lane_off + COL_P + half * (HALF / 2);
    const uint64_t scale2 = am::pack2f(p.scale_log2, p.scale_log2);
    const uint32_t always = key < a.sinks ? 0xffffffffu : 0u;
    for (int i = 0; i < steps; ++i) {
      const int st = i % STAGES, it = i0 + i;
      const int token0 = it * p.col_tokens, token1 = token0 + p.col_tokens - 1;
      // every query of the tile sees every key of this one
      const bool plain = token0 >= jt * TILE + TILE - 1 && (token1 - jt * TILE < a.window || (jt + 1) * TILE <= a.sinks);
      const float4* nlse4 = reinterpret_cast<const float4*>(nlse_smem + st * COLS + half * HALF);
      const float4* ndel4 = reinterpret_cast<const float4*>(ndelta_smem + st * COLS + half * HALF);
      float pr[HALF];
      uint32_t ra[32], rb[16];
      ptx::mbar_wait(&qdo_full[st], (i / STAGES) & 1, abort_flag, p.status, 110);
      ptx::mbar_wait(s_ready, i & 1, abort_flag, p.status, 111);
      ptx::tc_fence_after();
      ptx::tmem_ld32(s_addr, ra);
      ptx::tmem_ld16(s_addr + 32, rb);
      am::tmem_ld_wait_dep(ra);
      am::tmem_ld_wait_dep(rb);
      ptx::tc_fence_before();
      ptx::mbar_arrive(s_free);
      uint32_t pa[16], pb[8];
      // the arguments and conversions of neighbouring columns are issued between the exponentials
      auto probabilities = [&](auto masked, uint32_t seen0, uint32_t seen1) {
        constexpr int LAG = 3, PAIRS = HALF / 2;  // pairs between an exponential and its use
        auto argument = [&](int k) {
          const float4 nl = nlse4[k >> 1];
          const uint64_t v = k < 16 ? am::pack2u(ra[2 * k & 31], ra[(2 * k + 1) & 31]) : am::pack2u(rb[2 * k & 15], rb[(2 * k + 1) & 15]);
          am::unpack2f(am::fma2_ordered(v, scale2, k & 1 ? am::pack2f(nl.z, nl.w) : am::pack2f(nl.x, nl.y)), pr[2 * k], pr[2 * k + 1]);
        };
        argument(0);
#pragma unroll
        for (int k = 0; k < PAIRS + LAG; ++k) {
          if (k < PAIRS) pr[2 * k] = am::ex2_ordered(pr[2 * k]);
          if (k + 1 < PAIRS) argument(k + 1);
          if (k < PAIRS) pr[2 * k + 1] = am::ex2_ordered(pr[2 * k + 1]);
          if (k >= LAG) {
            const int d = k - LAG;
            if constexpr (decltype(masked)::value) {
              const uint32_t seen = d < 16 ? seen0 : seen1;
              if (!(seen & (1u << (2 * d & 31)))) pr[2 * d] = 0.f;
              if (!(seen & (2u << (2 * d & 31)))) pr[2 * d + 1] = 0.f;
            }
            const uint32_t both = am::cvt_ordered<T>(pr[2 * d], pr[2 * d + 1]);
            if (d < 16) pa[d & 15] = both;
            else pb[d & 7] = both;
          }
        }
      };
      if (plain) {
        probabilities(std::false_type{}, 0u, 0u);
      } else {
        // columns from `low` on are not before the key, those below `high` are within its window
        const int low = saturate((int64_t)(key - token0) * a.G) - half * HALF;
        const int high = saturate(((int64_t)key + a.window - token0) * a.G) - half * HALF;
        probabilities(std::true_type{}, ~low_bits(low) & (low_bits(high) | always),
                      ~low_bits(low - 32) & (low_bits(high - 32) | always));
      }
      {
        if (i > 0) {  // P^T(i) goes over P^T(i-1)
          ptx::mbar_wait(dv_done, (i - 1) & 1, abort_flag, p.status, 112);
          ptx::tc_fence_after();
        }
        ptx::tmem_st16(p_addr, pa);
        ptx::tmem_st8(p_addr + 16, pb);
        ptx::tmem_st_wait();
        ptx::tc_fence_before();
        ptx::mbar_arrive(p_ready);
      }
      ptx::mbar_wait(dp_ready, i & 1, abort_flag, p.status, 113);
      ptx::tc_fence_after();
      ptx::tmem_ld32(dp_addr, ra);
      ptx::tmem_ld16(dp_addr + 32, rb);
      am::tmem_ld_wait_dep(ra);
      am::tmem_ld_wait_dep(rb);
      {
        auto grad = [&](int g, uint32_t v0, uint32_t v1, uint32_t v2, uint32_t v3, uint32_t& o0, uint32_t& o1) {
          const float4 nd = ndel4[g];
          float d0, d1, d2, d3;
          am::unpack2f(am::mul2(am::pack2f(pr[g * 4], pr[g * 4 + 1]), am::add2(am::pack2u(v0, v1), am::pack2f(nd.x, nd.y))), d0, d1);
          am::unpack2f(am::mul2(am::pack2f(pr[g * 4 + 2], pr[g * 4 + 3]), am::add2(am::pack2u(v2, v3), am::pack2f(nd.z, nd.w))), d2, d3);
          o0 = am::cvt_pair<T>(d0, d1);
          o1 = am::cvt_pair<T>(d2, d3);
        };
#pragma unroll
        for (int g = 0; g < 8; ++g) grad(g, ra[g * 4], ra[g * 4 + 1], ra[g * 4 + 2], ra[g * 4 + 3], pa[g * 2], pa[g * 2 + 1]);
#pragma unroll
        for (int g = 0; g < 4; ++g) grad(8 + g, rb[g * 4], rb[g * 4 + 1], rb[g * 4 + 2], rb[g * 4 + 3], pb[g * 2], pb[g * 2 + 1]);
        ptx::tmem_st16(dp_addr, pa);
        ptx::tmem_st8(dp_addr + 16, pb);
        ptx::tmem_st_wait();
        ptx::tc_fence_before();
        ptx::mbar_arrive(ds_ready);
      }
    }
    // epilogue: the first half of the warps writes dV, the second dK
    ptx::mbar_wait(all_done, 0, abort_flag, p.status, 114);
    ptx::tc_fence_after();
    const bool is_k = half == 1, parted = jt < p.b.sink_tiles;
    const float mul = is_k ? a.scale : 1.f;
    const int64_t* ost = is_k ? p.b.dks : p.b.dvs;
    T* out = reinterpret_cast<T*>(is_k ? p.dk : p.dv) + (int64_t)s * ost[0] + hk * ost[1] + (int64_t)key * ost[2];
    float* part = p.b.part + ((((((int64_t)s * a.KV + hk) * p.b.sink_tiles + jt) * (p.b.far + 1) + piece + 1) * 2 + (is_k ? 0 : 1)) * TILE + r) * D;
#pragma unroll 1
    for (int c = 0; c < D / 32; ++c) {
      uint32_t v[32];
      __syncwarp();
      if (steps > 0) {
        ptx::tmem_ld32(tmem_base + lane_off + (is_k ? COL_DK : COL_DV) + c * 32, v);
        ptx::tmem_ld_wait();
      } else {
#pragma unroll
        for (int e = 0; e < 32; ++e) v[e] = 0;
      }
      if (parted) {
#pragma unroll
        for (int g = 0; g < 8; ++g)
          *reinterpret_cast<float4*>(part + c * 32 + g * 4) =
              make_float4(__uint_as_float(v[g * 4]) * mul, __uint_as_float(v[g * 4 + 1]) * mul,
                          __uint_as_float(v[g * 4 + 2]) * mul, __uint_as_float(v[g * 4 + 3]) * mul);
      } else if (key < a.tokens) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          uint4 o;
          o.x = am::cvt_pair<T>(__uint_as_float(v[g * 8 + 0]) * mul, __uint_as_float(v[g * 8 + 1]) * mul);
          o.y = am::cvt_pair<T>(__uint_as_float(v[g * 8 + 2]) * mul, __uint_as_float(v[g * 8 + 3]) * mul);
          o.z = am::cvt_pair<T>(__uint_as_float(v[g * 8 + 4]) * mul, __uint_as_float(v[g * 8 + 5]) * mul);
          o.w = am::cvt_pair<T>(__uint_as_float(v[g * 8 + 6]) * mul, __uint_as_float(v[g * 8 + 7]) * mul);
          *reinterpret_cast<uint4*>(out + c * 32 + g * 8) = o;
        }
      }
    }
  }
  ptx::tc_fence_before();
  __syncthreads();
  if (warp == 2) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

// ------------------------------------------------------------------ dQ
// warp 0: producer (rings of two K and two V tiles across all tiles of the CTA; Q and dO of the next tile land in
// shared memory during this one); warp 1: MMA issuer; warps 2, 3: -lse log2e and -delta of the next tile's rows; warps
// 4-11: compute.
template <typename T, int D>
__global__ void __launch_bounds__(THREADS, 1)
    local_dq_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_do,
                       const __grid_constant__ CUtensorMap map_dq,
                       const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                       const BwdParams p) {
  constexpr int TILE_BYTES = TILE * D * 2, NBOX = D / 64, BOX_BYTES = TILE * 128;
  constexpr bool IS_BF16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr uint32_t IDESC_S = ptx::make_idesc(IS_BF16, false, false, TILE, TILE);
  constexpr uint32_t IDESC_D = ptx::make_idesc(IS_BF16, false, true, TILE, D);
  constexpr uint32_t TMEM_COLS = 512, COL_S = 0, COL_DP = 128, COL_DQ = 256, COL_Q = 384, COL_DO = 448;

  // (at D = 128 the tiles leave 3 KB: the window starts at the CTA's shared memory, checked below)
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* k_smem = smem;                     // [2]
  uint8_t* v_smem = smem + 2 * TILE_BYTES;    // [2]
  uint8_t* land_smem = smem + 4 * TILE_BYTES; // Q, dO of the next tile
  uint8_t* out_smem = smem + 6 * TILE_BYTES;  // dQ of a tile on its way out
  float* stats = reinterpret_cast<float*>(smem + 7 * TILE_BYTES);  // [2][nlse, ndelta][128]
  uint64_t* bars = reinterpret_cast<uint64_t*>(stats + 4 * TILE);
  // Per step (g counts the steps of all tiles of this CTA), per tile (u): parity of g or u; rings: of g / 2.
  uint64_t* k_full = bars;           // [2]
  uint64_t* k_empty = bars + 2;      // [2] dQ(g) done
  uint64_t* v_full = bars + 4;       // [2]
  uint64_t* v_empty = bars + 6;      // [2] dP(g) done
  uint64_t* land_full = bars + 8;    // Q, dO of tile u have landed
  uint64_t* s_ready = bars + 9;      // S(g) computed
  uint64_t* dp_ready = bars + 10;    // dP(g) computed
  uint64_t* tile_done = bars + 11;   // all products of tile u done
  uint64_t* s_free = bars + 12;      // S(g) read                (256 arrivals)
  uint64_t* ds_ready = bars + 13;    // dS(g) written over dP(g) (256 arrivals)
  uint64_t* q_ready = bars + 14;     // Q, dO of tile u in tensor memory, dQ of tile u - 1 read (256 arrivals)
  uint64_t* stats_empty = bars + 15; // [2] (256 arrivals)
  uint64_t* stats_full = bars + 17;  // [2] (64 arrivals)
  uint64_t* out_free = bars + 19;    // dQ of tile u - 1 has left shared memory
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 20);
  volatile uint32_t* abort_flag = tmem_slot + 1;

  const LocalArgs& a = p.b.f;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int units = a.n * a.KV * p.row_tiles;
  struct Unit {
    int s, hk, t0, ntok;
  };
  // tile `unit`: longest walks (last tokens) of all sequences and key heads first
  auto unit_at = [&](int unit) {
    Unit w;
    const int rank = p.heads.quotient(unit), sh = unit - rank * (int)p.heads.d, it = p.row_tiles - 1 - rank;
    w.s = p.kv.quotient(sh);
    w.hk = sh - w.s * a.KV;
    w.t0 = it * p.tile_tokens;
    w.ntok = min(p.tile_tokens, a.tokens - w.t0);
    return w;
  };
  // (at least one key tile: a query sees itself)
  auto walk_of = [&](const Unit& w) { return key_range(a, w.t0, w.t0 + w.ntok - 1, a.tokens, TILE); };

  if (threadIdx.x == 0) {
    for (int i = 0; i < 12; ++i) ptx::mbar_init(&bars[i], 1);
    for (int i = 12; i < 17; ++i) ptx::mbar_init(&bars[i], 256);
    for (int i = 17; i < 19; ++i) ptx::mbar_init(&bars[i], 64);
    ptx::mbar_init(out_free, 1);
    abort_flag[0] = 0;
    abort_flag[1] = p.test_dq.units;
    if ((ptx::smem_u32(smem) & 1023u) != 0) {  // swizzled tiles need a 1024-byte aligned base
      abort_flag[0] = 1;
      atomicCAS(p.status, 0, 120);
    }
    ptx::fence_barrier_init();
    ptx::prefetch_tensormap(&map_q);
    ptx::prefetch_tensormap(&map_do);
    ptx::prefetch_tensormap(&map_dq);
    ptx::prefetch_tensormap(&map_k);
    ptx::prefetch_tensormap(&map_v);
  }
  if (warp == 1) {
    ptx::tmem_alloc(tmem_slot, TMEM_COLS);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      auto land = [&](int unit) {
        const Unit w = unit_at(unit);
        ptx::mbar_expect_tx(land_full, 2 * NBOX * p.tile_tokens * a.G * 128);
#pragma unroll
        for (int c = 0; c < NBOX; ++c) {
          tma_load_5d(land_smem + c * BOX_BYTES, &map_q, land_full, c * 64, 0, w.t0, w.hk, w.s);
          tma_load_5d(land_smem + TILE_BYTES + c * BOX_BYTES, &map_do, land_full, c * 64, 0, w.t0, w.hk, w.s);
        }
      };
      int g = 0, u = 0, keys = 0, landed = 1;  // steps, tiles; K tiles (g, or one more) and landings brought
      bool stop = false;                       // a wait has run out: nothing more is brought
      land(blockIdx.x);
      for (int unit = blockIdx.x; unit < units && !stop; unit += gridDim.x, ++u) {
        const Unit w = unit_at(unit);
        const KeyRange kr = walk_of(w);
        for (int i = 0; i < kr.count; ++i, ++g) {
          const int st = g & 1, j0 = kr.tile(i) * TILE;
          ptx::mbar_wait(&k_empty[st], ((g >> 1) & 1) ^ 1, abort_flag, p.status, 121);
          if ((stop = abort_flag[0] != 0)) break;
          ++keys;
          if (!(g == p.test_dq.skip && blockIdx.x == 0)) {  // (test hook)
            ptx::mbar_expect_tx(&k_full[st], TILE_BYTES);
#pragma unroll
            for (int c = 0; c < NBOX; ++c) tma_load_4d(k_smem + st * TILE_BYTES + c * BOX_BYTES, &map_k, &k_full[st], c * 64, j0, w.hk, w.s);
          }
          ptx::mbar_wait(&v_empty[st], ((g >> 1) & 1) ^ 1, abort_flag, p.status, 122);
          if ((stop = abort_flag[0] != 0)) break;
          ptx::mbar_expect_tx(&v_full[st], TILE_BYTES);
#pragma unroll
          for (int c = 0; c < NBOX; ++c) tma_load_4d(v_smem + st * TILE_BYTES + c * BOX_BYTES, &map_v, &v_full[st], c * 64, j0, w.hk, w.s);
          // the next tile's rows, once this tile's have been taken out (after the copies that are needed first)
          if (i == min(1, kr.count - 1) && unit + (int)gridDim.x < units) {
            ptx::mbar_wait(q_ready, u & 1, abort_flag, p.status, 123);
            if ((stop = abort_flag[0] != 0)) {
              ++g;  // (this step's V is under way)
              break;
            }
            land(unit + gridDim.x);
            ++landed;
          }
        }
      }
      // every copy has landed before the CTA gives up its shared memory
      ptx::mbar_wait_drain(land_full, (landed - 1) & 1, abort_flag, p.status, 124);
      for (int i = keys > 2 ? keys - 2 : 0; i < keys; ++i) ptx::mbar_wait_drain(&k_full[i & 1], (i >> 1) & 1, abort_flag, p.status, 124);
      for (int i = g > 2 ? g - 2 : 0; i < g; ++i) ptx::mbar_wait_drain(&v_full[i & 1], (i >> 1) & 1, abort_flag, p.status, 124);
    }
    __syncwarp();
  } else if (warp == 1) {
    // The whole warp walks the loop and waits; one elected lane issues. (With the waits in the elected lane
    // alone, a commit was seen to take effect only after that lane's next wait had given up.)
    const bool elected = ptx::elect_one();
    auto wait_ = [&](uint64_t* bar, uint32_t parity, int code) {
      ptx::mbar_wait(bar, parity, abort_flag, p.status, code);
      __syncwarp();
    };
    auto commit_ = [&](uint64_t* bar) {
      if (elected) ptx::umma_commit(bar);
    };
    const uint64_t dk = ptx::make_smem_desc(ptx::smem_u32(k_smem), 16, 1024), dv = ptx::make_smem_desc(ptx::smem_u32(v_smem), 16, 1024);
    const uint64_t dk_t = ptx::make_smem_desc(ptx::smem_u32(k_smem), BOX_BYTES, 1024);  // read along the keys
    constexpr uint64_t STAGE = static_cast<uint64_t>(TILE_BYTES >> 4);
    auto score = [&](uint32_t col, uint32_t from, uint64_t bd) {
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks)
        if (elected)
          ptx::umma_ts(tmem_base + col, tmem_base + from + ks * 8, bd + static_cast<uint64_t>(((ks >> 2) * BOX_BYTES + (ks & 3) * 32) >> 4),
                       IDESC_S, ks != 0);
    };
    auto scores_of = [&](int g) {
      if (g > 0) wait_(s_free, (g - 1) & 1, 125);
      wait_(&k_full[g & 1], (g >> 1) & 1, 126);
      ptx::tc_fence_after();
      score(COL_S, COL_Q, dk + (g & 1) * STAGE);
      commit_(s_ready);
    };
    auto gradients_of = [&](int g) {  // (over dS(g-1), which dQ(g-1) reads first on the in-order pipe)
      wait_(&v_full[g & 1], (g >> 1) & 1, 127);
      ptx::tc_fence_after();
      score(COL_DP, COL_DO, dv + (g & 1) * STAGE);
      commit_(dp_ready);
      commit_(&v_empty[g & 1]);
    };
    int g = 0, u = 0;
    for (int unit = blockIdx.x; unit < units; unit += gridDim.x, ++u) {
      const int steps = walk_of(unit_at(unit)).count;
      wait_(q_ready, u & 1, 128);
      ptx::tc_fence_after();
      scores_of(g);
      gradients_of(g);
      for (int i = 0; i < steps; ++i, ++g) {
        if (i + 1 < steps) scores_of(g + 1);
        wait_(ds_ready, g & 1, 129);
        ptx::tc_fence_after();
#pragma unroll
        for (int ks = 0; ks < TILE / 16; ++ks)  // (a thread packs dS into the first half of its own 64 columns)
          if (elected)
            ptx::umma_ts(tmem_base + COL_DQ, tmem_base + COL_DP + (ks >> 2) * 64 + (ks & 3) * 8,
                         dk_t + (g & 1) * STAGE + static_cast<uint64_t>((ks * 2048) >> 4), IDESC_D, (i | ks) != 0);
        commit_(&k_empty[g & 1]);
        if (i + 1 < steps) gradients_of(g + 1);
      }
      commit_(tile_done);
    }
    // everything issued has completed before tensor memory is freed
    ptx::mbar_wait_drain(tile_done, (u - 1) & 1, abort_flag, p.status, 130);
    __syncwarp();
  } else if (warp < 4) {
    // -------------------------------------------------------------- -lse log2e, -delta
    const int t = threadIdx.x - 64;
    int u = 0;
    for (int unit = blockIdx.x; unit < units; unit += gridDim.x, ++u) {
      const Unit w = unit_at(unit);
      float nlse[2], ndelta[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {  // rows t and t + 64
        const int r = t + 64 * i;
        nlse[i] = ndelta[i] = 0.f;
        if (r < w.ntok * a.G) {
          const int pos = w.t0 + r / a.G;
          const int64_t at = (((int64_t)w.s * a.KV + w.hk) * p.col_tiles + pos / p.col_tokens) * COLS + (pos % p.col_tokens) * a.G + r % a.G;
          nlse[i] = p.nlse2[at];
          ndelta[i] = p.ndelta[at];
        }
      }
      ptx::mbar_wait(&stats_empty[u & 1], ((u >> 1) & 1) ^ 1, abort_flag, p.status, 131);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = t + 64 * i;
        stats[(u & 1) * 2 * TILE + r] = nlse[i];
        stats[((u & 1) * 2 + 1) * TILE + r] = ndelta[i];
      }
      ptx::mbar_arrive(&stats_full[u & 1]);
    }
  } else {
    // -------------------------------------------------------------- compute
    const int quarter = warp & 3, half = (warp - 4) >> 2;
    const int r = quarter * 32 + lane;
    const int row_token = r / a.G;
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t s_addr = tmem_base + lane_off + COL_S + half * 64, dp_addr = tmem_base + lane_off + COL_DP + half * 64;
    const uint64_t scale2 = am::pack2f(p.scale_log2, p.scale_log2);
    int g = 0, u = 0;
    for (int unit = blockIdx.x; unit < units; unit += gridDim.x, ++u) {
      const Unit w = unit_at(unit);
      const KeyRange kr = walk_of(w);
      const bool live = r < w.ntok * a.G;
      const int pos = live ? w.t0 + row_token : -1;
      // half 0 puts the rows of Q into tensor memory, half 1 those of dO (the products that read the
      // previous tile's are done: tile_done)
      ptx::mbar_wait(land_full, u & 1, abort_flag, p.status, 132);
      {
        const uint8_t* src = land_smem + half * TILE_BYTES + r * 128;
#pragma unroll
        for (int c = 0; c < D / 64; ++c) {
          uint32_t v[32];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const uint4 x = *reinterpret_cast<const uint4*>(src + c * BOX_BYTES + ((e ^ (r & 7)) << 4));
            v[e * 4] = x.x;
            v[e * 4 + 1] = x.y;
            v[e * 4 + 2] = x.z;
            v[e * 4 + 3] = x.w;
          }
          ptx::tmem_st32(tmem_base + lane_off + (half ? COL_DO : COL_Q) + c * 32, v);
        }
        ptx::tmem_st_wait();
        ptx::fence_proxy_async_smem();  // (the landing zone is next written by copies)
        ptx::tc_fence_before();
        ptx::mbar_arrive(q_ready);
      }
      if (threadIdx.x == 128) {
        ptx::bulk_wait_read();
        ptx::mbar_arrive(out_free);
      }
      ptx::mbar_wait(&stats_full[u & 1], (u >> 1) & 1, abort_flag, p.status, 133);
      const float nlse = stats[(u & 1) * 2 * TILE + r], ndelta = stats[((u & 1) * 2 + 1) * TILE + r];
      ptx::mbar_arrive(&stats_empty[u & 1]);
      const uint64_t nlse_2 = am::pack2f(nlse, nlse), ndelta_2 = am::pack2f(ndelta, ndelta);
      for (int i = 0; i < kr.count; ++i, ++g) {
        const int j0 = kr.tile(i) * TILE;
        const bool plain = j0 + TILE - 1 <= w.t0 && (w.t0 + w.ntok - 1 - j0 < a.window || j0 + TILE <= a.sinks);
        float pr[64];
        uint32_t ra[32], rb[32];
        ptx::mbar_wait(s_ready, g & 1, abort_flag, p.status, 134);
        ptx::tc_fence_after();
        ptx::tmem_ld32(s_addr, ra);
        ptx::tmem_ld32(s_addr + 32, rb);
        am::tmem_ld_wait_dep(ra);
        am::tmem_ld_wait_dep(rb);
        ptx::tc_fence_before();
        ptx::mbar_arrive(s_free);
        if (plain) {
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            am::unpack2f(am::fma2(am::pack2u(ra[e], ra[e + 1]), scale2, nlse_2), pr[e], pr[e + 1]);
            am::unpack2f(am::fma2(am::pack2u(rb[e], rb[e + 1]), scale2, nlse_2), pr[32 + e], pr[33 + e]);
          }
#pragma unroll
          for (int e = 0; e < 64; ++e) pr[e] = am::ex2(pr[e]);
        } else {
          // by blocks of 32 columns: those that no row sees cost nothing, those that all rows see no mask
          auto block = [&](const uint32_t (&v)[32], int q) {
            const int b0 = j0 + half * 64 + 32 * q, last = w.t0 + w.ntok - 1;
            const bool none = b0 > last || (w.t0 - (b0 + 31) >= a.window && b0 >= a.sinks);
            const bool all = b0 + 31 <= w.t0 && (last - b0 < a.window || b0 + 32 <= a.sinks);
            if (none) {
#pragma unroll
              for (int e = 0; e < 32; ++e) pr[q * 32 + e] = 0.f;
              return;
            }
#pragma unroll
            for (int e = 0; e < 32; e += 2)
              am::unpack2f(am::fma2(am::pack2u(v[e], v[e + 1]), scale2, nlse_2), pr[q * 32 + e], pr[q * 32 + e + 1]);
#pragma unroll
            for (int e = 0; e < 32; ++e) pr[q * 32 + e] = am::ex2(pr[q * 32 + e]);
            if (all) return;
            // columns below pos + 1 - b0 are not in the future, those from pos - window + 1 - b0 on in the window
            const uint32_t seen = low_bits(pos + 1 - b0) & (~low_bits(saturate((int64_t)pos - a.window + 1 - b0)) | low_bits(a.sinks - b0));
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (!(seen & (1u << e))) pr[q * 32 + e] = 0.f;
          };
          block(ra, 0);
          block(rb, 1);
        }
        ptx::mbar_wait(dp_ready, g & 1, abort_flag, p.status, 135);
        ptx::tc_fence_after();
        ptx::tmem_ld32(dp_addr, ra);
        ptx::tmem_ld32(dp_addr + 32, rb);
        am::tmem_ld_wait_dep(ra);
        am::tmem_ld_wait_dep(rb);
        uint32_t packed[32];
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          float d0, d1;
          am::unpack2f(am::mul2(am::pack2f(pr[e], pr[e + 1]), am::add2(am::pack2u(ra[e], ra[e + 1]), ndelta_2)), d0, d1);
          packed[e >> 1] = am::cvt_pair<T>(d0, d1);
          am::unpack2f(am::mul2(am::pack2f(pr[32 + e], pr[33 + e]), am::add2(am::pack2u(rb[e], rb[e + 1]), ndelta_2)), d0, d1);
          packed[16 + (e >> 1)] = am::cvt_pair<T>(d0, d1);
        }
        ptx::tmem_st32(dp_addr, packed);
        ptx::tmem_st_wait();
        ptx::tc_fence_before();
        ptx::mbar_arrive(ds_ready);
      }
      // dQ out through shared memory, once the last tile's has left it: each half of the warps takes half of the features
      ptx::mbar_wait(out_free, u & 1, abort_flag, p.status, 137);
      ptx::mbar_wait(tile_done, u & 1, abort_flag, p.status, 136);
      ptx::tc_fence_after();
#pragma unroll
      for (int c = 0; c < D / 64; ++c) {
        uint32_t v[32];
        ptx::tmem_ld32(tmem_base + lane_off + COL_DQ + half * (D / 2) + c * 32, v);
        ptx::tmem_ld_wait();
        const int chunk0 = (half * (D / 2) + c * 32) / 8;  // first 16-byte chunk of the row
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint4 o;
          o.x = am::cvt_pair<T>(__uint_as_float(v[e * 8 + 0]) * a.scale, __uint_as_float(v[e * 8 + 1]) * a.scale);
          o.y = am::cvt_pair<T>(__uint_as_float(v[e * 8 + 2]) * a.scale, __uint_as_float(v[e * 8 + 3]) * a.scale);
          o.z = am::cvt_pair<T>(__uint_as_float(v[e * 8 + 4]) * a.scale, __uint_as_float(v[e * 8 + 5]) * a.scale);
          o.w = am::cvt_pair<T>(__uint_as_float(v[e * 8 + 6]) * a.scale, __uint_as_float(v[e * 8 + 7]) * a.scale);
          const int chunk = chunk0 + e;
          *reinterpret_cast<uint4*>(out_smem + (chunk >> 3) * BOX_BYTES + r * 128 + (((chunk & 7) ^ (r & 7)) << 4)) = o;
        }
      }
      ptx::tc_fence_before();
      ptx::fence_proxy_async_smem();
      asm volatile("bar.sync 1, 256;" ::: "memory");
      if (threadIdx.x == 128) {
#pragma unroll
        for (int c = 0; c < NBOX; ++c) ptx::tma_store_5d(&map_dq, out_smem + c * BOX_BYTES, c * 64, 0, w.t0, w.hk, w.s);
        ptx::bulk_commit();
      }
    }
    if (threadIdx.x == 128) ptx::bulk_wait_done();
  }
  ptx::tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

template <typename Kernel>
int optin(Kernel kern, int bytes, std::atomic<unsigned long long>& done) {
  const cudaError_t e = smem_optin_per_device(done, reinterpret_cast<const void*>(kern), bytes);
  if (e == cudaSuccess) return 0;
  set_error("window_attention_bwd: cudaFuncSetAttribute failed: %s", cudaGetErrorString(e));
  return (int)e;
}

}  // namespace

bool local_bwd_tc_supported(const LocalBwdArgs& b, int dtype, const void* q, const void* k, const void* v, const void* out,
                            const void* dout, const void* dq, const void* dk, const void* dv) {
  return (int64_t)b.f.n * b.f.KV * ceil_div(b.f.tokens, LOCAL_TC_TILE / b.f.G) < (1ll << 31) - (1 << 20) &&
         local_tc_supported(b.f, dtype, q, k, v, out) && local_rows_ok(dout, b.dos, b.f) && local_rows_ok(dq, b.dqs, b.f) &&
         local_keys_ok(dk, b.dks, b.f) && local_keys_ok(dv, b.dvs, b.f);
}

int launch_local_bwd_tc(void* dq, void* dk, void* dv, const void* dout, const void* q, const void* k, const void* v,
                        const void* out, const float* lse, float* row_scratch, const LocalBwdArgs& b, int dtype,
                        cudaStream_t st) {
  const LocalArgs& a = b.f;
  const int col_tokens = COLS / a.G;
  CUtensorMap mq, md, mq128, md128, mk, mv, mdq;
  bind_primary_context();
  if (!local_map_rows(&mq, q, a.qs, a, col_tokens, "q") || !local_map_rows(&md, dout, b.dos, a, col_tokens, "dout") ||
      !local_map_rows(&mq128, q, a.qs, a, TILE / a.G, "q") || !local_map_rows(&md128, dout, b.dos, a, TILE / a.G, "dout") ||
      !local_map_rows(&mdq, dq, b.dqs, a, TILE / a.G, "dq") || !local_map_keys(&mk, k, a.ks, a, TILE, "k") ||
      !local_map_keys(&mv, v, a.vs, a, TILE, "v"))
    return TB200_ERR_UNSUPPORTED;
  BwdParams p;
  p.b = b;
  p.dk = dk;
  p.dv = dv;
  p.lse = lse;
  p.nlse2 = row_scratch;
  p.ndelta = row_scratch + local_tc_rows(a);
  p.scale_log2 = a.scale * LOG2E;
  p.tile_tokens = TILE / a.G;
  p.row_tiles = (int)ceil_div(a.tokens, p.tile_tokens);
  p.col_tokens = col_tokens;
  p.col_tiles = (int)ceil_div(a.tokens, col_tokens);
  p.key_tiles = (int)ceil_div(a.tokens, TILE);
  p.heads = Divisor(a.n * a.KV);
  p.kv = Divisor(a.KV);
  p.status = device_status_ptr();
  p.test_dq = WaitTest::of_this_thread(1, 1);
  p.test_dkv = WaitTest::of_this_thread(2, 1);
  const int64_t parts = (int64_t)a.n * a.KV * (p.key_tiles + (int64_t)b.sink_tiles * b.far);
  TB200_REQUIRE(parts < (1ll << 31), TB200_ERR_UNSUPPORTED, "local_dkv_tc: %lld walks", (long long)parts);
  auto go = [&](auto tag, auto dsel) -> int {
    using T = decltype(tag);
    constexpr int D = decltype(dsel)::value;
    constexpr int DKV_SMEM = 2 * TILE * D * 2 + 6 * COLS * D * 2 + 6 * COLS * 4 + 256 + 1024;
    constexpr int DQ_SMEM = 7 * TILE * D * 2 + 4 * TILE * 4 + 256;
    static_assert(DKV_SMEM <= 227 * 1024 && DQ_SMEM <= 227 * 1024, "shared memory of one CTA");
    auto kkv = local_dkv_tc_kernel<T, D>;
    auto kq = local_dq_tc_kernel<T, D>;
    static std::atomic<unsigned long long> done_kv{0}, done_q{0};
    if (int rc = optin(kkv, DKV_SMEM, done_kv)) return rc;
    if (int rc = optin(kq, DQ_SMEM, done_q)) return rc;
    const int64_t units = (int64_t)a.n * a.KV * p.row_tiles;
    local_rows_tc_kernel<T, D><<<(unsigned)ceil_div(local_tc_rows(a), 16 * 8), 256, 0, st>>>((const T*)out, (const T*)dout, p);
    if (int rc = launch_status("local_rows_tc")) return rc;
    kq<<<(unsigned)(units < sm_count() ? units : sm_count()), THREADS, DQ_SMEM, st>>>(mq128, md128, mdq, mk, mv, p);
    if (int rc = launch_status("local_dq_tc")) return rc;
    kkv<<<(unsigned)parts, THREADS, DKV_SMEM, st>>>(mq, md, mk, mv, p);
    return launch_status("local_dkv_tc");
  };
  using D64 = std::integral_constant<int, 64>;
  using D128 = std::integral_constant<int, 128>;
  if (dtype == TB200_BF16) return a.D == 128 ? go(__nv_bfloat16{}, D128{}) : go(__nv_bfloat16{}, D64{});
  return a.D == 128 ? go(__half{}, D128{}) : go(__half{}, D64{});
}

}  // namespace tb200
