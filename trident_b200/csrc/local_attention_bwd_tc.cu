// tcgen05 backward of window attention with sinks, for 16-bit operands with head size 64 or 128.
//
// Two kernels, each of which owns what it sums, so that nothing is added with atomics and the same inputs
// give the same bits (one kernel for all three gradients would need 5 products a tile pair instead of 7,
// but has to add dQ across CTAs):
//
//   dK, dV  a CTA owns 128 keys (K_j, V_j resident) and walks the tiles of 128 packed query rows (token *
//           G + head) that see any of them; the sum over the heads of a group is part of the walk. All
//           transposed, keys on the tensor-memory lanes:
//             S^T = K_j Q^T, dP^T = V_j dO^T, P^T = exp2(S^T scale log2e - lse log2e), dS^T = P^T (dP^T - delta),
//             dV += P^T dO, dK += dS^T Q   (P^T, dS^T 16-bit in tensor memory over S^T and dP^T)
//           The tensor pipe runs dP^T(s) | dV(s) | S^T(s+1) | dK(s): while the compute warps are in one
//           of their two stages (exponentials; score gradients) it has the other's products to run.
//   dQ      a CTA owns a tile of 128 packed query rows (Q, dO resident) and walks the keys it sees:
//             S = Q K^T (two buffers), dP = dO V^T, dS = P (dP - delta) over S, dQ += dS K
//
// The queries beyond the window of a key tile that holds sinks ("far", LocalBwdArgs) are cut into pieces
// about as long as a walk inside the window, each a CTA of its own: a single CTA would walk all queries.
//
// A first kernel computes -delta = -sum_d out dout and -lse log2e, laid out by query tile; rows that do
// not exist get -lse = -inf, so that their probabilities are 0.
//
// Bound by the tensor pipe and, next to it, the exponentials: at D = 128 the four products of a step of
// the first kernel take 2048 cycles, the three of the second 1536, the 16 K exponentials of either 1024.
#include <type_traits>

#include "attn_math.cuh"
#include "local_attention_tc.cuh"
#include "ptx.cuh"

namespace tb200 {
namespace {

constexpr int TILE = LOCAL_TC_TILE;
constexpr int THREADS = 384;  // 4 service warps, 8 compute warps: two threads per row, 64 columns each
constexpr float LOG2E = 1.4426950408889634f;

struct BwdParams {
  LocalBwdArgs b;
  void *dq, *dk, *dv;
  const float* nlse2;   // [n * KV][query tiles][128]  -lse * log2(e)
  const float* ndelta;  // [n * KV][query tiles][128]
  float scale_log2;
  int tile_tokens;      // tokens of a query tile
  int query_tiles, key_tiles;
  int* status;
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
__device__ inline uint32_t low_bits(int n) { return n <= 0 ? 0u : (n >= 32 ? 0xffffffffu : (1u << n) - 1u); }
__device__ inline int saturate(int64_t v) { return v < -(1 << 20) ? -(1 << 20) : (v > (1 << 20) ? (1 << 20) : (int)v); }
// Column of the packed 16-bit copy of the 32 columns `c` of a score row: each compute thread packs into
// the 64 columns it has read itself.
__host__ __device__ constexpr uint32_t packed_col(int c) { return static_cast<uint32_t>((c >> 1) * 64 + (c & 1) * 16); }

// Rows [rows, 128) of `tiles` swizzled tiles set to zero (rows that no copy writes, but products read).
template <int NBOX>
__device__ inline void zero_rows(uint8_t* smem, int tiles, int rows) {
  const int per_box = (TILE - rows) * 8;  // 16-byte chunks
  for (int i = threadIdx.x; i < tiles * NBOX * per_box; i += THREADS)
    *reinterpret_cast<uint4*>(smem + (i / per_box) * (TILE * 128) + rows * 128 + (i % per_box) * 16) = make_uint4(0, 0, 0, 0);
}

// ------------------------------------------------------------------ dK, dV
template <typename T, int D>
__global__ void __launch_bounds__(THREADS, 1)
    local_dkv_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_do,
                        const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                        const BwdParams p) {
  constexpr int TILE_BYTES = TILE * D * 2, NBOX = D / 64, BOX_BYTES = TILE * 128;
  constexpr bool IS_BF16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr uint32_t IDESC_S = ptx::make_idesc(IS_BF16, false, false, TILE, TILE);
  constexpr uint32_t IDESC_D = ptx::make_idesc(IS_BF16, false, true, TILE, D);
  constexpr uint32_t TMEM_COLS = 512, COL_S = 0, COL_P = 128, COL_DV = 256, COL_DK = 256 + D;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* k_smem = smem;
  uint8_t* v_smem = smem + TILE_BYTES;
  uint8_t* q_smem = smem + 2 * TILE_BYTES;   // [2]
  uint8_t* do_smem = smem + 4 * TILE_BYTES;  // [2]
  float* nlse_smem = reinterpret_cast<float*>(smem + 6 * TILE_BYTES);  // [2][128]
  float* ndelta_smem = nlse_smem + 256;                                // [2][128]
  uint64_t* bars = reinterpret_cast<uint64_t*>(ndelta_smem + 256);
  uint64_t* kv_full = bars;
  uint64_t* qdo_full = bars + 1;   // [2]
  uint64_t* qdo_empty = bars + 3;  // [2]
  uint64_t* s_ready = bars + 5;    // S^T(s) computed
  uint64_t* p_ready = bars + 6;    // P^T(s) written      (256 arrivals)
  uint64_t* dp_ready = bars + 7;   // dP^T(s) computed
  uint64_t* ds_ready = bars + 8;   // dS^T(s) written     (256 arrivals)
  uint64_t* all_done = bars + 9;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 10);
  volatile uint32_t* abort_flag = tmem_slot + 1;

  const LocalArgs& a = p.b.f;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int s = blockIdx.z, hk = blockIdx.y;
  // the walk: query tiles [i0, i0 + steps)
  int jt = blockIdx.x, piece = -1, i0, i1;
  const bool far = jt >= p.key_tiles;
  if (far) {
    piece = (jt - p.key_tiles) % p.b.far;
    jt = (jt - p.key_tiles) / p.b.far;
  }
  const int beyond = (near_end(a, jt, TILE) + p.tile_tokens - 1) / p.tile_tokens;  // first query tile beyond the window
  if (far) {
    const int64_t span = p.query_tiles - beyond;
    i0 = beyond + (int)(span * piece / p.b.far);
    i1 = beyond + (int)(span * (piece + 1) / p.b.far);
  } else {
    i0 = jt * TILE / p.tile_tokens;
    i1 = beyond;
  }
  const int steps = i1 - i0;
  const int rows = p.tile_tokens * a.G;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 10; ++i) ptx::mbar_init(&bars[i], (i == 6 || i == 8) ? 256 : 1);
    abort_flag[0] = 0;
    abort_flag[1] = ptx::WAIT_LIMIT_UNITS;
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
  if (rows < TILE) {
    zero_rows<NBOX>(q_smem, 4, rows);
    ptx::fence_proxy_async_smem();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    if (lane == 0 && steps > 0) {
      ptx::mbar_expect_tx(kv_full, 2 * TILE_BYTES);
#pragma unroll
      for (int c = 0; c < NBOX; ++c) {
        tma_load_4d(k_smem + c * BOX_BYTES, &map_k, kv_full, c * 64, jt * TILE, hk, s);
        tma_load_4d(v_smem + c * BOX_BYTES, &map_v, kv_full, c * 64, jt * TILE, hk, s);
      }
      for (int i = 0; i < steps; ++i) {
        const int st = i & 1, it = i0 + i;
        ptx::mbar_wait(&qdo_empty[st], ((i >> 1) & 1) ^ 1, abort_flag, p.status, 101);
        ptx::mbar_expect_tx(&qdo_full[st], 2 * NBOX * rows * 128 + 2 * 512);
#pragma unroll
        for (int c = 0; c < NBOX; ++c) {
          tma_load_5d(q_smem + st * TILE_BYTES + c * BOX_BYTES, &map_q, &qdo_full[st], c * 64, 0, it * p.tile_tokens, hk, s);
          tma_load_5d(do_smem + st * TILE_BYTES + c * BOX_BYTES, &map_do, &qdo_full[st], c * 64, 0, it * p.tile_tokens, hk, s);
        }
        const int64_t row0 = (((int64_t)s * a.KV + hk) * p.query_tiles + it) * TILE;
        bulk_load(nlse_smem + st * 128, p.nlse2 + row0, 512, &qdo_full[st]);
        bulk_load(ndelta_smem + st * 128, p.ndelta + row0, 512, &qdo_full[st]);
      }
      // every copy has landed before the CTA gives up its shared memory
      ptx::mbar_wait_drain(kv_full, 0, abort_flag, p.status, 102);
      for (int i = steps > 2 ? steps - 2 : 0; i < steps; ++i)
        ptx::mbar_wait_drain(&qdo_full[i & 1], (i >> 1) & 1, abort_flag, p.status, 102);
    }
    __syncwarp();
  } else if (warp == 1) {
    const bool elected = ptx::elect_one();
    auto wait_ = [&](uint64_t* bar, uint32_t parity, int code) {
      if (elected) ptx::mbar_wait(bar, parity, abort_flag, p.status, code);
      __syncwarp();
    };
    auto commit_ = [&](uint64_t* bar) {
      if (elected) ptx::umma_commit(bar);
    };
    const uint64_t dk = ptx::make_smem_desc(ptx::smem_u32(k_smem), 16, 1024), dv = ptx::make_smem_desc(ptx::smem_u32(v_smem), 16, 1024);
    const uint64_t dq = ptx::make_smem_desc(ptx::smem_u32(q_smem), 16, 1024), dd = ptx::make_smem_desc(ptx::smem_u32(do_smem), 16, 1024);
    const uint64_t dq_t = ptx::make_smem_desc(ptx::smem_u32(q_smem), BOX_BYTES, 1024);   // read along the rows
    const uint64_t dd_t = ptx::make_smem_desc(ptx::smem_u32(do_smem), BOX_BYTES, 1024);
    constexpr uint64_t NEXT = static_cast<uint64_t>(TILE_BYTES >> 4);
    auto score = [&](uint32_t col, uint64_t ad, uint64_t bd) {  // [keys][rows] = A B^T over the features
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        const uint64_t off = static_cast<uint64_t>(((ks >> 2) * BOX_BYTES + (ks & 3) * 32) >> 4);
        if (elected) ptx::umma_ss(tmem_base + col, ad + off, bd + off, IDESC_S, ks != 0);
      }
    };
    auto gather = [&](uint32_t col, uint32_t from, uint64_t bd, bool accumulate) {  // [keys][features] += P B over the rows
#pragma unroll
      for (int ks = 0; ks < TILE / 16; ++ks)
        if (elected)
          ptx::umma_ts(tmem_base + col, tmem_base + from + packed_col(ks >> 1) + (ks & 1) * 8,
                       bd + static_cast<uint64_t>((ks * 2048) >> 4), IDESC_D, accumulate || ks != 0);
    };
    if (steps > 0) {
      wait_(kv_full, 0, 103);
      wait_(&qdo_full[0], 0, 104);
      ptx::tc_fence_after();
      score(COL_S, dk, dq);
      commit_(s_ready);
      for (int i = 0; i < steps; ++i) {
        const uint32_t ph = i & 1;
        const uint64_t cur = (i & 1) ? NEXT : 0, nxt = (i & 1) ? 0 : NEXT;
        score(COL_P, dv, dd + cur);  // dP^T(i): dK(i-1), issued before, has read dS^T(i-1)
        commit_(dp_ready);
        wait_(p_ready, ph, 105);
        ptx::tc_fence_after();
        gather(COL_DV, COL_S, dd_t + cur, i > 0);
        if (i + 1 < steps) {
          wait_(&qdo_full[(i + 1) & 1], ((i + 1) >> 1) & 1, 106);
          ptx::tc_fence_after();
          score(COL_S, dk, dq + nxt);  // (over P^T(i), which dV(i) reads first on the in-order pipe)
          commit_(s_ready);
        }
        wait_(ds_ready, ph, 107);
        ptx::tc_fence_after();
        gather(COL_DK, COL_P, dq_t + cur, i > 0);
        commit_(&qdo_empty[i & 1]);
      }
    }
    commit_(all_done);
    if (elected) ptx::mbar_wait_drain(all_done, 0, abort_flag, p.status, 108);
    __syncwarp();
  } else if (warp >= 4) {
    const int quarter = warp & 3, half = (warp - 4) >> 2;
    const int r = quarter * 32 + lane, key = jt * TILE + r;
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t s_addr = tmem_base + lane_off + COL_S + half * 64, p_addr = tmem_base + lane_off + COL_P + half * 64;
    const uint64_t scale2 = am::pack2f(p.scale_log2, p.scale_log2);
    const uint32_t always = key < a.sinks ? 0xffffffffu : 0u;
    for (int i = 0; i < steps; ++i) {
      const int st = i & 1, it = i0 + i;
      const int token0 = it * p.tile_tokens, token1 = token0 + p.tile_tokens - 1;
      // every query of the tile sees every key of this one
      const bool plain = token0 >= jt * TILE + TILE - 1 && (token1 - jt * TILE < a.window || (jt + 1) * TILE <= a.sinks);
      const float4* nlse4 = reinterpret_cast<const float4*>(nlse_smem + st * 128 + half * 64);
      const float4* ndel4 = reinterpret_cast<const float4*>(ndelta_smem + st * 128 + half * 64);
      float pr[64];
      ptx::mbar_wait(&qdo_full[st], (i >> 1) & 1, abort_flag, p.status, 109);
      ptx::mbar_wait(s_ready, i & 1, abort_flag, p.status, 110);
      ptx::tc_fence_after();
      {
        uint32_t ra[32], rb[32];
        // columns from `low` on are not before the key, those below `high` are within its window
        const int low = saturate((int64_t)(key - token0) * a.G) - half * 64;
        const int high = saturate(((int64_t)key + a.window - token0) * a.G) - half * 64;
        auto exp32 = [&](const uint32_t (&v)[32], int q) {
#pragma unroll
          for (int g = 0; g < 8; ++g) {
            const float4 nl = nlse4[q * 8 + g];
            am::unpack2f(am::fma2(am::pack2u(v[g * 4], v[g * 4 + 1]), scale2, am::pack2f(nl.x, nl.y)), pr[q * 32 + g * 4],
                         pr[q * 32 + g * 4 + 1]);
            am::unpack2f(am::fma2(am::pack2u(v[g * 4 + 2], v[g * 4 + 3]), scale2, am::pack2f(nl.z, nl.w)),
                         pr[q * 32 + g * 4 + 2], pr[q * 32 + g * 4 + 3]);
          }
#pragma unroll
          for (int e = 0; e < 32; ++e) pr[q * 32 + e] = am::ex2(pr[q * 32 + e]);
          if (!plain) {
            const uint32_t seen = ~low_bits(low - 32 * q) & (low_bits(high - 32 * q) | always);
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (!((seen >> e) & 1u)) pr[q * 32 + e] = 0.f;
          }
          uint32_t packed[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) packed[e] = am::cvt_pair<T>(pr[q * 32 + 2 * e], pr[q * 32 + 2 * e + 1]);
          ptx::tmem_st16(s_addr + q * 16, packed);
        };
        ptx::tmem_ld32(s_addr, ra);
        am::tmem_ld_wait_dep(ra);
        ptx::tmem_ld32(s_addr + 32, rb);
        am::tmem_ld_wait_dep(rb);  // (both blocks are read before the packed copy goes over them)
        exp32(ra, 0);
        exp32(rb, 1);
        ptx::tmem_st_wait();
        ptx::tc_fence_before();
        ptx::mbar_arrive(p_ready);
      }
      ptx::mbar_wait(dp_ready, i & 1, abort_flag, p.status, 111);
      ptx::tc_fence_after();
      {
        uint32_t ra[32], rb[32];
        auto grad32 = [&](const uint32_t (&v)[32], int q) {
          uint32_t packed[16];
#pragma unroll
          for (int g = 0; g < 8; ++g) {
            const float4 nd = ndel4[q * 8 + g];
            float d0, d1, d2, d3;
            am::unpack2f(am::mul2(am::pack2f(pr[q * 32 + g * 4], pr[q * 32 + g * 4 + 1]),
                                  am::add2(am::pack2u(v[g * 4], v[g * 4 + 1]), am::pack2f(nd.x, nd.y))), d0, d1);
            am::unpack2f(am::mul2(am::pack2f(pr[q * 32 + g * 4 + 2], pr[q * 32 + g * 4 + 3]),
                                  am::add2(am::pack2u(v[g * 4 + 2], v[g * 4 + 3]), am::pack2f(nd.z, nd.w))), d2, d3);
            packed[g * 2] = am::cvt_pair<T>(d0, d1);
            packed[g * 2 + 1] = am::cvt_pair<T>(d2, d3);
          }
          ptx::tmem_st16(p_addr + q * 16, packed);
        };
        ptx::tmem_ld32(p_addr, ra);
        am::tmem_ld_wait_dep(ra);
        ptx::tmem_ld32(p_addr + 32, rb);
        am::tmem_ld_wait_dep(rb);
        grad32(ra, 0);
        grad32(rb, 1);
        ptx::tmem_st_wait();
        ptx::tc_fence_before();
        ptx::mbar_arrive(ds_ready);
      }
    }
    // epilogue: the first half of the warps writes dV, the second dK
    ptx::mbar_wait(all_done, 0, abort_flag, p.status, 112);
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
template <typename T, int D>
__global__ void __launch_bounds__(THREADS, 1)
    local_dq_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_do,
                       const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                       const BwdParams p) {
  constexpr int TILE_BYTES = TILE * D * 2, NBOX = D / 64, BOX_BYTES = TILE * 128;
  constexpr bool IS_BF16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr uint32_t IDESC_S = ptx::make_idesc(IS_BF16, false, false, TILE, TILE);
  constexpr uint32_t IDESC_D = ptx::make_idesc(IS_BF16, false, true, TILE, D);
  constexpr uint32_t TMEM_COLS = 512, COL_S = 0, COL_DP = 256, COL_DQ = 384;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* q_smem = smem;
  uint8_t* do_smem = smem + TILE_BYTES;
  uint8_t* k_smem = smem + 2 * TILE_BYTES;  // [2]
  uint8_t* v_smem = smem + 4 * TILE_BYTES;  // [2]
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + 6 * TILE_BYTES);
  uint64_t* qdo_full = bars;
  uint64_t* k_full = bars + 1;    // [2]
  uint64_t* v_full = bars + 3;    // [2]
  uint64_t* kv_empty = bars + 5;  // [2]
  uint64_t* s_ready = bars + 7;   // [2] S(i) computed, by buffer i & 1
  uint64_t* ds_ready = bars + 9;  // [2] dS(i) written over S(i)   (256 arrivals)
  uint64_t* dp_ready = bars + 11; // dP(i) computed
  uint64_t* dp_free = bars + 12;  // dP(i) read                    (256 arrivals)
  uint64_t* all_done = bars + 13;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 14);
  volatile uint32_t* abort_flag = tmem_slot + 1;

  const LocalArgs& a = p.b.f;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int s = blockIdx.z, hk = blockIdx.y;
  const int it = (int)gridDim.x - 1 - (int)blockIdx.x;  // longest walks first
  const int t0 = it * p.tile_tokens, ntok = min(p.tile_tokens, a.tokens - t0);
  const KeyRange kr = key_range(a, t0, t0 + ntok - 1, a.tokens, TILE);
  const int steps = kr.count;  // (at least one: a query sees itself)

  if (threadIdx.x == 0) {
    for (int i = 0; i < 14; ++i) ptx::mbar_init(&bars[i], (i == 9 || i == 10 || i == 12) ? 256 : 1);
    abort_flag[0] = 0;
    abort_flag[1] = ptx::WAIT_LIMIT_UNITS;
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
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      const uint32_t bytes = NBOX * p.tile_tokens * a.G * 128;
      ptx::mbar_expect_tx(qdo_full, 2 * bytes);
#pragma unroll
      for (int c = 0; c < NBOX; ++c) {
        tma_load_5d(q_smem + c * BOX_BYTES, &map_q, qdo_full, c * 64, 0, t0, hk, s);
        tma_load_5d(do_smem + c * BOX_BYTES, &map_do, qdo_full, c * 64, 0, t0, hk, s);
      }
      for (int i = 0; i < steps; ++i) {
        const int st = i & 1, j0 = kr.tile(i) * TILE;
        ptx::mbar_wait(&kv_empty[st], ((i >> 1) & 1) ^ 1, abort_flag, p.status, 121);
        ptx::mbar_expect_tx(&k_full[st], TILE_BYTES);
#pragma unroll
        for (int c = 0; c < NBOX; ++c) tma_load_4d(k_smem + st * TILE_BYTES + c * BOX_BYTES, &map_k, &k_full[st], c * 64, j0, hk, s);
        ptx::mbar_expect_tx(&v_full[st], TILE_BYTES);
#pragma unroll
        for (int c = 0; c < NBOX; ++c) tma_load_4d(v_smem + st * TILE_BYTES + c * BOX_BYTES, &map_v, &v_full[st], c * 64, j0, hk, s);
      }
      ptx::mbar_wait_drain(qdo_full, 0, abort_flag, p.status, 122);
      for (int i = steps > 2 ? steps - 2 : 0; i < steps; ++i) {
        ptx::mbar_wait_drain(&k_full[i & 1], (i >> 1) & 1, abort_flag, p.status, 122);
        ptx::mbar_wait_drain(&v_full[i & 1], (i >> 1) & 1, abort_flag, p.status, 122);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    const bool elected = ptx::elect_one();
    auto wait_ = [&](uint64_t* bar, uint32_t parity, int code) {
      if (elected) ptx::mbar_wait(bar, parity, abort_flag, p.status, code);
      __syncwarp();
    };
    auto commit_ = [&](uint64_t* bar) {
      if (elected) ptx::umma_commit(bar);
    };
    const uint64_t dq = ptx::make_smem_desc(ptx::smem_u32(q_smem), 16, 1024), dd = ptx::make_smem_desc(ptx::smem_u32(do_smem), 16, 1024);
    const uint64_t dk = ptx::make_smem_desc(ptx::smem_u32(k_smem), 16, 1024), dv = ptx::make_smem_desc(ptx::smem_u32(v_smem), 16, 1024);
    const uint64_t dk_t = ptx::make_smem_desc(ptx::smem_u32(k_smem), BOX_BYTES, 1024);  // read along the keys
    constexpr uint64_t NEXT = static_cast<uint64_t>(TILE_BYTES >> 4);
    auto score = [&](uint32_t col, uint64_t ad, uint64_t bd) {
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        const uint64_t off = static_cast<uint64_t>(((ks >> 2) * BOX_BYTES + (ks & 3) * 32) >> 4);
        if (elected) ptx::umma_ss(tmem_base + col, ad + off, bd + off, IDESC_S, ks != 0);
      }
    };
    auto scores_of = [&](int i) {
      wait_(&k_full[i & 1], (i >> 1) & 1, 123);
      ptx::tc_fence_after();
      score(COL_S + (i & 1) * 128, dq, dk + ((i & 1) ? NEXT : 0));
      commit_(&s_ready[i & 1]);
    };
    auto gradients_of = [&](int i) {
      wait_(&v_full[i & 1], (i >> 1) & 1, 124);
      ptx::tc_fence_after();
      score(COL_DP, dd, dv + ((i & 1) ? NEXT : 0));
      commit_(dp_ready);
    };
    wait_(qdo_full, 0, 125);
    scores_of(0);
    gradients_of(0);
    for (int i = 0; i < steps; ++i) {
      if (i + 1 < steps) {
        scores_of(i + 1);  // (over dS(i-1), which dQ(i-1) reads first on the in-order pipe)
        wait_(dp_free, i & 1, 126);
        ptx::tc_fence_after();
        gradients_of(i + 1);
      }
      wait_(&ds_ready[i & 1], (i >> 1) & 1, 127);
      ptx::tc_fence_after();
#pragma unroll
      for (int ks = 0; ks < TILE / 16; ++ks)
        if (elected)
          ptx::umma_ts(tmem_base + COL_DQ, tmem_base + COL_S + (i & 1) * 128 + packed_col(ks >> 1) + (ks & 1) * 8,
                       dk_t + ((i & 1) ? NEXT : 0) + static_cast<uint64_t>((ks * 2048) >> 4), IDESC_D, (i | ks) != 0);
      commit_(&kv_empty[i & 1]);
    }
    commit_(all_done);
    if (elected) ptx::mbar_wait_drain(all_done, 0, abort_flag, p.status, 128);
    __syncwarp();
  } else if (warp >= 4) {
    const int quarter = warp & 3, half = (warp - 4) >> 2;
    const int r = quarter * 32 + lane;
    const bool live = r < ntok * a.G;
    const int pos = live ? t0 + r / a.G : -1;
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t s_addr = tmem_base + lane_off + COL_S + half * 64, dp_addr = tmem_base + lane_off + COL_DP + half * 64;
    const int64_t row = (((int64_t)s * a.KV + hk) * p.query_tiles + it) * TILE + r;
    const float nlse = p.nlse2[row], ndelta = p.ndelta[row];
    const uint64_t scale2 = am::pack2f(p.scale_log2, p.scale_log2), nlse_2 = am::pack2f(nlse, nlse), ndelta_2 = am::pack2f(ndelta, ndelta);
    for (int i = 0; i < steps; ++i) {
      const int j0 = kr.tile(i) * TILE;
      const bool plain = j0 + TILE - 1 <= t0 && (t0 + ntok - 1 - j0 < a.window || j0 + TILE <= a.sinks);
      float pr[64];
      ptx::mbar_wait(&s_ready[i & 1], (i >> 1) & 1, abort_flag, p.status, 129);
      ptx::tc_fence_after();
      {
        uint32_t ra[32], rb[32];
        const int high = pos - j0 + 1 - half * 64;  // columns below `high` are not in the future
        const int low = saturate((int64_t)pos - a.window + 1 - j0) - half * 64, sink = a.sinks - j0 - half * 64;
        auto exp32 = [&](const uint32_t (&v)[32], int q) {
#pragma unroll
          for (int e = 0; e < 32; e += 2)
            am::unpack2f(am::fma2(am::pack2u(v[e], v[e + 1]), scale2, nlse_2), pr[q * 32 + e], pr[q * 32 + e + 1]);
#pragma unroll
          for (int e = 0; e < 32; ++e) pr[q * 32 + e] = am::ex2(pr[q * 32 + e]);
          if (!plain) {
            const uint32_t seen = low_bits(high - 32 * q) & (~low_bits(low - 32 * q) | low_bits(sink - 32 * q));
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (!((seen >> e) & 1u)) pr[q * 32 + e] = 0.f;
          }
        };
        ptx::tmem_ld32(s_addr + (i & 1) * 128, ra);
        am::tmem_ld_wait_dep(ra);
        ptx::tmem_ld32(s_addr + (i & 1) * 128 + 32, rb);
        exp32(ra, 0);
        am::tmem_ld_wait_dep(rb);
        exp32(rb, 1);
      }
      ptx::mbar_wait(dp_ready, i & 1, abort_flag, p.status, 130);
      ptx::tc_fence_after();
      {
        uint32_t ra[32], rb[32];
        auto grad32 = [&](const uint32_t (&v)[32], int q) {
          uint32_t packed[16];
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            float d0, d1;
            am::unpack2f(am::mul2(am::pack2f(pr[q * 32 + e], pr[q * 32 + e + 1]), am::add2(am::pack2u(v[e], v[e + 1]), ndelta_2)),
                         d0, d1);
            packed[e >> 1] = am::cvt_pair<T>(d0, d1);
          }
          ptx::tmem_st16(s_addr + (i & 1) * 128 + q * 16, packed);
        };
        ptx::tmem_ld32(dp_addr, ra);
        ptx::tmem_ld32(dp_addr + 32, rb);
        am::tmem_ld_wait_dep(ra);
        am::tmem_ld_wait_dep(rb);
        ptx::tc_fence_before();
        ptx::mbar_arrive(dp_free);
        grad32(ra, 0);
        grad32(rb, 1);
        ptx::tmem_st_wait();
        ptx::tc_fence_before();
        ptx::mbar_arrive(&ds_ready[i & 1]);
      }
    }
    // epilogue: each half of the warps writes half of the features
    ptx::mbar_wait(all_done, 0, abort_flag, p.status, 131);
    ptx::tc_fence_after();
    T* out = reinterpret_cast<T*>(p.dq) + (int64_t)s * p.b.dqs[0] + (int64_t)(hk * a.G + r % a.G) * p.b.dqs[1] +
             (int64_t)(t0 + r / a.G) * p.b.dqs[2] + half * (D / 2);
#pragma unroll 1
    for (int c = 0; c < D / 64; ++c) {
      uint32_t v[32];
      __syncwarp();
      ptx::tmem_ld32(tmem_base + lane_off + COL_DQ + half * (D / 2) + c * 32, v);
      ptx::tmem_ld_wait();
      if (live) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          uint4 o;
          o.x = am::cvt_pair<T>(__uint_as_float(v[g * 8 + 0]) * a.scale, __uint_as_float(v[g * 8 + 1]) * a.scale);
          o.y = am::cvt_pair<T>(__uint_as_float(v[g * 8 + 2]) * a.scale, __uint_as_float(v[g * 8 + 3]) * a.scale);
          o.z = am::cvt_pair<T>(__uint_as_float(v[g * 8 + 4]) * a.scale, __uint_as_float(v[g * 8 + 5]) * a.scale);
          o.w = am::cvt_pair<T>(__uint_as_float(v[g * 8 + 6]) * a.scale, __uint_as_float(v[g * 8 + 7]) * a.scale);
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

// ------------------------------------------------------------------ -lse log2e and -delta by query tile
// D / 8 threads a row, each one 16-byte load of out and one of dout.
template <typename T, int D>
__global__ void __launch_bounds__(256)
    local_bwd_prep(float* __restrict__ nlse2, float* __restrict__ ndelta, const T* __restrict__ out, const T* __restrict__ dout,
                   const float* __restrict__ lse, const LocalBwdArgs b, int tile_tokens, int query_tiles) {
  constexpr int TPR = D / 8;
  const LocalArgs& a = b.f;
  const int sub = threadIdx.x % TPR;
  const int64_t row = (int64_t)blockIdx.x * (256 / TPR) + threadIdx.x / TPR;
  const int64_t total = (int64_t)a.n * a.KV * query_tiles * TILE;
  const int c = (int)(row % TILE), it = (int)(row / TILE % query_tiles);
  const int64_t sh = row / TILE / query_tiles;
  const int hk = (int)(sh % a.KV), head = hk * a.G + c % a.G, t = it * tile_tokens + c / a.G;
  const int64_t s = sh / a.KV;
  const bool live = row < total && c < tile_tokens * a.G && t < a.tokens;
  float acc = 0.f;
  if (live) {
    float o[8], g[8];
    unpack<T>(ld_stream(out + s * a.os[0] + head * a.os[1] + t * a.os[2] + sub * 8), o);
    unpack<T>(ld_stream(dout + s * b.dos[0] + head * b.dos[1] + t * b.dos[2] + sub * 8), g);
#pragma unroll
    for (int i = 0; i < 8; ++i) acc = fmaf(o[i], g[i], acc);
  }
#pragma unroll
  for (int off = TPR / 2; off > 0; off >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, off);
  if (row < total && sub == 0) {
    nlse2[row] = live ? -lse[(s * a.H + head) * a.tokens + t] * LOG2E : -INFINITY;
    ndelta[row] = -acc;
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
  return local_tc_supported(b.f, dtype, q, k, v, out) && local_rows_ok(dout, b.dos, b.f) && local_rows_ok(dq, b.dqs, b.f) &&
         local_keys_ok(dk, b.dks, b.f) && local_keys_ok(dv, b.dvs, b.f);
}

int launch_local_bwd_tc(void* dq, void* dk, void* dv, const void* dout, const void* q, const void* k, const void* v,
                        const void* out, const float* lse, float* row_scratch, const LocalBwdArgs& b, int dtype,
                        cudaStream_t st) {
  const LocalArgs& a = b.f;
  CUtensorMap mq, md, mk, mv;
  if (!local_map_rows(&mq, q, a.qs, a, "q") || !local_map_rows(&md, dout, b.dos, a, "dout") ||
      !local_map_keys(&mk, k, a.ks, a, TILE, "k") || !local_map_keys(&mv, v, a.vs, a, TILE, "v"))
    return TB200_ERR_UNSUPPORTED;
  const int64_t rows = local_tc_rows(a);
  BwdParams p;
  p.b = b;
  p.dq = dq;
  p.dk = dk;
  p.dv = dv;
  p.nlse2 = row_scratch;
  p.ndelta = row_scratch + rows;
  p.scale_log2 = a.scale * LOG2E;
  p.tile_tokens = TILE / a.G;
  p.query_tiles = (int)ceil_div(a.tokens, p.tile_tokens);
  p.key_tiles = (int)ceil_div(a.tokens, TILE);
  p.status = device_status_ptr();
  auto go = [&](auto tag, auto dsel) -> int {
    using T = decltype(tag);
    constexpr int D = decltype(dsel)::value;
    constexpr int DKV_SMEM = 6 * TILE * D * 2 + 2048 + 256 + 1024, DQ_SMEM = 6 * TILE * D * 2 + 256 + 1024;
    static_assert(DKV_SMEM <= 227 * 1024, "shared memory of one CTA");
    auto kkv = local_dkv_tc_kernel<T, D>;
    auto kq = local_dq_tc_kernel<T, D>;
    static std::atomic<unsigned long long> done_kv{0}, done_q{0};
    if (int rc = optin(kkv, DKV_SMEM, done_kv)) return rc;
    if (int rc = optin(kq, DQ_SMEM, done_q)) return rc;
    local_bwd_prep<T, D><<<(unsigned)ceil_div(rows, 256 / (D / 8)), 256, 0, st>>>(
        row_scratch, row_scratch + rows, (const T*)out, (const T*)dout, lse, b, p.tile_tokens, p.query_tiles);
    if (int rc = launch_status("local_bwd_prep")) return rc;
    kkv<<<dim3((unsigned)(p.key_tiles + b.sink_tiles * b.far), (unsigned)a.KV, (unsigned)a.n), THREADS, DKV_SMEM, st>>>(mq, md, mk, mv, p);
    if (int rc = launch_status("local_dkv_tc")) return rc;
    kq<<<dim3((unsigned)p.query_tiles, (unsigned)a.KV, (unsigned)a.n), THREADS, DQ_SMEM, st>>>(mq, md, mk, mv, p);
    return launch_status("local_dq_tc");
  };
  using D64 = std::integral_constant<int, 64>;
  using D128 = std::integral_constant<int, 128>;
  if (dtype == TB200_BF16) return a.D == 128 ? go(__nv_bfloat16{}, D128{}) : go(__nv_bfloat16{}, D64{});
  return a.D == 128 ? go(__half{}, D128{}) : go(__half{}, D64{});
}

}  // namespace tb200
