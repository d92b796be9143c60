// Attention of few query rows (up to 16 of one sequence and key head: single tokens of a group of heads) over
// the pages of a cache, for 16-bit operands with head size 64 or 128.
//
// Everything transposed, so that 128 keys lie on the tensor-memory lanes and the query rows in N = 16 columns:
// a tile of keys is then worked on by 128 threads with 16 scores each, where a tile with the rows on the lanes
// would leave all but 16 of them idle, one thread with 128 exponentials in a row.
//
//   S^T = K Q^T        [keys][rows], two buffers
//   P^T = exp2(S^T scale log2e - m), 16-bit, to shared memory as [row][key] (operand, 128-byte swizzle)
//   O^T += V^T P^T     [features][rows]  (at D = 64 lanes 64-127 compute on what follows the tile in shared
//                      memory, and are not read)
//
// The maximum m of a row is common to all 128 threads; it moves only when a score is more than 8 (log2
// units) above it, which a barrier with a vote finds out: a step costs one barrier, and the shuffles of a
// row maximum only when it moves. Row sums are kept per thread and added at the end.
//
//   warp 0      producer: one ring of three (D = 64: five) tiles, K and V in turn; one lane per piece of a page
//   warp 1      MMA issuer, tensor-memory allocation
//   warps 2-5   softmax: lane = key
// Two CTAs an SM: the start and end of one walk overlap the other's loads. Bound by HBM: 64 single tokens of 8 x 4
// heads over contexts of 512 to 8192, D = 128 (1.14 GB), 200 us and 5 for joining the parts, 5.7 TB/s. The products
// read each key and value once from shared memory, 512 cycles a tile, the pipe is 5 % busy.
#include <type_traits>

#include "attn_math.cuh"
#include "local_attention_tc.cuh"
#include "ptx.cuh"

namespace tb200 {
namespace {

constexpr int TILE = LOCAL_TC_TILE;
constexpr int N = LOCAL_FEW_ROWS;
constexpr int THREADS = 192;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;
constexpr float RESCALE_THRESHOLD = 8.f;

struct FewParams {
  LocalArgs a;
  void* out;
  float scale_log2;
  int piece;  // rows of one copy of keys
  WaitTest test;
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
__device__ inline uint32_t low_bits(int n) { return n <= 0 ? 0u : (n >= 32 ? 0xffffffffu : (1u << n) - 1u); }
__device__ inline int saturate(int64_t v) { return v < -(1 << 20) ? -(1 << 20) : (v > (1 << 20) ? (1 << 20) : (int)v); }
// barrier of the 128 softmax threads with the disjunction of their votes
__device__ inline bool vote128(bool mine) {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, 1, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
               : "=r"(r)
               : "r"(mine ? 1u : 0u)
               : "memory");
  return r != 0;
}
__device__ inline void sync128() { asm volatile("barrier.cta.sync 1, 128;" ::: "memory"); }

template <typename T, int D>
__global__ void __launch_bounds__(THREADS, 2)
    local_few_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                        const __grid_constant__ CUtensorMap map_v, const FewParams p) {
  constexpr int STAGES = D == 128 ? 3 : 5;  // tiles of the ring
  constexpr int TILE_BYTES = TILE * D * 2, NBOX = D / 64, BOX_BYTES = TILE * 128;
  constexpr int Q_BYTES = N * D * 2, P_BYTES = N * TILE * 2;
  constexpr bool IS_BF16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr uint32_t IDESC_S = ptx::make_idesc(IS_BF16, false, false, TILE, N);  // K-major x K-major
  constexpr uint32_t IDESC_O = ptx::make_idesc(IS_BF16, true, false, TILE, N);   // V^T along the features, P^T K-major
  constexpr uint32_t TMEM_COLS = 64;
  constexpr uint32_t COL_S = 0, COL_O = 2 * N;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* ring = smem;                                // [STAGES]
  uint8_t* p_smem = ring + STAGES * TILE_BYTES;        // [2] (at D = 64 the products of the last stage read on into
  uint8_t* q_smem = p_smem + 2 * P_BYTES;              //  what follows the ring, TILE_BYTES of which are allocated)
  float* m_smem = reinterpret_cast<float*>(q_smem + Q_BYTES);  // [N] running maximum of the rows
  float* w_smem = m_smem + N;                                  // [4][N] of the four warps
  uint64_t* bars = reinterpret_cast<uint64_t*>(w_smem + 4 * N);
  uint64_t* full = bars;                 // [STAGES]
  uint64_t* empty = bars + STAGES;       // [STAGES]
  uint64_t* q_full = bars + 2 * STAGES;
  uint64_t* s_full = q_full + 1;         // [2] S^T(i) computed, by buffer
  uint64_t* o_done = q_full + 3;         // [2] O^T += V^T P^T(i) done, by buffer
  uint64_t* s_free = q_full + 5;         // [2] S^T(i) read     (128 arrivals)
  uint64_t* p_full = q_full + 7;         // [2] P^T(i) written  (128 arrivals)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(q_full + 9);
  volatile uint32_t* abort_flag = tmem_slot + 1;

  const LocalArgs& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = blockIdx.x, hk = blockIdx.y, s = blockIdx.z;
  const Sequence seq = load_sequence(a, s);
  if (a.zero_rest && hk == 0) zero_rest_of(reinterpret_cast<T*>(p.out), a, s, seq, split, gridDim.x);
  if (seq.q_len == 0) return;
  const int base = seq.base;
  const int rows = min(seq.q_len, N / a.G) * a.G;
  const KeyRange kr = key_range(a, base, base + seq.q_len - 1, seq.kv_len, TILE);
  int m0, m1;
  split_range(a, kr.count, split, &m0, &m1);
  if (split > 0 && m0 >= m1) return;
  const int steps = m1 - m0;
  const bool whole = a.split_tiles == 0 || kr.count <= a.split_tiles;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2 * STAGES + 5; ++i) ptx::mbar_init(&bars[i], 1);
    for (int i = 0; i < 4; ++i) ptx::mbar_init(s_free + i, 128);
    abort_flag[0] = 0;
    abort_flag[1] = p.test.units;
    ptx::fence_barrier_init();
    ptx::prefetch_tensormap(&map_q);
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
    // ---------------------------------------------------------------- producer (whole warp)
    const int pieces = TILE / p.piece, from = first_key(a, max(base, 0));
    auto locate = [&](int j, int* page, int* row) {  // of this lane's piece (index `pages`: zeros)
      const int p0 = j * TILE + lane * p.piece;
      int id = -1;
      if (lane < pieces && p0 < seq.kv_len && (p0 + p.piece > from || p0 < a.sinks))
        id = a.table[s * a.table_stride + p0 / a.page];
      *page = id < 0 || id >= a.pages ? a.pages : id;
      *row = p0 % a.page;
    };
    int page = 0, row = 0;
    if (steps > 0) {
      locate(kr.tile(m0), &page, &row);
      if (lane == 0) {
        ptx::mbar_expect_tx(q_full, NBOX * (N / a.G) * a.G * 128);
#pragma unroll
        for (int c = 0; c < NBOX; ++c)
          tma_load_5d(q_smem + c * (N * 128), &map_q, q_full, c * 64, 0, seq.q_begin, hk, 0);
      }
    }
    int brought = 0;    // tiles
    bool stop = false;  // a wait has run out: nothing more is brought
    for (int i = 0; i < steps && !stop; ++i) {
      int next_page = 0, next_row = 0;
      if (i + 1 < steps) locate(kr.tile(m0 + i + 1), &next_page, &next_row);
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        const int g = 2 * i + kv, st = g % STAGES;
        if (stop) continue;
        if (lane == 0) ptx::mbar_wait(&empty[st], ((g / STAGES) & 1) ^ 1, abort_flag, a.status, 141);
        stop = __shfl_sync(0xffffffffu, lane == 0 ? abort_flag[0] : 0u, 0) != 0;
        if (stop) continue;
        brought = g + 1;
        const bool left_out = g == p.test.skip && blockIdx.x + blockIdx.y + blockIdx.z == 0;  // (test hook)
        if (lane == 0 && !left_out) ptx::mbar_expect_tx(&full[st], TILE_BYTES);
        __syncwarp();
        if (lane < pieces && !left_out) {
#pragma unroll
          for (int c = 0; c < NBOX; ++c)
            tma_load_4d(ring + st * TILE_BYTES + c * BOX_BYTES + lane * p.piece * 128, kv ? &map_v : &map_k, &full[st], c * 64, row,
                        hk, page);
        }
      }
      page = next_page;
      row = next_row;
    }
    // every copy has landed before the CTA gives up its shared memory
    if (lane == 0 && steps > 0) {
      ptx::mbar_wait_drain(q_full, 0, abort_flag, a.status, 142);
      for (int g = brought > STAGES ? brought - STAGES : 0; g < brought; ++g)
        ptx::mbar_wait_drain(&full[g % STAGES], (g / STAGES) & 1, abort_flag, a.status, 142);
    }
    __syncwarp();
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMA issuer (whole warp; one lane issues)
    const bool elected = ptx::elect_one();
    auto wait_ = [&](uint64_t* bar, uint32_t parity, int code) {
      ptx::mbar_wait(bar, parity, abort_flag, a.status, code);
      __syncwarp();
    };
    auto commit_ = [&](uint64_t* bar) {
      if (elected) ptx::umma_commit(bar);
    };
    const uint64_t dk = ptx::make_smem_desc(ptx::smem_u32(ring), 16, 1024);
    const uint64_t dv = ptx::make_smem_desc(ptx::smem_u32(ring), BOX_BYTES, 1024);  // along the features
    const uint64_t dq = ptx::make_smem_desc(ptx::smem_u32(q_smem), 16, 1024);
    const uint64_t dp = ptx::make_smem_desc(ptx::smem_u32(p_smem), 16, 1024);
    constexpr uint64_t STAGE = static_cast<uint64_t>(TILE_BYTES >> 4);
    auto scores_of = [&](int i) {
      const int g = 2 * i, st = g % STAGES;
      if (i >= 2) wait_(&s_free[i & 1], ((i - 2) >> 1) & 1, 143);
      wait_(&full[st], (g / STAGES) & 1, 144);
      ptx::tc_fence_after();
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        const uint64_t oa = static_cast<uint64_t>(((ks >> 2) * BOX_BYTES + (ks & 3) * 32) >> 4);
        const uint64_t ob = static_cast<uint64_t>(((ks >> 2) * (N * 128) + (ks & 3) * 32) >> 4);
        if (elected) ptx::umma_ss(tmem_base + COL_S + (i & 1) * N, dk + st * STAGE + oa, dq + ob, IDESC_S, ks != 0);
      }
      commit_(&s_full[i & 1]);
      commit_(&empty[st]);
    };
    if (steps > 0) {
      wait_(q_full, 0, 145);
      scores_of(0);
      for (int i = 0; i < steps; ++i) {
        if (i + 1 < steps) scores_of(i + 1);
        const int g = 2 * i + 1, st = g % STAGES;
        wait_(&p_full[i & 1], (i >> 1) & 1, 146);
        wait_(&full[st], (g / STAGES) & 1, 147);
        ptx::tc_fence_after();
#pragma unroll
        for (int ks = 0; ks < TILE / 16; ++ks) {
          const uint64_t ob = static_cast<uint64_t>(((ks >> 2) * (N * 128) + (ks & 3) * 32) >> 4);
          if (elected)
            ptx::umma_ss(tmem_base + COL_O, dv + st * STAGE + static_cast<uint64_t>((ks * 2048) >> 4),
                         dp + (i & 1) * static_cast<uint64_t>(P_BYTES >> 4) + ob, IDESC_O, (i | ks) != 0);
        }
        commit_(&o_done[i & 1]);
        commit_(&empty[st]);
      }
      // everything issued has completed before tensor memory is freed
      ptx::mbar_wait_drain(&o_done[(steps - 1) & 1], ((steps - 1) >> 1) & 1, abort_flag, a.status, 148);
    }
    __syncwarp();
  } else {
    // ---------------------------------------------------------------- softmax: lane = key
    const int quarter = warp & 3, r = quarter * 32 + lane;  // (tensor-memory lanes of the warp)
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const int wid = warp - 2, tid = threadIdx.x - 64;
    if (tid < N) m_smem[tid] = -INFINITY;
    sync128();
    float l[N];  // this thread's part of the rows' sums
#pragma unroll
    for (int n = 0; n < N; ++n) l[n] = 0.f;
    uint8_t* p_at = p_smem + (r >> 6) * (N * 128) + (r & 7) * 2;
    const int p_chunk = (r & 63) >> 3;
    const int pos0 = base;  // position of row 0's token
    for (int i = 0; i < steps; ++i) {
      const int j0 = kr.tile(m0 + i) * TILE, j = j0 + r;
      uint32_t sv[N];
      ptx::mbar_wait(&s_full[i & 1], (i >> 1) & 1, abort_flag, a.status, 149);
      ptx::tc_fence_after();
      ptx::tmem_ld16(tmem_base + lane_off + COL_S + (i & 1) * N, sv);
      am::tmem_ld_wait_dep(sv);
      ptx::tc_fence_before();
      ptx::mbar_arrive(&s_free[i & 1]);
      // rows that see this key: from `low` on they are not before it, below `high` within the window
      uint32_t seen;
      {
        const int low = saturate((int64_t)(j - pos0) * a.G), high = saturate(((int64_t)j - pos0 + a.window) * a.G);
        const uint32_t sink = j < a.sinks ? 0xffffffffu : 0u, exists = j < seq.kv_len ? 0xffffffffu : 0u;
        seen = exists & low_bits(rows) & ~low_bits(low) & (low_bits(high) | sink);
      }
      float x[N];
      bool above = false;
#pragma unroll
      for (int n = 0; n < N; ++n) {
        x[n] = (seen >> n) & 1u ? __uint_as_float(sv[n]) * p.scale_log2 : -INFINITY;
        above = above || x[n] > m_smem[n] + RESCALE_THRESHOLD;
      }
      if (vote128(above)) {  // the maxima move
        float mine[N];
#pragma unroll
        for (int n = 0; n < N; ++n) mine[n] = warp_max(x[n]);
        if (lane == 0) {
#pragma unroll
          for (int n = 0; n < N; ++n) w_smem[wid * N + n] = mine[n];
        }
        if (i > 0) {
          ptx::mbar_wait(&o_done[(i - 1) & 1], ((i - 1) >> 1) & 1, abort_flag, a.status, 150);
          ptx::tc_fence_after();
        }
        sync128();
        float f[N];
#pragma unroll
        for (int n = 0; n < N; ++n) {
          const float was = m_smem[n];
          const float now = fmaxf(fmaxf(fmaxf(w_smem[n], w_smem[N + n]), fmaxf(w_smem[2 * N + n], w_smem[3 * N + n])), was);
          f[n] = now == -INFINITY ? 1.f : exp2f(was - now);
          l[n] *= f[n];
          mine[n] = now;
        }
        if (i > 0) {
          uint32_t o[N];
          ptx::tmem_ld16(tmem_base + lane_off + COL_O, o);
          am::tmem_ld_wait_dep(o);
#pragma unroll
          for (int n = 0; n < N; ++n) o[n] = __float_as_uint(__uint_as_float(o[n]) * f[n]);
          ptx::tmem_st16(tmem_base + lane_off + COL_O, o);
          ptx::tmem_st_wait();
          ptx::tc_fence_before();
        }
        sync128();  // (all have read the old maxima)
#pragma unroll
        for (int n = 0; n < N; ++n)
          if (tid == n) m_smem[n] = mine[n];
        sync128();
      }
      // P^T(i) goes over P^T(i-2)
      if (i >= 2) ptx::mbar_wait(&o_done[i & 1], ((i - 2) >> 1) & 1, abort_flag, a.status, 151);
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const float m = m_smem[n];
        const float e = am::ex2(x[n] - (m == -INFINITY ? 0.f : m));
        l[n] += e;
        *reinterpret_cast<T*>(p_at + (i & 1) * P_BYTES + n * 128 + ((p_chunk ^ (n & 7)) << 4)) = Traits<T>::from_f(e);
      }
      if (j0 + TILE > seq.kv_len) {
        // rows of V behind the sequence's end hold anything (0 times that might not be 0): zeros
        const int g = 2 * i + 1, st = g % STAGES;
        ptx::mbar_wait(&full[st], (g / STAGES) & 1, abort_flag, a.status, 152);
        if (j >= seq.kv_len) {
#pragma unroll
          for (int c = 0; c < D / 8; ++c)
            *reinterpret_cast<uint4*>(ring + st * TILE_BYTES + (c >> 3) * BOX_BYTES + r * 128 + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
        }
      }
      ptx::fence_proxy_async_smem();
      ptx::mbar_arrive(&p_full[i & 1]);
    }
    // row sums over the keys of all threads
#pragma unroll
    for (int n = 0; n < N; ++n) l[n] = warp_sum(l[n]);
    sync128();
    if (lane == 0) {
#pragma unroll
      for (int n = 0; n < N; ++n) w_smem[wid * N + n] = l[n];
    }
    if (steps > 0) {
      ptx::mbar_wait(&o_done[(steps - 1) & 1], ((steps - 1) >> 1) & 1, abort_flag, a.status, 153);
      ptx::tc_fence_after();
    }
    sync128();
    uint32_t o[N];
    if (steps > 0) {
      ptx::tmem_ld16(tmem_base + lane_off + COL_O, o);
      am::tmem_ld_wait_dep(o);
    }
    // lane = feature
    if (r < D) {
#pragma unroll
      for (int n = 0; n < N; ++n) {
        if (n >= rows) continue;
        const float sum = w_smem[n] + w_smem[N + n] + w_smem[2 * N + n] + w_smem[3 * N + n];
        const float inv = sum > 0.f ? 1.f / sum : 0.f;  // a row without keys: zeros
        const float value = sum > 0.f ? __uint_as_float(o[n]) * inv : 0.f;
        const int head = hk * a.G + n % a.G;
        const int64_t token = seq.q_begin + n / a.G;
        if (whole) {
          reinterpret_cast<T*>(p.out)[token * a.os[2] + head * a.os[1] + r] = Traits<T>::from_f(value);
        } else {
          const int64_t row = ((int64_t)split * a.tokens + token) * a.H + head;
          a.part_out[row * D + r] = value;
          if (r == 0) a.part_lse[row] = sum > 0.f ? m_smem[n] * LN2 + logf(sum) : -INFINITY;
        }
      }
    }
  }
  ptx::tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

template <typename T, int D>
int launch_few(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const FewParams& p, cudaStream_t st) {
  constexpr int RING = (D == 128 ? 3 : 5) * TILE * D * 2;
  constexpr int REST = 2 * N * TILE * 2 + N * D * 2 + 5 * N * 4 + 256;
  // (at D = 64 a product on the last stage reads one tile beyond the ring)
  constexpr int SMEM = RING + (D == 64 && REST < TILE * D * 2 ? TILE * D * 2 : REST) + 1024;
  static_assert(SMEM <= 227 * 1024, "shared memory of one CTA");
  auto kern = local_few_tc_kernel<T, D>;
  static std::atomic<unsigned long long> done{0};
  const cudaError_t e = smem_optin_per_device(done, reinterpret_cast<const void*>(kern), SMEM);
  if (e != cudaSuccess) {
    set_error("local_few_tc: cudaFuncSetAttribute failed: %s", cudaGetErrorString(e));
    return (int)e;
  }
  kern<<<dim3((unsigned)p.a.splits, (unsigned)p.a.KV, (unsigned)p.a.n), THREADS, SMEM, st>>>(mq, mk, mv, p);
  return launch_status("local_few_tc");
}

}  // namespace

int launch_local_few_tc(void* out, const void* q, const void* k, const void* v, const LocalArgs& a, int dtype,
                        cudaStream_t st) {
  FewParams p;
  p.a = a;
  p.a.status = device_status_ptr();
  p.out = out;
  p.scale_log2 = a.scale * LOG2E;
  p.piece = local_piece(a);
  p.test = WaitTest::of_this_thread(1, 2);
  CUtensorMap mq, mk, mv;
  bind_primary_context();
  if (!local_map_rows(&mq, q, a.qs, a, N / a.G, "q") || !local_map_keys(&mk, k, a.ks, a, p.piece, "k") ||
      !local_map_keys(&mv, v, a.vs, a, p.piece, "v"))
    return TB200_ERR_UNSUPPORTED;
  auto go = [&](auto tag, auto dsel) -> int {
    using T = decltype(tag);
    constexpr int D = decltype(dsel)::value;
    return launch_few<T, D>(mq, mk, mv, p, st);
  };
  using D64 = std::integral_constant<int, 64>;
  using D128 = std::integral_constant<int, 128>;
  if (dtype == TB200_BF16) return a.D == 128 ? go(__nv_bfloat16{}, D128{}) : go(__nv_bfloat16{}, D64{});
  return a.D == 128 ? go(__half{}, D128{}) : go(__half{}, D64{});
}

}  // namespace tb200
