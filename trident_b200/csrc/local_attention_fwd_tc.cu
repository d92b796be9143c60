// tcgen05 forward of local attention (window and sinks), training and serving form, for 16-bit operands
// with head size 64 or 128.
//
// A unit of work is two adjacent tiles of 128 packed query rows (token * G + head of the group) of one sequence
// and key head, along the key tiles that any of them sees (KeyRange), or one part of that walk. A persistent
// CTA takes every gridDim-th unit: the next unit's queries, keys and first scores are under way while the
// last one's output is written (a CTA per unit spent 9500 of 51000 cycles on its start and end at a window
// of 1024). Both score tiles and both output accumulators live in tensor memory (S0, S1: 128 fp32 columns each;
// O0, O1: D columns each), so the tensor pipe works on one query tile while the softmax warps work on the
// other; a key tile that only one of the two sees is walked by that one alone.
//
//   warp 0      producer: Q0, Q1 of a unit, rings of two K and two V tiles. A tile of keys is 128 rows of a
//               sequence (training), or 128 / R pieces of R rows, R the largest divisor of the page size
//               and of 128: one lane per piece looks its page up and issues its copies. Pieces that no row
//               sees, or whose page is outside the pool, are read at a page index past the end: zeros.
//   warp 1      MMA issuer: S_t = Q_t K^T, O_t += P_t V (P_t from tensor memory, in two parts: the product
//               starts when three quarters of P_t are there)
//   warp 2      tensor-memory allocation; issues the bulk copies of output tiles
//   warp 3      looks the walks of coming units up for the MMA issuer; serving form: zeroes the rows of the last
//               V tile behind the sequence's end (a probability of 0 times what an unused row holds, which may
//               be NaN, would not be 0)
//   warps 4-7   softmax of query tile 0, warps 8-11 of tile 1: one thread per row; scores stay in registers
//               between maximum and exponentials. Warps without a row of the sequence only pass the
//               barriers (a single new token is G rows of one tile). Output tiles leave through shared memory
//               and bulk copies (by the threads themselves where a tile is not full or the walk is cut).
//
// Masks by blocks of 32 columns and warps of 32 rows: a block that no row of the warp sees costs nothing, one
// that all rows see no mask, the others a 32-bit mask per row. The running maximum used in the exponent moves
// only when the true one has moved by more than 8 (log2 units): the final division by the row sum undoes it
// exactly. The row sum adds the fp32 probabilities; P is rounded to 16 bits for the product with V, as the
// tensor cores take it.
//
// Bound, by size of the problem: HBM for single tokens, for chunks and training the chain of each of the two
// tiles. At D = 128 a step of it takes 3700 cycles: 800 from the issue of the scores (operands in shared memory:
// 94 cycles an instruction instead of 64) to the threads that read them, 800 to the maximum, 1500 for the
// exponentials (1024 of them the tile's share of the exponential unit), 600 until the next scores are issued behind
// P V on the in-order pipe; the other tile's step runs beside it. 2 x 32 heads x 4096 x 128 bf16, window 1024, 8 key
// heads: 169 us (713 TFLOP/s), tensor pipe 45 % busy; 4 chunks of up to 512 tokens over contexts to 16384: 55 us.
#include <mutex>
#include <type_traits>

#include "attn_math.cuh"
#include "local_attention_tc.cuh"
#include "ptx.cuh"

namespace tb200 {
namespace {

constexpr int TILE = LOCAL_TC_TILE;
constexpr int FWD_THREADS = 384;
// (launch registers x threads is the pool that setmaxnreg.inc draws on; checked below and by the host)
constexpr int REGS_LAUNCH = 168, REGS_SERVICE = 72, REGS_SOFTMAX = 216;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;
constexpr float RESCALE_THRESHOLD = 8.f;
constexpr int64_t MOST_UNITS = (1ll << 31) - (1 << 20);

struct FwdParams {
  LocalArgs a;
  void* out;
  float* lse;
  float scale_log2;
  int tile_tokens;  // tokens of a query tile
  int piece;        // R: rows of one copy of keys
  int pairs, units; // pairs of query tiles per sequence and key head; pairs * KV * sequences * parts
  Divisor outer, kv, splits;  // of a unit's number (unit_at)
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
// the lowest n bits
__device__ inline uint32_t low_bits(int n) { return n <= 0 ? 0u : (n >= 32 ? 0xffffffffu : (1u << n) - 1u); }

// P of a whole row of 128 raw scores: p = 2^(v scale - m), 16-bit, to tensor memory; returns the row's sum.
// One warp of a query tile is alone on its scheduler's exponential unit, which takes an instruction every 8
// cycles; the arguments, sums and conversions of neighbouring columns are issued in between (as three passes
// over blocks of 32 columns, one after the other, a row took 1870 cycles instead of the 1024 of its
// exponentials). `part` is called once the first 96 columns have been stored.
template <typename T, typename Part>
__device__ inline float exp_row(const uint32_t (&v)[4][32], uint64_t scale2, uint64_t negm2, uint32_t p_addr, Part part) {
  constexpr int LAG = 3;  // pairs between an exponential and its use
  uint64_t sum0 = am::pack2f(0.f, 0.f), sum1 = sum0;
  float x[128];
  uint32_t packed[16];
  am::unpack2f(am::fma2_ordered(am::pack2u(v[0][0], v[0][1]), scale2, negm2), x[0], x[1]);
#pragma unroll
  for (int k = 0; k < 64 + LAG; ++k) {
    if (k < 64) x[2 * k] = am::ex2_ordered(x[2 * k]);
    if (k + 1 < 64)
      am::unpack2f(am::fma2_ordered(am::pack2u(v[(k + 1) >> 4][(2 * k + 2) & 31], v[(k + 1) >> 4][(2 * k + 3) & 31]), scale2, negm2),
                   x[2 * k + 2], x[2 * k + 3]);
    if (k < 64) x[2 * k + 1] = am::ex2_ordered(x[2 * k + 1]);
    if (k >= LAG) {
      const int d = k - LAG;
      if (d & 1) sum1 = am::add2_ordered(sum1, am::pack2f(x[2 * d], x[2 * d + 1]));
      else sum0 = am::add2_ordered(sum0, am::pack2f(x[2 * d], x[2 * d + 1]));
      packed[d & 15] = am::cvt_ordered<T>(x[2 * d], x[2 * d + 1]);
      if ((d & 15) == 15) ptx::tmem_st16(p_addr + (d >> 4) * 16, packed);
      if (d == 47 + 6) part();  // (the stores have had the time of six pairs)
    }
  }
  float s0, s1;
  am::unpack2f(am::add2(sum0, sum1), s0, s1);
  return s0 + s1;
}

// Until `count` output tiles have been read from shared memory (a bounded wait, as ptx::mbar_wait).
__device__ inline void wait_copied(const uint32_t* copied, int count, volatile uint32_t* abort_flag, int* status) {
  const long long start = clock64();
  for (uint32_t polls = 1;; ++polls) {
    uint32_t now;
    asm volatile("ld.acquire.cta.shared::cta.u32 %0, [%1];" : "=r"(now) : "r"(ptx::smem_u32(copied)) : "memory");
    if ((int)now >= count) return;
    if ((polls & 1023u) == 0) {
      if (abort_flag[0]) return;
      if (clock64() - start > (static_cast<long long>(abort_flag[1]) << 16)) {
        abort_flag[0] = 1;
        if (status) atomicCAS(status, 0, 86);
        return;
      }
    }
  }
}

// A unit of work, as all roles of the CTA see it.
struct Unit {
  int s, hk, split, t0;   // t0: first token (within the sequence) of query tile 0
  Sequence seq;
  int base;               // position of the sequence's first new token
  KeyRange kr;
  int m0, m1;             // steps of the walk
  bool whole;
  int st_tiles, lo0, lo1, hi0, hi1;
  // whether query tile t takes part in key tile j: tiles below st_tiles (sinks) or from lo on, up to hi
  __device__ bool active(int t, int j) const { return (j < st_tiles || j >= (t ? lo1 : lo0)) && j <= (t ? hi1 : hi0); }
};
// What the MMA issuer needs of one (steps = 0: there are no more). Warp 3 looks it up ahead and hands it over in
// shared memory: code that runs once per unit is fetched at 5 cycles an instruction, which between one unit's last
// values and the next one's first scores was 3000 cycles without a product.
struct Walk {
  int steps, sink_tiles, skipped, first;  // key tile of step i: first + i, from step sink_tiles on `skipped` further
  int st_tiles, lo0, lo1, hi0, hi1;
  int last0, last1;  // last step of each query tile: its queries are not needed after that (-1: takes no part)
  __device__ int tile(int i) const { return first + i + (first + i < sink_tiles ? 0 : skipped); }
  __device__ bool active(int t, int j) const { return (j < st_tiles || j >= (t ? lo1 : lo0)) && j <= (t ? hi1 : hi0); }
};
// false: nothing to do
template <bool PAGED>
__device__ inline bool unit_at(const FwdParams& p, int unit, Unit* w) {
  const LocalArgs& a = p.a;
  int pair;
  if (PAGED && a.before) {
    const int tile = p.kv.quotient(unit);
    w->hk = unit - tile * a.KV;
    w->split = 0;
    listed_tile(a, tile, &w->s, &pair);
  } else {
    const int high = p.outer.quotient(unit), rest = unit - high * (int)p.outer.d;
    // Walks of a training step grow with the tile up to the window: longest first (3 sequences of 1111 tokens, 2 key
    // heads: 18.8 us by sequence and head, 17.1 so; 2 of 4096, 8 key heads: 169 and 170). Those of chunks hardly
    // grow, and their last tiles may be empty.
    pair = PAGED ? high : p.pairs - 1 - high;
    const int sequence_part = p.kv.quotient(rest);
    w->hk = rest - sequence_part * a.KV;
    w->s = p.splits.quotient(sequence_part);
    w->split = sequence_part - w->s * a.splits;
  }
  w->seq = load_sequence(a, w->s);
  w->t0 = pair * 2 * p.tile_tokens;
  if (w->t0 >= w->seq.q_len) return false;
  w->base = w->seq.base;
  const int last_token = min(w->t0 + 2 * p.tile_tokens, w->seq.q_len) - 1;
  w->kr = key_range(a, w->base + w->t0, w->base + last_token, w->seq.kv_len, TILE);
  split_range(a, w->kr.count, w->split, &w->m0, &w->m1);
  if (w->split > 0 && w->m0 >= w->m1) return false;
  w->whole = a.split_tiles == 0 || w->kr.count <= a.split_tiles;
  w->st_tiles = a.window != NO_WINDOW && a.sinks > 0 ? (a.sinks + TILE - 1) / TILE : 0;
  auto lowest = [&](int t) { return first_key(a, max(w->base + w->t0 + t * p.tile_tokens, 0)) / TILE; };
  auto highest = [&](int t) {
    const int first = w->t0 + t * p.tile_tokens, last = min(first + p.tile_tokens, w->seq.q_len) - 1;
    return first <= last && w->base + last >= 0 ? (w->base + last) / TILE : -1;
  };
  w->lo0 = lowest(0);
  w->lo1 = lowest(1);
  w->hi0 = highest(0);
  w->hi1 = highest(1);
  return true;
}

// LOW: also writes what the rounding of the output leaves (training form), by the threads themselves: 179 us instead of
// 167 at 2 x 32 heads x 4096 x 128, window 1024, 87 instead of 74 at a window of 128.
template <typename T, int D, bool PAGED, bool LOW>
__global__ void __launch_bounds__(FWD_THREADS, 1)
    local_fwd_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                        const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_out,
                        const FwdParams p) {
  constexpr int TILE_BYTES = TILE * D * 2;
  constexpr int NBOX = D / 64;
  constexpr int BOX_BYTES = TILE * 64 * 2;
  constexpr bool IS_BF16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr uint32_t IDESC_QK = ptx::make_idesc(IS_BF16, false, false, TILE, TILE);
  constexpr uint32_t IDESC_PV = ptx::make_idesc(IS_BF16, false, true, TILE, D);
  constexpr uint32_t TMEM_COLS = 512;
  constexpr uint32_t COL_S = 0, COL_O = 256;
  // At D = 64 the accumulators leave 128 columns free: P gets columns of its own, and the next score
  // product is issued as soon as the softmax threads hold the current scores in registers.
  constexpr bool P_SPLIT = D == 64;
  constexpr uint32_t COL_P = 384;
  constexpr int P_FIRST = 6;  // steps of 16 keys in the first part of P V

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* q_smem = smem;                      // [2][TILE_BYTES]
  uint8_t* k_smem = smem + 2 * TILE_BYTES;     // [2][TILE_BYTES]
  uint8_t* v_smem = smem + 4 * TILE_BYTES;     // [2][TILE_BYTES]
  uint8_t* out_smem = smem + 6 * TILE_BYTES;   // an output tile on its way out
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + 7 * TILE_BYTES);
  // Hand-overs. A ring barrier completes once per step of the walks, a barrier of query tile t once per step
  // that t takes part in, or once per unit: the waiter of phase c passes parity c & 1.
  //   k/v_full    copies (complete_tx), or warp 3 after its zeroes   MMA issuer
  //   k/v_empty   tcgen05.commit after the last product that reads   producer
  //   q_full[t]   copies, per unit in which t takes part             MMA issuer
  //   q_empty[t]  tcgen05.commit after the unit's last Q_t K^T       producer
  //   s_full[t]   tcgen05.commit after Q_t K^T                       softmax: load of S_t
  //   s_free[t]   128 softmax threads after the load of S_t (D = 64) MMA issuer: next Q_t K^T over S_t
  //   p_part[t]   128 softmax threads, first part of P_t stored      MMA issuer: first part of P_t V
  //   p_full[t]   128 softmax threads, all of P_t stored             MMA issuer: the rest
  //   o_done[t]   tcgen05.commit after P_t V                         softmax: rescale, P_t over P_t, epilogue
  //   walk_full   warp 3, after a unit's walk is in shared memory    MMA issuer
  //   walk_empty  MMA issuer, after it has read the walk             warp 3
  //   out_full    128 softmax threads of a tile, per output tile     warp 2: bulk copy
  //   copied      (a counter) warp 2, output tiles whose copy has    softmax: next output tile into shared memory
  //               read shared memory; the tiles of all units in order, tile 0 of a unit before tile 1. (Not a
  //               barrier: a query tile waits for every other number only, and one without keys to walk gets
  //               to its next output while its last is being copied, two phases before the one it waits for.)
  // Every barrier's next completion needs all waiters of the last one to have seen that: a waiter can
  // never be two phases behind.
  uint64_t* q_full = bars;           // [2]
  uint64_t* k_full = bars + 2;       // [2]
  uint64_t* k_empty = bars + 4;      // [2]
  uint64_t* v_full = bars + 6;       // [2]
  uint64_t* v_empty = bars + 8;      // [2]
  uint64_t* s_full = bars + 10;      // [2]
  uint64_t* o_done = bars + 12;      // [2]
  uint64_t* q_empty = bars + 14;     // [2]
  uint64_t* v_raw = bars + 16;       // [2] the copies of a V tile that warp 3 completes (by stage: the
                                     // producer may be two tiles ahead, both of them such)
  uint64_t* mma_drained = bars + 18;
  uint64_t* p_full = bars + 19;      // [2]
  uint64_t* p_part = bars + 21;      // [2]
  uint64_t* s_free = bars + 23;      // [2]
  uint64_t* out_full = bars + 25;
  uint32_t* copied = reinterpret_cast<uint32_t*>(bars + 26);
  uint64_t* walk_full = bars + 27;   // [2]
  uint64_t* walk_empty = bars + 29;  // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 31);
  volatile uint32_t* abort_flag = tmem_slot + 1;  // [0] abort flag, [1] wait limit (ptx::mbar_wait)
  Walk* walks = reinterpret_cast<Walk*>(bars + 33);  // [2], behind the two words of abort_flag

  const LocalArgs& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // query tile t's output leaves through shared memory: a full tile of a walk that is not cut
  auto is_bulk = [&](const Unit& w, int t) {
    const int tokens = w.seq.q_len - (w.t0 + t * p.tile_tokens);
    return w.whole && (PAGED ? tokens >= p.tile_tokens : tokens > 0);
  };
  // the last V tile has rows behind the sequence's end that its copies do not fill with zeros
  auto needs_fix = [&](const Unit& w) {
    return PAGED && w.m1 > w.m0 && w.kr.tile(w.m1 - 1) == (w.seq.kv_len - 1) / TILE && w.seq.kv_len % p.piece != 0;
  };

  if (threadIdx.x == 0) {
    for (int i = 0; i < 19; ++i) ptx::mbar_init(&bars[i], 1);
    for (int i = 19; i < 26; ++i) ptx::mbar_init(&bars[i], 128);
    for (int i = 27; i < 31; ++i) ptx::mbar_init(&bars[i], 1);
    *copied = 0;
    abort_flag[0] = 0;
    abort_flag[1] = p.test.units;
    ptx::fence_barrier_init();
    ptx::prefetch_tensormap(&map_q);
    ptx::prefetch_tensormap(&map_k);
    ptx::prefetch_tensormap(&map_v);
    ptx::prefetch_tensormap(&map_out);
  }
  if (warp == 2) {
    ptx::tmem_alloc(tmem_slot, TMEM_COLS);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  static_assert(REGS_LAUNCH * FWD_THREADS <= 65536, "launch allocation");
  static_assert(4 * 32 * REGS_SERVICE + 8 * 32 * REGS_SOFTMAX <= REGS_LAUNCH * FWD_THREADS,
                "register pool of the CTA exceeded: setmaxnreg.inc would never return");
  int units = p.units;
  if (PAGED && a.before) {
    const int64_t listed = (int64_t)a.before[a.n] * a.KV;
    units = (int)(listed < MOST_UNITS ? listed : MOST_UNITS);
  }
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_SERVICE));
    if (warp == 0) {
      // -------------------------------------------------------------- producer (whole warp)
      const int pieces = TILE / p.piece;
      int g = 0, queries0 = 0, queries1 = 0;  // steps so far, queries brought of each tile (lane 0)
      int keys = 0;                           // K tiles: g, or one more
      uint32_t fixed = 0;                     // bit s: the last V tile of stage s is completed by warp 3; 2 + s: parity
                                              // of that completion (of v_raw)
      bool stop = false;                      // a wait has run out: nothing more is brought
      auto stopped = [&]() { return __shfl_sync(0xffffffffu, lane == 0 ? abort_flag[0] : 0u, 0) != 0; };
      for (int unit = blockIdx.x; unit < units && !stop; unit += gridDim.x) {
        Unit w;
        if (!unit_at<PAGED>(p, unit, &w) || w.m1 <= w.m0) continue;
        const bool fix = needs_fix(w);
        const int from = first_key(a, max(w.base + w.t0, 0));
        // page and row of this lane's piece of key tile j (index `pages`: zeros)
        auto locate = [&](int j, int* page, int* row) {
          if constexpr (PAGED) {
            const int p0 = j * TILE + lane * p.piece;
            int id = -1;
            if (lane < pieces && p0 < w.seq.kv_len && (p0 + p.piece > from || p0 < a.sinks))
              id = a.table[w.s * a.table_stride + p0 / a.page];
            *page = id < 0 || id >= a.pages ? a.pages : id;
            *row = p0 % a.page;
          } else {
            *page = w.s;
            *row = j * TILE;
          }
        };
        int page = 0, row = 0;
        locate(w.kr.tile(w.m0), &page, &row);
        for (int m = w.m0; m < w.m1; ++m, ++g) {
          const int st = g & 1;
          const uint32_t ph = (g >> 1) & 1;
          if (lane == 0 && m == w.m0) {
            const uint32_t bytes = NBOX * p.tile_tokens * a.G * 128;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
              if ((t ? w.hi1 : w.hi0) < 0) continue;
              ptx::mbar_wait(&q_empty[t], ((t ? queries1 : queries0) & 1) ^ 1, abort_flag, a.status, 60);
              if (abort_flag[0]) break;
              ++(t ? queries1 : queries0);
              ptx::mbar_expect_tx(&q_full[t], bytes);
#pragma unroll
              for (int c = 0; c < NBOX; ++c)
                tma_load_5d(q_smem + t * TILE_BYTES + c * BOX_BYTES, &map_q, &q_full[t], c * 64, 0,
                            w.seq.q_begin + w.t0 + t * p.tile_tokens, w.hk, PAGED ? 0 : w.s);
            }
          }
          int next_page = 0, next_row = 0;  // (looked up while this step's copies wait for their stage)
          if (m + 1 < w.m1) locate(w.kr.tile(m + 1), &next_page, &next_row);
          if (lane == 0) ptx::mbar_wait(&k_empty[st], ph ^ 1, abort_flag, a.status, 61);
          if ((stop = stopped())) break;
          const bool left_out = g == p.test.skip && blockIdx.x == 0;  // (test hook)
          if (lane == 0 && !left_out) ptx::mbar_expect_tx(&k_full[st], TILE_BYTES);
          __syncwarp();
          ++keys;
          if (lane < pieces && !left_out) {
#pragma unroll
            for (int c = 0; c < NBOX; ++c)
              tma_load_4d(k_smem + st * TILE_BYTES + c * BOX_BYTES + lane * p.piece * 128, &map_k, &k_full[st], c * 64, row,
                          w.hk, page);
          }
          const bool fixed_tile = fix && m + 1 == w.m1;
          uint64_t* vbar = fixed_tile ? &v_raw[st] : &v_full[st];
          if (lane == 0) ptx::mbar_wait(&v_empty[st], ph ^ 1, abort_flag, a.status, 62);
          if ((stop = stopped())) break;
          fixed = ((fixed & ~(1u << st)) | (fixed_tile ? 1u << st : 0u)) ^ (fixed_tile ? 4u << st : 0u);
          if (lane == 0) ptx::mbar_expect_tx(vbar, TILE_BYTES);
          __syncwarp();
          if (lane < pieces) {
#pragma unroll
            for (int c = 0; c < NBOX; ++c)
              tma_load_4d(v_smem + st * TILE_BYTES + c * BOX_BYTES + lane * p.piece * 128, &map_v, vbar, c * 64, row, w.hk, page);
          }
          page = next_page;
          row = next_row;
        }
      }
      // Drain: every copy has landed before the CTA gives up its shared memory.
      if (lane == 0) {
        if (queries0 > 0) ptx::mbar_wait_drain(&q_full[0], (queries0 - 1) & 1, abort_flag, a.status, 63);
        if (queries1 > 0) ptx::mbar_wait_drain(&q_full[1], (queries1 - 1) & 1, abort_flag, a.status, 63);
        for (int i = keys > 2 ? keys - 2 : 0; i < keys; ++i)
          ptx::mbar_wait_drain(&k_full[i & 1], (i >> 1) & 1, abort_flag, a.status, 64);
        for (int i = g > 2 ? g - 2 : 0; i < g; ++i) {
          if (((fixed >> (i & 1)) & 1u)) ptx::mbar_wait_drain(&v_raw[i & 1], ((fixed >> (2 + (i & 1))) & 1u) ^ 1u, abort_flag, a.status, 65);
          else ptx::mbar_wait_drain(&v_full[i & 1], (i >> 1) & 1, abort_flag, a.status, 65);
        }
      }
      __syncwarp();
    } else if (warp == 1) {
      // -------------------------------------------------------------- MMA issuer
      // The whole warp walks the loop and waits; one elected lane issues. (With the waits in the elected lane
      // alone, a commit was seen to take effect only after that lane's next wait had given up.)
      const bool elected = ptx::elect_one();
      auto wait_ = [&](uint64_t* bar, uint32_t parity, int code) {
        ptx::mbar_wait(bar, parity, abort_flag, a.status, code);
        __syncwarp();
      };
      auto commit_ = [&](uint64_t* bar) {
        if (elected) ptx::umma_commit(bar);
      };
      const uint64_t dq0 = ptx::make_smem_desc(ptx::smem_u32(q_smem), 16, 1024);
      const uint64_t dk0 = ptx::make_smem_desc(ptx::smem_u32(k_smem), 16, 1024);
      const uint64_t dv0 = ptx::make_smem_desc(ptx::smem_u32(v_smem), BOX_BYTES, 1024);
      constexpr uint64_t NEXT_TILE = static_cast<uint64_t>(TILE_BYTES >> 4);
      // Counts of each query tile over all units: score products, value products, units with queries.
      int scores0 = 0, scores1 = 0, values0 = 0, values1 = 0, queries0 = 0, queries1 = 0;
      auto issue_qk = [&](int t, int st) {
        const uint64_t qd = dq0 + (t ? NEXT_TILE : 0), kd = dk0 + (st ? NEXT_TILE : 0);
        const uint32_t d_tmem = tmem_base + COL_S + t * 128;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          const uint64_t off = static_cast<uint64_t>(((ks >> 2) * BOX_BYTES + (ks & 3) * 32) >> 4);
          if (elected) ptx::umma_ss(d_tmem, qd + off, kd + off, IDESC_QK, ks != 0);
        }
      };
      auto issue_pv = [&](int t, int st, int ks0, int ks1, bool accumulate) {
        const uint64_t vd = dv0 + (st ? NEXT_TILE : 0);
        const uint32_t d_tmem = tmem_base + COL_O + t * D;
        const uint32_t p_tmem = tmem_base + (P_SPLIT ? COL_P + t * 64 : COL_S + t * 128);
#pragma unroll
        for (int ks = 0; ks < TILE / 16; ++ks) {
          if (ks < ks0 || ks >= ks1) continue;
          if (elected)
            ptx::umma_ts(d_tmem, p_tmem + ks * 8, vd + static_cast<uint64_t>((ks * 2048) >> 4), IDESC_PV,
                         accumulate || ks != 0);
        }
      };
      // One walk over the steps of all units: the scores of step g next to the values of step g - 1, also
      // where g begins a new unit. The keys and values of both are waited for ahead of the probabilities: a
      // wait for a barrier that has long completed costs 150 to 250 cycles of this warp, which stood
      // between a tile's probabilities and its next scores.
      int g = 0;
      uint32_t todo = 0;  // values of step g - 1: bit t: of query tile t, bit 2 + t: the first of its unit
      auto do_values = [&](auto tag, uint32_t which) {
        constexpr int t = decltype(tag)::value;
        if (!((which >> t) & 1u)) return;
        int& values = t ? values1 : values0;
        const int st = (g - 1) & 1;
        // (a unit's first probabilities also say that the output of the one before has been read)
        wait_(&p_part[t], values & 1, 76 + t);
        ptx::tc_fence_after();
        issue_pv(t, st, 0, P_FIRST, !((which >> (2 + t)) & 1u));
        wait_(&p_full[t], values & 1, 76 + t);
        ptx::tc_fence_after();
        issue_pv(t, st, P_FIRST, TILE / 16, true);
        commit_(&o_done[t]);
        ++values;
      };
      using T0 = std::integral_constant<int, 0>;
      using T1 = std::integral_constant<int, 1>;
      for (int units = 0;; ++units) {
        wait_(&walk_full[units & 1], (units >> 1) & 1, 70);
        const Walk w = walks[units & 1];
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(&walk_empty[units & 1]);
        if (__any_sync(0xffffffffu, w.steps == 0 || abort_flag[0])) break;
        const int steps = w.steps;
        bool fresh0 = true, fresh1 = true;  // no scores of the tile yet
        for (int i = 0; i < steps; ++i, ++g) {
          const int j = w.tile(i);
          const bool active0 = w.active(0, j), active1 = w.active(1, j);
          const uint32_t old = todo;
          todo = (active0 ? (fresh0 ? 5u : 1u) : 0u) | (active1 ? (fresh1 ? 10u : 2u) : 0u);
          if (g > 0) wait_(&v_full[(g - 1) & 1], ((g - 1) >> 1) & 1, 78);
          if (i > 0) wait_(&k_full[g & 1], (g >> 1) & 1, 75);
          auto do_scores = [&](auto tag) {
            constexpr int t = decltype(tag)::value;
            if (!(t ? active1 : active0)) return;
            int& scores = t ? scores1 : scores0;
            bool& fresh = t ? fresh1 : fresh0;
            if (fresh) wait_(&q_full[t], (t ? queries1 : queries0) & 1, 71 + t);
            fresh = false;
            if (P_SPLIT && scores > 0) wait_(&s_free[t], (scores - 1) & 1, 73 + t);
            if (i == 0) wait_(&k_full[g & 1], (g >> 1) & 1, 75);
            ptx::tc_fence_after();
            issue_qk(t, g & 1);
            commit_(&s_full[t]);
            if (i == (t ? w.last1 : w.last0)) commit_(&q_empty[t]);
            ++scores;
          };
          if constexpr (P_SPLIT) {
            // next scores of a tile before its values
            do_scores(T0{});
            do_values(T0{}, old);
            do_scores(T1{});
            commit_(&k_empty[g & 1]);
            do_values(T1{}, old);
            if (g > 0) commit_(&v_empty[(g - 1) & 1]);
          } else {
            // P overwrites S: the next scores follow the values on the in-order pipe
            do_values(T0{}, old);
            do_scores(T0{});
            do_values(T1{}, old);
            if (g > 0) commit_(&v_empty[(g - 1) & 1]);
            do_scores(T1{});
            commit_(&k_empty[g & 1]);
          }
        }
        // (a tile whose queries were brought, but that takes no part in this part of the walk, counts too)
        if (w.hi0 >= 0) {
          if (fresh0) {
            wait_(&q_full[0], queries0 & 1, 71);
            commit_(&q_empty[0]);
          }
          ++queries0;
        }
        if (w.hi1 >= 0) {
          if (fresh1) {
            wait_(&q_full[1], queries1 & 1, 72);
            commit_(&q_empty[1]);
          }
          ++queries1;
        }
      }
      if (g > 0) {
        wait_(&v_full[(g - 1) & 1], ((g - 1) >> 1) & 1, 78);
        do_values(T0{}, todo);
        do_values(T1{}, todo);
      }
      // everything issued has completed before tensor memory is freed
      commit_(mma_drained);
      ptx::mbar_wait_drain(mma_drained, 0, abort_flag, a.status, 79);
      __syncwarp();
    } else if (warp == 2) {
      // -------------------------------------------------------------- output tiles (one lane)
      if (lane == 0) {
        int outs = 0;
        for (int unit = blockIdx.x; unit < units; unit += gridDim.x) {
          Unit w;
          if (abort_flag[0]) break;
          if (!unit_at<PAGED>(p, unit, &w)) continue;
#pragma unroll 1
          for (int t = 0; t < 2; ++t) {
            if (!is_bulk(w, t)) continue;
            ptx::mbar_wait(out_full, outs & 1, abort_flag, a.status, 67);
#pragma unroll
            for (int c = 0; c < NBOX; ++c)
              ptx::tma_store_5d(&map_out, out_smem + c * BOX_BYTES, c * 64, 0, w.seq.q_begin + w.t0 + t * p.tile_tokens, w.hk,
                                PAGED ? 0 : w.s);
            ptx::bulk_commit();
            ptx::bulk_wait_read();
            ++outs;
            asm volatile("st.release.cta.shared::cta.u32 [%0], %1;" ::"r"(ptx::smem_u32(copied)), "r"(outs) : "memory");
          }
        }
        ptx::bulk_wait_done();
      }
      __syncwarp();
    } else if (warp == 3) {
      // -------------------------------------------------------------- walks for the issuer, zeros behind the sequence's end
      int g = 0, n = 0;     // steps, units
      uint32_t phases = 0;  // bit s: parity of the next completion of stage s
      auto publish = [&](const Walk& w) {
        ptx::mbar_wait(&walk_empty[n & 1], ((n >> 1) & 1) ^ 1, abort_flag, a.status, 68);
        if (lane == 0) {
          walks[n & 1] = w;
          ptx::mbar_arrive(&walk_full[n & 1]);
        }
        __syncwarp();
        ++n;
      };
      // the last V tile of the unit with steps up to g, when its sequence has `keys` keys
      auto fix = [&](int keys) {
        const int st = (g - 1) & 1;
        ptx::mbar_wait_drain(&v_raw[st], (phases >> st) & 1u, abort_flag, a.status, 66);
        phases ^= 1u << st;
        const int first = keys % TILE, end = min(TILE, ((first + p.piece - 1) / p.piece) * p.piece);
        // (whole pieces behind the end were read as zeros)
        for (int r = first + lane / 8; r < end; r += 4)
#pragma unroll
          for (int c = 0; c < NBOX; ++c)
            *reinterpret_cast<uint4*>(v_smem + st * TILE_BYTES + c * BOX_BYTES + r * 128 + (lane & 7) * 16) = make_uint4(0, 0, 0, 0);
        ptx::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(&v_full[st]);
      };
      int fix_keys = 0;  // of the unit before
      for (int unit = blockIdx.x; unit < units; unit += gridDim.x) {
        Unit w;
        if (__any_sync(0xffffffffu, abort_flag[0] != 0)) break;
        if (!unit_at<PAGED>(p, unit, &w) || w.m1 <= w.m0) continue;
        int last0 = w.m1 - w.m0 - 1, last1 = last0;
        while (last0 >= 0 && !w.active(0, w.kr.tile(w.m0 + last0))) --last0;
        while (last1 >= 0 && !w.active(1, w.kr.tile(w.m0 + last1))) --last1;
        publish(Walk{w.m1 - w.m0, w.kr.sink_tiles, w.kr.lo - w.kr.sink_tiles, w.m0, w.st_tiles, w.lo0, w.lo1, w.hi0, w.hi1,
                     last0, last1});
        if (PAGED && fix_keys > 0) fix(fix_keys);
        g += w.m1 - w.m0;
        fix_keys = needs_fix(w) ? w.seq.kv_len : 0;
      }
      publish(Walk{});
      if (PAGED && fix_keys > 0) fix(fix_keys);
    }
  } else {
    // ---------------------------------------------------------------- softmax + epilogue
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS_SOFTMAX));
    if (PAGED && a.zero_rest) {  // (these warps have nothing else to do until the first scores are there)
      T* out = reinterpret_cast<T*>(p.out);
      const int thread = threadIdx.x - 128;
      zero_rows(out, a, 0, load_sequence(a, 0).q_begin, blockIdx.x, gridDim.x, thread, 256);
      zero_rows(out, a, load_sequence(a, a.n - 1).q_end, a.tokens, blockIdx.x, gridDim.x, thread, 256);
      if (a.max_q < a.tokens)  // a warp looks 32 sequences up, and takes the rows beyond max_q of each in turn
        for (int s0 = thread & ~31; s0 < a.n; s0 += 256) {
          int begin = 0, end = 0;
          if (s0 + lane < a.n) {
            const Sequence seq = load_sequence(a, s0 + lane);
            begin = seq.q_begin + seq.q_len;
            end = seq.q_end;
          }
          for (uint32_t some = __ballot_sync(0xffffffffu, begin < end); some; some &= some - 1) {
            const int l = __ffs(some) - 1;
            const int from = __shfl_sync(0xffffffffu, begin, l), to = __shfl_sync(0xffffffffu, end, l);
            zero_rows(out, a, from, to, blockIdx.x, gridDim.x, lane, 32);
          }
        }
    }
    const int t = (warp - 4) >> 2;
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;
    const int row_token = r / a.G, row_head = r % a.G;
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t s_addr = tmem_base + lane_off + COL_S + t * 128;
    const uint32_t o_addr = tmem_base + lane_off + COL_O + t * D;
    const uint32_t p_addr = tmem_base + lane_off + (P_SPLIT ? COL_P + t * 64 : COL_S + t * 128);
    const int warp_first = quarter * 32 / a.G, warp_last = (quarter * 32 + 31) / a.G;
    int count = 0, outs = 0;  // steps of this tile, output tiles of both (over all units of the CTA)
    Unit w;
    auto next_unit = [&](int unit) {  // the first from `unit` on that has something to do
      while (unit < units && !unit_at<PAGED>(p, unit, &w)) unit += gridDim.x;
      return unit;
    };
    for (int unit = next_unit(blockIdx.x); unit < units;) {
      if (__any_sync(0xffffffffu, abort_flag[0] != 0)) break;
      const int first_token = w.t0 + t * p.tile_tokens;
      const int tokens = min(p.tile_tokens, w.seq.q_len - first_token);
      const int rows = tokens > 0 ? tokens * a.G : 0;
      const bool warp_live = quarter * 32 < rows, live = r < rows;
      const int token = first_token + row_token;  // of the sequence
      const int pos = live ? w.base + token : -1;
      // positions of the warp's rows
      const int wmin = w.base + first_token + warp_first;
      const int wmax = w.base + first_token + min(warp_last, tokens - 1);
      // (positions may lie behind the last key: see load_sequence)
      const int end = PAGED ? w.seq.kv_len - 1 : MOST_KEYS, pos_end = min(pos, end), wmin_end = min(wmin, end), wmax_end = min(wmax, end);
      float m_used = -INFINITY, l = 0.f;
      const int before = count;
      for (int m = w.m0; m < w.m1; ++m) {
        const int j = w.kr.tile(m);
        if (!w.active(t, j)) continue;
        const int c = count++;
        const bool first = c == before;
        ptx::mbar_wait(&s_full[t], c & 1, abort_flag, a.status, 81);
        ptx::tc_fence_after();
        if (!warp_live) {
          if constexpr (P_SPLIT) ptx::mbar_arrive(&s_free[t]);
          // (P of these rows is never read into a stored result; the barriers' phases stay in step)
          if (P_SPLIT && c > 0) ptx::mbar_wait(&o_done[t], (c - 1) & 1, abort_flag, a.status, 82);
          ptx::tc_fence_before();
          ptx::mbar_arrive(&p_part[t]);
          ptx::mbar_arrive(&p_full[t]);
          continue;
        }
        const int j0 = j * TILE;
        // blocks of 32 columns that no row of the warp sees, and that all see
        uint32_t none = 0, all = 0;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int b0 = j0 + 32 * q;
          if (b0 > wmax_end || (wmin - (b0 + 31) >= a.window && b0 >= a.sinks)) none |= 1u << q;
          if (b0 + 31 <= wmin_end && (wmax - b0 < a.window || b0 + 32 <= a.sinks)) all |= 1u << q;
        }
        const bool plain = all == 15u && p.scale_log2 >= 0.f;
        uint32_t sr[4][32];
        float mx = -INFINITY;
        if (plain) {
          float x[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int q = 0; q < 4; ++q) ptx::tmem_ld32(s_addr + 32 * q, sr[q]);
#pragma unroll
          for (int q = 0; q < 4; ++q) am::tmem_ld_wait_dep(sr[q]);
#pragma unroll
          for (int i = 0; i < 32; i += 2)
#pragma unroll
            for (int q = 0; q < 4; ++q) x[q] = am::max3(x[q], __uint_as_float(sr[q][i]), __uint_as_float(sr[q][i + 1]));
          mx = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])) * p.scale_log2;
        } else {
          const uint64_t sc2 = am::pack2f(p.scale_log2, p.scale_log2);
          float x0 = -INFINITY, x1 = -INFINITY;
          auto scale32 = [&](uint32_t (&v)[32], int q) {
            if ((none >> q) & 1u) return;
            // columns below pos + 1 - b0 are not in the future, those from pos - window + 1 - b0 on in the window
            const int b0 = j0 + 32 * q;
            const int64_t low = (int64_t)pos - a.window + 1 - b0;
            if ((all >> q) & 1u) {
#pragma unroll
              for (int i = 0; i < 32; i += 2) {
                float s0, s1;
                am::unpack2f(am::mul2(am::pack2u(v[i], v[i + 1]), sc2), s0, s1);
                if (i & 2) x1 = am::max3(x1, s0, s1);
                else x0 = am::max3(x0, s0, s1);
                v[i] = __float_as_uint(s0);
                v[i + 1] = __float_as_uint(s1);
              }
              return;
            }
            const uint32_t seen = low_bits(pos_end + 1 - b0) & (~low_bits(low < 0 ? 0 : (int)low) | low_bits(a.sinks - b0));
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              float s0, s1;
              am::unpack2f(am::mul2(am::pack2u(v[i], v[i + 1]), sc2), s0, s1);
              s0 = seen & (1u << i) ? s0 : -INFINITY;
              s1 = seen & (2u << i) ? s1 : -INFINITY;
              if (i & 2) x1 = am::max3(x1, s0, s1);
              else x0 = am::max3(x0, s0, s1);
              v[i] = __float_as_uint(s0);
              v[i + 1] = __float_as_uint(s1);
            }
          };
          ptx::tmem_ld32(s_addr, sr[0]);
          am::tmem_ld_wait_dep(sr[0]);
          ptx::tmem_ld32(s_addr + 32, sr[1]);
          scale32(sr[0], 0);
          am::tmem_ld_wait_dep(sr[1]);
          ptx::tmem_ld32(s_addr + 64, sr[2]);
          scale32(sr[1], 1);
          am::tmem_ld_wait_dep(sr[2]);
          ptx::tmem_ld32(s_addr + 96, sr[3]);
          scale32(sr[2], 2);
          am::tmem_ld_wait_dep(sr[3]);
          scale32(sr[3], 3);
          mx = fmaxf(x0, x1);
        }
        if constexpr (P_SPLIT) {
          ptx::tc_fence_before();
          ptx::mbar_arrive(&s_free[t]);
        }
        const float m_new = fmaxf(m_used, mx);
        if (first) {
          m_used = m_new;
        } else {
          const bool need = live && m_new > m_used + RESCALE_THRESHOLD;  // (other rows may hold anything)
          if (__any_sync(0xffffffffu, need)) {
            ptx::mbar_wait(&o_done[t], (c - 1) & 1, abort_flag, a.status, 83);
            ptx::tc_fence_after();
            const float factor = m_new == -INFINITY ? 1.f : exp2f(m_used - m_new);
#pragma unroll 1
            for (int q = 0; q < D / 32; ++q) {
              uint32_t v[32];
              ptx::tmem_ld32(o_addr + q * 32, v);
              ptx::tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * factor);
              ptx::tmem_st32(o_addr + q * 32, v);
            }
            ptx::tmem_st_wait();
            l *= factor;
            m_used = m_new;
          }
        }
        const float m_safe = m_used == -INFINITY ? 0.f : m_used;
        if constexpr (P_SPLIT) {
          if (c > 0) {  // P(c) goes over P(c-1)
            ptx::mbar_wait(&o_done[t], (c - 1) & 1, abort_flag, a.status, 84);
            ptx::tc_fence_after();
          }
        }
        const uint64_t negm2 = am::pack2f(-m_safe, -m_safe);
        auto first_part = [&]() {
          ptx::tmem_st_wait();
          ptx::tc_fence_before();
          ptx::mbar_arrive(&p_part[t]);
        };
        if (plain) {
          l += exp_row<T>(sr, am::pack2f(p.scale_log2, p.scale_log2), negm2, p_addr, first_part);
        } else {
          uint64_t lsum = am::pack2f(0.f, 0.f), lsum_b = am::pack2f(0.f, 0.f);
          auto exp32 = [&](const uint32_t (&v)[32], int q) {
            uint32_t packed[16];
            if ((none >> q) & 1u) {
#pragma unroll
              for (int i = 0; i < 16; ++i) packed[i] = 0u;
              ptx::tmem_st16(p_addr + q * 16, packed);
              return;
            }
            float x[32];
#pragma unroll
            for (int i = 0; i < 32; i += 2)
              am::unpack2f(am::add2(am::pack2u(v[i], v[i + 1]), negm2), x[i], x[i + 1]);
#pragma unroll
            for (int i = 0; i < 32; ++i) x[i] = am::ex2(x[i]);
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
              lsum = am::add2(lsum, am::pack2f(x[i], x[i + 1]));
              lsum_b = am::add2(lsum_b, am::pack2f(x[i + 2], x[i + 3]));
              packed[i >> 1] = am::cvt_pair<T>(x[i], x[i + 1]);
              packed[(i >> 1) + 1] = am::cvt_pair<T>(x[i + 2], x[i + 3]);
            }
            ptx::tmem_st16(p_addr + q * 16, packed);
          };
          exp32(sr[0], 0);
          exp32(sr[1], 1);
          exp32(sr[2], 2);
          first_part();
          exp32(sr[3], 3);
          float l0, l1;
          am::unpack2f(am::add2(lsum, lsum_b), l0, l1);
          l += l0 + l1;
        }
        ptx::tmem_st_wait();
        ptx::tc_fence_before();
        ptx::mbar_arrive(&p_full[t]);
      }
      // What the epilogue needs of this unit; the next one is looked up while the last product runs.
      const bool counted = count > before, whole = w.whole, bulk0 = is_bulk(w, 0), bulk1 = is_bulk(w, 1), bulk = t ? bulk1 : bulk0;
      const int head = w.hk * a.G + row_head;
      const long long tok = w.seq.q_begin + token;
      const bool some = l > 0.f;  // (a row without keys: zeros)
      const float inv = some ? 1.f / l : 0.f;
      const long long oat = (long long)w.s * a.os[0] + head * a.os[1] + tok * a.os[2];
      T* orow = reinterpret_cast<T*>(p.out) + oat;
      const long long prow = ((long long)w.split * a.tokens + tok) * a.H + head;
      if (live) {
        const float ls = some ? m_used * LN2 + logf(l) : -INFINITY;
        if (!whole) a.part_lse[prow] = ls;
        else if (!PAGED && p.lse) p.lse[((long long)w.s * a.H + head) * a.tokens + tok] = ls;
      }
      unit = next_unit(unit + gridDim.x);
      if (counted) {
        ptx::mbar_wait(&o_done[t], (count - 1) & 1, abort_flag, a.status, 85);
        ptx::tc_fence_after();
      }
      const int mine = outs + (t && bulk0 ? 1 : 0);  // number of this output tile
      outs += (bulk0 ? 1 : 0) + (bulk1 ? 1 : 0);
      if (bulk) wait_copied(copied, mine, abort_flag, a.status);
      if (warp_live) {
        const uint64_t inv2 = am::pack2f(inv, inv);
        const bool zeros = !__all_sync(0xffffffffu, some || !live);  // (the columns hold what was there before)
#pragma unroll 1
        for (int h = 0; h < D / 64; ++h) {  // (not unrolled: run once per unit, its code is fetched anew each time)
          uint32_t v[2][32];
          __syncwarp();
          ptx::tmem_ld32(o_addr + h * 64, v[0]);
          ptx::tmem_ld32(o_addr + h * 64 + 32, v[1]);
          am::tmem_ld_wait_dep(v[0]);
          am::tmem_ld_wait_dep(v[1]);
          if (zeros) {
#pragma unroll
            for (int e = 0; e < 64; ++e) v[e >> 5][e & 31] = some ? v[e >> 5][e & 31] : 0u;
          }
#pragma unroll
          for (int e = 0; e < 64; e += 2) {
            float x, y;
            am::unpack2f(am::mul2(am::pack2u(v[e >> 5][e & 31], v[e >> 5][(e & 31) + 1]), inv2), x, y);
            v[e >> 5][e & 31] = __float_as_uint(x);
            v[e >> 5][(e & 31) + 1] = __float_as_uint(y);
          }
          if (whole) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const uint32_t* x = &v[e >> 2][(e & 3) * 8];
              uint4 o;
              o.x = am::cvt_pair<T>(__uint_as_float(x[0]), __uint_as_float(x[1]));
              o.y = am::cvt_pair<T>(__uint_as_float(x[2]), __uint_as_float(x[3]));
              o.z = am::cvt_pair<T>(__uint_as_float(x[4]), __uint_as_float(x[5]));
              o.w = am::cvt_pair<T>(__uint_as_float(x[6]), __uint_as_float(x[7]));
              if (LOW && live) {  // what the rounding leaves
                float y[8];
                unpack<T>(o, y);
                uint4 low;
                low.x = am::cvt_pair<T>(__uint_as_float(x[0]) - y[0], __uint_as_float(x[1]) - y[1]);
                low.y = am::cvt_pair<T>(__uint_as_float(x[2]) - y[2], __uint_as_float(x[3]) - y[3]);
                low.z = am::cvt_pair<T>(__uint_as_float(x[4]) - y[4], __uint_as_float(x[5]) - y[5]);
                low.w = am::cvt_pair<T>(__uint_as_float(x[6]) - y[6], __uint_as_float(x[7]) - y[7]);
                *reinterpret_cast<uint4*>(reinterpret_cast<T*>(a.low) + oat + h * 64 + e * 8) = low;
              }
              if (bulk)
                *reinterpret_cast<uint4*>(out_smem + h * BOX_BYTES + r * 128 + ((e ^ (r & 7)) << 4)) = o;
              else if (live)
                *reinterpret_cast<uint4*>(orow + h * 64 + e * 8) = o;
            }
          } else if (live && some) {  // (a part without keys is known by its lse)
            uint4* dst = reinterpret_cast<uint4*>(a.part_out + prow * D + h * 64);
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const uint32_t* x = &v[e >> 3][(e & 7) * 4];
              dst[e] = make_uint4(x[0], x[1], x[2], x[3]);
            }
          }
        }
      }
      ptx::tc_fence_before();
      if (bulk) {
        ptx::fence_proxy_async_smem();
        ptx::mbar_arrive(out_full);
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

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn encode_fn() {
  static EncodeFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* sym = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &sym, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeFn>(sym);
    else
      cudaGetLastError();
  });
  return fn;
}

bool encode(CUtensorMap* map, int rank, const void* base, const cuuint64_t* dims, const cuuint64_t* strides,
            const cuuint32_t* box, const char* what) {
  cuuint32_t elem[5] = {1, 1, 1, 1, 1};
  const CUresult r = encode_fn()(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, (cuuint32_t)rank, const_cast<void*>(base), dims, strides,
                                 box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                 CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r == CUDA_SUCCESS) return true;
  set_error("local attention: tensor map of %s refused with CUresult %d", what, (int)r);
  return false;
}

int gcd(int a, int b) { return b == 0 ? a : gcd(b, a % b); }

// stride of a dimension; one of extent 1 may carry any
cuuint64_t stride_of(int64_t st, int64_t extent) { return (cuuint64_t)(extent > 1 ? st : 64) * 2; }

bool stride_ok(int64_t st, int64_t extent) { return extent <= 1 || (st > 0 && st % 8 == 0 && st < (1ll << 38)); }

}  // namespace

// packed rows of q (or a tensor laid out like it): [features, head of the group, token, key head, sequence],
// box of `tokens` tokens of one key head
bool local_map_rows(CUtensorMap* map, const void* q, const int64_t* st, const LocalArgs& a, int tokens, const char* what) {
  const bool paged = a.table != nullptr;
  const cuuint64_t dims[5] = {(cuuint64_t)a.D, (cuuint64_t)a.G, (cuuint64_t)a.tokens, (cuuint64_t)a.KV,
                              (cuuint64_t)(paged ? 1 : a.n)};
  const cuuint64_t strides[4] = {stride_of(st[1], a.G), stride_of(st[2], a.tokens), stride_of(st[1] * a.G, a.KV),
                                 stride_of(st[0], paged ? 1 : a.n)};
  const cuuint32_t box[5] = {64, (cuuint32_t)a.G, (cuuint32_t)tokens, 1, 1};
  return encode(map, 5, q, dims, strides, box, what);
}
// keys (or values): [features, position (of a page), key head, sequence or page], box of one piece
bool local_map_keys(CUtensorMap* map, const void* k, const int64_t* st, const LocalArgs& a, int piece, const char* what) {
  const bool paged = a.table != nullptr;
  const int64_t rows = paged ? a.page : a.tokens, outer = paged ? a.pages : a.n;
  const cuuint64_t dims[4] = {(cuuint64_t)a.D, (cuuint64_t)rows, (cuuint64_t)a.KV, (cuuint64_t)outer};
  const cuuint64_t strides[3] = {stride_of(st[2], rows), stride_of(st[1], a.KV), stride_of(st[0], outer)};
  const cuuint32_t box[4] = {64, (cuuint32_t)piece, 1, 1};
  return encode(map, 4, k, dims, strides, box, what);
}
bool local_rows_ok(const void* p, const int64_t* st, const LocalArgs& a) {
  return aligned16(p) && st[3] == 1 && stride_ok(st[1], a.H) && stride_ok(st[2], a.tokens) &&
         (a.table || stride_ok(st[0], a.n)) && st[1] * (int64_t)a.G < (1ll << 38);
}
bool local_keys_ok(const void* p, const int64_t* st, const LocalArgs& a) {
  return aligned16(p) && st[3] == 1 && stride_ok(st[1], a.KV) && stride_ok(st[2], a.table ? a.page : a.tokens) &&
         stride_ok(st[0], a.table ? a.pages : a.n);
}
int local_piece(const LocalArgs& a) { return a.table ? gcd(a.page, LOCAL_TC_TILE) : LOCAL_TC_TILE; }

bool local_tc_supported(const LocalArgs& a, int dtype, const void* q, const void* k, const void* v, const void* out) {
  if (dtype != TB200_F16 && dtype != TB200_BF16) return false;
  if (a.D != 64 && a.D != 128) return false;
  if (a.table && (local_piece(a) < 8 || a.pages == 0)) return false;
  return local_rows_ok(q, a.qs, a) && local_rows_ok(out, a.os, a) && local_keys_ok(k, a.ks, a) && local_keys_ok(v, a.vs, a) &&
         encode_fn() != nullptr;
}

namespace {

template <typename T, int D, bool PAGED, bool LOW>
int launch_fwd(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const CUtensorMap& mo, const FwdParams& p,
               cudaStream_t st) {
  constexpr int SMEM = 7 * TILE * D * 2 + 1024 + 384;  // (tiles, alignment, barriers and what follows them)
  static_assert(33 * 8 + 2 * sizeof(Walk) <= 384, "barriers, flags and walks");
  static_assert(SMEM <= 227 * 1024, "shared memory of one CTA");
  auto kern = local_fwd_tc_kernel<T, D, PAGED, LOW>;
  static std::atomic<unsigned long long> optin_done{0};
  static std::atomic<int> regs_cached{0};
  cudaError_t e = smem_optin_per_device(optin_done, reinterpret_cast<const void*>(kern), SMEM);
  int regs = regs_cached.load(std::memory_order_relaxed);
  if (e == cudaSuccess && regs == 0) {
    cudaFuncAttributes fa;
    if ((e = cudaFuncGetAttributes(&fa, kern)) == cudaSuccess) {
      regs = fa.numRegs;
      regs_cached.store(regs, std::memory_order_relaxed);
    }
  }
  if (e != cudaSuccess) {
    set_error("local_fwd_tc: cudaFuncSetAttribute failed: %s", cudaGetErrorString(e));
    return (int)e;
  }
  // (the register allowances of the kernel's warps come from its launch allocation)
  if (regs * FWD_THREADS < 4 * 32 * REGS_SERVICE + 8 * 32 * REGS_SOFTMAX) {
    set_error("local_fwd_tc: kernel compiled with %d registers per thread, the register rebalancing needs %d", regs, REGS_LAUNCH);
    return TB200_ERR_UNSUPPORTED;
  }
  const int sms = sm_count();
  kern<<<(unsigned)(p.units < sms ? p.units : sms), FWD_THREADS, SMEM, st>>>(mq, mk, mv, mo, p);
  return launch_status("local_fwd_tc");
}

}  // namespace

int launch_local_fwd_tc(void* out, float* lse, const void* q, const void* k, const void* v, const LocalArgs& a, int max_q,
                        int dtype, cudaStream_t st) {
  FwdParams p;
  p.a = a;
  p.a.status = device_status_ptr();
  p.out = out;
  p.lse = lse;
  p.scale_log2 = a.scale * LOG2E;
  p.tile_tokens = TILE / a.G;
  p.piece = local_piece(a);
  p.pairs = (int)ceil_div(max_q, 2 * p.tile_tokens);
  const int64_t units = (int64_t)p.pairs * a.KV * a.n * a.splits;
  TB200_REQUIRE(a.before || units < MOST_UNITS, TB200_ERR_UNSUPPORTED, "local_fwd_tc: %lld units of work", (long long)units);
  p.units = (int)(units < MOST_UNITS ? units : MOST_UNITS);  // (list form: the kernel finds the number)
  p.outer = Divisor(a.before ? 1 : p.units / p.pairs);
  p.kv = Divisor(a.KV);
  p.splits = Divisor(a.splits);
  p.test = WaitTest::of_this_thread(1, 1);
  CUtensorMap mq, mk, mv, mo;
  bind_primary_context();
  if (!local_map_rows(&mq, q, a.qs, a, p.tile_tokens, "q") || !local_map_rows(&mo, out, a.os, a, p.tile_tokens, "out") || !local_map_keys(&mk, k, a.ks, a, p.piece, "k") ||
      !local_map_keys(&mv, v, a.vs, a, p.piece, "v"))
    return TB200_ERR_UNSUPPORTED;
  auto go = [&](auto tag, auto dsel) -> int {
    using T = decltype(tag);
    constexpr int D = decltype(dsel)::value;
    return a.table ? launch_fwd<T, D, true, false>(mq, mk, mv, mo, p, st)
           : a.low ? launch_fwd<T, D, false, true>(mq, mk, mv, mo, p, st) : launch_fwd<T, D, false, false>(mq, mk, mv, mo, p, st);
  };
  using D64 = std::integral_constant<int, 64>;
  using D128 = std::integral_constant<int, 128>;
  if (dtype == TB200_BF16) return a.D == 128 ? go(__nv_bfloat16{}, D128{}) : go(__nv_bfloat16{}, D64{});
  return a.D == 128 ? go(__half{}, D128{}) : go(__half{}, D64{});
}

}  // namespace tb200
