// Attention of a prompt (or a chunk of one) over the KV cache on the tensor cores, with a sliding window and leading
// tokens that stay visible.
//
// Mathematics: for every query row the running maximum m and sum l of 2^(s - m) over key tiles of 128, O = sum 2^(s - m) v
// accumulated in tensor memory, rescaled only when the maximum has grown by more than 2^8.  4 T n D operations per head
// against n D elements of keys and values that stay in L2: bound by the tensor pipe and, next to it, by the 128 x 128
// exponentials of a tile (16 a clock per SM, 1024 clocks; a tile's two products take 1024 at D = 128, 2048 at 256).
//
// * A query tile is 128 rows: the heads of one KV head for consecutive tokens (tc_common.cuh); a unit of work has two.
//   D <= 128: one CTA takes both, each with its score columns and accumulator in tensor memory and two softmax
//   warpgroups; the tiles take turns, one's products run under the other's exponentials, and a key tile is
//   loaded once for both.  D = 256: the accumulator takes half of the tensor memory, so a pair of CTAs takes a unit with
//   products of 256 rows across the two SMs (cta_group::2), each holding its query tile, two score buffers, half of the
//   keys of a tile and half of the value columns.  One CTA alone would read 128 KiB of keys and
//   values from L2 for each 128 x 128 tile: that ran at 4600 clocks a tile, waiting for L2 and for shared memory.
// * Warps: 0 loads queries and keys, 1 values, 2 issues S = Q K^T, 3 issues O += P V (P replaces S in tensor memory,
//   in the inputs' type: the product needs a 16-bit operand; f16: lifted first, mma_sync.cuh), the others softmax, two threads a row: with one
//   the row's 128 exponentials were a chain of 4000 clocks.
// * Only the key tiles that some row of the unit sees are visited; only those that some row does not see whole are masked.
//   Value rows behind the sequence's length are zeroed in shared memory before the product, whatever the cache holds there.
// * Persistent CTAs, one per SM.  plan_kernel cuts the key tiles of all units into equal ranges (ranges.cuh), so that unequal
//   lengths, causal triangles and few query rows over a long cache all fill the GPU.  A unit cut in pieces leaves (O, m, l) per piece in the workspace and
//   join_kernel adds them up in order.
//
// Measured (B200, the whole call): 16 query / 2 KV heads, D = 256, a prompt of 8192 0.46 ms = 1.19 PFLOP/s (0.73 of what cuBLAS
// reaches in a burst, 0.85 of what it sustains under the power cap), a chunk of 2048 over 10240 tokens 0.26 ms (0.73), 48 rows
// over 32768 0.057 ms; a key
// tile takes 2670 clocks, 2048 of them on the tensor pipe.  32 / 8 heads, D = 128, two prompts of 8192 with a window of 1024:
// 0.41 ms (0.41; a causal prompt of 8192 0.65 ms = 0.52, at D = 64 0.51 ms = 0.33): 4300 clocks for the two tiles' 2048 of products and 2048 of exponentials, the softmax threads' waits
// (tensor-memory loads and stores, the other half's maximum, the hand-over of P) are most of the rest.  Five prompts of up to 193:
// 23 us, three launches' latency.
#include "ranges.cuh"
#include "tc_common.cuh"

namespace dflash {
namespace {

using namespace tc;

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kRescale = 8.f;              // in log2 units
constexpr int kUnitCost = 3;                 // what a unit costs besides its key tiles (loading queries, storing rows), in tiles

struct PromptParams {
  CacheArgs a;
  Tiling t;
  Ranges ranges;               // rows of units of two query tiles
  int box;
  float scale_log2;
  int out32;                   // `out` is 32-byte aligned
  float4* part_o;              // [2 * grid][D / 4][256]
  float2* part_ml;             // [2 * grid][256]
};

template <int D> struct Cfg {
  static constexpr bool PAIR = D == 256;                    // two CTAs on one unit, a query tile each
  static constexpr int NC = D / 64;                         // 64-column chunks of a row
  static constexpr int QT = PAIR ? 1 : 2;                   // query tiles of one CTA (a unit has two)
  static constexpr int threads = 128 + QT * 256;            // four helper warps, eight softmax warps a query tile
  // registers a thread at launch; what the helper warps give up the softmax warps take
  static constexpr int regs_launch = PAIR ? 168 : 96, regs_helper = 56, regs_softmax = PAIR ? 216 : 104;
  static_assert(128 * regs_helper + (threads - 128) * regs_softmax <= threads * regs_launch, "register split");
  static constexpr int k_rows = PAIR ? 64 : 128;            // this CTA's share of a key tile: rows ...
  static constexpr int v_chunks = PAIR ? NC / 2 : NC;       // ... and of a value tile: columns
  static constexpr int k_chunk = k_rows * 128, k_stage = NC * k_chunk, v_stage = v_chunks * kChunk;
  // A pair's key stages: the next tile's keys are wanted a period after the stage's last use, its values two; copies take
  // about 2000 clocks under load (two key and three value stages waited 500 clocks a tile for keys).
  static constexpr int KS = D == 64 ? 4 : (PAIR ? 3 : 2), VS = D == 64 ? 6 : (PAIR ? 2 : 3);
  static constexpr int q = 0;
  static constexpr int k = QT * NC * kChunk, v = k + KS * k_stage;
  static constexpr int bars = v + VS * v_stage;
  // barriers
  static constexpr int b_q_full = 0, b_q_empty = 1, b_s_full = 2, b_p_half = 4, b_pv_done = 8, b_tail = 10, b_k_full = 11, b_k_empty = b_k_full + KS, b_v_full = b_k_empty + KS, b_v_empty = b_v_full + VS,
                       n_bars = b_v_empty + VS;
  static constexpr int misc = bars + (8 * n_bars + 15) / 16 * 16;   // tensor-memory base, abort flag
  static constexpr int xch = misc + 16;                     // row maxima (sums) of the two halves: [QT][slots][2][128]
  static constexpr int slots = PAIR ? 2 : 1;
  static constexpr int total = xch + QT * slots * 2 * 128 * 4;
  // tensor-memory columns: accumulators first, score buffers in the upper half
  __host__ __device__ static constexpr int col_o(int qi) { return qi * 128; }
  __host__ __device__ static constexpr int col_s(int i) { return 256 + i * 128; }
};
static_assert(Cfg<256>::total <= 232448 && Cfg<128>::total <= 232448 && Cfg<64>::total <= 232448, "shared memory");

// ---- the plan ----
__device__ __forceinline__ int unit_steps(const CacheArgs& a, RowLens len, int u, int tokens) {
  const int t0 = u * tokens;
  if (t0 >= len.rows) return 0;
  return key_tiles(a, len, t0, t0 + tokens < len.rows ? t0 + tokens : len.rows).count;
}
__global__ void __launch_bounds__(1024) plan_kernel(const PromptParams p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  plan_ranges<kUnitCost>(p.ranges, p.a, [&](RowLens len, int u) { return unit_steps(p.a, len, u, 2 * p.t.Tt); });
}

struct Unit {
  int b, h, gc, t0;            // t0: first token of the unit
  RowLens len;
  KeyTiles k;
};

struct Segment {
  Unit u;
  int lo, hi;                  // key tiles [lo, hi) of u.k
  int nq;                      // query tiles with rows in use
  int slot;                    // -1: the whole unit
};
__device__ __forceinline__ Unit unit_at(const PromptParams& p, const Cursor& c) {
  Unit u;
  u.b = c.b;
  u.h = p.t.GC == 1 ? c.hg : c.hg / p.t.GC;
  u.gc = c.hg - u.h * p.t.GC;
  u.t0 = c.u * 2 * p.t.Tt;
  u.len = c.len;
  const int t1 = u.t0 + 2 * p.t.Tt;
  u.k = key_tiles(p.a, c.len, u.t0, t1 < c.len.rows ? t1 : c.len.rows);
  return u;
}
struct Walker {
  const PromptParams& p;
  RangeWalker w;
  __device__ Walker(const PromptParams& p_, int worker) : p(p_), w(p_.ranges, p_.a, worker) {}
  __device__ bool next(Segment& s) {
    const int tokens = 2 * p.t.Tt;
    if (!w.find([&](RowLens len, int u) { return u * tokens < len.rows ? u : p.ranges.per_row; }, s.lo)) return false;
    s.u = unit_at(p, w.c);
    s.nq = s.u.t0 + p.t.Tt < s.u.len.rows ? 2 : 1;
    s.hi = w.take(s.lo, s.u.k.count, s.slot);
    return true;
  }
};

// row r of query tile qi of a unit: token, output row; false: not in use
__device__ __forceinline__ bool row_of(const PromptParams& p, const Unit& u, int qi, int r, int& t, long long& row) {
  const int g = u.gc * p.t.Gt + r % p.t.Gt;
  t = u.t0 + qi * p.t.Tt + r / p.t.Gt;
  row = ((long long)u.b * p.a.Hq + u.h * p.t.G + g) * p.a.T + t;
  return r < p.t.Gt * p.t.Tt && g < p.t.G && t < u.len.rows;
}

__device__ __forceinline__ uint32_t low_bits(int n) {      // bits [0, n), n clamped to [0, 32]
  return n <= 0 ? 0u : (n >= 32 ? 0xffffffffu : (1u << n) - 1u);
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
template <typename T, int D>
__global__ void __launch_bounds__(Cfg<D>::threads, 1)
prompt_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
              const __grid_constant__ CUtensorMap map_v, const PromptParams p) {
  using C = Cfg<D>;
  constexpr bool PAIR = C::PAIR;
  constexpr int NC = C::NC, KS = C::KS, VS = C::VS;
  extern __shared__ __align__(1024) uint8_t sm[];
  const CacheArgs& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = PAIR ? (int)ptx::cluster_rank() : 0, worker = PAIR ? blockIdx.x >> 1 : blockIdx.x;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + C::bars);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sm + C::misc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(sm + C::misc + 4);
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (threadIdx.x == 0) {
    ptx::prefetch_tensormap(&map_q);
    ptx::prefetch_tensormap(&map_k);
    ptx::prefetch_tensormap(&map_v);
    // Arrivals.  P, in two halves: one a softmax warp (4 a query tile; 8 in each CTA of a pair).  Values: the
    // loading lane of each CTA.  A pair's leader has the barriers that its issuing lanes wait for.
    for (int i = 0; i < C::n_bars; ++i) {
      const bool soft = i >= C::b_p_half && i < C::b_p_half + 4;
      const bool val = i >= C::b_v_full && i < C::b_v_full + VS;
      ptx::mbar_init(&bars[i], soft ? (PAIR ? 16 : 8) : (val && PAIR ? 2 : 1));
    }
    *abort_flag = (ptx::smem_u32(sm) & 1023u) != 0u;      // swizzled tiles need 1024-byte alignment; never seen violated
    if (*abort_flag) atomicExch(a.status, kStatusSmemAlign);
    ptx::fence_mbar_init();
  }
  if (warp == 2) {
    if constexpr (PAIR) {
      ptx::tmem_alloc_pair(tmem_slot, 512);
      ptx::tmem_relinquish_pair();
    } else {
      ptx::tmem_alloc(tmem_slot, 512);
      ptx::tmem_relinquish();
    }
  }
  ptx::tc_fence_before();
  if constexpr (PAIR) ptx::cluster_sync();
  __syncthreads();
  ptx::tc_fence_after();
  asm volatile("griddepcontrol.wait;" ::: "memory");     // the plan
  const uint32_t tmem = *tmem_slot;
  // A wait that gives up raises the abort flags, after which every wait of the CTA (or pair) returns at once: the roles run
  // through their loops without results, meet at the end and leave.
  auto wait_as = [&](int bar, uint32_t parity, bool cluster) {
#pragma unroll 1
    for (uint32_t i = 0; i < ptx::kWaitPolls; ++i) {
      if (PAIR && cluster ? ptx::mbar_try_wait_cluster(&bars[bar], parity) : ptx::mbar_try_wait(&bars[bar], parity)) return true;
      if ((i & 63u) == 63u) {
        if (*abort_flag) return false;
        __nanosleep(40);
      }
    }
    *abort_flag = 1;
    if constexpr (PAIR) ptx::cluster_store(ptx::cluster_addr(const_cast<int*>(abort_flag), rank ^ 1), 1);
    atomicExch(a.status, kStatusMbarWait);
    return false;
  };
  // Every wait is made by a whole warp, whose lanes agree on the outcome: none leaves a loop that the others stay in.  (The
  // softmax warps' loops do not depend on it: they call wait_as.)
  auto wait = [&](int bar, uint32_t parity) { return __all_sync(0xffffffffu, wait_as(bar, parity, false)); };
  auto wait_pair = [&](int bar, uint32_t parity) { return __all_sync(0xffffffffu, wait_as(bar, parity, true)); };   // the other CTA's stores among what is waited for
  auto commit = [&](int bar) {
    if constexpr (PAIR) ptx::umma_commit_pair(&bars[bar]);
    else ptx::umma_commit(&bars[bar]);
  };
  // the leader's barrier, for arrivals and copies of both CTAs
  auto arrive_leader = [&](int bar) {
    if (PAIR) ptx::cluster_arrive_tc(ptx::cluster_addr(&bars[bar], 0));
    else ptx::mbar_arrive(&bars[bar]);
  };
  auto load = [&](void* dst, const CUtensorMap* m, int x, int y, int z, int w, int bar) {
    if constexpr (PAIR) ptx::tma_load_4d_pair(dst, m, x, y, z, w, ptx::cluster_addr(&bars[bar], 0));
    else ptx::tma_load_4d(dst, m, x, y, z, w, &bars[bar]);
  };

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::regs_helper));
    Walker walk(p, worker);
    Segment s;
    if (warp == 0) {
      // ------------------------------ queries and keys ------------------------------
      uint32_t fill = 0, seg = 0;
      bool ok = __all_sync(0xffffffffu, !*abort_flag);
      while (ok && walk.next(s)) {
        if (seg > 0) ok = wait(C::b_q_empty, (seg - 1) & 1);
        if (!ok) break;
        if (lane == 0) {
          const int tiles = PAIR ? 2 : s.nq;                  // a pair's tile without rows in use reads as zeros
          if (rank == 0) ptx::mbar_arrive_expect_tx(&bars[C::b_q_full], tiles * NC * p.t.Gt * p.t.Tt * 128);
          for (int qi = 0; qi < (PAIR ? 1 : tiles); ++qi)
            for (int c = 0; c < NC; ++c)
              load(sm + C::q + (qi * NC + c) * kChunk, &map_q, c * 64, s.u.gc * p.t.Gt, s.u.t0 + (PAIR ? rank : qi) * p.t.Tt,
                   s.u.b * a.Hkv + s.u.h, C::b_q_full);
        }
        __syncwarp();
        for (int j = s.lo; j < s.hi; ++j, ++fill) {
          const int n0 = tile_key(s.u.k, j) + rank * 64;
          const uint32_t st = fill % KS;
          if (fill >= KS) ok = wait(C::b_k_empty + st, (fill / KS - 1) & 1);
          if (!ok) break;
          if (lane == 0 && rank == 0) ptx::mbar_arrive_expect_tx(&bars[C::b_k_full + st], (PAIR ? 2 : 1) * C::k_stage);
          __syncwarp();
          const int box = p.box < C::k_rows ? p.box : C::k_rows, pieces = C::k_rows / box;
          for (int i = lane; i < NC * pieces; i += 32) {
            const int c = i / pieces, n = n0 + (i - c * pieces) * box;
            const TilePlace at = place_of(a, s.u.b, n, s.u.len.keys);
            load(sm + C::k + st * C::k_stage + c * C::k_chunk + (n - n0) * 128, &map_k, c * 64, at.row, s.u.h, at.outer, C::b_k_full + st);
          }
          __syncwarp();
        }
        ++seg;
      }
    } else if (warp == 1) {
      // ----------------------------------- values -----------------------------------
      uint32_t fill = 0, tails = 0;
      bool ok = __all_sync(0xffffffffu, !*abort_flag);
      while (ok && walk.next(s)) {
        for (int j = s.lo; j < s.hi; ++j, ++fill) {
          const int n0 = tile_key(s.u.k, j), rows = s.u.len.keys - n0;
          const uint32_t st = fill % VS;
          if (fill >= VS) ok = wait(C::b_v_empty + st, (fill / VS - 1) & 1);
          if (!ok) break;
          // Rows behind the sequence's length: a weight of zero times whatever the cache holds there would not be zero, so
          // such a tile lands under a barrier of its own and the rows are cleared before the tile is announced.
          const bool tail = rows < kKeys;
          if (lane == 0) {
            if (tail) ptx::mbar_arrive_expect_tx(&bars[C::b_tail], C::v_stage);
            else if (rank == 0) ptx::mbar_arrive_expect_tx(&bars[C::b_v_full + st], (PAIR ? 2 : 1) * C::v_stage);
            else arrive_leader(C::b_v_full + st);
          }
          __syncwarp();
          uint8_t* dst = sm + C::v + st * C::v_stage;
          const int pieces = kKeys / p.box;
          for (int i = lane; i < C::v_chunks * pieces; i += 32) {
            const int c = i / pieces, n = n0 + (i - c * pieces) * p.box;
            const TilePlace at = place_of(a, s.u.b, n, s.u.len.keys);
            uint8_t* d = dst + c * kChunk + (n - n0) * 128;
            const int col = (rank * C::v_chunks + c) * 64;
            if (tail) ptx::tma_load_4d(d, &map_v, col, at.row, s.u.h, at.outer, &bars[C::b_tail]);
            else load(d, &map_v, col, at.row, s.u.h, at.outer, C::b_v_full + st);
          }
          __syncwarp();
          if (tail) {
            ok = wait(C::b_tail, tails++ & 1);
            if (!ok) break;
            for (int c = 0; c < C::v_chunks; ++c)
              for (int e = (rows > 0 ? rows : 0) * 8 + lane; e < kKeys * 8; e += 32)
                *reinterpret_cast<uint4*>(dst + c * kChunk + e * 16) = make_uint4(0, 0, 0, 0);
            ptx::fence_proxy_async();
            __syncwarp();
            if (lane == 0) {
              if (PAIR) ptx::cluster_arrive(ptx::cluster_addr(&bars[C::b_v_full + st], 0));
              else arrive_leader(C::b_v_full + st);
            }
          }
        }
      }
    } else if (warp == 2) {
      // --------------------------------- S = Q K^T ----------------------------------
      constexpr uint32_t kI = idesc<T>(PAIR ? 256 : 128, kKeys, false);
      if (rank == 0) {
        uint32_t drain = 0, seg = 0, n_s[2] = {0, 0};       // n_s: score tiles issued per buffer
        const uint32_t q_addr = ptx::smem_u32(sm + C::q), k_addr = ptx::smem_u32(sm + C::k);
        bool ok = true;
        while (ok && walk.next(s)) {
          ok = wait(C::b_q_full, seg & 1);
          const int nq = PAIR ? 1 : s.nq;
          for (int j = s.lo; ok && j < s.hi; ++j, ++drain) {
            const uint32_t st = drain % KS;
            ok = wait(C::b_k_full + st, (drain / KS) & 1);
            for (int qi = 0; ok && qi < nq; ++qi) {
              // the buffer is free once the product that read P from it has retired
              const int buf = PAIR ? (int)(drain & 1) : qi;
              if (n_s[buf] > 0) ok = wait(C::b_pv_done + buf, (n_s[buf] - 1) & 1);
              if (!ok) break;
              ptx::tc_fence_after();
              if (ptx::elect_one()) {
                const uint32_t d = tmem + C::col_s(buf);
#pragma unroll 1
                for (int c = 0; c < NC; ++c) {
                  const uint64_t da = make_desc(q_addr + (qi * NC + c) * kChunk, 16, 1024);
                  const uint64_t db = make_desc(k_addr + st * C::k_stage + c * C::k_chunk, 16, 1024);
#pragma unroll
                  for (int k = 0; k < 4; ++k) {
                    if constexpr (PAIR) ptx::umma_ss_pair(d, da + 2 * k, db + 2 * k, kI, c + k > 0);
                    else ptx::umma_ss(d, da + 2 * k, db + 2 * k, kI, c + k > 0);
                  }
                }
                commit(C::b_s_full + buf);
                if (qi == nq - 1) commit(C::b_k_empty + st);
                if (qi == nq - 1 && j == s.hi - 1) commit(C::b_q_empty);
              }
              __syncwarp();
              ++n_s[buf];
            }
          }
          ++seg;
        }
      }
    } else {
      // --------------------------------- O += P V -----------------------------------
      constexpr uint32_t kI = idesc<T>(PAIR ? 256 : 128, D, true);
      if (rank == 0) {
        uint32_t drain = 0, n_p[2] = {0, 0};
        const uint32_t v_addr = ptx::smem_u32(sm + C::v);
        bool ok = true;
        while (ok && walk.next(s)) {
          const int nq = PAIR ? 1 : s.nq;
          for (int j = s.lo; ok && j < s.hi; ++j, ++drain) {
            const uint32_t st = drain % VS;
            ok = wait_pair(C::b_v_full + st, (drain / VS) & 1);
            for (int qi = 0; ok && qi < nq; ++qi) {
              const int buf = PAIR ? (int)(drain & 1) : qi;
              // The weights come in two halves (of every thread's columns), so that the first products run under the
              // second half's exponentials.  The first half of a segment's first tile also says that the last
              // segment's accumulator has been read.
              const uint64_t db = make_desc(v_addr + st * C::v_stage, kChunk, 1024);
              const uint32_t d = tmem + C::col_o(qi), pt = tmem + C::col_s(buf);
#pragma unroll 1
              for (int half = 0; half < 2; ++half) {
                ok = ok && wait(C::b_p_half + 2 * half + buf, n_p[buf] & 1);
                if (!ok) break;
                ptx::tc_fence_after();
                if (ptx::elect_one()) {
                  // 16 keys a step: 2048 bytes of values, 8 columns of P (those of the second 64 keys start at column 64); 64-column
                  // chunks of values lie 16 KiB apart
#pragma unroll
                  for (int i = 0; i < 4; ++i) {
                    const int k = 4 * (i / 2) + 2 * half + i % 2, pc = 64 * (i / 2) + 16 * half + 8 * (i % 2);
                    if constexpr (PAIR) ptx::umma_ts_pair(d, pt + pc, db + (uint64_t)k * 128, kI, j > s.lo || half + i > 0);
                    else ptx::umma_ts(d, pt + pc, db + (uint64_t)k * 128, kI, j > s.lo || half + i > 0);
                  }
                  if (half) {
                    commit(C::b_pv_done + buf);
                    if (qi == nq - 1) commit(C::b_v_empty + st);
                  }
                }
                __syncwarp();
              }
              if (!ok) break;
              ++n_p[buf];
            }
          }
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::regs_softmax));
    // ----------------------------------- softmax ------------------------------------
    Walker walk(p, worker);
    Segment s;
    const int wq = warp & 3, grp = ((warp - 4) >> 2) & 1;     // tensor-memory lane quarter; half of the row
    const int r = wq * 32 + lane;
    const uint32_t lane_addr = tmem + ((uint32_t)(wq * 32) << 16);
    const int qi = (warp - 4) >> 3, tile = PAIR ? rank : qi;  // query tile of this CTA, of the unit
    constexpr int NS = 64;                                    // score columns of this thread
    const int col0 = grp * 64;
    float* xch = reinterpret_cast<float*>(sm + C::xch) + qi * C::slots * 256;
    uint32_t n_s = 0, n_x = 0;                                // score tiles and exchanges done
    auto pv_done = [&](uint32_t n) { wait_as(C::b_pv_done + (PAIR ? (int)(n & 1) : qi), PAIR ? (n >> 1) & 1 : n & 1, false); };
    // Value of the thread that has the other half of this row; the two warps always meet the same number of times.  With
    // one slot the next value is written only after this one has been read: the next tile's scores take both threads' P.
    auto other_half = [&](float mine) {
      float* x = xch + n_x++ % C::slots * 256;
      x[grp * 128 + r] = mine;
      asm volatile("bar.sync %0, 64;" ::"r"(1 + qi * 4 + wq) : "memory");
      return x[(grp ^ 1) * 128 + r];
    };
    while (walk.next(s)) {
      if (!PAIR && qi >= s.nq) continue;
      int t;
      long long row;
      const bool used = row_of(p, s.u, tile, r, t, row);
      const int pos = s.u.len.keys - s.u.len.rows + t;       // of an unused row too: it sees what it sees, nobody reads it
      const int p_min = s.u.len.keys - s.u.len.rows + s.u.t0 + tile * p.t.Tt, p_max = p_min + p.t.Tt - 1;
      float m = -INFINITY, l = 0.f;
      for (int j = s.lo; j < s.hi; ++j, ++n_s) {
        const int buf = PAIR ? (int)(n_s & 1) : qi;
        wait_as(C::b_s_full + buf, PAIR ? (n_s >> 1) & 1 : n_s & 1, false);
        __syncwarp();
        ptx::tc_fence_after();
        const uint32_t s_addr = lane_addr + C::col_s(buf) + col0;
        const int n0 = tile_key(s.u.k, j);
        const bool whole = n0 + kKeys - 1 <= p_min && (a.window == 0 || n0 > p_max - a.window || n0 + kKeys <= a.sinks);
        // Loops of 32 scores, read from tensor memory a second time for the exponentials; a pair's CTA, with half as many
        // warps, takes 64 at a time.  (Two query tiles with 64 scores a thread kept in registers: spills, a fifth of the
        // instruction fetches missing, 500 instead of 458 us for two prompts of 8192 with a window.)
        constexpr int kAt = PAIR ? 2 : 1;
        float mx = -INFINITY;
#pragma unroll 1
        for (int g = 0; g < NS; g += 32 * kAt) {
          uint32_t x[kAt][32];
#pragma unroll
          for (int u = 0; u < kAt; ++u) ptx::tmem_ld32(s_addr + g + u * 32, x[u]);
          ptx::tmem_ld_wait();
          float m4[4] = {mx, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int u = 0; u < kAt; ++u) {
            if (!whole) {                                     // hidden scores go back as -infinity
              const int at = col0 + g + u * 32, hi = pos - n0 - at + 1, lo = a.window > 0 ? hi - a.window : 0, sink = a.sinks - n0 - at;
              const uint32_t seen = low_bits(hi) & (~low_bits(lo) | low_bits(sink));
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (!((seen >> i) & 1u)) x[u][i] = __float_as_uint(-INFINITY);
              ptx::tmem_st32(s_addr + g + u * 32, x[u]);
            }
#pragma unroll
            for (int i = 0; i < 32; i += 2) m4[(i >> 1) & 3] = max3(m4[(i >> 1) & 3], __uint_as_float(x[u][i]), __uint_as_float(x[u][i + 1]));
          }
          mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
        }
        if (!whole) ptx::tmem_st_wait();
        mx = fmaxf(mx, other_half(mx));
        float f = 1.f;
        const bool grow = mx > m && (m == -INFINITY || (mx - m) * p.scale_log2 > kRescale);
        if (grow) {
          f = m == -INFINITY ? 0.f : mma::exp2_approx((m - mx) * p.scale_log2);
          m = mx;
          l *= f;
        }
        const bool rescale = j > s.lo && __any_sync(0xffffffffu, grow);
        const float neg = m == -INFINITY ? 0.f : mma::kLift<T> - m * p.scale_log2;
        // the last product is done with the accumulator
        if (rescale) {
          constexpr int kCols = D / 2;
          pv_done(n_s - 1);
          __syncwarp();
          ptx::tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < kCols; c += 32) {
            uint32_t o[32];
            const uint32_t o_addr = lane_addr + C::col_o(qi) + grp * kCols + c;
            ptx::tmem_ld32(o_addr, o);
            ptx::tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
            ptx::tmem_st32(o_addr, o);
          }
        }
        // P over the front half of this thread's own columns, in two halves
        float2 add[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        uint32_t xs[kAt][32];
#pragma unroll kAt
        for (int half = 0; half < 2; ++half) {
          uint32_t pr[16];
          if (half % kAt == 0) {
#pragma unroll
            for (int u = 0; u < kAt; ++u) ptx::tmem_ld32(s_addr + (half + u) * 32, xs[u]);
            ptx::tmem_ld_wait();
          }
          const uint32_t(&x)[32] = xs[half % kAt];
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            float2 w = fma2v(__uint_as_float(x[i]), __uint_as_float(x[i + 1]), p.scale_log2, neg, neg);
            w.x = mma::exp2_approx(w.x);
            w.y = mma::exp2_approx(w.y);
            add[(i >> 1) & 1] = add2(add[(i >> 1) & 1], w);
            pr[i / 2] = mma::pack<T>(w.x, w.y);
          }
          ptx::tmem_st16(s_addr + half * 16, pr);
          ptx::tmem_st_wait();
          ptx::tc_fence_before();
          // Every phase is waited for, in order (a parity wait that skips one cannot tell "done" from "two phases behind"),
          // and before the next one can end, which takes this warp's arrival.
          if (half && n_s > 0) pv_done(n_s - 1);
          __syncwarp();
          if (lane == 0) arrive_leader(C::b_p_half + 2 * half + buf);
        }
        l += (add[0].x + add[0].y) + (add[1].x + add[1].y);
      }
      // ---- the segment's result ----
      pv_done(n_s - 1);
      __syncwarp();
      ptx::tc_fence_after();
      {                                                        // the same order of the two halves in both threads
        const float x = other_half(l);
        l = grp == 0 ? l + x : x + l;
        if (C::slots == 1) asm volatile("bar.sync %0, 64;" ::"r"(1 + qi * 4 + wq) : "memory");
      }
      constexpr int kCols = D / 2;
      const int c0 = grp * kCols;
      const float inv = l == 0.f ? 0.f : 1.f / l;             // 0: nothing was visible; NaN stays NaN
#pragma unroll 1
      for (int c = 0; c < kCols; c += 32) {
        uint32_t o[32];
        ptx::tmem_ld32(lane_addr + C::col_o(qi) + c0 + c, o);
        ptx::tmem_ld_wait();
        if (s.slot < 0) {
          if (used) {
            T* dst = reinterpret_cast<T*>(a.out) + row * D + c0 + c;
            uint32_t x[16];
#pragma unroll
            for (int i = 0; i < 32; i += 2) x[i / 2] = mma::pack<T>(__uint_as_float(o[i]) * inv, __uint_as_float(o[i + 1]) * inv);
            if (p.out32) {                       // whole sectors; the rows of a warp are far apart
              ptx::st_global_v8(dst, x);
              ptx::st_global_v8(dst + 16, x + 8);
            } else {
#pragma unroll
              for (int i = 0; i < 16; i += 4) reinterpret_cast<uint4*>(dst)[i / 4] = make_uint4(x[i], x[i + 1], x[i + 2], x[i + 3]);
            }
          }
        } else {
          // [D / 4][rows]: the 32 rows of a warp store 512 bytes in a row
          float4* dst = p.part_o + ((long long)s.slot * (D / 4) + (c0 + c) / 4) * 256 + tile * 128 + r;
#pragma unroll
          for (int i = 0; i < 32; i += 4)
            dst[(i / 4) * 256] = make_float4(__uint_as_float(o[i]), __uint_as_float(o[i + 1]), __uint_as_float(o[i + 2]), __uint_as_float(o[i + 3]));
        }
      }
      ptx::tc_fence_before();              // the next segment's first half of P says that the accumulator has been read
      if (grp == 0) {
        if (s.slot >= 0) p.part_ml[(long long)s.slot * 256 + tile * 128 + r] = make_float2(m * p.scale_log2 - mma::kLift<T>, l);
        else if (used && a.lse) a.lse[row] = l == 0.f ? -INFINITY : (m * p.scale_log2 - mma::kLift<T> + log2f(l)) * kLn2;
      }
    }
  }
  __syncwarp();
  __syncthreads();
  if (*abort_flag) __nanosleep(100000);        // copies that were still in flight land before the memory is given back
  if constexpr (PAIR) {
    ptx::cluster_sync();                       // the other CTA's products and arrivals use this one's memory
    if (warp == 2) ptx::tmem_dealloc_pair(tmem, 512);
  } else {
    if (warp == 2) ptx::tmem_dealloc(tmem, 512);
  }
}

// Joins the pieces of a cut unit: 32 rows and 64 columns a block, weights 2^(m_i - max m), added in the order of the pieces.
template <typename T, int D>
__global__ void __launch_bounds__(128) join_kernel(const PromptParams p) {
  constexpr int R = 256;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (p.a.lse && p.a.q_len) {                  // rows behind a sequence's last query
    const long long rows = (long long)p.a.B * p.a.Hq * p.a.T, threads = (long long)gridDim.x * gridDim.y * gridDim.z * 128;
    const long long block = ((long long)blockIdx.z * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x;
    for (long long i = block * 128 + threadIdx.x; i < rows; i += threads) {
      const long long bh = i / p.a.T;
      if ((int)(i - bh * p.a.T) >= lens_of(p.a, (int)(bh / p.a.Hq)).rows) p.a.lse[i] = -INFINITY;
    }
  }
  const Cut cut = p.ranges.cuts[blockIdx.x];
  if (cut.count == 0) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Unit u = unit_at(p, Cursor(p.ranges, p.a, cut.unit));
  const int rr = blockIdx.y * 32 + lane, qi = rr / 128, r = rr % 128;
  const int col = blockIdx.z * 64 + warp * 16;
  int t;
  long long row;
  if (!row_of(p, u, qi, r, t, row)) return;
  auto slot = [&](int i) { return (long long)piece_slot(cut, i); };
  float top = -INFINITY;
  for (int i = 0; i < cut.count; ++i) top = fmaxf(top, p.part_ml[slot(i) * R + rr].x);
  const float z = top == -INFINITY ? 0.f : top;
  float sum = 0.f;
  float4 o[4] = {};
#pragma unroll 2
  for (int i = 0; i < cut.count; ++i) {
    const float2 ml = p.part_ml[slot(i) * R + rr];
    const float w = mma::exp2_approx(ml.x - z);
    sum = fmaf(w, ml.y, sum);
    const float4* src = p.part_o + (slot(i) * (D / 4) + col / 4) * R + rr;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float4 v = src[k * R];
      o[k].x = fmaf(w, v.x, o[k].x); o[k].y = fmaf(w, v.y, o[k].y); o[k].z = fmaf(w, v.z, o[k].z); o[k].w = fmaf(w, v.w, o[k].w);
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  uint4 x[2];
  uint32_t* xp = reinterpret_cast<uint32_t*>(x);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    xp[2 * k] = mma::pack<T>(o[k].x * inv, o[k].y * inv);
    xp[2 * k + 1] = mma::pack<T>(o[k].z * inv, o[k].w * inv);
  }
  uint4* dst = reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.a.out) + row * D + col);
  dst[0] = x[0];
  dst[1] = x[1];
  if (p.a.lse && blockIdx.z == 0 && warp == 0) p.a.lse[row] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2;
}

size_t up256(size_t x) { return (x + 255) / 256 * 256; }

struct Plan {
  Tiling t;
  int per_row, grid;           // grid: workers, a CTA each (D <= 128) or a pair of CTAs
  size_t part_ml, part_o, total;
};
Plan plan_of(int B, int Hq, int Hkv, int T, int D, int N) {
  Plan x;
  x.t = tiling_of(Hq, Hkv);
  x.per_row = (T + 2 * x.t.Tt - 1) / (2 * x.t.Tt);
  const long long tiles = (long long)B * Hkv * x.t.GC * x.per_row * ((N + kKeys - 1) / kKeys);
  int most = D == 256 ? sm_count() / 2 : sm_count();
  if (most > kMaxGrid) most = kMaxGrid;
  x.grid = (int)(tiles < most ? tiles : most);
  x.part_ml = up256((size_t)2 * x.grid * 256 * sizeof(float2));
  x.part_o = up256((size_t)2 * x.grid * 256 * D * 4);
  x.total = ranges_bytes(B, x.per_row, x.grid) + x.part_ml + x.part_o;
  return x;
}

template <typename T, int D>
int32_t launch_typed(const CacheArgs& a, cudaStream_t stream) {
  using C = Cfg<D>;
  const Plan x = plan_of(a.B, a.Hq, a.Hkv, a.T, D, a.N);
  PromptParams p{};
  p.a = a;
  p.t = x.t;
  p.ranges = Ranges{a.B, a.Hkv * x.t.GC, x.per_row, x.grid, nullptr, nullptr, nullptr};
  p.box = box_rows(a);
  p.scale_log2 = a.scale * kLog2e;
  p.out32 = (reinterpret_cast<uintptr_t>(a.out) & 31) == 0;
  uint8_t* ws = ranges_at(p.ranges, reinterpret_cast<uint8_t*>(a.workspace));
  p.part_ml = reinterpret_cast<float2*>(ws);
  p.part_o = reinterpret_cast<float4*>(ws + x.part_ml);
  CUtensorMap mq, mk, mv;
  CUresult r = encode_q(&mq, a, x.t);
  if (r == CUDA_SUCCESS) r = encode_kv(&mk, a.k, a, p.box < C::k_rows ? p.box : C::k_rows);
  if (r == CUDA_SUCCESS) r = encode_kv(&mv, a.v, a, p.box);
  if (r != CUDA_SUCCESS) { set_error("prompt_sdpa: cuTensorMapEncodeTiled failed with CUresult %d", (int)r); return DFLASH_ERR_CUDA; }
  if (!ranges_fit(a.B, x.per_row)) { set_error("prompt_sdpa: unsupported: more than 2^30 units of work"); return DFLASH_ERR_UNSUPPORTED; }
  auto kernel = prompt_kernel<T, D>;
  static std::atomic<uint64_t> ready{0};
  DFLASH_CUDA_CHECK(allow_shared(ready, kernel, C::total));
  // the register hand-over waits for good if the launch gives the CTA fewer than it takes
  static const int regs = [&] { cudaFuncAttributes f; return cudaFuncGetAttributes(&f, kernel) == cudaSuccess ? f.numRegs : 0; }();
  if (regs != C::regs_launch) { set_error("prompt_sdpa: the kernel is launched with %d registers a thread, %d expected", regs, C::regs_launch); return DFLASH_ERR_CUDA; }
  plan_kernel<<<1, 1024, 0, stream>>>(p);
  DFLASH_LAUNCH_CHECK();
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 2;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = C::PAIR ? 2 : 1;
  cfg.stream = stream;
  cfg.gridDim = dim3(x.grid * (C::PAIR ? 2 : 1));
  cfg.blockDim = dim3(C::threads);
  cfg.dynamicSmemBytes = C::total;
  DFLASH_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, mq, mk, mv, p));
  cfg.numAttrs = 1;
  cfg.gridDim = dim3(x.grid, 8, D / 64);
  cfg.blockDim = dim3(128);
  cfg.dynamicSmemBytes = 0;
  DFLASH_CUDA_CHECK(cudaLaunchKernelEx(&cfg, join_kernel<T, D>, p));
  count_launch(3);
  return DFLASH_OK;
}

template <typename T>
int32_t launch_dims(const CacheArgs& a, cudaStream_t s) {
  if (a.D == 64) return launch_typed<T, 64>(a, s);
  if (a.D == 128) return launch_typed<T, 128>(a, s);
  return launch_typed<T, 256>(a, s);
}

}  // namespace

size_t prompt_workspace_bytes(int B, int Hq, int Hkv, int T, int D, int N) { return plan_of(B, Hq, Hkv, T, D, N).total; }

int32_t launch_prompt(const CacheArgs& a, cudaStream_t stream) {
  return a.dtype == DFLASH_BF16 ? launch_dims<__nv_bfloat16>(a, stream) : launch_dims<__half>(a, stream);
}

}  // namespace dflash
