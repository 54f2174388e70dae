// The weight that cached tokens receive from queries whose log-sum-exp is known:
//     mass[b, h, n] += sum over the rows r of h's query heads that see n of 2^(scale log2(e) q_r . k_n - log2(e) lse_r)
//
// Computed as S^T = K Q^T on the tensor cores (tcgen05): 128 keys are the lanes of tensor memory and 128 query rows its
// columns, so that the sum over rows stays inside a thread and nothing is reduced across lanes; two threads share a key.
// A unit of work is 256 keys (two key tiles), its steps are the query tiles that see some of them.  Few rows (a verify
// block, the last rows of a prompt: one query tile): every key is read once and used by 128 rows, bound by HBM; the query
// tile stays in shared memory and keys stream.  Many rows: 2 D operations and one exponential a pair of row and key, bound by
// the 16 exponentials a clock of an SM (1024 clocks a tile against 512 of products at D = 128); the keys stay and query
// tiles stream, each used for both key tiles: with one key tile they took 32 KiB from L2 every 1000 clocks, and L2 set the pace.
//
// Warps: 0 loads keys and queries, 1 the rows' -log2(e) lse, 2 issues the products, 3 walks the steps, 4-11
// sum the first key tile, 12-19 the second.  Four score buffers in tensor memory let the products run a step ahead.  Units
// are cut into equal ranges per CTA (ranges.cuh); pieces of a cut unit leave 256 sums in the workspace, added in order by
// mass_join_kernel: the order of every sum is fixed.
//
// Measured (B200, the whole call): 2048 rows of 32 / 8 heads over 16384 tokens, D = 128, 0.385 ms = 0.67 PFLOP/s; 1.0e9
// exponentials take 0.24 ms at 16 a clock and SM.  16 rows of 32 sequences of 1.4 to 4.1 thousand tokens, D = 256: 35 us, the 94 MB
// take 14 at the HBM's rate; the plan and the start of the CTAs are behind most of the rest.  2048 rows of 16 / 2 heads over 16384
// tokens, D = 256, 0.31 ms = 0.82 PFLOP/s: its ring holds one query tile, whose successor loads when the last product has read it.
#include "ranges.cuh"
#include "tc_common.cuh"

namespace dflash {
namespace {

using namespace tc;

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kUnitCost = 1;                 // what a unit costs besides its query tiles
constexpr int kSumWarps = 16, kThreads = 128 + kSumWarps * 32;
constexpr int kUnitKeys = 2 * kKeys;
constexpr int kBuffers = 4;                  // steps whose log-sum-exps are in shared memory; score buffers of two steps
constexpr int kRing = 16;                    // steps that are described ahead

struct MassParams {
  CacheArgs a;
  Tiling t;
  Ranges ranges;               // rows of key tiles
  int box, k_stages, q_stages; // stages of keys and of queries in shared memory
  float scale_log2;
  float* part;                 // [2 * grid][256]
  int* nan_seen;               // a row in use has an lse of NaN
};

// One step: a key tile against a query tile.
// the first step of a unit; another query tile than before; the last step of the unit; of the query tile; one key tile; no step
enum : int { kNewKeys = 1, kNewQueries = 2, kLast = 4, kQueriesLast = 8, kOneTile = 16, kEnd = 32 };
struct __align__(16) Step {
  int b, h, n0, gc;
  int t0, keys, rows, flags;   // t0: first token of the query tile; the sequence's lengths
  int slot, pad[3];            // of the unit (see RangeWalker::take)
};

template <int D> struct Cfg {
  static constexpr int NC = D / 64;
  // Stages of two chunks (one at D = 64), of keys and queries together: a wait and an issue for every 8 products.  (For
  // every 4 the issuing warp was the slowest part: 470 us for 411.)
  static constexpr int SC = NC < 2 ? NC : 2, NS = NC / SC, stages = 12 / SC, stage = SC * kChunk;
  static constexpr int bars = stages * stage;
  static constexpr int b_full = 0, b_empty = stages, b_s_full = 2 * stages, b_s_free = b_s_full + 4, b_z_full = b_s_free + 4,
                       b_z_free = b_z_full + kBuffers, b_step = b_z_free + kBuffers, b_meet = b_step + kRing, n_bars = b_meet + 2;
  static constexpr int misc = bars + (8 * n_bars + 15) / 16 * 16;
  static constexpr int z = misc + 16;                       // [kBuffers][128] -log2(e) lse of the rows
  static constexpr int sums = z + kBuffers * 128 * 4;       // [2 key tiles][2][2 halves][128]
  static constexpr int steps = sums + 2 * 2 * 2 * 128 * 4;  // [kRing] Step
  static constexpr int total = steps + kRing * (int)sizeof(Step);
};
static_assert(Cfg<256>::total <= 232448 && Cfg<128>::total <= 232448 && Cfg<64>::total <= 232448, "shared memory");

// Place in a ring of a length known at run time: stage and round by counting, not by division.
struct RingAt {
  int stage = 0;
  uint32_t round = 0;
  __device__ void next(int stages, int by = 1) {
    stage += by;
    if (stage >= stages) { stage -= stages; ++round; }
  }
};

// query tokens of sequence (len) that see some key of [n0, n0 + 256): first and last; last < first: none
struct Seeing { int first, last; };
__device__ __forceinline__ Seeing seeing(const CacheArgs& a, RowLens len, int n0) {
  const int past = len.keys - len.rows, n1 = (n0 + kUnitKeys < len.keys ? n0 + kUnitKeys : len.keys) - 1;
  Seeing s{n0 > past ? n0 - past : 0, len.rows - 1};
  if (a.window > 0 && n0 >= a.sinks && n1 + a.window - 1 - past < s.last) s.last = n1 + a.window - 1 - past;
  if (n1 < n0) s.last = -1;
  return s;
}
// query tiles (times head groups) of a unit
__device__ __forceinline__ int unit_steps(const CacheArgs& a, const Tiling& t, RowLens len, int u) {
  const Seeing s = seeing(a, len, u * kUnitKeys);
  return s.last < s.first ? 0 : t.GC * (s.last / t.Tt - s.first / t.Tt + 1);
}
// first unit at or behind u that is seen
__device__ __forceinline__ int next_unit(const CacheArgs& a, RowLens len, int u, int per_row) {
  const int tiles = (len.keys + kUnitKeys - 1) / kUnitKeys;
  if (len.rows == 0 || u >= tiles) return per_row;
  const int past = len.keys - len.rows;
  const int lo = a.window > 0 && past - a.window + 1 > 0 ? (past - a.window + 1) / kUnitKeys : 0;   // of the first row's window
  const int sinks = a.window > 0 ? (a.sinks + kUnitKeys - 1) / kUnitKeys : 0;
  if (u >= sinks && u < lo) u = lo;
  return u < tiles ? u : per_row;
}

__global__ void __launch_bounds__(1024) mass_plan_kernel(const MassParams p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (threadIdx.x == 0) *p.nan_seen = 0;
  plan_ranges<kUnitCost>(p.ranges, p.a, [&](RowLens len, int u) { return unit_steps(p.a, p.t, len, u); });
}

struct Steps {
  const MassParams& p;
  RangeWalker w;
  Step s;
  int tt0, per_gc, i, hi;      // first query tile and query tiles per head group of the unit; step, end
  bool any;
  __device__ Steps(const MassParams& p_, int worker) : p(p_), w(p_.ranges, p_.a, worker), i(0), hi(0), any(false) {}
  __device__ bool next() {
    const int b = s.b, h = s.h, gc = s.gc, t0 = s.t0;
    int flags = ++i >= hi || !any ? kNewKeys : 0;
    if (flags) {
      if (!w.find([&](RowLens len, int u) {
            u = next_unit(p.a, len, u, p.ranges.per_row);
            while (u < p.ranges.per_row && unit_steps(p.a, p.t, len, u) == 0) u = next_unit(p.a, len, u + 1, p.ranges.per_row);
            return u;
          }, i)) return false;
      s.b = w.c.b;
      s.h = w.c.hg;
      s.keys = w.c.len.keys;
      s.rows = w.c.len.rows;
      s.n0 = w.c.u * kUnitKeys;
      const Seeing x = seeing(p.a, w.c.len, s.n0);
      tt0 = x.first / p.t.Tt;
      per_gc = x.last / p.t.Tt - tt0 + 1;
      hi = w.take(i, p.t.GC * per_gc, s.slot);
    }
    s.gc = p.t.GC == 1 ? 0 : i / per_gc;
    s.t0 = (tt0 + i - s.gc * per_gc) * p.t.Tt;
    if (!any || b != s.b || h != s.h || gc != s.gc || t0 != s.t0) flags |= kNewQueries;
    if (i == hi - 1) flags |= kLast;
    if (s.n0 + kKeys >= s.keys) flags |= kOneTile;
    s.flags = flags;
    any = true;
    return true;
  }
};

__device__ __forceinline__ uint32_t bits_below(int n) {     // bits [0, n), n clamped to [0, 32]
  return n <= 0 ? 0u : (n >= 32 ? 0xffffffffu : (1u << n) - 1u);
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1)
mass_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const MassParams p) {
  using C = Cfg<D>;
  constexpr int NS = C::NS, SC = C::SC;
  extern __shared__ __align__(1024) uint8_t sm[];
  const CacheArgs& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + C::bars);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sm + C::misc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(sm + C::misc + 4);
  int* nan_flag = reinterpret_cast<int*>(sm + C::misc + 8);
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (threadIdx.x == 0) {
    ptx::prefetch_tensormap(&map_q);
    ptx::prefetch_tensormap(&map_k);
    for (int i = 0; i < C::n_bars; ++i)
      ptx::mbar_init(&bars[i], (i >= C::b_s_free && i < C::b_z_full) || i >= C::b_meet ? kSumWarps / 2 : (i >= C::b_z_free && i < C::b_step ? kSumWarps : 1));
    *abort_flag = (ptx::smem_u32(sm) & 1023u) != 0u;      // swizzled tiles need 1024-byte alignment; never seen violated
    if (*abort_flag) atomicExch(a.status, kStatusSmemAlign);
    *nan_flag = 0;
    ptx::fence_mbar_init();
  }
  // rows of a query tile behind Gt * Tt are never loaded: zeros, so that their scores are numbers
  const int q0 = p.k_stages;                   // first stage of the queries' ring
  if (p.t.Gt * p.t.Tt < kRows) {
    for (int e = threadIdx.x; e < p.q_stages * C::stage / 16; e += kThreads) *reinterpret_cast<uint4*>(sm + q0 * C::stage + e * 16) = make_uint4(0, 0, 0, 0);
    ptx::fence_proxy_async();
  }
  if (warp == 2) {
    ptx::tmem_alloc(tmem_slot, 512);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  asm volatile("griddepcontrol.wait;" ::: "memory");     // the plan
  const uint32_t tmem = *tmem_slot;
  // A wait that gives up raises the abort flag, after which every wait returns at once: the roles run through their loops
  // without results, meet at the end and leave.
  // Every wait is made by a whole warp.  wait(): its lanes agree on the outcome, none leaves a loop that the others stay in;
  // wait_lane(): where the outcome decides nothing, or the lanes agree on it behind the next wait.
  auto wait_lane = [&](int bar, uint32_t parity) { return ptx::mbar_wait_or_abort(&bars[bar], parity, abort_flag, a.status, kStatusMbarWait); };
  auto wait = [&](int bar, uint32_t parity) { return __all_sync(0xffffffffu, wait_lane(bar, parity)); };
  // Warp 3 walks the CTA's steps and describes them in a ring; the others read.  (Every role walking for itself was five
  // copies of that code: an eighth of the instruction fetches missed and each step took 2350 clocks.)
  Step* ring = reinterpret_cast<Step*>(sm + C::steps);
  auto step_at = [&](uint32_t n) {                            // step n; flags = kEnd behind the last
    Step x;
    if (!wait(C::b_step + n % kRing, (n / kRing) & 1)) { x.flags = kEnd; return x; }
    const int4* src = reinterpret_cast<const int4*>(&ring[n % kRing]);
    int4* dst = reinterpret_cast<int4*>(&x);
    dst[0] = src[0];
    dst[1] = src[1];
    dst[2] = src[2];
    return x;
  };

  if (warp == 0) {
    // ------------------------------- keys and queries -------------------------------
    RingAt k, q;
    const int pieces = kKeys / p.box, q_bytes = SC * p.t.Gt * p.t.Tt * 128;
    bool ok = __all_sync(0xffffffffu, !*abort_flag);
    for (uint32_t n = 0; ok; ++n) {
      const Step s = step_at(n);
      if (s.flags & kEnd) break;
      if (s.flags & kNewKeys) {
        const int uses = (s.flags & kOneTile ? 1 : 2) * NS;
        const TilePlace x0 = place_of(a, s.b, s.n0 + lane * p.box, lane < 2 * pieces ? s.keys : 0);   // lane i: box i of the unit
        for (int i = 0; i < uses; ++i) {
          const int tile = i / NS, c0 = i % NS * SC;
          if (k.round > 0) ok = wait(C::b_empty + k.stage, (k.round - 1) & 1);
          if (!ok) break;
          if (lane == 0) ptx::mbar_arrive_expect_tx(&bars[C::b_full + k.stage], C::stage);
          __syncwarp();
          const int box = lane - tile * pieces;
          if (box >= 0 && box < pieces)
            for (int c = 0; c < SC; ++c)
              ptx::tma_load_4d(sm + k.stage * C::stage + c * kChunk + box * p.box * 128, &map_k, (c0 + c) * 64, x0.row, s.h, x0.outer, &bars[C::b_full + k.stage]);
          __syncwarp();
          k.next(p.k_stages);
        }
        if (!ok) break;
      }
      if (s.flags & kNewQueries) {
        for (int i = 0; i < NS; ++i) {
          if (q.round > 0) ok = wait(C::b_empty + q0 + q.stage, (q.round - 1) & 1);
          if (!ok) break;
          if (lane == 0) ptx::mbar_arrive_expect_tx(&bars[C::b_full + q0 + q.stage], q_bytes);
          __syncwarp();
          if (lane < SC)
            ptx::tma_load_4d(sm + (q0 + q.stage) * C::stage + lane * kChunk, &map_q, (i * SC + lane) * 64, s.gc * p.t.Gt, s.t0, s.b * a.Hkv + s.h, &bars[C::b_full + q0 + q.stage]);
          __syncwarp();
          q.next(p.q_stages);
        }
      }
    }
  } else if (warp == 3) {
    // ------------------------------------- steps -------------------------------------
    // A slot is written again when the sums of sixteen steps ago are done; those of twelve ago are waited for, in order.
    Steps st(p, blockIdx.x);
    bool more = st.next(), ok = true;
    for (uint32_t n = 0; ok; ++n) {
      Step s = st.s;
      if (!more) s.flags = kEnd;
      else {
        more = st.next();
        if (!more || (st.s.flags & kNewQueries)) s.flags |= kQueriesLast;
      }
      if (n >= kRing - kBuffers) {
        const uint32_t done = n - (kRing - kBuffers);
        ok = wait(C::b_z_free + done % kBuffers, (done / kBuffers) & 1);
      }
      if (lane == 0) {
        ring[n % kRing] = s;
        ptx::mbar_arrive(&bars[C::b_step + n % kRing]);
      }
      __syncwarp();
      if (s.flags & kEnd) break;
    }
  } else if (warp == 1) {
    // --------------------------------- log-sum-exp ----------------------------------
    float* z = reinterpret_cast<float*>(sm + C::z);
    long long off[4];                                         // lane i has the rows 4 i ... 4 i + 3 of a query tile
    int tok[4], head[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = lane * 4 + i;
      head[i] = r < p.t.Gt * p.t.Tt ? r % p.t.Gt : p.t.G;     // G: no such head
      tok[i] = r / p.t.Gt;
      off[i] = (long long)head[i] * a.T + tok[i];
    }
    auto fetch = [&](uint32_t n, float (&v)[4]) {             // false: there is no step n
      const Step s = step_at(n);
      if (s.flags & kEnd) return false;
      const float* base = a.lse + ((long long)s.b * a.Hq + s.h * p.t.G + s.gc * p.t.Gt) * a.T + s.t0;
#pragma unroll
      for (int i = 0; i < 4; ++i)                             // rows not in use add nothing
        v[i] = s.gc * p.t.Gt + head[i] < p.t.G && s.t0 + tok[i] < s.rows ? base[off[i]] : -INFINITY;
      return true;
    };
    float v[kBuffers][4];                                     // values on their way
    uint32_t have = 0;
#pragma unroll
    for (int i = 0; i < kBuffers - 1; ++i)
      if (have == (uint32_t)i && fetch(i, v[i])) ++have;
    bool ok = true, more = have == kBuffers - 1;
    for (uint32_t n0 = 0; ok && n0 < have; n0 += kBuffers) {
#pragma unroll
      for (int k = 0; k < kBuffers; ++k) {
        const uint32_t n = n0 + k;
        if (!ok || n >= have) break;
        if (more) {
          more = fetch(n + kBuffers - 1, v[(k + kBuffers - 1) % kBuffers]);
          have += more;
        }
        if (n >= kBuffers) ok = wait(C::b_z_free + k, (n / kBuffers - 1) & 1);
        // Neither do rows that see nothing (their lse is -infinity), nor those whose lse is NaN: it would reach the keys that the
        // row does not see, by way of their score of -infinity.  mass_join_kernel marks what such rows see.
        if (v[k][0] != v[k][0] || v[k][1] != v[k][1] || v[k][2] != v[k][2] || v[k][3] != v[k][3]) *nan_flag = 1;
        float4 x;
        x.x = v[k][0] > -INFINITY ? -v[k][0] * kLog2e : -INFINITY;
        x.y = v[k][1] > -INFINITY ? -v[k][1] * kLog2e : -INFINITY;
        x.z = v[k][2] > -INFINITY ? -v[k][2] * kLog2e : -INFINITY;
        x.w = v[k][3] > -INFINITY ? -v[k][3] * kLog2e : -INFINITY;
        *reinterpret_cast<float4*>(z + k * 128 + lane * 4) = x;
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(&bars[C::b_z_full + k]);
      }
    }
  } else if (warp == 2) {
    // ---------------------------------- S^T = K Q^T ----------------------------------
    constexpr uint32_t kI = idesc<T>(kKeys, kRows, false);
    RingAt k, q, k_unit, q_tile;                              // the chunks to come; those of the unit and query tile in use
    uint32_t used = 0;                                        // second key tile's two score buffers: bits 0, 1 in use, bits 2, 3 the phase
    const uint32_t base = ptx::smem_u32(sm);
    bool ok = true;
    for (uint32_t n = 0; ok; ++n) {
      ok = wait(C::b_step + n % kRing, (n / kRing) & 1);
      const int flags = ok ? ring[n % kRing].flags : kEnd;
      if (flags & kEnd) break;
      const int tiles = flags & kOneTile ? 1 : 2;
      if (flags & kNewKeys) { k_unit = k; k.next(p.k_stages, tiles * NS); }
      if (flags & kNewQueries) { q_tile = q; q.next(p.q_stages, NS); }
      RingAt ka = k_unit;
#pragma unroll 1
      for (int tile = 0; ok && tile < tiles; ++tile) {
        const uint32_t buf = (n & 1) * 2 + tile, par = n & 1;
        if (tile == 0) {
          if (n >= 2) ok = wait_lane(C::b_s_free + buf, ((n >> 1) - 1) & 1);
        } else {
          if (used >> par & 1) ok = wait_lane(C::b_s_free + buf, used >> (2 + par) & 1);
          used = (used ^ (used >> par & 1) << (2 + par)) | 1u << par;
        }
        RingAt qa = q_tile;
#pragma unroll
        for (int i = 0; i < NS; ++i) {
          // a stage of new queries (keys) is used as soon as it is there
          if ((flags & kNewQueries) && tile == 0) ok &= wait_lane(C::b_full + q0 + qa.stage, qa.round & 1);
          if (flags & kNewKeys) ok &= wait_lane(C::b_full + ka.stage, ka.round & 1);
          if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
          ptx::tc_fence_after();
          if (ptx::elect_one()) {
            const uint32_t d = tmem + buf * 128, k_addr = base + ka.stage * C::stage, q_addr = base + (q0 + qa.stage) * C::stage;
#pragma unroll
            for (int c = 0; c < SC; ++c) {
              const uint64_t da = make_desc(k_addr + c * kChunk, 16, 1024), db = make_desc(q_addr + c * kChunk, 16, 1024);
#pragma unroll
              for (int kk = 0; kk < 4; ++kk) ptx::umma_ss(d, da + 2 * kk, db + 2 * kk, kI, i + c + kk > 0);
            }
            if (i == NS - 1) ptx::umma_commit(&bars[C::b_s_full + buf]);
            if (flags & kLast) ptx::umma_commit(&bars[C::b_empty + ka.stage]);
            if ((flags & kQueriesLast) && tile == tiles - 1) ptx::umma_commit(&bars[C::b_empty + q0 + qa.stage]);
          }
          __syncwarp();
          ka.next(p.k_stages);
          qa.next(p.q_stages);
        }
      }
    }
  } else if (warp >= 4) {
    // ------------------------------------- sums --------------------------------------
    const int wq = warp & 3, tile = (warp - 4) >> 3, half = ((warp - 4) >> 2) & 1;    // wq: tensor-memory lane quarter
    const int key = wq * 32 + lane;
    const float* z = reinterpret_cast<const float*>(sm + C::z);
    float* sums = reinterpret_cast<float*>(sm + C::sums) + tile * 512;
    uint32_t phase = 0, units = 0;                            // phase bits of this tile's two score buffers
    float2 acc[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
    float before = 0.f;
    for (uint32_t n = 0;; ++n) {
      const Step s = step_at(n);
      if (s.flags & kEnd) break;
      const uint32_t zb = n % kBuffers;
      // waited for by the warps that have no tile here too: running ahead, they would arrive twice in one phase of z_free
      wait_lane(C::b_z_full + zb, (n / kBuffers) & 1);
      if (tile == 0 || !(s.flags & kOneTile)) {
        const int n0 = s.n0 + tile * kKeys, nn = n0 + key;
        float* out = a.mass + ((long long)s.b * a.Hkv + s.h) * a.mass_stride + nn;
        const bool writer = half == 0 && nn < s.keys;
        if (s.flags & kNewKeys) {
          acc[0] = acc[1] = make_float2(0.f, 0.f);
          if (writer && s.slot < 0) before = *out;            // wanted at the unit's end
        }
        const int buf = (n & 1) * 2 + tile;
        wait_lane(C::b_s_full + buf, phase >> (n & 1) & 1);
        phase ^= 1u << (n & 1);
        __syncwarp();
        ptx::tc_fence_after();
        const int p0 = s.keys - s.rows + s.t0, p1 = p0 + p.t.Tt - 1;              // positions of the tile's tokens
        const bool whole = n0 + kKeys - 1 <= p0 && (a.window == 0 || n0 > p1 - a.window || n0 + kKeys <= a.sinks) && s.t0 + p.t.Tt <= s.rows;
        // otherwise rows [lo, hi) of the tile see this key: the tokens from it on, up to a window behind it, that are in use
        int lo = nn - p0, hi = p.t.Tt < s.rows - s.t0 ? p.t.Tt : s.rows - s.t0;
        if (a.window > 0 && nn >= a.sinks && nn + a.window - p0 < hi) hi = nn + a.window - p0;
        lo = lo < 0 ? 0 : (lo > kRows ? kRows : lo);
        hi = hi < 0 ? 0 : hi;
#pragma unroll 1
        for (int col = half * 64; col < half * 64 + 64; col += 32) {
          uint32_t x[32];
          ptx::tmem_ld32(tmem + ((uint32_t)(wq * 32) << 16) + buf * 128 + col, x);
          ptx::tmem_ld_wait();
          if (!whole) {
            const uint32_t seen = bits_below(hi * p.t.Gt - col) & ~bits_below(lo * p.t.Gt - col);
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (!((seen >> i) & 1u)) x[i] = 0xff800000u;    // -infinity
          }
          const float4* zp = reinterpret_cast<const float4*>(z + zb * 128 + col);
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            const float4 zi = zp[i / 4];
            float2 u = fma2v(__uint_as_float(x[i]), __uint_as_float(x[i + 1]), p.scale_log2, zi.x, zi.y);
            float2 w = fma2v(__uint_as_float(x[i + 2]), __uint_as_float(x[i + 3]), p.scale_log2, zi.z, zi.w);
            u.x = mma::exp2_approx(u.x); u.y = mma::exp2_approx(u.y);
            w.x = mma::exp2_approx(w.x); w.y = mma::exp2_approx(w.y);
            acc[0] = add2(acc[0], u);
            acc[1] = add2(acc[1], w);
          }
        }
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(&bars[C::b_s_free + buf]);
        if (s.flags & kLast) {
          // a key's two threads; the slot of two units ago was read before the last unit's meeting
          float* slot = sums + (units & 1) * 256;
          slot[half * 128 + key] = (acc[0].x + acc[0].y) + (acc[1].x + acc[1].y);
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive(&bars[C::b_meet + tile]);
          // a bounded wait: after one that gave up, a tile's warps may be at different steps
          if (wait(C::b_meet + tile, units++ & 1)) {
            const float total = slot[key] + slot[128 + key];
            if (half == 0 && s.slot >= 0) p.part[(long long)s.slot * kUnitKeys + tile * kKeys + key] = total;
            else if (writer) *out = before + total;
          }
        }
      }
      if (lane == 0) ptx::mbar_arrive(&bars[C::b_z_free + zb]);
      __syncwarp();
    }
  }
  __syncwarp();
  __syncthreads();
  if (threadIdx.x == 0 && *nan_flag) *p.nan_seen = 1;
  if (*abort_flag) __nanosleep(100000);        // copies that were still in flight land before the memory is given back
  if (warp == 2) ptx::tmem_dealloc(tmem, 512);
}

// does a row that sees key n of (b, h) have an lse of NaN?
__device__ __forceinline__ bool nan_row(const MassParams& p, int b, int h, RowLens len, int n) {
  const CacheArgs& a = p.a;
  const int past = len.keys - len.rows, first = n > past ? n - past : 0;
  int end = len.rows;
  if (a.window > 0 && n >= a.sinks && n + a.window - past < end) end = n + a.window - past;
  const float* lse = a.lse + ((long long)b * a.Hq + h * p.t.G) * a.T;
  for (int g = 0; g < p.t.G; ++g, lse += a.T)
    for (int i = first; i < end; ++i)
      if (lse[i] != lse[i]) return true;
  return false;
}

// Adds up the pieces of a cut unit, in order.  Where some row has an lse of NaN, which a working program never meets, every key
// is looked at again here, for all rows that see it: done by the summing threads of mass_kernel it cost every call 2 to 5 %
// (387 to 400 us for 381 in 2048 rows over 16384 tokens, with bits of such rows beside each step's log-sum-exps or a flag a unit; 385 so).
__global__ void __launch_bounds__(kUnitKeys) mass_join_kernel(const MassParams p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const Cut cut = p.ranges.cuts[blockIdx.x];
  const bool nan = *p.nan_seen != 0;
  auto at = [&](const Cursor& c, int n) { return p.a.mass + ((long long)c.b * p.a.Hkv + c.hg) * p.a.mass_stride + n; };
  if (cut.count > 0) {
    const Cursor c(p.ranges, p.a, cut.unit);
    const int n = c.u * kUnitKeys + threadIdx.x;
    if (n < c.len.keys) {
      float total = 0.f;
      for (int i = 0; i < cut.count; ++i) total += p.part[(long long)piece_slot(cut, i) * kUnitKeys + threadIdx.x];
      if (nan && nan_row(p, c.b, c.hg, c.len, n)) total = __int_as_float(0x7fffffff);
      *at(c, n) += total;
    }
  }
  if (!nan) return;
  const long long units = (long long)p.a.B * p.a.Hkv * p.ranges.per_row;
  for (long long unit = blockIdx.x; unit < units; unit += gridDim.x) {
    bool is_cut = false;                       // another block adds to it
    for (int i = 0; i < p.ranges.grid; ++i) is_cut |= p.ranges.cuts[i].count > 0 && p.ranges.cuts[i].unit == unit;
    const Cursor c(p.ranges, p.a, unit);
    const int n = c.u * kUnitKeys + threadIdx.x;
    if (!is_cut && n < c.len.keys && nan_row(p, c.b, c.hg, c.len, n)) *at(c, n) = __int_as_float(0x7fffffff);
  }
}

struct Plan { Tiling t; int per_row, grid; size_t total; };
Plan plan_of(int B, int Hq, int Hkv, int T, int N) {
  Plan x;
  x.t = tiling_of(Hq, Hkv);
  x.per_row = (N + kUnitKeys - 1) / kUnitKeys;
  const long long tiles = (long long)B * Hkv * x.per_row * x.t.GC * ((T + x.t.Tt - 1) / x.t.Tt);
  const int n_sm = sm_count(), most = n_sm < kMaxGrid ? n_sm : kMaxGrid;
  x.grid = (int)(tiles < most ? tiles : most);
  x.total = ranges_bytes(B, x.per_row, x.grid) + (size_t)2 * x.grid * kUnitKeys * 4 + 16;
  return x;
}

template <typename T, int D>
int32_t launch_typed(const CacheArgs& a, cudaStream_t stream) {
  using C = Cfg<D>;
  const Plan x = plan_of(a.B, a.Hq, a.Hkv, a.T, a.N);
  MassParams p{};
  p.a = a;
  p.t = x.t;
  p.ranges = Ranges{a.B, a.Hkv, x.per_row, x.grid, nullptr, nullptr, nullptr};
  p.box = box_rows(a);
  // one query tile in all: it stays, keys stream; else queries stream past two key tiles
  const bool one = x.t.GC == 1 && a.T <= x.t.Tt;
  p.q_stages = one ? C::NS : C::stages - 2 * C::NS;
  p.k_stages = C::stages - p.q_stages;
  p.scale_log2 = a.scale * kLog2e;
  p.part = reinterpret_cast<float*>(ranges_at(p.ranges, reinterpret_cast<uint8_t*>(a.workspace)));
  p.nan_seen = reinterpret_cast<int*>(p.part + (size_t)2 * x.grid * kUnitKeys);
  CUtensorMap mq, mk;
  CUresult r = encode_q(&mq, a, x.t);
  if (r == CUDA_SUCCESS) r = encode_kv(&mk, a.k, a, p.box);
  if (r != CUDA_SUCCESS) { set_error("attention_mass: cuTensorMapEncodeTiled failed with CUresult %d", (int)r); return DFLASH_ERR_CUDA; }
  if (!ranges_fit(a.B, x.per_row)) { set_error("attention_mass: unsupported: more than 2^30 units of work"); return DFLASH_ERR_UNSUPPORTED; }
  auto kernel = mass_kernel<T, D>;
  static std::atomic<uint64_t> ready{0};
  DFLASH_CUDA_CHECK(allow_shared(ready, kernel, C::total));
  mass_plan_kernel<<<1, 1024, 0, stream>>>(p);
  DFLASH_LAUNCH_CHECK();
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cfg.stream = stream;
  cfg.gridDim = dim3(x.grid);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = C::total;
  DFLASH_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, mq, mk, p));
  cfg.blockDim = dim3(kUnitKeys);
  cfg.dynamicSmemBytes = 0;
  DFLASH_CUDA_CHECK(cudaLaunchKernelEx(&cfg, mass_join_kernel, p));
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

size_t mass_workspace_bytes(int B, int Hq, int Hkv, int T, int, int N) { return plan_of(B, Hq, Hkv, T, N).total; }

int32_t launch_mass(const CacheArgs& a, cudaStream_t stream) {
  return a.dtype == DFLASH_BF16 ? launch_dims<__nv_bfloat16>(a, stream) : launch_dims<__half>(a, stream);
}

}  // namespace dflash
