// Attention of a prompt (or a chunk of one) over the KV cache on the tensor cores, with a sliding window and leading
// tokens that stay visible.
//
// Mathematics: for every query row the running maximum m and sum l of 2^(s - m) over key tiles of 128, O = sum 2^(s - m) v
// accumulated in tensor memory, rescaled only when the maximum has grown by more than 2^8.  4 T n D operations per head
// against n D elements of keys and values that stay in L2: bound by the tensor pipe and, next to it, by the 128 x 128
// exponentials of a tile (16 a clock per SM, 1024 clocks; a tile's two products take 1024 at D = 128, 2048 at 256).
//
// * A query tile is 128 rows: the heads of one KV head for consecutive tokens (tc_common.cuh).  D <= 128: two query
//   tiles a CTA, each with its score columns and accumulator in tensor memory and a softmax warpgroup (one thread a
//   row); the tiles take turns, one's products run under the other's exponentials, and a key tile is loaded once for both.
//   D = 256: the accumulator takes half of the tensor memory, so one query tile with two score buffers; two threads
//   share a row.
// * Warps: 0 loads queries and keys, 1 values, 2 issues S = Q K^T, 3 issues O += P V (P replaces S in tensor memory,
//   in the inputs' type: the product needs a 16-bit operand), 4-11 softmax.
// * Only the key tiles that some row of the unit sees are visited; only those that some row does not see whole are masked.
//   Value rows behind the sequence's length are zeroed in shared memory before the product, whatever the cache holds there.
// * One persistent CTA per SM.  plan_kernel lays the key tiles of all units in a row and cuts them into equal ranges, so
//   that unequal lengths, causal triangles and few query rows over a long cache all fill the GPU; a cut closer than kMinCut
//   tiles to a unit's edge moves to the edge.  A unit cut in pieces leaves (O, m, l) per piece in the workspace and
//   join_kernel adds them up in order.
#include "tc_common.cuh"

namespace dflash {
namespace {

using namespace tc;

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kRescale = 8.f;              // in log2 units
constexpr int kThreads = 384;
constexpr int kMinCut = 4;
// registers: 384 threads launched with 168 each; what the four helper warps give up the softmax warps take
constexpr int kRegsLaunch = 168, kRegsHelper = 56, kRegsSoftmax = 216;
static_assert(128 * kRegsHelper + 256 * kRegsSoftmax <= kThreads * kRegsLaunch, "register split");

struct Boundary { long long unit; int off, pad; long long pos; };
struct Cut { long long unit; int first, count; };

struct PromptParams {
  CacheArgs a;
  Tiling t;
  int NTT;                     // units (of NQ query tiles) per (sequence, KV head, head group)
  int box;
  int grid;
  float scale_log2;
  int negate;                  // scale < 0: the scores change sign first
  long long* steps;            // [B * NTT + 1] key tiles in front of every (sequence, unit)
  Boundary* bounds;            // [grid + 1]
  Cut* cuts;                   // [grid]
  float4* part_o;              // [2 * grid][D / 4][128 NQ]
  float2* part_ml;             // [2 * grid][128 NQ]
};

template <int D> struct Cfg {
  static constexpr int NQ = D == 256 ? 1 : 2;               // query tiles
  static constexpr int NC = D / 64;                         // 64-column chunks of a row
  static constexpr int ring = 10;                           // 16 KiB chunks of keys and values
  static constexpr int KS = D == 64 ? 4 : 4, VS = ring - KS;
  static constexpr int q = 0;
  static constexpr int kv = NQ * NC * kChunk;
  static constexpr int bars = kv + ring * kChunk;
  // barriers
  static constexpr int b_q_full = 0, b_q_empty = 1, b_s_full = 2, b_p_full = 4, b_s_free = 6, b_pv_done = 8, b_o_free = 10,
                       b_kv_full = 12, b_kv_empty = 12 + ring, n_bars = 12 + 2 * ring;
  static constexpr int misc = bars + 8 * n_bars;            // tensor-memory base, abort flag
  static constexpr int xch = misc + 16;                     // [2][2][128] row maxima of the two halves (D = 256)
  static constexpr int total = xch + 2 * 2 * 128 * 4;
  // tensor-memory columns: accumulators first, score buffers in the upper half
  __host__ __device__ static constexpr int col_o(int qi) { return qi * 128; }
  __host__ __device__ static constexpr int col_s(int i) { return 256 + i * 128; }
};
static_assert(Cfg<256>::total <= 232448 && Cfg<128>::total <= 232448, "shared memory");

// ---- the plan ----
__device__ __forceinline__ int unit_steps(const PromptParams& p, RowLens len, int tt, int tokens) {
  const int t0 = tt * tokens;
  if (t0 >= len.rows) return 0;
  const int t1 = t0 + tokens < len.rows ? t0 + tokens : len.rows;
  return key_tiles(p.a, len, t0, t1).count;
}

__global__ void __launch_bounds__(1024) plan_kernel(const PromptParams p, int tokens) {
  __shared__ long long warp_sums[32];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const long long E = (long long)p.a.B * p.NTT, HG = (long long)p.a.Hkv * p.t.GC;
  const long long per_thread = (E + 1023) / 1024, e0 = tid * per_thread, e1 = e0 + per_thread < E ? e0 + per_thread : E;
  long long mine = 0;
  int b = -1;
  RowLens len{0, 0};
  for (long long e = e0; e < e1; ++e) {
    const int eb = (int)(e / p.NTT);
    if (eb != b) { b = eb; len = lens_of(p.a, b, true); }
    mine += unit_steps(p, len, (int)(e - (long long)b * p.NTT), tokens);
  }
  long long x = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  long long at = x - mine;
  for (int w = 0; w < warp; ++w) at += warp_sums[w];
  b = -1;
  for (long long e = e0; e < e1; ++e) {
    const int eb = (int)(e / p.NTT);
    if (eb != b) { b = eb; len = lens_of(p.a, b); }
    p.steps[e] = at;
    at += unit_steps(p, len, (int)(e - (long long)b * p.NTT), tokens);
  }
  long long all = 0;
  for (int w = 0; w < 32; ++w) all += warp_sums[w];
  if (tid == 0) p.steps[E] = all;
  __syncthreads();               // the table is read by other threads of this block below
  const long long total = all * HG;
  long long per = (total + p.grid - 1) / p.grid;
  if (per < kMinCut) per = kMinCut;
  for (int c = tid; c <= p.grid; c += 1024) {
    long long pos = c * per;
    Boundary r{E * HG, 0, 0, total};
    if (pos < total) {
      int lo = 0, hi = p.a.B - 1;             // the last sequence that starts at or before pos
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (p.steps[(long long)mid * p.NTT] * HG <= pos) lo = mid; else hi = mid - 1;
      }
      const long long base = p.steps[(long long)lo * p.NTT], len_b = p.steps[(long long)(lo + 1) * p.NTT] - base;
      const long long hg = (pos - base * HG) / len_b, rem = pos - base * HG - hg * len_b;
      int ta = 0, tb = p.NTT - 1;             // the last unit that starts at or before rem
      while (ta < tb) {
        const int mid = (ta + tb + 1) >> 1;
        if (p.steps[(long long)lo * p.NTT + mid] - base <= rem) ta = mid; else tb = mid - 1;
      }
      const long long s = p.steps[(long long)lo * p.NTT + ta] - base, e = p.steps[(long long)lo * p.NTT + ta + 1] - base;
      const long long unit = ((long long)lo * HG + hg) * p.NTT + ta;
      const int off = (int)(rem - s), size = (int)(e - s);
      if (off < kMinCut) r = Boundary{unit, 0, 0, pos - off};
      else if (size - off < kMinCut) r = Boundary{unit + 1, 0, 0, pos - off + size};
      else r = Boundary{unit, off, 0, pos};
    }
    p.bounds[c] = r;
  }
  __syncthreads();
  for (int c = tid; c < p.grid; c += 1024) {
    Cut cut{0, 0, 0};
    if (c >= 1 && p.bounds[c].off > 0 && !(p.bounds[c - 1].off > 0 && p.bounds[c - 1].unit == p.bounds[c].unit)) {
      int n = 1;
      while (c + n <= p.grid && p.bounds[c + n].off > 0 && p.bounds[c + n].unit == p.bounds[c].unit) ++n;
      cut = Cut{p.bounds[c].unit, c - 1, n + 1};
    }
    p.cuts[c] = cut;
  }
}

struct Unit {
  int b, h, gc, t0;            // t0: first token of the unit
  RowLens len;
  KeyTiles k;
};
__device__ __forceinline__ Unit unit_at(const PromptParams& p, long long unit, int tokens) {
  Unit u;
  const int HG = p.a.Hkv * p.t.GC;
  const long long bhg = unit / p.NTT;
  u.t0 = (int)(unit - bhg * p.NTT) * tokens;
  u.b = (int)(bhg / HG);
  const int hg = (int)(bhg - (long long)u.b * HG);
  u.h = hg / p.t.GC;
  u.gc = hg - u.h * p.t.GC;
  u.len = lens_of(p.a, u.b);
  const int t1 = u.t0 + tokens < u.len.rows ? u.t0 + tokens : u.len.rows;
  u.k = key_tiles(p.a, u.len, u.t0, t1);
  return u;
}

struct Segment {
  Unit u;
  int lo, hi;                  // key tiles [lo, hi) of u.k
  int nq;                      // query tiles with rows in use
  int slot;                    // -1: the whole unit
};
// the segments of one CTA, in order; every role walks them for itself
template <int NQ>
struct Walker {
  const PromptParams& p;
  long long unit, left;
  int off;
  bool first;
  __device__ explicit Walker(const PromptParams& p_) : p(p_), first(true) {
    const Boundary x = p.bounds[blockIdx.x], y = p.bounds[blockIdx.x + 1];
    unit = x.unit;
    off = x.off;
    left = y.pos - x.pos;
  }
  __device__ bool next(Segment& s) {
    if (left <= 0) return false;
    const int tokens = NQ * p.t.Tt;
    for (;;) {
      s.u = unit_at(p, unit, tokens);
      if (s.u.t0 < s.u.len.rows) break;
      unit = (unit / p.NTT + 1) * p.NTT;       // the rest of this head's units has no rows either
    }
    s.lo = off;
    const int size = s.u.k.count;
    s.hi = left < size - off ? off + (int)left : size;
    s.nq = NQ == 2 && s.u.t0 + p.t.Tt < s.u.len.rows ? 2 : 1;
    s.slot = (s.lo == 0 && s.hi == size) ? -1 : 2 * (int)blockIdx.x + (s.lo > 0 ? 0 : 1);
    left -= s.hi - s.lo;
    off = 0;
    ++unit;
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

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1)
prompt_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
              const __grid_constant__ CUtensorMap map_v, const PromptParams p) {
  using C = Cfg<D>;
  constexpr int NQ = C::NQ, NC = C::NC, KS = C::KS, VS = C::VS;
  extern __shared__ __align__(1024) uint8_t sm[];
  const CacheArgs& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if ((ptx::smem_u32(sm) & 1023u) != 0u) {   // swizzled tiles need 1024-byte alignment; never seen violated
    if (threadIdx.x == 0) atomicExch(a.status, kStatusSmemAlign);
    return;
  }
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + C::bars);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sm + C::misc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(sm + C::misc + 4);
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (threadIdx.x == 0) {
    ptx::prefetch_tensormap(&map_q);
    ptx::prefetch_tensormap(&map_k);
    ptx::prefetch_tensormap(&map_v);
    // arrivals: P and the freed accumulator come from softmax warps (4 a query tile, 8 when two threads share a row)
    for (int i = 0; i < C::n_bars; ++i) {
      const bool soft = (i >= C::b_p_full && i < C::b_p_full + 2) || (i >= C::b_o_free && i < C::b_o_free + 2);
      ptx::mbar_init(&bars[i], soft ? (NQ == 2 ? 4 : 8) : 1);
    }
    *abort_flag = 0;
    ptx::fence_mbar_init();
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
  // A wait that gives up raises the CTA's abort flag, after which every wait returns at once: the roles run through
  // their loops without results, meet at the end and leave.
  auto wait = [&](int bar, uint32_t parity) { return ptx::mbar_wait_or_abort(&bars[bar], parity, abort_flag, a.status, kStatusMbarWait); };

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsHelper));
    Walker<NQ> walk(p);
    Segment s;
    if (warp == 0) {
      // ------------------------------ queries and keys ------------------------------
      uint32_t fill = 0, seg = 0;
      bool ok = true;
      while (ok && walk.next(s)) {
        if (seg > 0) ok = wait(C::b_q_empty, (seg - 1) & 1);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (lane == 0) {
          ptx::mbar_arrive_expect_tx(&bars[C::b_q_full], s.nq * NC * p.t.Gt * p.t.Tt * 128);
          for (int qi = 0; qi < s.nq; ++qi)
            for (int c = 0; c < NC; ++c)
              ptx::tma_load_4d(sm + C::q + (qi * NC + c) * kChunk, &map_q, c * 64, s.u.gc * p.t.Gt, s.u.t0 + qi * p.t.Tt,
                               s.u.b * a.Hkv + s.u.h, &bars[C::b_q_full]);
        }
        __syncwarp();
        for (int j = s.lo; ok && j < s.hi; ++j) {
          const int n0 = tile_key(s.u.k, j);
          for (int c = 0; ok && c < NC; ++c, ++fill) {
            const uint32_t st = fill % KS;
            if (fill >= KS) ok = wait(C::b_kv_empty + st, (fill / KS - 1) & 1);
            ok = __all_sync(0xffffffffu, ok);
            if (ok) load_chunk(sm + C::kv + st * kChunk, &map_k, a, p.box, s.u.b, s.u.h, n0, s.u.len.keys, c * 64, &bars[C::b_kv_full + st], lane);
          }
        }
        ++seg;
      }
    } else if (warp == 1) {
      // ----------------------------------- values -----------------------------------
      uint32_t fill = 0;
      bool ok = true;
      while (ok && walk.next(s)) {
        for (int j = s.lo; ok && j < s.hi; ++j) {
          const int n0 = tile_key(s.u.k, j);
          for (int c = 0; ok && c < NC; ++c, ++fill) {
            const uint32_t st = KS + fill % VS;
            if (fill >= VS) ok = wait(C::b_kv_empty + st, (fill / VS - 1) & 1);
            ok = __all_sync(0xffffffffu, ok);
            if (ok) load_chunk(sm + C::kv + st * kChunk, &map_v, a, p.box, s.u.b, s.u.h, n0, s.u.len.keys, c * 64, &bars[C::b_kv_full + st], lane);
          }
        }
      }
    } else if (warp == 2) {
      // --------------------------------- S = Q K^T ----------------------------------
      constexpr uint32_t kI = idesc<T>(kRows, kKeys, false);
      if (lane == 0) {
        uint32_t drain = 0, seg = 0, n_s[2] = {0, 0};       // n_s: score tiles issued per buffer
        const uint32_t q_addr = ptx::smem_u32(sm + C::q), kv_addr = ptx::smem_u32(sm + C::kv);
        bool ok = true;
        while (ok && walk.next(s)) {
          ok = wait(C::b_q_full, seg & 1);
          ptx::tc_fence_after();
          for (int j = s.lo; ok && j < s.hi; ++j) {
            for (int qi = 0; ok && qi < s.nq; ++qi) {
              // the buffer is free once the product that read P from it has retired
              const int buf = NQ == 2 ? qi : (int)((n_s[0] + n_s[1]) & 1);
              if (n_s[buf] > 0) ok = wait(C::b_s_free + buf, (n_s[buf] - 1) & 1);
              if (!ok) break;
              ptx::tc_fence_after();
              const uint32_t d = tmem + C::col_s(buf);
              for (int c = 0; ok && c < NC; ++c) {
                const uint32_t f = drain + c, st = f % KS;
                if (qi == 0) {
                  ok = wait(C::b_kv_full + st, (f / KS) & 1);
                  ptx::tc_fence_after();
                }
                const uint64_t da = make_desc(q_addr + (qi * NC + c) * kChunk, 16, 1024), db = make_desc(kv_addr + st * kChunk, 16, 1024);
                if (c == 0) ptx::umma_ss_first(d, da, db, kI);
                else ptx::umma_ss_acc(d, da, db, kI);
                ptx::umma_ss_acc(d, da + 2, db + 2, kI);
                ptx::umma_ss_acc(d, da + 4, db + 4, kI);
                ptx::umma_ss_acc(d, da + 6, db + 6, kI);
                if (qi == s.nq - 1) ptx::umma_commit(&bars[C::b_kv_empty + st]);
              }
              ptx::umma_commit(&bars[C::b_s_full + buf]);
              ++n_s[buf];
            }
            drain += NC;
          }
          ptx::umma_commit(&bars[C::b_q_empty]);
          ++seg;
        }
      }
    } else {
      // --------------------------------- O += P V -----------------------------------
      constexpr int kN = D == 64 ? 64 : 128;                 // columns of one product: one or two chunks
      constexpr uint32_t kI = idesc<T>(kRows, kN, true);
      uint32_t drain = 0, n_p[2] = {0, 0}, n_seg[2] = {0, 0};
      bool ok = true;
      while (ok && walk.next(s)) {
        for (int j = s.lo; ok && j < s.hi; ++j) {
          // value rows behind the sequence's length: zero, whatever the cache holds there
          const int n0 = tile_key(s.u.k, j), rows = s.u.len.keys - n0;
          if (rows < kKeys) {
            for (int c = 0; c < NC; ++c) {
              const uint32_t f = drain + c, st = KS + f % VS;
              ok = __all_sync(0xffffffffu, wait(C::b_kv_full + st, (f / VS) & 1)) && ok;
              uint8_t* v = sm + C::kv + st * kChunk;
              for (int e = (rows > 0 ? rows : 0) * 8 + lane; e < kKeys * 8; e += 32) *reinterpret_cast<uint4*>(v + e * 16) = make_uint4(0, 0, 0, 0);
            }
            ptx::fence_proxy_async();
            __syncwarp();
          }
          if (lane == 0) {
            for (int qi = 0; ok && qi < s.nq; ++qi) {
              const int buf = NQ == 2 ? qi : (int)((n_p[0] + n_p[1]) & 1);
              // the first product of a segment overwrites the accumulator: the last segment's result must be out
              if (j == s.lo && n_seg[qi] > 0) ok = wait(C::b_o_free + qi, (n_seg[qi] - 1) & 1);
              ok = ok && wait(C::b_p_full + buf, n_p[buf] & 1);
              if (!ok) break;
              ptx::tc_fence_after();
              const uint32_t pt = tmem + C::col_s(buf);
              for (int c = 0; ok && c < NC; c += kN / 64) {
                const uint32_t f = drain + c, st = KS + f % VS;
                if (qi == 0) {
                  ok = wait(C::b_kv_full + st, (f / VS) & 1);
                  if (kN == 128) ok = ok && wait(C::b_kv_full + st + 1, (f / VS) & 1);
                  ptx::tc_fence_after();
                }
                // 16 keys a step: 2048 bytes of values, 8 columns of P; the second chunk of a pair lies 16 KiB on
                const uint64_t db = make_desc(ptx::smem_u32(sm + C::kv + st * kChunk), kChunk, 1024);
                const uint32_t d = tmem + C::col_o(qi) + c * 64;
                if (j == s.lo) ptx::umma_ts_first(d, pt, db, kI);
                else ptx::umma_ts_acc(d, pt, db, kI);
#pragma unroll
                for (int k = 1; k < kKeys / 16; ++k) ptx::umma_ts_acc(d, pt + k * 8, db + (uint64_t)k * 128, kI);
                if (qi == s.nq - 1) {
                  ptx::umma_commit(&bars[C::b_kv_empty + st]);
                  if (kN == 128) ptx::umma_commit(&bars[C::b_kv_empty + st + 1]);
                }
              }
              ptx::umma_commit(&bars[C::b_s_free + buf]);
              ptx::umma_commit(&bars[C::b_pv_done + qi]);
              ++n_p[buf];
            }
            for (int qi = 0; j == s.hi - 1 && qi < s.nq; ++qi) ++n_seg[qi];
          }
          drain += NC;
          ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
    // ----------------------------------- softmax ------------------------------------
    Walker<NQ> walk(p);
    Segment s;
    const int wq = warp & 3, grp = (warp - 4) >> 2;           // tensor-memory lane quarter; query tile, or half of the row
    const int r = wq * 32 + lane;
    const uint32_t lane_addr = tmem + ((uint32_t)(wq * 32) << 16);
    const int qi = NQ == 2 ? grp : 0;
    constexpr int NS = NQ == 2 ? 128 : 64;                    // score columns of this thread
    const int col0 = NQ == 2 ? 0 : grp * 64;
    float* xch = reinterpret_cast<float*>(sm + C::xch);
    uint32_t n_s = 0, n_x = 0;                                // score tiles and exchanges done
    // value of the thread that has the other half of this row; the two warps always meet the same number of times
    auto other_half = [&](float mine) {
      float* x = xch + (n_x++ & 1) * 256;
      x[grp * 128 + r] = mine;
      asm volatile("bar.sync %0, 64;" ::"r"(1 + wq) : "memory");
      return x[(grp ^ 1) * 128 + r];
    };
    while (walk.next(s)) {
      if (NQ == 2 && qi >= s.nq) continue;
      int t;
      long long row;
      const bool used = row_of(p, s.u, qi, r, t, row);
      const int pos = s.u.len.keys - s.u.len.rows + t;       // of an unused row too: it sees what it sees, nobody reads it
      const int p_min = s.u.len.keys - s.u.len.rows + s.u.t0 + qi * p.t.Tt, p_max = p_min + p.t.Tt - 1;
      float m = -INFINITY, l = 0.f;
      for (int j = s.lo; j < s.hi; ++j, ++n_s) {
        const int buf = NQ == 2 ? qi : (int)(n_s & 1);
        const uint32_t par = NQ == 2 ? n_s & 1 : (n_s >> 1) & 1;
        wait(C::b_s_full + buf, par);
        __syncwarp();
        ptx::tc_fence_after();
        const uint32_t s_addr = lane_addr + C::col_s(buf);
        uint32_t sr[NS / 32][32];
#pragma unroll
        for (int i = 0; i < NS / 32; ++i) ptx::tmem_ld32(s_addr + col0 + i * 32, sr[i]);
        ptx::tmem_ld_wait();
        const int n0 = tile_key(s.u.k, j);
        if (p.negate) {
#pragma unroll
          for (int i = 0; i < NS; ++i) sr[i / 32][i % 32] ^= 0x80000000u;
        }
        const bool whole = n0 + kKeys - 1 <= p_min && (a.window == 0 || n0 > p_max - a.window || n0 + kKeys <= a.sinks);
        if (!whole) {
          const int hi = pos - n0 - col0, lo = a.window > 0 ? hi - a.window : -1, sink = a.sinks - n0 - col0;
#pragma unroll
          for (int i = 0; i < NS; ++i)
            if (i > hi || (i <= lo && i >= sink)) sr[i / 32][i % 32] = __float_as_uint(-INFINITY);
        }
        float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < NS; ++i) mx4[i & 3] = fmaxf(mx4[i & 3], __uint_as_float(sr[i / 32][i % 32]));
        float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
        if (NQ == 1) mx = fmaxf(mx, other_half(mx));
        float f = 1.f;
        const bool grow = mx > m && (m == -INFINITY || (mx - m) * p.scale_log2 > kRescale);
        if (grow) {
          f = m == -INFINITY ? 0.f : mma::exp2_approx((m - mx) * p.scale_log2);
          m = mx;
          l *= f;
        }
        const bool rescale = j > s.lo && __any_sync(0xffffffffu, grow);
        const float neg = m == -INFINITY ? 0.f : -m * p.scale_log2;
        uint32_t pr[NS / 2];
        float add4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < NS; i += 2) {
          const float w0 = mma::exp2_approx(fmaf(__uint_as_float(sr[i / 32][i % 32]), p.scale_log2, neg));
          const float w1 = mma::exp2_approx(fmaf(__uint_as_float(sr[i / 32][i % 32 + 1]), p.scale_log2, neg));
          add4[(i >> 1) & 3] += w0 + w1;
          pr[i / 2] = mma::pack<T>(w0, w1);
        }
        l += (add4[0] + add4[1]) + (add4[2] + add4[3]);
        // the last product is done with the accumulator; waited for every time and in order (a parity wait that skips a
        // phase cannot tell "done" from "two phases behind"), after the exponentials, when it rarely waits
        if (n_s > 0) wait(C::b_pv_done + qi, (n_s - 1) & 1);
        if (rescale) {
          constexpr int kCols = NQ == 2 ? D : D / 2;
          __syncwarp();
          ptx::tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < kCols; c += 32) {
            uint32_t o[32];
            const uint32_t o_addr = lane_addr + C::col_o(qi) + (NQ == 2 ? 0 : grp * kCols) + c;
            ptx::tmem_ld32(o_addr, o);
            ptx::tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
            ptx::tmem_st32(o_addr, o);
          }
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < NS / 64; ++i) ptx::tmem_st32(s_addr + col0 / 2 + i * 32, *reinterpret_cast<uint32_t(*)[32]>(&pr[i * 32]));
        ptx::tmem_st_wait();
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(&bars[C::b_p_full + buf]);
      }
      // ---- the segment's result ----
      wait(C::b_pv_done + qi, (n_s - 1) & 1);
      __syncwarp();
      ptx::tc_fence_after();
      if (NQ == 1) {                                           // the same order of the two halves in both threads
        const float x = other_half(l);
        l = grp == 0 ? l + x : x + l;
      }
      constexpr int kCols = NQ == 2 ? D : D / 2;
      const int c0 = NQ == 2 ? 0 : grp * kCols;
      const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll 1
      for (int c = 0; c < kCols; c += 32) {
        uint32_t o[32];
        ptx::tmem_ld32(lane_addr + C::col_o(qi) + c0 + c, o);
        ptx::tmem_ld_wait();
        if (s.slot < 0) {
          if (used) {
            uint4* dst = reinterpret_cast<uint4*>(reinterpret_cast<T*>(a.out) + row * D + c0 + c);
#pragma unroll
            for (int i = 0; i < 32; i += 8) {
              uint4 x;
              x.x = mma::pack<T>(__uint_as_float(o[i]) * inv, __uint_as_float(o[i + 1]) * inv);
              x.y = mma::pack<T>(__uint_as_float(o[i + 2]) * inv, __uint_as_float(o[i + 3]) * inv);
              x.z = mma::pack<T>(__uint_as_float(o[i + 4]) * inv, __uint_as_float(o[i + 5]) * inv);
              x.w = mma::pack<T>(__uint_as_float(o[i + 6]) * inv, __uint_as_float(o[i + 7]) * inv);
              dst[i / 8] = x;
            }
          }
        } else {
          // [D / 4][rows]: the 32 rows of a warp store 512 bytes in a row
          float4* dst = p.part_o + ((long long)s.slot * (D / 4) + (c0 + c) / 4) * (128 * NQ) + qi * 128 + r;
#pragma unroll
          for (int i = 0; i < 32; i += 4)
            dst[(i / 4) * (128 * NQ)] = make_float4(__uint_as_float(o[i]), __uint_as_float(o[i + 1]), __uint_as_float(o[i + 2]), __uint_as_float(o[i + 3]));
        }
      }
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(&bars[C::b_o_free + qi]);
      if (NQ == 2 || grp == 0) {
        if (s.slot >= 0) p.part_ml[(long long)s.slot * (128 * NQ) + qi * 128 + r] = make_float2(m * p.scale_log2, l);
        else if (used && a.lse) a.lse[row] = l > 0.f ? (m * p.scale_log2 + log2f(l)) * kLn2 : -INFINITY;
      }
    }
  }
  __syncwarp();
  __syncthreads();
  if (*abort_flag) __nanosleep(100000);        // copies that were still in flight land before the memory is given back
  if (warp == 2) ptx::tmem_dealloc(tmem, 512);
}

// Joins the pieces of a cut unit: 32 rows and 64 columns a block, weights 2^(m_i - max m), added in the order of the pieces.
template <typename T, int D>
__global__ void __launch_bounds__(128) join_kernel(const PromptParams p) {
  constexpr int NQ = Cfg<D>::NQ, R = 128 * NQ;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const Cut cut = p.cuts[blockIdx.x];
  if (cut.count == 0) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Unit u = unit_at(p, cut.unit, NQ * p.t.Tt);
  const int rr = blockIdx.y * 32 + lane, qi = rr / 128, r = rr % 128;
  const int col = blockIdx.z * 64 + warp * 16;
  int t;
  long long row;
  if (!row_of(p, u, qi, r, t, row)) return;
  auto slot = [&](int i) { return (long long)(2 * (cut.first + i) + (i == 0 ? 1 : 0)); };
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
  const float inv = sum > 0.f ? 1.f / sum : 0.f;
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
  if (p.a.lse && blockIdx.z == 0 && warp == 0) p.a.lse[row] = sum > 0.f ? (top + log2f(sum)) * kLn2 : -INFINITY;
}

size_t up256(size_t x) { return (x + 255) / 256 * 256; }

struct Plan {
  Tiling t;
  int NQ, NTT, grid;
  size_t steps, bounds, cuts, part_ml, part_o, total;
};
Plan plan_of(int B, int Hq, int Hkv, int T, int D, int N) {
  Plan x;
  x.t = tiling_of(Hq, Hkv);
  x.NQ = D == 256 ? 1 : 2;
  x.NTT = (T + x.NQ * x.t.Tt - 1) / (x.NQ * x.t.Tt);
  const long long tiles = (long long)B * Hkv * x.t.GC * x.NTT * ((N + kKeys - 1) / kKeys);
  const int n_sm = sm_count();
  x.grid = (int)(tiles < n_sm ? tiles : n_sm);
  x.steps = up256(((size_t)B * x.NTT + 1) * 8);
  x.bounds = up256((size_t)(x.grid + 1) * sizeof(Boundary));
  x.cuts = up256((size_t)x.grid * sizeof(Cut));
  x.part_ml = up256((size_t)2 * x.grid * 128 * x.NQ * sizeof(float2));
  x.part_o = up256((size_t)2 * x.grid * 128 * x.NQ * D * 4);
  x.total = x.steps + x.bounds + x.cuts + x.part_ml + x.part_o;
  return x;
}

template <typename T, int D>
int32_t launch_typed(const CacheArgs& a, cudaStream_t stream) {
  using C = Cfg<D>;
  const Plan x = plan_of(a.B, a.Hq, a.Hkv, a.T, D, a.N);
  PromptParams p{};
  p.a = a;
  p.t = x.t;
  p.NTT = x.NTT;
  p.box = box_rows(a);
  p.grid = x.grid;
  // a scale of zero as one too small to matter: -inf times it has to stay -inf
  const float s = a.scale < 0.f ? -a.scale : a.scale;
  p.scale_log2 = (s < 1e-30f ? 1e-30f : s) * kLog2e;
  p.negate = a.scale < 0.f;
  uint8_t* ws = reinterpret_cast<uint8_t*>(a.workspace);
  p.steps = reinterpret_cast<long long*>(ws);
  p.bounds = reinterpret_cast<Boundary*>(ws += x.steps);
  p.cuts = reinterpret_cast<Cut*>(ws += x.bounds);
  p.part_ml = reinterpret_cast<float2*>(ws += x.cuts);
  p.part_o = reinterpret_cast<float4*>(ws += x.part_ml);
  CUtensorMap mq, mk, mv;
  CUresult r = encode_q(&mq, a, x.t);
  if (r == CUDA_SUCCESS) r = encode_kv(&mk, a.k, a, p.box);
  if (r == CUDA_SUCCESS) r = encode_kv(&mv, a.v, a, p.box);
  if (r != CUDA_SUCCESS) { set_error("prompt_sdpa: cuTensorMapEncodeTiled failed with CUresult %d", (int)r); return DFLASH_ERR_CUDA; }
  auto kernel = prompt_kernel<T, D>;
  DFLASH_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::total));
  // the register hand-over waits for good if the launch gives the CTA fewer than it takes
  static const int regs = [&] { cudaFuncAttributes f; return cudaFuncGetAttributes(&f, kernel) == cudaSuccess ? f.numRegs : 0; }();
  if (regs != kRegsLaunch) { set_error("prompt_sdpa: the kernel is launched with %d registers a thread, %d expected", regs, kRegsLaunch); return DFLASH_ERR_CUDA; }
  plan_kernel<<<1, 1024, 0, stream>>>(p, C::NQ * x.t.Tt);
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
  DFLASH_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, mq, mk, mv, p));
  cfg.gridDim = dim3(x.grid, 4 * C::NQ, D / 64);
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
