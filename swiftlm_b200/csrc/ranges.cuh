// Work of unequal size cut into equal ranges on the device.
//
// The units of a call form rows: HG rows (heads) per sequence, per_row units each, the same costs in every row of a
// sequence.  All units in a row, weighted by their cost (steps that a worker may be cut out of, plus what a unit costs
// besides), are cut into `grid` ranges, one a worker; a cut falls on a multiple of kMinCut steps of a unit, or on its edge where
// the rest would be shorter.  Lengths are read here, on the device: the host needs no copy of them.
#pragma once

#include "cache_ops.cuh"

namespace dflash {

constexpr int kMinCut = 4;                   // steps of the smallest piece of a cut unit
constexpr int kMaxGrid = 1023;               // workers at most: a boundary for each thread of plan_ranges
constexpr int kNearCosts = 2048;             // entries of the cost table that are kept in shared memory: searching the other
                                             // way, through L2, was 5 of the plan's 8 us

struct Boundary { long long unit; int off, pad; };   // in front of step `off` of a unit
struct Cut { long long unit; int first, count; };    // a unit in `count` pieces, of the workers first, first + 1, ...
struct Ranges {
  int B, HG, per_row, grid;
  long long* cost;             // [B * per_row + 1] cost of what is in front of every (sequence, unit), where that is a long table
  Boundary* bounds;            // [grid + 1]
  Cut* cuts;                   // [grid]
};

inline bool ranges_fit(long long B, long long per_row) { return B * per_row < (1ll << 30); }
inline size_t ranges_bytes(long long B, long long per_row, int grid) {
  auto up = [](size_t x) { return (x + 255) / 256 * 256; };
  return up((size_t)(B * per_row + 1) * 8) + up((size_t)(grid + 1) * sizeof(Boundary)) + up((size_t)grid * sizeof(Cut));
}
// lays the plan out at `ws`, returns what is behind it
inline uint8_t* ranges_at(Ranges& r, uint8_t* ws) {
  auto up = [](size_t x) { return (x + 255) / 256 * 256; };
  r.cost = reinterpret_cast<long long*>(ws);
  ws += up(((size_t)r.B * r.per_row + 1) * 8);
  r.bounds = reinterpret_cast<Boundary*>(ws);
  ws += up((size_t)(r.grid + 1) * sizeof(Boundary));
  r.cuts = reinterpret_cast<Cut*>(ws);
  return ws + up((size_t)r.grid * sizeof(Cut));
}

// One block of 1024 threads.  steps(len, unit in its row): 0 for a unit without work.
static_assert(sizeof(Boundary) * (kMaxGrid + 1) <= 8 * (kNearCosts + 2), "the boundaries take the costs' place");
template <int UnitCost, typename Steps>
__device__ __forceinline__ void plan_ranges(const Ranges& p, const CacheArgs& a, Steps steps) {
  __shared__ long long warp_sums[32];
  __shared__ __align__(16) long long near[kNearCosts + 2];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int E = p.B * p.per_row;             // the host sees to it that this is an int
  const long long HG = p.HG;
  auto cost = [&](RowLens len, int u) { const int n = steps(len, u); return n > 0 ? n + UnitCost : 0; };
  const int per_thread = (E - 1) / 1024 + 1, e0 = tid * per_thread < E ? tid * per_thread : E, e1 = E - e0 < per_thread ? E : e0 + per_thread;
  const bool is_near = E <= kNearCosts;
  const long long* table = is_near ? near : p.cost;
  long long mine = 0;
  int b = -1;
  RowLens len{0, 0};
  for (int e = e0; e < e1; ++e) {
    const int eb = e / p.per_row;
    if (eb != b) { b = eb; len = lens_of(a, b, true); }
    mine += cost(len, e - b * p.per_row);
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
  for (int e = e0; e < e1; ++e) {
    (is_near ? near : p.cost)[e] = at;
    if (e + 1 == e1) break;
    const int eb = e / p.per_row;
    if (eb != b) { b = eb; len = lens_of(a, b); }
    at += cost(len, e - b * p.per_row);
  }
  long long all = 0;
  for (int w = 0; w < 32; ++w) all += warp_sums[w];
  if (tid == 0) (is_near ? near : p.cost)[E] = all;
  __syncthreads();               // the table is read by other threads of this block below
  const long long total = all * HG;
  const long long per = total > p.grid ? (total + p.grid - 1) / p.grid : 1;
  __shared__ Boundary raw[kMaxGrid + 1];
  if (tid <= p.grid) {
    const int c = tid;
    const long long pos = c * per;
    Boundary r{E * HG, 0, 0};
    if (pos < total) {
      int lo = 0, hi = p.B - 1;             // the last sequence that starts at or before pos
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (table[(long long)mid * p.per_row] * HG <= pos) lo = mid; else hi = mid - 1;
      }
      const long long base = table[(long long)lo * p.per_row], len_b = table[(long long)(lo + 1) * p.per_row] - base;
      const long long hg = (pos - base * HG) / len_b, rem = pos - base * HG - hg * len_b;
      int ta = 0, tb = p.per_row - 1;             // the last unit that starts at or before rem
      while (ta < tb) {
        const int mid = (ta + tb + 1) >> 1;
        if (table[(long long)lo * p.per_row + mid] - base <= rem) ta = mid; else tb = mid - 1;
      }
      const long long s = table[(long long)lo * p.per_row + ta] - base, e = table[(long long)lo * p.per_row + ta + 1] - base;
      const long long unit = ((long long)lo * HG + hg) * p.per_row + ta;
      const int size = (int)(e - s) - UnitCost;
      int off = (int)(rem - s) - UnitCost;
      off = off < 0 ? 0 : off / kMinCut * kMinCut;
      const bool back = size < kMinCut ? 2 * (rem - s) >= e - s : size - off < kMinCut;    // the unit's end is nearer
      r = back ? Boundary{unit + 1, 0, 0} : Boundary{unit, off, 0};
    }
    raw[c] = r;
  }
  __syncthreads();
  Boundary* bounds = reinterpret_cast<Boundary*>(near);      // the costs are done with
  // equal boundaries become one, so that the pieces of a cut unit belong to workers in a row
  {
    const bool fresh = tid <= p.grid && (tid == 0 || raw[tid].unit != raw[tid - 1].unit || raw[tid].off != raw[tid - 1].off);
    const uint32_t in_warp = __ballot_sync(0xffffffffu, fresh);
    if (lane == 0) warp_sums[warp] = __popc(in_warp);
    __syncthreads();
    int before = 0, all_fresh = 0;
    for (int w = 0; w < 32; ++w) {
      before += w < warp ? (int)warp_sums[w] : 0;
      all_fresh += (int)warp_sums[w];
    }
    if (fresh) bounds[before + __popc(in_warp & ((1u << lane) - 1u))] = raw[tid];
    if (tid >= all_fresh && tid <= p.grid) bounds[tid] = Boundary{E * HG, 0, 0};
  }
  __syncthreads();
  if (tid <= p.grid) p.bounds[tid] = bounds[tid];
  if (tid < p.grid) {
    const int c = tid;
    Cut cut{0, 0, 0};
    if (c >= 1 && bounds[c].off > 0 && !(bounds[c - 1].off > 0 && bounds[c - 1].unit == bounds[c].unit)) {
      int n = 1;
      while (c + n <= p.grid && bounds[c + n].off > 0 && bounds[c + n].unit == bounds[c].unit) ++n;
      cut = Cut{bounds[c].unit, c - 1, n + 1};
    }
    p.cuts[c] = cut;
  }
}

// The units from number `unit` on, one after another; a sequence's lengths are read once.
struct Cursor {
  const Ranges& p;
  const CacheArgs& a;
  int b, hg, u;                // sequence, row, unit in its row
  RowLens len;
  __device__ Cursor(const Ranges& p_, const CacheArgs& a_, long long unit) : p(p_), a(a_) {
    const long long row = unit / p.per_row;
    u = (int)(unit - row * p.per_row);
    b = (int)(row / p.HG);
    hg = (int)(row - (long long)b * p.HG);
    len = b < p.B ? lens_of(a, b) : RowLens{0, 0};
  }
  __device__ long long number() const { return ((long long)b * p.HG + hg) * p.per_row + u; }
  __device__ void move_to(int v) {             // unit v of the row, or the next row
    u = v;
    if (v < p.per_row) return;
    u = 0;
    if (++hg == p.HG) {
      hg = 0;
      ++b;
      len = b < p.B ? lens_of(a, b) : RowLens{0, 0};
    }
  }
};

// The units (or pieces) of one worker, in order; every role of a kernel walks them for itself.
struct RangeWalker {
  Cursor c;
  long long last;              // unit in which the range ends, in front of step last_off
  int off, last_off, worker;
  __device__ RangeWalker(const Ranges& p, const CacheArgs& a, int worker_)
      : c(p, a, p.bounds[worker_].unit), last(p.bounds[worker_ + 1].unit), off(p.bounds[worker_].off),
        last_off(p.bounds[worker_ + 1].off), worker(worker_) {}
  // first(len, u): the first unit of a row at or behind u that has work, per_row if there is none.  True: c stands at the next
  // unit of the range, whose steps begin with `lo`; the caller finishes it with take().
  template <typename First>
  __device__ bool find(First first, int& lo) {
    for (;;) {
      const long long at = c.number();
      if (at > last || (at == last && off >= last_off)) return false;
      const int v = first(c.len, c.u);
      if (v == c.u) break;
      c.move_to(v);
    }
    lo = off;
    return true;
  }
  // end of the steps of this unit that belong to the range, and the slot of a piece (-1: the whole unit)
  __device__ int take(int lo, int size, int& slot) {
    const int hi = c.number() == last ? last_off : size;
    slot = (lo == 0 && hi == size) ? -1 : 2 * worker + (lo > 0 ? 0 : 1);
    off = 0;
    c.move_to(c.u + 1);
    return hi;
  }
};
__device__ __forceinline__ int piece_slot(const Cut& cut, int i) { return 2 * (cut.first + i) + (i == 0 ? 1 : 0); }

}  // namespace dflash
