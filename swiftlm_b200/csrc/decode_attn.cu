// Attention of one new token per sequence over the KV cache: out = softmax(scale q K^T over the visible tokens) V.
//
// Every visible key and value is read once and used by the G query heads of its KV head (more than 16 of them: once for every
// group of 16, each group's units a pass of their own): G operations a byte, far below what the tensor cores need to be busy, so
// the kernel is built to keep HBM reads in flight and nothing else.  (On the CUDA
// cores G = 8 would take 4096 fused multiply-adds per kilobyte, which is 0.8 of the fp32 rate at full HBM speed; as
// warp-level matrix products it is some 200 issue slots per 16 keys.)
//
// * Work: a unit is one (sequence, KV head, group of up to 8 NT query heads); its visible tokens are a list of 16-key
//   chunks, first those of the sinks, then those of the window (a chunk never crosses a page: page sizes are multiples
//   of 16).  A tile is W chunks, one per warp.  The tiles of all units, in a row, are cut into equal ranges, one per resident
//   CTA, whatever the lengths are; lengths are read on the device, the host needs no copy of them.
// * Loads: a ring of tiles in shared memory filled by 16-byte asynchronous copies, each warp its own chunk (one page
//   look-up per 16 keys), two to five tiles ahead, across the ends of units.  Rows behind the sequence's length are
//   filled with zeros and never read: whatever they hold cannot reach a product.
// * S^T = K Q^T (16 keys x 8 NT heads per warp, m16n8k16): the heads are the narrow side, so a group of 8 wastes
//   nothing.  The W warps agree on the tile's maxima through shared memory, write P as 16-bit rows, and each warp then
//   owns D / W rows of O^T = V^T P^T for all the tile's keys: one accumulator per CTA, no merge of warps, two
//   barriers a tile.  O is rescaled only when a maximum grows by more than 2^8 (its scale is exact in fp32).
//   P is rounded to the inputs' type (the sum of the weights is not): the product needs a 16-bit operand (f16: lifted
//   first, mma_sync.cuh).
// * A unit that one CTA covers is normalised and written at once; the others leave (O, maximum, sum) in the workspace
//   and decode_finish_kernel, chained by a programmatic launch, joins them in a fixed order.
// * With `mass`, the scaled scores of the visible tokens are kept and decode_finish_kernel turns them into weights when every
//   head's sum is known.  A key has 4 bytes for each of 8 or 16 heads, whether there are as many or not: written and read
//   again, 6 % of the bytes of K and V at D = 256 and up to 8 heads, where reading K again would be half of them; 25 % at
//   D = 64, however few the heads.
//
// Measured (B200, the whole call; of the 6.57 TB/s that a copy reaches): 8 sequences of 34 to 102 thousand tokens at D = 256
// 175 to 189 us, from card to card (1.02 to 0.94); 32 of 3 to 8 thousand with weights 78 us (0.71: the main kernel takes 63, the
// second 14); 64 sequences x 8 KV heads at D = 128 with a window of 1024 and 64 sinks 58 us (0.75); one sequence of
// 517 tokens 18 us, bound by the host (12 us of kernels, 6 and 5.5).
#include <type_traits>

#include "cache_ops.cuh"
#include "mma_sync.cuh"
#include "ptx.cuh"

namespace dflash {
namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kRescale = 8.f;            // in log2 units
constexpr int kMaxBatch = 512;             // sequences per launch (the prefix of their tile counts lives in shared memory)

// Warps (16 keys each), ring stages and CTAs per SM: 192 KiB of keys and values in an SM's rings.
template <int D> struct Shape;
template <> struct Shape<64> { static constexpr int W = 4, S = 6, per_sm = 2; };
template <> struct Shape<128> { static constexpr int W = 4, S = 3, per_sm = 2; };
template <> struct Shape<256> { static constexpr int W = 4, S = 3, per_sm = 1; };

template <int D, int NT> struct Layout {
  static constexpr int W = Shape<D>::W, S = Shape<D>::S;
  static constexpr int chunk = 16 * D * 2;                  // bytes of 16 key (or value) rows
  static constexpr int stage = 2 * W * chunk;               // K chunks of the W warps, then V chunks
  static constexpr int q = S * stage;                       // two query tiles [8 NT][D]
  static constexpr int q_bytes = 8 * NT * D * 2;
  static constexpr int p = q + 2 * q_bytes;                 // P: [NT][16 W keys][8 heads], 16-bit
  static constexpr int mx = p + NT * 16 * W * 16;           // per warp maxima (and sums) of the heads
  static constexpr int prefix = mx + W * 8 * NT * 4;        // tiles of the sequences before b, long long
  static constexpr int fixed = prefix + 8;
};

struct DecodeParams {
  CacheArgs a;
  int b0, nb;                  // the launch's sequences
  int G, GC;                   // heads per KV head, head groups per KV head
  int heads;                   // query heads a block of decode_finish_kernel joins
  int max_chunks;              // upper bound of a unit's chunks
  float scale_log2;
  float *part_o, *part_m, *part_l;   // [2 * grid][8 NT][D], [2 * grid][8 NT] twice
  int2* unit_info;             // [units]: first CTA and number of its ranges; ranges = 0: written already
  float* scores;               // [units][max_chunks][16][8 NT] or null
  float* lse2;                 // [B * Hq] log2 of the sum of weights, for the mass
};

// the visible chunks of a sequence with n tokens whose newest one asks
struct Visible {
  int n, lo, sinks;            // tokens [0, sinks) and [lo, n)
  int head, first, count;      // chunk c of the list is chunk c (c < head) or first + c - head
};
__device__ __forceinline__ Visible visible_of(const CacheArgs& a, int n) {
  Visible v;
  v.n = n;
  v.lo = (a.window > 0 && n > a.window) ? n - a.window : 0;
  v.sinks = a.sinks < v.lo ? a.sinks : v.lo;
  v.first = v.lo >> 4;
  v.head = (v.sinks + 15) >> 4;
  if (v.head > v.first) v.head = v.first;
  v.count = v.head + ((n + 15) >> 4) - v.first;
  if (v.count < 1) v.count = 1;               // an empty sequence: one chunk in which nothing is visible
  return v;
}
__device__ __forceinline__ int chunk_key(const Visible& v, int c) { return (c < v.head ? c : v.first + c - v.head) << 4; }

struct Segment {
  long long unit;
  int b, h, gc;                // b: sequence of the whole call
  int tile, end, tiles;        // its tiles [tile, end) of the unit's `tiles`
  Visible v;
};

// walks the units that a range of tiles touches
template <int W>
struct Walker {
  const DecodeParams& p;
  const long long* prefix;
  long long pos, end;
  int b;
  __device__ Walker(const DecodeParams& p_, const long long* prefix_, long long begin, long long end_) : p(p_), prefix(prefix_), pos(begin), end(end_), b(0) {
    if (pos < end) {           // the last b with prefix[b] <= pos
      int lo = 0, hi = p.nb - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (prefix[mid] <= pos) lo = mid; else hi = mid - 1;
      }
      b = lo;
    }
  }
  __device__ bool next(Segment& s) {
    if (pos >= end) return false;
    while (pos >= prefix[b + 1]) ++b;
    s.b = p.b0 + b;
    s.v = visible_of(p.a, lens_of(p.a, s.b).keys);
    s.tiles = (s.v.count + W - 1) / W;
    const long long off = pos - prefix[b];
    const int u = (int)(off / s.tiles);
    s.tile = (int)(off - (long long)u * s.tiles);
    s.h = u / p.GC;
    s.gc = u - s.h * p.GC;
    s.unit = (long long)s.b * p.a.Hkv * p.GC + u;
    const long long left = end - pos;
    s.end = left < s.tiles - s.tile ? s.tile + (int)left : s.tiles;
    pos += s.end - s.tile;
    return true;
  }
};

template <typename T, int D, int NT>
__global__ void __launch_bounds__(Shape<D>::W * 32, Shape<D>::per_sm) decode_kernel(const DecodeParams p) {
  using L = Layout<D, NT>;
  constexpr int W = L::W, S = L::S, kThreads = W * 32, H = 8 * NT;
  constexpr int U = D / 8;                    // 16-byte units of a row
  constexpr int MT = D / W / 16;              // 16-row tiles of O^T per warp
  extern __shared__ __align__(128) uint8_t sm[];
  const CacheArgs& a = p.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // ---- tiles in front of every sequence, and this CTA's range ----
  long long* prefix = reinterpret_cast<long long*>(sm + L::prefix);
  {
    constexpr int per = (kMaxBatch + kThreads - 1) / kThreads;
    long long mine = 0;
    int cnt[per];
#pragma unroll
    for (int i = 0; i < per; ++i) {
      const int b = tid * per + i;
      cnt[i] = 0;
      if (b < p.nb) cnt[i] = (visible_of(a, lens_of(a, p.b0 + b, blockIdx.x == 0).keys).count + W - 1) / W;
      mine += cnt[i];
    }
    long long x = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    long long* ws = reinterpret_cast<long long*>(sm);      // the ring is not in use yet
    if (lane == 31) ws[warp] = x;
    __syncthreads();
    long long at = x - mine;
    for (int w = 0; w < warp; ++w) at += ws[w];
    const long long units_b = (long long)a.Hkv * p.GC;
#pragma unroll
    for (int i = 0; i < per; ++i) {
      const int b = tid * per + i;
      if (b < p.nb) prefix[b] = at * units_b;
      at += cnt[i];
      if (b == p.nb - 1) prefix[p.nb] = at * units_b;
    }
    __syncthreads();
  }
  const long long total = prefix[p.nb], per_cta = (total + gridDim.x - 1) / gridDim.x;
  const long long begin = per_cta * blockIdx.x < total ? per_cta * blockIdx.x : total;
  const long long end = begin + per_cta < total ? begin + per_cta : total;
  if (begin >= end) return;

  // ---- loading side: one cursor over the CTA's tiles ----
  Walker<W> lw(p, prefix, begin, end);
  Segment ls;
  bool l_more = lw.next(ls);
  int l_tile = ls.tile, l_stage = 0;
  auto load_tile = [&]() {
    if (l_more) {
      const int c = l_tile * W + warp;
      uint8_t* kd = sm + l_stage * L::stage + warp * L::chunk;
      uint8_t* vd = kd + W * L::chunk;
      const int n0 = c < ls.v.count ? chunk_key(ls.v, c) : 0;
      int rows = c < ls.v.count ? ls.v.n - n0 : 0;          // rows of the chunk that exist
      long long row0 = 0;
      if (rows > 0) {
        row0 = kv_row(a, ls.b, ls.h, n0);
        if (row0 < 0) { row0 = 0; rows = 0; }              // a page outside the pool reads as zeros
      }
      const uint8_t* ks = reinterpret_cast<const uint8_t*>(a.k) + row0 * (D * 2);
      const uint8_t* vs = reinterpret_cast<const uint8_t*>(a.v) + row0 * (D * 2);
#pragma unroll
      for (int i = 0; i < 16 * U / 32; ++i) {
        const int e = i * 32 + lane, r = e / U, u = e % U;
        const int off = r * (D * 2) + ((u ^ (r & 7)) << 4);
        const bool ok = r < rows;
        const int src = ok ? e * 16 : 0;
        ptx::cp_async16_zfill(kd + off, ks + src, ok);
        ptx::cp_async16_zfill(vd + off, vs + src, ok);
      }
      if (++l_tile == ls.end) {
        l_more = lw.next(ls);
        l_tile = ls.tile;
      }
    }
    ptx::cp_async_commit();
    l_stage = l_stage + 1 == S ? 0 : l_stage + 1;
  };
#pragma unroll
  for (int i = 0; i < S - 1; ++i) load_tile();

  // ---- queries: fetched into registers a segment ahead, zero behind the last head ----
  constexpr int kQVecs = (H * U + kThreads - 1) / kThreads;
  uint4 qv[kQVecs];
  auto fetch_q = [&](const Segment& s) {
#pragma unroll
    for (int i = 0; i < kQVecs; ++i) {
      const int e = i * kThreads + tid, g = s.gc * H + e / U;
      qv[i] = make_uint4(0, 0, 0, 0);
      if (e < H * U && g < p.G)
        qv[i] = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(a.q) +
                                                (((long long)s.b * a.Hq + s.h * p.G + g) * D) * 2 + (e % U) * 16);
    }
  };
  auto store_q = [&](int buf) {
#pragma unroll
    for (int i = 0; i < kQVecs; ++i) {
      const int e = i * kThreads + tid, r = e / U, u = e % U;
      if (e < H * U) *reinterpret_cast<uint4*>(sm + L::q + buf * L::q_bytes + r * (D * 2) + ((u ^ (r & 7)) << 4)) = qv[i];
    }
  };
  Walker<W> cw(p, prefix, begin, end);
  Segment s, s_next;
  cw.next(s);
  fetch_q(s);
  store_q(0);
  __syncthreads();

  float* mx = reinterpret_cast<float*>(sm + L::mx);
  int stage = 0, q_buf = 0;
  const int hc = 2 * (lane & 3);               // this thread's heads in an 8-head tile: hc, hc + 1
  bool more = true;
  while (more) {
    more = cw.next(s_next);
    if (more) fetch_q(s_next);
    float o[MT][NT][4] = {};
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) m[t][0] = m[t][1] = -INFINITY, l[t][0] = l[t][1] = 0.f;

    for (int tile = s.tile; tile < s.end; ++tile) {
      ptx::cp_async_wait<S - 2>();
      __syncwarp();
      const uint8_t* kd = sm + stage * L::stage + warp * L::chunk;
      const uint8_t* vd = sm + stage * L::stage + W * L::chunk;
      const uint8_t* qd = sm + L::q + q_buf * L::q_bytes;
      // ---- S^T = K Q^T for this warp's 16 keys: two accumulators a tile keep the chain of products short ----
      float c[2][NT][4] = {};
      {
        const int kr = lane & 15, ku = lane >> 4;
        const int qr = lane & 7, qu = lane >> 3;
#pragma unroll
        for (int k2 = 0; k2 < D / 32; ++k2) {
          uint32_t ka[2][4];
          mma::ldmatrix_x4(ka[0], kd + kr * (D * 2) + (((4 * k2 + ku) ^ (kr & 7)) << 4));
          mma::ldmatrix_x4(ka[1], kd + kr * (D * 2) + (((4 * k2 + 2 + ku) ^ (kr & 7)) << 4));
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            uint32_t qb[4];
            mma::ldmatrix_x4(qb, qd + (t * 8 + qr) * (D * 2) + (((4 * k2 + qu) ^ (qr & 7)) << 4));
            mma::mma16816<T>(c[0][t], ka[0], qb[0], qb[1]);
            mma::mma16816<T>(c[1][t], ka[1], qb[2], qb[3]);
          }
        }
      }
      // ---- scale, hide, maxima ----
      const int ci = tile * W + warp;
      const int n0 = ci < s.v.count ? chunk_key(s.v, ci) : s.v.n;
      const int r0 = n0 + (lane >> 2), r1 = r0 + 8;
      const bool on0 = r0 < s.v.n && (r0 >= s.v.lo || r0 < s.v.sinks), on1 = r1 < s.v.n && (r1 >= s.v.lo || r1 < s.v.sinks);
      float x[NT][4];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[t][i] = (i < 2 ? on0 : on1) ? (c[0][t][i] + c[1][t][i]) * p.scale_log2 : -INFINITY;
        float a0 = fmaxf(x[t][0], x[t][2]), a1 = fmaxf(x[t][1], x[t][3]);
#pragma unroll
        for (int sh = 4; sh < 32; sh <<= 1) {
          a0 = fmaxf(a0, __shfl_xor_sync(0xffffffffu, a0, sh));
          a1 = fmaxf(a1, __shfl_xor_sync(0xffffffffu, a1, sh));
        }
        if (lane < 4) *reinterpret_cast<float2*>(&mx[warp * H + t * 8 + hc]) = make_float2(a0, a1);
        if (p.scores && ci < s.v.count) {
          float* sc = p.scores + ((s.unit * p.max_chunks + ci) * 16 + (lane >> 2)) * H + t * 8 + hc;
          *reinterpret_cast<float2*>(sc) = make_float2(x[t][0], x[t][1]);
          *reinterpret_cast<float2*>(sc + 8 * H) = make_float2(x[t][2], x[t][3]);
        }
      }
      __syncthreads();          // maxima of all warps; every warp's values have landed; the previous tile is done with
      load_tile();              // ... so its stage may be filled again
      // ---- weights ----
      bool grow = false;
      float f[NT][2];
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float top = mx[t * 8 + hc + i];
#pragma unroll
          for (int w = 1; w < W; ++w) top = fmaxf(top, mx[w * H + t * 8 + hc + i]);
          f[t][i] = 1.f;
          if (top > m[t][i] + kRescale || (m[t][i] == -INFINITY && top > -INFINITY)) {
            f[t][i] = mma::exp2_approx(m[t][i] - top);       // 0 where nothing was visible before
            m[t][i] = top;
            grow = true;
          }
        }
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const float z0 = m[t][0] == -INFINITY ? 0.f : m[t][0] - mma::kLift<T>, z1 = m[t][1] == -INFINITY ? 0.f : m[t][1] - mma::kLift<T>;
        const float w0 = mma::exp2_approx(x[t][0] - z0), w1 = mma::exp2_approx(x[t][1] - z1);
        const float w2 = mma::exp2_approx(x[t][2] - z0), w3 = mma::exp2_approx(x[t][3] - z1);
        l[t][0] = l[t][0] * f[t][0] + (w0 + w2);
        l[t][1] = l[t][1] * f[t][1] + (w1 + w3);
        uint32_t* pd = reinterpret_cast<uint32_t*>(sm + L::p + t * (16 * W * 16) + (warp * 16 + (lane >> 2)) * 16) + (lane & 3);
        pd[0] = mma::pack<T>(w0, w1);
        pd[32] = mma::pack<T>(w2, w3);          // 8 rows of 16 bytes on
      }
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            o[i][t][0] *= f[t][0]; o[i][t][1] *= f[t][1];
            o[i][t][2] *= f[t][0]; o[i][t][3] *= f[t][1];
          }
      }
      __syncthreads();          // P of all warps
      // ---- O^T += V^T P^T: this warp's D / W rows, all keys ----
#pragma unroll
      for (int kk = 0; kk < W; kk += 2) {       // two 16-key steps
        uint32_t pb[NT][4];
#pragma unroll
        for (int t = 0; t < NT; ++t) mma::ldmatrix_x4_trans(pb[t], sm + L::p + t * (16 * W * 16) + (kk * 16 + lane) * 16);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int vr = ((lane >> 4) << 3) + (lane & 7), vu = (lane >> 3) & 1;
          const uint8_t* vrow = vd + (kk + j) * L::chunk + vr * (D * 2);
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            uint32_t va[4];
            mma::ldmatrix_x4_trans(va, vrow + (((warp * (2 * MT) + 2 * i + vu) ^ (vr & 7)) << 4));
#pragma unroll
            for (int t = 0; t < NT; ++t) mma::mma16816<T>(o[i][t], va, pb[t][2 * j], pb[t][2 * j + 1]);
          }
        }
      }
      stage = stage + 1 == S ? 0 : stage + 1;
    }

    // ---- the segment's end: sums over lanes and warps, then the output or a partial ----
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int sh = 4; sh < 32; sh <<= 1) l[t][i] += __shfl_xor_sync(0xffffffffu, l[t][i], sh);
        if (lane < 4) mx[warp * H + t * 8 + hc + i] = l[t][i];
      }
    if (more) store_q(q_buf ^ 1);
    __syncthreads();
    const bool whole = s.tile == 0 && s.end == s.tiles;
    const int slot = 2 * blockIdx.x + (s.tile == 0 ? 1 : 0);
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int j = t * 8 + hc + i, g = s.gc * H + j;
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) sum += mx[w * H + j];
        if (whole) {
          if (g < p.G) {
            const long long row = (long long)s.b * a.Hq + s.h * p.G + g;
            const float inv = sum == 0.f ? 0.f : 1.f / sum;     // 0: nothing was visible; NaN stays NaN
            T* dst = reinterpret_cast<T*>(a.out) + row * D + warp * (D / W) + (lane >> 2);
#pragma unroll
            for (int k = 0; k < MT; ++k) {
              dst[k * 16] = from_f32<T>(o[k][t][i] * inv);
              dst[k * 16 + 8] = from_f32<T>(o[k][t][i + 2] * inv);
            }
            if (warp == 0 && lane < 4) {
              const float z = sum == 0.f ? -INFINITY : m[t][i] - mma::kLift<T> + log2f(sum);
              if (a.lse) a.lse[row] = z * kLn2;
              if (p.lse2) p.lse2[row] = z;
            }
          }
        } else {
          float* dst = p.part_o + ((long long)slot * H + j) * D + warp * (D / W) + (lane >> 2);
#pragma unroll
          for (int k = 0; k < MT; ++k) {
            dst[k * 16] = o[k][t][i];
            dst[k * 16 + 8] = o[k][t][i + 2];
          }
          if (warp == 0 && lane < 4) {
            p.part_m[slot * H + j] = m[t][i] - mma::kLift<T>;
            p.part_l[slot * H + j] = sum;
          }
        }
      }
    if (tid == 0 && s.tile == 0) {
      const int left = s.tiles - (s.end - s.tile);      // tiles of the unit behind this CTA's range
      p.unit_info[s.unit] = make_int2(blockIdx.x, whole ? 0 : 1 + (int)((left + per_cta - 1) / per_cta));
    }
    __syncthreads();            // mx and the query buffer are used again
    q_buf ^= 1;
    s = s_next;
  }
}

// Behind the main kernel, one launch for two things.
// Join: the ranges of a cut unit with weights 2^(m_r - max m), summed in the order of the ranges.  A block takes p.heads heads of
// one unit; where a unit has few ranges a group of D / 4 threads takes a head each, else all groups share a head's ranges.
// Mass: mass[b, h, n] += sum over the heads of 2^(score - lse), one thread per visible key, the heads in order.  The
// log-sum-exps of a cut unit's heads are computed again by every block that needs them: a few loads, against a launch.
constexpr int kFinishThreads = 256;
template <typename T, int D, int NT>
__global__ void __launch_bounds__(kFinishThreads) decode_finish_kernel(const DecodeParams p) {
  constexpr int H = 8 * NT, V = D / 4, R = kFinishThreads / V;       // float4 columns, groups of threads
  __shared__ float acc_s[R][V][4];
  __shared__ float zs[H];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const CacheArgs& a = p.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int blocks = (p.G < H ? p.G + p.heads - 1 : H + p.heads - 1) / p.heads;      // head blocks of a unit
  const int u = blockIdx.x / blocks, j0 = (blockIdx.x - u * blocks) * p.heads;
  const int bh = u / p.GC, gc = u - bh * p.GC, b = p.b0 + bh / a.Hkv, h = bh % a.Hkv;
  auto slot_of = [&](const int2& info, int r) { return 2 * (info.x + r) + (r == 0 ? 1 : 0); };
  if (blockIdx.y == 0) {
    const long long unit = ((long long)b * a.Hkv + h) * p.GC + gc;
    const int2 info = p.unit_info[unit];
    const int n = info.y, col = tid % V, grp = tid / V;
    int j1 = p.G - gc * H < H ? p.G - gc * H : H;            // heads of the unit
    if (j1 > j0 + p.heads) j1 = j0 + p.heads;
    auto store = [&](int j, float4 o, float top, float sum) {
      const long long row = (long long)b * a.Hq + h * p.G + gc * H + j;
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      uint2 pk;
      pk.x = mma::pack<T>(o.x * inv, o.y * inv);
      pk.y = mma::pack<T>(o.z * inv, o.w * inv);
      *reinterpret_cast<uint2*>(reinterpret_cast<T*>(a.out) + row * D + col * 4) = pk;
      if (col == 0 && a.lse) a.lse[row] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2;
    };
    auto add = [&](int j, int r, float z, float4& o, float& sum) {
      const int sl = slot_of(info, r) * H + j;
      const float w = mma::exp2_approx(p.part_m[sl] - z);
      sum = fmaf(w, p.part_l[sl], sum);
      const float4 v = *reinterpret_cast<const float4*>(p.part_o + (long long)sl * D + col * 4);
      o.x = fmaf(w, v.x, o.x); o.y = fmaf(w, v.y, o.y); o.z = fmaf(w, v.z, o.z); o.w = fmaf(w, v.w, o.w);
    };
    if (n > 0 && n <= 8 && j1 - j0 > 1) {
      for (int j = j0 + grp; j < j1; j += R) {
        float top = -INFINITY, sum = 0.f;
        for (int r = 0; r < n; ++r) top = fmaxf(top, p.part_m[slot_of(info, r) * H + j]);
        const float z = top == -INFINITY ? 0.f : top;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int r = 0; r < n; ++r) add(j, r, z, o, sum);
        store(j, o, top, sum);
      }
    } else if (n > 0) {
      for (int j = j0; j < j1; ++j) {
        float top = -INFINITY, sum = 0.f;
        for (int r = lane; r < n; r += 32) top = fmaxf(top, p.part_m[slot_of(info, r) * H + j]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float z = top == -INFINITY ? 0.f : top;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int r = grp; r < n; r += R) add(j, r, z, o, sum);      // this group's ranges
        *reinterpret_cast<float4*>(acc_s[grp][col]) = o;
        sum = 0.f;                                               // of all ranges, by every warp alike
        for (int r = lane; r < n; r += 32) {
          const int sl = slot_of(info, r) * H + j;
          sum = fmaf(mma::exp2_approx(p.part_m[sl] - z), p.part_l[sl], sum);
        }
#pragma unroll
        for (int q = 16; q > 0; q >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, q);
        __syncthreads();
        if (grp == 0) {                                          // the groups' shares, in order
#pragma unroll
          for (int k = 1; k < R; ++k) {
            const float4 v = *reinterpret_cast<const float4*>(acc_s[k][col]);
            o.x += v.x; o.y += v.y; o.z += v.z; o.w += v.w;
          }
          store(j, o, top, sum);
        }
        __syncthreads();
      }
    }
    return;
  }
  if (gc != 0 || j0 != 0) return;              // rows of blocks from 1 on: mass
  const Visible v = visible_of(a, lens_of(a, b).keys);
  const long long keys = (long long)v.count * 16;
  const long long first = (long long)(blockIdx.y - 1) * kFinishThreads;
  for (long long e0 = first; e0 < keys; e0 += (long long)(gridDim.y - 1) * kFinishThreads) {
    const long long e = e0 + tid;
    const int n = e < keys ? chunk_key(v, (int)(e >> 4)) + ((int)e & 15) : 0;
    const bool on = e < keys && n < v.n && (n >= v.lo || n < v.sinks);
    float total = 0.f;
    for (int g = 0; g < p.GC; ++g) {
      const long long unit = ((long long)b * a.Hkv + h) * p.GC + g;
      const int heads = p.G - g * H < H ? p.G - g * H : H;
      const int2 info = p.unit_info[unit];
      const bool known = p.GC == 1 && e0 > first;              // one group of heads: its log-sum-exps stay in shared memory
      __syncthreads();
      for (int j = known ? heads : warp; j < heads; j += kFinishThreads / 32) {
        float z;
        if (info.y == 0) {
          z = p.lse2[(long long)b * a.Hq + h * p.G + g * H + j];
        } else {
          float top = -INFINITY, sum = 0.f;
          for (int r = lane; r < info.y; r += 32) top = fmaxf(top, p.part_m[slot_of(info, r) * H + j]);
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
          const float zz = top == -INFINITY ? 0.f : top;
          for (int r = lane; r < info.y; r += 32) {
            const int sl = slot_of(info, r) * H + j;
            sum = fmaf(mma::exp2_approx(p.part_m[sl] - zz), p.part_l[sl], sum);
          }
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
          z = sum == 0.f ? -INFINITY : top + log2f(sum);
        }
        if (lane == 0) zs[j] = z;
      }
      __syncthreads();
      if (!on) continue;
      const float* sc = p.scores + (unit * p.max_chunks * 16 + e) * H;
      float x[H];
#pragma unroll
      for (int i = 0; i < H; i += 4) *reinterpret_cast<float4*>(&x[i]) = *reinterpret_cast<const float4*>(sc + i);
#pragma unroll
      for (int i = 0; i < H; ++i)
        if (i < heads) total += mma::exp2_approx(x[i] - zs[i]);
    }
    if (on) a.mass[((long long)b * a.Hkv + h) * a.mass_stride + n] += total;
  }
}

size_t up256(size_t x) { return (x + 255) / 256 * 256; }

struct Plan {
  int G, GC, NT, W, grid_max, max_chunks;
  long long units;
  size_t part, info, scores, lse2, total;
};
Plan plan_of(int B, int Hq, int Hkv, int D, int N, int window, int sinks, bool with_mass) {
  Plan t;
  t.G = Hq / Hkv;
  t.NT = t.G <= 8 ? 1 : 2;
  t.GC = (t.G + 8 * t.NT - 1) / (8 * t.NT);
  t.W = 4;
  static_assert(Shape<64>::W == 4 && Shape<128>::W == 4 && Shape<256>::W == 4, "");
  t.max_chunks = (N + 15) / 16;
  if (window > 0) {
    const long long c = (long long)(sinks + 15) / 16 + (window + 15) / 16 + 1;
    if (c < t.max_chunks) t.max_chunks = (int)c;
  }
  t.units = (long long)B * Hkv * t.GC;
  const int nb = B < kMaxBatch ? B : kMaxBatch;
  const long long tiles = (long long)nb * Hkv * t.GC * ((t.max_chunks + t.W - 1) / t.W);
  const int ctas = sm_count() * (D == 256 ? Shape<256>::per_sm : Shape<128>::per_sm);
  t.grid_max = (int)(tiles < ctas ? tiles : ctas);
  const size_t rows = 2 * (size_t)t.grid_max * 8 * t.NT;
  t.part = up256(rows * D * 4) + 2 * up256(rows * 4);
  t.info = up256((size_t)t.units * sizeof(int2));
  t.scores = with_mass ? up256((size_t)t.units * t.max_chunks * 16 * 8 * t.NT * 4) : 0;
  t.lse2 = with_mass ? up256((size_t)B * Hq * 4) : 0;
  t.total = t.part + t.info + t.scores + t.lse2;
  return t;
}

template <typename F>
cudaError_t launch_chained(F kernel, dim3 grid, int threads, const DecodeParams& p, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

template <typename T, int D, int NT>
int32_t launch_typed(const CacheArgs& a, const Plan& t, cudaStream_t stream) {
  using L = Layout<D, NT>;
  DecodeParams p{};
  p.a = a;
  p.G = t.G;
  p.GC = t.GC;
  p.max_chunks = t.max_chunks;
  p.scale_log2 = a.scale * kLog2e;
  uint8_t* ws = reinterpret_cast<uint8_t*>(a.workspace);
  const size_t rows = 2 * (size_t)t.grid_max * 8 * NT;
  p.part_o = reinterpret_cast<float*>(ws);
  p.part_m = reinterpret_cast<float*>(ws + up256(rows * D * 4));
  p.part_l = reinterpret_cast<float*>(ws + up256(rows * D * 4) + up256(rows * 4));
  p.unit_info = reinterpret_cast<int2*>(ws + t.part);
  p.scores = a.mass ? reinterpret_cast<float*>(ws + t.part + t.info) : nullptr;
  p.lse2 = a.mass ? reinterpret_cast<float*>(ws + t.part + t.info + t.scores) : nullptr;
  auto kernel = decode_kernel<T, D, NT>;
  static std::atomic<uint64_t> ready{0};
  DFLASH_CUDA_CHECK(allow_shared(ready, kernel, L::fixed + kMaxBatch * 8));
  for (int b0 = 0; b0 < a.B; b0 += kMaxBatch) {
    p.b0 = b0;
    p.nb = a.B - b0 < kMaxBatch ? a.B - b0 : kMaxBatch;
    const long long tiles = (long long)p.nb * a.Hkv * t.GC * ((t.max_chunks + L::W - 1) / L::W);
    const int grid = (int)(tiles < t.grid_max ? tiles : t.grid_max);
    kernel<<<grid, L::W * 32, L::fixed + p.nb * 8, stream>>>(p);
    DFLASH_LAUNCH_CHECK();
    // Units that are hardly cut: a block for all heads of one (64 sequences of 8 KV heads with a window: 58 us the whole
    // call, 60 with 2048 blocks of a head each).  A unit in many ranges: a block a head.
    const long long units = (long long)p.nb * a.Hkv * t.GC;
    const int heads = t.G < 8 * NT ? t.G : 8 * NT;
    p.heads = units >= grid / 4 ? heads : 1;
    const long long x = units * ((heads + p.heads - 1) / p.heads), blocks = 1 + (a.mass ? ((long long)t.max_chunks * 16 + kFinishThreads - 1) / kFinishThreads : 0);
    // Rows of blocks for the mass: six blocks an SM in all, as each finds the log-sum-exps for itself.  Of a row, one block a
    // (sequence, KV head) works, the first of its head blocks; the others return.  With a block a head (few units, long
    // caches) those that work are fewer by the number of heads: 112 for one sequence with 2 KV heads of 8 query heads each.
    const long long once = 1 + (6 * (long long)sm_count() + x - 1) / x;
    const unsigned y = (unsigned)(blocks < once ? blocks : (once < 65535 ? once : 65535));
    DFLASH_CUDA_CHECK(launch_chained(decode_finish_kernel<T, D, NT>, dim3((unsigned)x, y), kFinishThreads, p, stream));
    count_launch(2);
  }
  return DFLASH_OK;
}

template <typename T>
int32_t launch_dims(const CacheArgs& a, const Plan& t, cudaStream_t s) {
  if (t.NT == 1) {
    if (a.D == 64) return launch_typed<T, 64, 1>(a, t, s);
    if (a.D == 128) return launch_typed<T, 128, 1>(a, t, s);
    return launch_typed<T, 256, 1>(a, t, s);
  }
  if (a.D == 64) return launch_typed<T, 64, 2>(a, t, s);
  if (a.D == 128) return launch_typed<T, 128, 2>(a, t, s);
  return launch_typed<T, 256, 2>(a, t, s);
}

}  // namespace

size_t decode_workspace_bytes(int B, int Hq, int Hkv, int D, int N, int window, int sinks, bool with_mass) {
  return plan_of(B, Hq, Hkv, D, N, window, sinks, with_mass).total;
}

int32_t launch_decode(const CacheArgs& a, cudaStream_t stream) {
  const Plan t = plan_of(a.B, a.Hq, a.Hkv, a.D, a.N, a.window, a.sinks, a.mass != nullptr);
  return a.dtype == DFLASH_BF16 ? launch_dims<__nv_bfloat16>(a, t, stream) : launch_dims<__half>(a, t, stream);
}

}  // namespace dflash
