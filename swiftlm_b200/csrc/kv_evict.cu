// Eviction from the KV cache by accumulated attention weight.
//
// For every (sequence, KV head) with n > budget tokens: keep the first S, the last R and the need = budget - S - R
// heaviest of the m = n - S - R between, move the kept rows to the front in the order they are in.
//
// select_kernel, one cluster of 1 to 8 CTAs per (sequence, KV head), a CTA for every 4096 tokens: the need-th largest mass by
// radix selection on the masses' bits (32-bit keys whose unsigned order is the floats' order; 11 + 11 + 10 bits, a
// histogram in each CTA's shared memory per digit, added up through distributed shared memory), then one pass that writes
// the kept places in ascending order by counts in front: a token stays when its key is above the threshold, or equal to it and
// among the first (need - above) equals.  No atomic decides an order, so ties go to the lowest index on every run.
// Up to 32768 tokens masses are read once and stay in shared memory, beyond that four times; one CTA for 32768 tokens took 38 us.
// move_kernel: a kept row only moves towards the front (its new place j <= its old place) and the places ascend,
// so a CTA that owns one column slice of one (sequence, KV head) may go through the rows in chunks in place: it loads a whole
// chunk, meets at a barrier, and stores it.  What later chunks still have to read lies at or behind their own places,
// in front of which the stores of this chunk end: the next chunk's loads are in flight while this one is stored, and one
// barrier a chunk is enough.  Bound by HBM: every row that moves is read once and written once.
//
// Measured (B200, the whole call; fp32 rows of as many bytes take the same): 32 sequences x 2 heads from 1104 to 1088 tokens
// (135 MB) 41 us, selection 11 and move 26 (20.6 at the HBM's rate); 8 x 2 heads from up to 32768 to 4096 53 us, selection 22 and move 27.  (With masses read once a digit, a
// second meeting a digit and places written by the threads that found them: 43 and 60 us.)
#include "cache_ops.cuh"
#include "ptx.cuh"

namespace dflash {
namespace {

struct EvictParams {
  uint8_t *k, *v;
  const int32_t *page_table, *kv_len;
  const float* mass;
  int32_t* kv_len_out;
  float* mass_out;
  int32_t* kept;          // [B*Hkv, budget] or null
  int2* moves;            // [B*Hkv] rows that stay, first of them that moves
  longlong2* places;      // [B*Hkv, stride] byte offsets of a row that stays: where it is, where it goes; .x < 0: nothing to do
  int B, Hkv, N, page_tokens, max_pages, num_pages, mass_stride, budget, recent, sinks, stride;
  int row_bytes;
  int* status;
  uint32_t page_mul, page_shift;
  // n / page_tokens for 0 <= n < 2^31: multiplication by a rounded-up 2^32+shift / page_tokens
  __device__ int by_page(int n) const { return (int)((__umulhi((uint32_t)n, page_mul) + (uint32_t)n) >> page_shift); }
};

constexpr int kMaxCluster = 8;
constexpr int kSelThreads = 512, kPer = 8, kChunk = kSelThreads * kPer;   // tokens of one CTA at a time

// unsigned order of the key = order of the float; -0 and +0 are equal, every NaN is above +inf
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// Sum over the CTA of two packed counts (each below 2^16 per chunk), exclusive prefix in `before`.
__device__ __forceinline__ uint32_t block_prefix(uint32_t mine, uint32_t& total, uint32_t* warp_sums) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t x = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  uint32_t w = lane < kSelThreads / 32 ? warp_sums[lane] : 0u;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, w, o);
    if (lane >= o) w += y;
  }
  total = __shfl_sync(0xffffffffu, w, 31);
  const uint32_t base = __shfl_sync(0xffffffffu, w, (warp + 31) & 31);
  __syncthreads();
  return x - mine + (warp ? base : 0u);
}

__device__ __forceinline__ void peer_add(const uint32_t* mine, uint32_t rank, uint32_t x) {
  asm volatile("red.shared::cluster.add.u32 [%0], %1;" ::"r"(ptx::cluster_addr(mine, rank)), "r"(x) : "memory");
}
__device__ __forceinline__ uint32_t peer_load(const uint32_t* mine, uint32_t rank) {   // the same word in CTA `rank` of the cluster
  uint32_t x;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(x) : "r"(ptx::cluster_addr(mine, rank)) : "memory");
  return x;
}

__global__ void __launch_bounds__(kSelThreads, 2) select_kernel(const EvictParams p, int C) {
  __shared__ uint32_t hist[2048], hist_all[5120];          // this CTA's counts; the cluster's, for each of the three digits
  __shared__ float vals[kChunk];                           // masses of this CTA's tokens of a round
  __shared__ uint32_t warp_sums[32];
  __shared__ uint32_t s_digit, s_left, s_count, s_counts[kMaxCluster], s_first;
  uint16_t* list = reinterpret_cast<uint16_t*>(hist);      // when the digits are known: tokens that stay, from the round's first
  static_assert(kChunk * sizeof(uint16_t) <= sizeof(hist) && kChunk <= 65536, "list");
  const int unit = blockIdx.x / C, b = unit / p.Hkv, h = unit - b * p.Hkv, tid = threadIdx.x;
  const uint32_t rank = blockIdx.x - unit * C;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  auto meet = [&]() {
    __syncwarp();
    if (C > 1) ptx::cluster_sync();
    else __syncthreads();
  };
  int n = p.kv_len[b];
  if (n < 0 || n > p.N) {
    if (tid == 0 && h == 0 && rank == 0) atomicExch(p.status, kStatusCacheLen);
    n = n < 0 ? 0 : p.N;
  }
  const float* mass = p.mass + (long long)unit * p.mass_stride;
  float* mass_out = p.mass_out + (long long)unit * p.mass_stride;
  int32_t* kept = p.kept ? p.kept + (long long)unit * p.budget : nullptr;
  longlong2* places = p.places + (long long)unit * p.stride;
  const int left = n < p.budget ? n : p.budget;
  const int all = tid + (int)rank * kSelThreads, stride = C * kSelThreads;
  if (kept)
    for (int i = left + all; i < p.budget; i += stride) kept[i] = -1;
  if (n <= p.budget) {                                      // the same in every CTA of the cluster
    for (int i = all; i < n; i += stride) {
      if (kept) kept[i] = i;
      mass_out[i] = mass[i];
    }
    if (all == 0) p.moves[unit] = make_int2(left, left);
    return;
  }
  const int lo = p.sinks, hi = n - p.recent;
  uint32_t need = (uint32_t)(p.budget - p.sinks - p.recent);
  if (tid == 0) s_first = (uint32_t)left;
  // A round is C * span tokens, CTA r of the cluster has the r-th span of it, a thread `per` of these in a row.  Up to
  // 4096 tokens a CTA there is one round, and the masses are read once.
  const int even = ((n - 1) / stride + 1) * kSelThreads, span = even < kChunk ? even : kChunk, per = span / kSelThreads;
  const bool once = n <= C * span;
  auto fetch = [&](int base) {                              // this thread reads back what it has written
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const int i = base + (int)rank * span + k * kSelThreads + tid;
      if (k < per) vals[k * kSelThreads + tid] = i < n ? mass[i] : 0.f;
    }
  };
  if (once) fetch(0);
  // ---- the need-th largest key of [lo, hi), digit by digit ----
  uint32_t threshold = 0, mask = 0;
  if (need > 0) {
    for (int i = tid; i < 2048; i += kSelThreads) hist[i] = 0;
    for (int i = tid; i < 5120; i += kSelThreads) hist_all[i] = 0;
    meet();
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0), bins = pass == 2 ? 1024 : 2048, bins_thread = bins / kSelThreads;
      uint32_t* sums = hist_all + pass * 2048;
      uint32_t* mine = C > 1 ? hist : sums;
      for (int base = 0; base < n; base += C * span) {
        if (!once) fetch(base);
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
          const int i = base + (int)rank * span + k * kSelThreads + tid;
          if (k >= per || i < lo || i >= hi) continue;
          const uint32_t key = order_key(vals[k * kSelThreads + tid]);
          if ((key & mask) == threshold) atomicAdd(&mine[(key >> shift) & (bins - 1)], 1u);
        }
      }
      if (C > 1) {
        // Masses have few leading digits: a CTA adds its few counts to every CTA's sums.  (Each thread reading its bins
        // from eight CTAs took 14000 clocks a digit.)
        __syncthreads();
        for (int i = tid; i < bins; i += kSelThreads) {
          const uint32_t c = hist[i];
          if (c) {
            for (int r = 0; r < C; ++r) peer_add(&sums[i], r, c);
            hist[i] = 0;
          }
        }
      }
      meet();
      // from the top: the digit in which the running count reaches `need`; thread 0 has the highest of 4 or 2 bins a thread
      const int top = bins - 1 - tid * bins_thread;
      uint32_t c[4], total;
#pragma unroll
      for (int j = 0; j < 4; ++j) c[j] = j < bins_thread ? sums[top - j] : 0u;
      uint32_t before = block_prefix(c[0] + c[1] + c[2] + c[3], total, warp_sums);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (before < need && need <= before + c[j]) { s_digit = top - j; s_left = need - before; }
        before += c[j];
      }
      __syncthreads();
      threshold |= s_digit << shift;
      mask |= (uint32_t)(bins - 1) << shift;
      need = s_left;
    }
  }
  const uint32_t equals = need;                          // how many tokens equal to the threshold stay
  const bool any = p.budget > p.sinks + p.recent;
  // ---- kept places, ascending ----
  uint32_t done = 0, eq_done = 0, first = 0xffffffffu;
  for (int base = 0; base < n; base += C * span) {
    const int from = base + (int)rank * span;
    if (!once) fetch(base);
    __syncthreads();
    uint32_t sure = 0, eq = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int at = tid * per + j, i = from + at;
      if (j >= per || i >= n) continue;
      if (i < lo || i >= hi) sure |= 1u << j;
      else if (any) {
        const uint32_t key = order_key(vals[at]);
        sure |= key > threshold ? 1u << j : 0u;
        eq |= key == threshold ? 1u << j : 0u;
      }
    }
    uint32_t total;                                       // both counts of a span are at most 4096
    const uint32_t at = block_prefix(__popc(sure) | (__popc(eq) << 16), total, warp_sums);
    if (tid == 0) s_count = total;
    meet();                                               // every CTA has read its span and counted
    if (tid < C) s_counts[tid] = C == 1 ? total : peer_load(&s_count, tid);
    __syncthreads();
    uint32_t cta_sure = done, cta_eq = eq_done;
    for (int r = 0; r < C; ++r) {
      const uint32_t c = s_counts[r];
      if (r < (int)rank) { cta_sure += c & 0xffffu; cta_eq += c >> 16; }
      done += c & 0xffffu;
      eq_done += c >> 16;
    }
    // What stays of a span goes to places in a row: first into a list, so that the rows are shared out evenly below (few threads
    // have many, where much stays; most have none, where little does).
    auto place = [&](uint32_t n_sure, uint32_t n_eq) { return n_sure + (n_eq < equals ? n_eq : equals); };
    const uint32_t slot0 = place(cta_sure, cta_eq), slot1 = place(cta_sure + (total & 0xffffu), cta_eq + (total >> 16));
    uint32_t sure_at = cta_sure + (at & 0xffffu), eq_at = cta_eq + (at >> 16);
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const bool s = (sure >> j) & 1u, e = (eq >> j) & 1u;
      if (s || (e && eq_at < equals)) list[place(sure_at, eq_at) - slot0] = (uint16_t)(tid * per + j);
      sure_at += s;
      eq_at += e;
    }
    __syncthreads();
    // Addresses are looked up here, once a row, and not by every thread that moves a part of it.
    const int32_t* table = p.page_table ? p.page_table + (long long)b * p.max_pages : nullptr;
#pragma unroll 2
    for (int slot = (int)slot0 + tid; slot < (int)slot1; slot += kSelThreads) {
      const int at = list[slot - slot0], i = from + at;
      if (kept) kept[slot] = i;
      mass_out[slot] = vals[at];                          // slot <= token, and this round has been read
      longlong2 at2 = make_longlong2(-1, -1);
      if (slot != i) {
        if ((uint32_t)slot < first) first = (uint32_t)slot;
        if (!table) {
          const long long row = (long long)unit * p.N;
          at2 = make_longlong2((row + i) * p.row_bytes, (row + slot) * p.row_bytes);
        } else {
          const int page_i = p.by_page(i), page_s = p.by_page(slot), pf = table[page_i], pt = table[page_s];
          if ((unsigned)pf >= (unsigned)p.num_pages || (unsigned)pt >= (unsigned)p.num_pages) {
            atomicExch(p.status, kStatusKvRange);         // a page outside the pool: the row is skipped
          } else {
            at2 = make_longlong2((((long long)pf * p.Hkv + h) * p.page_tokens + i - page_i * p.page_tokens) * p.row_bytes,
                                 (((long long)pt * p.Hkv + h) * p.page_tokens + slot - page_s * p.page_tokens) * p.row_bytes);
          }
        }
      }
      places[slot] = at2;
    }
    if (!once) meet();                                    // the counts, the masses and the list are used again
  }
  first = __reduce_min_sync(0xffffffffu, first);
  if ((tid & 31) == 0 && first != 0xffffffffu) atomicMin(&s_first, first);
  for (int i = left + all; i < n; i += stride) mass_out[i] = 0.f;
  meet();
  // the first row that moves
  if (rank == 0 && tid < 32) {
    uint32_t x = tid < C ? (C == 1 ? s_first : peer_load(&s_first, tid)) : 0xffffffffu;
    x = __reduce_min_sync(0xffffffffu, x);
    if (tid == 0) p.moves[unit] = make_int2(left, (int)x);
  }
  meet();                                                 // no CTA leaves while another reads its shared memory
}

// Rows a thread has in flight in one chunk, with 64 bytes of a row a CTA (`vecs` below).  Measured, the whole call, at 32 x 2
// heads from 1104 to 1088 tokens, 8 x 2 from up to 32768 to 4096 (512-byte rows both) and 8 x 8 from up to 4000 to 2000 (128-byte
// rows): 4 rows 41, 53 and 29 us, 2 rows 39, 65 and 34, 8 rows 46, 68 and 35; 32 bytes a CTA 45, 61 and 33, 128 bytes 41, 63 and 35.
constexpr int kMoveThreads = 256, kMoveRows = 4;
// One CTA: `vecs` 16-byte columns from vecs * blockIdx.x on, of K (z = 0) or V (z = 1) of one (b, h).
__global__ void __launch_bounds__(kMoveThreads) move_kernel(const EvictParams p, int vecs) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int unit = blockIdx.y, b = unit / p.Hkv, h = unit - b * p.Hkv;
  const int2 range = p.moves[unit];
  if (blockIdx.x == 0 && blockIdx.z == 0 && h == 0 && threadIdx.x == 0) p.kv_len_out[b] = range.x;   // kv_len may be the same array
  const int per = kMoveThreads / vecs, row = threadIdx.x / vecs, col = (blockIdx.x * vecs + threadIdx.x - row * vecs) * 16;
  const longlong2* places = p.places + (long long)unit * p.stride + row;
  uint8_t* x = (blockIdx.z ? p.v : p.k) + col;
  const int end = col < p.row_bytes ? range.x - row : 0, chunk = per * kMoveRows;
  if (range.y >= range.x) return;                // nothing moves
  // Three chunks are under way: the places of one are read, the rows of the next are loaded, those of the last stored.
  longlong2 at[kMoveRows];
  uint4 val[2][kMoveRows];
  long long to[2][kMoveRows];
  auto read = [&](int j0) {
#pragma unroll
    for (int u = 0; u < kMoveRows; ++u) at[u] = j0 + u * per < end ? places[j0 + u * per] : make_longlong2(-1, -1);
  };
  auto load = [&](uint4 (&v)[kMoveRows], long long (&t)[kMoveRows]) {
#pragma unroll
    for (int u = 0; u < kMoveRows; ++u) {
      t[u] = at[u].x >= 0 ? at[u].y : -1;
      if (at[u].x >= 0) v[u] = *reinterpret_cast<const uint4*>(x + at[u].x);
    }
  };
  auto store = [&](const uint4 (&v)[kMoveRows], const long long (&t)[kMoveRows]) {
#pragma unroll
    for (int u = 0; u < kMoveRows; ++u)
      if (t[u] >= 0) *reinterpret_cast<uint4*>(x + t[u]) = v[u];
  };
  read(range.y);
  load(val[0], to[0]);
  read(range.y + chunk);
  for (int j0 = range.y; j0 < range.x; j0 += 2 * chunk) {
    __syncthreads();
    load(val[1], to[1]);
    read(j0 + 2 * chunk);
    store(val[0], to[0]);
    __syncthreads();
    load(val[0], to[0]);
    read(j0 + 3 * chunk);
    store(val[1], to[1]);
  }
}

}  // namespace
}  // namespace dflash

static size_t moves_bytes(int B, int Hkv) { return ((size_t)B * Hkv * sizeof(int2) + 255) / 256 * 256; }

extern "C" size_t dflash_kv_evict_workspace_bytes(int32_t B, int32_t Hkv, int32_t N, int32_t budget) {
  if (B <= 0 || Hkv <= 0 || N <= 0 || N > dflash::kMaxTokens || budget <= 0) return 0;
  return moves_bytes(B, Hkv) + (size_t)B * Hkv * (size_t)(budget < N ? budget : N) * sizeof(longlong2);
}

extern "C" int32_t dflash_kv_evict(void* k_cache, void* v_cache, const int32_t* page_table, const int32_t* kv_len, const float* mass,
                                   int32_t* kv_len_out, float* mass_out, int32_t* kept, void* workspace, size_t workspace_bytes,
                                   int32_t B, int32_t Hkv, int32_t D, int32_t N, int32_t page_tokens, int32_t max_pages,
                                   int32_t num_pages, int32_t mass_stride, int32_t budget, int32_t recent, int32_t sinks,
                                   int32_t dtype, void* stream) {
  using namespace dflash;
  auto invalid = [](const char* what) { set_error("kv_evict: invalid argument: %s", what); return (int32_t)DFLASH_ERR_INVALID_ARG; };
  if (!k_cache || !v_cache || !kv_len || !mass || !kv_len_out || !mass_out) return invalid("null pointer");
  if (B <= 0 || Hkv <= 0 || D <= 0 || N <= 0) return invalid("non-positive dimension");
  if (dtype != DFLASH_BF16 && dtype != DFLASH_F16 && dtype != DFLASH_F32) { set_error("kv_evict: unsupported dtype %d", dtype); return DFLASH_ERR_UNSUPPORTED; }
  if (budget <= 0 || recent < 0 || sinks < 0 || (long long)recent + sinks > budget) return invalid("need budget > 0 and sinks + recent <= budget");
  if (N > kMaxTokens) { set_error("kv_evict: unsupported length N=%d (at most 2^29)", N); return DFLASH_ERR_UNSUPPORTED; }
  if (mass_stride < N) return invalid("mass_stride smaller than N");
  if (page_table && (page_tokens <= 0 || max_pages <= 0 || num_pages <= 0 || (long long)max_pages * page_tokens < N))
    return invalid("paged cache needs page_tokens, num_pages and max_pages * page_tokens >= N");
  const long long row_bytes = (long long)D * (dtype == DFLASH_F32 ? 4 : 2);
  auto off = [](const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) != 0; };
  if (row_bytes % 16 != 0 || row_bytes > (1 << 20) || off(k_cache, 16) || off(v_cache, 16))
    return invalid("rows must be multiples of 16 bytes (at most 1 MiB) and the caches 16-byte aligned");
  if (off(page_table, 4) || off(kv_len, 4) || off(mass, 4) || off(kv_len_out, 4) || off(mass_out, 4) || off(kept, 4) || off(workspace, 16))
    return invalid("misaligned pointer");
  if ((long long)B * Hkv > 65535) { set_error("kv_evict: more than 65535 (sequence, head) pairs"); return DFLASH_ERR_UNSUPPORTED; }
  const size_t need = dflash_kv_evict_workspace_bytes(B, Hkv, N, budget);
  if (!workspace || workspace_bytes < need) {
    set_error("kv_evict: workspace of %zu bytes needed, %zu given", need, workspace ? workspace_bytes : (size_t)0);
    return DFLASH_ERR_WORKSPACE;
  }
  // kv_len_out and mass_out may be kv_len and mass; two arrays of masses may lie in each other's gaps
  const unsigned long long heads = (unsigned long long)B * Hkv, mass_bytes = ((heads - 1) * mass_stride + N) * 4;
  const unsigned long long kv = (page_table ? (unsigned long long)num_pages * Hkv * page_tokens : heads * N) * row_bytes;
  const Span old{mass == mass_out ? nullptr : mass, mass_bytes};
  const Span s[] = {{k_cache, kv}, {v_cache, kv}, {kv_len_out, 4ull * B}, {kept, heads * budget * 4}, {workspace, need}, {mass_out, mass_bytes},
                    {kv_len == kv_len_out ? nullptr : kv_len, 4ull * B}, {page_table, 4ull * B * max_pages}};
  bool ok = apart(s, 6);
  for (int i = 0; i < 5; ++i) ok = ok && !s[i].meets(old);
  if (s[5].meets(old)) {
    const unsigned long long a = reinterpret_cast<uintptr_t>(mass), b = reinterpret_cast<uintptr_t>(mass_out), row = 4ull * mass_stride;
    const unsigned long long off = (a < b ? b - a : a - b) % row;
    ok = ok && off >= 4ull * N && row - off >= 4ull * N;
  }
  if (!ok) return invalid("an output or the workspace overlaps another argument");
  int* status = device_status_word();
  if (!status) { set_error("no CUDA device"); return DFLASH_ERR_CUDA; }
  EvictParams p{reinterpret_cast<uint8_t*>(k_cache), reinterpret_cast<uint8_t*>(v_cache), page_table, kv_len, mass, kv_len_out, mass_out,
                kept, reinterpret_cast<int2*>(workspace),
                reinterpret_cast<longlong2*>(reinterpret_cast<uint8_t*>(workspace) + moves_bytes(B, Hkv)), B, Hkv, N, page_tokens, max_pages, num_pages, mass_stride, budget, recent, sinks,
                budget < N ? budget : N, (int)row_bytes, status, 0, 0};
  if (page_table) {
    while ((1ull << p.page_shift) < (uint64_t)page_tokens) ++p.page_shift;
    p.page_mul = (uint32_t)(((1ull << 32) * ((1ull << p.page_shift) - (uint64_t)page_tokens)) / (uint64_t)page_tokens + 1);
  }
  int C = 1;
  while (C < kMaxCluster && N > C * kChunk) C *= 2;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = C;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cfg.stream = reinterpret_cast<cudaStream_t>(stream);
  cfg.gridDim = dim3(B * Hkv * C);
  cfg.blockDim = dim3(kSelThreads);
  DFLASH_CUDA_CHECK(cudaLaunchKernelEx(&cfg, select_kernel, p, C));
  const int vecs = 4;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3((unsigned)((row_bytes / 16 + vecs - 1) / vecs), B * Hkv, 2);
  cfg.blockDim = dim3(kMoveThreads);
  DFLASH_CUDA_CHECK(cudaLaunchKernelEx(&cfg, move_kernel, p, vecs));
  count_launch(2);
  return DFLASH_OK;
}
