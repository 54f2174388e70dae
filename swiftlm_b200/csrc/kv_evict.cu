// Eviction from the KV cache by accumulated attention weight.
//
// For every (sequence, KV head) with n > budget tokens: keep the first S, the last R and the need = budget - S - R
// heaviest of the m = n - S - R between, move the kept rows to the front in the order they are in.
//
// select_kernel, one CTA per (sequence, KV head): the need-th largest mass by radix selection on the masses' bits
// (32-bit keys whose unsigned order is the floats' order; 11 + 11 + 10 bits, one histogram in shared memory per digit),
// then one pass that writes the kept places in ascending order by a block-wide count: a token stays when its key is above
// the threshold, or equal to it and among the first (need - above) equals.  No atomic decides an order, so ties
// go to the lowest index on every run.
// move_kernel: a kept row only moves towards the front (its new place j <= its old place idx[j]) and the places
// ascend, so a CTA that owns one column slice of one (sequence, KV head) may go through the rows in chunks in place:
// it loads a whole chunk, meets at a barrier, and stores it.  What later chunks still have to read lies at or behind their
// own places, in front of which the stores of this chunk end.
#include "common.cuh"

namespace dflash {
namespace {

struct EvictParams {
  uint8_t *k, *v;
  const int32_t *page_table, *kv_len;
  const float* mass;
  int32_t* kv_len_out;
  float* mass_out;
  int32_t* kept;          // [B*Hkv, kept_stride]
  int B, Hkv, N, page_tokens, max_pages, num_pages, mass_stride, budget, recent, sinks, kept_stride;
  int row_bytes;
  int* status;
};

constexpr int kSelThreads = 1024;

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
  uint32_t w = warp_sums[lane];
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

__global__ void __launch_bounds__(kSelThreads) select_kernel(const EvictParams p) {
  __shared__ uint32_t hist[2048];
  __shared__ uint32_t warp_sums[32];
  __shared__ uint32_t s_digit, s_left;
  const int b = blockIdx.y, h = blockIdx.x, tid = threadIdx.x;
  const long long unit = (long long)b * p.Hkv + h;
  int n = p.kv_len[b];
  if (n < 0 || n > p.N) {
    if (tid == 0 && h == 0) atomicExch(p.status, kStatusCacheLen);
    n = n < 0 ? 0 : p.N;
  }
  const float* mass = p.mass + unit * p.mass_stride;
  float* mass_out = p.mass_out + unit * p.mass_stride;
  int32_t* kept = p.kept + unit * p.kept_stride;
  const int left = n < p.budget ? n : p.budget;
  for (int i = left + tid; i < p.kept_stride; i += kSelThreads) kept[i] = -1;
  if (n <= p.budget) {
    for (int i = tid; i < n; i += kSelThreads) {
      kept[i] = i;
      mass_out[i] = mass[i];
    }
    return;
  }
  const int lo = p.sinks, hi = n - p.recent;
  uint32_t need = (uint32_t)(p.budget - p.sinks - p.recent);
  // ---- the need-th largest key of [lo, hi), digit by digit ----
  uint32_t threshold = 0, mask = 0;
  if (need > 0) {
#pragma unroll
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0), bins = pass == 2 ? 1024 : 2048;
      for (int i = tid; i < bins; i += kSelThreads) hist[i] = 0;
      __syncthreads();
      for (int i = lo + tid; i < hi; i += kSelThreads) {
        const uint32_t key = order_key(mass[i]);
        if ((key & mask) == threshold) atomicAdd(&hist[(key >> shift) & (bins - 1)], 1u);
      }
      __syncthreads();
      // from the top: the digit in which the running count reaches `need`
      const int per = bins / kSelThreads;                 // 2 or 1 bins a thread, thread 0 has the highest
      uint32_t c[2] = {hist[bins - 1 - tid * per], per == 2 ? hist[bins - 2 - tid * per] : 0u};
      uint32_t total;
      const uint32_t before = block_prefix(c[0] + c[1], total, warp_sums);
      if (before < need && need <= before + c[0]) { s_digit = bins - 1 - tid * per; s_left = need - before; }
      else if (before + c[0] < need && need <= before + c[0] + c[1]) { s_digit = bins - 2 - tid * per; s_left = need - before - c[0]; }
      __syncthreads();
      threshold |= s_digit << shift;
      mask |= (uint32_t)(bins - 1) << shift;
      need = s_left;
      __syncthreads();
    }
  }
  const uint32_t equals = need;                          // how many tokens equal to the threshold stay
  const bool any = p.budget > p.sinks + p.recent;
  // ---- kept places, ascending ----
  uint32_t done = 0, eq_done = 0;
  for (int base = 0; base < n; base += kSelThreads) {
    const int i = base + tid;
    float w = 0.f;
    bool sure = false, eq = false;
    if (i < n) {
      w = mass[i];
      if (i < lo || i >= hi) sure = true;
      else if (any) {
        const uint32_t key = order_key(w);
        sure = key > threshold;
        eq = key == threshold;
      }
    }
    uint32_t total;
    const uint32_t at = block_prefix((sure ? 1u : 0u) | (eq ? 0x10000u : 0u), total, warp_sums);
    const uint32_t eq_at = eq_done + (at >> 16);
    const uint32_t eq_before = eq_at < equals ? eq_at : equals;          // equals in front of this one that stay
    const uint32_t slot = done + (at & 0xffffu) + eq_before;              // done counts the sure ones only
    if (sure || (eq && eq_at < equals)) {
      kept[slot] = i;
      mass_out[slot] = w;                                               // slot <= i, and this chunk has been read
    }
    done += total & 0xffffu;
    eq_done += total >> 16;
    __syncthreads();
  }
  for (int i = left + tid; i < n; i += kSelThreads) mass_out[i] = 0.f;
}

__global__ void lens_kernel(const EvictParams p) {
  const int b = blockIdx.x * blockDim.x + threadIdx.x;
  if (b >= p.B) return;
  int n = p.kv_len[b];
  n = n < 0 ? 0 : (n > p.N ? p.N : n);
  p.kv_len_out[b] = n < p.budget ? n : p.budget;
}

// byte address of token n's row of (b, h), or -1
__device__ __forceinline__ long long row_at(const EvictParams& p, int b, int h, int n) {
  if (!p.page_table) return (((long long)b * p.Hkv + h) * p.N + n) * p.row_bytes;
  const int page = p.page_table[(long long)b * p.max_pages + n / p.page_tokens];
  if ((unsigned)page >= (unsigned)p.num_pages) {
    atomicExch(p.status, kStatusKvRange);
    return -1;
  }
  return (((long long)page * p.Hkv + h) * p.page_tokens + n % p.page_tokens) * p.row_bytes;
}

constexpr int kMoveThreads = 256, kMoveVecs = 4;
// One CTA: columns [16 * vecs * blockIdx.x, ...) of K (z = 0) or V (z = 1) of one (b, h).
__global__ void __launch_bounds__(kMoveThreads) move_kernel(const EvictParams p, int vecs) {
  const int unit = blockIdx.y, b = unit / p.Hkv, h = unit % p.Hkv;
  const int32_t* kept = p.kept + (long long)unit * p.kept_stride;
  uint8_t* x = blockIdx.z ? p.v : p.k;
  const int rows_per = kMoveThreads / vecs, col = (blockIdx.x * vecs + threadIdx.x % vecs) * 16;
  const int limit = p.kept_stride < p.budget ? p.kept_stride : p.budget;
  if (threadIdx.x / vecs >= rows_per) return;   // never: vecs is a power of two
  const bool live = col < p.row_bytes;
  for (int j0 = 0; j0 < limit; j0 += rows_per * kMoveVecs) {
    uint4 val[kMoveVecs];
    long long dst[kMoveVecs];
#pragma unroll
    for (int u = 0; u < kMoveVecs; ++u) {
      const int j = j0 + u * rows_per + threadIdx.x / vecs;
      dst[u] = -1;
      const int src = j < limit ? kept[j] : -1;
      if (live && src > j) {                     // src == j: the row is where it belongs
        const long long from = row_at(p, b, h, src), to = row_at(p, b, h, j);
        if (from >= 0 && to >= 0) {
          val[u] = *reinterpret_cast<const uint4*>(x + from + col);
          dst[u] = to + col;
        }
      }
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kMoveVecs; ++u)
      if (dst[u] >= 0) *reinterpret_cast<uint4*>(x + dst[u]) = val[u];
    __syncthreads();
  }
}

}  // namespace
}  // namespace dflash

extern "C" size_t dflash_kv_evict_workspace_bytes(int32_t B, int32_t Hkv, int32_t N, int32_t budget) {
  if (B <= 0 || Hkv <= 0 || N <= 0 || budget <= 0) return 0;
  return ((size_t)B * Hkv * (size_t)(budget < N ? budget : N) * 4 + 255) / 256 * 256;
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
  if (mass_stride < N) return invalid("mass_stride smaller than N");
  if (page_table && (page_tokens <= 0 || max_pages <= 0 || num_pages <= 0 || (long long)max_pages * page_tokens < N))
    return invalid("paged cache needs page_tokens, num_pages and max_pages * page_tokens >= N");
  const long long row_bytes = (long long)D * (dtype == DFLASH_F32 ? 4 : 2);
  auto off = [](const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) != 0; };
  if (row_bytes % 16 != 0 || row_bytes > (1 << 20) || off(k_cache, 16) || off(v_cache, 16))
    return invalid("rows must be multiples of 16 bytes (at most 1 MiB) and the caches 16-byte aligned");
  if (off(page_table, 4) || off(kv_len, 4) || off(mass, 4) || off(kv_len_out, 4) || off(mass_out, 4) || off(kept, 4) || off(workspace, 4))
    return invalid("misaligned pointer");
  if ((long long)B * Hkv > 65535 || B > 65535) { set_error("kv_evict: more than 65535 (sequence, head) pairs"); return DFLASH_ERR_UNSUPPORTED; }
  const int stride = kept ? budget : (budget < N ? budget : N);
  if (!kept) {
    const size_t need = dflash_kv_evict_workspace_bytes(B, Hkv, N, budget);
    if (!workspace || workspace_bytes < need) {
      set_error("kv_evict: workspace of %zu bytes needed, %zu given", need, workspace ? workspace_bytes : (size_t)0);
      return DFLASH_ERR_WORKSPACE;
    }
    kept = reinterpret_cast<int32_t*>(workspace);
  }
  int* status = device_status_word();
  if (!status) { set_error("no CUDA device"); return DFLASH_ERR_CUDA; }
  EvictParams p{reinterpret_cast<uint8_t*>(k_cache), reinterpret_cast<uint8_t*>(v_cache), page_table, kv_len, mass, kv_len_out, mass_out,
                kept, B, Hkv, N, page_tokens, max_pages, num_pages, mass_stride, budget, recent, sinks, stride, (int)row_bytes, status};
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  select_kernel<<<dim3(Hkv, B), kSelThreads, 0, s>>>(p);
  DFLASH_LAUNCH_CHECK();
  lens_kernel<<<(B + 127) / 128, 128, 0, s>>>(p);      // behind select_kernel, which reads kv_len: the two may be one array
  DFLASH_LAUNCH_CHECK();
  if (budget < N) {                                    // else no sequence can be longer than the budget
    const int vecs = 4;
    move_kernel<<<dim3((unsigned)((row_bytes / 16 + vecs - 1) / vecs), B * Hkv, 2), kMoveThreads, 0, s>>>(p, vecs);
    DFLASH_LAUNCH_CHECK();
    count_launch();
  }
  count_launch(2);
  return DFLASH_OK;
}
