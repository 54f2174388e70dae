// Shared by the operators on the KV cache outside the verify cycle (decode_attn.cu, prompt_attn.cu, attn_mass.cu):
// arguments, lengths and visibility.
#pragma once

#include <atomic>

#include "common.cuh"

namespace dflash {

struct CacheArgs {
  const void *q, *k, *v;
  const int32_t *page_table, *q_len, *kv_len;
  void* out;
  float* lse;          // decode / prompt: output or null; mass: input
  float* mass;
  void* workspace;
  size_t workspace_bytes;
  int B, Hq, Hkv, T, D, N;
  int page_tokens, max_pages, num_pages, mass_stride;
  int window, sinks;   // window <= N (0: none), sinks <= N
  float scale;
  int dtype;
  int* status;
};

constexpr int kMaxTokens = 1 << 29;   // N and T at most: sums of two positions and a window stay in 32 bits

struct RowLens { int keys, rows; };   // cached tokens, query rows in use

// Lengths of sequence b, clamped to [0, N] and [0, T]; one thread of the grid passes report = true.
__device__ __forceinline__ RowLens lens_of(const CacheArgs& a, int b, bool report = false) {
  int n = a.kv_len ? a.kv_len[b] : a.N, t = a.q_len ? a.q_len[b] : a.T;
  const int n0 = n, t0 = t;
  n = n < 0 ? 0 : (n > a.N ? a.N : n);
  t = t < 0 ? 0 : (t > a.T ? a.T : t);
  if (report && (n != n0 || t != t0)) atomicExch(a.status, kStatusCacheLen);
  return RowLens{n, t};
}

// Row index (in rows of D elements) of token n of (b, h); -1: the page is outside the pool.  n < N.
__device__ __forceinline__ long long kv_row(const CacheArgs& a, int b, int h, int n) {
  if (!a.page_table) return ((long long)b * a.Hkv + h) * a.N + n;
  const int page = a.page_table[(long long)b * a.max_pages + n / a.page_tokens];
  if ((unsigned)page >= (unsigned)a.num_pages) {
    atomicExch(a.status, kStatusKvRange);
    return -1;
  }
  return ((long long)page * a.Hkv + h) * a.page_tokens + n % a.page_tokens;
}

__device__ __forceinline__ bool sees(const CacheArgs& a, int p, int n) {
  return n <= p && (a.window == 0 || n > p - a.window || n < a.sinks);
}

// A range of memory that a call reads or writes, for the refusal of calls that would read what they have written.
struct Span {
  const void* at;
  unsigned long long bytes;
  bool meets(const Span& o) const {
    const uintptr_t a = reinterpret_cast<uintptr_t>(at), b = reinterpret_cast<uintptr_t>(o.at);
    return at && o.at && a < b + o.bytes && b < a + bytes;
  }
};
// The first `written` of the spans meet none of the others?
template <int N>
inline bool apart(const Span (&s)[N], int written) {
  for (int i = 0; i < written; ++i)
    for (int j = i + 1; j < N; ++j)
      if (s[i].meets(s[j])) return false;
  return true;
}

// Dynamic shared memory of a kernel, set once per device (a driver call of a microsecond); `ready` belongs to the kernel.
template <typename F>
inline cudaError_t allow_shared(std::atomic<uint64_t>& ready, F kernel, int bytes) {
  int dev = 0;
  if (cudaError_t e = cudaGetDevice(&dev)) return e;
  if (dev < 64 && (ready.load(std::memory_order_acquire) >> dev & 1)) return cudaSuccess;
  if (cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes)) return e;
  if (dev < 64) ready.fetch_or(1ull << dev, std::memory_order_release);
  return cudaSuccess;
}

size_t decode_workspace_bytes(int B, int Hq, int Hkv, int D, int N, int window, int sinks, bool with_mass);
int32_t launch_decode(const CacheArgs& a, cudaStream_t stream);
size_t prompt_workspace_bytes(int B, int Hq, int Hkv, int T, int D, int N);
int32_t launch_prompt(const CacheArgs& a, cudaStream_t stream);
size_t mass_workspace_bytes(int B, int Hq, int Hkv, int T, int D, int N);
int32_t launch_mass(const CacheArgs& a, cudaStream_t stream);

}  // namespace dflash
