// Attention over the KV cache, first form: one warp per (sequence, query head, row) walks the row's visible tokens with
// a running maximum and sum; lanes split the head dimension.  Weights: one warp per cached token.
#include "cache_ops.cuh"

namespace dflash {
namespace {

template <typename T, int D>
__device__ __forceinline__ void load_row(const T* p, float (&x)[D / 32], int lane) {
#pragma unroll
  for (int i = 0; i < D / 32; ++i) x[i] = to_f32(p[lane * (D / 32) + i]);
}

__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

template <typename T, int D>
__global__ void __launch_bounds__(128) rows_kernel(const CacheArgs a, float* lse_out) {
  const int lane = threadIdx.x & 31;
  const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (row >= (long long)a.B * a.Hq * a.T) return;
  const int r = (int)(row % a.T), hq = (int)(row / a.T % a.Hq), b = (int)(row / a.T / a.Hq);
  const int h = hq / (a.Hq / a.Hkv);
  const RowLens len = lens_of(a, b, hq == 0 && r == 0 && lane == 0);
  if (r >= len.rows) return;
  const int p = len.keys - len.rows + r;
  float q[D / 32], o[D / 32] = {};
  load_row<T, D>(reinterpret_cast<const T*>(a.q) + row * D, q, lane);
  float m = -INFINITY, l = 0.f;
  for (int n = 0; n <= p; ++n) {
    if (!sees(a, p, n)) {
      n = p - a.window;       // the next one is the first token of the window
      if (n + 1 > p) break;
      continue;
    }
    const long long at = kv_row(a, b, h, n);
    float kx[D / 32] = {}, vx[D / 32] = {};
    if (at >= 0) {
      load_row<T, D>(reinterpret_cast<const T*>(a.k) + at * D, kx, lane);
      load_row<T, D>(reinterpret_cast<const T*>(a.v) + at * D, vx, lane);
    }
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) s = fmaf(q[i], kx[i], s);
    s = warp_sum(s) * a.scale;
    const float m2 = fmaxf(m, s), f = expf(m - m2), w = expf(s - m2);
    l = l * f + w;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) o[i] = fmaf(w, vx[i], o[i] * f);
    m = m2;
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
  for (int i = 0; i < D / 32; ++i) reinterpret_cast<T*>(a.out)[row * D + lane * (D / 32) + i] = from_f32<T>(o[i] * inv);
  if (lse_out && lane == 0) lse_out[row] = l > 0.f ? m + logf(l) : -INFINITY;
}

template <typename T, int D>
__global__ void __launch_bounds__(128) mass_kernel(const CacheArgs a, const float* lse) {
  const int lane = threadIdx.x & 31;
  const long long item = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (item >= (long long)a.B * a.Hkv * a.N) return;
  const int n = (int)(item % a.N), h = (int)(item / a.N % a.Hkv), b = (int)(item / a.N / a.Hkv);
  const RowLens len = lens_of(a, b, n == 0 && h == 0 && lane == 0);
  if (n >= len.keys) return;
  const long long at = kv_row(a, b, h, n);
  float kx[D / 32] = {};
  if (at >= 0) load_row<T, D>(reinterpret_cast<const T*>(a.k) + at * D, kx, lane);
  const int G = a.Hq / a.Hkv;
  float total = 0.f;
  for (int g = 0; g < G; ++g)
    for (int r = 0; r < len.rows; ++r) {
      if (!sees(a, len.keys - len.rows + r, n)) continue;
      const long long row = ((long long)b * a.Hq + h * G + g) * a.T + r;
      float q[D / 32];
      load_row<T, D>(reinterpret_cast<const T*>(a.q) + row * D, q, lane);
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) s = fmaf(q[i], kx[i], s);
      s = warp_sum(s) * a.scale;
      const float z = lse[row];
      if (z > -INFINITY) total += expf(s - z);
    }
  if (lane == 0) a.mass[((long long)b * a.Hkv + h) * a.mass_stride + n] += total;
}

template <typename T>
int32_t rows_typed(const CacheArgs& a, float* lse, cudaStream_t s) {
  const unsigned grid = (unsigned)(((long long)a.B * a.Hq * a.T + 3) / 4);
  if (a.D == 64) rows_kernel<T, 64><<<grid, 128, 0, s>>>(a, lse);
  else if (a.D == 128) rows_kernel<T, 128><<<grid, 128, 0, s>>>(a, lse);
  else rows_kernel<T, 256><<<grid, 128, 0, s>>>(a, lse);
  DFLASH_LAUNCH_CHECK();
  count_launch();
  return DFLASH_OK;
}
template <typename T>
int32_t mass_typed(const CacheArgs& a, const float* lse, cudaStream_t s) {
  const unsigned grid = (unsigned)(((long long)a.B * a.Hkv * a.N + 3) / 4);
  if (a.D == 64) mass_kernel<T, 64><<<grid, 128, 0, s>>>(a, lse);
  else if (a.D == 128) mass_kernel<T, 128><<<grid, 128, 0, s>>>(a, lse);
  else mass_kernel<T, 256><<<grid, 128, 0, s>>>(a, lse);
  DFLASH_LAUNCH_CHECK();
  count_launch();
  return DFLASH_OK;
}
int32_t rows_any(const CacheArgs& a, float* lse, cudaStream_t s) {
  return a.dtype == DFLASH_BF16 ? rows_typed<__nv_bfloat16>(a, lse, s) : rows_typed<__half>(a, lse, s);
}
int32_t mass_any(const CacheArgs& a, const float* lse, cudaStream_t s) {
  return a.dtype == DFLASH_BF16 ? mass_typed<__nv_bfloat16>(a, lse, s) : mass_typed<__half>(a, lse, s);
}

}  // namespace

size_t prompt_workspace_bytes(int, int, int, int, int, int) { return 0; }
int32_t launch_prompt(const CacheArgs& a, cudaStream_t s) { return rows_any(a, a.lse, s); }
size_t mass_workspace_bytes(int, int, int, int, int, int) { return 0; }
int32_t launch_mass(const CacheArgs& a, cudaStream_t s) { return mass_any(a, a.lse, s); }

}  // namespace dflash
