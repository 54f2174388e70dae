// The weights of the cached tokens, first form: one warp per cached token, lanes split the head dimension.
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
int32_t mass_typed(const CacheArgs& a, const float* lse, cudaStream_t s) {
  const unsigned grid = (unsigned)(((long long)a.B * a.Hkv * a.N + 3) / 4);
  if (a.D == 64) mass_kernel<T, 64><<<grid, 128, 0, s>>>(a, lse);
  else if (a.D == 128) mass_kernel<T, 128><<<grid, 128, 0, s>>>(a, lse);
  else mass_kernel<T, 256><<<grid, 128, 0, s>>>(a, lse);
  DFLASH_LAUNCH_CHECK();
  count_launch();
  return DFLASH_OK;
}
int32_t mass_any(const CacheArgs& a, const float* lse, cudaStream_t s) {
  return a.dtype == DFLASH_BF16 ? mass_typed<__nv_bfloat16>(a, lse, s) : mass_typed<__half>(a, lse, s);
}

}  // namespace

size_t mass_workspace_bytes(int, int, int, int, int, int) { return 0; }
int32_t launch_mass(const CacheArgs& a, cudaStream_t s) { return mass_any(a, a.lse, s); }

}  // namespace dflash
