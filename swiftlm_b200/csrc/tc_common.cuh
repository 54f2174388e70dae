// What the tcgen05 kernels on the KV cache share (prompt_attn.cu, attn_mass.cu): operand descriptors, tiles, tensor maps.
#pragma once

#include <cuda.h>

#include <type_traits>

#include "cache_ops.cuh"
#include "mma_sync.cuh"
#include "ptx.cuh"

namespace dflash {
namespace tc {

constexpr int kRows = 128, kKeys = 128;       // rows of a query tile, keys of a key tile
constexpr int kChunk = 128 * 128;             // bytes of 128 rows x 64 16-bit elements, 128-byte swizzle

// shared-memory operand: start address, leading / stride byte offsets (all >> 4), descriptor version 1, 128-byte swizzle
__device__ __forceinline__ uint64_t make_desc(uint32_t smem_addr, uint32_t lbo_bytes, uint32_t sbo_bytes) {
  return (uint64_t)((smem_addr & 0x3FFFFu) >> 4) | ((uint64_t)(lbo_bytes >> 4) << 16) | ((uint64_t)(sbo_bytes >> 4) << 32) |
         (1ull << 46) | (2ull << 61);
}
// fp32 accumulator, A and B of type T, both K-major unless b_mn
template <typename T>
__host__ __device__ constexpr uint32_t idesc(int m, int n, bool b_mn) {
  const uint32_t f = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  return (1u << 4) | (f << 7) | (f << 10) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

// packed fp32: (x, y) * s + (u, v) and (x, y) + (u, v), one instruction each
__device__ __forceinline__ float2 fma2v(float x, float y, float s, float u, float v) {
  return __ffma2_rn(make_float2(x, y), make_float2(s, s), make_float2(u, v));
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) { return __fadd2_rn(a, b); }

// Rows of a query tile: the Gt query heads of one KV head for consecutive tokens, head fastest, so that a tile spans as
// few positions as possible and a group of heads fills it even when there are few tokens.
struct Tiling {
  int G, Gt, GC, Tt;           // heads per KV head; heads in a tile; head groups; tokens in a tile (Gt * Tt <= 128)
};
inline Tiling tiling_of(int Hq, int Hkv) {
  Tiling t;
  t.G = Hq / Hkv;
  t.GC = (t.G + kRows - 1) / kRows;
  t.Gt = (t.G + t.GC - 1) / t.GC;
  t.Tt = kRows / t.Gt;
  return t;
}

// The key tiles that the tokens [t0, t1) of a sequence see between them: `head` tiles of the sinks, then tiles
// first, first + 1, ...
struct KeyTiles { int head, first, count; };
__device__ __forceinline__ KeyTiles key_tiles(const CacheArgs& a, RowLens len, int t0, int t1) {
  KeyTiles k{0, 0, 1};
  const int p0 = len.keys - len.rows + t0, p1 = len.keys - len.rows + t1 - 1;
  if (p1 < 0) return k;                                   // nothing visible: one tile, all of it masked
  const int lo = a.window > 0 && p0 - a.window + 1 > 0 ? p0 - a.window + 1 : 0;
  const int s = a.sinks < lo ? a.sinks : lo;
  k.first = lo / kKeys;
  k.head = (s + kKeys - 1) / kKeys;
  if (k.head > k.first) k.head = k.first;
  k.count = k.head + p1 / kKeys - k.first + 1;
  return k;
}
__device__ __forceinline__ int tile_key(const KeyTiles& k, int c) { return (c < k.head ? c : k.first + c - k.head) * kKeys; }

inline int box_rows(const CacheArgs& a) {                  // rows of one copy: a page holds a whole number of them
  if (!a.page_table) return kKeys;
  int h = kKeys;
  while (a.page_tokens % h) h >>= 1;
  return h;                                               // 16 .. 128: page_tokens is a multiple of 16
}

// 64-element columns of keys / values: (d, token, head, sequence or page).  Tokens behind the array and a page id at or
// behind num_pages read as zeros.
inline CUresult encode_kv(CUtensorMap* m, const void* base, const CacheArgs& a, int rows) {
  EncodeTiledFn encode = tensor_map_encoder();
  if (!encode) return CUDA_ERROR_NOT_FOUND;
  const cuuint64_t n = a.page_table ? a.page_tokens : a.N, outer = a.page_table ? a.num_pages : a.B;
  const cuuint64_t dims[4] = {(cuuint64_t)a.D, n, (cuuint64_t)a.Hkv, outer};
  const cuuint64_t strides[3] = {(cuuint64_t)a.D * 2, n * a.D * 2, (cuuint64_t)a.Hkv * n * a.D * 2};
  const cuuint32_t box[4] = {64, (cuuint32_t)rows, 1, 1}, es[4] = {1, 1, 1, 1};
  return encode(m, a.dtype == DFLASH_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                const_cast<void*>(base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
}
// queries as (d, head, token, sequence x KV head), box (64, Gt, Tt): rows in the order of Tiling
inline CUresult encode_q(CUtensorMap* m, const CacheArgs& a, const Tiling& t) {
  EncodeTiledFn encode = tensor_map_encoder();
  if (!encode) return CUDA_ERROR_NOT_FOUND;
  const cuuint64_t dims[4] = {(cuuint64_t)a.D, (cuuint64_t)t.G, (cuuint64_t)a.T, (cuuint64_t)a.B * a.Hkv};
  const cuuint64_t strides[3] = {(cuuint64_t)a.T * a.D * 2, (cuuint64_t)a.D * 2, (cuuint64_t)t.G * a.T * a.D * 2};
  const cuuint32_t box[4] = {64, (cuuint32_t)t.Gt, (cuuint32_t)t.Tt, 1}, es[4] = {1, 1, 1, 1};
  return encode(m, a.dtype == DFLASH_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                const_cast<void*>(a.q), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
}

// Where the copy that starts at token n of sequence b begins.  Tokens at and behind `len` may be anything that was in the
// cache; their pages are not looked up.
struct TilePlace { int row, outer; };
__device__ __forceinline__ TilePlace place_of(const CacheArgs& a, int b, int n, int len) {
  if (!a.page_table) return TilePlace{n, b};
  TilePlace t{n % a.page_tokens, a.num_pages};            // behind the pool: zeros
  if (n < len) {
    const int page = a.page_table[(long long)b * a.max_pages + n / a.page_tokens];
    if ((unsigned)page < (unsigned)a.num_pages) t.outer = page;
    else atomicExch(a.status, kStatusKvRange);
  }
  return t;
}

}  // namespace tc
}  // namespace dflash
