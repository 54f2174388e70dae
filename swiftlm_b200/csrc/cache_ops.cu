// Entry points of the operators on the KV cache outside the verify cycle: arguments checked here, kernels in
// decode_attn.cu, prompt_attn.cu and attn_mass.cu.  Every refusal happens before the device is touched.
#include "cache_ops.cuh"

namespace dflash {
namespace {

bool aligned(const void* p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

int32_t invalid(const char* op, const char* what) {
  set_error("%s: invalid argument: %s", op, what);
  return DFLASH_ERR_INVALID_ARG;
}

// What the three attention operators refuse alike; fills the parts of `a` that need no device.
int32_t check(const char* op, CacheArgs& a) {
  if (a.B <= 0 || a.Hq <= 0 || a.Hkv <= 0 || a.T <= 0 || a.D <= 0 || a.N <= 0) return invalid(op, "non-positive dimension");
  if (a.dtype != DFLASH_BF16 && a.dtype != DFLASH_F16) { set_error("%s: unsupported dtype %d (bf16 or f16)", op, a.dtype); return DFLASH_ERR_UNSUPPORTED; }
  if (a.D != 64 && a.D != 128 && a.D != 256) { set_error("%s: unsupported head_dim %d (64, 128 or 256)", op, a.D); return DFLASH_ERR_UNSUPPORTED; }
  if (a.Hq % a.Hkv != 0) { set_error("%s: unsupported heads: Hq=%d not a multiple of Hkv=%d", op, a.Hq, a.Hkv); return DFLASH_ERR_UNSUPPORTED; }
  if (a.N > kMaxTokens || a.T > kMaxTokens) { set_error("%s: unsupported length: N=%d, T=%d (at most 2^29)", op, a.N, a.T); return DFLASH_ERR_UNSUPPORTED; }
  if (a.window < 0 || a.sinks < 0) return invalid(op, "negative window or sinks");
  if (!(a.scale >= 1e-30f && a.scale <= 1e30f)) return invalid(op, "scale must be positive and finite");   // running maxima assume its sign
  if (a.page_table) {
    if (a.page_tokens <= 0 || a.max_pages <= 0 || a.num_pages <= 0 || (long long)a.max_pages * a.page_tokens < a.N)
      return invalid(op, "paged KV needs page_tokens, num_pages and max_pages * page_tokens >= N");
    if (a.page_tokens % 16 != 0) { set_error("%s: unsupported page_tokens %d (a multiple of 16)", op, a.page_tokens); return DFLASH_ERR_UNSUPPORTED; }
  } else {
    a.page_tokens = a.max_pages = a.num_pages = 0;
  }
  if (a.mass && a.mass_stride < a.N) return invalid(op, "mass_stride smaller than N");
  if (!aligned(a.q, 16) || !aligned(a.k, 16) || !aligned(a.v, 16) || !aligned(a.out, 16) || !aligned(a.workspace, 16))
    return invalid(op, "tensor base pointers must be 16-byte aligned");
  if (!aligned(a.lse, 4) || !aligned(a.mass, 4) || !aligned(a.page_table, 4) || !aligned(a.kv_len, 4) || !aligned(a.q_len, 4))
    return invalid(op, "misaligned pointer");
  // a position is below N, so a window of N tokens or more hides nothing
  if (a.window >= a.N) a.window = 0;
  if (a.sinks > a.N) a.sinks = a.N;
  return DFLASH_OK;
}

int32_t check_workspace(const char* op, const CacheArgs& a, size_t need) {
  if (need > 0 && (!a.workspace || a.workspace_bytes < need)) {
    set_error("%s: workspace of %zu bytes needed, %zu given", op, need, a.workspace ? a.workspace_bytes : (size_t)0);
    return DFLASH_ERR_WORKSPACE;
  }
  return DFLASH_OK;
}

// Outputs and workspace against each other and the inputs.  out may be q itself: a unit's queries are read before its rows are
// written, by the one CTA that has all of it or by the launch in front of the join.
int32_t check_apart(const char* op, const CacheArgs& a, bool lse_written, size_t workspace) {
  const unsigned long long rows = (unsigned long long)a.B * a.Hq * a.T, heads = (unsigned long long)a.B * a.Hkv, row_bytes = 2ull * a.D;
  const unsigned long long kv = a.page_table ? (unsigned long long)a.num_pages * a.Hkv * a.page_tokens * row_bytes : heads * a.N * row_bytes;
  const Span lse{a.lse, rows * 4}, none{nullptr, 0};
  const Span s[] = {{a.out, rows * row_bytes}, {a.mass, ((heads - 1) * a.mass_stride + a.N) * 4}, {a.workspace, workspace}, lse_written ? lse : none,
                    lse_written ? none : lse, {a.out == a.q ? nullptr : a.q, rows * row_bytes}, {a.k, kv}, {a.v, kv},
                    {a.page_table, 4ull * a.B * a.max_pages}, {a.q_len, 4ull * a.B}, {a.kv_len, 4ull * a.B}};
  return apart(s, 4) ? DFLASH_OK : invalid(op, "an output or the workspace overlaps another argument");
}

int32_t with_status(CacheArgs& a) {
  a.status = device_status_word();
  if (!a.status) { set_error("no CUDA device"); return DFLASH_ERR_CUDA; }
  return DFLASH_OK;
}

}  // namespace
}  // namespace dflash

using namespace dflash;

extern "C" {

int32_t dflash_decode_sdpa(const void* q, const void* k, const void* v, const int32_t* page_table, const int32_t* kv_len,
                           void* out, float* lse, float* mass, void* workspace, size_t workspace_bytes, int32_t B,
                           int32_t Hq, int32_t Hkv, int32_t D, int32_t N, int32_t page_tokens, int32_t max_pages,
                           int32_t num_pages, int32_t mass_stride, int32_t window, int32_t sinks, float scale,
                           int32_t dtype, void* stream) {
  const char* op = "decode_sdpa";
  if (!q || !k || !v || !out) return invalid(op, "null tensor pointer");
  CacheArgs a{q, k, v, page_table, nullptr, kv_len, out, lse, mass, workspace, workspace_bytes, B, Hq, Hkv, 1, D, N,
              page_tokens, max_pages, num_pages, mass_stride, window, sinks, scale, dtype, nullptr};
  if (int32_t st = check(op, a)) return st;
  const size_t need = decode_workspace_bytes(B, Hq, Hkv, D, N, a.window, a.sinks, mass != nullptr);
  if (int32_t st = check_workspace(op, a, need)) return st;
  if (int32_t st = check_apart(op, a, true, need)) return st;
  if (int32_t st = with_status(a)) return st;
  return launch_decode(a, reinterpret_cast<cudaStream_t>(stream));
}

size_t dflash_decode_sdpa_workspace_bytes(int32_t B, int32_t Hq, int32_t Hkv, int32_t D, int32_t N, int32_t window,
                                          int32_t sinks, int32_t with_mass) {
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || D <= 0 || N <= 0 || N > kMaxTokens || Hq % Hkv != 0 || window < 0 || sinks < 0) return 0;
  return decode_workspace_bytes(B, Hq, Hkv, D, N, window >= N ? 0 : window, sinks > N ? N : sinks, with_mass != 0);
}

int32_t dflash_prompt_sdpa(const void* q, const void* k, const void* v, const int32_t* page_table, const int32_t* q_len,
                           const int32_t* kv_len, void* out, float* lse, void* workspace, size_t workspace_bytes,
                           int32_t B, int32_t Hq, int32_t Hkv, int32_t T, int32_t D, int32_t N, int32_t page_tokens,
                           int32_t max_pages, int32_t num_pages, int32_t window, int32_t sinks, float scale,
                           int32_t dtype, void* stream) {
  const char* op = "prompt_sdpa";
  if (!q || !k || !v || !out) return invalid(op, "null tensor pointer");
  CacheArgs a{q, k, v, page_table, q_len, kv_len, out, lse, nullptr, workspace, workspace_bytes, B, Hq, Hkv, T, D, N,
              page_tokens, max_pages, num_pages, 0, window, sinks, scale, dtype, nullptr};
  if (int32_t st = check(op, a)) return st;
  const size_t need = prompt_workspace_bytes(B, Hq, Hkv, T, D, N);
  if (int32_t st = check_workspace(op, a, need)) return st;
  if (int32_t st = check_apart(op, a, true, need)) return st;
  if (int32_t st = with_status(a)) return st;
  return launch_prompt(a, reinterpret_cast<cudaStream_t>(stream));
}

size_t dflash_prompt_sdpa_workspace_bytes(int32_t B, int32_t Hq, int32_t Hkv, int32_t T, int32_t D, int32_t N) {
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || T <= 0 || D <= 0 || N <= 0 || N > kMaxTokens || T > kMaxTokens || Hq % Hkv != 0) return 0;
  return prompt_workspace_bytes(B, Hq, Hkv, T, D, N);
}

int32_t dflash_attention_mass(const void* q, const void* k, const int32_t* page_table, const int32_t* q_len,
                              const int32_t* kv_len, const float* lse, float* mass, void* workspace,
                              size_t workspace_bytes, int32_t B, int32_t Hq, int32_t Hkv, int32_t T, int32_t D, int32_t N,
                              int32_t page_tokens, int32_t max_pages, int32_t num_pages, int32_t mass_stride,
                              int32_t window, int32_t sinks, float scale, int32_t dtype, void* stream) {
  const char* op = "attention_mass";
  if (!q || !k || !lse || !mass) return invalid(op, "null tensor pointer");
  CacheArgs a{q, k, nullptr, page_table, q_len, kv_len, nullptr, const_cast<float*>(lse), mass, workspace, workspace_bytes,
              B, Hq, Hkv, T, D, N, page_tokens, max_pages, num_pages, mass_stride, window, sinks, scale, dtype, nullptr};
  if (int32_t st = check(op, a)) return st;
  const size_t need = mass_workspace_bytes(B, Hq, Hkv, T, D, N);
  if (int32_t st = check_workspace(op, a, need)) return st;
  if (int32_t st = check_apart(op, a, false, need)) return st;
  if (int32_t st = with_status(a)) return st;
  return launch_mass(a, reinterpret_cast<cudaStream_t>(stream));
}

size_t dflash_attention_mass_workspace_bytes(int32_t B, int32_t Hq, int32_t Hkv, int32_t T, int32_t D, int32_t N) {
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || T <= 0 || D <= 0 || N <= 0 || N > kMaxTokens || T > kMaxTokens || Hq % Hkv != 0) return 0;
  return mass_workspace_bytes(B, Hq, Hkv, T, D, N);
}

}  // extern "C"
