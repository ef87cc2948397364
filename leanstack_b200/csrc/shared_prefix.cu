// Attention of a batch whose sequences share a prefix held once (head_dim 128).
//
// Query row (token i of sequence b, head h) attends over the P keys of the
// shared prefix of its kv head and over keys 0 .. cache_pos[b] + i of its own
// static cache strip, one softmax over both (the mask of
// src/leanstack/runtime/qwen_explicit.py:551-563 with the prefix in front).
//
// One CTA per (token, query head): four warps take every fourth key, each lane
// four of the 128 dims, online softmax in fp32 (base 2), merged in shared
// memory.  Every row reads the prefix for itself.
#include "common.cuh"

namespace lsb {

constexpr int kSpHeadDim = 128;

struct SpParams {
  const __nv_bfloat16* q;         // [M, Hq, D]
  const __nv_bfloat16* k_prefix;  // [Hkv, prefix_cap, D]
  const __nv_bfloat16* v_prefix;
  const __nv_bfloat16* k_cache;   // [B, Hkv, S, D]
  const __nv_bfloat16* v_cache;
  const int* cache_pos;           // [B] or null (then uniform_past)
  int uniform_past;
  __nv_bfloat16* out;             // [M, Hq * D]
  int* err;
  int q_len, Hq, Hkv, G, P, prefix_cap, max_seq;
  float scale_log2;
};

__global__ void __launch_bounds__(128) shared_prefix_attention_kernel(SpParams p) {
  __shared__ float sm_m[4], sm_l[4], sm_o[4][kSpHeadDim];
  grid_dep_wait();
  grid_dep_launch();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int t = blockIdx.x, h = blockIdx.y, hkv = h / p.G;
  const int b = t / p.q_len, i = t - b * p.q_len;
  const int cp = p.cache_pos ? p.cache_pos[b] : p.uniform_past;
  if ((cp < 0 || cp > p.max_seq - p.q_len) && threadIdx.x == 0) raise_device_error(p.err, LS_ERR_KV_OVERFLOW);
  const int own = min(max(min(cp, p.max_seq) + i + 1, 0), p.max_seq);
  const size_t pbase = (size_t)hkv * p.prefix_cap * kSpHeadDim;
  const size_t cbase = ((size_t)b * p.Hkv + hkv) * p.max_seq * kSpHeadDim;
  const uint2 qu = *reinterpret_cast<const uint2*>(p.q + ((size_t)t * p.Hq + h) * kSpHeadDim + lane * 4);
  float m = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f, o2 = 0.f, o3 = 0.f;
  for (int j = warp; j < p.P + own; j += 4) {
    const size_t off = (j < p.P ? pbase + (size_t)j * kSpHeadDim : cbase + (size_t)(j - p.P) * kSpHeadDim) + lane * 4;
    const uint2 ku = *reinterpret_cast<const uint2*>((j < p.P ? p.k_prefix : p.k_cache) + off);
    const uint2 vu = *reinterpret_cast<const uint2*>((j < p.P ? p.v_prefix : p.v_cache) + off);
    float s = bf16_lo(qu.x) * bf16_lo(ku.x) + bf16_hi(qu.x) * bf16_hi(ku.x) + bf16_lo(qu.y) * bf16_lo(ku.y) +
              bf16_hi(qu.y) * bf16_hi(ku.y);
    s = warp_sum(s) * p.scale_log2;
    const float mn = fmaxf(m, s);
    if (mn == -INFINITY) continue;
    const float c = exp2f(m - mn), e = exp2f(s - mn);
    m = mn;
    l = l * c + e;
    o0 = o0 * c + e * bf16_lo(vu.x);
    o1 = o1 * c + e * bf16_hi(vu.x);
    o2 = o2 * c + e * bf16_lo(vu.y);
    o3 = o3 * c + e * bf16_hi(vu.y);
  }
  if (lane == 0) sm_m[warp] = m, sm_l[warp] = l;
  *reinterpret_cast<float4*>(&sm_o[warp][lane * 4]) = make_float4(o0, o1, o2, o3);
  __syncthreads();
  const float mx = fmaxf(fmaxf(sm_m[0], sm_m[1]), fmaxf(sm_m[2], sm_m[3]));
  float ls = 0.f, acc = 0.f;
  if (mx != -INFINITY)
    for (int w = 0; w < 4; ++w) {
      const float c = exp2f(sm_m[w] - mx);
      ls += sm_l[w] * c;
      acc += sm_o[w][threadIdx.x] * c;
    }
  p.out[((size_t)t * p.Hq + h) * kSpHeadDim + threadIdx.x] = f_to_bf16(ls > 0.f ? acc / ls : 0.f);
}

}  // namespace lsb

namespace lsb_host {
using namespace lsb;

int shared_prefix_workspace_bytes(int64_t batch, int64_t q_len, int64_t hq, int64_t hkv, int64_t prefix_len,
                                  int64_t* bytes) {
  (void)batch, (void)q_len, (void)hq, (void)hkv, (void)prefix_len;
  *bytes = 0;
  return LS_OK;
}

int launch_shared_prefix_attention(const void* q, const void* k_prefix, const void* v_prefix, int64_t prefix_len,
                                   int64_t prefix_cap, const void* k_cache, const void* v_cache,
                                   const int32_t* cache_pos, int64_t uniform_past, int64_t batch, int64_t q_len,
                                   int64_t hq, int64_t hkv, int64_t max_seq, float scale, void* out, void* workspace,
                                   cudaStream_t stream) {
  (void)workspace;
  SpParams p = {};
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.k_prefix = static_cast<const __nv_bfloat16*>(k_prefix);
  p.v_prefix = static_cast<const __nv_bfloat16*>(v_prefix);
  p.k_cache = static_cast<const __nv_bfloat16*>(k_cache);
  p.v_cache = static_cast<const __nv_bfloat16*>(v_cache);
  p.cache_pos = cache_pos;
  p.uniform_past = (int)uniform_past;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.err = device_error_ptr();
  p.q_len = (int)q_len;
  p.Hq = (int)hq;
  p.Hkv = (int)hkv;
  p.G = (int)(hq / hkv);
  p.P = (int)prefix_len;
  p.prefix_cap = (int)prefix_cap;
  p.max_seq = (int)max_seq;
  p.scale_log2 = scale * 1.4426950408889634f;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(batch * q_len), (unsigned)hq);
  cfg.blockDim = dim3(128);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, shared_prefix_attention_kernel, p);
  return e == cudaSuccess ? LS_OK : set_error(LS_ERR_CUDA, "shared_prefix_attention launch: %s", cudaGetErrorString(e));
}

}  // namespace lsb_host

using namespace lsb_host;

extern "C" {

int ls_shared_prefix_attention_workspace_bytes(int64_t batch, int64_t q_len, int64_t num_heads, int64_t num_kv_heads,
                                               int64_t head_dim, int64_t prefix_len, int64_t* bytes) {
  LS_REQUIRE(bytes, LS_ERR_INVALID_ARGUMENT, "ls_shared_prefix_attention_workspace_bytes: bytes is null");
  LS_REQUIRE(head_dim == 128, LS_ERR_UNSUPPORTED_SHAPE, "head_dim=%lld (only 128 is implemented)",
             (long long)head_dim);
  LS_REQUIRE(batch > 0 && batch <= 65535 && q_len > 0 && q_len < (1ll << 31) && num_kv_heads > 0 && num_heads > 0 &&
                 num_heads <= 65535 && num_heads % num_kv_heads == 0 && prefix_len >= 0 && prefix_len < (1ll << 30),
             LS_ERR_INVALID_ARGUMENT, "ls_shared_prefix_attention_workspace_bytes: bad sizes");
  return shared_prefix_workspace_bytes(batch, q_len, num_heads, num_kv_heads, prefix_len, bytes);
}

int ls_shared_prefix_attention(const void* q, const void* k_prefix, const void* v_prefix, int64_t prefix_len,
                               int64_t prefix_cap, const void* k_cache, const void* v_cache, const int32_t* cache_pos,
                               int64_t uniform_past, int64_t batch, int64_t q_len, int64_t num_heads,
                               int64_t num_kv_heads, int64_t head_dim, int64_t max_seq, float scale, void* out,
                               void* workspace, int64_t workspace_bytes, ls_stream_t stream) {
  LS_REQUIRE(q && k_cache && v_cache && out, LS_ERR_INVALID_ARGUMENT, "ls_shared_prefix_attention: null pointer");
  int64_t need = 0;
  int rc = ls_shared_prefix_attention_workspace_bytes(batch, q_len, num_heads, num_kv_heads, head_dim, prefix_len,
                                                      &need);
  if (rc) return rc;
  LS_REQUIRE(prefix_len == 0 || (k_prefix && v_prefix), LS_ERR_INVALID_ARGUMENT,
             "ls_shared_prefix_attention: prefix_len=%lld without prefix pointers", (long long)prefix_len);
  LS_REQUIRE(prefix_len <= prefix_cap && prefix_cap < (1ll << 30), LS_ERR_KV_OVERFLOW,
             "prefix_len=%lld beyond prefix_cap=%lld", (long long)prefix_len, (long long)prefix_cap);
  LS_REQUIRE(max_seq > 0 && max_seq < (1ll << 30) && batch * q_len < (1ll << 31), LS_ERR_INVALID_ARGUMENT,
             "ls_shared_prefix_attention: bad sizes");
  LS_REQUIRE(cache_pos || (uniform_past >= 0 && uniform_past + q_len <= max_seq), LS_ERR_KV_OVERFLOW,
             "uniform_past=%lld + q_len=%lld beyond max_seq=%lld", (long long)uniform_past, (long long)q_len,
             (long long)max_seq);
  LS_REQUIRE(aligned16(q) && aligned16(k_prefix) && aligned16(v_prefix) && aligned16(k_cache) && aligned16(v_cache) &&
                 aligned16(out) && aligned16(workspace),
             LS_ERR_MISALIGNED, "ls_shared_prefix_attention: pointers must be 16-byte aligned");
  LS_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), LS_ERR_WORKSPACE,
             "ls_shared_prefix_attention: workspace needs %lld bytes", (long long)need);
  return launch_shared_prefix_attention(q, k_prefix, v_prefix, prefix_len, prefix_cap, k_cache, v_cache, cache_pos,
                                        uniform_past, batch, q_len, num_heads, num_kv_heads, max_seq, scale, out,
                                        workspace, (cudaStream_t)stream);
}

}  // extern "C"
