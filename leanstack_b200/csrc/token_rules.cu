// Rules on the next token: penalties for repeated tokens, biases and grammar
// masks on a row of logits, then the greedy pick (lowest id on ties).
//
// Per allowed token v of row b, in fp32 and in this order, each step rounded:
//   l = logit;  seen: l = l > 0 ? l / repetition : l * repetition;
//   count > 0:  l = (l - frequency * count) - presence;
//   l = l + (the row's biases of v, added in list order).
// Tokens whose grammar bit is clear are no candidates, whatever their logit
// holds, and read -inf in the optional output; NaN is never picked.  A row
// with no candidate gives -1.
//
// Seen tokens (prompt or answer) and grammars are bit sets of 32-bit words, so
// an unmasked bf16 row costs 2 bytes and two bits a token and the counts are
// read only where the seen bit is set; groups of 8 tokens that the grammar
// bans outright are not read at all.  The groups are aligned in the flattened
// [m, vocab] array, not in the row, so that every vocabulary size takes 16-byte
// accesses; a group's bits are cut from two words.  A row is split over a
// cluster of CTAs whose winners meet in the first CTA's shared memory: no
// workspace, no counters, so captured graphs share nothing.  A thread keeps
// several groups in flight: the bound is the chain bits -> logits -> counts of dependent
// loads for few rows, and HBM for many.
#include "common.cuh"

namespace lsb {

constexpr int kTrMaxThreads = 512;
constexpr int kTrMaxCluster = 16;

struct TrParams {
  const void* logits;        // [M, V] bf16 or fp32
  int* counts;               // [M, V] or null
  uint32_t* seen;            // [M, W] or null
  const float* repetition;   // [M] or null (1)
  const float* frequency;    // [M] or null (0)
  const float* presence;     // [M] or null (0)
  const int* bias_ids;       // [M, bias_cap] or null; entries outside the vocabulary are skipped
  const float* bias_values;  // [M, bias_cap]
  const uint32_t* allowed;   // [M, W] or null (all)
  int64_t* out_ids;          // [M]
  float* out_logits;         // [M, V] or null
  int V, W, bias_cap, record;
};

// 8 consecutive logits as loaded, and as fp32.
template <typename T>
struct TrRaw {};
template <>
struct TrRaw<__nv_bfloat16> {
  uint4 v;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { v = ldg16(p); }  // 16-byte aligned
  __device__ __forceinline__ void load(const __nv_bfloat16* p, int lo, int hi) {  // elements lo .. hi - 1 only
    uint32_t h[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) h[j] = j >= lo && j < hi ? (uint32_t)__bfloat16_as_ushort(p[j]) : 0u;
    v = make_uint4(h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16);
  }
  __device__ __forceinline__ void get(float f[8]) const { unpack8(v, f); }
};
template <>
struct TrRaw<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = *reinterpret_cast<const float4*>(p);
    b = *reinterpret_cast<const float4*>(p + 4);
  }
  __device__ __forceinline__ void load(const float* p, int lo, int hi) {
    float f[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = j >= lo && j < hi ? p[j] : 0.f;
    a = make_float4(f[0], f[1], f[2], f[3]);
    b = make_float4(f[4], f[5], f[6], f[7]);
  }
  __device__ __forceinline__ void get(float f[8]) const {
    f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
  }
};

// Bits v0 .. v0 + 7 of a set of `words` words (v0 >= -7); bits outside are 0.
__device__ __forceinline__ uint32_t tr_bits8(const uint32_t* set, int words, int v0) {
  const int w = v0 >> 5, sh = v0 & 31;
  const uint32_t lo = w >= 0 && w < words ? set[w] : 0u;
  const uint32_t hi = sh > 24 && w + 1 < words ? set[w + 1] : 0u;
  return __funnelshift_r(lo, hi, sh) & 0xffu;
}

__device__ __forceinline__ bool tr_better(float v, int i, float best, int besti) {
  return v > best || (v == best && i < besti);
}

template <typename T>
__global__ void __launch_bounds__(kTrMaxThreads, 2) constrained_argmax_kernel(TrParams p) {
  extern __shared__ uint32_t tr_bias[];  // bit set of this CTA's biased tokens (bias lists only)
  __shared__ float bv[kTrMaxThreads / 32], cv[kTrMaxCluster];
  __shared__ int bi[kTrMaxThreads / 32], ci[kTrMaxCluster];
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");  // this CTA is running
  grid_dep_wait();
  grid_dep_launch();
  const int row = blockIdx.y, c = blockIdx.x, ncta = gridDim.x, nt = blockDim.x;
  // Groups of 8 flattened indices; the row's first and last group may reach into
  // its neighbours.  Group g of the row starts at token 8 g - a.
  const long long row0 = (long long)row * p.V;
  const int a = (int)(row0 & 7), ngroups = (p.V + a + 7) / 8;
  // The CTAs take tiles of nt groups (a power of two) in turn: frequent tokens have
  // low ids, and with them the counts to read.
  constexpr int kGroups = sizeof(T) == 2 ? 4 : 2;  // groups in flight per thread
  const int lg = __ffs(nt) - 1, tiles = (ngroups + nt - 1) >> lg;
  const T* logits = static_cast<const T*>(p.logits) + row0;
  const uint32_t* seen = p.seen ? p.seen + (size_t)row * p.W : nullptr;
  const uint32_t* allowed = p.allowed ? p.allowed + (size_t)row * p.W : nullptr;
  const int* counts = p.counts + row0;
  float* out = p.out_logits ? p.out_logits + row0 : nullptr;
  const bool last_row = row == (int)gridDim.y - 1;
  const int* bias_ids = p.bias_ids + (size_t)row * p.bias_cap;
  // Biased tokens as bits of the CTA's own tiles, 8 a group.
  unsigned char* bias_bits = reinterpret_cast<unsigned char*>(tr_bias);
  if (p.bias_cap) {
    for (int w = threadIdx.x; w < ((tiles + ncta - 1) / ncta << lg) / 4; w += nt) tr_bias[w] = 0u;
    __syncthreads();
    for (int k = threadIdx.x; k < p.bias_cap; k += nt) {
      const int v = bias_ids[k], g = (v + a) >> 3, tile = g >> lg;
      if (v < 0 || v >= p.V || tile % ncta != c) continue;
      const int at = (tile / ncta << lg) + (g & (nt - 1));
      atomicOr(&tr_bias[at >> 2], 1u << ((at & 3) * 8 + ((v + a) & 7)));
    }
    __syncthreads();
  }
  const float rep = p.repetition ? p.repetition[row] : 1.f;
  const float freq = p.frequency ? p.frequency[row] : 0.f;
  const float pres = p.presence ? p.presence[row] : 0.f;
  float best = -INFINITY;
  int besti = 0x7fffffff;
  for (int tile = c; tile < tiles; tile += kGroups * ncta) {
    uint32_t ab[kGroups], sb[kGroups];
    int n0[kGroups];  // count of the group's first seen token
    TrRaw<T> raw[kGroups];
#pragma unroll
    for (int u = 0; u < kGroups; ++u) {
      const int g = ((tile + u * ncta) << lg) + threadIdx.x, v0 = g * 8 - a;
      const uint32_t live = g >= ngroups ? 0u : (v0 < 0 ? 0xffu << -v0 & 0xffu : p.V - v0 >= 8 ? 0xffu : (1u << (p.V - v0)) - 1u);
      ab[u] = live && allowed ? tr_bits8(allowed, p.W, v0) & live : live;
      sb[u] = live && seen ? tr_bits8(seen, p.W, v0) : 0u;
    }
#pragma unroll
    for (int u = 0; u < kGroups; ++u) {
      const int v0 = (((tile + u * ncta) << lg) + (int)threadIdx.x) * 8 - a;
      sb[u] &= ab[u];
      if (ab[u] == 0u) continue;
      if (sb[u]) n0[u] = counts[v0 + __ffs(sb[u]) - 1];
      if (last_row && v0 + 8 > p.V) raw[u].load(logits + v0, max(-v0, 0), p.V - v0);  // the array ends inside the group
      else raw[u].load(logits + v0);
    }
#pragma unroll
    for (int u = 0; u < kGroups; ++u) {
      const int lt = (tile + u * ncta) / ncta;  // tile = c + lt ncta
      const int g = ((tile + u * ncta) << lg) + threadIdx.x, v0 = g * 8 - a;
      if (g >= ngroups) break;
      float f[8];
      if (ab[u]) {
        raw[u].get(f);
        // Few tokens are seen or biased: one at a time, not eight predicated divisions.
        for (uint32_t m = sb[u]; m; m &= m - 1u) {
          const int j = __ffs(m) - 1, n = m == sb[u] ? n0[u] : counts[v0 + j];
          float x = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (e == j) x = f[e];
          x = x > 0.f ? x / rep : __fmul_rn(x, rep);
          if (n > 0) x = __fsub_rn(__fsub_rn(x, __fmul_rn(freq, (float)n)), pres);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (e == j) f[e] = x;
        }
        for (uint32_t m = p.bias_cap ? bias_bits[(lt << lg) + threadIdx.x] & ab[u] : 0u; m; m &= m - 1u) {
          const int j = __ffs(m) - 1;
          float add = 0.f;  // the token's biases in list order
          for (int k = 0; k < p.bias_cap; ++k)
            if (bias_ids[k] == v0 + j) add = __fadd_rn(add, p.bias_values[(size_t)row * p.bias_cap + k]);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (e == j) f[e] = __fadd_rn(f[e], add);
        }
      }
      if (ab[u] != 0xffu) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (!(ab[u] >> j & 1u)) f[j] = -INFINITY;
      }
      // The group's maximum (NaN drops out); a thread meets its tokens in order, so
      // a later equal one does not win.  -inf counts while there is nothing else.
      const float top = fmaxf(fmaxf(fmaxf(f[0], f[1]), fmaxf(f[2], f[3])), fmaxf(fmaxf(f[4], f[5]), fmaxf(f[6], f[7])));
      if (top > best || (besti == 0x7fffffff && ab[u])) {
#pragma unroll
        for (int j = 7; j >= 0; --j)
          if (f[j] == top && (ab[u] >> j & 1u)) best = top, besti = v0 + j;
      }
      if (out) {
        if (v0 >= 0 && v0 + 8 <= p.V) {
          *reinterpret_cast<float4*>(out + v0) = make_float4(f[0], f[1], f[2], f[3]);
          *reinterpret_cast<float4*>(out + v0 + 4) = make_float4(f[4], f[5], f[6], f[7]);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (v0 + j >= 0 && v0 + j < p.V) out[v0 + j] = f[j];
        }
      }
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float ov = __shfl_xor_sync(0xffffffffu, best, o);
    const int oi = __shfl_xor_sync(0xffffffffu, besti, o);
    if (tr_better(ov, oi, best, besti)) best = ov, besti = oi;
  }
  if ((threadIdx.x & 31) == 0) bv[threadIdx.x >> 5] = best, bi[threadIdx.x >> 5] = besti;
  __syncthreads();
  asm volatile("barrier.cluster.wait.aligned;" ::: "memory");  // the first CTA runs: its shared memory may be written
  if (threadIdx.x == 0) {
    for (int w = 1; w < nt / 32; ++w)
      if (tr_better(bv[w], bi[w], best, besti)) best = bv[w], besti = bi[w];
    uint32_t rv, ri;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(rv) : "r"(smem_u32(&cv[c])));
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(ri) : "r"(smem_u32(&ci[c])));
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(rv), "f"(best) : "memory");
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(ri), "r"(besti) : "memory");
  }
  // Every CTA's winner is in place and every read of the row's state is done.
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (c != 0 || threadIdx.x != 0) return;
  for (int w = 0; w < ncta; ++w)
    if (w == 0 || tr_better(cv[w], ci[w], best, besti)) best = cv[w], besti = ci[w];
  const bool found = besti != 0x7fffffff;
  p.out_ids[row] = found ? besti : -1;
  if (p.record && found) {  // atomics only so that nothing waits for the old value
    atomicAdd(p.counts + row0 + besti, 1);
    atomicOr(p.seen + (size_t)row * p.W + besti / 32, 1u << (besti & 31));
  }
}

// Tokens of each sequence into its seen bits and, for an answer's tokens, its
// counts.  Negative ids are padding; ids past the vocabulary are reported.
constexpr int kTsThreads = 256;
__global__ void __launch_bounds__(kTsThreads) token_stats_add_kernel(const int64_t* ids, int len, int V, int W,
                                                                     int* counts, uint32_t* seen, int* err) {
  grid_dep_wait();
  grid_dep_launch();
  const int row = blockIdx.y;
  for (int i = blockIdx.x * kTsThreads + threadIdx.x; i < len; i += gridDim.x * kTsThreads) {
    const int64_t v = ids[(size_t)row * len + i];
    if (v < 0) continue;
    if (v >= V) {
      raise_device_error(err, LS_ERR_INVALID_ARGUMENT);
      continue;
    }
    atomicOr(seen + (size_t)row * W + v / 32, 1u << (v & 31));
    if (counts) atomicAdd(counts + (size_t)row * V + v, 1);
  }
}

}  // namespace lsb

namespace lsb_host {
using namespace lsb;

template <typename T>
static int launch_constrained_argmax(const TrParams& p, int64_t m, cudaStream_t stream) {
  static bool configured[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    cudaError_t e =
        cudaFuncSetAttribute(constrained_argmax_kernel<T>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return set_error(LS_ERR_CUDA, "constrained_argmax attribute: %s", cudaGetErrorString(e));
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  // Threads of a row: what the GPU holds at once (1024 an SM at 64 registers) over
  // the rows, between 8 x 128 and 16 x 512.
  const int64_t share = 1024 * (int64_t)sm_count() / m;
  const int cluster = share >= 16 * 512 ? 16 : 8;
  const int threads = share >= 8 * 512 ? 512 : share >= 8 * 256 ? 256 : 128;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)cluster, (unsigned)m);
  cfg.blockDim = dim3((unsigned)threads);
  // One byte of bias bits per group of the CTA's tiles.
  const int64_t tiles = ((int64_t)(p.V + 14) / 8 + threads - 1) / threads;
  cfg.dynamicSmemBytes = p.bias_cap ? (size_t)((tiles + cluster - 1) / cluster * threads) : 0;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  cudaError_t e = cudaLaunchKernelEx(&cfg, constrained_argmax_kernel<T>, p);
  return e == cudaSuccess ? LS_OK : set_error(LS_ERR_CUDA, "constrained_argmax launch: %s", cudaGetErrorString(e));
}

// Largest vocabulary: the bias bit set of one CTA (vocab / 8 / cluster bytes)
// stays within the 48 KB of shared memory that need no opt-in.
constexpr int64_t kTrMaxVocab = 1 << 21;

}  // namespace lsb_host

using namespace lsb_host;

extern "C" {

int ls_constrained_argmax(const void* logits, int logits_f32, int64_t m, int64_t vocab, int32_t* counts, uint32_t* seen,
                          const float* repetition, const float* frequency, const float* presence,
                          const int32_t* bias_ids, const float* bias_values, int64_t bias_cap, const uint32_t* allowed,
                          int record, int64_t* out_ids, float* out_logits, ls_stream_t stream) {
  LS_REQUIRE(logits && out_ids, LS_ERR_INVALID_ARGUMENT, "ls_constrained_argmax: null pointer");
  LS_REQUIRE(m > 0 && m <= 65535 && vocab > 0, LS_ERR_INVALID_ARGUMENT, "ls_constrained_argmax: bad sizes");
  LS_REQUIRE(vocab <= kTrMaxVocab, LS_ERR_UNSUPPORTED_SHAPE, "ls_constrained_argmax: vocab=%lld beyond %lld",
             (long long)vocab, (long long)kTrMaxVocab);
  LS_REQUIRE((counts == nullptr) == (seen == nullptr), LS_ERR_INVALID_ARGUMENT,
             "ls_constrained_argmax: counts and seen come together");
  LS_REQUIRE(counts || !(repetition || frequency || presence || record), LS_ERR_INVALID_ARGUMENT,
             "ls_constrained_argmax: penalties and record need counts and seen");
  LS_REQUIRE((bias_ids == nullptr) == (bias_values == nullptr) && (bias_ids != nullptr) == (bias_cap > 0) &&
                 bias_cap >= 0 && bias_cap < (1ll << 31),
             LS_ERR_INVALID_ARGUMENT, "ls_constrained_argmax: bias_ids, bias_values and bias_cap come together");
  LS_REQUIRE(aligned16(logits) && aligned16(out_logits), LS_ERR_MISALIGNED,
             "ls_constrained_argmax: logits must be 16-byte aligned");
  TrParams p = {};
  p.logits = logits;
  p.counts = counts;
  p.seen = seen;
  p.repetition = repetition;
  p.frequency = frequency;
  p.presence = presence;
  p.bias_ids = bias_ids;
  p.bias_values = bias_values;
  p.allowed = allowed;
  p.out_ids = out_ids;
  p.out_logits = out_logits;
  p.V = (int)vocab;
  p.W = (int)((vocab + 31) / 32);
  p.bias_cap = (int)bias_cap;
  p.record = record ? 1 : 0;
  return logits_f32 ? launch_constrained_argmax<float>(p, m, (cudaStream_t)stream)
                    : launch_constrained_argmax<__nv_bfloat16>(p, m, (cudaStream_t)stream);
}

int ls_token_stats_add(const int64_t* ids, int64_t batch, int64_t len, int64_t vocab, int32_t* counts, uint32_t* seen,
                       ls_stream_t stream) {
  LS_REQUIRE(ids && seen, LS_ERR_INVALID_ARGUMENT, "ls_token_stats_add: null pointer");
  LS_REQUIRE(batch > 0 && batch <= 65535 && len > 0 && len < (1ll << 31) && vocab > 0 && vocab <= kTrMaxVocab,
             LS_ERR_INVALID_ARGUMENT, "ls_token_stats_add: bad sizes");
  const int64_t blocks = (len + kTsThreads - 1) / kTsThreads;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(blocks < 64 ? blocks : 64), (unsigned)batch);
  cfg.blockDim = dim3(kTsThreads);
  cfg.stream = (cudaStream_t)stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, token_stats_add_kernel, ids, (int)len, (int)vocab,
                                     (int)((vocab + 31) / 32), counts, seen, device_error_ptr());
  return e == cudaSuccess ? LS_OK : set_error(LS_ERR_CUDA, "token_stats_add launch: %s", cudaGetErrorString(e));
}

}  // extern "C"
