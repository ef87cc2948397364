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
// bans outright are not read at all.  A row is split over a cluster of CTAs
// whose winners meet in the first CTA's shared memory: no workspace, no
// counters, so captured graphs share nothing.
#include "common.cuh"

namespace lsb {

constexpr int kTrThreads = 256;
constexpr int kTrCluster = 8;

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

template <typename T>
__device__ __forceinline__ void tr_load8(const T* row, int v0, int V, bool vec, float f[8]);
template <>
__device__ __forceinline__ void tr_load8(const __nv_bfloat16* row, int v0, int V, bool vec, float f[8]) {
  if (vec) {
    unpack8(ldg16(row + v0), f);
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = v0 + j < V ? bf16_to_f(row[v0 + j]) : 0.f;
}
template <>
__device__ __forceinline__ void tr_load8(const float* row, int v0, int V, bool vec, float f[8]) {
  if (vec) {
    const float4 a = *reinterpret_cast<const float4*>(row + v0), b = *reinterpret_cast<const float4*>(row + v0 + 4);
    f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = v0 + j < V ? row[v0 + j] : 0.f;
}

__device__ __forceinline__ bool tr_better(float v, int i, float best, int besti) {
  return v > best || (v == best && i < besti);
}

template <typename T>
__global__ void __launch_bounds__(kTrThreads) constrained_argmax_kernel(TrParams p) {
  extern __shared__ uint32_t tr_bias[];  // bit set of this CTA's biased tokens (bias lists only)
  __shared__ float bv[kTrThreads / 32], cv[kTrCluster];
  __shared__ int bi[kTrThreads / 32], ci[kTrCluster];
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");  // this CTA is running
  grid_dep_wait();
  grid_dep_launch();
  const int row = blockIdx.y, c = blockIdx.x;
  const int w0 = (int)((long long)p.W * c / kTrCluster), w1 = (int)((long long)p.W * (c + 1) / kTrCluster);
  const T* logits = static_cast<const T*>(p.logits) + (size_t)row * p.V;
  const uint32_t* seen = p.seen ? p.seen + (size_t)row * p.W : nullptr;
  const uint32_t* allowed = p.allowed ? p.allowed + (size_t)row * p.W : nullptr;
  const int* counts = p.counts + (size_t)row * p.V;
  float* out = p.out_logits ? p.out_logits + (size_t)row * p.V : nullptr;
  const float rep = p.repetition ? p.repetition[row] : 1.f;
  const float freq = p.frequency ? p.frequency[row] : 0.f;
  const float pres = p.presence ? p.presence[row] : 0.f;
  const bool vec = p.V % 8 == 0;  // every row 16-byte aligned and in whole groups
  if (p.bias_cap) {
    for (int w = threadIdx.x; w < w1 - w0; w += kTrThreads) tr_bias[w] = 0u;
    __syncthreads();
    for (int k = threadIdx.x; k < p.bias_cap; k += kTrThreads) {
      const int v = p.bias_ids[(size_t)row * p.bias_cap + k];
      if (v >= w0 * 32 && v < w1 * 32 && v < p.V) atomicOr(&tr_bias[v / 32 - w0], 1u << (v & 31));
    }
    __syncthreads();
  }
  float best = -INFINITY;
  int besti = 0x7fffffff;
  for (int g = w0 * 4 + threadIdx.x; g < w1 * 4; g += kTrThreads) {  // groups of 8 tokens, a quarter word each
    const int v0 = g * 8, sh = (g & 3) * 8;
    if (v0 >= p.V) break;
    const int nv = min(8, p.V - v0);
    const uint32_t live = nv == 8 ? 0xffu : (1u << nv) - 1u;
    const uint32_t ab = (allowed ? allowed[g >> 2] >> sh : 0xffu) & live;
    if (ab == 0u) {
      if (out)
        for (int j = 0; j < nv; ++j) out[v0 + j] = -INFINITY;
      continue;
    }
    const uint32_t sb = seen ? seen[g >> 2] >> sh & ab : 0u;
    const uint32_t bb = p.bias_cap ? tr_bias[(g >> 2) - w0] >> sh & ab : 0u;
    float f[8];
    tr_load8(logits, v0, p.V, vec, f);
    if (sb | bb) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (sb >> j & 1u) {
          f[j] = f[j] > 0.f ? f[j] / rep : __fmul_rn(f[j], rep);
          const int n = counts[v0 + j];
          if (n > 0) f[j] = __fsub_rn(__fsub_rn(f[j], __fmul_rn(freq, (float)n)), pres);
        }
        if (bb >> j & 1u) {
          float add = 0.f;
          for (int k = 0; k < p.bias_cap; ++k)
            if (p.bias_ids[(size_t)row * p.bias_cap + k] == v0 + j)
              add = __fadd_rn(add, p.bias_values[(size_t)row * p.bias_cap + k]);
          f[j] = __fadd_rn(f[j], add);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (!(ab >> j & 1u)) f[j] = -INFINITY;
      else if (tr_better(f[j], v0 + j, best, besti)) best = f[j], besti = v0 + j;
      if (out && j < nv) out[v0 + j] = f[j];
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
    for (int w = 1; w < kTrThreads / 32; ++w)
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
  for (int w = 0; w < kTrCluster; ++w)
    if (w == 0 || tr_better(cv[w], ci[w], best, besti)) best = cv[w], besti = ci[w];
  const bool found = besti != 0x7fffffff;
  p.out_ids[row] = found ? besti : -1;
  if (p.record && found) {
    p.counts[(size_t)row * p.V + besti] += 1;
    p.seen[(size_t)row * p.W + besti / 32] |= 1u << (besti & 31);
  }
}

// Tokens of each sequence into its seen bits and, for an answer's tokens, its
// counts.  Negative ids are padding; ids past the vocabulary are reported.
__global__ void __launch_bounds__(kTrThreads) token_stats_add_kernel(const int64_t* ids, int len, int V, int W,
                                                                     int* counts, uint32_t* seen, int* err) {
  grid_dep_wait();
  grid_dep_launch();
  const int row = blockIdx.y;
  for (int i = blockIdx.x * kTrThreads + threadIdx.x; i < len; i += gridDim.x * kTrThreads) {
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
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(kTrCluster, (unsigned)m);
  cfg.blockDim = dim3(kTrThreads);
  cfg.dynamicSmemBytes = p.bias_cap ? (size_t)(p.W / kTrCluster + 1) * 4 : 0;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = kTrCluster;
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
  const int64_t blocks = (len + kTrThreads - 1) / kTrThreads;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(blocks < 64 ? blocks : 64), (unsigned)batch);
  cfg.blockDim = dim3(kTrThreads);
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
