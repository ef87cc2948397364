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
// bans outright are not read at all.  Where the vocabulary is no multiple of 8 the
// groups are aligned in the flattened [m, vocab] array, not in the row, so that
// these sizes take 16-byte accesses too, and a group's bits are cut from two
// words.  The CTAs of a row leave one key each, of a value and the group of 8 that holds
// it, and a second, small kernel finds the token in that group, meets it with the biased
// ones and enters it into the row's state: no counters to zero, no order of
// arrival, nothing that two captured graphs share.  (With a row as a cluster of
// CTAs whose winners met in shared memory, 64 rows of 151936 took 17 us instead of
// 10: clusters are placed slowly and wait for one another.)  What bounds it: for
// few rows the chain bits -> logits, counts -> pick of dependent latencies; for
// many, instruction issue beside the loads, so a group is kept short: bits as bytes,
// masks by byte permutes, a packed maximum and no index (161 -> 70 instructions a
// group of 8 bf16 tokens), seen tokens one at a time.
// Measured: 1 row of 151936 bf16 4.6 us (launch and latency), 32 rows of it under a
// grammar of 300 tokens 7.0, 128 rows with everything and written logits 34 (3.5 TB/s).
#include <algorithm>

#include "common.cuh"
#include "token_groups.cuh"

namespace lsb {

constexpr int kTrThreads = 256;
constexpr int kTrPickThreads = 128;

constexpr int64_t kTrNoKey = INT64_MIN;  // below every argmax_key: a CTA without a candidate

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
  int64_t* keys;             // [M, CTAs of a row]: the workspace
  float* out_logits;         // [M, V] or null
  int V, W, bias_cap;
};

// 8 consecutive logits as loaded; kept(): with -inf in place of the tokens whose bit is
// clear, from which their maximum (NaN drops out) and their fp32 are taken.
template <typename T>
struct TrRaw {};
template <>
struct TrRaw<__nv_bfloat16> {
  uint32_t w[4];
  __device__ __forceinline__ void load(const __nv_bfloat16* p) {  // 16-byte aligned
    const uint4 v = ldg16(p);
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  }
  __device__ __forceinline__ void load(const __nv_bfloat16* p, int lo, int hi) {  // elements lo .. hi - 1 only
    uint32_t h[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) h[j] = j >= lo && j < hi ? (uint32_t)__bfloat16_as_ushort(p[j]) : 0u;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = h[2 * i] | h[2 * i + 1] << 16;
  }
  __device__ __forceinline__ float value(int j) const {
    const uint32_t x = j & 4 ? (j & 2 ? w[3] : w[2]) : (j & 2 ? w[1] : w[0]);
    return __uint_as_float(j & 1 ? x & 0xffff0000u : x << 16);
  }
  // Four bits become the sign bits of four bytes, and two byte permutes that repeat
  // signs make 16-bit masks of them.
  __device__ __forceinline__ TrRaw kept(uint32_t bits) const {
    TrRaw r = *this;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t sign = ((bits >> 4 * i & 15u) * 0x10204080u) & 0x80808080u;
      uint32_t m0, m1;
      asm("prmt.b32 %0, %1, 0, 0x9988;" : "=r"(m0) : "r"(sign));
      asm("prmt.b32 %0, %1, 0, 0xbbaa;" : "=r"(m1) : "r"(sign));
      r.w[2 * i] = (w[2 * i] & m0) | (0xff80ff80u & ~m0);
      r.w[2 * i + 1] = (w[2 * i + 1] & m1) | (0xff80ff80u & ~m1);
    }
    return r;
  }
  __device__ __forceinline__ float top() const {
    __nv_bfloat162 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = *reinterpret_cast<const __nv_bfloat162*>(&w[i]);
    const float2 t = __bfloat1622float2(__hmax2(__hmax2(v[0], v[1]), __hmax2(v[2], v[3])));
    return fmaxf(t.x, t.y);
  }
  __device__ __forceinline__ void get(float f[8]) const { unpack8(make_uint4(w[0], w[1], w[2], w[3]), f); }
};
template <>
struct TrRaw<float> {
  float f[8];
  __device__ __forceinline__ void load(const float* p) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
  }
  __device__ __forceinline__ void load(const float* p, int lo, int hi) {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = j >= lo && j < hi ? p[j] : 0.f;
  }
  __device__ __forceinline__ float value(int j) const {
    float x = f[0];
#pragma unroll
    for (int e = 1; e < 8; ++e)
      if (e == j) x = f[e];
    return x;
  }
  __device__ __forceinline__ TrRaw kept(uint32_t bits) const {
    TrRaw r;
#pragma unroll
    for (int j = 0; j < 8; ++j) r.f[j] = bits >> j & 1u ? f[j] : -INFINITY;
    return r;
  }
  __device__ __forceinline__ float top() const {
    return fmaxf(fmaxf(fmaxf(f[0], f[1]), fmaxf(f[2], f[3])), fmaxf(fmaxf(f[4], f[5]), fmaxf(f[6], f[7])));
  }
  __device__ __forceinline__ void get(float o[8]) const {
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = f[j];
  }
};

// Bits of group g, tokens v0 .. v0 + 7 (v0 >= -7), of a set of `words` words; bits
// outside the row come from its edges and are not live.
template <bool VEC>
__device__ __forceinline__ uint32_t tr_bits8(const uint32_t* set, int words, int g, int v0) {
  if (VEC) return reinterpret_cast<const unsigned char*>(set)[g];
  const int w = v0 >> 5, sh = v0 & 31;
  const uint32_t lo = set[max(w, 0)], hi = sh > 24 ? set[min(w + 1, words - 1)] : lo;
  return __funnelshift_r(lo, hi, sh) & 0xffu;
}

__device__ __forceinline__ bool tr_better(float v, int i, float best, int besti) {
  return v > best || (v == best && i < besti);
}

__device__ __forceinline__ float tr_penalise(float x, float rep, int n, float freq, float pres) {  // a seen token
  x = x > 0.f ? x / rep : __fmul_rn(x, rep);
  return n > 0 ? __fsub_rn(__fsub_rn(x, __fmul_rn(freq, (float)n)), pres) : x;
}
__device__ __forceinline__ float tr_value(__nv_bfloat16 v) { return bf16_to_f(v); }
__device__ __forceinline__ float tr_value(float v) { return v; }

// VEC: the vocabulary is a multiple of 8.  U: groups in flight per thread.
template <typename T, bool VEC, int U>
__global__ void __launch_bounds__(kTrThreads, 4) constrained_argmax_kernel(TrParams p) {
  extern __shared__ uint32_t tr_bias[];  // bias lists only: 8 bits for each group of this CTA's tiles
  __shared__ float bv[kTrThreads / 32];
  __shared__ int bi[kTrThreads / 32];
  grid_dep_wait();
  grid_dep_launch();
  constexpr int nt = kTrThreads, lg = 8;
  const int row = blockIdx.y, c = blockIdx.x, ncta = gridDim.x;
  // Groups of 8 flattened indices; the row's first and last group may reach into
  // its neighbours.  Group g of the row starts at token 8 g - a.  The CTAs take
  // tiles of 256 groups in turn: frequent tokens have low ids, and
  // with them the counts to read.
  const long long row0 = (long long)row * p.V;
  const int a = VEC ? 0 : tr_offset(row, p.V), ngroups = tr_groups(a, p.V);
  const int left = VEC ? 0 : tr_left(row, p.V, gridDim.y);
  const int stride = ncta << lg;  // groups from one own tile to the next
  const T* logits = static_cast<const T*>(p.logits) + row0 - a;
  const uint32_t* seen = p.seen ? p.seen + (size_t)row * p.W : nullptr;
  const uint32_t* allowed = p.allowed ? p.allowed + (size_t)row * p.W : nullptr;
  const int* counts = p.counts + row0 - a;
  float* out = p.out_logits ? p.out_logits + row0 - a : nullptr;
  const int* bias_ids = p.bias_ids + (size_t)row * p.bias_cap;
  const unsigned char* bias_bits = reinterpret_cast<const unsigned char*>(tr_bias) + threadIdx.x;
  const int own = (ngroups + stride - 1) / stride;  // tiles, at most
  int biased = threadIdx.x < p.bias_cap ? bias_ids[threadIdx.x] : -1;
  const float rep = p.repetition ? p.repetition[row] : 1.f;
  const float freq = p.frequency ? p.frequency[row] : 0.f;
  const float pres = p.presence ? p.presence[row] : 0.f;

  // A batch: U groups of this thread, one in each of U successive own tiles.
  uint32_t ab[U], sb[U];  // allowed bits, allowed and seen bits
  int n0[U];              // count of the group's first seen token
  TrRaw<T> raw[U];
  auto fetch_bits = [&](int gb) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int g = gb + u * stride, v0 = g * 8 - a;
      ab[u] = sb[u] = 0u;
      if (g >= ngroups) continue;
      ab[u] = allowed ? tr_bits8<VEC>(allowed, p.W, g, v0) : 0xffu;
      if (seen) sb[u] = tr_bits8<VEC>(seen, p.W, g, v0);
      if (!VEC && v0 < 0) ab[u] &= 0xffu << -v0;
      if (!VEC && v0 + 8 > p.V) ab[u] &= (1u << (p.V - v0)) - 1u;
    }
  };
  auto fetch_values = [&](int gb) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int g = gb + u * stride;
      sb[u] &= ab[u];
      raw[u] = {};  // (a value in any case: what no bit keeps is masked, not unknown)
      if (ab[u] == 0u) continue;
      if (!VEC && g * 8 + 8 > left) raw[u].load(logits + g * 8, 0, left - g * 8);  // (the array ends inside the group)
      else raw[u].load(logits + g * 8);
      if (sb[u]) n0[u] = counts[g * 8 + __ffs(sb[u]) - 1];
    }
  };
  // The first loads are on their way while the biased tokens are marked: the CTAs
  // run in several waves, and every wave would pay for one after the other.
  int gb = (c << lg) + threadIdx.x;
  fetch_bits(gb);
  if (p.bias_cap) {
    for (int w = threadIdx.x; w < own << lg >> 2; w += nt) tr_bias[w] = 0u;
    __syncthreads();
  }
  fetch_values(gb);
  if (p.bias_cap) {
    for (int k = threadIdx.x; k < p.bias_cap; k += nt) {
      const int v = biased, g = (v + a) >> 3, tile = g >> lg;
      biased = k + nt < p.bias_cap ? bias_ids[k + nt] : -1;
      if (v < 0 || v >= p.V || tile % ncta != c) continue;
      const int at = (tile / ncta << lg) + (g & (nt - 1));
      atomicOr(&tr_bias[at >> 2], 1u << ((at & 3) * 8 + ((v + a) & 7)));
    }
    __syncthreads();
  }
  float best = -INFINITY;
  int bestg = 0x7fffffff, at = 0;  // at: where this thread's group of the batch's first tile has its bias bits
#pragma unroll 1
  for (; gb < ngroups; at += U << lg) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int g = gb + u * stride;
      if (g >= ngroups) break;
      // Seen tokens are few: one at a time beside the group's maximum, not eight
      // predicated divisions.  Biased ones are the pick's.
      const uint32_t bb = p.bias_cap ? bias_bits[at + (u << lg)] : 0u, keep = ab[u] & ~(sb[u] | bb);
      TrRaw<T> kept = raw[u];
      if (keep != 0xffu) kept = raw[u].kept(keep);
      if (out) {
        float f[8];
        kept.get(f);
        float* o = out + g * 8;
        if (VEC || (g * 8 >= a && g * 8 - a + 8 <= p.V)) {
          *reinterpret_cast<float4*>(o) = make_float4(f[0], f[1], f[2], f[3]);
          *reinterpret_cast<float4*>(o + 4) = make_float4(f[4], f[5], f[6], f[7]);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (g * 8 + j >= a && g * 8 - a + j < p.V) o[j] = f[j];
        }
      }
      float top = kept.top();
#pragma unroll 1
      for (uint32_t m = sb[u]; m; m &= m - 1u) {
        const int j = __ffs(m) - 1;
        const float x = tr_penalise(raw[u].value(j), rep, m == sb[u] ? n0[u] : counts[g * 8 + j], freq, pres);
        if (out) out[g * 8 + j] = x;
        if (!(bb >> j & 1u)) top = fmaxf(top, x);
      }
      if (top > best) best = top, bestg = g;  // a thread meets its groups in order: the first of equals stays
    }
    gb += U * stride;
    if (gb >= ngroups) break;
    fetch_bits(gb);
    fetch_values(gb);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float ov = __shfl_xor_sync(0xffffffffu, best, o);
    const int og = __shfl_xor_sync(0xffffffffu, bestg, o);
    if (tr_better(ov, og, best, bestg)) best = ov, bestg = og;
  }
  if ((threadIdx.x & 31) == 0) bv[threadIdx.x >> 5] = best, bi[threadIdx.x >> 5] = bestg;
  __syncthreads();
  if (threadIdx.x < nt / 32) {
    best = bv[threadIdx.x], bestg = bi[threadIdx.x];
#pragma unroll
    for (int o = nt / 64; o > 0; o >>= 1) {
      const float ov = __shfl_xor_sync((1u << nt / 32) - 1u, best, o);
      const int og = __shfl_xor_sync((1u << nt / 32) - 1u, bestg, o);
      if (tr_better(ov, og, best, bestg)) best = ov, bestg = og;
    }
    if (threadIdx.x == 0) p.keys[(size_t)row * ncta + c] = bestg != 0x7fffffff ? argmax_key(best, bestg) : kTrNoKey;
  }
}

__device__ __forceinline__ int64_t tr_warp_max(int64_t key) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) key = max(key, (int64_t)__shfl_xor_sync(0xffffffffu, (long long)key, o));
  return key;
}
__device__ __forceinline__ int64_t tr_block_max(int64_t key, int64_t* warps) {  // of all kTrPickThreads threads
  key = tr_warp_max(key);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) warps[threadIdx.x >> 5] = key;
  __syncthreads();
  for (int w = 0; w < kTrPickThreads / 32; ++w) key = max(key, warps[w]);
  return key;
}

// The row's token.  Its CTAs' keys name a value and the group of 8 that holds it; the
// group's tokens are worked out again here and the best of them, lowest id first, meets
// the biased tokens.  Those are worked out here, a thread each at their first place in
// the list, the first 128 before the wait: they need nothing of the kernel before, and a
// list of 60 took 8 us behind it.  Where no token is above -inf, one that is -inf itself
// is looked for.  record: the pick into the row's state.
template <typename T>
__global__ void __launch_bounds__(kTrPickThreads) constrained_pick_kernel(TrParams p, int ncta, int record, int64_t* out_ids) {
  constexpr int kStage = 512;
  __shared__ __align__(16) int ids[kStage];
  __shared__ float values[kStage];
  __shared__ int64_t warps[kTrPickThreads / 32];
  __shared__ int s_first;
  // The kernel before lets this one start only after every kernel before it is
  // complete: logits, state and rules may be used at once, its keys after the wait.
  grid_dep_launch();
  const int row = blockIdx.x, tid = threadIdx.x;
  const size_t row_v = (size_t)row * p.V, row_w = (size_t)row * p.W;
  const T* logits = static_cast<const T*>(p.logits) + row_v;
  const int* bias_ids = p.bias_ids + (size_t)row * p.bias_cap;
  const float* bias_values = p.bias_values + (size_t)row * p.bias_cap;
  const float rep = p.repetition ? p.repetition[row] : 1.f;
  const float freq = p.frequency ? p.frequency[row] : 0.f;
  const float pres = p.presence ? p.presence[row] : 0.f;
  // Token v without its biases, and whether it is allowed; all it needs is loaded at once.
  auto token = [&](int v, bool& free) {
    const uint32_t aw = p.allowed ? p.allowed[row_w + (v >> 5)] : 0xffffffffu, sw = p.seen ? p.seen[row_w + (v >> 5)] : 0u;
    const int n = p.seen ? p.counts[row_v + v] : 0;
    const float x = tr_value(logits[v]);
    free = aw >> (v & 31) & 1u;
    return sw >> (v & 31) & 1u ? tr_penalise(x, rep, n, freq, pres) : x;
  };
  auto unbiased = [&](int v) {
    for (int k = 0; k < p.bias_cap; ++k)
      if (bias_ids[k] == v) return false;
    return true;
  };
  // Place k of the list: its token if this is the token's first place and it is allowed, else -1.
  auto biased = [&](int k, float& x) {
    int v = k < p.bias_cap ? bias_ids[k] : -1;
    if (v >= p.V) v = -1;
    bool free = false, first = true;
    x = v >= 0 ? token(v, free) : 0.f;
    float add = 0.f;  // its biases in list order
    for (int q0 = 0; q0 < p.bias_cap; q0 += kStage) {
      const int n = min(kStage, p.bias_cap - q0);
      __syncthreads();
      for (int q = tid; q < ((n + 3) & ~3); q += kTrPickThreads) {
        ids[q] = q < n ? bias_ids[q0 + q] : -1;
        values[q] = q < n ? bias_values[q0 + q] : 0.f;
      }
      __syncthreads();
      for (int q = 0; q < n; q += 4) {
        const int4 four = *reinterpret_cast<const int4*>(ids + q);
        const int id[4] = {four.x, four.y, four.z, four.w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (id[e] == v) {
            first = first && q0 + q + e >= k;
            add = __fadd_rn(add, values[q + e]);
          }
      }
    }
    x = __fadd_rn(x, add);
    return free && first ? v : -1;
  };
  int64_t key = kTrNoKey;  // of the biased tokens; the same in every thread
  float x = 0.f;
  int v = -1;
  if (p.bias_cap) {
    v = biased(tid, x);
    key = tr_block_max(v >= 0 && x == x ? argmax_key(x, v) : kTrNoKey, warps);
  }
  grid_dep_wait();
  for (int k0 = 0;; v = biased(k0 + tid, x)) {  // (with the block: biased() has barriers)
    if (v >= 0 && p.out_logits) p.out_logits[row_v + v] = x;
    if (k0 > 0) key = max(key, tr_block_max(v >= 0 && x == x ? argmax_key(x, v) : kTrNoKey, warps));
    k0 += kTrPickThreads;
    if (k0 >= p.bias_cap) break;
  }
  // Every warp finds the winning key, the first one the token: no barrier on this way.
  int64_t top = kTrNoKey;
  for (int i0 = tid & 31; i0 < ncta; i0 += 128) {
    int64_t k[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = i0 + 32 * u;
      k[u] = i < ncta ? (int64_t)__ldcg(reinterpret_cast<const long long*>(p.keys) + (size_t)row * ncta + i) : kTrNoKey;
    }
    top = max(top, max(max(k[0], k[1]), max(k[2], k[3])));
  }
  top = tr_warp_max(top);
  if (top != kTrNoKey) {
    if (tid >= 32) return;
    const int v0 = (int)argmax_key_id(top) * 8 - tr_offset(row, p.V);
    bool free = false;
    v = v0 + tid;
    if (tid < 8 && v >= 0 && v < p.V) x = token(v, free);
    uint32_t hit = 0u;  // tokens of the group that have a bias
    for (int k = tid; k < p.bias_cap; k += 32) {
      const unsigned d = (unsigned)(bias_ids[k] - v0);
      if (d < 8u) hit |= 1u << d;
    }
    hit = __reduce_or_sync(0xffffffffu, hit);
    key = max(key, tr_warp_max(free && x == x && !(hit >> tid & 1u) ? argmax_key(x, v) : kTrNoKey));
  } else {
    // Nothing above -inf without a bias.  Unless a biased token is, a word of tokens a
    // thread, until a block of words holds one that is allowed, not biased and -inf.
    for (int w0 = 0; w0 < p.W && key <= argmax_key(-INFINITY, 0); w0 += kTrPickThreads) {
      if (tid == 0) s_first = p.V;
      __syncthreads();
      const int w = w0 + tid;
      uint32_t free = w >= p.W ? 0u : p.allowed ? p.allowed[row_w + w] : 0xffffffffu;
      for (; free; free &= free - 1u) {
        const int t = w * 32 + __ffs(free) - 1;
        if (t >= p.V) break;
        bool is_free;
        if (token(t, is_free) == -INFINITY && unbiased(t)) {
          atomicMin(&s_first, t);
          break;
        }
      }
      __syncthreads();
      if (s_first < p.V) {
        key = max(key, argmax_key(-INFINITY, s_first));
        break;
      }
      __syncthreads();
    }
  }
  if (tid != 0) return;
  const int64_t id = key == kTrNoKey ? -1 : argmax_key_id(key);
  out_ids[row] = id;
  if (record && id >= 0) {  // atomics only so that nothing waits for the old value
    atomicAdd(p.counts + row_v + id, 1);
    atomicOr(p.seen + row_w + id / 32, 1u << (id & 31));
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

// CTAs of a row: a group per thread while that does not fill the GPU several times;
// then four groups (those a thread has in flight); from 16 groups a thread for one wave
// of CTAs (four an SM) on, that wave: 128 rows of 151936 bf16 with penalties, biases and
// masks, logits written, four groups / one wave: 37.8 / 33.9 us, 64 rows (which make 8)
// 14.2 / 15.7.  At most 64 tiles a CTA: their bias bits are 16 KB.
static int64_t tr_ctas(int64_t m, int64_t vocab) {
  const int64_t tiles = (vocab + 14) / 8 / kTrThreads + 1, sms = sm_count();
  if (m * tiles <= 8 * sms) return tiles;
  int64_t per = 4;
  if (m * tiles >= 16 * 4 * sms) {
    const int64_t ctas = std::max<int64_t>(4 * sms / m, 1);
    per = std::min<int64_t>((tiles + ctas - 1) / ctas, 64);
  }
  return (tiles + per - 1) / per;
}
constexpr int64_t kTrMaxVocab = 1 << 20;
constexpr int64_t kTrMaxBiases = 1 << 14;  // the pick compares each with each: about 10 ms there, and four times that for twice as many

template <typename T, bool VEC>
static int launch_constrained_argmax(const TrParams& p, int64_t m, int record, int64_t* out_ids, cudaStream_t stream) {
  const int64_t ncta = tr_ctas(m, p.V), tiles = ((int64_t)(p.V + 14) / 8 + kTrThreads - 1) / kTrThreads;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ncta, (unsigned)m);
  cfg.blockDim = dim3(kTrThreads);
  cfg.dynamicSmemBytes = p.bias_cap ? (size_t)((tiles + ncta - 1) / ncta * kTrThreads) : 0;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  // 64 bytes of groups a thread; bf16 with a tile a CTA one group: 4 rows of 151936 5.4
  // us, with four 5.8 (fp32 with one group is 3% slower than with two).
  constexpr int U = sizeof(T) == 2 ? 4 : 2, kSingle = sizeof(T) == 2 ? 1 : U;
  cudaError_t e = ncta >= tiles ? cudaLaunchKernelEx(&cfg, constrained_argmax_kernel<T, VEC, kSingle>, p)
                                : cudaLaunchKernelEx(&cfg, constrained_argmax_kernel<T, VEC, U>, p);
  if (e == cudaSuccess) {
    cfg.gridDim = dim3((unsigned)m);
    cfg.blockDim = dim3(kTrPickThreads);
    cfg.dynamicSmemBytes = 0;
    e = cudaLaunchKernelEx(&cfg, constrained_pick_kernel<T>, p, (int)ncta, record, out_ids);
  }
  return e == cudaSuccess ? LS_OK : set_error(LS_ERR_CUDA, "constrained_argmax launch: %s", cudaGetErrorString(e));
}

}  // namespace lsb_host

using namespace lsb_host;

extern "C" {

int ls_constrained_argmax_workspace_bytes(int64_t m, int64_t vocab, int64_t* bytes) {
  LS_REQUIRE(bytes && m > 0 && m <= 65535 && vocab > 0, LS_ERR_INVALID_ARGUMENT,
             "ls_constrained_argmax_workspace_bytes: bad arguments");
  LS_REQUIRE(vocab <= kTrMaxVocab, LS_ERR_UNSUPPORTED_SHAPE, "ls_constrained_argmax: vocab=%lld beyond %lld",
             (long long)vocab, (long long)kTrMaxVocab);
  *bytes = m * tr_ctas(m, vocab) * 8;
  return LS_OK;
}

int ls_constrained_argmax(const void* logits, int logits_f32, int64_t m, int64_t vocab, int32_t* counts, uint32_t* seen,
                          const float* repetition, const float* frequency, const float* presence,
                          const int32_t* bias_ids, const float* bias_values, int64_t bias_cap, const uint32_t* allowed,
                          int record, int64_t* out_ids, float* out_logits, void* workspace,
                          int64_t workspace_bytes, ls_stream_t stream) {
  LS_REQUIRE(logits && out_ids, LS_ERR_INVALID_ARGUMENT, "ls_constrained_argmax: null pointer");
  int64_t need = 0;
  int rc = ls_constrained_argmax_workspace_bytes(m, vocab, &need);
  if (rc) return rc;
  LS_REQUIRE((counts == nullptr) == (seen == nullptr), LS_ERR_INVALID_ARGUMENT,
             "ls_constrained_argmax: counts and seen come together");
  LS_REQUIRE(counts || !(repetition || frequency || presence || record), LS_ERR_INVALID_ARGUMENT,
             "ls_constrained_argmax: penalties and record need counts and seen");
  LS_REQUIRE((bias_ids == nullptr) == (bias_values == nullptr) && (bias_ids != nullptr) == (bias_cap > 0) &&
                 bias_cap >= 0 && bias_cap < (1ll << 31),
             LS_ERR_INVALID_ARGUMENT, "ls_constrained_argmax: bias_ids, bias_values and bias_cap come together");
  LS_REQUIRE(bias_cap <= kTrMaxBiases, LS_ERR_UNSUPPORTED_SHAPE, "ls_constrained_argmax: %lld biases a row, beyond %lld",
             (long long)bias_cap, (long long)kTrMaxBiases);
  LS_REQUIRE(aligned16(logits) && aligned16(out_logits), LS_ERR_MISALIGNED,
             "ls_constrained_argmax: logits must be 16-byte aligned");
  LS_REQUIRE(workspace && workspace_bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 7u) == 0, LS_ERR_WORKSPACE,
             "ls_constrained_argmax: workspace needs %lld bytes, 8-byte aligned", (long long)need);
  // The pick reads the logits of a group again after the main pass has written them processed.
  const uintptr_t in = reinterpret_cast<uintptr_t>(logits), to = reinterpret_cast<uintptr_t>(out_logits);
  const uint64_t elements = (uint64_t)m * (uint64_t)vocab;
  LS_REQUIRE(!out_logits || to >= in + elements * (logits_f32 ? 4 : 2) || in >= to + elements * 4, LS_ERR_INVALID_ARGUMENT,
             "ls_constrained_argmax: out_logits overlaps logits (not in place)");
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
  p.keys = static_cast<int64_t*>(workspace);
  p.out_logits = out_logits;
  p.V = (int)vocab;
  p.W = (int)((vocab + 31) / 32);
  p.bias_cap = (int)bias_cap;
  const cudaStream_t st = (cudaStream_t)stream;
  if (vocab % 8 == 0)
    return logits_f32 ? launch_constrained_argmax<float, true>(p, m, record ? 1 : 0, out_ids, st)
                      : launch_constrained_argmax<__nv_bfloat16, true>(p, m, record ? 1 : 0, out_ids, st);
  return logits_f32 ? launch_constrained_argmax<float, false>(p, m, record ? 1 : 0, out_ids, st)
                    : launch_constrained_argmax<__nv_bfloat16, false>(p, m, record ? 1 : 0, out_ids, st);
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
