// Low-rank adapters of many requests beside a projection they share.
//
// delta[t, n] = scaling[id] * sum_r u[t, r] * b[id, n, r],
// u[t, r] = sum_k x[t, k] * a[id, r, k], id = adapter_ids[t / q_len]; tokens of
// a sequence without an adapter (id < 0) get zeros.  The fp32 result has the
// layout of one more split partial of the shared projection (LS_EPI_SPLIT_F32),
// so the kernel that adds the partials adds the adapter too and the projection
// plus its adapter round once.
//
// Two halves, both on mma.sync m16n8k16 (16 tokens x 8 ranks or outputs); the
// operands go from global memory straight into the fragments, since both sides may
// take k in any order as long as it is the same one: a lane's 16 (8) bytes of a
// row are its k's of two (one) MMA steps.
//   * Shrink, u over up to 8 k splits: a cluster of CTAs whose partials meet in shared
//     memory and are added in split order (left to the expand kernel, every one of
//     its CTAs added them again: 20 us of 30 at rank 64 and 16 splits).
//   * Expand: u keeps its 24 bits as a sum of three bf16 (8 bits each), three
//     products per step.  Up to 8 tokens in a tile: outputs are the rows, tokens the
//     columns, half the products of the other way round (32 tokens with an adapter each
//     to 19456 outputs: 10.8 us instead of 11.7).  A lane's outputs are neighbours.
// Two launches, or one in which a cluster does both halves of a tile (lora_one_launch).
// Short sequences (decode, verify): the tokens of one adapter (within a window of 1024
// sequences) make tiles of 16, and the CTA of a tile's first sequence works for all of
// it, so an adapter is read once for every 16 of its tokens; one CTA for all of them
// walked its tiles one by one (64 tokens of one adapter, 2560 -> 6144: 23 us, in tiles
// at once 7.4).  Long ones (prompts, q_len >= 16): a CTA takes tokens of one sequence.
// What bounds it: memory -- A and B of the adapters in use for short sequences
// (where a few MB are latency), x and the fp32 output for prompts.  Tensor cores of
// the tcgen05 kind would wait: 2 r flops per byte of x.
// Measured: 1 token 2560 -> 6144 at rank 16 5.2 us (launch, three dependent loads, a
// cluster's exchange), 32 tokens with an adapter each 2560 -> 19456 10.8 us (1.5 TB/s),
// 7 prompts of 701 tokens 2560 -> 6144 at rank 32 39.5 us (3.7 TB/s: 13 of it shrink
// at 1.9, the rest writes the output).
#include <type_traits>

#include "mma_sync.cuh"

namespace lsb {

constexpr int kLoThreads = 128;
constexpr int kLoWarps = 4;
constexpr int kLoOneRanks = 64;   // of the one-launch kernel (its sums: 16 tokens x ranks of every warp)
constexpr int kLoWindow = 1024;   // sequences among which equal adapters share a CTA
constexpr int kLoPrompt = 16;     // q_len from which a CTA takes tokens of one sequence
constexpr int kLoTile = 128;      // shrink: tokens of a prompt CTA (32 a pair of warps)
constexpr int kLoPromptThreads = 256;
constexpr int kLoRanks = 16;      // shrink: ranks of a CTA, at most (16 x 5 tokens at rank 64: 13.6 us; all 64: 14.7)
constexpr int kLoRanksPrompt = 32;
constexpr int kLoTileOut = 64;    // expand: tokens of a prompt CTA (16 a warp)

struct LoraParams {
  const __nv_bfloat16* x;  // [M, K]
  const __nv_bfloat16* a;  // [adapters, R, K]
  const __nv_bfloat16* b;  // [adapters, N, R]
  const float* scaling;    // [adapters]
  const int* ids;          // [batch]
  float* u;                // [M, R]
  float* out;              // [M, N]
  int* err;
  int M, batch, q_len, K, N, R, adapters, accumulate;
  int splits, k_chunk;     // shrink: k split s is [s k_chunk, (s + 1) k_chunk)
  int n_block;             // expand: outputs of a CTA
};

// The adapter of sequence b, -1 for none; an id past the bank counts as none and is reported.
__device__ __forceinline__ int lora_adapter(const LoraParams& p, int b) {
  const int id = p.ids[b];
  if (id >= p.adapters) {
    if (threadIdx.x == 0) raise_device_error(p.err, LS_ERR_INVALID_ARGUMENT);
    return -1;
  }
  return id < 0 ? -1 : id;
}

// Short sequences: the sequences that the CTA of sequence b works for, a tile of at most
// 16 tokens: those of its adapter in its window are counted through, and the first of
// every 16 / q_len works for itself and those up to the next such.  Returns their number
// (0: b is not such a first); `members` holds their indices, in order.
template <int WARPS = kLoWarps>
__device__ __forceinline__ int lora_group(const LoraParams& p, int b, int id, int first, int (&members)[16]) {
  __shared__ int s_before[WARPS], s_from[WARPS];
  const int w0 = b / kLoWindow * kLoWindow, w1 = min(w0 + kLoWindow, p.batch), most = 16 / p.q_len;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int before = 0, n = 0;
  for (int i0 = w0; i0 < w1; i0 += WARPS * 32) {
    const int i = i0 + threadIdx.x;
    const bool same = i < w1 && (i0 == w0 ? first : p.ids[i]) == id;
    const uint32_t vote = __ballot_sync(0xffffffffu, same && i < b), from = __ballot_sync(0xffffffffu, same && i >= b);
    if (lane == 0) {
      s_before[warp] = __popc(vote);
      s_from[warp] = __popc(from);
    }
    __syncthreads();
    int at = n + __popc(from & ((1u << lane) - 1u));
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      if (w < warp) at += s_from[w];
      n += s_from[w];
      before += s_before[w];
    }
    if ((from >> lane & 1u) && at < most) members[at] = i;
    __syncthreads();
  }
  return before % most ? 0 : min(n, most);
}

// What lora_group compares first, loaded beside the id that it compares with.
__device__ __forceinline__ int lora_first(const LoraParams& p, int b) {
  const int i = b / kLoWindow * kLoWindow + threadIdx.x;
  return i < p.batch ? p.ids[i] : -1;
}

// The lines of `bytes` bytes into L2, while the previous kernel is still at work.
__device__ __forceinline__ void lora_prefetch(const void* base, int bytes) {
  for (int i = threadIdx.x * 128; i < bytes; i += blockDim.x * 128)
    asm volatile("prefetch.global.L2 [%0];" ::"l"(static_cast<const char*>(base) + i));
}

__device__ __forceinline__ uint32_t lo_part(const uint4& v, int i) {
  return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
}

// acc += x a^T over k in [k0, k1) in steps of `step` (each of 32 k): MT tiles of 16
// tokens (rows g8 and g8 + 8 at xr), NT tiles of 8 of the R ranks at a.  Every xr is a row
// of x, a missing token's any other's, and so are the rows of a past R: rows and columns
// of the products are independent, and those are not used.  Only k's past k1 are zeros.
template <int MT, int NT>
__device__ __forceinline__ void lora_dot(const __nv_bfloat16* const (&xr)[MT][2], const __nv_bfloat16* a, int K, int R, int k0,
                                         int k1, int step, float (&acc)[MT][NT][4]) {
  const int lane = threadIdx.x & 31, g8 = lane >> 2, t4 = lane & 3;
  const __nv_bfloat16* ar[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) ar[j] = a + (size_t)(j * 8 + g8 < R ? j * 8 + g8 : 0) * K;
  auto products = [&](const uint4 (&xv)[MT][2], const uint4 (&av)[NT]) {
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const uint32_t fa[4] = {lo_part(xv[i][0], 2 * s), lo_part(xv[i][1], 2 * s), lo_part(xv[i][0], 2 * s + 1),
                                lo_part(xv[i][1], 2 * s + 1)};
#pragma unroll
        for (int j = 0; j < NT; ++j) mma_bf16(acc[i][j], fa, lo_part(av[j], 2 * s), lo_part(av[j], 2 * s + 1));
      }
  };
  int k = k0;
#pragma unroll (NT <= 4 ? 4 : 2)  // (64 ranks: 140 registers with 4 leave an SM one CTA, 32 sequences 23 us instead of 15)
  for (; k + 32 <= k1; k += step) {
    const int kk = k + t4 * 8;
    uint4 xv[MT][2], av[NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) xv[i][h] = ldg16(xr[i][h] + kk);
#pragma unroll
    for (int j = 0; j < NT; ++j) av[j] = ldg16(ar[j] + kk);
    products(xv, av);
  }
  if (k < k1) {  // k1 is a multiple of 8: a lane's 8 are there or not
    const int kk = k + t4 * 8;
    const uint4 none = make_uint4(0, 0, 0, 0);
    uint4 xv[MT][2], av[NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) xv[i][h] = kk < k1 ? ldg16(xr[i][h] + kk) : none;
#pragma unroll
    for (int j = 0; j < NT; ++j) av[j] = kk < k1 ? ldg16(ar[j] + kk) : none;
    products(xv, av);
  }
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// An fp32 at the same place as `local` in CTA `cta` of the cluster.
__device__ __forceinline__ float ld_cluster(const float* local, int cta) {
  uint32_t at;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(local)), "r"(cta));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ void st_cluster(float* local, int cta, float v) {
  uint32_t at;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(local)), "r"(cta));
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at), "f"(v) : "memory");
}

// Elements [0, n) of the cluster's CTAs' partials, added in split order; CTA c of
// them takes every ncta-th run of THREADS elements and hands its sums to store(i, v).
template <int THREADS, typename Store>
__device__ __forceinline__ void lora_join_splits(const float* part, int n, Store store) {
  const int c = blockIdx.x, ncta = gridDim.x;  // the cluster is the grid's x extent
  if (ncta > 1) cluster_sync();
  else __syncthreads();
  for (int i = c * THREADS + threadIdx.x; i < n; i += ncta * THREADS) {
    float v = 0.f;
    if (ncta == 1) {
      v = part[i];
    } else {
      float w[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) w[q] = ld_cluster(part + i, q < ncta ? q : 0);
#pragma unroll
      for (int q = 0; q < 8; ++q)
        if (q < ncta) v += w[q];
    }
    store(i, v);
  }
  // The partials are read by others: they stay until all are done.
  if (ncta > 1) cluster_sync();
  else __syncthreads();
}

// Short sequences: the four warps share the CTA's k range; their sums meet in shared memory.
template <int NT>
__global__ void __launch_bounds__(kLoThreads) lora_shrink_kernel(LoraParams p) {
  __shared__ int members[16];
  __shared__ float red[kLoWarps][16][NT * 8 + 1], part[16 * NT * 8];
  grid_dep_wait();
  grid_dep_launch();
  const int b = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g8 = lane >> 2, t4 = lane & 3;
  const int first = lora_first(p, b), id = lora_adapter(p, b);
  if (id < 0) return;
  const int tokens = lora_group(p, b, id, first, members) * p.q_len;
  if (!tokens) return;  // the whole cluster
  const int k0 = blockIdx.x * p.k_chunk, k1 = min(k0 + p.k_chunk, p.K);
  const int r0 = blockIdx.z * kLoRanks, ranks = min(kLoRanks, p.R - r0);
  auto token = [&](int i) { return members[i / p.q_len] * p.q_len + i % p.q_len; };
  const __nv_bfloat16* xr[1][2];
#pragma unroll
  for (int h = 0; h < 2; ++h) xr[0][h] = p.x + (size_t)token(g8 + 8 * h < tokens ? g8 + 8 * h : 0) * p.K;
  float acc[1][NT][4] = {};
  lora_dot<1, NT>(xr, p.a + ((size_t)id * p.R + r0) * p.K, p.K, ranks, k0 + warp * 32, k1, 32 * kLoWarps, acc);
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) red[warp][g8 + 8 * (e >> 1)][j * 8 + 2 * t4 + (e & 1)] = acc[0][j][e];
  __syncthreads();
  for (int i = threadIdx.x; i < 16 * NT * 8; i += kLoThreads) {
    const int t = i / (NT * 8), r = i % (NT * 8);
    part[i] = (red[0][t][r] + red[1][t][r]) + (red[2][t][r] + red[3][t][r]);
  }
  lora_join_splits<kLoThreads>(part, 16 * NT * 8, [&](int i, float v) {
    const int t = i / (NT * 8), r = i % (NT * 8);
    if (t < tokens && r < ranks) p.u[(size_t)token(t) * p.R + r0 + r] = v;
  });
}

// Prompts: two warps take 32 tokens, each every other step of the CTA's k range.
template <int NT>
__global__ void __launch_bounds__(kLoPromptThreads) lora_shrink_prompt_kernel(LoraParams p) {
  __shared__ __align__(16) float part[kLoTile * NT * 8];
  grid_dep_wait();
  grid_dep_launch();
  const int b = blockIdx.z, lane = threadIdx.x & 31, g8 = lane >> 2, t4 = lane & 3;
  const int warp = threadIdx.x >> 5 & 3, odd = threadIdx.x >> 7;
  const int id = lora_adapter(p, b);
  if (id < 0) return;
  const int groups = (p.R + kLoRanksPrompt - 1) / kLoRanksPrompt, t0 = blockIdx.y / groups * kLoTile, i0 = t0 + warp * 32;
  const int r0 = blockIdx.y % groups * kLoRanksPrompt, ranks = min(kLoRanksPrompt, p.R - r0);
  const int k0 = blockIdx.x * p.k_chunk, k1 = min(k0 + p.k_chunk, p.K);
  const __nv_bfloat16* xr[2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int t = i0 + i * 16 + h * 8 + g8;
      xr[i][h] = p.x + ((size_t)b * p.q_len + min(t, p.q_len - 1)) * p.K;
    }
  float acc[2][NT][4] = {};
  lora_dot<2, NT>(xr, p.a + ((size_t)id * p.R + r0) * p.K, p.K, ranks, k0 + odd * 32, k1, 64, acc);
  for (int half = 1; half >= 0; --half) {  // the odd steps' warp stores its sums, the other adds its own
    if (odd == half) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            float2* to = reinterpret_cast<float2*>(part + (warp * 32 + i * 16 + h * 8 + g8) * (NT * 8) + j * 8 + 2 * t4);
            const float2 had = half ? make_float2(0.f, 0.f) : *to;
            *to = make_float2(had.x + acc[i][j][2 * h], had.y + acc[i][j][2 * h + 1]);
          }
    }
    __syncthreads();
  }
  lora_join_splits<kLoPromptThreads>(part, kLoTile * NT * 8, [&](int i, float v) {
    const int t = t0 + i / (NT * 8), r = i % (NT * 8);
    if (t < p.q_len && r < ranks) p.u[((size_t)b * p.q_len + t) * p.R + r0 + r] = v;
  });
}

// Four values as sums of three bf16, each part as two pairs.
__device__ __forceinline__ void lora_three(const float4& v, uint32_t (&lo)[3], uint32_t (&hi)[3]) {
  float r[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int q = 0; q < 3; ++q) {
    float c[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      c[e] = round_bf16(r[e]);
      r[e] = fabsf(c[e]) < INFINITY ? r[e] - c[e] : 0.f;  // (infinity and NaN are whole in the first part)
    }
    lo[q] = pack_bf16(c[0], c[1]);
    hi[q] = pack_bf16(c[2], c[3]);
  }
}

// u of a tile's tokens as fragments of KS steps, each value a sum of three bf16: TOK = 16
// as the MMA's rows (a lane's are g8 and g8 + 8), TOK = 8 as its columns (a lane's is g8).
template <int KS, int TOK>
struct LoraU {
  static constexpr int H = TOK / 8;
  uint32_t f[KS][3][2 * H];
  // value(h, k): u of rank k .. k + 3 of token g8 + 8 h
  template <typename Value>
  __device__ __forceinline__ void split(int R, Value value) {
    const int t4 = threadIdx.x & 3;
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int h = 0; h < H; ++h) {
        const int k = s * 16 + t4 * 4;
        uint32_t lo[3], hi[3];
        lora_three(k < R ? value(h, k) : make_float4(0.f, 0.f, 0.f, 0.f), lo, hi);
#pragma unroll
        for (int q = 0; q < 3; ++q) f[s][q][h] = lo[q], f[s][q][H + h] = hi[q];
      }
  }
  // From the workspace; tok: the tokens, < 0: zeros.
  __device__ __forceinline__ void load(const LoraParams& p, const int (&tok)[H]) {
    split(p.R, [&](int h, int k) {
      return tok[h] < 0 ? make_float4(0.f, 0.f, 0.f, 0.f)
                        : __ldcg(reinterpret_cast<const float4*>(p.u + (size_t)tok[h] * p.R + k));
    });
  }
};

// The rows of b of outputs n .. n + 15 as fragments of KS steps.  TOK = 16: columns of two
// products, column 2 t4 + e of product j is output 4 t4 + 2 j + e, so that a lane's four
// outputs of a token are neighbours; TOK = 8: rows of one, rows g8 and g8 + 8 are outputs
// 2 g8 and 2 g8 + 1, so that a lane's two of a token are.
template <int KS, int TOK>
struct LoraB {
  uint2 v[2][KS];
  __device__ __forceinline__ void load(const __nv_bfloat16* b, int n, int n1, int R) {
    const int lane = threadIdx.x & 31, g8 = lane >> 2, t4 = lane & 3;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int row = n + (TOK == 8 ? 2 * g8 + j : (g8 >> 1) * 4 + j * 2 + (g8 & 1));
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const int k = s * 16 + t4 * 4;
        v[j][s] = row < n1 && k < R ? __ldg(reinterpret_cast<const uint2*>(b + (size_t)row * R + k)) : make_uint2(0u, 0u);
      }
    }
  }
};

// Outputs n .. n + 15 of a tile.  tok: the tokens that this lane stores, g8 and g8 + 8
// (TOK = 16) or 2 t4 and 2 t4 + 1 (TOK = 8); < 0: none.
template <int KS, int TOK>
__device__ __forceinline__ void lora_store(const LoraParams& p, const LoraU<KS, TOK>& u, const LoraB<KS, TOK>& b,
                                           float scale, const int (&tok)[2], int n, int n1) {
  const int g8 = (threadIdx.x & 31) >> 2, t4 = threadIdx.x & 3;
  if constexpr (TOK == 8) {
    float acc[4] = {};
#pragma unroll
    for (int q = 2; q >= 0; --q)  // the small parts first
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const uint32_t fa[4] = {b.v[0][s].x, b.v[1][s].x, b.v[0][s].y, b.v[1][s].y};
        mma_bf16(acc, fa, u.f[s][q][0], u.f[s][q][1]);
      }
    if (n + 2 * g8 >= n1) return;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (tok[h] < 0) continue;
      float2* o = reinterpret_cast<float2*>(p.out + (size_t)tok[h] * p.N + n + 2 * g8);
      float2 v = make_float2(acc[h] * scale, acc[2 + h] * scale);
      if (p.accumulate) {
        const float2 w = *o;
        v = make_float2(w.x + v.x, w.y + v.y);
      }
      *o = v;
    }
  } else {
    float acc[2][4] = {};
#pragma unroll
    for (int q = 2; q >= 0; --q)
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int j = 0; j < 2; ++j) mma_bf16(acc[j], u.f[s][q], b.v[j][s].x, b.v[j][s].y);
    if (n + t4 * 4 >= n1) return;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (tok[h] < 0) continue;
      float4* o = reinterpret_cast<float4*>(p.out + (size_t)tok[h] * p.N + n + t4 * 4);
      float4 v = make_float4(acc[0][2 * h] * scale, acc[0][2 * h + 1] * scale, acc[1][2 * h] * scale,
                             acc[1][2 * h + 1] * scale);
      if (p.accumulate) {
        const float4 w = *o;
        v = make_float4(w.x + v.x, w.y + v.y, w.z + v.z, w.w + v.w);
      }
      *o = v;
    }
  }
}

// Outputs [n0, n1) of a tile, 16 at a time, `step` apart.
template <int KS, int TOK>
__device__ __forceinline__ void lora_outputs(const LoraParams& p, const LoraU<KS, TOK>& u, int id, const int (&tok)[2],
                                             int n0, int n1, int step) {
  const __nv_bfloat16* b = p.b + (size_t)id * p.N * p.R;
  const float scale = p.scaling[id];
#pragma unroll (KS == 1 ? 8 : 4)
  for (int n = n0; n < n1; n += step) {
    LoraB<KS, TOK> f;
    f.load(b, n, n1, p.R);
    lora_store<KS, TOK>(p, u, f, scale, tok, n, n1);
  }
}

// Token i of a tile of short sequences, -1 behind its last.
__device__ __forceinline__ int lora_token(const LoraParams& p, const int (&members)[16], int tokens, int i) {
  return i < tokens ? members[i / p.q_len] * p.q_len + i % p.q_len : -1;
}

// Zeros into outputs [n0, n1) of `count` tokens from token t0 on.
__device__ __forceinline__ void lora_zeros(const LoraParams& p, int t0, int count, int n0, int n1) {
  const int w = (n1 - n0) / 4;
  for (int i = threadIdx.x; i < count * w; i += blockDim.x)
    *reinterpret_cast<float4*>(p.out + (size_t)(t0 + i / w) * p.N + n0 + i % w * 4) = make_float4(0.f, 0.f, 0.f, 0.f);
}

template <int KS>
__global__ void __launch_bounds__(kLoThreads, KS == 1 ? 10 : KS <= 4 ? 4 : 3) lora_expand_kernel(LoraParams p) {
  __shared__ int members[16];
  // The shrink kernel's CTAs let this one start only after every kernel before them
  // is complete: ids, b and out may be used at once, u after the wait.
  grid_dep_launch();
  const int b = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g8 = lane >> 2;
  const int n0 = blockIdx.x * p.n_block, n1 = min(n0 + p.n_block, p.N);
  const int id = lora_adapter(p, b);
  if (id < 0) {
    if (!p.accumulate) lora_zeros(p, b * p.q_len, p.q_len, n0, n1);
    grid_dep_wait();
    return;
  }
  const int tokens = lora_group(p, b, id, lora_first(p, b), members) * p.q_len;
  if (tokens > 0) lora_prefetch(p.b + ((size_t)id * p.N + n0) * p.R, (n1 - n0) * p.R * 2);
  grid_dep_wait();
  if (!tokens) return;
  const int t4 = lane & 3;
  if (tokens <= 8) {
    const int of[1] = {lora_token(p, members, tokens, g8)};
    const int tok[2] = {lora_token(p, members, tokens, 2 * t4), lora_token(p, members, tokens, 2 * t4 + 1)};
    LoraU<KS, 8> u;
    u.load(p, of);
    lora_outputs<KS, 8>(p, u, id, tok, n0 + warp * 16, n1, 16 * kLoWarps);
  } else {
    const int tok[2] = {lora_token(p, members, tokens, g8), lora_token(p, members, tokens, g8 + 8)};
    LoraU<KS, 16> u;
    u.load(p, tok);
    lora_outputs<KS, 16>(p, u, id, tok, n0 + warp * 16, n1, 16 * kLoWarps);
  }
}

template <int KS>
__global__ void __launch_bounds__(kLoThreads) lora_expand_prompt_kernel(LoraParams p) {
  grid_dep_launch();
  const int b = blockIdx.z, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g8 = lane >> 2;
  const int n0 = blockIdx.x * p.n_block, n1 = min(n0 + p.n_block, p.N);
  const int t0 = blockIdx.y * kLoTileOut;
  const int id = lora_adapter(p, b);
  if (id < 0) {
    if (!p.accumulate) lora_zeros(p, b * p.q_len + t0, min(kLoTileOut, p.q_len - t0), n0, n1);
    grid_dep_wait();
    return;
  }
  lora_prefetch(p.b + ((size_t)id * p.N + n0) * p.R, (n1 - n0) * p.R * 2);
  grid_dep_wait();
  int tok[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int t = t0 + warp * 16 + h * 8 + g8;
    tok[h] = t < p.q_len ? b * p.q_len + t : -1;
  }
  if (t0 + warp * 16 >= p.q_len) return;
  LoraU<KS, 16> u;
  u.load(p, tok);
  lora_outputs<KS, 16>(p, u, id, tok, n0, n1, 16);
}

// Short sequences, both halves in one launch: a cluster of 8 CTAs per sequence.  CTA c
// takes k split c for every rank; its partials meet those of the others in shared memory
// (each CTA adds an eighth of them, in split order, and hands its sums to all), then it
// takes outputs [c n_block, (c + 1) n_block).
template <int KS, int THREADS>
__global__ void __launch_bounds__(THREADS, KS == 1 ? 1024 / THREADS : 512 / THREADS) lora_one_kernel(LoraParams p) {  // registers for 1024 threads an SM at rank 16, else for 512
  constexpr int NT = KS * 2, RP = KS * 16, WARPS = THREADS / 32;
  __shared__ int members[16];
  __shared__ float red[WARPS / 2][16][RP + 1], part[16 * RP];
  __shared__ __align__(16) float sum[16][RP];
  grid_dep_wait();
  grid_dep_launch();
  const int b = blockIdx.y, c = blockIdx.x;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g8 = lane >> 2, t4 = lane & 3;
  const int n0 = min(c * p.n_block, p.N), n1 = min(n0 + p.n_block, p.N);
  const int first = lora_first(p, b), id = lora_adapter(p, b);
  if (id < 0) {  // the whole cluster
    if (!p.accumulate) lora_zeros(p, b * p.q_len, p.q_len, n0, n1);
    return;
  }
  const int tokens = lora_group<WARPS>(p, b, id, first, members) * p.q_len;
  if (!tokens) return;
  const __nv_bfloat16* pb = p.b + (size_t)id * p.N * p.R;
  lora_prefetch(pb + (size_t)n0 * p.R, (n1 - n0) * p.R * 2);
  const int k0 = c * p.k_chunk, k1 = min(k0 + p.k_chunk, p.K);
  const __nv_bfloat16* xr[1][2];
  int tok[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int i = g8 + 8 * h;
    tok[h] = i < tokens ? members[i / p.q_len] * p.q_len + i % p.q_len : -1;
    xr[0][h] = p.x + (size_t)(tok[h] >= 0 ? tok[h] : members[0] * p.q_len) * p.K;
  }
  float acc[1][NT][4] = {};
  lora_dot<1, NT>(xr, p.a + (size_t)id * p.R * p.K, p.K, p.R, k0 + warp * 32, k1, 32 * WARPS, acc);
  // Two warps share a place of the sums: the upper one stores, then the lower one adds.
#pragma unroll
  for (int half = 1; half >= 0; --half) {
    if (warp / (WARPS / 2) == half) {
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float& to = red[warp % (WARPS / 2)][g8 + 8 * (e >> 1)][j * 8 + 2 * t4 + (e & 1)];
          to = half ? acc[0][j][e] : to + acc[0][j][e];
        }
    }
    __syncthreads();
  }
  for (int i = threadIdx.x; i < 16 * RP; i += THREADS) {
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS / 2; ++w) v += red[w][i / RP][i % RP];
    part[i] = v;
  }
  auto exchange = [&]() {
    cluster_sync();
    for (int i = c * (2 * RP) + threadIdx.x; i < (c + 1) * (2 * RP); i += THREADS) {
      float w[8], v = 0.f;
#pragma unroll
      for (int q = 0; q < 8; ++q) w[q] = ld_cluster(part + i, q);
#pragma unroll
      for (int q = 0; q < 8; ++q) v += w[q];
#pragma unroll
      for (int q = 0; q < 8; ++q) st_cluster(&sum[0][0] + i, q, v);
    }
    cluster_sync();  // (and no CTA reads or writes another's memory any more)
  };
  const float scale = p.scaling[id];
  // The rows of b of the warp's first outputs are loaded while the CTAs exchange their sums.
  auto expand = [&](auto tile, const int (&to)[2]) {
    constexpr int TOK = decltype(tile)::value, kPre = KS == 1 ? 2 : 1;
    const int nw = n0 + warp * 16;
    LoraB<KS, TOK> pre[kPre];
#pragma unroll
    for (int q = 0; q < kPre; ++q) pre[q].load(pb, nw + q * 16 * WARPS, n1, p.R);
    exchange();
    LoraU<KS, TOK> u;
    u.split(p.R, [&](int h, int k) { return *reinterpret_cast<const float4*>(&sum[g8 + 8 * h][k]); });
#pragma unroll
    for (int q = 0; q < kPre; ++q) lora_store<KS, TOK>(p, u, pre[q], scale, to, nw + q * 16 * WARPS, n1);
    lora_outputs<KS, TOK>(p, u, id, to, nw + kPre * 16 * WARPS, n1, 16 * WARPS);
  };
  if (tokens <= 8) {  // (for the whole cluster)
    const int to[2] = {lora_token(p, members, tokens, 2 * t4), lora_token(p, members, tokens, 2 * t4 + 1)};
    expand(std::integral_constant<int, 8>(), to);
  } else {
    expand(std::integral_constant<int, 16>(), tok);
  }
}

}  // namespace lsb

namespace lsb_host {
using namespace lsb;

// k splits: with the sequences (or token tiles), about two CTAs an SM; at least 128
// k's a CTA (32 a warp), at most a cluster of 8.
static int64_t lora_splits(int64_t batch, int64_t q_len, int64_t k) {
  const int64_t groups = q_len >= kLoPrompt ? batch * ((q_len + kLoTile - 1) / kLoTile) : batch;
  int64_t s = 2 * (int64_t)sm_count() / groups;
  const int64_t most = (k + 127) / 128;
  if (s > most) s = most;
  if (s > 8) s = 8;
  return s < 1 ? 1 : s;
}

// Short sequences of rank <= 64, one launch or two.  One saves a launch (about 2 us of
// host time) and, for many sequences, the CTAs of those that another works for; but eight
// CTAs a tile are few for wide outputs, and rank 64 wants more of them.  us one / two:
// rank 16, 6144 outputs: 5.6 / 5.5 (1 sequence; 5.7 / 8.9 with the host's), 7.4 / 8.7
// (32), 9.0 / 10.8 (100); 19456 outputs: 8.1 / 5.7, 11.7 / 12.3, 14.8 / 18.7; rank 64,
// 6144 outputs: 9.6 / 6.7, 15.3 / 16.4, 16.4 / 23.0.
// Threads: 512 halve a CTA's steps, 256 let more CTAs stay: rank 16, 6144 outputs,
// 256 / 512: 6.1 / 5.6 (1 sequence), 7.4 / 8.1 (32); 19456 outputs: 16.5 / 14.8 (100);
// rank 64: 15.3 / 22.9 (32).
static bool lora_one_launch(int64_t batch, int64_t q_len, int64_t n, int64_t rank) {
  return q_len < kLoPrompt && rank <= kLoOneRanks && (batch >= 32 || (rank <= 32 && n <= 8192));
}

static int64_t lora_workspace(int64_t batch, int64_t q_len, int64_t k, int64_t rank) {
  (void)k;
  return batch * q_len * rank * 4;
}

static cudaError_t launch_lora_kernel(void (*kernel)(LoraParams), dim3 grid, unsigned cluster, const LoraParams& p,
                                      cudaStream_t stream, int threads = kLoThreads) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

static int launch_lora(LoraParams p, cudaStream_t stream) {
  const bool prompt = p.q_len >= kLoPrompt;
  if (lora_one_launch(p.batch, p.q_len, p.N, p.R)) {
    p.k_chunk = ((p.K + 7) / 8 + 31) / 32 * 32;
    p.n_block = ((p.N + 7) / 8 + 15) / 16 * 16;
    const bool wide = p.R <= 32 && (p.batch < 16 || p.N > 8192);
    void (*one)(LoraParams) = p.R <= 16   ? (wide ? lora_one_kernel<1, 512> : lora_one_kernel<1, 256>)
                              : p.R <= 32 ? (wide ? lora_one_kernel<2, 512> : lora_one_kernel<2, 256>)
                                          : lora_one_kernel<4, 256>;
    const cudaError_t e = launch_lora_kernel(one, dim3(8, (unsigned)p.batch), 8, p, stream, wide ? 512 : 256);
    return e == cudaSuccess ? LS_OK : set_error(LS_ERR_CUDA, "lora_delta launch: %s", cudaGetErrorString(e));
  }
  p.splits = (int)lora_splits(p.batch, p.q_len, p.K);
  p.k_chunk = ((p.K + p.splits - 1) / p.splits + 31) / 32 * 32;
  const int most = prompt ? kLoRanksPrompt : kLoRanks;  // ranks of a shrink CTA
  const int nt = (p.R < most ? p.R : most) / 8, ks = (p.R + 15) / 16;
  const unsigned groups = (unsigned)((p.R + most - 1) / most);
  void (*shrink)(LoraParams);
  void (*expand)(LoraParams);
  if (prompt) {
    shrink = nt <= 1 ? lora_shrink_prompt_kernel<1> : nt <= 2 ? lora_shrink_prompt_kernel<2> : lora_shrink_prompt_kernel<4>;
    expand = ks <= 1   ? lora_expand_prompt_kernel<1>
             : ks <= 2 ? lora_expand_prompt_kernel<2>
             : ks <= 4 ? lora_expand_prompt_kernel<4>
                       : lora_expand_prompt_kernel<8>;
  } else {
    shrink = nt <= 1 ? lora_shrink_kernel<1> : lora_shrink_kernel<2>;
    expand = ks <= 1   ? lora_expand_kernel<1>
             : ks <= 2 ? lora_expand_kernel<2>
             : ks <= 4 ? lora_expand_kernel<4>
                       : lora_expand_kernel<8>;
  }
  // Outputs of a CTA: 64 (16 a warp) for few sequences, more as the grid grows
  // beyond about 1200 CTAs; prompts 128 (64 / 256 / 512 were 4 / 7 / 20% slower).
  const int64_t blocks = (int64_t)((p.N + 63) / 64) * p.batch;
  const int64_t per = (blocks + 1199) / 1200;
  p.n_block = prompt ? 128 : 64 * (int)(per < 1 ? 1 : per > 16 ? 16 : per);
  const unsigned nb = (unsigned)((p.N + p.n_block - 1) / p.n_block);
  auto tiles = [&](int tile) { return (unsigned)((p.q_len + tile - 1) / tile); };
  const dim3 gs = prompt ? dim3((unsigned)p.splits, tiles(kLoTile) * groups, (unsigned)p.batch)
                         : dim3((unsigned)p.splits, (unsigned)p.batch, groups);
  const dim3 ge = prompt ? dim3(nb, tiles(kLoTileOut), (unsigned)p.batch) : dim3(nb, (unsigned)p.batch);
  cudaError_t e = launch_lora_kernel(shrink, gs, (unsigned)p.splits, p, stream, prompt ? kLoPromptThreads : kLoThreads);
  if (e == cudaSuccess) e = launch_lora_kernel(expand, ge, 1, p, stream);
  return e == cudaSuccess ? LS_OK : set_error(LS_ERR_CUDA, "lora_delta launch: %s", cudaGetErrorString(e));
}

}  // namespace lsb_host

using namespace lsb_host;

extern "C" {

int ls_lora_delta_workspace_bytes(int64_t batch, int64_t q_len, int64_t k, int64_t n, int64_t rank, int64_t* bytes) {
  LS_REQUIRE(bytes, LS_ERR_INVALID_ARGUMENT, "ls_lora_delta_workspace_bytes: bytes is null");
  LS_REQUIRE(batch > 0 && q_len > 0 && batch < (1ll << 31) && q_len < (1ll << 31) && batch * q_len < (1ll << 31) &&
                 k > 0 && k < (1ll << 31) && n > 0 && n < (1ll << 24) && rank > 0,
             LS_ERR_INVALID_ARGUMENT, "ls_lora_delta: bad sizes");
  LS_REQUIRE(k % 8 == 0 && n % 8 == 0 && rank % 8 == 0, LS_ERR_MISALIGNED,
             "ls_lora_delta: k=%lld, n=%lld and rank=%lld must be multiples of 8", (long long)k, (long long)n,
             (long long)rank);
  LS_REQUIRE(rank <= 128, LS_ERR_UNSUPPORTED_SHAPE, "ls_lora_delta: rank=%lld beyond 128", (long long)rank);
  LS_REQUIRE(batch <= 65535 && (q_len + 63) / 64 * 2 <= 65535, LS_ERR_UNSUPPORTED_SHAPE,
             "ls_lora_delta: %lld sequences of %lld tokens exceed the grid", (long long)batch, (long long)q_len);
  *bytes = lora_workspace(batch, q_len, k, rank);
  return LS_OK;
}

int ls_lora_delta_launches(int64_t batch, int64_t q_len, int64_t k, int64_t n, int64_t rank, int64_t* launches) {
  LS_REQUIRE(launches, LS_ERR_INVALID_ARGUMENT, "ls_lora_delta_launches: launches is null");
  int64_t bytes = 0;
  const int rc = ls_lora_delta_workspace_bytes(batch, q_len, k, n, rank, &bytes);
  if (rc) return rc;
  *launches = lora_one_launch(batch, q_len, n, rank) ? 1 : 2;
  return LS_OK;
}

int ls_lora_delta(const void* x, int64_t batch, int64_t q_len, int64_t k, const void* a, const void* b,
                  const float* scaling, int64_t adapters, int64_t n, int64_t rank, const int32_t* adapter_ids,
                  int accumulate, float* out, void* workspace, int64_t workspace_bytes, ls_stream_t stream) {
  LS_REQUIRE(x && a && b && scaling && adapter_ids && out, LS_ERR_INVALID_ARGUMENT, "ls_lora_delta: null pointer");
  LS_REQUIRE(adapters > 0 && adapters < (1ll << 24), LS_ERR_INVALID_ARGUMENT, "ls_lora_delta: bad sizes");
  int64_t need = 0;
  int rc = ls_lora_delta_workspace_bytes(batch, q_len, k, n, rank, &need);
  if (rc) return rc;
  LS_REQUIRE(aligned16(x) && aligned16(a) && aligned16(b) && aligned16(out) && aligned16(workspace), LS_ERR_MISALIGNED,
             "ls_lora_delta: pointers must be 16-byte aligned");
  LS_REQUIRE(workspace && workspace_bytes >= need, LS_ERR_WORKSPACE, "ls_lora_delta: workspace needs %lld bytes",
             (long long)need);
  LoraParams p = {};
  p.x = static_cast<const __nv_bfloat16*>(x);
  p.a = static_cast<const __nv_bfloat16*>(a);
  p.b = static_cast<const __nv_bfloat16*>(b);
  p.scaling = scaling;
  p.ids = adapter_ids;
  p.u = static_cast<float*>(workspace);
  p.out = out;
  p.err = device_error_ptr();
  p.M = (int)(batch * q_len);
  p.batch = (int)batch;
  p.q_len = (int)q_len;
  p.K = (int)k;
  p.N = (int)n;
  p.R = (int)rank;
  p.adapters = (int)adapters;
  p.accumulate = accumulate ? 1 : 0;
  return launch_lora(p, (cudaStream_t)stream);
}

}  // extern "C"
