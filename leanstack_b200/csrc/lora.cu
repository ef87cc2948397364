// Low-rank adapters of many requests beside a projection they share.
//
// delta[t, n] = scaling[id] * sum_r u[t, r] * b[id, n, r],
// u[t, r] = sum_k x[t, k] * a[id, r, k], id = adapter_ids[t / q_len]; tokens of
// a sequence without an adapter (id < 0) get zeros.  The fp32 result has the
// layout of one more split partial of the shared projection (LS_EPI_SPLIT_F32),
// so the kernel that adds the partials adds the adapter too and the projection
// plus its adapter round once.  u stays in fp32 (workspace).
//
// Shrink: one CTA per token, one warp per rank row.  Expand: one thread per
// output.
#include "common.cuh"

namespace lsb {

struct LoraParams {
  const __nv_bfloat16* x;        // [M, K]
  const __nv_bfloat16* a;        // [adapters, R, K]
  const __nv_bfloat16* b;        // [adapters, N, R]
  const float* scaling;          // [adapters]
  const int* ids;                // [batch]
  float* u;                      // [M, R]
  float* out;                    // [M, N]
  int* err;
  int q_len, K, N, R, adapters, accumulate;
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

__global__ void __launch_bounds__(256) lora_shrink_kernel(LoraParams p) {
  grid_dep_wait();
  grid_dep_launch();
  const int t = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int id = lora_adapter(p, t / p.q_len);
  if (id < 0) return;
  const __nv_bfloat16* xr = p.x + (size_t)t * p.K;
  for (int r = warp; r < p.R; r += 8) {
    const __nv_bfloat16* ar = p.a + ((size_t)id * p.R + r) * p.K;
    float acc = 0.f;
    for (int v = lane; v < p.K / 8; v += 32) acc = dot8(ldg16(ar + v * 8), ldg16(xr + v * 8), acc);
    acc = warp_sum(acc);
    if (lane == 0) p.u[(size_t)t * p.R + r] = acc;
  }
}

__global__ void __launch_bounds__(256) lora_expand_kernel(LoraParams p) {
  grid_dep_wait();
  grid_dep_launch();
  const int t = blockIdx.x, n = blockIdx.y * 256 + threadIdx.x;
  const int id = lora_adapter(p, t / p.q_len);
  if (n >= p.N) return;
  float acc = 0.f;
  if (id >= 0) {
    const __nv_bfloat16* br = p.b + ((size_t)id * p.N + n) * p.R;
    const float* ur = p.u + (size_t)t * p.R;
    for (int r = 0; r < p.R; r += 8) {
      float f[8];
      unpack8(ldg16(br + r), f);
#pragma unroll
      for (int j = 0; j < 8; ++j) acc = fmaf(ur[r + j], f[j], acc);
    }
    acc *= p.scaling[id];
  }
  float* o = p.out + (size_t)t * p.N + n;
  *o = p.accumulate ? *o + acc : acc;
}

}  // namespace lsb

namespace lsb_host {
using namespace lsb;

static int64_t lora_workspace(int64_t batch, int64_t q_len, int64_t rank) { return batch * q_len * rank * 4; }

template <typename Kernel>
static cudaError_t launch_lora_kernel(Kernel kernel, dim3 grid, const LoraParams& p, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

static int launch_lora(const LoraParams& p, int64_t batch, cudaStream_t stream) {
  const unsigned m = (unsigned)(batch * p.q_len);
  cudaError_t e = launch_lora_kernel(lora_shrink_kernel, dim3(m), p, stream);
  if (e == cudaSuccess) e = launch_lora_kernel(lora_expand_kernel, dim3(m, (unsigned)((p.N + 255) / 256)), p, stream);
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
  *bytes = lora_workspace(batch, q_len, rank);
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
  p.q_len = (int)q_len;
  p.K = (int)k;
  p.N = (int)n;
  p.R = (int)rank;
  p.adapters = (int)adapters;
  p.accumulate = accumulate ? 1 : 0;
  return launch_lora(p, batch, (cudaStream_t)stream);
}

}  // extern "C"
