// Attention of a batch whose sequences share a prefix held once (head_dim 128).
//
// Query row (token i of sequence b, head h) attends over the P keys of the
// shared prefix of its kv head and over keys 0 .. cache_pos[b] + i of its own
// static cache strip, one softmax over both (the mask of
// src/leanstack/runtime/qwen_explicit.py:551-563 with the prefix in front).
//
// The softmax splits over the keys: with m the maximum of a group of scores,
// l = sum e^(s - m) and O = sum e^(s - m) v, groups join as
//   M = max m,  o = sum_g e^(m_g - M) O_g / sum_g e^(m_g - M) l_g.
// So the prefix is one group per key split, formed once for ALL query rows of a
// kv head (B q_len G rows, whatever sequence they belong to) by prefix_tc_kernel;
// a sequence's cache strip is a few more, formed beside it by strip_groups_kernel;
// prefix_join_kernel joins them.  Per prefix key and kv head 512 bytes are read
// once for R rows and 4 D R flops done on them: memory is the bound below about
// 250 rows, the tensor cores above.
//
// prefix_tc_kernel:
//   * warp 8 streams 64-key K and V tiles with TMA (128-byte swizzle, boxes of
//     32 keys so that a split's last tile fetches little more than it needs)
//     through a ring of 16 KB slots;
//   * warps 9 and 10 issue S = Q K^T into TMEM (fp32, 64 columns) and O += P V
//     with P taken from TMEM, where it replaces the S it came from.  A warp needs
//     about 1100 cycles to wait for and issue a tile's two products, more than
//     they take, so each stream has its own where both use every tile (kRows,
//     kFull: every slot is then seen, in ring order, and released by both).  With
//     kKeys one warp issues for both streams: a slot belongs to one of them, and
//     only a reader that has seen a slot's every use can tell their parities
//     apart.  There memory (1400 cycles a tile at its share of HBM) is slower;
//   * warps 0-7 are two softmax streams of 128 threads, one thread per row, a
//     whole 64-key row of S in registers: no shuffles, no shared memory on the
//     way from S to P.  Each stream has two S buffers, so the scores of its next
//     tile are there when it is done with one.  Rows (kRows): the streams hold
//     two 128-row tiles and share every K/V tile.  Keys (kKeys, at most 128
//     rows): they hold the same rows and take alternate K/V tiles; their results
//     join in the epilogue, and 114 KB of shared memory and 128 registers leave
//     room for five strip CTAs on the same SM.
//   * P goes into the product as two bf16, hi = bf16(p) and lo = bf16(p - hi), so
//     to 2^-16 of itself, as in the attention kernels without a prefix; one bf16
//     (2^-8) shifts every key of equal score the same way, against a row sum that
//     is taken in fp32.  The pair takes the place of the scores: columns 0 - 31 and
//     32 - 63 of their buffer.  The maximum in use moves only when a score exceeds
//     it by 2^8; then O is rescaled in TMEM.
//   * kFull: a prompt's rows.  A CTA owns 256 rows of one (sequence, kv head)
//     and walks the prefix tiles, then the sequence's own tiles with the causal
//     mask, and writes the finished rows: no partials, no join.
//
// Measured with 32 / 8 heads, all kernels together: 32 sequences behind 8192 keys, 372
// own ones each, 27.9 us (83 MB, 3.0 TB/s; each kernel alone and cold: prefix 16.7, strips
// 15.4 in two to three waves of single warps, join 6.3); 13 x 5 rows (16 / 8 heads) behind
// 5003 keys 24.9 us; 6 prompts of 384 behind 8192 keys 351 us (909 TFLOP/s, 1360 with the
// products of the low halves; 410 in runs long enough for the power cap); 2 sequences
// behind 300 keys 6.6 us.  With P as one bf16 these were 26.7, 23.5, 293 and 6.1 us.
#include <algorithm>
#include <cmath>

#include "mma_sync.cuh"
#include "tcgen05.cuh"

namespace lsb {

constexpr int kSpHeadDim = 128;
constexpr int kSpRows = 128;                       // rows of one stream (MMA M)
constexpr int kSpKeys = 64;                        // keys per tile
constexpr int kSpBox = 32;                         // keys per TMA box
constexpr int kSpQHalf = kSpRows * 128;            // 64 dims of 128 rows: 16 KB
constexpr int kSpQ = 2 * kSpQHalf;                 // one 128-row Q tile: 32 KB
constexpr int kSpKvHalf = kSpKeys * 128;           // 64 dims of 64 keys: 8 KB
constexpr int kSpSlot = 2 * kSpKvHalf;             // one K or V tile: 16 KB
constexpr int kSpSoft = 256;
constexpr float kSpRescaleLog2 = 8.f;
enum SpMode { kKeys = 0, kRows = 1, kFull = 2, kFew = 3 };  // (kFew: without prefix_tc_kernel)
constexpr int sp_threads(int mode) { return mode == kKeys ? 320 : 352; }
constexpr int sp_slots(int mode) { return mode == kKeys ? 5 : 8; }
constexpr int sp_ahead(int mode) { return mode == kKeys ? 4 : 2; }  // tiles whose S is issued before the first PV
constexpr int sp_ring(int mode) { return mode == kKeys ? kSpQ : 2 * kSpQ; }  // ring offset, behind Q
constexpr int sp_bars(int mode) { return sp_ring(mode) + sp_slots(mode) * kSpSlot; }
constexpr int sp_smem(int mode) { return 1024 + sp_bars(mode) + 256; }

struct SpParams {
  const __nv_bfloat16* q;  // [M, Hq, D]
  const int* cache_pos;    // [B] or null (then uniform_past); kFull only
  int uniform_past;
  float* part_o;           // [Hkv][rows][n_part][D]: unnormalised O of each key group
  float2* part_ml;         // [Hkv][rows][n_part]: (m, l)
  __nv_bfloat16* out;      // kFull: [M, Hq * D]
  int* err;
  int rows;                // kKeys / kRows: B q_len G; kFull: q_len G
  int q_len, Hq, Hkv, G, P, prefix_cap, max_seq, splits, n_part;
  // The maximum is taken before the scale, which is positive here: the sign of the
  // caller's goes to the query rows (q ^ q_flip), and a scale of 0 makes them 0 (q & q_keep).
  float scale_log2;
  uint32_t q_keep, q_flip;
};

template <int MODE>
__global__ void __launch_bounds__(MODE == kKeys ? 512 : sp_threads(MODE), 1)  // kKeys: at most 128 registers
    prefix_tc_kernel(const __grid_constant__ CUtensorMap tm_kp, const __grid_constant__ CUtensorMap tm_vp,
                     const __grid_constant__ CUtensorMap tm_kc, const __grid_constant__ CUtensorMap tm_vc, SpParams p) {
  constexpr int kSlots = sp_slots(MODE), kAhead = sp_ahead(MODE);
  extern __shared__ unsigned char sp_smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<size_t>(sp_smem_raw) + 1023) & ~size_t(1023));
  unsigned char* ring = smem + sp_ring(MODE);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + sp_bars(MODE));
  uint64_t* empty = full + kSlots;
  uint64_t* s_full = empty + kSlots;  // [stream][buffer]: scores are in TMEM
  uint64_t* p_full = s_full + 4;      // [stream][buffer]: probabilities are in TMEM
  uint64_t* o_part = p_full + 4;      // [stream][buffer]: the product that read them is done
  uint64_t* o_done = o_part + 4;      // [issuing warp]: its last product is done
  uint64_t* q_full = o_done + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(q_full + 1);
  __shared__ int s_abort;
  __shared__ float2 s_ml[2][kSpRows];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row_blk = MODE == kFull ? gridDim.x - 1 - blockIdx.x : blockIdx.y;  // kFull: the longest first
  const int r0 = row_blk * (MODE == kKeys ? kSpRows : 2 * kSpRows);
  const bool both = MODE != kKeys && r0 + kSpRows < p.rows;  // two row tiles: both streams use every K/V tile
  if (threadIdx.x == 0) {
    for (int s = 0; s < kSlots; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], both ? 2 : 1);
    }
    for (int w = 0; w < 4; ++w) {
      mbar_init(&s_full[w], 1);
      mbar_init(&p_full[w], kSpRows);
      mbar_init(&o_part[w], 1);
    }
    mbar_init(q_full, kSpSoft);
    mbar_init(&o_done[0], 1);
    mbar_init(&o_done[1], 1);
    s_abort = 0;
    mbar_fence_init();
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;  // stream w: S buffers at columns 128 w and 128 w + 64, O at 256 + 128 w

  // Every CTA waits before it lets the next kernel start: what that kernel reads
  // besides this one's results was complete before.
  grid_dep_wait();
  grid_dep_launch();

  // This CTA's rows and keys.
  const int h = MODE == kFull ? blockIdx.y : blockIdx.z;
  const int b = MODE == kFull ? blockIdx.z : 0;
  const int split = MODE == kFull ? 0 : blockIdx.x;
  int k0 = 0, k1 = p.P;  // prefix keys
  if (MODE != kFull) {   // 16-key units, evenly over the splits
    const int units = (p.P + 15) / 16;
    k0 = (int)((long long)units * split / p.splits) * 16;
    k1 = min((int)((long long)units * (split + 1) / p.splits) * 16, p.P);
  }
  const int n_pre = (k1 - k0 + kSpKeys - 1) / kSpKeys;
  int cp = 0, own = 0;  // kFull: cursor, and own keys that the last row of the block sees
  if (MODE == kFull) {
    cp = p.cache_pos ? __ldcg(p.cache_pos + b) : p.uniform_past;
    if ((cp < 0 || cp > p.max_seq - p.q_len) && threadIdx.x == 0 && blockIdx.x == 0)
      raise_device_error(p.err, LS_ERR_KV_OVERFLOW);
    cp = min(cp, p.max_seq);
    own = min(max(cp + (min(r0 + 2 * kSpRows, p.rows) - 1) / p.G + 1, 0), p.max_seq);
  }
  const int ntiles = n_pre + (MODE == kFull ? (own + kSpKeys - 1) / kSpKeys : 0);
  const bool two = MODE == kKeys ? ntiles > 1 : both;  // the second stream has work
  // Keys of tile t, and its first row in the K/V tensor maps.
  auto tile_keys = [&](int t) -> int {
    return t < n_pre ? min(kSpKeys, k1 - k0 - t * kSpKeys) : min(kSpKeys, own - (t - n_pre) * kSpKeys);
  };
  // The ring holds K of the first kAhead tiles, then V_0, K_kAhead, V_1, ...: the
  // order in which they are used.  Position of V_t:
  auto idx_v = [&](int t) { return min(ntiles, kAhead) + t + max(0, min(t, ntiles - kAhead)); };

  if (warp == 8) {
    // ---------------- TMA producer ----------------
    if (lane == 0) {
      int it = 0;
      bool ok = true;
      auto load = [&](int t, bool key) {
        const int s = it % kSlots;
        if (!ok || *(volatile int*)&s_abort ||
            (it >= kSlots && !mbar_wait(&empty[s], (uint32_t)(it / kSlots - 1) & 1u, p.err, 0x31))) {
          ok = false;
          return;
        }
        const bool pre = t < n_pre;
        const CUtensorMap* map = pre ? (key ? &tm_kp : &tm_vp) : (key ? &tm_kc : &tm_vc);
        const int y = pre ? h * p.prefix_cap + k0 + t * kSpKeys : (b * p.Hkv + h) * p.max_seq + (t - n_pre) * kSpKeys;
        const int boxes = (tile_keys(t) + kSpBox - 1) / kSpBox;
        unsigned char* st = ring + s * kSpSlot;
        mbar_arrive_expect_tx(&full[s], (uint32_t)boxes * kSpBox * 256);
        for (int x = 0; x < boxes; ++x) {
          tma_load_2d(st + x * kSpBox * 128, map, 0, y + x * kSpBox, &full[s]);
          tma_load_2d(st + kSpKvHalf + x * kSpBox * 128, map, 64, y + x * kSpBox, &full[s]);
        }
        ++it;
      };
      for (int t = 0; t < min(ntiles, kAhead); ++t) load(t, true);
      for (int t = 0; t < ntiles; ++t) {
        load(t, false);
        if (t + kAhead < ntiles) load(t + kAhead, true);
      }
      // After a timeout nobody reads the last copies: wait until they have landed.
      for (int j = max(0, it - kSlots); !ok && j < it; ++j) mbar_wait(&full[j % kSlots], (uint32_t)(j / kSlots) & 1u, p.err, 0x32);
    }
  } else if (warp >= 9) {
    // ---------------- MMA issuers: the whole warp, uniformly ----------------
    const int w0 = __shfl_sync(0xffffffffu, warp - 9, 0);
    if (ntiles > 0 && (w0 == 0 || two)) {
      constexpr uint32_t idesc_s = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(kSpKeys >> 3) << 17) |
                                   ((uint32_t)(kSpRows >> 4) << 24);
      constexpr uint32_t idesc_pv = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) |
                                    ((uint32_t)(kSpHeadDim >> 3) << 17) | ((uint32_t)(kSpRows >> 4) << 24);  // V MN-major
      const uint64_t q_desc = umma_desc_sw128(smem_u32(smem) + w0 * kSpQ);
      const uint64_t k_desc = umma_desc_sw128(smem_u32(ring)), v_desc = umma_desc_sw128_mn(smem_u32(ring), kSpKvHalf);
      bool ok = mbar_wait(q_full, 0u, p.err, 0x35);
      // The ring is consumed in order: the next slot and its parity.
      int slot = 0;
      uint32_t parity = 0;
      auto take = [&]() -> int {
        const int s = slot;
        ok = ok && mbar_wait(&full[s], parity, p.err, 0x33);
        if (++slot == kSlots) slot = 0, parity ^= 1u;
        return s;
      };
      // Stream w's j-th tile: S = Q K^T into buffer j & 1.  Products run in the order
      // of issue, so the P that the buffer held has been read.
      auto issue_s = [&](int w, int j, int s) {
        umma_k128_n64(tmem + w * 128 + (j & 1) * kSpKeys, q_desc, k_desc + s * (kSpSlot >> 4), idesc_s, 0u);
        umma_commit_warp(&s_full[2 * w + (j & 1)]);
        umma_commit_warp(&empty[s]);
      };
      for (int t = 0; ok && t < min(ntiles, kAhead); ++t) {
        const int s = take();
        if (!ok) break;
        tc_fence_after();
        if (MODE == kKeys) issue_s(t & 1, t >> 1, s);
        else issue_s(w0, t, s);
      }
      for (int t = 0; ok && t < ntiles; ++t) {
        const int w = MODE == kKeys ? t & 1 : w0, j = MODE == kKeys ? t >> 1 : t;
        const bool more = t + kAhead < ntiles;
        const int sv = take();
        const int sk = more ? take() : 0;
        ok = ok && mbar_wait(&p_full[2 * w + (j & 1)], (uint32_t)(j >> 1) & 1u, p.err, 0x34);
        if (!ok) break;
        tc_fence_after();
        const uint32_t tP = tmem + w * 128 + (j & 1) * kSpKeys;
        umma_ta_k64(tmem + 256 + w * 128, tP, v_desc + sv * (kSpSlot >> 4), idesc_pv, j > 0 ? 1u : 0u);  // O += P V
        umma_ta_k64(tmem + 256 + w * 128, tP + kSpKeys / 2, v_desc + sv * (kSpSlot >> 4), idesc_pv, 1u);
        if (more) issue_s(w, j + 2, sk);
        umma_commit_warp(&o_part[2 * w + (j & 1)]);
        umma_commit_warp(&empty[sv]);
      }
      if (!ok && lane == 0) s_abort = 1;
      umma_commit_warp(&o_done[w0]);
      mbar_wait(&o_done[w0], 0u, p.err, 0x36);  // every product issued here is done before TMEM is given back
    }
  } else {
    // ---------------- softmax streams: warps 0-3 and 4-7, one thread per row ----------------
    const int w = warp >> 2, quad = warp & 3, r = quad * 32 + lane;
    const int row = r0 + (MODE == kKeys ? r : w * kSpRows + r);
    const bool valid = row < p.rows;
    const bool warp_valid = __any_sync(0xffffffffu, valid);
    // Query rows into the swizzled tiles: 16 lanes a row, zeros behind the end;
    // eight loads in flight per thread before the first store.
#pragma unroll
    for (int tile = 0; tile < (MODE == kKeys ? 1 : 2); ++tile) {
      uint4 v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int gr = r0 + tile * kSpRows + (int)(threadIdx.x >> 4) + 16 * u, t = gr / p.G;
        v[u] = make_uint4(0, 0, 0, 0);
        if (gr < p.rows)
          v[u] = __ldcg(reinterpret_cast<const uint4*>(
                            p.q + (((size_t)b * p.q_len + t) * p.Hq + h * p.G + (gr - t * p.G)) * kSpHeadDim) +
                        (threadIdx.x & 15));
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        v[u].x = (v[u].x & p.q_keep) ^ p.q_flip;
        v[u].y = (v[u].y & p.q_keep) ^ p.q_flip;
        v[u].z = (v[u].z & p.q_keep) ^ p.q_flip;
        v[u].w = (v[u].w & p.q_keep) ^ p.q_flip;
        *reinterpret_cast<uint4*>(smem + tile * kSpQ + pt_off((threadIdx.x >> 4) + 16 * u, threadIdx.x & 15, kSpQHalf)) = v[u];
      }
    }
    fence_proxy_async_smem();
    mbar_arrive(q_full);

    const int lim = MODE == kFull ? (valid ? cp + row / p.G : -1) : 0;  // kFull: the row's last own key
    const uint32_t lane_off = (uint32_t)(quad * 32) << 16;
    const uint32_t tO = tmem + 256 + w * 128 + lane_off;
    float m_run = -INFINITY, l_run = 0.f;
    bool ok = true;
    const int step = MODE == kKeys ? 2 : 1;
    const int t_end = w == 0 || two ? ntiles : 0;
    for (int t = MODE == kKeys ? w : 0, j = 0; t < t_end; t += step, ++j) {
      // Wait results are made warp-uniform: the TMEM accesses are warp-collective.
      if (!__all_sync(0xffffffffu, mbar_wait(&s_full[2 * w + (j & 1)], (uint32_t)(j >> 1) & 1u, p.err, 0x37))) {
        ok = false;
        break;
      }
      tc_fence_after();
      const int nk = tile_keys(t);
      if (warp_valid) {
        const int vis = t < n_pre ? nk : min(nk, lim + 1 - (t - n_pre) * kSpKeys);  // keys of the tile the row sees
        const uint32_t tS = tmem + w * 128 + (j & 1) * kSpKeys + lane_off;
        uint32_t sv[kSpKeys];
        tmem_ld64(tS, sv);
        if (!__all_sync(0xffffffffu, vis >= kSpKeys)) {
#pragma unroll
          for (int e = 0; e < kSpKeys; ++e)
            if (e >= vis) sv[e] = 0xff800000u;  // -inf
        }
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int e = 0; e < kSpKeys; e += 4) {
#pragma unroll
          for (int a = 0; a < 4; ++a) mx[a] = fmaxf(mx[a], __uint_as_float(sv[e + a]));
        }
        const float mraw = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
        const float mt = mraw == -INFINITY ? -INFINITY : mraw * p.scale_log2;
        float corr = 1.f;
        if (m_run == -INFINITY) {
          m_run = mt;  // the row's first visible keys: nothing accumulated yet
        } else if (mt > m_run + kSpRescaleLog2) {
          corr = ex2_approx(m_run - mt);
          m_run = mt;
        }
        // O is rescaled once the product of the tile before is in it; the whole
        // warp joins when any of its rows needs the new scale.
        if (__any_sync(0xffffffffu, corr != 1.f)) {
          if (!__all_sync(0xffffffffu, mbar_wait(&o_part[2 * w + ((j - 1) & 1)], (uint32_t)((j - 1) >> 1) & 1u, p.err, 0x3a))) {
            ok = false;
            break;
          }
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < 8; ++c) {
            float ov[16];
            tmem_ld16(tO + (uint32_t)(c * 16), ov);
#pragma unroll
            for (int e = 0; e < 16; ++e) ov[e] *= corr;
            tmem_st16(tO + (uint32_t)(c * 16), ov);
          }
        }
        const float neg_m = m_run == -INFINITY ? 0.f : -m_run;  // a row without keys so far: exp2(-inf) = 0
        const float2 scale2 = make_float2(p.scale_log2, p.scale_log2), neg2 = make_float2(neg_m, neg_m);
        float2 ls[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        uint32_t hi[kSpKeys / 2], lo[kSpKeys / 2];
#pragma unroll
        for (int e = 0; e < kSpKeys / 2; ++e) {
          float2 x = fma2(make_float2(__uint_as_float(sv[2 * e]), __uint_as_float(sv[2 * e + 1])), scale2, neg2);
          x.x = ex2_approx(x.x);
          x.y = ex2_approx(x.y);
          ls[e & 1] = add2(ls[e & 1], x);
          hi[e] = pack_bf16(x.x, x.y);
          x = fma2(make_float2(__uint_as_float(hi[e] << 16), __uint_as_float(hi[e] & 0xffff0000u)), make_float2(-1.f, -1.f), x);
          lo[e] = pack_bf16(x.x, x.y);
        }
        tmem_st32(tS, hi);
        tmem_st32(tS + kSpKeys / 2, lo);
        l_run = l_run * corr + ((ls[0].x + ls[0].y) + (ls[1].x + ls[1].y));
        tmem_st_wait();
      }
      if (nk < kSpKeys) {
        // The product takes 64 keys: clear the V rows past the tile's end (the
        // memory there is the caller's or not loaded, and 0 x NaN is NaN).  Two
        // streams that share the tile both do: neither waits for the other.
        const int it = idx_v(t);
        if (!__all_sync(0xffffffffu, mbar_wait(&full[it % kSlots], (uint32_t)(it / kSlots) & 1u, p.err, 0x38))) {
          ok = false;
          break;
        }
        unsigned char* vt = ring + (it % kSlots) * kSpSlot;
        for (int c = r; c < (kSpKeys - nk) * 16; c += kSpRows)
          *reinterpret_cast<uint4*>(vt + pt_off(nk + (c >> 4), c & 15, kSpKvHalf)) = make_uint4(0, 0, 0, 0);
        fence_proxy_async_smem();
      }
      tc_fence_before();
      mbar_arrive(&p_full[2 * w + (j & 1)]);
    }
    if (!ok) s_abort = 1;
    // ---------------- epilogue ----------------
    const int wd = MODE == kKeys ? 0 : w;  // the warp that issued this stream's products
    // kRows with two row tiles: the ring is idle only when the other stream's products are
    // done too, which read the same tiles and may be some behind.
    const bool fin = ntiles > 0 &&
                     __all_sync(0xffffffffu, ok && (wd == 1 && !two ? true : mbar_wait(&o_done[wd], 0u, p.err, 0x39)) &&
                                                 (MODE != kRows || !both || mbar_wait(&o_done[wd ^ 1], 0u, p.err, 0x3b)));
    tc_fence_after();
    // Partials go out through shared memory (the ring, idle now): a thread holds
    // a row, a warp writes whole 512-byte rows.  16-byte chunk c of row x sits at
    // chunk c ^ (x mod 32): no bank conflicts either way.
    float4* stage = reinterpret_cast<float4*>(ring) + (MODE == kKeys ? 0 : w * kSpRows * 32);
    if (MODE == kKeys) {
      // Join the two streams: each forms one half of the dims of the rows.
      s_ml[w][r] = make_float2(m_run, l_run);
      named_bar_sync(1, kSpSoft);
      if (fin && warp_valid) {
        const float2 a = s_ml[0][r], c = s_ml[1][r];
        const float m = fmaxf(a.x, c.x);
        const float fa = a.x == -INFINITY ? 0.f : ex2_approx(a.x - m), fc = c.x == -INFINITY ? 0.f : ex2_approx(c.x - m);
        if (w == 0 && valid)
          p.part_ml[((size_t)h * p.rows + row) * p.n_part + split] = make_float2(m, a.y * fa + c.y * fc);
#pragma unroll 1
        for (int c32 = 0; c32 < 2; ++c32) {
          float o0[32], o1[32];
          tmem_ld32(tmem + 256 + lane_off + (uint32_t)(w * 64 + c32 * 32), o0);
          if (two) tmem_ld32(tmem + 384 + lane_off + (uint32_t)(w * 64 + c32 * 32), o1);
#pragma unroll
          for (int e = 0; e < 32; ++e) o0[e] = o0[e] * fa + (two ? o1[e] * fc : 0.f);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            stage[r * 32 + ((w * 16 + c32 * 8 + e) ^ (r & 31))] =
                make_float4(o0[4 * e], o0[4 * e + 1], o0[4 * e + 2], o0[4 * e + 3]);
          __syncwarp();
        }
      }
      named_bar_sync(1, kSpSoft);
    } else if (fin && warp_valid) {
      const int tok = valid ? row / p.G : 0;
      // A row without a key has no weight at all and gives zeros; a NaN or infinite score
      // makes the sum NaN, and NaN goes out.
      const float inv = l_run == 0.f ? 0.f : 1.f / l_run;
      if (MODE == kRows && valid) p.part_ml[((size_t)h * p.rows + row) * p.n_part + split] = make_float2(m_run, l_run);
#pragma unroll 1
      for (int c16 = 0; c16 < 8; ++c16) {
        float ov[16];
        tmem_ld16(tO + (uint32_t)(c16 * 16), ov);
        if (MODE == kRows) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            stage[r * 32 + ((c16 * 4 + e) ^ (r & 31))] =
                make_float4(ov[4 * e], ov[4 * e + 1], ov[4 * e + 2], ov[4 * e + 3]);
        } else if (valid) {
          uint32_t pk[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const __nv_bfloat162 v2 = __floats2bfloat162_rn(l_run == 0.f ? 0.f : ov[2 * e] * inv,
                                                            l_run == 0.f ? 0.f : ov[2 * e + 1] * inv);
            pk[e] = *reinterpret_cast<const uint32_t*>(&v2);
          }
          uint4* dst = reinterpret_cast<uint4*>(
              p.out + (((size_t)b * p.q_len + tok) * p.Hq + h * p.G + (row - tok * p.G)) * kSpHeadDim + c16 * 16);
          dst[0] = make_uint4(pk[0], pk[1], pk[2], pk[3]);
          dst[1] = make_uint4(pk[4], pk[5], pk[6], pk[7]);
        }
        __syncwarp();
      }
    }
    if (MODE != kFull && fin) {  // kRows: a warp's own rows; kKeys: 16 of the joined ones
      const int x0 = MODE == kKeys ? warp * 16 : quad * 32, n = MODE == kKeys ? 16 : 32;
      const int g0 = r0 + (MODE == kKeys ? 0 : w * kSpRows);
      float4* dst = reinterpret_cast<float4*>(p.part_o) + (((size_t)h * p.rows + g0) * p.n_part + split) * 32 + lane;
#pragma unroll 8
      for (int x = x0; x < x0 + n && g0 + x < p.rows; ++x)
        dst[(size_t)x * p.n_part * 32] = stage[x * 32 + (lane ^ (x & 31))];
    }
    if (MODE == kFull && ntiles == 0 && valid) {  // no key at all (a cursor outside the cache): zeros
      const int tok = row / p.G;
      uint4* dst = reinterpret_cast<uint4*>(
          p.out + (((size_t)b * p.q_len + tok) * p.Hq + h * p.G + (row - tok * p.G)) * kSpHeadDim);
      for (int c = 0; c < 16; ++c) dst[c] = make_uint4(0, 0, 0, 0);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
}

// Groups of a sequence's own strip: one warp per (sequence, kv head, 16 query
// rows, key chunk), mma.sync m16n8k16 on 16-key tiles from a 2-stage cp.async
// ring, online softmax in registers, P as two bf16 as in prefix_tc_kernel.
// A chunk is a row's share of its sequence's keys, at least kStMinBlocks tiles; a
// chunk behind the end leaves a group without weight.  Single warps: nothing to
// merge, and the SM's scheduler evens out strips of different lengths.  kFew: a short
// prefix of at most 16 rows in all is taken as one more sequence, whose rows see all of it.
constexpr int kStMinBlocks = 4;
constexpr int kStStages = 2;
constexpr int kStTile = 16 * kTaHeadDim * 2;  // 16 keys of K or V: 4 KB

struct StParams {
  const __nv_bfloat16* q;
  const __nv_bfloat16* k_cache;
  const __nv_bfloat16* v_cache;
  const int* cache_pos;
  int uniform_past;
  float* part_o;    // groups n_pre .. n_part - 1 are written here
  float2* part_ml;
  int* err;
  const __nv_bfloat16* k_prefix;  // kFew: the prefix is sequence `batch`, its rows those of all (16 at most)
  const __nv_bfloat16* v_prefix;
  int batch, P, prefix_cap, own;  // own: groups of a sequence's strip
  int q_len, Hq, Hkv, G, R, RG, max_seq, n_pre, n_part;
  int behind;       // prefix_tc_kernel was launched before
  float scale_log2;
};

__global__ void __launch_bounds__(32) strip_groups_kernel(StParams p) {
  __shared__ __align__(128) unsigned char sm[kStStages * 2 * kStTile + kStTile];
  // Behind a prefix: that kernel's CTAs let this one start only after every kernel
  // before is complete, so what is read here is there, and one CTA waits for it at
  // the end, so that whoever waits for this kernel has both.
  if (!p.behind) grid_dep_wait();
  grid_dep_launch();
  const int lane = threadIdx.x, g8 = lane >> 2, t4 = lane & 3;
  const bool pre = (int)blockIdx.z == p.batch;
  const int hkv = blockIdx.y / p.RG, r0 = (blockIdx.y - hkv * p.RG) * 16;
  const int b = pre ? 0 : blockIdx.z, R = pre ? p.batch * p.R : p.R, groups = pre ? p.n_pre : p.own;
  if ((int)blockIdx.x >= groups) return;  // (only where `pre` makes the grid wider)
  const int nrows = min(16, R - r0);
  int L = p.P, cp = 0;  // the first L keys; row r sees those up to cp + r / G, of the prefix all
  if (!pre) {
    cp = p.cache_pos ? __ldcg(p.cache_pos + b) : p.uniform_past;
    if ((cp < 0 || cp > p.max_seq - p.q_len) && lane == 0) raise_device_error(p.err, LS_ERR_KV_OVERFLOW);
    cp = min(cp, p.max_seq);
    L = min(max(cp + p.q_len, 0), p.max_seq);
  }
  const int blocks = (L + 15) / 16;
  const int per = max((blocks + groups - 1) / groups, kStMinBlocks);
  const int blk0 = min((int)blockIdx.x * per, blocks), nb = min(per, blocks - blk0);
  // row r: + r n_part
  const size_t at = (((size_t)hkv * p.batch + b) * p.R + r0) * p.n_part + (pre ? 0 : p.n_pre) + blockIdx.x;
  if (nb <= 0) {
    if (lane < nrows) p.part_ml[at + (size_t)lane * p.n_part] = make_float2(-INFINITY, 0.f);
  } else {
    const size_t base = pre ? (size_t)hkv * p.prefix_cap * kTaHeadDim : ((size_t)b * p.Hkv + hkv) * p.max_seq * kTaHeadDim;
    const __nv_bfloat16 *keys = pre ? p.k_prefix : p.k_cache, *values = pre ? p.v_prefix : p.v_cache;
    const uint32_t ring = smem_u32(sm), sq = ring + kStStages * 2 * kStTile;
#pragma unroll
    for (int it = 0; it < 8; ++it) {  // the query rows, zeros behind the end; with the first tiles' copies
      const int r = (lane >> 4) + 2 * it, row = r0 + (r < nrows ? r : 0);
      const int i = row / p.G, gq = row - i * p.G;
      cp_async16(sq + ta_swz(r, lane & 15),
                 p.q + (((size_t)b * p.q_len + i) * p.Hq + hkv * p.G + gq) * kTaHeadDim + (lane & 15) * 8,
                 r < nrows ? 16u : 0u);
    }
    auto load_block = [&](int n) {
      const uint32_t st = ring + (n % kStStages) * 2 * kStTile;
#pragma unroll
      for (int it = 0; it < 8; ++it) {
        const int r = (lane >> 4) + 2 * it, j = (blk0 + n) * 16 + r;
        const bool ok = j < L;
        const size_t off = base + (size_t)(ok ? j : 0) * kTaHeadDim + (lane & 15) * 8;
        cp_async16(st + ta_swz(r, lane & 15), keys + off, ok ? 16u : 0u);
        cp_async16(st + kStTile + ta_swz(r, lane & 15), values + off, ok ? 16u : 0u);
      }
    };
#pragma unroll
    for (int n = 0; n < kStStages; ++n) {
      if (n < nb) load_block(n);
      cp_async_commit();
    }
    int lim[2];  // last key the rows g8 and g8 + 8 see
#pragma unroll
    for (int hr = 0; hr < 2; ++hr) lim[hr] = g8 + 8 * hr >= nrows ? -1 : pre ? L - 1 : cp + (r0 + g8 + 8 * hr) / p.G;
    uint32_t qa[8][4];
    float o[16][4];
#pragma unroll
    for (int nt = 0; nt < 16; ++nt) o[nt][0] = o[nt][1] = o[nt][2] = o[nt][3] = 0.f;
    float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f};
    for (int n = 0; n < nb; ++n) {
      cp_async_wait<kStStages - 1>();
      __syncwarp();
      if (n == 0) {
#pragma unroll
        for (int ks = 0; ks < 8; ++ks)
          ldsm_x4(sq + ta_swz((lane & 7) + ((lane >> 3) & 1) * 8, 2 * ks + (lane >> 4)), qa[ks][0], qa[ks][1], qa[ks][2],
                  qa[ks][3]);
      }
      const uint32_t stK = ring + (n % kStStages) * 2 * kStTile, stV = stK + kStTile;
      const int jb = (blk0 + n) * 16;
      float sc[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int ks = 0; ks < 8; ++ks) {
        uint32_t b00, b01, b10, b11;
        ldsm_x4(stK + ta_swz((lane & 7) + ((lane >> 4) << 3), 2 * ks + ((lane >> 3) & 1)), b00, b01, b10, b11);
        mma_bf16(sc[0], qa[ks], b00, b01);
        mma_bf16(sc[1], qa[ks], b10, b11);
      }
      float corr[2];
#pragma unroll
      for (int hr = 0; hr < 2; ++hr) {  // row g8 + 8 hr: elements 2 hr, 2 hr + 1 of both tiles
        float mx = -INFINITY;
#pragma unroll
        for (int nt = 0; nt < 2; ++nt)
#pragma unroll
          for (int e = 2 * hr; e < 2 * hr + 2; ++e) {
            const int j = jb + nt * 8 + 2 * t4 + (e & 1);
            const float v = j < L && j <= lim[hr] ? sc[nt][e] * p.scale_log2 : -INFINITY;
            sc[nt][e] = v;
            mx = fmaxf(mx, v);
          }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float mn = fmaxf(m_run[hr], mx);
        corr[hr] = m_run[hr] == mn ? 1.f : ex2_approx(m_run[hr] - mn);
        m_run[hr] = mn;
        const float neg = mn == -INFINITY ? 0.f : -mn;
        float ps = 0.f;
#pragma unroll
        for (int nt = 0; nt < 2; ++nt)
#pragma unroll
          for (int e = 2 * hr; e < 2 * hr + 2; ++e) {
            sc[nt][e] = ex2_approx(sc[nt][e] + neg);
            ps += sc[nt][e];
          }
        l_run[hr] = l_run[hr] * corr[hr] + ps;
      }
      if (__any_sync(0xffffffffu, corr[0] != 1.f || corr[1] != 1.f)) {
#pragma unroll
        for (int nt = 0; nt < 16; ++nt) {
          o[nt][0] *= corr[0];
          o[nt][1] *= corr[0];
          o[nt][2] *= corr[1];
          o[nt][3] *= corr[1];
        }
      }
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const float x0 = sc[x >> 1][(x & 1) * 2], x1 = sc[x >> 1][(x & 1) * 2 + 1];
        hi[x] = pack_bf16(x0, x1);
        lo[x] = pack_bf16(x0 - __uint_as_float(hi[x] << 16), x1 - __uint_as_float(hi[x] & 0xffff0000u));
      }
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        uint32_t v0, v1, v2, v3;
        ldsm_x4_t(stV + ta_swz((lane & 7) + (((lane >> 3) & 1) << 3), 2 * c + (lane >> 4)), v0, v1, v2, v3);
        mma_bf16(o[2 * c], hi, v0, v1);
        mma_bf16(o[2 * c + 1], hi, v2, v3);
        mma_bf16(o[2 * c], lo, v0, v1);
        mma_bf16(o[2 * c + 1], lo, v2, v3);
      }
      __syncwarp();
      if (n + kStStages < nb) load_block(n + kStStages);
      cp_async_commit();
    }
    cp_async_wait<0>();
#pragma unroll
    for (int hr = 0; hr < 2; ++hr) {
      l_run[hr] += __shfl_xor_sync(0xffffffffu, l_run[hr], 1);
      l_run[hr] += __shfl_xor_sync(0xffffffffu, l_run[hr], 2);
      const int r = g8 + 8 * hr;
      if (r >= nrows) continue;
      const size_t g = at + (size_t)r * p.n_part;
      if (t4 == 0) p.part_ml[g] = make_float2(m_run[hr], l_run[hr]);
#pragma unroll
      for (int nt = 0; nt < 16; ++nt)
        *reinterpret_cast<float2*>(p.part_o + g * kTaHeadDim + nt * 8 + 2 * t4) =
            make_float2(o[nt][2 * hr], o[nt][2 * hr + 1]);
    }
  }
  if (p.behind && blockIdx.x == gridDim.x - 1 && blockIdx.y == gridDim.y - 1 && blockIdx.z == gridDim.z - 1)
    grid_dep_wait();
}

// Join of a row's key groups: one warp per row (kv head, token, group member) and
// half of its dims, a lane two of them.  The groups' weights e^(m_g - M) sit in
// the lanes, their O is read 32 groups at a time.  14 MB of partials in 3 us beside
// the launch: latency.
constexpr int kSpJoinWarps = 4;
__global__ void __launch_bounds__(kSpJoinWarps * 32) prefix_join_kernel(const float* part_o, const float2* part_ml,
                                                                        int n_part, int rows, int G, int Hq,
                                                                        __nv_bfloat16* out) {
  grid_dep_wait();
  grid_dep_launch();
  const int lane = threadIdx.x & 31, h = blockIdx.y;
  const int row = (blockIdx.x * kSpJoinWarps + (threadIdx.x >> 5)) >> 1;
  const int dim = ((threadIdx.x >> 5) & 1) * (kSpHeadDim / 2) + lane * 2;
  if (row >= rows) return;
  const size_t at = ((size_t)h * rows + row) * n_part;
  const float2* po = reinterpret_cast<const float2*>(part_o + at * kSpHeadDim + dim);
  float M = -INFINITY, l = 0.f;
  float2 o = make_float2(0.f, 0.f);
  for (int c0 = 0; c0 < n_part; c0 += 32) {
    const int n = min(32, n_part - c0);
    float2 v[32];
#pragma unroll
    for (int u = 0; u < 32; ++u)
      if (u < n) v[u] = __ldcg(po + (size_t)(c0 + u) * (kSpHeadDim / 2));
    const float2 ml = lane < n ? __ldcg(part_ml + at + c0 + lane) : make_float2(-INFINITY, 0.f);
    const float mn = fmaxf(M, warp_max(ml.x));
    if (mn == -INFINITY) {  // no key so far, or scores that are all NaN: then the sum is
      l += warp_sum(ml.y);
      continue;
    }
    const float corr = exp2f(M - mn), f = exp2f(ml.x - mn);
    const uint32_t some = __ballot_sync(0xffffffffu, ml.y != 0.f);  // a group without keys may hold anything
    M = mn;
    l = l * corr + warp_sum(ml.y * f);
    o.x *= corr, o.y *= corr;
#pragma unroll
    for (int u = 0; u < 32; ++u) {
      const float fu = __shfl_sync(0xffffffffu, f, u);
      if (u < n && (some >> u & 1u)) {
        o.x = fmaf(v[u].x, fu, o.x);
        o.y = fmaf(v[u].y, fu, o.y);
      }
    }
  }
  const float inv = 1.f / l;
  const __nv_bfloat162 v2 = l == 0.f ? __floats2bfloat162_rn(0.f, 0.f) : __floats2bfloat162_rn(o.x * inv, o.y * inv);
  const int t = row / G;
  *reinterpret_cast<__nv_bfloat162*>(out + ((size_t)t * Hq + h * G + (row - t * G)) * kSpHeadDim + dim) = v2;
}

}  // namespace lsb

namespace lsb_host {
using namespace lsb;

struct SpPlan {
  int mode, row_blocks, splits, chunks;  // key groups: the prefix's splits and the strips' chunks
  int64_t ml_bytes, bytes;
};

constexpr int kSpMaxChunks = 32;
constexpr int64_t kSpFewKeys = 2048;
// kFull when the prompt rows alone give three quarters of the SMs a CTA (one
// launch, nothing written in between); else the prefix is split over the SMs.
static SpPlan sp_plan(int64_t batch, int64_t q_len, int64_t hq, int64_t hkv, int64_t prefix_len, int64_t max_seq) {
  SpPlan pl = {};
  const int64_t g = hq / hkv, sms = sm_count();
  const int64_t own_blocks = (q_len * g + 2 * kSpRows - 1) / (2 * kSpRows);
  if (q_len * g >= 2 * kSpRows && own_blocks * hkv * batch * 4 >= sms * 3) {
    pl.mode = kFull;
    pl.row_blocks = (int)own_blocks;
    return pl;
  }
  const int64_t rows = batch * q_len * g;
  // Few rows: each K/V tile serves 128 rows and what little is computed leaves room
  // for the strips on the same SM; many: 256 rows share a tile.  Measured at 32 / 8
  // heads and 8192 shared keys, kKeys / kRows, up to 20 own keys: 192 rows 21.8 / 25.2
  // us, 384 rows 32.2 / 34.2, 768 rows 50.6 / 49.7; 40 to 700 own keys: 36.7 / 40.3,
  // 58.8 / 64.3, 104.5 / 107.9.
  pl.mode = rows <= 512 ? kKeys : kRows;
  // One row tile and a short prefix: its keys go to the strips' kernel, a launch less.
  // us without / with, and with the host's time, 4 sequences of 4 rows: 64 keys 7.4 / 6.5
  // and 8.9 / 7.4, 300 keys 7.9 / 6.6 and 9.0 / 7.3, 2000 keys 8.6 / 8.7 and 9.4 / 9.4,
  // 8192 keys 13.3 / 18.1; 1 sequence: 2000 keys 8.1 / 7.5, 8192 keys 12.7 / 17.0.
  const bool few = rows <= 16 && prefix_len <= kSpFewKeys;
  if (few) pl.mode = kFew;
  const int64_t per = pl.mode == kKeys ? kSpRows : 2 * kSpRows;
  pl.row_blocks = (int)((rows + per - 1) / per);
  // As many splits as fill the SMs once, of at least 128 keys each.
  const int64_t most = (prefix_len + 127) / 128;
  int64_t splits = sms / (hkv * pl.row_blocks);
  if (splits < 1) splits = 1;
  if (splits > most) splits = most;
  pl.splits = prefix_len > 0 ? (int)splits : 0;
  const int64_t few_splits = (std::min<int64_t>(prefix_len, kSpFewKeys) + 16 * kStMinBlocks - 1) / (16 * kStMinBlocks);
  if (few) pl.splits = (int)few_splits;
  // Strip chunks: about 2048 warps in all (14 an SM, of which 7 fit at once).
  const int64_t strips = batch * hkv * ((q_len * g + 15) / 16);
  int64_t chunks = 2048 / strips;
  const int64_t longest = (max_seq + 16 * kStMinBlocks - 1) / (16 * kStMinBlocks);
  if (chunks > longest) chunks = longest;
  if (chunks > kSpMaxChunks) chunks = kSpMaxChunks;
  pl.chunks = chunks < 1 ? 1 : (int)chunks;
  // (A longer prefix never needs less, although it may leave kFew.)
  const int64_t groups = (rows <= 16 ? std::max<int64_t>(pl.splits, few_splits) : pl.splits) + pl.chunks;
  pl.ml_bytes = (hkv * rows * groups * 8 + 255) / 256 * 256;
  pl.bytes = pl.ml_bytes + hkv * rows * groups * kSpHeadDim * 4;
  return pl;
}

// The workspace serves every max_seq: as many chunks as any length takes.
static int64_t shared_prefix_workspace(int64_t batch, int64_t q_len, int64_t hq, int64_t hkv, int64_t prefix_len) {
  return sp_plan(batch, q_len, hq, hkv, prefix_len, (int64_t)1 << 30).bytes;
}

template <int MODE>
static int launch_prefix_tc(const CUtensorMap& kp, const CUtensorMap& vp, const CUtensorMap& kc, const CUtensorMap& vc,
                            const SpParams& p, dim3 grid, cudaStream_t stream) {
  static bool configured[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    cudaError_t e = cudaFuncSetAttribute(prefix_tc_kernel<MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, sp_smem(MODE));
    // All of the SM's memory as shared memory, or the strips' kernel does not fit beside this one.
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(prefix_tc_kernel<MODE>, cudaFuncAttributePreferredSharedMemoryCarveout,
                               cudaSharedmemCarveoutMaxShared);
    if (e != cudaSuccess) return set_error(LS_ERR_CUDA, "shared_prefix_attention attribute: %s", cudaGetErrorString(e));
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(sp_threads(MODE));
  cfg.dynamicSmemBytes = sp_smem(MODE);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, prefix_tc_kernel<MODE>, kp, vp, kc, vc, p);
  return e == cudaSuccess ? LS_OK : set_error(LS_ERR_CUDA, "shared_prefix_attention launch: %s", cudaGetErrorString(e));
}

static int launch_shared_prefix_attention(const void* q, const void* k_prefix, const void* v_prefix, int64_t prefix_len,
                                          int64_t prefix_cap, const void* k_cache, const void* v_cache,
                                          const int32_t* cache_pos, int64_t uniform_past, int64_t batch, int64_t q_len,
                                          int64_t hq, int64_t hkv, int64_t max_seq, float scale, void* out,
                                          void* workspace, cudaStream_t stream) {
  const SpPlan pl = sp_plan(batch, q_len, hq, hkv, prefix_len, max_seq);
  SpParams p = {};
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.cache_pos = cache_pos;
  p.uniform_past = (int)uniform_past;
  p.part_ml = static_cast<float2*>(workspace);
  p.part_o = reinterpret_cast<float*>(static_cast<unsigned char*>(workspace) + pl.ml_bytes);
  p.out = static_cast<__nv_bfloat16*>(out);
  p.err = device_error_ptr();
  p.rows = (int)((pl.mode == kFull ? 1 : batch) * q_len * (hq / hkv));
  p.q_len = (int)q_len;
  p.Hq = (int)hq;
  p.Hkv = (int)hkv;
  p.G = (int)(hq / hkv);
  p.P = (int)prefix_len;
  p.prefix_cap = (int)prefix_cap;
  p.max_seq = (int)max_seq;
  p.splits = pl.splits;
  p.n_part = pl.splits + pl.chunks;
  const float scale_log2 = scale * 1.4426950408889634f;
  p.scale_log2 = scale == 0.f ? 1.f : std::fabs(scale_log2);
  p.q_keep = scale == 0.f ? 0u : 0xffffffffu;
  p.q_flip = scale < 0.f ? 0x80008000u : 0u;
  CUtensorMap kp, vp, kc, vc;
  int rc = LS_OK;
  if (prefix_len > 0 && pl.mode != kFew) {
    rc = make_map(&kp, k_prefix, hkv * prefix_cap, kSpHeadDim, kSpBox);
    if (!rc) rc = make_map(&vp, v_prefix, hkv * prefix_cap, kSpHeadDim, kSpBox);
  }
  if (pl.mode == kFull) {
    if (!rc) rc = make_map(&kc, k_cache, batch * hkv * max_seq, kSpHeadDim, kSpBox);
    if (!rc) rc = make_map(&vc, v_cache, batch * hkv * max_seq, kSpHeadDim, kSpBox);
    if (rc) return rc;
    if (prefix_len == 0) kp = kc, vp = vc;  // no tile of it is read
    return launch_prefix_tc<kFull>(kp, vp, kc, vc, p, dim3((unsigned)pl.row_blocks, (unsigned)hkv, (unsigned)batch),
                                   stream);
  }
  if (rc) return rc;
  if (prefix_len > 0 && pl.mode != kFew) {
    const dim3 grid((unsigned)pl.splits, (unsigned)pl.row_blocks, (unsigned)hkv);
    rc = pl.mode == kKeys ? launch_prefix_tc<kKeys>(kp, vp, kp, vp, p, grid, stream)
                          : launch_prefix_tc<kRows>(kp, vp, kp, vp, p, grid, stream);
    if (rc) return rc;
  }
  StParams st = {};
  st.q = p.q;
  st.k_cache = static_cast<const __nv_bfloat16*>(k_cache);
  st.v_cache = static_cast<const __nv_bfloat16*>(v_cache);
  st.cache_pos = cache_pos;
  st.uniform_past = p.uniform_past;
  st.part_o = p.part_o;
  st.part_ml = p.part_ml;
  st.err = p.err;
  st.q_len = p.q_len;
  st.Hq = p.Hq;
  st.Hkv = p.Hkv;
  st.G = p.G;
  st.R = p.q_len * p.G;
  const bool few = pl.mode == kFew && prefix_len > 0;
  st.RG = (st.R + 15) / 16;
  st.k_prefix = static_cast<const __nv_bfloat16*>(k_prefix);
  st.v_prefix = static_cast<const __nv_bfloat16*>(v_prefix);
  st.batch = (int)batch;
  st.P = p.P;
  st.prefix_cap = p.prefix_cap;
  st.own = pl.chunks;
  st.behind = prefix_len > 0 && !few;
  st.max_seq = p.max_seq;
  st.n_pre = pl.splits;
  st.n_part = p.n_part;
  st.scale_log2 = scale_log2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(few && pl.splits > pl.chunks ? pl.splits : pl.chunks), (unsigned)(hkv * st.RG),
                     (unsigned)(few ? batch + 1 : batch));
  cfg.blockDim = dim3(32);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, strip_groups_kernel, st);
  if (e == cudaSuccess) {
    cfg.gridDim = dim3((unsigned)((2 * (int64_t)p.rows + kSpJoinWarps - 1) / kSpJoinWarps), (unsigned)hkv);
    cfg.blockDim = dim3(kSpJoinWarps * 32);
    e = cudaLaunchKernelEx(&cfg, prefix_join_kernel, (const float*)p.part_o, (const float2*)p.part_ml, p.n_part, p.rows,
                           p.G, p.Hq, p.out);
  }
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
  *bytes = shared_prefix_workspace(batch, q_len, num_heads, num_kv_heads, prefix_len);
  return LS_OK;
}

int ls_shared_prefix_attention_launches(int64_t batch, int64_t q_len, int64_t num_heads, int64_t num_kv_heads,
                                        int64_t head_dim, int64_t prefix_len, int64_t* launches) {
  LS_REQUIRE(launches, LS_ERR_INVALID_ARGUMENT, "ls_shared_prefix_attention_launches: launches is null");
  int64_t bytes = 0;
  const int rc = ls_shared_prefix_attention_workspace_bytes(batch, q_len, num_heads, num_kv_heads, head_dim, prefix_len,
                                                            &bytes);
  if (rc) return rc;
  const int mode = sp_plan(batch, q_len, num_heads, num_kv_heads, prefix_len, 1).mode;  // (for any max_seq)
  *launches = mode == kFull ? 1 : prefix_len > 0 && mode != kFew ? 3 : 2;
  return LS_OK;
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
  LS_REQUIRE(max_seq > 0 && max_seq < (1ll << 30), LS_ERR_INVALID_ARGUMENT, "ls_shared_prefix_attention: bad sizes");
  LS_REQUIRE(num_kv_heads * ((q_len * (num_heads / num_kv_heads) + 15) / 16) <= 65535, LS_ERR_UNSUPPORTED_SHAPE,
             "ls_shared_prefix_attention: %lld query rows per kv head exceed the grid",
             (long long)(q_len * (num_heads / num_kv_heads)));
  LS_REQUIRE(batch * num_kv_heads * max_seq < (1ll << 31) - 256 && num_kv_heads * prefix_cap < (1ll << 31) - 256 &&
                 batch * q_len * num_heads < (1ll << 31) - 256,
             LS_ERR_UNSUPPORTED_SHAPE, "ls_shared_prefix_attention: %lld x %lld strips of %lld or %lld positions, %lld rows",
             (long long)batch, (long long)num_kv_heads, (long long)max_seq, (long long)prefix_cap,
             (long long)(batch * q_len * num_heads));
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
