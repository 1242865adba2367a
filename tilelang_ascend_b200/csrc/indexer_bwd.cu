// Backward of the lightning indexer's scores at listed keys (sm_100a, tcgen05; 128 dims, at most 64 heads):
//
//   score_j = sum_h w_h relu(z_jh),  z_jh = q_h . k_j         for the listed keys j of a query, with gradients g_j
//   dw_h = sum_j g_j relu(z_jh),     dz_jh = g_j w_h [z_jh > 0],    dq_h = sum_j dz_jh k_j,    dk_j += sum_h dz_jh q_h
//
// One CTA per query, two per SM.  Per tile of 128 listed keys (gathered rows of 256 bytes, K-major chunks in the 128-byte swizzle):
//   Z   [128 keys x 64 heads]   A = keys, B = the query's heads               (contraction over 128 dims)
//   dZ  to shared memory in the inputs' type: 128 rows of 64 heads; dw stays in the workers' registers, in fp32
//   dQ^T[128 dims x 64 heads]  += A = the same keys read MN-major, B = dZ read MN-major     (over 128 keys, stays in tensor memory)
//   dK^T[128 dims x 128 keys]   = A = the heads read MN-major, B = dZ read K-major          (over 64 heads)
// dK^T has a dim per lane, so a warp adds 32 consecutive dims of a key to the fp32 gradient with one 128-byte request.
// dz is rounded to the inputs' type (a tensor-core operand); its magnitude is that of the gradient, so fp16 takes it times a power
// of two that brings the largest of a query's list near 1.  Sums are fp32.
#include <type_traits>

#include "fwd_common.cuh"
#include "indexer_bwd.h"
#include "launch_util.h"

namespace dsa {

namespace ib {
constexpr int kD = 128, kKeys = 128, kHeads = 64;
constexpr uint32_t kQChunk = kHeads * 128, kQBytes = 2 * kQChunk;     // two chunks of 64 dims
constexpr uint32_t kKChunk = kKeys * 128, kKBytes = 2 * kKChunk;
constexpr uint32_t kDzBytes = kKeys * 128;
constexpr int kStages = 2;
constexpr int kMaxWords = 8192 / 32;
constexpr int kWorkers = 8, kGatherWarp = 8, kMmaWarp = 12, kThreads = 13 * 32;
constexpr uint32_t kOffK = kQBytes, kOffDz = kOffK + kStages * kKBytes;
constexpr uint32_t kOffBar = kOffDz + kDzBytes;
constexpr uint32_t kOffW = kOffBar + 128;                             // 64 weights
constexpr uint32_t kOffRow = kOffW + kHeads * 4;                      // rows of dk of the keys of two tiles, -1: none
constexpr uint32_t kOffDw = kOffRow + 2 * kKeys * 4;                  // four partial sums of 64 heads
constexpr uint32_t kOffBits = kOffDw + 4 * kHeads * 4;
constexpr uint32_t kSmemBytes = kOffBits + kMaxWords * 4;
constexpr uint32_t kColZ = 0, kColDq = 64, kColDk = 128, kTmemCols = 256;
static_assert(2 * (kSmemBytes + 1024) <= 233472, "two CTAs per SM");
}  // namespace ib

template <bool kBF16>
__global__ void __launch_bounds__(ib::kThreads, 2) indexer_bwd_kernel(const __grid_constant__ IndexerBwdParams p) {
  using namespace ib;
  using T = typename std::conditional<kBF16, __nv_bfloat16, __half>::type;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t sQ = smem_u32(smem);
  if (sQ & 1023u) {
    if (threadIdx.x == 0) atomicCAS(p.status, kStatusOk, kStatusBadLayout);
    return;
  }
  const uint32_t sK = sQ + kOffK, sDz = sQ + kOffDz;
  uint64_t* k_full = reinterpret_cast<uint64_t*>(smem + kOffBar);   // [2] count 4: the gather warps' copies have landed
  uint64_t* k_empty = k_full + 2;    // [2] count 1: commit after the MMAs that read the stage
  uint64_t* z_full = k_full + 4;     // count 1: commit after Z
  uint64_t* z_free = k_full + 5;     // count 8: the workers have read Z
  uint64_t* dz_full = k_full + 6;    // count 8: dZ is in shared memory
  uint64_t* dz_free = k_full + 7;    // count 1: commit after the MMAs that read dZ
  uint64_t* dk_full = k_full + 8;    // count 1: commit after dK^T
  uint64_t* dk_free = k_full + 9;    // count 8: the workers have read dK^T
  uint64_t* q_full = k_full + 10;    // count 256: the query's heads have landed
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(k_full + 11);
  int* start_status = reinterpret_cast<int*>(k_full + 12);
  float* s_w = reinterpret_cast<float*>(smem + kOffW);
  int* s_row = reinterpret_cast<int*>(smem + kOffRow);
  float* s_dw = reinterpret_cast<float*>(smem + kOffDw);
  uint32_t* s_bits = reinterpret_cast<uint32_t*>(smem + kOffBits);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int bt = p.B * p.S1 - 1 - static_cast<int>(blockIdx.x), b = bt / p.S1;
  const int tiles = (p.K + kKeys - 1) / kKeys;
  const int32_t* idx_row = p.indices + static_cast<int64_t>(bt) * p.K;
  const float* g_row = p.grad + static_cast<int64_t>(bt) * p.K;

  if (tid == 0) {
    *start_status = *reinterpret_cast<volatile int*>(p.status);
    for (int i = 0; i < kStages; ++i) { mbar_init(&k_full[i], 4); mbar_init(&k_empty[i], 1); }
    mbar_init(z_full, 1); mbar_init(z_free, kWorkers); mbar_init(dz_full, kWorkers); mbar_init(dz_free, 1);
    mbar_init(dk_full, 1); mbar_init(dk_free, kWorkers); mbar_init(q_full, kWorkers * 32);
    mbar_init_fence();
  }
  if (tid < kHeads) s_w[tid] = tid < p.N1 ? p.w[static_cast<int64_t>(bt) * p.N1 + tid] : 0.f;
  float top = 0.f;   // largest |g| of this thread's entries
  for (int w = warp; w < 4 * tiles; w += kThreads / 32) {
    const int j = w * 32 + lane, idx = j < p.K ? __ldg(idx_row + j) : -1;
    const bool valid = idx >= 0 && idx < p.S2;
    const uint32_t bits = __ballot_sync(0xffffffffu, valid);
    if (lane == 0) s_bits[w] = bits;
    if (!kBF16 && valid) top = fmaxf(top, fabsf(__ldg(g_row + j)));
  }
  if (warp == kMmaWarp) { tmem_alloc(tmem_slot, kTmemCols); tmem_relinquish(); }
  float scale = 1.f, unscale = 1.f;
  if (!kBF16) {
    // 2^-e with 2^e the exponent of max|g| max|w|: dz keeps fp16's range from the largest of the list downwards (what falls below
    // 2^-24 of it is lost, as it is below fp32's last place of the sums)
    uint32_t* s_top = reinterpret_cast<uint32_t*>(s_dw);
    if (tid < 2) s_top[tid] = 0u;
    __syncthreads();
    atomicMax(&s_top[0], __float_as_uint(top));   // (non-negative floats order like their bits)
    if (tid < kHeads) atomicMax(&s_top[1], __float_as_uint(fabsf(s_w[tid])));
    __syncthreads();
    const float most = __uint_as_float(s_top[0]), most_w = __uint_as_float(s_top[1]);
    int eg = 0, ew = 0;
    if (most > 0.f && most < INFINITY) eg = ilogbf(most);
    if (most_w > 0.f && most_w < INFINITY) ew = ilogbf(most_w);
    const int e = max(-120, min(120, eg + ew));
    scale = ldexpf(1.f, -e);
    unscale = ldexpf(1.f, e);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const bool run = *start_status == kStatusOk;
  auto any_key = [&](int tile) { return (s_bits[4 * tile] | s_bits[4 * tile + 1] | s_bits[4 * tile + 2] | s_bits[4 * tile + 3]) != 0u; };
  auto next_tile = [&](int tile) {
    while (tile < tiles && !any_key(tile)) ++tile;
    return tile;
  };

  if (warp >= kGatherWarp && warp < kMmaWarp) {
    // ================================ gather: 32 keys of every tile per warp ========================
    const int key0 = (warp - kGatherWarp) * 32 + (lane >> 3), unit = lane & 7;   // keys key0 + 4 i, one 16-byte unit of both chunks
    const T* kbase = reinterpret_cast<const T*>(p.k) + static_cast<int64_t>(b) * p.S2 * kD;
    int g = 0;
    bool ok = run;
    for (int tile = next_tile(0); ok && tile < tiles; tile = next_tile(tile + 1), ++g) {
      const int s = g % kStages;
      int idx[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int slot = tile * kKeys + key0 + 4 * i;
        idx[i] = ((s_bits[slot >> 5] >> (slot & 31)) & 1u) ? __ldg(idx_row + slot) : -1;
      }
      if (g >= kStages && !__all_sync(0xffffffffu, mbar_wait(&k_empty[s], ((g / kStages) + 1) & 1, p.status))) { ok = false; break; }
      const uint32_t dst = sK + s * kKBytes;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const T* src = kbase + static_cast<int64_t>(idx[i] < 0 ? 0 : idx[i]) * kD + unit * 8;
        cp_async16(dst + sw128_offset(key0 + 4 * i, unit), src, idx[i] < 0 ? 0u : 16u);
        cp_async16(dst + kKChunk + sw128_offset(key0 + 4 * i, unit), src + 64, idx[i] < 0 ? 0u : 16u);
      }
      cp_async_commit();
      // a warp announces a tile once, when its copies have landed (128 threads arriving by themselves hold the barrier up)
      cp_async_wait<0>();
      __syncwarp();
      if (lane == 0) mbar_arrive(&k_full[s]);
    }
  } else if (warp == kMmaWarp) {
    // ================================ MMA issuer (converged, one elected lane issues) ===============
    constexpr uint32_t id_z = make_idesc_f16(kBF16, kKeys, kHeads, 0, 0);
    constexpr uint32_t id_dq = make_idesc_f16(kBF16, kD, kHeads, 1, 1);
    constexpr uint32_t id_dk = make_idesc_f16(kBF16, kD, kKeys, 1, 0);
    const uint32_t go = elect_one_lane();
    bool ok = run;
    int tile = next_tile(0);
    if (ok && tile < tiles) ok = __all_sync(0xffffffffu, mbar_wait(q_full, 0, p.status));
    // Z of tile number g (its keys are in stage g % 2)
    auto issue_z = [&](int g) {
      const int s = g % kStages;
      if (!__all_sync(0xffffffffu, mbar_wait(&k_full[s], (g / kStages) & 1, p.status))) return false;
      if (g >= 1 && !__all_sync(0xffffffffu, mbar_wait(z_free, (g + 1) & 1, p.status))) return false;
      fence_proxy_async_smem();   // keys and heads were written by cp.async of other threads
      tc_fence_after();
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const uint64_t da = make_smem_desc(sK + s * kKBytes + c * kKChunk, 16, 1024, kSwizzle128B);
        const uint64_t db = make_smem_desc(sQ + c * kQChunk, 16, 1024, kSwizzle128B);
#pragma unroll
        for (int k = 0; k < 4; ++k) umma_ss_if(go, tmem_base + kColZ, da + 2 * k, db + 2 * k, id_z, (c | k) != 0);
      }
      umma_commit_if(go, z_full);
      return true;
    };
    if (ok && tile < tiles) ok = issue_z(0);
    int g = 0;
    while (ok && tile < tiles) {
      const int s = g % kStages, after = next_tile(tile + 1);
      if (after < tiles && !issue_z(g + 1)) { ok = false; break; }   // the next tile's Z while the workers are at this one's
      if (!__all_sync(0xffffffffu, mbar_wait(dz_full, g & 1, p.status))) { ok = false; break; }
      if (g >= 1 && !__all_sync(0xffffffffu, mbar_wait(dk_free, (g + 1) & 1, p.status))) { ok = false; break; }
      fence_proxy_async_smem();
      tc_fence_after();
      const uint64_t dz_k = make_smem_desc(sDz, 16, 1024, kSwizzle128B);              // K-major: contraction over heads
      const uint64_t q_mn = make_smem_desc(sQ, kQChunk, 1024, kSwizzle128B);          // rows are heads, two chunks of 64 dims
      const uint64_t k_mn = make_smem_desc(sK + s * kKBytes, kKChunk, 1024, kSwizzle128B);
      const uint64_t dz_mn = make_smem_desc(sDz, kDzBytes, 1024, kSwizzle128B);       // rows are keys, one chunk of 64 heads
#pragma unroll
      for (int k = 0; k < kHeads / 16; ++k) umma_ss_if(go, tmem_base + kColDk, q_mn + k * (2048 >> 4), dz_k + 2 * k, id_dk, k != 0);
      umma_commit_if(go, dk_full);
#pragma unroll
      for (int k = 0; k < kKeys / 16; ++k) umma_ss_if(go, tmem_base + kColDq, k_mn + k * (2048 >> 4), dz_mn + k * (2048 >> 4), id_dq, (g | k) != 0);
      umma_commit_if(go, &k_empty[s]);
      umma_commit_if(go, dz_free);
      tile = after;
      ++g;
    }
  } else {
    // ================================ workers =======================================================
    // warp = (lane quarter of tensor memory, half of the columns): key 32 quarter + lane and heads 32 half .. + 31 of Z; dims
    // 32 quarter + lane and keys 64 half .. + 63 of dK^T; the same dims and heads of dQ^T.
    const int quarter = warp & 3, half = warp >> 2, key = quarter * 32 + lane;
    const uint32_t lane_base = static_cast<uint32_t>(quarter * 32) << 16;
    const T* q = reinterpret_cast<const T*>(p.q) + static_cast<int64_t>(bt) * p.N1 * kD;
    for (int i = tid; i < kHeads * 16; i += kWorkers * 32) {
      const int h = i >> 4, unit = i & 15;
      const bool copy = h < p.N1;
      cp_async16(sQ + (unit >> 3) * kQChunk + sw128_offset(h, unit & 7), copy ? q + h * kD + unit * 8 : q, copy ? 16u : 0u);
    }
    cp_async_arrive_noinc(q_full);
    float dw[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) dw[i] = 0.f;
    float* dk = p.d_k + static_cast<int64_t>(b) * p.S2 * kD + quarter * 32 + lane;
    auto add_keys = [&](int g) {   // dK^T of tile number g to global memory
      if (!__all_sync(0xffffffffu, mbar_wait(dk_full, g & 1, p.status))) return false;
      tc_fence_after();
      const int4* rows = reinterpret_cast<const int4*>(s_row + (g & 1) * kKeys + half * 64);
#pragma unroll
      for (int c0 = 0; c0 < 64; c0 += 16) {
        uint32_t v[16];
        tmem_ld16(tmem_base + kColDk + half * 64 + c0 + lane_base, v);
        tmem_wait_ld();
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int4 r = rows[c0 / 4 + j];
          const int row[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (row[i] >= 0) atomicAdd(dk + static_cast<int64_t>(row[i]) * kD, __uint_as_float(v[4 * j + i]) * unscale);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(dk_free);
      return true;
    };
    // dZ of tile number g, and its part of dw
    auto score_keys = [&](int tile, int g) {
      const int slot = tile * kKeys + key;
      const bool valid = (s_bits[slot >> 5] >> (slot & 31)) & 1u;
      const float gr = valid ? __ldg(g_row + slot) : 0.f, gs = gr * scale;
      if (half == 0) s_row[(g & 1) * kKeys + key] = valid ? __ldg(idx_row + slot) : -1;
      if (!__all_sync(0xffffffffu, mbar_wait(z_full, g & 1, p.status))) return false;
      if (g >= 1 && !__all_sync(0xffffffffu, mbar_wait(dz_free, (g + 1) & 1, p.status))) return false;
      tc_fence_after();
#pragma unroll
      for (int c0 = 0; c0 < 32; c0 += 16) {
        uint32_t v[16], w[8];
        tmem_ld16(tmem_base + kColZ + half * 32 + c0 + lane_base, v);
        tmem_wait_ld();
        const float4* w4 = reinterpret_cast<const float4*>(s_w + half * 32 + c0);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float4 wt = w4[j];
          float z[4], d[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            z[i] = __uint_as_float(v[4 * j + i]);
            dw[c0 + 4 * j + i] = fmaf(gr, fmaxf(z[i], 0.f), dw[c0 + 4 * j + i]);
          }
          d[0] = z[0] > 0.f ? gs * wt.x : 0.f;
          d[1] = z[1] > 0.f ? gs * wt.y : 0.f;
          d[2] = z[2] > 0.f ? gs * wt.z : 0.f;
          d[3] = z[3] > 0.f ? gs * wt.w : 0.f;
          w[2 * j] = pack2<kBF16>(d[0], d[1]);
          w[2 * j + 1] = pack2<kBF16>(d[2], d[3]);
        }
        const int unit = half * 4 + c0 / 8;
        st_shared_v4(sDz + sw128_offset(key, unit), w[0], w[1], w[2], w[3]);
        st_shared_v4(sDz + sw128_offset(key, unit + 1), w[4], w[5], w[6], w[7]);
      }
      tc_fence_before();
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(z_free);
        mbar_arrive(dz_full);
      }
      return true;
    };
    int g = 0;
    bool ok = run;
    for (int tile = next_tile(0); tile < tiles; tile = next_tile(tile + 1), ++g) {
      ok = ok && score_keys(tile, g);
      ok = ok && (g == 0 || add_keys(g - 1));
      // s_row of the tile before has been read, this tile's is complete (every worker comes here for every tile, also when a wait
      // has given up)
      named_bar_sync(1, kWorkers * 32);
    }
    if (ok && g > 0) ok = add_keys(g - 1);
    // ---- dQ: complete with the last tile (dz_free comes after its MMAs) ----------------------------
    T* dq = reinterpret_cast<T*>(p.d_q) + static_cast<int64_t>(bt) * p.N1 * kD + quarter * 32 + lane;
    if (ok && g > 0) ok = __all_sync(0xffffffffu, mbar_wait(dz_free, (g + 1) & 1, p.status));
    if (ok) {
      tc_fence_after();
#pragma unroll
      for (int c0 = 0; c0 < 32; c0 += 16) {
        uint32_t v[16];
        if (g > 0) {
          tmem_ld16(tmem_base + kColDq + half * 32 + c0 + lane_base, v);
          tmem_wait_ld();
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int h = half * 32 + c0 + i;
          if (h < p.N1) dq[h * kD] = static_cast<T>(g > 0 ? __uint_as_float(v[i]) * unscale : 0.f);
        }
      }
      // ---- dw: over the lanes (lane l ends with head 32 half + l), then over the four quarters -----
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const bool upper = lane & o;
#pragma unroll
        for (int i = 0; i < o; ++i) {
          const float give = upper ? dw[i] : dw[i + o], mine = upper ? dw[i + o] : dw[i];
          dw[i] = mine + __shfl_xor_sync(0xffffffffu, give, o);
        }
      }
      s_dw[quarter * kHeads + half * 32 + lane] = dw[0];
    }
    named_bar_sync(1, kWorkers * 32);
    if (ok && tid < p.N1)
      p.d_w[static_cast<int64_t>(bt) * p.N1 + tid] = (s_dw[tid] + s_dw[kHeads + tid]) + (s_dw[2 * kHeads + tid] + s_dw[3 * kHeads + tid]);
    cp_async_wait<0>();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) tmem_dealloc(tmem_base, kTmemCols);
}

bool indexer_bwd_supported(const IndexerBwdParams& p) { return p.D == ib::kD && p.N1 <= ib::kHeads && p.K <= ib::kMaxWords * 32; }

int launch_indexer_bwd(const IndexerBwdParams& p, bool bf16, cudaStream_t stream) {
  int dev = 0, sms = 0;
  cudaError_t e = current_device_sms(&dev, &sms);
  if (e != cudaSuccess) return static_cast<int>(e);
  auto kern = bf16 ? indexer_bwd_kernel<true> : indexer_bwd_kernel<false>;
  if ((e = ensure_dynamic_smem(kern, dev, static_cast<int>(ib::kSmemBytes))) != cudaSuccess) return static_cast<int>(e);
  kern<<<static_cast<unsigned>(p.B) * p.S1, ib::kThreads, ib::kSmemBytes, stream>>>(p);
  return static_cast<int>(cudaGetLastError());
}

}  // namespace dsa
