// Attention weights of the listed keys, averaged over the heads (sm_100a, tcgen05):
//
//   w[b, t, j] = 1/H sum_h exp(sm_scale q[b, t, h] . kv[b, idx_j] - lse[b, t, h])        0 for entries that take no part
//
// what the sparse MLA forward's softmax gives each key of a query's list; the forward keeps only its normaliser (lse).
//
// Bound by the tensor cores on paper (2 H D operations against 2 D gathered bytes per key).  The MMA is issued transposed:
// A = 128 gathered keys x 64 dims at a time (UMMA M = keys), B = up to 128 heads of the query, so that the accumulator holds a
// key per lane and the sum over heads is each thread's own, without exchange; 128 exponentials per key cost half of its MMA time.
// The query's heads stay in shared memory, the keys pass through a ring of chunks of [128 keys x 64 dims].  One CTA per query,
// long (late) queries first; more than 128 heads take further passes over the list.
#include <type_traits>

#include "fwd_common.cuh"
#include "launch_util.h"

namespace dsa {

namespace kw {
constexpr int kKeys = 128;                        // keys per tile = UMMA M
constexpr int kHeads = 128;                       // heads per pass, at most (UMMA N = the next multiple of 16)
constexpr uint32_t kChunkBytes = kKeys * 128;     // 128 keys x 64 dims
constexpr int kMaxStages = 12;
constexpr int kMaxWords = 8192 / 32;              // validity bits of a list
constexpr int kGatherWarps = 8, kMmaWarp = 12, kThreads = 13 * 32;   // warps 0-3: query rows, then epilogue
constexpr uint32_t kFixedBytes = 256 + kHeads * 4 + kMaxWords * 4;   // barriers, lse, bits
constexpr uint32_t kMaxSmem = 232448;
constexpr uint32_t kTmemCols = 2 * kHeads;        // two accumulators
struct Shape {
  int chunks, n, stages;                          // 64-dim chunks of a row; UMMA N; stages of the ring
};
}  // namespace kw

template <bool kBF16>
__global__ void __launch_bounds__(kw::kThreads, 1)
    sparse_mla_key_weights_kernel(const __grid_constant__ FwdParams p, float* __restrict__ weights, const kw::Shape sh) {
  using namespace kw;
  using T = typename std::conditional<kBF16, __nv_bfloat16, __half>::type;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t sQ = smem_u32(smem);
  if (sQ & 1023u) {
    if (threadIdx.x == 0) atomicCAS(p.status, kStatusOk, kStatusBadLayout);
    return;
  }
  const uint32_t q_chunk = static_cast<uint32_t>(sh.n) * 128;      // one chunk of the query's heads
  const uint32_t sK = sQ + sh.chunks * q_chunk;
  uint8_t* fixed = smem + sh.chunks * q_chunk + sh.stages * kChunkBytes;
  uint64_t* k_full = reinterpret_cast<uint64_t*>(fixed);   // [kMaxStages] count 256: the gather threads' copies have landed
  uint64_t* k_empty = k_full + kMaxStages;                 // [kMaxStages] count 1: commit after the MMAs that read the stage
  uint64_t* acc_full = k_empty + kMaxStages;               // [2] count 1: commit after a tile's last MMA
  uint64_t* acc_empty = acc_full + 2;                      // [2] count 128
  uint64_t* q_full = acc_empty + 2;                        // count 128: this pass's heads have landed
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(q_full + 1);
  int* start_status = reinterpret_cast<int*>(tmem_slot + 1);
  float* s_lse = reinterpret_cast<float*>(fixed + 256);    // in log2 units; +inf: no weight
  uint32_t* s_bits = reinterpret_cast<uint32_t*>(fixed + 256 + kHeads * 4);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int bt = p.B * p.S - 1 - static_cast<int>(blockIdx.x);
  const RowCtx c = make_row_ctx(p, bt);
  const int words = (p.topk + 31) >> 5, tiles = (p.topk + kKeys - 1) / kKeys;
  float* out = weights + static_cast<int64_t>(bt) * p.topk;

  if (tid == 0) {
    *start_status = *reinterpret_cast<volatile int*>(p.status);
    for (int i = 0; i < sh.stages; ++i) { mbar_init(&k_full[i], kGatherWarps * 32); mbar_init(&k_empty[i], 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(&acc_full[i], 1); mbar_init(&acc_empty[i], 128); }
    mbar_init(q_full, 128);
    mbar_init_fence();
  }
  for (int w = warp; w < 4 * tiles; w += kThreads / 32) {
    const int j = w * 32 + lane;
    const bool valid = w < words && j < p.topk && c.active && index_valid(c, __ldg(c.idx_row + j));
    const uint32_t bits = __ballot_sync(0xffffffffu, valid);
    if (lane == 0) s_bits[w] = bits;
  }
  if (warp == kMmaWarp) { tmem_alloc(tmem_slot, kTmemCols); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const bool run = *start_status == kStatusOk;
  const int passes = (p.H + kHeads - 1) / kHeads;
  auto any_key = [&](int tile) { return (s_bits[4 * tile] | s_bits[4 * tile + 1] | s_bits[4 * tile + 2] | s_bits[4 * tile + 3]) != 0u; };

  if (warp >= 4 && warp < kMmaWarp) {
    // ================================ gather: 16 keys of every chunk per warp =======================
    const int key0 = (warp - 4) * 16 + (lane >> 3), unit = lane & 7;   // this thread's keys: key0 + 4 i, one 16-byte unit of each
    const T* kv = reinterpret_cast<const T*>(p.kv) + static_cast<int64_t>(c.b) * p.S_kv * p.D;
    int stage = 0;
    uint32_t phase = 1;   // (the first round of the ring finds its stages empty)
    bool ok = run;
    for (int pass = 0; ok && pass < passes; ++pass)
      for (int tile = 0; ok && tile < tiles; ++tile) {
        if (!any_key(tile)) continue;
        const T* src[4];
        uint32_t there = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = key0 + 4 * i, slot = tile * kKeys + key;
          const bool valid = (s_bits[slot >> 5] >> (slot & 31)) & 1u;
          const int idx = valid ? __ldg(c.idx_row + slot) : 0;
          src[i] = kv + static_cast<int64_t>(idx) * p.D + unit * 8;
          there |= valid ? 1u << i : 0u;
        }
        for (int ch = 0; ch < sh.chunks; ++ch) {
          if (!__all_sync(0xffffffffu, mbar_wait(&k_empty[stage], phase, p.status))) { ok = false; break; }
          const bool dims = ch * 64 + unit * 8 < p.D;
          const uint32_t dst = sK + stage * kChunkBytes;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const bool copy = dims && ((there >> i) & 1u);
            cp_async16(dst + sw128_offset(key0 + 4 * i, unit), copy ? src[i] + ch * 64 : reinterpret_cast<const T*>(p.kv), copy ? 16u : 0u);
          }
          cp_async_arrive_noinc(&k_full[stage]);
          if (++stage == sh.stages) { stage = 0; phase ^= 1u; }
        }
      }
    cp_async_wait<0>();
  } else if (warp == kMmaWarp) {
    // ================================ MMA issuer (converged, one elected lane issues) ===============
    const uint32_t idesc = make_idesc_f16(kBF16, kKeys, sh.n, 0, 0), go = elect_one_lane();
    int stage = 0, g = 0;
    uint32_t phase = 0;
    bool ok = run;
    for (int pass = 0; ok && pass < passes; ++pass) {
      bool first = true;
      for (int tile = 0; ok && tile < tiles; ++tile) {
        if (!any_key(tile)) continue;
        if (first) {
          if (!__all_sync(0xffffffffu, mbar_wait(q_full, pass & 1, p.status))) { ok = false; break; }
          first = false;
        }
        const int a = g & 1;
        if (g >= 2 && !__all_sync(0xffffffffu, mbar_wait(&acc_empty[a], ((g >> 1) + 1) & 1, p.status))) { ok = false; break; }
        for (int ch = 0; ch < sh.chunks; ++ch) {
          if (!__all_sync(0xffffffffu, mbar_wait(&k_full[stage], phase, p.status))) { ok = false; break; }
          fence_proxy_async_smem();   // the rows were written by cp.async of other threads
          tc_fence_after();
          const uint64_t da = make_smem_desc(sK + stage * kChunkBytes, 16, 1024, kSwizzle128B);
          const uint64_t db = make_smem_desc(sQ + ch * q_chunk, 16, 1024, kSwizzle128B);
#pragma unroll
          for (int k = 0; k < 4; ++k) umma_ss_if(go, tmem_base + a * kHeads, da + 2 * k, db + 2 * k, idesc, (ch | k) != 0);
          umma_commit_if(go, &k_empty[stage]);
          if (++stage == sh.stages) { stage = 0; phase ^= 1u; }
        }
        if (!ok) break;
        umma_commit_if(go, &acc_full[a]);
        ++g;
      }
    }
  } else {
    // ================================ query rows, then epilogue: thread = key ========================
    const uint32_t lane_base = static_cast<uint32_t>(warp * 32) << 16;
    const float inv_h = 1.f / static_cast<float>(p.H);
    int g = 0;
    bool ok = run;
    for (int pass = 0; pass < passes; ++pass) {   // (also when a wait has given up: the barriers below count every thread)
      const int h0 = pass * kHeads, heads = min(kHeads, p.H - h0);
      // (the last pass's MMAs are done: their accumulators have been read below)
      const T* q = reinterpret_cast<const T*>(p.q) + (static_cast<int64_t>(bt) * p.H + h0) * p.D;
      for (int i = tid; i < sh.chunks * sh.n * 8; i += 128) {
        const int unit = i & 7, row = (i >> 3) % sh.n, ch = (i >> 3) / sh.n;
        const bool copy = row < heads && ch * 64 + unit * 8 < p.D;
        cp_async16(sQ + ch * q_chunk + sw128_offset(row, unit), copy ? q + static_cast<int64_t>(row) * p.D + ch * 64 + unit * 8 : q, copy ? 16u : 0u);
      }
      cp_async_arrive_noinc(q_full);
      named_bar_sync(1, 128);   // the last pass's normalisers have been used
      {
        // a head without any key has lse = -inf: no weight (neither have the rows that pad the heads)
        const float l = tid < heads ? p.lse[static_cast<int64_t>(bt) * p.H + h0 + tid] : INFINITY;
        s_lse[tid] = l == -INFINITY ? INFINITY : l * 1.4426950408889634f;
      }
      named_bar_sync(1, 128);
      for (int tile = 0; ok && tile < tiles; ++tile) {
        const int slot = tile * kKeys + tid;
        float sum = 0.f;
        if (any_key(tile)) {
          const int a = g & 1;
          if (!__all_sync(0xffffffffu, mbar_wait(&acc_full[a], (g >> 1) & 1, p.status))) { ok = false; break; }
          tc_fence_after();
          float part[4] = {0.f, 0.f, 0.f, 0.f};
          for (int c0 = 0; c0 < sh.n; c0 += 16) {
            uint32_t v[16];
            tmem_ld16(tmem_base + a * kHeads + c0 + lane_base, v);
            tmem_wait_ld();
            const float4* l4 = reinterpret_cast<const float4*>(s_lse + c0);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float4 l = l4[j];
              part[0] += exp2f(fmaf(__uint_as_float(v[4 * j]), p.scale_log2, -l.x));
              part[1] += exp2f(fmaf(__uint_as_float(v[4 * j + 1]), p.scale_log2, -l.y));
              part[2] += exp2f(fmaf(__uint_as_float(v[4 * j + 2]), p.scale_log2, -l.z));
              part[3] += exp2f(fmaf(__uint_as_float(v[4 * j + 3]), p.scale_log2, -l.w));
            }
          }
          tc_fence_before();
          mbar_arrive(&acc_empty[a]);
          ++g;
          sum = ((s_bits[slot >> 5] >> (slot & 31)) & 1u) ? ((part[0] + part[1]) + (part[2] + part[3])) * inv_h : 0.f;
        }
        if (slot < p.topk) out[slot] = pass ? out[slot] + sum : sum;
      }
    }
    cp_async_wait<0>();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) tmem_dealloc(tmem_base, kTmemCols);
}

bool sparse_mla_key_weights_supported(const FwdParams& p) { return p.D % 8 == 0 && p.D <= 640 && p.topk <= kw::kMaxWords * 32; }

// p.lse is read; p.out is not used.
int launch_sparse_mla_key_weights(const FwdParams& p, float* weights, bool bf16, cudaStream_t stream) {
  int dev = 0, sms = 0;
  cudaError_t e = current_device_sms(&dev, &sms);
  if (e != cudaSuccess) return static_cast<int>(e);
  kw::Shape sh;
  sh.chunks = (p.D + 63) / 64;
  sh.n = p.H >= kw::kHeads ? kw::kHeads : (p.H + 15) / 16 * 16;
  // as many stages as shared memory holds beside the heads (576 dims: 128 heads 5, 64 heads 9)
  const uint32_t q_bytes = static_cast<uint32_t>(sh.chunks) * sh.n * 128;
  sh.stages = static_cast<int>((kw::kMaxSmem - kw::kFixedBytes - q_bytes) / kw::kChunkBytes);
  if (sh.stages > kw::kMaxStages) sh.stages = kw::kMaxStages;
  const int smem = static_cast<int>(q_bytes + sh.stages * kw::kChunkBytes + kw::kFixedBytes);
  auto kern = bf16 ? sparse_mla_key_weights_kernel<true> : sparse_mla_key_weights_kernel<false>;
  if ((e = ensure_dynamic_smem(kern, dev, smem)) != cudaSuccess) return static_cast<int>(e);
  kern<<<static_cast<unsigned>(p.B) * p.S, kw::kThreads, smem, stream>>>(p, weights, sh);
  return static_cast<int>(cudaGetLastError());
}

}  // namespace dsa
