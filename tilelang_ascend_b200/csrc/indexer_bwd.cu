// Backward of the lightning indexer's scores at listed keys (sm_100a, tcgen05; 128 dims, at most 64 heads):
//
//   score_j = sum_h w_h relu(z_jh),  z_jh = q_h . k_j         for the listed keys j of a query, with gradients g_j
//   dw_h = sum_j g_j relu(z_jh),     dz_jh = g_j w_h [z_jh > 0],    dq_h = sum_j dz_jh k_j,    dk_j += sum_h dz_jh q_h
//
// Persistent CTAs, one per SM, long (late) queries first.  Per tile of 128 listed keys (gathered rows of 256 bytes, K-major chunks in
// the 128-byte swizzle):
//   Z   [128 keys x 64 heads]   A = keys, B = the query's heads               (contraction over 128 dims)
//   dZ  to shared memory in the inputs' type: 128 rows of 64 heads; dw stays in registers, in fp32
//   dQ^T[128 dims x 64 heads]  += A = the same keys read MN-major, B = dZ read MN-major     (over 128 keys, stays in tensor memory)
//   dK^T[128 dims x 128 keys]   = A = the heads read MN-major, B = dZ read K-major          (over 64 heads)
// dK^T has a dim per lane, so a warp adds 32 consecutive dims of a key to the fp32 gradient with one 128-byte request; these additions
// (512 bytes per pair of query and key) are what bounds the kernel.  So everything else is kept out of their way: eight warps do
// nothing else, eight others make dZ, four gather, one issues Z's MMAs and one the sums', one reads the next query's list; Z, dZ, dK^T and
// dQ^T exist twice.  Measured for 4096 queries x 2048 of 4096 keys, 64 heads (3.2 GB of additions): 674 us, 4.8 TB/s; without the additions 478; fp16 698.
// (Two CTAs per SM whose warps made dZ and added in turn spent 8500 clocks on a tile, half of them without an addition on its way: 790 us;
// one warp for all MMAs: 710.)
// dz is rounded to the inputs' type (a tensor-core operand); its magnitude is that of the gradient, so fp16 takes it times a power
// of two that brings the largest of a query's list close under fp16's end.  Sums are fp32.
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
constexpr int kStages = 4;
constexpr int kMaxWords = 8192 / 32, kMaxTiles = 8192 / kKeys;
constexpr int kDzWarps = 8, kAddWarp = 8, kAddWarps = 8, kGatherWarp = 16, kGatherWarps = 4, kZWarp = 20, kMmaWarp = 21, kListWarp = 22, kThreads = 23 * 32;
constexpr int kUsers = kDzWarps + kAddWarps + kGatherWarps + 2;       // warps that read a list
// A query's list: what all roles need to know of it.
struct List {
  int query;                 // b * S1 + s, -1: no more
  int tiles;                 // tiles with a key
  float scale, unscale;      // of a gradient; of the sums
  float w[kHeads];           // scaled too
  uint32_t bits[kMaxWords];  // which entries take part
  uint8_t tile[kMaxTiles];   // the tiles with a key
};
constexpr uint32_t kOffK = 2 * kQBytes, kOffDz = kOffK + kStages * kKBytes;
constexpr uint32_t kOffBar = kOffDz + 2 * kDzBytes;
constexpr uint32_t kOffRow = kOffBar + 256;                           // rows of dk of the 64 keys of each adding warp
constexpr uint32_t kOffDw = kOffRow + kAddWarps * 64 * 4;                  // four partial sums of 64 heads
constexpr uint32_t kOffList = kOffDw + 4 * kHeads * 4;
constexpr uint32_t kSmemBytes = kOffList + 2 * sizeof(List);
constexpr uint32_t kColZ = 0, kColDq = 128, kColDk = 256, kTmemCols = 512;   // two of each: 64, 64 and 128 columns
static_assert(kSmemBytes <= 232448 && sizeof(List) % 16 == 0, "shared memory per CTA");

// A NaN stays one, as in autograd's relu (whose gradient at NaN is that of a positive value).
__device__ __forceinline__ float relu(float z) {
  float r;
  asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(r) : "f"(z));
  return r;
}
}  // namespace ib

template <bool kBF16>
__global__ void __launch_bounds__(ib::kThreads, 1) indexer_bwd_kernel(const __grid_constant__ IndexerBwdParams p) {
  using namespace ib;
  using T = typename std::conditional<kBF16, __nv_bfloat16, __half>::type;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t sQ = smem_u32(smem);
  if (sQ & 1023u) {
    if (threadIdx.x == 0) atomicCAS(p.status, kStatusOk, kStatusBadLayout);
    return;
  }
  const uint32_t sK = sQ + kOffK, sDz = sQ + kOffDz;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kOffBar);
  uint64_t* k_full = bars;           // [4] count 4: the gather warps' copies have landed
  uint64_t* k_empty = bars + 4;      // [4] count 1: commit after the MMAs that read the stage
  uint64_t* z_full = bars + 8;       // [2] count 1: commit after Z
  uint64_t* z_free = bars + 10;      // [2] count 8: Z has been read
  uint64_t* dz_full = bars + 12;     // [2] count 8: dZ is in shared memory
  uint64_t* dz_free = bars + 14;     // [2] count 1: commit after the MMAs that read dZ
  uint64_t* dk_full = bars + 16;     // [2] count 1: commit after dK^T
  uint64_t* dk_free = bars + 18;     // [2] count 8: dK^T has been read
  uint64_t* q_full = bars + 20;      // [2] count 4: the query's heads have landed
  uint64_t* q_done = bars + 22;      // [2] count 1: commit after a query's last MMAs: its heads are free, dQ^T is complete
  uint64_t* dq_free = bars + 24;     // [2] count 8: dQ^T has been read
  uint64_t* list_full = bars + 26;   // [2] count 1
  uint64_t* list_free = bars + 28;   // [2] count kUsers
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 30);
  int* start_status = reinterpret_cast<int*>(bars + 31);
  int* s_row = reinterpret_cast<int*>(smem + kOffRow);
  float* s_dw = reinterpret_cast<float*>(smem + kOffDw);
  List* lists = reinterpret_cast<List*>(smem + kOffList);

  if (p.only_if && *p.only_if == 0) return;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    *start_status = *reinterpret_cast<volatile int*>(p.status);
    for (int i = 0; i < kStages; ++i) { mbar_init(&k_full[i], kGatherWarps); mbar_init(&k_empty[i], 1); }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&z_full[i], 1); mbar_init(&z_free[i], kDzWarps); mbar_init(&dz_full[i], kDzWarps); mbar_init(&dz_free[i], 1);
      mbar_init(&dk_full[i], 1); mbar_init(&dk_free[i], kAddWarps); mbar_init(&q_full[i], kGatherWarps); mbar_init(&q_done[i], 1);
      mbar_init(&dq_free[i], kAddWarps); mbar_init(&list_full[i], 1); mbar_init(&list_free[i], kUsers);
    }
    mbar_init_fence();
  }
  if (warp == kMmaWarp) { tmem_alloc(tmem_slot, kTmemCols); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  bool ok = *start_status == kStatusOk;
  auto wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity, p.status)) != 0; };
  // Item n of this CTA (its n-th query with a key): parity of the n-th use of a pair of barriers, and of the use before it.
  auto use = [](int n) { return static_cast<uint32_t>(n >> 1) & 1u; };
  auto before = [](int n) { return (static_cast<uint32_t>(n >> 1) + 1u) & 1u; };
  auto done_with = [&](int n) {
    __syncwarp();
    if (lane == 0) mbar_arrive(&list_free[n & 1]);
  };

  if (warp == kListWarp) {
    // ================================ lists, one query ahead; queries without keys ==================
    int n = 0;
    for (int i = blockIdx.x; ok && i < p.B * p.S1; i += gridDim.x) {
      const int bt = p.B * p.S1 - 1 - i;
      if (n >= 2 && !wait(&list_free[n & 1], before(n))) { ok = false; break; }
      List& list = lists[n & 1];
      const int32_t* idx_row = p.indices + static_cast<int64_t>(bt) * p.K;
      const float* g_row = p.grad + static_cast<int64_t>(bt) * p.K;
      int tiles = 0;
      float top = 0.f;   // largest finite |g| of this lane's entries
      for (int j0 = 0; j0 < p.K; j0 += 4 * kKeys) {   // four tiles' entries on their way at once
        int idx[16];
        float size[16];   // (fp16)
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          const int j = j0 + 32 * k + lane;
          idx[k] = j < p.K ? __ldg(idx_row + j) : -1;
          if (!kBF16) size[k] = j < p.K ? fabsf(__ldg(g_row + j)) : 0.f;
        }
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          uint32_t any = 0;
#pragma unroll
          for (int k = 4 * t; k < 4 * t + 4; ++k) {
            const bool valid = idx[k] >= 0 && idx[k] < p.S2;
            const uint32_t bits = __ballot_sync(0xffffffffu, valid);
            if (lane == 0 && j0 + 32 * k < kMaxWords * 32) list.bits[j0 / 32 + k] = bits;
            if (!kBF16) top = fmaxf(top, valid && size[k] < INFINITY ? size[k] : 0.f);
            any |= bits;
          }
          if (any) {
            if (lane == 0) list.tile[tiles] = static_cast<uint8_t>(j0 / kKeys + t);
            ++tiles;
          }
        }
      }
      const float* w_row = p.w + static_cast<int64_t>(bt) * p.N1;
      if (!tiles) {
        T* dq = reinterpret_cast<T*>(p.d_q) + static_cast<int64_t>(bt) * p.N1 * kD;
        if ((reinterpret_cast<uintptr_t>(dq) & 15u) == 0) {
          for (int k = lane; k < p.N1 * kD / 8; k += 32) reinterpret_cast<uint4*>(dq)[k] = make_uint4(0, 0, 0, 0);
        } else {   // (d_q may start at any element)
          for (int k = lane; k < p.N1 * kD; k += 32) dq[k] = static_cast<T>(0.f);
        }
        for (int k = lane; k < p.N1; k += 32) p.d_w[static_cast<int64_t>(bt) * p.N1 + k] = 0.f;
        continue;
      }
      float w[2], top_w = 0.f;   // (largest finite |w|)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int h = 32 * k + lane;
        w[k] = h < p.N1 ? __ldg(w_row + h) : 0.f;
        if (fabsf(w[k]) < INFINITY) top_w = fmaxf(top_w, fabsf(w[k]));
      }
      float scale_w = 1.f, scale = 1.f, unscale = 1.f;
      if (!kBF16) {
        // |dz| goes to 2^13 .. 2^15 at most, close under fp16's end: a head's or a key's sum need not hold the largest of the list, so all that lies
        // below it counts.  A dz down to 2^-27 of the list's largest keeps fp16's 11 bits, what is smaller is off by 2^-38 of that largest.
        // Gradients and weights take a power of two each, so that neither product leaves fp32.
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
          top_w = fmaxf(top_w, __shfl_xor_sync(0xffffffffu, top_w, o));
        }
        int eg = 0, ew = 0;
        if (top > 0.f) eg = max(-113, ilogbf(top));
        if (top_w > 0.f) ew = max(-126, min(126, ilogbf(top_w)));
        const int e = max(-126, min(126, eg + ew - 13));
        scale_w = ldexpf(1.f, -ew);
        scale = ldexpf(1.f, ew - e);
        unscale = ldexpf(1.f, e);
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) list.w[32 * k + lane] = w[k] * scale_w;
      __syncwarp();
      if (lane == 0) {
        list.query = bt;
        list.tiles = tiles;
        list.scale = scale;
        list.unscale = unscale;
        mbar_arrive(&list_full[n & 1]);
      }
      __syncwarp();
      ++n;
    }
    if (ok && n >= 2) ok = wait(&list_free[n & 1], before(n));
    if (ok && lane == 0) {
      lists[n & 1].query = -1;
      mbar_arrive(&list_full[n & 1]);
    }
  } else if (warp >= kGatherWarp && warp < kZWarp) {
    // ================================ gather: a quarter of the rows of everything per warp ==========
    const int quarter = warp - kGatherWarp, sub = lane >> 3, unit = lane & 7;   // row sub + 4 i of the quarter, one 16-byte unit of both chunks
    int g = 0;   // tiles so far
    for (int n = 0; ok; ++n) {
      if (!wait(&list_full[n & 1], use(n))) { ok = false; break; }
      const List& list = lists[n & 1];
      const int bt = list.query;
      if (bt < 0) break;
      const int32_t* idx_row = p.indices + static_cast<int64_t>(bt) * p.K;
      const T* kbase = reinterpret_cast<const T*>(p.k) + static_cast<int64_t>(bt / p.S1) * p.S2 * kD + unit * 8;
      const T* q = reinterpret_cast<const T*>(p.q) + static_cast<int64_t>(bt) * p.N1 * kD + unit * 8;
      auto rows_of = [&](int i, int (&row)[8]) {
        const int slot0 = list.tile[i] * kKeys + quarter * 32 + sub;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int slot = slot0 + 4 * k, idx = slot < p.K ? __ldg(idx_row + slot) : -1;
          row[k] = idx < p.S2 ? idx : -1;
        }
      };
      int next[8];
      rows_of(0, next);
      if (n >= 2 && !wait(&q_done[n & 1], before(n))) { ok = false; break; }
      {
        const uint32_t dst = sQ + (n & 1) * kQBytes;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int h = quarter * 16 + 4 * i + sub;
          const T* src = h < p.N1 ? q + h * kD : q;
          cp_async16(dst + sw128_offset(h, unit), src, h < p.N1 ? 16u : 0u);
          cp_async16(dst + kQChunk + sw128_offset(h, unit), src + 64, h < p.N1 ? 16u : 0u);
        }
        cp_async_commit();
        cp_async_wait<0>();
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_full[n & 1]);
      }
      for (int i = 0; ok && i < list.tiles; ++i, ++g) {
        int row[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) row[k] = next[k];
        if (i + 1 < list.tiles) rows_of(i + 1, next);   // one tile ahead of its copies
        const int s = g % kStages;
        if (g >= kStages && !wait(&k_empty[s], ((g / kStages) + 1) & 1)) { ok = false; break; }
        const uint32_t dst = sK + s * kKBytes;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const uint32_t r = quarter * 32 + 4 * k + sub;
          const T* src = kbase + static_cast<int64_t>(row[k] < 0 ? 0 : row[k]) * kD;
          cp_async16(dst + sw128_offset(r, unit), src, row[k] < 0 ? 0u : 16u);
          cp_async16(dst + kKChunk + sw128_offset(r, unit), src + 64, row[k] < 0 ? 0u : 16u);
        }
        cp_async_commit();
        cp_async_wait<0>();
        __syncwarp();
        if (lane == 0) mbar_arrive(&k_full[s]);
      }
      done_with(n);
    }
  } else if (warp == kZWarp) {
    // ================================ MMA issuer of Z (converged, one elected lane issues) ==========
    constexpr uint32_t id_z = make_idesc_f16(kBF16, kKeys, kHeads, 0, 0);
    const uint32_t go = elect_one_lane();
    const uint32_t tmem = __reduce_or_sync(0xffffffffu, tmem_base);   // (known to be the same in all lanes: the MMAs' operands are uniform registers)
    int g = 0;
    for (int n = 0; ok; ++n) {
      if (!wait(&list_full[n & 1], use(n))) { ok = false; break; }
      const int tiles = __reduce_or_sync(0xffffffffu, lists[n & 1].query < 0 ? 0u : static_cast<uint32_t>(lists[n & 1].tiles));
      if (!tiles) break;
      if (!wait(&q_full[n & 1], use(n))) { ok = false; break; }
      for (int i = 0; i < tiles; ++i, ++g) {
        const int s = g % kStages;
        if (!wait(&k_full[s], (g / kStages) & 1)) { ok = false; break; }
        if (g >= 2 && !wait(&z_free[g & 1], before(g))) { ok = false; break; }
        fence_proxy_async_smem();   // keys and heads were written by cp.async of other threads
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const uint64_t da = make_smem_desc(sK + s * kKBytes + c * kKChunk, 16, 1024, kSwizzle128B);
          const uint64_t db = make_smem_desc(sQ + (n & 1) * kQBytes + c * kQChunk, 16, 1024, kSwizzle128B);
#pragma unroll
          for (int k = 0; k < 4; ++k) umma_ss_if(go, tmem + kColZ + (g & 1) * kHeads, da + 2 * k, db + 2 * k, id_z, (c | k) != 0);
        }
        umma_commit_if(go, &z_full[g & 1]);
      }
      if (!ok) break;
      done_with(n);
    }
  } else if (warp == kMmaWarp) {
    // ================================ MMA issuer of dK^T and dQ^T ===================================
    constexpr uint32_t id_dq = make_idesc_f16(kBF16, kD, kHeads, 1, 1);
    constexpr uint32_t id_dk = make_idesc_f16(kBF16, kD, kKeys, 1, 0);
    const uint32_t go = elect_one_lane();
    const uint32_t tmem = __reduce_or_sync(0xffffffffu, tmem_base);
    int g = 0;
    for (int n = 0; ok; ++n) {
      if (!wait(&list_full[n & 1], use(n))) { ok = false; break; }
      const int tiles = __reduce_or_sync(0xffffffffu, lists[n & 1].query < 0 ? 0u : static_cast<uint32_t>(lists[n & 1].tiles));
      if (!tiles) break;
      if (n >= 2 && !wait(&dq_free[n & 1], before(n))) { ok = false; break; }
      for (int i = 0; i < tiles; ++i, ++g) {
        const int s = g % kStages;
        if (g >= 2 && !wait(&dk_free[g & 1], before(g))) { ok = false; break; }
        if (!wait(&dz_full[g & 1], use(g))) { ok = false; break; }
        fence_proxy_async_smem();
        tc_fence_after();
        const uint32_t dz = sDz + (g & 1) * kDzBytes;
        const uint64_t dz_k = make_smem_desc(dz, 16, 1024, kSwizzle128B);                                   // K-major: contraction over heads
        const uint64_t q_mn = make_smem_desc(sQ + (n & 1) * kQBytes, kQChunk, 1024, kSwizzle128B);          // rows are heads, two chunks of 64 dims
        const uint64_t k_mn = make_smem_desc(sK + s * kKBytes, kKChunk, 1024, kSwizzle128B);
        const uint64_t dz_mn = make_smem_desc(dz, kDzBytes, 1024, kSwizzle128B);                            // rows are keys, one chunk of 64 heads
#pragma unroll
        for (int k = 0; k < kHeads / 16; ++k)
          umma_ss_if(go, tmem + kColDk + (g & 1) * kKeys, q_mn + k * (2048 >> 4), dz_k + 2 * k, id_dk, k != 0);
        umma_commit_if(go, &dk_full[g & 1]);
#pragma unroll
        for (int k = 0; k < kKeys / 16; ++k)
          umma_ss_if(go, tmem + kColDq + (n & 1) * kHeads, k_mn + k * (2048 >> 4), dz_mn + k * (2048 >> 4), id_dq, (i | k) != 0);
        umma_commit_if(go, &k_empty[s]);
        umma_commit_if(go, &dz_free[g & 1]);
      }
      if (!ok) break;
      umma_commit_if(go, &q_done[n & 1]);
      done_with(n);
    }
  } else if (warp < kDzWarps) {
    // ================================ dZ and dw =====================================================
    // warp = (quarter of the keys, half of the heads): thread = key 32 quarter + lane, heads 32 half .. + 31
    const int quarter = warp & 3, half = warp >> 2, key = quarter * 32 + lane;
    const uint32_t lane_base = static_cast<uint32_t>(quarter * 32) << 16;
    int g = 0;
    // (Every warp of the group takes the same turns, also when a wait has given up: the barriers count them all.  Whether a list can be
    // trusted is agreed on; that barrier also keeps a query's sums of dw apart from the next one's.)
    for (int n = 0;; ++n) {
      ok = bar_and(1, kDzWarps * 32, ok && wait(&list_full[n & 1], use(n)));
      if (!ok) break;
      const List& list = lists[n & 1];
      const int bt = list.query;
      if (bt < 0) break;
      const float* g_row = p.grad + static_cast<int64_t>(bt) * p.K;
      const float scale = list.scale;
      // this thread's key of the list's tile number i: does it take part, and its gradient
      auto takes_part = [&](int i) { return ((list.bits[list.tile[i] * (kKeys / 32) + quarter] >> lane) & 1u) != 0; };
      auto gradient = [&](int i) { return takes_part(i) ? __ldg(g_row + list.tile[i] * kKeys + key) : 0.f; };
      float dw[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) dw[i] = 0.f;
      float next = gradient(0);
      for (int i = 0; i < list.tiles; ++i, ++g) {
        const float gr = next;
        const bool there = takes_part(i);
        if (i + 1 < list.tiles) next = gradient(i + 1);
        ok = ok && wait(&z_full[g & 1], use(g));
        ok = ok && (g < 2 || wait(&dz_free[g & 1], before(g)));
        if (!ok) continue;
        tc_fence_after();
        const float gs = gr * scale;
        const uint32_t dz = sDz + (g & 1) * kDzBytes;
#pragma unroll
        for (int c0 = 0; c0 < 32; c0 += 16) {
          uint32_t v[16], w[8];
          tmem_ld16(tmem_base + kColZ + (g & 1) * kHeads + half * 32 + c0 + lane_base, v);
          tmem_wait_ld();
          if (!there) {   // (its row is zeros, but the query need not be finite)
#pragma unroll
            for (int k = 0; k < 16; ++k) v[k] = 0u;
          }
          const float4* w4 = reinterpret_cast<const float4*>(list.w + half * 32 + c0);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float4 wt = w4[j];
            float z[4], d[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              z[k] = __uint_as_float(v[4 * j + k]);
              dw[c0 + 4 * j + k] = fmaf(gr, relu(z[k]), dw[c0 + 4 * j + k]);
            }
            d[0] = z[0] <= 0.f ? 0.f : gs * wt.x;
            d[1] = z[1] <= 0.f ? 0.f : gs * wt.y;
            d[2] = z[2] <= 0.f ? 0.f : gs * wt.z;
            d[3] = z[3] <= 0.f ? 0.f : gs * wt.w;
            w[2 * j] = pack2<kBF16>(d[0], d[1]);
            w[2 * j + 1] = pack2<kBF16>(d[2], d[3]);
          }
          const int unit = half * 4 + c0 / 8;
          st_shared_v4(dz + sw128_offset(key, unit), w[0], w[1], w[2], w[3]);
          st_shared_v4(dz + sw128_offset(key, unit + 1), w[4], w[5], w[6], w[7]);
        }
        tc_fence_before();
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&z_free[g & 1]);
          mbar_arrive(&dz_full[g & 1]);
        }
      }
      // over the lanes (lane l ends with head 32 half + l), then over the four quarters
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
      named_bar_sync(1, kDzWarps * 32);
      if (ok && tid < p.N1)
        p.d_w[static_cast<int64_t>(bt) * p.N1 + tid] = (s_dw[tid] + s_dw[kHeads + tid]) + (s_dw[2 * kHeads + tid] + s_dw[3 * kHeads + tid]);
      done_with(n);
    }
  } else {
    // ================================ dK to global memory; dQ =======================================
    // warp = (quarter of the dims, half of the columns): thread = dim 32 quarter + lane, keys 64 half .. + 63 of dK^T, heads 32 half .. + 31 of dQ^T
    const int quarter = warp & 3, half = (warp - kAddWarp) >> 2;
    const uint32_t lane_base = static_cast<uint32_t>(quarter * 32) << 16;
    int g = 0;
    for (int n = 0; ok; ++n) {
      if (!wait(&list_full[n & 1], use(n))) { ok = false; break; }
      const List& list = lists[n & 1];
      const int bt = list.query;
      if (bt < 0) break;
      const float unscale = list.unscale;
      const int32_t* idx_row = p.indices + static_cast<int64_t>(bt) * p.K;
      float* dk = p.d_k + static_cast<int64_t>(bt / p.S1) * p.S2 * kD + quarter * 32 + lane;
      // the rows of this warp's 64 keys, read a tile ahead by the lanes and handed round through shared memory; -1: takes no part
      int* my_rows = s_row + (warp - kAddWarp) * 64;
      auto rows_of = [&](int i, int (&row)[2]) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int slot = list.tile[i] * kKeys + half * 64 + k * 32 + lane;
          row[k] = (list.bits[slot >> 5] >> lane) & 1u ? __ldg(idx_row + slot) : -1;
        }
      };
      int next[2];
      rows_of(0, next);
      for (int i = 0; i < list.tiles; ++i, ++g) {
        __syncwarp();
        my_rows[lane] = next[0];
        my_rows[32 + lane] = next[1];
        __syncwarp();
        if (i + 1 < list.tiles) rows_of(i + 1, next);
        if (!wait(&dk_full[g & 1], use(g))) { ok = false; break; }
        tc_fence_after();
        const int4* rows = reinterpret_cast<const int4*>(my_rows);
        const uint32_t* words = list.bits + list.tile[i] * 4 + half * 2;
        auto add = [&](auto all_keys) {
#pragma unroll
          for (int c0 = 0; c0 < 64; c0 += 16) {
            uint32_t v[16];
            tmem_ld16(tmem_base + kColDk + (g & 1) * kKeys + half * 64 + c0 + lane_base, v);
            tmem_wait_ld();
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int4 r = rows[c0 / 4 + j];
              const int row[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const float d = kBF16 ? __uint_as_float(v[4 * j + k]) : __uint_as_float(v[4 * j + k]) * unscale;
                if (decltype(all_keys)::value || row[k] >= 0) atomicAdd(dk + static_cast<int64_t>(row[k]) * kD, d);
              }
            }
          }
        };
        // (a branch per key holds a warp up more than its addition)
        if ((words[0] & words[1]) == 0xffffffffu) add(std::true_type{});
        else add(std::false_type{});
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&dk_free[g & 1]);
      }
      if (!ok) break;
      if (!wait(&q_done[n & 1], use(n))) { ok = false; break; }
      tc_fence_after();
      T* dq = reinterpret_cast<T*>(p.d_q) + static_cast<int64_t>(bt) * p.N1 * kD + quarter * 32 + lane;
#pragma unroll
      for (int c0 = 0; c0 < 32; c0 += 16) {
        uint32_t v[16];
        tmem_ld16(tmem_base + kColDq + (n & 1) * kHeads + half * 32 + c0 + lane_base, v);
        tmem_wait_ld();
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          const int h = half * 32 + c0 + k;
          if (h < p.N1) dq[h * kD] = static_cast<T>(__uint_as_float(v[k]) * unscale);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&dq_free[n & 1]);
      done_with(n);
    }
  }
  cp_async_wait<0>();
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
  const long long n = static_cast<long long>(p.B) * p.S1;
  kern<<<static_cast<unsigned>(n < sms ? n : sms), ib::kThreads, ib::kSmemBytes, stream>>>(p);
  return static_cast<int>(cudaGetLastError());
}

}  // namespace dsa
