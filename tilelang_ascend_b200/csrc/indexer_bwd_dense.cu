// Backward of the lightning indexer's listed scores when the lists hold a large part of the keys that their queries may see (sm_100a, tcgen05; bf16, 128 dims, 16,
// 32 or 64 heads).  The mathematics is that of indexer_bwd.cu; what differs is how the key gradient is summed.  There every (query, listed key)
// pair adds 512 bytes to global memory, and those additions are what it takes; here both gradients are products over whole
// tiles, each owned by the CTA that sums it in tensor memory:
//
//   spread   the lists' gradients become a matrix G [B, S1, S2 padded to 128] (0 where not listed) and a flag per (query, tile of 128 keys)
//   kQueries a CTA owns 128 (query, head) rows and walks the key tiles:    dQ^T[128 dims x 128 rows] += K^T dZ,  and dw
//   kKeys    a CTA owns 128 keys and walks blocks of 128 (query, head) rows:  dK^T[128 dims x 128 keys] += Q^T dZ^T
//
// with Z[128 keys x 128 rows] = K Q^T and dZ = G w [Z > 0] made once in each.  Tiles are dense, so they come by TMA, without
// indices; (block, tile) pairs without a listed key are skipped by the flags (the upper half of a causal step).  1024 clocks of MMAs
// per pair of tiles and kernel.
// A dense product also multiplies what is not listed, by 0.  Where that holds infinities or NaN (padding that was never written), 0
// is the wrong answer, so `spread` looks through q and k for them; if there are any, these kernels do nothing and the other kernel,
// launched behind them, does it all.
#include <stdint.h>
#include <string.h>

#include "fwd_common.cuh"
#include "indexer_bwd.h"
#include "launch_util.h"
#include "tensor_map.h"

namespace dsa {

namespace ibd {
constexpr int kD = 128, kTile = 128;                                  // dims; keys or (query, head) rows of a tile
constexpr uint32_t kChunk = kTile * 128, kTileBytes = 2 * kChunk;     // two chunks of 64 dims (dZ: of 64 rows)
constexpr int kStages = 3;
constexpr int kMaxSteps = 1024;                                       // tiles an item may walk
constexpr int kWorkers = 16, kLoadWarp = 16, kZWarp = 17, kMmaWarp = 18, kListWarp = 19, kThreads = 20 * 32;
constexpr int kUsers = kWorkers + 3;
struct Steps {
  int item, count;               // item -1: no more
  int pad[2];
  uint16_t step[kMaxSteps];
};
constexpr uint32_t kOffRing = kTileBytes, kOffDz = kOffRing + kStages * kTileBytes;
constexpr uint32_t kOffBar = kOffDz + 2 * kTileBytes;
constexpr uint32_t kOffW = kOffBar + 256;                             // head weights of the stages' rows, and of the own ones
constexpr uint32_t kOffDw = kOffW + (kStages + 1) * kTile * 4;        // four quarters' sums of 128 rows
constexpr uint32_t kOffSteps = kOffDw + 4 * kTile * 4;
constexpr uint32_t kSmemBytes = kOffSteps + 2 * sizeof(Steps);
constexpr uint32_t kColZ = 0, kColAcc = 256, kTmemCols = 512;         // two of each, 128 columns
static_assert(kSmemBytes <= 232448, "shared memory per CTA");

__device__ __forceinline__ bool bar_and(uint32_t id, uint32_t nthreads, bool yes) {
  uint32_t all;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "bar.red.and.pred q, %2, %3, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(all)
      : "r"(yes ? 1u : 0u), "r"(id), "r"(nthreads)
      : "memory");
  return all != 0;
}

// Contiguous global -> shared copy (16-byte aligned addresses, size a multiple of 16); its bytes count on the barrier.
__device__ __forceinline__ void bulk_load(uint32_t smem_dst, const void* src, uint32_t bytes, uint32_t mbar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_dst), "l"(src), "r"(bytes), "r"(mbar)
               : "memory");
}

struct Dense {
  const int* dirty;       // not 0: q or k hold infinities or NaN, nothing is done
  int* next;              // [2] items handed out so far
  const float* grad;      // G [B, S1, width]
  const uint8_t* flags;   // [B, S1, width / 128]
  int width, tiles;       // S2 rounded up to 128; width / 128
  int queries;            // per block of 128 rows
  int blocks;             // of a batch entry's queries
  int splits, per_split;  // kKeys: parts a key tile's blocks are walked in
};
}  // namespace ibd

// -------------------------------------------------------------------------------------------------
// spread: block = (query, 8192 columns of G).  The blocks also look through q (each its query) and k (each its share of the rows).
// -------------------------------------------------------------------------------------------------
__global__ void __launch_bounds__(256)
    indexer_bwd_spread_kernel(const __grid_constant__ IndexerBwdParams p, float* G, uint8_t* flags, int* dirty, const int width, const int parts, const int k_units) {
  // bf16 infinities and NaN: all bits of the exponent
  auto odd_pair = [](uint32_t w) { return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u; };
  auto odd = [&](const uint4& v) { return odd_pair(v.x) || odd_pair(v.y) || odd_pair(v.z) || odd_pair(v.w); };
  constexpr int kCols = 8192;
  __shared__ __align__(16) float acc[kCols];
  __shared__ uint8_t s_flags[kCols / 128];
  const int64_t bt = blockIdx.x / parts;
  const int c0 = static_cast<int>(blockIdx.x - bt * parts) * kCols, n = min(width - c0, kCols);
  const int tid = threadIdx.x;
  // the list's first entries travel while the rest is prepared
  constexpr int kAhead = 8;
  int idx[kAhead];
  float gr[kAhead];
#pragma unroll
  for (int i = 0; i < kAhead; ++i) {
    const int j = tid + 256 * i;
    idx[i] = j < p.K ? __ldg(p.indices + bt * p.K + j) : -1;
    gr[i] = j < p.K ? __ldg(p.grad + bt * p.K + j) : 0.f;
  }
  for (int i = tid * 4; i < n; i += 1024) *reinterpret_cast<float4*>(acc + i) = make_float4(0.f, 0.f, 0.f, 0.f);
  if (tid < kCols / 128) s_flags[tid] = 0;
  bool found = false;
  if (c0 == 0) {
    const uint4* q = reinterpret_cast<const uint4*>(p.q) + bt * p.N1 * 16;
#pragma unroll 4
    for (int i = tid; i < p.N1 * 16; i += 256) found |= odd(__ldg(q + i));
    const uint4* k = reinterpret_cast<const uint4*>(p.k);
    const int64_t last = min(static_cast<int64_t>(p.B) * p.S2 * 16, (bt + 1) * k_units);
    for (int64_t i = bt * k_units + tid; i < last; i += 256) found |= odd(__ldg(k + i));
  }
  if (found) *dirty = 1;
  __syncthreads();
  auto put = [&](int key, float g) {
    const int c = key - c0;
    if (key >= 0 && key < p.S2 && c >= 0 && c < n) {
      atomicAdd(&acc[c], g);   // (a key listed twice counts twice)
      s_flags[c >> 7] = 1;
    }
  };
#pragma unroll
  for (int i = 0; i < kAhead; ++i) put(idx[i], gr[i]);
  for (int j = tid + 256 * kAhead; j < p.K; j += 256) put(__ldg(p.indices + bt * p.K + j), __ldg(p.grad + bt * p.K + j));
  __syncthreads();
  for (int i = tid * 4; i < n; i += 1024) *reinterpret_cast<float4*>(G + bt * width + c0 + i) = *reinterpret_cast<const float4*>(acc + i);
  if (tid < n / 128) flags[bt * (width / 128) + c0 / 128 + tid] = s_flags[tid];
}

// -------------------------------------------------------------------------------------------------
// the two products
// -------------------------------------------------------------------------------------------------
enum { kQueries, kKeys };

template <int kOwner, int N1>
__global__ void __launch_bounds__(ibd::kThreads, 1)
    indexer_bwd_dense_kernel(const __grid_constant__ IndexerBwdParams p, const __grid_constant__ ibd::Dense d, const __grid_constant__ CUtensorMap q_map,
                             const __grid_constant__ CUtensorMap k_map) {
  using namespace ibd;
  constexpr int kCols = 32, kMine = N1 < kCols ? kCols / N1 : 1;   // a worker's columns; queries among them when they are rows
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t sOwn = smem_u32(smem);
  if (sOwn & 1023u) {
    if (threadIdx.x == 0) atomicCAS(p.status, kStatusOk, kStatusBadLayout);
    return;
  }
  const uint32_t sRing = sOwn + kOffRing, sDz = sOwn + kOffDz;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kOffBar);
  uint64_t* own_full = bars;         // count 1 + transaction bytes: the item's own tile has landed
  uint64_t* own_done = bars + 1;     // count 1: commit after an item's last MMAs: its own tile is free, its sum is complete
  uint64_t* full = bars + 2;         // [3] count 1 + transaction bytes
  uint64_t* empty = bars + 5;        // [3] count 1: commit after the MMAs that read the stage
  uint64_t* z_full = bars + 8;       // [2] count 1: commit after Z
  uint64_t* z_free = bars + 10;      // [2] count 16: Z has been read
  uint64_t* dz_full = bars + 12;     // [2] count 16: dZ is in shared memory
  uint64_t* dz_free = bars + 14;     // [2] count 1: commit after the MMAs that read dZ
  uint64_t* acc_free = bars + 16;    // [2] count 16: the sum has been read
  uint64_t* list_full = bars + 18;   // [2] count 1
  uint64_t* list_free = bars + 20;   // [2] count kUsers
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 22);
  int* start_status = reinterpret_cast<int*>(bars + 23);
  float* s_w = reinterpret_cast<float*>(smem + kOffW);
  float* s_dw = reinterpret_cast<float*>(smem + kOffDw);
  Steps* lists = reinterpret_cast<Steps*>(smem + kOffSteps);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (*d.dirty) return;
  if (tid == 0) {
    *start_status = *reinterpret_cast<volatile int*>(p.status);
    mbar_init(own_full, 1); mbar_init(own_done, 1);
    for (int i = 0; i < kStages; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&z_full[i], 1); mbar_init(&z_free[i], kWorkers); mbar_init(&dz_full[i], kWorkers); mbar_init(&dz_free[i], 1);
      mbar_init(&acc_free[i], kWorkers); mbar_init(&list_full[i], 1); mbar_init(&list_free[i], kUsers);
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
  // two at once: the answer of a barrier takes 200 clocks and more on this busy shared memory
  auto wait_both = [&](uint64_t* a, uint32_t parity_a, uint64_t* b, uint32_t parity_b, bool b_needed) {
    const bool got_a = mbar_try_wait(a, parity_a), got_b = !b_needed || mbar_try_wait(b, parity_b);
    return __all_sync(0xffffffffu, got_a && got_b) || (wait(a, parity_a) && (!b_needed || wait(b, parity_b)));
  };
  auto use = [](int n) { return static_cast<uint32_t>(n >> 1) & 1u; };           // parity of the n-th use of one of two
  auto before = [](int n) { return (static_cast<uint32_t>(n >> 1) + 1u) & 1u; }; // of the use before it
  auto done_with = [&](int n) {
    __syncwarp();
    if (lane == 0) mbar_arrive(&list_free[n & 1]);
  };
  const int per_batch = kOwner == kQueries ? d.blocks : d.tiles * d.splits, items = p.B * per_batch;
  // an item's batch entry, and the block of rows or the key tile that it owns
  auto batch_of = [&](int item) { return item / per_batch; };
  auto owned = [&](int item) { return kOwner == kQueries ? item % per_batch : item % per_batch / d.splits; };

  if (warp == kListWarp) {
    // ================================ which tiles an item walks, one item ahead =====================
    // Items are handed out one by one: how many tiles one walks is known here only.
    int n = 0;
    while (ok) {
      int i = 0;
      if (lane == 0) i = atomicAdd(d.next + kOwner, 1);
      i = __shfl_sync(0xffffffffu, i, 0);
      if (i >= items) break;
      const int item = kOwner == kQueries ? items - 1 - i : i;   // (late queries walk the most tiles)
      if (n >= 2 && !wait(&list_free[n & 1], before(n))) { ok = false; break; }
      Steps& list = lists[n & 1];
      const int b = batch_of(item), own = owned(item);
      const int first = kOwner == kQueries ? 0 : (item % d.splits) * d.per_split;
      const int last = kOwner == kQueries ? d.tiles : min(d.blocks, first + d.per_split);
      const uint8_t* flags = d.flags + static_cast<int64_t>(b) * p.S1 * d.tiles;
      int count = 0;
      for (int s0 = first; s0 < last; s0 += 32) {
        const int s = s0 + lane, tile = kOwner == kQueries ? s : own, block = kOwner == kQueries ? own : s;
        bool any = false;
        if (s < last)
          for (int k = 0; k < d.queries; ++k) {
            const int query = block * d.queries + k;
            any |= query < p.S1 && __ldg(flags + static_cast<int64_t>(query) * d.tiles + tile) != 0;
          }
        const uint32_t bits = __ballot_sync(0xffffffffu, any);
        if (any) list.step[count + __popc(bits & ((1u << lane) - 1))] = static_cast<uint16_t>(s);
        count += __popc(bits);
      }
      if (!count) {
        if (kOwner == kQueries) {   // rows without a key: zeros
          const int rows = min(kTile, (p.S1 - own * d.queries) * N1);
          const int64_t row0 = (static_cast<int64_t>(b) * p.S1 + own * d.queries) * N1;
          uint4* dq = reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(p.d_q) + row0 * kD);
          for (int k = lane; k < rows * kD / 8; k += 32) dq[k] = make_uint4(0, 0, 0, 0);
          for (int k = lane; k < rows; k += 32) p.d_w[row0 + k] = 0.f;
        }
        continue;
      }
      __syncwarp();
      if (lane == 0) {
        list.item = item;
        list.count = count;
        mbar_arrive(&list_full[n & 1]);
      }
      __syncwarp();
      ++n;
    }
    if (ok && n >= 2) ok = wait(&list_free[n & 1], before(n));
    if (ok && lane == 0) {
      lists[n & 1].item = -1;
      mbar_arrive(&list_full[n & 1]);
    }
  } else if (warp == kLoadWarp) {
    // ================================ tile loads (one lane issues) ==================================
    const CUtensorMap* own_map = kOwner == kQueries ? &q_map : &k_map;
    const CUtensorMap* walk_map = kOwner == kQueries ? &k_map : &q_map;
    if (lane == 0) { prefetch_tensormap(own_map); prefetch_tensormap(walk_map); }
    int g = 0;
    for (int n = 0; ok; ++n) {
      if (!wait(&list_full[n & 1], use(n))) { ok = false; break; }
      const Steps& list = lists[n & 1];
      const int item = list.item;
      if (item < 0) break;
      const int b = batch_of(item), own = owned(item);
      const int q_row0 = b * p.S1 * N1, k_row0 = b * p.S2;
      if (n >= 1 && !wait(own_done, (n + 1) & 1)) { ok = false; break; }
      // the head weights of a block of rows travel with them
      auto weight_bytes = [&](int block) { return static_cast<uint32_t>(min(kTile, p.S1 * N1 - block * kTile)) * 4u; };
      const float* weights = p.w + static_cast<int64_t>(q_row0);
      if (lane == 0) {
        mbar_arrive_expect_tx(own_full, kTileBytes + (kOwner == kQueries ? weight_bytes(own) : 0u));
        if (kOwner == kQueries) bulk_load(smem_u32(s_w + kStages * kTile), weights + own * kTile, weight_bytes(own), smem_u32(own_full));
        for (int c = 0; c < 2; ++c) tma_load_2d(sOwn + c * kChunk, own_map, smem_u32(own_full), c * 64, (kOwner == kQueries ? q_row0 : k_row0) + own * kTile);
      }
      __syncwarp();
      for (int i = 0; i < list.count; ++i, ++g) {
        const int s = g % kStages;
        if (g >= kStages && !wait(&empty[s], ((g / kStages) + 1) & 1)) { ok = false; break; }
        if (lane == 0) {
          mbar_arrive_expect_tx(&full[s], kTileBytes + (kOwner == kKeys ? weight_bytes(list.step[i]) : 0u));
          if (kOwner == kKeys) bulk_load(smem_u32(s_w + s * kTile), weights + list.step[i] * kTile, weight_bytes(list.step[i]), smem_u32(&full[s]));
          for (int c = 0; c < 2; ++c)
            tma_load_2d(sRing + s * kTileBytes + c * kChunk, walk_map, smem_u32(&full[s]), c * 64, (kOwner == kQueries ? k_row0 : q_row0) + list.step[i] * kTile);
        }
        __syncwarp();
      }
      if (!ok) break;
      done_with(n);
    }
  } else if (warp == kZWarp) {
    // ================================ MMA issuer of Z (converged, one elected lane issues) ==========
    constexpr uint32_t idesc = make_idesc_f16(true, kTile, kTile, 0, 0);
    const uint32_t go = elect_one_lane(), tmem = __reduce_or_sync(0xffffffffu, tmem_base);
    int g = 0;
    for (int n = 0; ok; ++n) {
      if (!wait(&list_full[n & 1], use(n))) { ok = false; break; }
      const int count = __reduce_or_sync(0xffffffffu, lists[n & 1].item < 0 ? 0u : static_cast<uint32_t>(lists[n & 1].count));
      if (!count) break;
      if (!wait(own_full, n & 1)) { ok = false; break; }
      for (int i = 0; i < count; ++i, ++g) {
        const int s = g % kStages;
        if (!wait_both(&full[s], (g / kStages) & 1, &z_free[g & 1], before(g), g >= 2)) { ok = false; break; }
        tc_fence_after();
        const uint32_t walked = sRing + s * kTileBytes, keys = kOwner == kQueries ? walked : sOwn, rows = kOwner == kQueries ? sOwn : walked;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const uint64_t da = make_smem_desc(keys + c * kChunk, 16, 1024, kSwizzle128B), db = make_smem_desc(rows + c * kChunk, 16, 1024, kSwizzle128B);
#pragma unroll
          for (int k = 0; k < 4; ++k) umma_ss_if(go, tmem + kColZ + (g & 1) * kTile, da + 2 * k, db + 2 * k, idesc, (c | k) != 0);
        }
        umma_commit_if(go, &z_full[g & 1]);
      }
      if (!ok) break;
      done_with(n);
    }
  } else if (warp == kMmaWarp) {
    // ================================ MMA issuer of the sums ========================================
    constexpr uint32_t idesc = make_idesc_f16(true, kD, kTile, 1, kOwner == kQueries ? 1 : 0);
    const uint32_t go = elect_one_lane(), tmem = __reduce_or_sync(0xffffffffu, tmem_base);
    int g = 0;
    for (int n = 0; ok; ++n) {
      if (!wait(&list_full[n & 1], use(n))) { ok = false; break; }
      const int count = __reduce_or_sync(0xffffffffu, lists[n & 1].item < 0 ? 0u : static_cast<uint32_t>(lists[n & 1].count));
      if (!count) break;
      if (n >= 2 && !wait(&acc_free[n & 1], before(n))) { ok = false; break; }
      for (int i = 0; i < count; ++i, ++g) {
        const int s = g % kStages;
        if (!wait(&dz_full[g & 1], use(g))) { ok = false; break; }
        fence_proxy_async_smem();
        tc_fence_after();
        // A: the walked tile read MN-major (128 dims; contraction over its keys or rows); B: dZ, rows are keys, two chunks of 64 (query, head) rows:
        // MN-major over the keys (kQueries), K-major over the rows (kKeys)
        const uint32_t dz = sDz + (g & 1) * kTileBytes;
        const uint64_t da = make_smem_desc(sRing + s * kTileBytes, kChunk, 1024, kSwizzle128B);
        const uint64_t db = kOwner == kQueries ? make_smem_desc(dz, kChunk, 1024, kSwizzle128B) : make_smem_desc(dz, 16, 1024, kSwizzle128B);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const uint32_t step = kOwner == kQueries ? k * (2048 >> 4) : ((k >> 2) * (kChunk >> 4) + 2 * (k & 3));
          umma_ss_if(go, tmem + kColAcc + (n & 1) * kTile, da + k * (2048 >> 4), db + step, idesc, (i | k) != 0);
        }
        umma_commit_if(go, &empty[s]);
        umma_commit_if(go, &dz_free[g & 1]);
      }
      if (!ok) break;
      umma_commit_if(go, own_done);
      done_with(n);
    }
  } else {
    // ================================ dZ and dw; the sums to global memory ==========================
    // warp = (quarter, group): key 32 quarter + lane and rows 32 group .. + 31 of Z; dim 32 quarter + lane and columns 32 group .. + 31 of a sum
    const int quarter = warp & 3, group = warp >> 2, key = quarter * 32 + lane;
    const uint32_t lane_base = static_cast<uint32_t>(quarter * 32) << 16;
    int g = 0;
    // (Every warp of the group takes the same turns, also when a wait has given up: the barriers count them all.)
    for (int n = 0;; ++n) {
      ok = bar_and(1, kWorkers * 32, ok && wait(&list_full[n & 1], use(n)));
      if (!ok) break;
      const Steps& list = lists[n & 1];
      const int item = list.item;
      if (item < 0) break;
      const int b = batch_of(item), own = owned(item), count = list.count;
      const float* grad = d.grad + static_cast<int64_t>(b) * p.S1 * d.width + key;
      // this thread's gradients of a step: of its key, for the queries of its rows (0 behind the last query)
      auto gradients = [&](int i, float (&to)[kMine]) {
        const int step = list.step[i], tile = kOwner == kQueries ? step : own, query0 = (kOwner == kQueries ? own : step) * d.queries + group * kCols / N1;
#pragma unroll
        for (int k = 0; k < kMine; ++k) to[k] = query0 + k < p.S1 ? __ldg(grad + static_cast<int64_t>(query0 + k) * d.width + tile * kTile) : 0.f;
      };
      float dw[kOwner == kQueries ? kCols : 1];
#pragma unroll
      for (int k = 0; k < (kOwner == kQueries ? kCols : 1); ++k) dw[k] = 0.f;
      float next[kMine];
      gradients(0, next);
      for (int i = 0; i < count; ++i, ++g) {
        float gr[kMine], above[kMine];   // dz where z is above: nowhere without a gradient, whatever the weight is
#pragma unroll
        for (int k = 0; k < kMine; ++k) {
          gr[k] = next[k];
          above[k] = gr[k] != 0.f ? 0.f : INFINITY;
        }
        if (i + 1 < count) gradients(i + 1, next);
        ok = ok && wait_both(&z_full[g & 1], use(g), &dz_free[g & 1], before(g), g >= 2);
        if (!ok) continue;
        tc_fence_after();
        const uint32_t dz = sDz + (g & 1) * kTileBytes + (group >> 1) * kChunk;
        const float4* w4 = reinterpret_cast<const float4*>(s_w + (kOwner == kQueries ? kStages : g % kStages) * kTile + group * kCols);
#pragma unroll
        for (int c0 = 0; c0 < kCols; c0 += 16) {
          const int k = c0 / N1;   // which of this thread's queries
          uint32_t v[16], w[8];
          tmem_ld16(tmem_base + kColZ + (g & 1) * kTile + group * kCols + c0 + lane_base, v);
          tmem_wait_ld();
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float4 wt = w4[c0 / 4 + j];
            const float2 gg = make_float2(gr[k], gr[k]), lo = fmul2(gg, make_float2(wt.x, wt.y)), hi = fmul2(gg, make_float2(wt.z, wt.w));
            float z[4];
#pragma unroll
            for (int m = 0; m < 4; ++m) z[m] = __uint_as_float(v[4 * j + m]);
            if constexpr (kOwner == kQueries) {
              float* e = dw + c0 + 4 * j;
              const float2 lo_w = ffma2(gg, make_float2(fmaxf(z[0], 0.f), fmaxf(z[1], 0.f)), make_float2(e[0], e[1]));
              const float2 hi_w = ffma2(gg, make_float2(fmaxf(z[2], 0.f), fmaxf(z[3], 0.f)), make_float2(e[2], e[3]));
              e[0] = lo_w.x; e[1] = lo_w.y; e[2] = hi_w.x; e[3] = hi_w.y;
            }
            w[2 * j] = pack2<true>(z[0] > above[k] ? lo.x : 0.f, z[1] > above[k] ? lo.y : 0.f);
            w[2 * j + 1] = pack2<true>(z[2] > above[k] ? hi.x : 0.f, z[3] > above[k] ? hi.y : 0.f);
          }
          const int unit = (group & 1) * 4 + c0 / 8;
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
      if constexpr (kOwner == kQueries) {
        // dw over the lanes (lane l ends with row l of the group), then over the four quarters
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          const bool upper = lane & o;
#pragma unroll
          for (int k = 0; k < o; ++k) {
            const float give = upper ? dw[k] : dw[k + o], mine = upper ? dw[k + o] : dw[k];
            dw[k] = mine + __shfl_xor_sync(0xffffffffu, give, o);
          }
        }
        s_dw[quarter * kTile + group * kCols + lane] = dw[0];
        named_bar_sync(1, kWorkers * 32);
        const int rows = min(kTile, (p.S1 - own * d.queries) * N1);
        if (ok && tid < rows)
          p.d_w[(static_cast<int64_t>(b) * p.S1 + own * d.queries) * N1 + tid] =
              (s_dw[tid] + s_dw[kTile + tid]) + (s_dw[2 * kTile + tid] + s_dw[3 * kTile + tid]);
      }
      ok = ok && wait(own_done, n & 1);
      if (ok) {
        tc_fence_after();
#pragma unroll 1
        for (int c0 = 0; c0 < kCols; c0 += 16) {
          uint32_t v[16];
          tmem_ld16(tmem_base + kColAcc + (n & 1) * kTile + group * kCols + c0 + lane_base, v);
          tmem_wait_ld();
          const int first = own * kTile + group * kCols + c0, dim = quarter * 32 + lane;   // the sum's first column among the batch entry's rows or keys
          const int limit = kOwner == kQueries ? p.S1 * N1 : p.S2;
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            if (first + k >= limit) continue;
            const int64_t at = (static_cast<int64_t>(b) * limit + first + k) * kD + dim;
            if (kOwner == kQueries) reinterpret_cast<__nv_bfloat16*>(p.d_q)[at] = __float2bfloat16(__uint_as_float(v[k]));
            else atomicAdd(p.d_k + at, __uint_as_float(v[k]));
          }
        }
        tc_fence_before();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_free[n & 1]);
      done_with(n);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) tmem_dealloc(tmem_base, kTmemCols);
}

// -------------------------------------------------------------------------------------------------
// host side
// -------------------------------------------------------------------------------------------------
namespace {
int padded_width(const IndexerBwdParams& p) { return (p.S2 + ibd::kTile - 1) / ibd::kTile * ibd::kTile; }

template <int kOwner, int N1>
int launch_owner(const IndexerBwdParams& p, const ibd::Dense& d, const CUtensorMap& q_map, const CUtensorMap& k_map, int dev, int sms, cudaStream_t stream) {
  auto kern = indexer_bwd_dense_kernel<kOwner, N1>;
  const cudaError_t e = ensure_dynamic_smem(kern, dev, static_cast<int>(ibd::kSmemBytes));
  if (e != cudaSuccess) return static_cast<int>(e);
  const long long items = static_cast<long long>(p.B) * (kOwner == kQueries ? d.blocks : d.tiles * d.splits);
  kern<<<static_cast<unsigned>(items < sms ? items : sms), ibd::kThreads, ibd::kSmemBytes, stream>>>(p, d, q_map, k_map);
  return static_cast<int>(cudaGetLastError());
}
template <int N1>
int launch_both(const IndexerBwdParams& p, const ibd::Dense& d, const CUtensorMap& q_map, const CUtensorMap& k_map, int dev, int sms, cudaStream_t stream) {
  const int err = launch_owner<kQueries, N1>(p, d, q_map, k_map, dev, sms, stream);
  return err ? err : launch_owner<kKeys, N1>(p, d, q_map, k_map, dev, sms, stream);
}
}  // namespace

// Which kernel: the other one takes about 105 ps per (query, listed key), whatever the heads; these take 60 ps per (query, key that it may
// see) with 64 heads, half and a quarter of that with 32 and 16, and 20 us more for G and three more launches.  Both counts as they are
// in a causal step (keys up to S2 - S1 + t) with full lists.  Measured, other / these, us: 4096 queries x 4096 keys, lists of 2048:
// 671 / 540, of 1024: 410 / 530; 4096 x 8192, 2048: 855 / 1416; 1024 x 4096, 2048: 223 / 278; 4096 x 1024, 512, 16 heads: 258 / 118; 2048 x 2048,
// 2048, 32 heads: 251 / 121.  fp16 stays with the other kernel: its range needs a scale per query.
static bool dense_preferred(const IndexerBwdParams& p, bool bf16) {
  if (!bf16 || p.D != ibd::kD || (p.N1 != 16 && p.N1 != 32 && p.N1 != 64)) return false;
  const long long B = p.B, S1 = p.S1, S2 = p.S2, K = p.K < p.S2 ? p.K : p.S2;
  if (B * S1 * padded_width(p) > (1LL << 28) || padded_width(p) / ibd::kTile > ibd::kMaxSteps || B * S1 * p.N1 >= (1LL << 30) || B * S2 >= (1LL << 30)) return false;
  const long long seen = S1 <= S2 ? S1 * (2 * S2 - S1 + 1) / 2 : S1 * S2;
  const long long first = S2 - S1 + 1;   // keys that query 0 may see
  const long long shorter = S1 > S2 || first >= K ? 0 : (K - first < S1 ? K - first : S1);   // queries that see fewer than K
  const long long listed = S1 * K - (shorter ? shorter * (2 * K - 2 * first - shorter + 1) / 2 : 0);
  return B * listed * 105 > B * seen * 60 * p.N1 / 64 + 20 * 1000 * 1000;
}

namespace {
struct Layout {
  size_t flags, dirty, bytes;   // offsets behind G
};
Layout layout(const IndexerBwdParams& p) {
  const size_t cells = static_cast<size_t>(p.B) * p.S1 * padded_width(p);
  Layout l;
  l.flags = cells * sizeof(float);
  l.dirty = (l.flags + cells / ibd::kTile + 15) & ~static_cast<size_t>(15);
  l.bytes = l.dirty + 16;
  return l;
}
}  // namespace

// 0: the other kernel is preferred.
size_t indexer_bwd_workspace_bytes(const IndexerBwdParams& p, bool bf16) { return dense_preferred(p, bf16) ? layout(p).bytes : 0; }

// Is a call that brought this workspace, 16-byte aligned, taken here?
bool indexer_bwd_dense_fits(const IndexerBwdParams& p, bool bf16) {
  return dense_preferred(p, bf16) && (reinterpret_cast<uintptr_t>(p.w) & 15u) == 0 && encode_tiled_fn() != nullptr;
}

// *dirty_out: where the device says whether the call is left to launch_indexer_bwd.
int launch_indexer_bwd_dense(const IndexerBwdParams& p, void* workspace, const int** dirty_out, cudaStream_t stream) {
  using namespace ibd;
  int dev = 0, sms = 0;
  cudaError_t e = current_device_sms(&dev, &sms);
  if (e != cudaSuccess) return static_cast<int>(e);
  Dense d;
  d.width = padded_width(p);
  d.tiles = d.width / kTile;
  d.queries = kTile / p.N1;
  d.blocks = (p.S1 + d.queries - 1) / d.queries;
  // a key tile's blocks in parts: about eight items per SM, so that their unequal lengths even out
  int splits = (8 * sms + p.B * d.tiles - 1) / (p.B * d.tiles);
  if (splits > d.blocks) splits = d.blocks;
  d.per_split = (d.blocks + splits - 1) / splits;
  if (d.per_split > kMaxSteps) d.per_split = kMaxSteps;
  d.splits = (d.blocks + d.per_split - 1) / d.per_split;
  const Layout l = layout(p);
  float* G = static_cast<float*>(workspace);
  uint8_t* flags = static_cast<uint8_t*>(workspace) + l.flags;
  int* dirty = reinterpret_cast<int*>(static_cast<uint8_t*>(workspace) + l.dirty);
  d.grad = G;
  d.flags = flags;
  d.dirty = *dirty_out = dirty;
  d.next = dirty + 1;
  alignas(64) CUtensorMap q_map, k_map;
  memset(&q_map, 0, sizeof(q_map));
  memset(&k_map, 0, sizeof(k_map));
  if (!encode_rows_map(p.q, static_cast<long long>(p.B) * p.S1 * p.N1, kD, true, kTile, &q_map) ||
      !encode_rows_map(p.k, static_cast<long long>(p.B) * p.S2, kD, true, kTile, &k_map))
    return static_cast<int>(cudaErrorInvalidValue);
  const int parts = (d.width + 8191) / 8192;
  const long long spread = static_cast<long long>(p.B) * p.S1 * parts;
  if (spread > 0x7fffffffLL) return static_cast<int>(cudaErrorInvalidValue);
  if ((e = cudaMemsetAsync(dirty, 0, 3 * sizeof(int), stream)) != cudaSuccess) return static_cast<int>(e);
  const int k_units = static_cast<int>((static_cast<long long>(p.S2) * 16 + p.S1 - 1) / p.S1);   // 16-byte units of k per query
  indexer_bwd_spread_kernel<<<static_cast<unsigned>(spread), 256, 0, stream>>>(p, G, flags, dirty, d.width, parts, k_units);
  if ((e = cudaGetLastError()) != cudaSuccess) return static_cast<int>(e);
  if (p.N1 == 64) return launch_both<64>(p, d, q_map, k_map, dev, sms, stream);
  if (p.N1 == 32) return launch_both<32>(p, d, q_map, k_map, dev, sms, stream);
  return launch_both<16>(p, d, q_map, k_map, dev, sms, stream);
}

}  // namespace dsa
