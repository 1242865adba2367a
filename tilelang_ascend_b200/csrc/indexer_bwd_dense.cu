// Backward of the lightning indexer's listed scores when the lists hold a large part of the keys that their queries may see (sm_100a, tcgen05; bf16, 128 dims, 16,
// 32 or 64 heads).  The mathematics is that of indexer_bwd.cu; what differs is how the key gradient is summed.  There every (query, listed key)
// pair adds 512 bytes to global memory, and those additions are what it takes; here both gradients are products over whole
// tiles, each owned by the CTA that sums it in tensor memory:
//
//   spread   the lists' gradients become a matrix G [B, S1, S2 padded to 128] (0 where not listed) and a flag per (query, tile of 128 keys)
//   kQueries a CTA owns 128 (query, head) rows and walks the key tiles:              dQ[128 rows x 128 dims] += dZ K,  and dw
//   kKeys    a CTA owns 128 keys and walks blocks of 128 (query, head) rows:         dK[128 keys x 128 dims] += dZ Q
//
// with Z[128 own x 128 walked] = own . walked and dZ = G w [Z > 0], made once in each.  The walked tile is read twice from shared memory,
// K-major for Z and MN-major for the sum; dZ goes to tensor memory, over the columns of Z that have been read, so that the sum takes its
// first operand there.  What bounds a step is the way from Z to dZ to the sum's MMAs (about 3900 clocks, of which the two
// products are 1024), so three steps are under way: three places for Z, each with four warps that turn Z into dZ all by themselves
// (no barrier among them), and the group that has an item's last step reads the sum out while the others go on.  Measured for 4096 queries x 2048
// of 4096 keys, 64 heads: kQueries 206 and kKeys 207 us (1370 TFLOP/s of what they multiply); with dZ in shared memory and all 16 warps at one
// step 257 and 244, of which the MMAs and the loads were not the bound (left out, the time stayed), the warps' 3200 clocks for two steps were.
// Tiles are dense, so they come by TMA, without indices; (block, tile) pairs without a listed key are skipped by the flags (the upper
// half of a causal step).
// A dense product also multiplies what is not listed, by 0.  Where that holds infinities, NaN or values whose products overflow
// (padding that was never written), 0 is the wrong answer, so `spread` looks through q, k and w for them; if there are any, these
// kernels do nothing and the other kernel, launched behind them, does it all.
#include <stdint.h>
#include <string.h>

#include "fwd_common.cuh"
#include "indexer_bwd.h"
#include "launch_util.h"
#include "tensor_map.h"

namespace dsa {

namespace ibd {
constexpr int kD = 128, kTile = 128;                                  // dims; keys or (query, head) rows of a tile
constexpr uint32_t kChunk = kTile * 128, kTileBytes = 2 * kChunk;     // two chunks of 64 dims
constexpr uint32_t kSideBytes = 4096;                                 // beside a walked tile: its gradients (kQueries: up to eight queries' 128 keys) or head weights
constexpr int kStages = 4, kSlots = 3;                                // walked tiles in shared memory; Z and dZ in tensor memory
constexpr int kMaxSteps = 1024;                                       // tiles an item may walk
constexpr int kWorkers = 4 * kSlots, kLoadWarp = kWorkers, kZWarp = kWorkers + 1, kMmaWarp = kWorkers + 2, kListWarp = kWorkers + 3, kThreads = (kWorkers + 4) * 32;
constexpr int kUsers = kWorkers + 3;
struct Steps {
  int item, count;               // item -1: no more
  int first, pad;                // tile `first` + step
  uint16_t step[kMaxSteps];
};
constexpr int kDwItems = 3;
constexpr uint32_t kOffRing = 2 * kTileBytes, kOffSide = kOffRing + kStages * kTileBytes;   // (two own tiles first)
constexpr uint32_t kOffBar = kOffSide + kStages * kSideBytes;
constexpr uint32_t kOffDw = kOffBar + 256;                            // sums of 128 rows by the groups, of three items
constexpr uint32_t kOffSteps = kOffDw + kDwItems * kSlots * kTile * 4;
constexpr uint32_t kSmemBytes = kOffSteps + 2 * sizeof(Steps);
constexpr uint32_t kColZ = 0, kColAcc = kSlots * kTile, kTmemCols = 512;      // three of Z (dZ takes the first 64 columns of its own), the sum
static_assert(kSmemBytes <= 232448, "shared memory per CTA");

// Contiguous global -> shared copy (16-byte aligned addresses, size a multiple of 16); its bytes count on the barrier.
__device__ __forceinline__ void bulk_load(uint32_t smem_dst, const void* src, uint32_t bytes, uint32_t mbar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_dst), "l"(src), "r"(bytes), "r"(mbar)
               : "memory");
}

// Adds four fp32 values (given as bits) to 16-byte aligned global memory.
__device__ __forceinline__ void red_add_v4(float* dst, uint32_t a, uint32_t b, uint32_t c, uint32_t e) {
  asm volatile("red.relaxed.gpu.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(dst), "f"(__uint_as_float(a)), "f"(__uint_as_float(b)),
               "f"(__uint_as_float(c)), "f"(__uint_as_float(e))
               : "memory");
}

// Four lanes' four 16-byte pieces transposed: piece j of lane l becomes piece l of lane j (within the lanes 4 i .. 4 i + 3).  Rows of which a
// lane has one each then leave in 64-byte pieces, eight rows per request instead of thirty-two.
__device__ __forceinline__ void quad_transpose(uint32_t* c, int lane) {
#pragma unroll
  for (int bit = 1; bit <= 2; bit <<= 1) {
    const bool up = lane & bit;
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      if (a & bit) continue;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        uint32_t &lo = c[4 * a + w], &hi = c[4 * (a + bit) + w];
        const uint32_t got = __shfl_xor_sync(0xffffffffu, up ? lo : hi, bit);
        lo = up ? got : lo;
        hi = up ? hi : got;
      }
    }
  }
}

struct Dense {
  const int* dirty;       // not 0: q, k or w hold what must not be multiplied by 0; nothing is done
  int* next;              // [2] items handed out so far
  const float* grad;      // G [B, S1, width]
  const uint8_t* flags;   // [B, S1, width / 128]
  int width, tiles;       // S2 rounded up to 128; width / 128
  int blocks;             // of a batch entry's queries
  int big, per_big, small, per_small;   // kKeys: a key tile's blocks are walked in `big` parts of per_big, then `small` ones of per_small
};
}  // namespace ibd

// -------------------------------------------------------------------------------------------------
// spread: block = (query, 8192 columns of G).  The blocks also look through q and w (each its query) and k (each its share of the rows).
// -------------------------------------------------------------------------------------------------
__global__ void __launch_bounds__(256)
    indexer_bwd_spread_kernel(const __grid_constant__ IndexerBwdParams p, float* G, uint8_t* flags, int* dirty, const int width, const int parts, const int k_units) {
  // bf16 infinities, NaN and values from 2^60 on (128 products of smaller ones stay finite)
  auto odd_pair = [](uint32_t w) { return (w & 0x7f80u) >= 0x5d80u || (w & 0x7f800000u) >= 0x5d800000u; };
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
    if (tid < p.N1) found |= !(fabsf(__ldg(p.w + bt * p.N1 + tid)) < 0x1p60f);
    const uint4* k = reinterpret_cast<const uint4*>(p.k);
    const int64_t last = min(static_cast<int64_t>(p.B) * p.S2 * 16, (bt + 1) * k_units);
    for (int64_t i = bt * k_units + tid; i < last; i += 256) found |= odd(__ldg(k + i));
  }
  if (found) *dirty = 1;
  __syncthreads();
  auto put = [&](int key, float g) {
    const int c = key - c0;
    if (key >= 0 && key < p.S2 && c >= 0 && c < n) {
      atomicAdd(&acc[c], g);   // (a key listed twice counts twice; of three entries the order is not fixed)
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
  constexpr int kMine = kTile / N1;   // queries of a block of rows
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t sOwn = smem_u32(smem), sRing = sOwn + kOffRing, sSide = sOwn + kOffSide;
  if (sOwn & 1023u) {
    if (threadIdx.x == 0) atomicCAS(p.status, kStatusOk, kStatusBadLayout);
    return;
  }
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kOffBar);
  uint64_t* full = bars;             // [4] count 1 + transaction bytes
  uint64_t* empty = bars + 4;        // [4] count 1: commit after the MMAs that read the stage
  uint64_t* own_full = bars + 8;     // [2] count 1 + transaction bytes
  uint64_t* own_free = bars + 10;    // [2] count 1: commit after an item's last Z
  uint64_t* dw_full = bars + 12;     // count kWorkers: an item's dw by group
  uint64_t* acc_free = bars + 13;    // count 4: the sum has been read
  uint64_t* z_full = bars + 14;      // [3] count 1: commit after Z
  uint64_t* dz_full = bars + 17;     // [3] count 4: dZ is in tensor memory
  uint64_t* dz_free = bars + 20;     // [3] count 1: commit after the MMAs that read dZ
  uint64_t* list_full = bars + 23;   // [2] count 1
  uint64_t* list_free = bars + 25;   // [2] count kUsers
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 27);
  int* start_status = reinterpret_cast<int*>(bars + 28);
  float* s_dw = reinterpret_cast<float*>(smem + kOffDw);
  Steps* lists = reinterpret_cast<Steps*>(smem + kOffSteps);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (*d.dirty) return;
  if (tid == 0) {
    *start_status = *reinterpret_cast<volatile int*>(p.status);
    for (int i = 0; i < kStages; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
    for (int i = 0; i < kSlots; ++i) { mbar_init(&z_full[i], 1); mbar_init(&dz_full[i], 4); mbar_init(&dz_free[i], 1); }
    mbar_init(dw_full, kWorkers); mbar_init(acc_free, 4);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&own_full[i], 1); mbar_init(&own_free[i], 1);
      mbar_init(&list_full[i], 1); mbar_init(&list_free[i], kUsers);
    }
    mbar_init_fence();
  }
  if constexpr (kOwner == kKeys) {
    // a block's rows may end before its tile: what the stage held before is multiplied by 0, so it has to be finite
    for (int i = tid; i < kStages * kTile; i += kThreads) reinterpret_cast<float*>(smem + kOffSide + i / kTile * kSideBytes)[i % kTile] = 0.f;
    fence_proxy_async_smem();
  }
  if (warp == kMmaWarp) { tmem_alloc(tmem_slot, kTmemCols); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  bool ok = *start_status == kStatusOk;
  auto wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity, p.status)) != 0; };
  // two at once: the answer of a barrier takes 200 clocks and more on a busy shared memory
  auto wait_both = [&](uint64_t* a, uint32_t parity_a, uint64_t* b, uint32_t parity_b, bool b_needed) {
    const bool got_a = mbar_try_wait(a, parity_a), got_b = !b_needed || mbar_try_wait(b, parity_b);
    return __all_sync(0xffffffffu, got_a && got_b) || (wait(a, parity_a) && (!b_needed || wait(b, parity_b)));
  };
  auto use = [](int n) { return static_cast<uint32_t>(n >> 1) & 1u; };           // parity of the n-th use of one of two
  auto before = [](int n) { return (static_cast<uint32_t>(n >> 1) + 1u) & 1u; }; // of the use before it
  // step g of all items: its stage and its slot, and the parity of their use number g / count (the one before it: ^ 1)
  auto stage_of = [](int g) { return g % kStages; };
  auto lap = [](int g) { return static_cast<uint32_t>(g / kStages) & 1u; };
  auto slot_of = [](int g) { return g % kSlots; };
  auto turn = [](int g) { return static_cast<uint32_t>(g / kSlots) & 1u; };
  auto done_with = [&](int n) {
    __syncwarp();
    if (lane == 0) mbar_arrive(&list_free[n & 1]);
  };
  const int per_batch = kOwner == kQueries ? d.blocks : d.tiles * (d.big + d.small), items = p.B * per_batch;
  // an item's batch entry, and the block of rows or the key tile that it owns
  auto batch_of = [&](int item) { return item / per_batch; };
  auto owned = [&](int item) {
    const int i = item % per_batch, most = d.tiles * d.big;
    return kOwner == kQueries ? i : i < most ? i / d.big : (i - most) / d.small;
  };

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
      int first = 0, last = d.tiles;
      if constexpr (kOwner == kKeys) {
        const int i = item % per_batch, most = d.tiles * d.big;
        if (i < most) {
          first = i % d.big * d.per_big;
          last = first + d.per_big;
        } else {
          first = d.big * d.per_big + (i - most) % d.small * d.per_small;
          last = min(d.blocks, first + d.per_small);
        }
      }
      const uint8_t* flags = d.flags + static_cast<int64_t>(b) * p.S1 * d.tiles;
      int count = 0;
      for (int s0 = first; s0 < last; s0 += 32) {
        const int s = s0 + lane, tile = kOwner == kQueries ? s : own, block = kOwner == kQueries ? own : s;
        uint32_t any = 0;
        if (s < last) {
#pragma unroll
          for (int k = 0; k < kMine; ++k) any |= __ldg(flags + static_cast<int64_t>(min(block * kMine + k, p.S1 - 1)) * d.tiles + tile);
        }
        const uint32_t bits = __ballot_sync(0xffffffffu, any != 0);
        if (any) list.step[count + __popc(bits & ((1u << lane) - 1))] = static_cast<uint16_t>(s - first);
        count += __popc(bits);
      }
      if (!count) {
        if (kOwner == kQueries) {   // rows without a key: zeros
          const int rows = min(kTile, (p.S1 - own * kMine) * N1);
          const int64_t row0 = (static_cast<int64_t>(b) * p.S1 + own * kMine) * N1;
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
        list.first = first;
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
    int g = 0, n = 0;   // steps and own tiles asked for
    while (ok) {
      if (!wait(&list_full[n & 1], use(n))) { ok = false; break; }
      const Steps& list = lists[n & 1];
      const int item = list.item;
      if (item < 0) break;
      const int b = batch_of(item), own = owned(item), count = list.count;
      const int q_row0 = b * p.S1 * N1, k_row0 = b * p.S2, own_row0 = kOwner == kQueries ? q_row0 : k_row0, walk_row0 = kOwner == kQueries ? k_row0 : q_row0;
      const int own_queries = min(kMine, p.S1 - own * kMine);   // (kQueries)
      if (n >= 2 && !wait(&own_free[n & 1], before(n))) { ok = false; break; }
      if (lane == 0) {
        mbar_arrive_expect_tx(&own_full[n & 1], kTileBytes);
        for (int c = 0; c < 2; ++c)
          tma_load_2d(sOwn + (n & 1) * kTileBytes + c * kChunk, own_map, smem_u32(&own_full[n & 1]), c * 64, own_row0 + own * kTile);
      }
      __syncwarp();
      for (int i = 0; i < count; ++i, ++g) {
        const int s = stage_of(g);
        if (g >= kStages && !wait(&empty[s], lap(g) ^ 1u)) { ok = false; break; }
        if (lane == 0) {
          const int tile = list.first + list.step[i];
          const uint32_t bar = smem_u32(&full[s]), side = sSide + s * kSideBytes;
          // beside a key tile the gradients of the own block's queries, beside a block of rows their head weights
          const uint32_t side_bytes = kOwner == kQueries ? static_cast<uint32_t>(own_queries) * kTile * 4u : static_cast<uint32_t>(min(kTile, p.S1 * N1 - tile * kTile)) * 4u;
          mbar_arrive_expect_tx(&full[s], kTileBytes + side_bytes);
          for (int c = 0; c < 2; ++c) tma_load_2d(sRing + s * kTileBytes + c * kChunk, walk_map, bar, c * 64, walk_row0 + tile * kTile);
          if constexpr (kOwner == kQueries) {
            for (int k = 0; k < own_queries; ++k)
              bulk_load(side + k * kTile * 4, d.grad + (static_cast<int64_t>(b) * p.S1 + own * kMine + k) * d.width + tile * kTile, kTile * 4, bar);
          } else {
            bulk_load(side, p.w + static_cast<int64_t>(q_row0) + tile * kTile, side_bytes, bar);
          }
        }
        __syncwarp();
      }
      if (!ok) { ++n; break; }
      done_with(n++);
    }
    // given up: the copies in flight land before the shared memory goes
    auto landed = [&](uint64_t* bar, uint32_t parity) { for (int tries = 0; tries < (1 << 16) && !mbar_try_wait(bar, parity); ++tries) {} };
    for (int i = max(g - kStages, 0); !ok && i < g; ++i) landed(&full[stage_of(i)], lap(i));
    for (int i = max(n - 2, 0); !ok && i < n; ++i) landed(&own_full[i & 1], use(i));
  } else if (warp == kZWarp) {
    // ================================ MMA issuer of Z (converged, one elected lane issues) ==========
    constexpr uint32_t idesc = make_idesc_f16(true, kTile, kTile, 0, 0);
    const uint32_t go = elect_one_lane(), tmem = __reduce_or_sync(0xffffffffu, tmem_base);
    int g = 0;
    for (int n = 0; ok; ++n) {
      if (!wait(&list_full[n & 1], use(n))) { ok = false; break; }
      const int count = __reduce_or_sync(0xffffffffu, lists[n & 1].item < 0 ? 0u : static_cast<uint32_t>(lists[n & 1].count));
      if (!count) break;
      if (!wait(&own_full[n & 1], use(n))) { ok = false; break; }
      const uint64_t da = make_smem_desc(sOwn + (n & 1) * kTileBytes, 16, 1024, kSwizzle128B);
      for (int i = 0; i < count; ++i, ++g) {
        const int s = stage_of(g), slot = slot_of(g);
        if (!wait_both(&full[s], lap(g), &dz_free[slot], turn(g) ^ 1u, g >= kSlots)) { ok = false; break; }
        tc_fence_after();
        const uint64_t db = make_smem_desc(sRing + s * kTileBytes, 16, 1024, kSwizzle128B);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const uint32_t at = (k >> 2) * (kChunk >> 4) + 2 * (k & 3);
          umma_ss_if(go, tmem + kColZ + slot * kTile, da + at, db + at, idesc, k != 0);
        }
        umma_commit_if(go, &z_full[slot]);
      }
      if (!ok) break;
      umma_commit_if(go, &own_free[n & 1]);
      done_with(n);
    }
  } else if (warp == kMmaWarp) {
    // ================================ MMA issuer of the sums ========================================
    constexpr uint32_t idesc = make_idesc_f16(true, kTile, kD, 0, 1);
    const uint32_t go = elect_one_lane(), tmem = __reduce_or_sync(0xffffffffu, tmem_base);
    int g = 0;
    for (int n = 0; ok; ++n) {
      if (!wait(&list_full[n & 1], use(n))) { ok = false; break; }
      const int count = __reduce_or_sync(0xffffffffu, lists[n & 1].item < 0 ? 0u : static_cast<uint32_t>(lists[n & 1].count));
      if (!count) break;
      if (n >= 1 && !wait(acc_free, (n + 1) & 1)) { ok = false; break; }
      for (int i = 0; i < count; ++i, ++g) {
        const int s = stage_of(g), slot = slot_of(g);
        if (!wait(&dz_full[slot], turn(g))) { ok = false; break; }
        tc_fence_after();
        const uint64_t db = make_smem_desc(sRing + s * kTileBytes, kChunk, 1024, kSwizzle128B);   // the walked tile read MN-major: 128 dims, contraction over its rows
#pragma unroll
        for (int k = 0; k < 8; ++k)
          umma_ts_if(go, tmem + kColAcc, tmem + kColZ + slot * kTile + k * 8, db + k * (2048 >> 4), idesc, (i | k) != 0);
        umma_commit_if(go, &empty[s]);
        umma_commit_if(go, &dz_free[slot]);
      }
      if (!ok) break;
      done_with(n);
    }
  } else {
    // ================================ dZ and dw; the sums to global memory ==========================
    // Group = four warps = the steps of one slot; warp = a quarter of its lanes: own row or key 32 quarter + lane, all 128 walked columns.
    const int quarter = warp & 3, group = warp >> 2, row = quarter * 32 + lane;
    const uint32_t lane_base = static_cast<uint32_t>(quarter * 32) << 16;
    int g = 0;
    // The group of an item's last step reads the sums, while the others go on to the next item; it has its turn there last.
    for (int n = 0; ok; ++n) {
      if (!wait(&list_full[n & 1], use(n))) { ok = false; break; }
      const Steps& list = lists[n & 1];
      const int item = list.item;
      if (item < 0) break;
      const int b = batch_of(item), own = owned(item), count = list.count;
      // kKeys: this thread's gradients of a step, of its key for the queries of its columns (0 behind the last query)
      const float* grad = d.grad + static_cast<int64_t>(b) * p.S1 * d.width + own * kTile + row;
      auto gradients = [&](int i, float (&to)[kMine]) {
        const int query0 = (list.first + list.step[i]) * kMine;
#pragma unroll
        for (int k = 0; k < kMine; ++k) to[k] = query0 + k < p.S1 ? __ldg(grad + static_cast<int64_t>(query0 + k) * d.width) : 0.f;
      };
      const int first = (group + kSlots - g % kSlots) % kSlots;   // this group's first step of the item
      float next[kMine];
      if constexpr (kOwner == kKeys) {
        if (first < count) gradients(first, next);
      }
      // kQueries: the weight of this thread's row
      const int own_rows = min(kTile, (p.S1 - own * kMine) * N1);   // (kQueries)
      const float weight = kOwner == kQueries && row < own_rows ? __ldg(p.w + (static_cast<int64_t>(b) * p.S1 + own * kMine) * N1 + row) : 0.f;
      float2 dw = make_float2(0.f, 0.f), dw2 = make_float2(0.f, 0.f);
      for (int i = first; i < count; i += kSlots) {
        const int s = stage_of(g + i);
        float gr[kMine];
        if constexpr (kOwner == kKeys) {
#pragma unroll
          for (int k = 0; k < kMine; ++k) gr[k] = next[k];
          if (i + kSlots < count) gradients(i + kSlots, next);
        }
        if (!wait(&z_full[group], turn(g + i))) { ok = false; break; }
        tc_fence_after();
        const uint32_t z_at = tmem_base + kColZ + group * kTile + lane_base;
        uint32_t v[2][32];
        tmem_ld32(z_at, v[0]);
        // what came beside the tile (only now: before Z of this step, the stage may be a lap behind)
        ok = wait(&full[s], lap(g + i));   // (if not, this step still ends: a load is under way)
        // kQueries: the gradients of this row's query for its keys; kKeys: the weights of its columns
        const float4* side = reinterpret_cast<const float4*>(smem + kOffSide + s * kSideBytes) + (kOwner == kQueries ? row / N1 * (kTile / 4) : 0);
#pragma unroll
        for (int c = 0; c < 4; ++c) {   // dZ takes columns of Z that have been read
          uint32_t w[16];
          tmem_wait_ld();
          if (c < 3) tmem_ld32(z_at + (c + 1) * 32, v[(c + 1) & 1]);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float4 f = side[c * 8 + j];
            float z[4];
#pragma unroll
            for (int m = 0; m < 4; ++m) z[m] = __uint_as_float(v[c & 1][4 * j + m]);
            float2 lo = make_float2(f.x, f.y), hi = make_float2(f.z, f.w), scale;
            if constexpr (kOwner == kQueries) {
              dw = ffma2(lo, make_float2(fmaxf(z[0], 0.f), fmaxf(z[1], 0.f)), dw);
              dw2 = ffma2(hi, make_float2(fmaxf(z[2], 0.f), fmaxf(z[3], 0.f)), dw2);
              scale = make_float2(weight, weight);
            } else {
              scale = make_float2(gr[(32 * c + 4 * j) / N1], gr[(32 * c + 4 * j) / N1]);
            }
            lo = fmul2(lo, scale);
            hi = fmul2(hi, scale);
            w[2 * j] = pack2<true>(z[0] > 0.f ? lo.x : 0.f, z[1] > 0.f ? lo.y : 0.f);
            w[2 * j + 1] = pack2<true>(z[2] > 0.f ? hi.x : 0.f, z[3] > 0.f ? hi.y : 0.f);
          }
          tmem_st16(z_at + c * 16, w);
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&dz_full[group]);
        if (!ok) break;
      }
      if (!ok) break;
      g += count;
      done_with(n);
      // dw by group, in the order of their first steps (which group has which varies).  Three items' worth: the list
      // of n + 3 comes when every warp is done with that of n + 1, so behind its reading of n.
      float* dw_at = s_dw + (n % kDwItems) * kSlots * kTile + row;
      if constexpr (kOwner == kQueries) {
        dw_at[first * kTile] = (dw.x + dw.y) + (dw2.x + dw2.y);
        __syncwarp();
        if (lane == 0) mbar_arrive(dw_full);
      }
      if ((g - 1) % kSlots != group) continue;
      if (!wait(&dz_free[group], turn(g - 1))) { ok = false; break; }   // all MMAs up to the last step's are done
      tc_fence_after();
      auto read = [&] {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(acc_free);
      };
      const uint32_t acc = tmem_base + kColAcc + lane_base;
      if constexpr (kOwner == kQueries) {
        uint32_t o[kD / 2];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t v[32];
          tmem_ld32(acc + c * 32, v);
          tmem_wait_ld();
#pragma unroll
          for (int k = 0; k < 16; ++k) o[16 * c + k] = pack2<true>(__uint_as_float(v[2 * k]), __uint_as_float(v[2 * k + 1]));
        }
        if (!wait(dw_full, n & 1)) { ok = false; break; }
        float sum = dw_at[0];
        for (int k = 1; k < kSlots; ++k) sum += dw_at[k * kTile];
        read();
        const int64_t row0 = (static_cast<int64_t>(b) * p.S1 + own * kMine) * N1;
        if (row < own_rows) p.d_w[row0 + row] = sum;
        uint4* dq = reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(p.d_q) + (row0 + (row & ~3)) * kD) + (lane & 3);
#pragma unroll
        for (int h = 0; h < 4; ++h) {   // 32 dims
          quad_transpose(o + 16 * h, lane);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if ((row & ~3) + j < own_rows) dq[j * (kD / 8) + 4 * h] = make_uint4(o[16 * h + 4 * j], o[16 * h + 4 * j + 1], o[16 * h + 4 * j + 2], o[16 * h + 4 * j + 3]);
        }
      } else {
        const int row4 = own * kTile + (row & ~3);
        float* dk = p.d_k + (static_cast<int64_t>(b) * p.S2 + row4) * kD + 4 * (lane & 3);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t v[32];
          tmem_ld32(acc + c * 32, v);
          tmem_wait_ld();
          if (c == 3) read();
#pragma unroll
          for (int h = 0; h < 2; ++h) {   // 16 dims
            uint32_t* u = v + 16 * h;
            quad_transpose(u, lane);
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (row4 + j < p.S2) red_add_v4(dk + j * kD + c * 32 + 16 * h, u[4 * j], u[4 * j + 1], u[4 * j + 2], u[4 * j + 3]);
          }
          __syncwarp();
        }
      }
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
  const long long items = static_cast<long long>(p.B) * (kOwner == kQueries ? d.blocks : d.tiles * (d.big + d.small));
  kern<<<static_cast<unsigned>(items < sms ? items : sms), ibd::kThreads, ibd::kSmemBytes, stream>>>(p, d, q_map, k_map);
  return static_cast<int>(cudaGetLastError());
}
template <int N1>
int launch_both(const IndexerBwdParams& p, const ibd::Dense& d, const CUtensorMap& q_map, const CUtensorMap& k_map, int dev, int sms, cudaStream_t stream) {
  const int err = launch_owner<kQueries, N1>(p, d, q_map, k_map, dev, sms, stream);
  return err ? err : launch_owner<kKeys, N1>(p, d, q_map, k_map, dev, sms, stream);
}
}  // namespace

// Which kernel: the other one takes about 100 ps per (query, listed key), whatever the heads; these take 8 ps per (query, key that it may see) for
// G, 42 more with 64 heads, half and a quarter of that with 32 and 16, and 30 us for three more launches.  Both counts as they are
// in a causal step (keys up to S2 - S1 + t) with full lists.  Measured, other / these, us (queries x keys, list): 64 heads: 4096 x 4096, 2048:
// 674 / 459, 1024: 416 / 459; 4096 x 8192, 2048: 862 / 1206; 1024 x 4096, 2048: 233 / 238; 32 heads: 2048 x 2048, 2048: 258 / 119; 4096 x 8192,
// 2048: 854 / 625; 16 heads: 4096 x 4096, 512: 260 / 184; 4096 x 1024, 512: 262 / 122.  fp16 stays with the other kernel: its range needs a
// scale per query.
static bool dense_preferred(const IndexerBwdParams& p, bool bf16) {
  if (!bf16 || p.D != ibd::kD || (p.N1 != 16 && p.N1 != 32 && p.N1 != 64)) return false;
  const long long B = p.B, S1 = p.S1, S2 = p.S2, K = p.K < p.S2 ? p.K : p.S2;
  if (B * S1 * padded_width(p) > (1LL << 28) || padded_width(p) / ibd::kTile > ibd::kMaxSteps || B * S1 * p.N1 >= (1LL << 30) || B * S2 >= (1LL << 30)) return false;
  const long long seen = S1 <= S2 ? S1 * (2 * S2 - S1 + 1) / 2 : S1 * S2;
  const long long first = S2 - S1 + 1;   // keys that query 0 may see
  const long long shorter = S1 > S2 || first >= K ? 0 : (K - first < S1 ? K - first : S1);   // queries that see fewer than K
  const long long listed = S1 * K - (shorter ? shorter * (2 * K - 2 * first - shorter + 1) / 2 : 0);
  return B * listed * 100 > B * seen * (8 + 42 * p.N1 / 64) + 30 * 1000 * 1000;
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
  const uintptr_t bases = reinterpret_cast<uintptr_t>(p.w) | reinterpret_cast<uintptr_t>(p.d_q) | reinterpret_cast<uintptr_t>(p.d_k);
  return dense_preferred(p, bf16) && (bases & 15u) == 0 && encode_tiled_fn() != nullptr;
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
  const int queries = kTile / p.N1;   // per block of 128 rows
  d.blocks = (p.S1 + queries - 1) / queries;
  // A key tile's blocks in parts, as many as make about six items per SM; the last quarter of them in smaller ones, handed out last, so
  // that the SMs end together (all of one size, eight per SM: 224 us; so 212, with four per SM 240, with half of them small 232).
  int parts_of_tile = (6 * sms + p.B * d.tiles - 1) / (p.B * d.tiles);
  if (parts_of_tile > d.blocks) parts_of_tile = d.blocks;
  d.per_big = (d.blocks + parts_of_tile - 1) / parts_of_tile;
  if (d.per_big > kMaxSteps) d.per_big = kMaxSteps;
  d.big = 3 * (d.blocks / 4) / d.per_big;
  d.per_small = (d.per_big + 3) / 4;
  d.small = (d.blocks - d.big * d.per_big + d.per_small - 1) / d.per_small;
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
