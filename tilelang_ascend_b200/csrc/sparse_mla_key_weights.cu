// Attention weights of the listed keys, averaged over the heads (sm_100a, tcgen05):
//
//   w[b, t, j] = 1/H sum_h exp(sm_scale q[b, t, h] . kv[b, idx_j] - lse[b, t, h])        0 for entries that take no part
//
// what the sparse MLA forward's softmax gives each key of a query's list; the forward keeps only its normaliser (lse).
//
// Bound by the tensor cores on paper (2 H D operations against 2 D gathered bytes per key), by shared memory in practice: a
// tile of 128 keys x 576 dims is written once (1152 clocks of the SM's 128 B/clk) and read once by the MMAs that take 2304 clocks.
// So the other operand must not come from there: S = Q K^T with A = the query's 128 heads, eight of their 64-dim chunks in tensor
// memory (256 columns, beside two score accumulators of 128), the rest in shared memory, B = the gathered keys.  (With the
// heads in shared memory too -- transposed product, a key per lane and no exchange in the sum over heads -- a tile's operands
// take 3456 clocks of shared memory and leave room for five stages of the ring: 1093 us for 4096 queries of 2048 keys x 128 heads.)
// Persistent CTAs, one per SM, long (late) queries first.  A query's heads ride the ring ahead of its keys and are moved to
// tensor memory by the epilogue warps as soon as the last MMAs of the query before are done, so that the gather never stops.
// Warps: 8 epilogue (quarter of the heads x half of the keys), 8 gather, the MMA issuer, and one that reads the next query's list.
// Shuffles, copies and barriers share one pipe, so the sum over heads uses few: a thread takes four heads of the same keys out of
// tensor memory and seven shuffles join 32 keys over a warp (one head per thread: 31; with that the epilogue took 3600 of the 2304
// clocks that a tile's MMAs take, and the copies waited behind it: 848 us).
// The exponentials are the hardware's ex2.approx of fp32 arguments: the weights are within 6e-7 of the definition (1e-7 with an exact
// exponential), far inside what bf16 or fp16 queries and keys carry.
// Measured there: 812 us, 1140 TFLOP/s.  A tile takes about 3200 clocks and a change of queries about 6000; what shares the tile's time is shared
// memory: without the copies 650 us, without the epilogue 755.
#include <type_traits>

#include "fwd_common.cuh"
#include "launch_util.h"

namespace dsa {

namespace kw {
constexpr int kKeys = 128;                        // keys per tile = UMMA N
constexpr int kHeads = 128;                       // heads per pass over the list = UMMA M
constexpr uint32_t kChunkBytes = 128 * 128;       // 128 keys (or heads) x 64 dims
constexpr int kTmemChunks = 8;                    // chunks of the heads in tensor memory
constexpr int kPerStage = 3;                       // chunks of a stage of the ring
constexpr uint32_t kStageBytes = kPerStage * kChunkBytes;
constexpr int kMaxStages = 4;
constexpr int kMaxWords = 8192 / 32;              // validity bits of a list
constexpr int kEpilogueWarps = 8, kGatherWarps = 8, kMmaWarp = 16, kListWarp = 17, kThreads = 18 * 32;
constexpr int kUsers = kEpilogueWarps + kGatherWarps + 1;   // warps that read a list
constexpr uint32_t kOffBits = 512;                              // after the barriers: two lists
constexpr uint32_t kListBytes = kMaxWords * 4 + 16 + kMaxWords / 4;   // validity bits; number of tiles with a key; those tiles
constexpr uint32_t kOffPart = kOffBits + 2 * kListBytes;        // two tiles' sums of the four quarters
constexpr uint32_t kFixedBytes = kOffPart + 2 * 4 * kKeys * 4;
constexpr uint32_t kMaxSmem = 232448;
constexpr uint32_t kColS = kTmemChunks * 32, kTmemCols = 512;
static_assert(kColS + 2 * kKeys <= kTmemCols, "tensor memory columns");
struct Shape {
  int chunks, parts;         // 64-dim chunks of a row; stages that a row tile passes through
  int smem_chunks, stages;   // chunks of the heads in shared memory; stages of the ring
};

// Position in the ring.
struct Ring {
  int stage = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next(int stages) {
    if (++stage == stages) { stage = 0; phase ^= 1u; }
  }
  __device__ __forceinline__ void skip(int n, int stages) {
    stage += n;
    while (stage >= stages) { stage -= stages; phase ^= 1u; }
  }
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
  const uint32_t sK = sQ + sh.smem_chunks * kChunkBytes;
  uint8_t* fixed = smem + sh.smem_chunks * kChunkBytes + sh.stages * kStageBytes;
  uint64_t* k_full = reinterpret_cast<uint64_t*>(fixed);   // [kMaxStages] count 128: a gather group's copies have landed
  uint64_t* k_empty = k_full + kMaxStages;                 // [kMaxStages] count 1: commit after the MMAs that read the stage, or the heads have been moved on
  uint64_t* acc_full = k_empty + kMaxStages;               // [2] count 1: commit after a tile's last MMA
  uint64_t* acc_free = acc_full + 2;                       // [2] count 8: the epilogue warps have read the scores
  uint64_t* q_ready = acc_free + 2;                        // count 8: a pass's heads are in place
  uint64_t* list_full = q_ready + 1;                       // [2] count 1
  uint64_t* list_free = list_full + 2;                     // [2] count kUsers
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(list_free + 2);
  int* start_status = reinterpret_cast<int*>(tmem_slot + 1);
  float* s_part = reinterpret_cast<float*>(fixed + kOffPart);
  auto bits_of = [&](int item) { return reinterpret_cast<uint32_t*>(fixed + kOffBits + (item & 1) * kListBytes); };
  auto tiles_of = [&](int item) { return fixed + kOffBits + (item & 1) * kListBytes + kMaxWords * 4 + 16; };

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int n = p.B * p.S, tiles = (p.topk + kKeys - 1) / kKeys;
  const int passes = (p.H + kHeads - 1) / kHeads;
  // items of this CTA: queries n - 1 - blockIdx.x, then every gridDim.x-th before it
  const int items = (n - static_cast<int>(blockIdx.x) + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x);
  auto query_of = [&](int item) { return n - 1 - static_cast<int>(blockIdx.x) - item * static_cast<int>(gridDim.x); };

  if (tid == 0) {
    *start_status = *reinterpret_cast<volatile int*>(p.status);
    for (int i = 0; i < sh.stages; ++i) { mbar_init(&k_full[i], kGatherWarps * 16); mbar_init(&k_empty[i], 1); }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1); mbar_init(&acc_free[i], kEpilogueWarps);
      mbar_init(&list_full[i], 1); mbar_init(&list_free[i], kUsers);
    }
    mbar_init(q_ready, kEpilogueWarps);
    mbar_init_fence();
  }
  if (warp == kMmaWarp) { tmem_alloc(tmem_slot, kTmemCols); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  bool ok = *start_status == kStatusOk;
  auto wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity, p.status)); };
  if (warp == kListWarp) {
    // ================================ lists: validity bits, one query ahead =========================
    for (int item = 0; ok && item < items; ++item) {
      if (item >= 2 && !wait(&list_free[item & 1], ((item >> 1) + 1) & 1)) { ok = false; break; }
      const RowCtx c = make_row_ctx(p, query_of(item));
      uint32_t* bits = bits_of(item);
      uint8_t* list = tiles_of(item);
      uint32_t count = 0;
      for (int t0 = 0; t0 < tiles; t0 += 4) {   // four tiles' indices on their way at once
        int idx[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int j = t0 * kKeys + i * 32 + lane;
          idx[i] = j < p.topk ? __ldg(c.idx_row + j) : -1;
        }
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          uint32_t any = 0;
#pragma unroll
          for (int i = 4 * t; i < 4 * t + 4; ++i) {
            const uint32_t b = __ballot_sync(0xffffffffu, c.active && index_valid(c, idx[i]));
            if (lane == 0 && t0 + t < tiles) bits[t0 * 4 + i] = b;
            any |= b;
          }
          if (any) {
            if (lane == 0) list[count] = static_cast<uint8_t>(t0 + t);
            ++count;
          }
        }
      }
      if (lane == 0) {
        bits[kMaxWords] = count;
        mbar_arrive(&list_full[item & 1]);
      }
      __syncwarp();
    }
  } else if (warp >= kEpilogueWarps && warp < kMmaWarp) {
    // ================================ gather: 32 rows of every other stage per warp =================
    // Two groups of four warps take alternate stages: waiting for a stage, announcing it and the loop around cost a warp as much as
    // twelve copies.
    const int group = (warp - kEpilogueWarps) >> 2, row0 = ((warp - kEpilogueWarps) & 3) * 32 + (lane >> 3), unit = lane & 7;   // rows row0 + 4 i
    const T* none = reinterpret_cast<const T*>(p.kv);
    Ring ring;
    ring.phase = 1;   // (the first round of the ring finds its stages empty)
    ring.skip(group, sh.stages);
    int turn = group;   // stages until this group's next one
    // eight rows per thread, stage by stage (base: this thread's unit of row 0's first chunk; row -1: zeros)
    auto load_rows = [&](const T* base, const int (&row)[8]) {
      for (; turn < sh.parts; turn += 2) {
        if (!wait(&k_empty[ring.stage], ring.phase)) return false;
#pragma unroll
        for (int c = 0; c < kPerStage; ++c) {
          const int ch = turn * kPerStage + c;
          if (ch < sh.chunks) {
            const bool dims = ch * 64 + unit * 8 < p.D;
            const uint32_t dst = sK + ring.stage * kStageBytes + c * kChunkBytes;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const bool copy = dims && row[i] >= 0;
              cp_async16(dst + sw128_offset(row0 + 4 * i, unit), copy ? base + static_cast<int64_t>(row[i]) * p.D + ch * 64 : none, copy ? 16u : 0u);
            }
          }
        }
        cp_async_arrive_noinc(&k_full[ring.stage]);
        ring.skip(2, sh.stages);
      }
      turn -= sh.parts;
      return true;
    };
    for (int item = 0; ok && item < items; ++item) {
      if (!wait(&list_full[item & 1], (item >> 1) & 1)) { ok = false; break; }
      const uint32_t* bits = bits_of(item);
      const uint8_t* list = tiles_of(item);
      const int count = bits[kMaxWords];
      if (count) {
        const int bt = query_of(item);
        const RowCtx c = make_row_ctx(p, bt);
        const T* kv = reinterpret_cast<const T*>(p.kv) + static_cast<int64_t>(c.b) * p.S_kv * p.D + unit * 8;
        const T* q = reinterpret_cast<const T*>(p.q) + static_cast<int64_t>(bt) * p.H * p.D + unit * 8;
        auto indices = [&](int i, int (&row)[8]) {   // of the list's tile number i
          const int slot0 = list[i] * kKeys + row0;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const int slot = slot0 + 4 * k, idx = slot < p.topk ? __ldg(c.idx_row + slot) : -1;
            row[k] = index_valid(c, idx) ? idx : -1;
          }
        };
        for (int pass = 0; ok && pass < passes; ++pass) {
          int row[8], next[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int h = pass * kHeads + row0 + 4 * i;
            row[i] = h < p.H ? h : -1;
          }
          indices(0, next);
          ok = load_rows(q, row);
          for (int i = 0; ok && i < count; ++i) {
#pragma unroll
            for (int k = 0; k < 8; ++k) row[k] = next[k];
            if (i + 1 < count) indices(i + 1, next);   // one tile ahead of its copies
            ok = load_rows(kv, row);
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&list_free[item & 1]);
    }
    cp_async_wait<0>();
  } else if (warp == kMmaWarp) {
    // ================================ MMA issuer (converged, one elected lane issues) ===============
    constexpr uint32_t idesc = make_idesc_f16(kBF16, kHeads, kKeys, 0, 0);
    const uint32_t go = elect_one_lane();
    // (a reduction's result is known to be the same in all lanes, a word from shared memory is not: the operands of an MMA are uniform
    // registers, and moving them there one by one cost more than the MMA)
    const uint32_t tmem = __reduce_or_sync(0xffffffffu, tmem_base);
    Ring ring;
    int g = 0, loads = 0;   // tiles and passes so far
    // The next stage and the next accumulator are looked at in the middle of a stage's MMAs (the answer of a barrier takes 200 clocks on
    // this busy shared memory, the fence 50 to 100); `yes`: it was complete, and what it announces has been fenced.
    auto look = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_try_wait(bar, parity)) != 0; };
    auto fence = [&]() {
      fence_proxy_async_smem();   // the rows were written by cp.async of other threads
      tc_fence_after();
    };
    for (int item = 0; ok && item < items; ++item) {
      if (!wait(&list_full[item & 1], (item >> 1) & 1)) { ok = false; break; }
      const int count = __reduce_or_sync(0xffffffffu, bits_of(item)[kMaxWords]);
      for (int pass = 0; ok && count && pass < passes; ++pass) {
        ring.skip(sh.parts, sh.stages);   // the heads' slots are the epilogue warps'
        if (!wait(q_ready, loads & 1)) { ok = false; break; }
        ++loads;
        bool full = false, room = g < 2;
        for (int i = 0; ok && i < count; ++i) {
          const int a = g & 1;
          if (!room) {
            if (!wait(&acc_free[a], ((g >> 1) + 1) & 1)) { ok = false; break; }
            tc_fence_after();   // (the stage may have been seen, and fenced, before)
          }
          const uint32_t acc = tmem + kColS + a * kKeys;
          room = g < 1;   // the tile after this one
          for (int part = 0; part < sh.parts; ++part) {
            if (!full) {
              if (!wait(&k_full[ring.stage], ring.phase)) { ok = false; break; }
              fence();
            }
            Ring after = ring;
            after.next(sh.stages);
            const uint64_t db = make_smem_desc(sK + ring.stage * kStageBytes, 16, 1024, kSwizzle128B);
#pragma unroll
            for (int c = 0; c < kPerStage; ++c) {
              const int ch = part * kPerStage + c;
              if (ch < kTmemChunks && ch < sh.chunks) {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                  umma_ts_if(go, acc, tmem + (ch * 4 + k) * 8, db + ((c * kChunkBytes + k * 32) >> 4), idesc, (ch | k) != 0);
              } else if (ch < sh.chunks) {
                const uint64_t da = make_smem_desc(sQ + (ch - kTmemChunks) * kChunkBytes, 16, 1024, kSwizzle128B);
#pragma unroll
                for (int k = 0; k < 4; ++k) umma_ss_if(go, acc, da + 2 * k, db + ((c * kChunkBytes + k * 32) >> 4), idesc, 1);
              }
              if (c == 1) {
                // (the last stage of a pass is followed by heads, which are not this warp's)
                full = (part + 1 < sh.parts || i + 1 < count) && look(&k_full[after.stage], after.phase);
                if (part + 1 == sh.parts && !room) room = look(&acc_free[(g + 1) & 1], (((g + 1) >> 1) + 1) & 1);
                if (full) fence();
              }
            }
            umma_commit_if(go, &k_empty[ring.stage]);
            ring = after;
          }
          if (!ok) break;
          umma_commit_if(go, &acc_full[a]);
          ++g;
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&list_free[item & 1]);
    }
  } else {
    // ================================ heads to tensor memory; epilogue ==============================
    const int quarter = warp & 3, half = warp >> 2, row = quarter * 32 + lane;   // this thread's head and half of the keys
    const uint32_t lane_base = static_cast<uint32_t>(quarter * 32) << 16;
    const float inv_h = 1.f / static_cast<float>(p.H);
    Ring ring;
    // The heads of a pass: the two halves take alternate chunks out of the ring.  All MMAs that read the heads before are done: every
    // warp has seen the commit of the last of them.
    auto move_heads = [&](bool go) {
      for (int part = 0; part < sh.parts; ++part) {
        go = go && wait(&k_full[ring.stage], ring.phase);
#pragma unroll 1
        for (int c = 0; c < kPerStage; ++c) {
          const int ch = part * kPerStage + c;
          if ((ch & 1) != half || ch >= sh.chunks) continue;
          const uint32_t src = sK + ring.stage * kStageBytes + c * kChunkBytes;
          uint32_t w[32];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const uint4 v = ld_shared_v4(src + sw128_offset(row, j));
            w[4 * j] = v.x; w[4 * j + 1] = v.y; w[4 * j + 2] = v.z; w[4 * j + 3] = v.w;
          }
          if (ch < kTmemChunks) {
            if (go) tmem_st32(tmem_base + lane_base + ch * 32, w);
          } else {
            const uint32_t dst = sQ + (ch - kTmemChunks) * kChunkBytes;
#pragma unroll
            for (int j = 0; j < 8; ++j) st_shared_v4(dst + sw128_offset(row, j), w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
          }
        }
        named_bar_sync(1, kEpilogueWarps * 32);   // all warps have read the stage
        if (tid == 0 && go) mbar_arrive(&k_empty[ring.stage]);
        ring.next(sh.stages);
      }
      tmem_wait_st();
      fence_proxy_async_smem();
      tc_fence_before();
      __syncwarp();
      if (lane == 0 && go) mbar_arrive(q_ready);
      return go;
    };
    // Normalisers of this thread's four heads, in log2 units; a head without any key has lse = -inf: no weight (neither have the rows
    // that pad the heads).
    auto load_lse = [&](int bt, int pass, float (&to)[4]) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int h = pass * kHeads + quarter * 32 + (lane >> 2) + 8 * i;
        const float l = h < p.H ? __ldg(p.lse + static_cast<int64_t>(bt) * p.H + h) : INFINITY;
        to[i] = l == -INFINITY ? INFINITY : l * 1.4426950408889634f;
      }
    };
    int g = 0;
    bool moved = false;      // the next pass's heads are in place already
    float lse[4] = {0.f, 0.f, 0.f, 0.f}, next_lse[4] = {0.f, 0.f, 0.f, 0.f};
    // (Every warp of the group takes the same turns through these loops, also when a wait has given up: the barriers inside count
    // them all.  Whether a list can be trusted is agreed on.)
    for (int item = 0; item < items; ++item) {
      ok = bar_and(1, kEpilogueWarps * 32, ok && wait(&list_full[item & 1], (item >> 1) & 1));
      if (!ok) break;
      const uint32_t* bits = bits_of(item);
      const int bt = query_of(item);
      float* out = weights + static_cast<int64_t>(bt) * p.topk;
      if (!bits[kMaxWords]) {
        for (int i = tid; i < p.topk; i += kEpilogueWarps * 32) out[i] = 0.f;
      } else {
        const uint8_t* list = tiles_of(item);
        const int count = bits[kMaxWords];
        // tiles without a key
        for (int tile = 0; tile < tiles; ++tile) {
          const int slot = tile * kKeys + tid;
          if (tid < kKeys && slot < p.topk && !(bits[4 * tile] | bits[4 * tile + 1] | bits[4 * tile + 2] | bits[4 * tile + 3])) out[slot] = 0.f;
        }
        for (int pass = 0; pass < passes; ++pass) {
          if (!moved) {
            load_lse(bt, pass, next_lse);
            ok = move_heads(ok);
          }
          moved = false;
#pragma unroll
          for (int k = 0; k < 4; ++k) lse[k] = next_lse[k];
          for (int i = 0; i < count; ++i) {
            const int slot = list[i] * kKeys + tid;   // (of the combining threads, tid < 128)
            const int a = g & 1;
            ok = ok && __all_sync(0xffffffffu, mbar_wait<true>(&acc_full[a], (g >> 1) & 1, p.status));
            tc_fence_after();   // ahead of the scores' loads and of the next heads' stores
            ring.skip(sh.parts, sh.stages);   // this tile's slots were the MMAs'
            if (i + 1 == count) {               // no MMA reads these heads any more: the next ones take their place before the epilogue
              if (pass + 1 < passes) {
                load_lse(bt, pass + 1, next_lse);
                ok = move_heads(ok);
                moved = true;
              } else if (item + 1 < items) {
                ok = bar_and(1, kEpilogueWarps * 32, ok && wait(&list_full[(item + 1) & 1], ((item + 1) >> 1) & 1));
                if (ok && bits_of(item + 1)[kMaxWords]) {
                  load_lse(query_of(item + 1), 0, next_lse);
                  ok = move_heads(ok);
                  moved = true;
                }
              }
            }
            // 32 keys at a time: this thread has two keys of every eight for four heads of its quarter, adds those up itself and ends, after
            // three halving exchanges with the lanes of the other heads, with the quarter's sum for one key.
            float* part = s_part + (a * 4 + quarter) * kKeys + half * 64;
#pragma unroll
            for (int grp = 0; grp < 2; ++grp) {
              uint32_t lo[16], hi[16];
              if (ok) {
                const uint32_t from = tmem_base + kColS + a * kKeys + half * 64 + grp * 32 + lane_base;
                tmem_ld_16x32(from, lo);
                tmem_ld_16x32(from + (16u << 16), hi);
                tmem_wait_ld();
              }
              if (grp == 1) {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&acc_free[a]);
              }
              float e[8];
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                const int r = 4 * (k >> 1) + (k & 1);
                e[k] = (exp2f(fmaf(__uint_as_float(lo[r]), p.scale_log2, -lse[0])) + exp2f(fmaf(__uint_as_float(lo[r + 2]), p.scale_log2, -lse[1]))) +
                       (exp2f(fmaf(__uint_as_float(hi[r]), p.scale_log2, -lse[2])) + exp2f(fmaf(__uint_as_float(hi[r + 2]), p.scale_log2, -lse[3])));
              }
#pragma unroll
              for (int o = 16; o >= 4; o >>= 1) {
                const bool upper = lane & o;
#pragma unroll
                for (int k = 0; k < o / 4; ++k) {
                  const float give = upper ? e[k] : e[k + o / 4], mine = upper ? e[k + o / 4] : e[k];
                  e[k] = mine + __shfl_xor_sync(0xffffffffu, give, o);
                }
              }
              part[grp * 32 + 8 * (lane >> 3) + 2 * (lane & 3) + ((lane >> 2) & 1)] = e[0];
            }
            named_bar_sync(1, kEpilogueWarps * 32);
            if (tid < kKeys && slot < p.topk && ok) {
              const float* q4 = s_part + a * 4 * kKeys + tid;
              const float sum = ((bits[slot >> 5] >> (slot & 31)) & 1u) ? ((q4[0] + q4[kKeys]) + (q4[2 * kKeys] + q4[3 * kKeys])) * inv_h : 0.f;
              out[slot] = pass ? out[slot] + sum : sum;
            }
            ++g;
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&list_free[item & 1]);
    }
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
  sh.parts = (sh.chunks + kw::kPerStage - 1) / kw::kPerStage;
  sh.smem_chunks = sh.chunks > kw::kTmemChunks ? sh.chunks - kw::kTmemChunks : 0;
  sh.stages = static_cast<int>((kw::kMaxSmem - kw::kFixedBytes - sh.smem_chunks * kw::kChunkBytes) / kw::kStageBytes);   // 4; 640 dims: 3
  const int smem = static_cast<int>(sh.smem_chunks * kw::kChunkBytes + sh.stages * kw::kStageBytes + kw::kFixedBytes);
  auto kern = bf16 ? sparse_mla_key_weights_kernel<true> : sparse_mla_key_weights_kernel<false>;
  if ((e = ensure_dynamic_smem(kern, dev, smem)) != cudaSuccess) return static_cast<int>(e);
  const long long n = static_cast<long long>(p.B) * p.S;
  kern<<<static_cast<unsigned>(n < sms ? n : sms), kw::kThreads, smem, stream>>>(p, weights, sh);
  return static_cast<int>(cudaGetLastError());
}

}  // namespace dsa
