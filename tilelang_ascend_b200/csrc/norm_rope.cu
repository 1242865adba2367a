// Norm of every head's row and rotation by its token's position, in one pass (sm_100a).
//
//   y = rot(norm(x))      norm over the leading norm_dim dims (none, RMS, layer; weight and bias shared by the heads),
//                         rotation of the dims [rope_start, rope_start + R), pairs (2i, 2i+1) or (i, i + R/2):
//                         (a, b) -> (a cos - b sin, b cos + a sin), angle = position * inv_freq[i]
//   backward: u = rot^T(dy); with n = (x - mean) rstd:  dweight = sum u n, dbias = sum u, g = u weight,
//             dx = rstd (g - mean(g n) n [- mean(g)])
//
// Bound by memory: a row is read once and written once.  A group of 8 lanes owns a row (above 576 dims: 16 lanes) and asks for all
// of it at once, up to nine 16-byte units per lane, so that a warp has four rows on their way and no lane is without a unit for the
// usual sizes (a warp per row left a quarter of its lanes idle at 576 dims and had one row on its way: 4096 tokens x 129 rows
// of 576 dims 264 us).  A block owns a tile of tokens x heads; the cosines and sines of its tokens are made once per block, the
// angle as an exact product reduced in 64 bits (a far position times a frequency has no fraction left in 32).
// That call takes 188 us now, 6.5 TB/s.  Short rows are bound by their instructions (390 per warp and four rows of 128 dims with a division
// per row and the lanes' angles in the same banks): forward and backward of 4096 tokens x 65 rows of 128 dims, layer norm on one of
// them, 96 us then, 74 now.
// Everything is computed in fp32 and rounded once, on the store.  The gradient of rows without a norm is the forward with the angles
// turned round.
//
// Rows that do not come in 16-byte units (odd sizes, offsets or strides) take the *_any kernels: a warp per row, one element
// at a time, the same arithmetic.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "launch_util.h"
#include "norm_rope.h"

namespace dsa {

namespace nr {
constexpr int kThreads = 256;
constexpr int kMaxPairs = 2048;      // (token, pair) angles a block keeps: 16 KB
constexpr int kMaxNormDim = 1024;    // widest row of the 16-byte kernels

// cos and sin of position * inv_freq (p.back: of its negative), times the rotation's scale.
__device__ __forceinline__ float2 turn_of(const NormRopeParams& p, long long position, float inv_freq) {
  const double angle = static_cast<double>(position) * static_cast<double>(inv_freq);
  const double turns = rint(angle * 0.15915494309189533577);          // 1 / 2 pi
  double r = fma(-turns, 6.283185307179586232, angle);                // 2 pi in two parts
  r = fma(-turns, 2.4492935982947064e-16, r);
  float s, c;
  sincosf(static_cast<float>(r), &s, &c);
  return make_float2(c * p.rope_scale, s * (p.back ? -p.rope_scale : p.rope_scale));
}

__device__ __forceinline__ long long position_of(const NormRopeParams& p, int token) {
  return p.positions64 ? static_cast<const long long*>(p.positions)[token] : static_cast<const int*>(p.positions)[token];
}

// A norm's weight or bias: fp32, or the rows' own type.
template <typename T>
__device__ __forceinline__ float param_at(const void* w, int fp32, int i) {
  return fp32 ? static_cast<const float*>(w)[i] : static_cast<float>(static_cast<const T*>(w)[i]);
}

template <typename T>
__device__ __forceinline__ void unpack8(const uint4& w, float (&v)[8]) {
  const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = static_cast<float>(e[j]);
}
template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&v)[8]) {
  uint4 w;
  T* e = reinterpret_cast<T*>(&w);
#pragma unroll
  for (int j = 0; j < 8; ++j) e[j] = static_cast<T>(v[j]);
  return w;
}
template <int G>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ uint4 ld_stream(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// Address of element 0 of row (token, head) of a strided [B, S, H, D] tensor.
template <typename T>
__device__ __forceinline__ const T* row_of(const RowView& v, int S, int token, int head) {
  const int b = token / S, s = token - b * S;
  return static_cast<const T*>(v.base) + b * v.stride_b + s * v.stride_s + head * v.stride_h;
}

// Row number the output of (token, head) goes to, -1: it is not written.
__device__ __forceinline__ long long out_row(const RopeSide& sd, int token, int head) {
  if (!sd.slots) return static_cast<long long>(token) * sd.H + head;
  const long long slot = sd.slots64 ? static_cast<const long long*>(sd.slots)[token] : static_cast<const int*>(sd.slots)[token];
  return slot >= 0 && slot < sd.y_slots ? slot * sd.H + head : -1;
}

// Where angle i of a token's `half` sits in shared memory: the 16-byte pieces (two angles) that make up a unit's angles -- four, or with
// interleaved pairs two -- lie apart, so that lanes with neighbouring units read neighbouring pieces.  (All of a unit's angles side
// by side: the lanes' reads met in a quarter of the banks.)
__device__ __forceinline__ int turn_slot(int i, int half, int interleaved) {
  const int log_pieces = interleaved ? 1 : 2, piece = (i >> 1) & ((1 << log_pieces) - 1), unit = (i >> 1) >> log_pieces;
  return 2 * (piece * (half >> (log_pieces + 1)) + unit) + (i & 1);
}
// The angles of a block's tokens.
__device__ __forceinline__ void make_turns(const NormRopeParams& p, float2* turns, int token0, int tokens) {
  const int half = p.R >> 1;
  for (int i = threadIdx.x; i < tokens * half; i += kThreads) {
    const int tk = i / half, pair = i - tk * half;
    turns[tk * half + turn_slot(pair, half, p.interleaved)] = turn_of(p, position_of(p, token0 + tk), p.inv_freq[pair]);
  }
}

// The rotation of unit e0 .. e0 + 7 (dims relative to rope_start) of a row: v = this unit, o = its partner unit (halves only).
__device__ __forceinline__ void rotate8(float (&v)[8], const float (&o)[8], const float2* turns, int e0, int half, bool interleaved) {
  const float4* t4 = reinterpret_cast<const float4*>(turns);
  if (interleaved) {
    t4 += e0 >> 3;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float4 t = t4[j * (half >> 2)];
      const float c[2] = {t.x, t.z}, s[2] = {t.y, t.w};
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const float a = v[4 * j + 2 * k], b = v[4 * j + 2 * k + 1];
        v[4 * j + 2 * k] = a * c[k] - b * s[k];
        v[4 * j + 2 * k + 1] = b * c[k] + a * s[k];
      }
    }
  } else {
    const bool second = e0 >= half;
    t4 += (second ? e0 - half : e0) >> 3;
    const float sign = second ? 1.f : -1.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float4 t = t4[j * (half >> 3)];
      v[2 * j] = v[2 * j] * t.x + o[2 * j] * (sign * t.y);
      v[2 * j + 1] = v[2 * j + 1] * t.z + o[2 * j + 1] * (sign * t.w);
    }
  }
}

struct Tile {
  int side, token0, head0, tokens, heads;
};
// A group's rows of a tile, `step` rows apart: their tokens and heads without a division each.
struct Walk {
  int tk, head, step_tk, step_head;
  __device__ __forceinline__ Walk(const Tile& t, int row, int step) {
    tk = row / t.heads;
    head = row - tk * t.heads;
    step_tk = step_head = 0;
    if (t.tokens * t.heads > step) {   // (there is a next one)
      step_tk = step / t.heads;
      step_head = step - step_tk * t.heads;
    }
  }
  __device__ __forceinline__ void next(const Tile& t) {
    tk += step_tk;
    head += step_head;
    if (head >= t.heads) { head -= t.heads; ++tk; }
  }
};
// Element 0 of the row of a tile's token number tk and head: b0 and s0 are those of its first token.
template <typename T>
__device__ __forceinline__ const T* row_in(const RowView& v, const Tile& t, int S, int b0, int s0, int tk, int head) {
  int b = b0, s = s0 + tk;
  if (s >= S) {   // (few tiles reach into the next sequence)
    const int more = s / S;
    b += more;
    s -= more * S;
  }
  return static_cast<const T*>(v.base) + b * v.stride_b + s * v.stride_s + (t.head0 + head) * v.stride_h;
}
__device__ __forceinline__ Tile tile_of(const NormRopeParams& p, int block) {
  Tile t;
  t.side = block >= p.side[0].blocks;
  const RopeSide& sd = p.side[t.side];
  if (t.side) block -= p.side[0].blocks;
  const int hb = (sd.H + sd.tile_heads - 1) / sd.tile_heads;
  const int tb = block / hb;
  t.token0 = tb * sd.tile_tokens;
  t.head0 = (block - tb * hb) * sd.tile_heads;
  t.tokens = min(sd.tile_tokens, p.tokens - t.token0);
  t.heads = min(sd.tile_heads, sd.H - t.head0);
  return t;
}
}  // namespace nr

// -------------------------------------------------------------------------------------------------
// forward, 16-byte units
// -------------------------------------------------------------------------------------------------
// (blocks per SM, in registers: short rows keep few bytes per thread on their way and need more threads: rows of 128 dims, the call above:
// four blocks 80 us, five 76, six 80)
template <typename T, int G, int NV>
__global__ void __launch_bounds__(nr::kThreads, NV <= 2 ? 5 : 3) norm_rope_kernel(const __grid_constant__ NormRopeParams p) {
  using namespace nr;
  extern __shared__ __align__(16) float2 turns[];         // [tile_tokens][R / 2]
  __shared__ __align__(16) float sw[kMaxNormDim], sb[kMaxNormDim];
  const Tile t = tile_of(p, blockIdx.x);
  const RopeSide& sd = p.side[t.side];
  const int tid = threadIdx.x, lane = tid % G, group = tid / G;
  constexpr int kGroups = kThreads / G;
  const int units = p.D >> 3, half = p.R >> 1, rows = t.tokens * t.heads;

  const int b0 = t.token0 / p.S, s0 = t.token0 - b0 * p.S;
  Walk at(t, group, kGroups);
  const T* x = nullptr;   // this group's row
  uint4 raw[NV];
  auto fetch = [&]() {
    x = row_in<T>(sd.x, t, p.S, b0, s0, at.tk, at.head);
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (lane + G * i < units) raw[i] = ld_stream(x + (lane + G * i) * 8);
  };
#pragma unroll
  for (int i = 0; i < NV; ++i) raw[i] = make_uint4(0, 0, 0, 0);   // (units beyond the row stay zero)
  if (group < rows) fetch();   // the first row travels while the angles are made
  make_turns(p, turns, t.token0, t.tokens);
  if (sd.norm)
    for (int i = tid; i < p.norm_dim; i += kThreads) {
      sw[i] = sd.weight ? param_at<T>(sd.weight, sd.param_fp32, i) : 1.f;
      sb[i] = sd.bias ? param_at<T>(sd.bias, sd.param_fp32, i) : 0.f;
    }
  __syncthreads();

  // (groups of one warp take the same number of turns through the loop, so that its shuffles see all lanes)
  for (int row0 = 0; row0 < rows; row0 += kGroups, at.next(t)) {
    const bool live = row0 + group < rows;
    const int tk = live ? at.tk : 0;
    if (row0 && live) fetch();
    float mean = 0.f, rstd = 1.f;
    if (sd.norm) {
      if (sd.norm == kNormLayer) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
          if ((lane + G * i) * 8 < p.norm_dim) {
            float v[8];
            unpack8<T>(raw[i], v);
#pragma unroll
            for (int j = 0; j < 8; ++j) s += v[j];
          }
        mean = group_sum<G>(s) * p.inv_norm_dim;
      }
      float q = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if ((lane + G * i) * 8 < p.norm_dim) {
          float v[8];
          unpack8<T>(raw[i], v);
#pragma unroll
          for (int j = 0; j < 8; ++j) q += (v[j] - mean) * (v[j] - mean);
        }
      rstd = rsqrtf(group_sum<G>(q) * p.inv_norm_dim + p.eps);
    }
    auto norm8 = [&](float (&v)[8], int e) {
      if (sd.norm && e < p.norm_dim) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = (v[j] - mean) * rstd * sw[e + j] + sb[e + j];
      }
    };
    const long long orow = live ? out_row(sd, t.token0 + at.tk, t.head0 + at.head) : -1;
    T* const y_lo = static_cast<T*>(sd.y) + orow * sd.split;
    T* const y_hi = sd.split < p.D ? static_cast<T*>(sd.y_tail) + (orow * (p.D - sd.split) - sd.split) : y_lo;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e = (lane + G * i) * 8, r = e - p.rope_start;
      float v[8], o[8];
      unpack8<T>(raw[i], v);
      norm8(v, e);
      // (the same for all lanes: does the rotation touch these G units?)
      if (G * i * 8 < p.rope_start + p.R && G * (i + 1) * 8 > p.rope_start) {
        const bool turned = r >= 0 && r < p.R;
        if (!p.interleaved) {   // the pairs' other members are another unit
          const int pe = r < half ? e + half : e - half;
          uint4 w = make_uint4(0, 0, 0, 0);
          if (p.partner_xor) {  // ... of the same turn of lane ^ partner_xor
            w.x = __shfl_xor_sync(0xffffffffu, raw[i].x, p.partner_xor);
            w.y = __shfl_xor_sync(0xffffffffu, raw[i].y, p.partner_xor);
            w.z = __shfl_xor_sync(0xffffffffu, raw[i].z, p.partner_xor);
            w.w = __shfl_xor_sync(0xffffffffu, raw[i].w, p.partner_xor);
          } else if (live && turned) {   // ... read once more, from L2
            w = __ldg(reinterpret_cast<const uint4*>(x + pe));
          }
          unpack8<T>(w, o);
          if (turned) norm8(o, pe);
        }
        if (turned) rotate8(v, o, turns + tk * half, r, half, p.interleaved);
      }
      if (orow >= 0 && e < p.D) *reinterpret_cast<uint4*>((e < sd.split ? y_lo : y_hi) + e) = pack8<T>(v);
    }
  }
}

// -------------------------------------------------------------------------------------------------
// backward of one side with a norm, 16-byte units.  Every block leaves the sums of its rows for dweight and dbias in its own
// line of the workspace (norm_rope_param_grad_kernel adds the lines up in a fixed order).
// -------------------------------------------------------------------------------------------------
template <typename T, int G, int NV>
__global__ void __launch_bounds__(nr::kThreads) norm_rope_bwd_kernel(const __grid_constant__ NormRopeParams p) {
  using namespace nr;
  extern __shared__ __align__(16) float2 turns[];
  __shared__ __align__(16) float sw[kMaxNormDim], sdw[kMaxNormDim], sdb[kMaxNormDim];
  const RopeSide& sd = p.side[0];
  const int tid = threadIdx.x, lane = tid % G, group = tid / G;
  constexpr int kGroups = kThreads / G;
  const int units = p.D >> 3, half = p.R >> 1;
  float dw[NV][8], db[NV][8];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
#pragma unroll
    for (int j = 0; j < 8; ++j) dw[i][j] = db[i][j] = 0.f;
  }
  for (int i = tid; i < p.norm_dim; i += kThreads) {
    sw[i] = sd.weight ? param_at<T>(sd.weight, sd.param_fp32, i) : 1.f;
    sdw[i] = sdb[i] = 0.f;
  }
  for (int tile = blockIdx.x; tile < sd.blocks; tile += gridDim.x) {
    const Tile t = tile_of(p, tile);
    const int rows = t.tokens * t.heads;
    __syncthreads();   // the last tile's angles have been used
    make_turns(p, turns, t.token0, t.tokens);
    __syncthreads();
    const int b0 = t.token0 / p.S, s0 = t.token0 - b0 * p.S;
    Walk at(t, group, kGroups);
    for (int row0 = 0; row0 < rows; row0 += kGroups, at.next(t)) {
      const bool live = row0 + group < rows;
      const int tk = live ? at.tk : 0, head = live ? at.head : 0;
      const T* dy = row_in<T>(sd.dy, t, p.S, b0, s0, tk, head);
      const T* x_row = row_in<T>(sd.x, t, p.S, b0, s0, tk, head);
      float v[NV][8], x[NV][8];
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        uint4 w = make_uint4(0, 0, 0, 0), wx = w;
        if (live && lane + G * i < units) {
          w = ld_stream(dy + (lane + G * i) * 8);
          if ((lane + G * i) * 8 < p.norm_dim) wx = ld_stream(x_row + (lane + G * i) * 8);
        }
        unpack8<T>(w, v[i]);
        unpack8<T>(wx, x[i]);
      }
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int e = (lane + G * i) * 8, r = e - p.rope_start;
        if (live && e < p.D && r >= 0 && r < p.R) {
          float o[8];
          if (!p.interleaved) unpack8<T>(__ldg(reinterpret_cast<const uint4*>(dy + (r < half ? e + half : e - half))), o);
          rotate8(v[i], o, turns + tk * half, r, half, p.interleaved);
        }
      }
      float mean = 0.f;
      if (sd.norm == kNormLayer) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
#pragma unroll
          for (int j = 0; j < 8; ++j) s += x[i][j];   // (units beyond norm_dim hold zeros)
        }
        mean = group_sum<G>(s) * p.inv_norm_dim;
      }
      float q = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if ((lane + G * i) * 8 < p.norm_dim) {
#pragma unroll
          for (int j = 0; j < 8; ++j) { x[i][j] -= mean; q += x[i][j] * x[i][j]; }
        }
      const float square = group_sum<G>(q) * p.inv_norm_dim + p.eps;
      const float rstd = live ? rsqrtf(square) : 0.f;   // (a group without a row holds zeros, and they stay zeros without an eps too)
      float gn = 0.f, gs = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int e = (lane + G * i) * 8;
        if (e < p.norm_dim) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            x[i][j] *= rstd;
            dw[i][j] += v[i][j] * x[i][j];
            db[i][j] += v[i][j];
            v[i][j] *= sw[e + j];
            gn += v[i][j] * x[i][j];
            gs += v[i][j];
          }
        }
      }
      gn = group_sum<G>(gn) * p.inv_norm_dim;
      gs = sd.norm == kNormLayer ? group_sum<G>(gs) * p.inv_norm_dim : 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if ((lane + G * i) * 8 < p.norm_dim) {
#pragma unroll
          for (int j = 0; j < 8; ++j) v[i][j] = rstd * (v[i][j] - gn * x[i][j] - gs);
        }
      if (live) {
        T* dx = static_cast<T*>(sd.y) + (static_cast<long long>(t.token0 + tk) * sd.H + t.head0 + head) * p.D;
#pragma unroll
        for (int i = 0; i < NV; ++i)
          if (lane + G * i < units) *reinterpret_cast<uint4*>(dx + (lane + G * i) * 8) = pack8<T>(v[i]);
      }
    }
  }
  if (!sd.partials) return;
  // the groups of the block add their sums one after the other: the same order in every run
  for (int turn = 0; turn < kGroups; ++turn) {
    __syncthreads();
    if (group == turn) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int e = (lane + G * i) * 8;
        if (e < p.norm_dim) {
#pragma unroll
          for (int j = 0; j < 8; ++j) { sdw[e + j] += dw[i][j]; sdb[e + j] += db[i][j]; }
        }
      }
    }
  }
  __syncthreads();
  float* line = sd.partials + static_cast<long long>(blockIdx.x) * 2 * p.norm_dim;
  for (int i = tid; i < p.norm_dim; i += kThreads) { line[i] = sdw[i]; line[p.norm_dim + i] = sdb[i]; }
}

// dweight and dbias from the blocks' lines: a block takes 32 columns of the 2 * norm_dim, its warps every 32nd line (every eighth, of twice
// as many lines: 8.8 us for 128 dims).
template <typename T>
__global__ void __launch_bounds__(1024) norm_rope_param_grad_kernel(const float* partials, int lines, int norm_dim, void* d_weight, void* d_bias, int fp32) {
  __shared__ float sums[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  float s = 0.f;
  if (c < 2 * norm_dim)
#pragma unroll 4
    for (int l = warp; l < lines; l += 32) s += partials[static_cast<long long>(l) * 2 * norm_dim + c];
  sums[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && c < 2 * norm_dim) {
    s = 0.f;
    for (int w = 0; w < 32; ++w) s += sums[w][lane];
    void* out = c < norm_dim ? d_weight : d_bias;
    const int i = c < norm_dim ? c : c - norm_dim;
    if (out) {
      if (fp32) static_cast<float*>(out)[i] = s;
      else static_cast<T*>(out)[i] = static_cast<T>(s);
    }
  }
}

// -------------------------------------------------------------------------------------------------
// any size, offset and stride: a warp per row, element by element.  kBack: backward (dweight / dbias sums through the lines of
// the workspace, one per block, added by one warp of the block after the other).
// -------------------------------------------------------------------------------------------------
namespace nr {
template <typename T>
__device__ __forceinline__ void any_stats(const NormRopeParams& p, const RopeSide& sd, const T* x, int lane, float* mean, float* rstd) {
  const int n = p.norm_dim;
  *mean = 0.f;
  *rstd = 1.f;
  if (!sd.norm) return;
  if (sd.norm == kNormLayer) {
    float s = 0.f;
    for (int e = lane; e < n; e += 32) s += static_cast<float>(x[e]);
    *mean = group_sum<32>(s) * p.inv_norm_dim;
  }
  float q = 0.f;
  for (int e = lane; e < n; e += 32) { const float d = static_cast<float>(x[e]) - *mean; q += d * d; }
  *rstd = rsqrtf(group_sum<32>(q) * p.inv_norm_dim + p.eps);
}

// Element e of the rotated row whose elements `at` gives.
template <typename At>
__device__ __forceinline__ float any_rotated(const NormRopeParams& p, long long position, int e, At at) {
  const int d = e - p.rope_start, half = p.R >> 1;
  if (d < 0 || d >= p.R) return at(e);
  const bool second = p.interleaved ? (d & 1) != 0 : d >= half;
  const int pair = p.interleaved ? d >> 1 : (second ? d - half : d);
  const int partner = p.interleaved ? p.rope_start + (d ^ 1) : (second ? e - half : e + half);
  const float2 t = turn_of(p, position, p.inv_freq[pair]);
  return at(e) * t.x + at(partner) * (second ? t.y : -t.y);
}

template <typename T, bool kBack>
__device__ __forceinline__ void any_row(const NormRopeParams& p, const RopeSide& sd, long long r, int token, int head, int lane) {
  const T* x = row_of<T>(sd.x, p.S, token, head);
  const int n = p.norm_dim;
  const long long position = position_of(p, token);
  float mean = 0.f, rstd = 1.f;
  if (sd.norm) any_stats(p, sd, x, lane, &mean, &rstd);
  auto weight = [&](int e) { return sd.weight ? param_at<T>(sd.weight, sd.param_fp32, e) : 1.f; };
  if constexpr (!kBack) {
    const long long orow = out_row(sd, token, head);
    if (orow < 0) return;
    auto normed = [&](int e) {
      const float v = static_cast<float>(x[e]);
      if (!sd.norm || e >= n) return v;
      return (v - mean) * rstd * weight(e) + (sd.bias ? param_at<T>(sd.bias, sd.param_fp32, e) : 0.f);
    };
    for (int e = lane; e < p.D; e += 32) {
      T* y = e < sd.split ? static_cast<T*>(sd.y) + orow * sd.split + e : static_cast<T*>(sd.y_tail) + orow * (p.D - sd.split) + (e - sd.split);
      *y = static_cast<T>(any_rotated(p, position, e, normed));
    }
  } else {
    const T* dy = row_of<T>(sd.dy, p.S, token, head);
    auto grad = [&](int e) { return static_cast<float>(dy[e]); };
    float gn = 0.f, gs = 0.f;
    if (sd.norm) {
      for (int e = lane; e < n; e += 32) {
        const float u = any_rotated(p, position, e, grad) * weight(e);
        gn += u * (static_cast<float>(x[e]) - mean) * rstd;
        gs += u;
      }
      gn = group_sum<32>(gn) * p.inv_norm_dim;
      gs = sd.norm == kNormLayer ? group_sum<32>(gs) * p.inv_norm_dim : 0.f;
    }
    T* dx = static_cast<T*>(sd.y) + r * p.D;
    for (int e = lane; e < p.D; e += 32) {
      float u = any_rotated(p, position, e, grad);
      if (sd.norm && e < n) u = rstd * (u * weight(e) - gn * (static_cast<float>(x[e]) - mean) * rstd - gs);
      dx[e] = static_cast<T>(u);
    }
  }
}
}  // namespace nr

template <typename T, bool kBack>
__global__ void __launch_bounds__(nr::kThreads) norm_rope_any_kernel(const __grid_constant__ NormRopeParams p) {
  using namespace nr;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = kThreads / 32;
  const long long rows0 = static_cast<long long>(p.tokens) * p.side[0].H, rows1 = kBack ? 0 : static_cast<long long>(p.tokens) * p.side[1].H;
  float* line = kBack && p.side[0].partials ? p.side[0].partials + static_cast<long long>(blockIdx.x) * 2 * p.norm_dim : nullptr;
  if (line) {
    for (int i = threadIdx.x; i < 2 * p.norm_dim; i += kThreads) line[i] = 0.f;
    __syncthreads();
  }
  const long long total = rows0 + rows1, step = static_cast<long long>(gridDim.x) * warps;
  for (long long base = static_cast<long long>(blockIdx.x) * warps; base < total; base += step) {
    const long long g = base + warp;
    if (g < total) {
      const RopeSide& sd = p.side[g >= rows0 ? 1 : 0];
      const long long r = g >= rows0 ? g - rows0 : g;
      const int token = static_cast<int>(r / sd.H), head = static_cast<int>(r - static_cast<long long>(token) * sd.H);
      any_row<T, kBack>(p, sd, r, token, head, lane);
    }
    if (line)   // the block's warps add their rows' sums one after the other
      for (int turn = 0; turn < warps; ++turn) {
        __syncthreads();
        if (warp == turn && g < total) {
          const RopeSide& sd = p.side[0];
          const int token = static_cast<int>(g / sd.H), head = static_cast<int>(g - static_cast<long long>(token) * sd.H);
          const T* x = row_of<T>(sd.x, p.S, token, head);
          const T* dy = row_of<T>(sd.dy, p.S, token, head);
          float mean, rstd;
          any_stats(p, sd, x, lane, &mean, &rstd);
          const long long position = position_of(p, token);
          for (int e = lane; e < p.norm_dim; e += 32) {
            const float u = any_rotated(p, position, e, [&](int i) { return static_cast<float>(dy[i]); });
            line[e] += u * (static_cast<float>(x[e]) - mean) * rstd;
            line[p.norm_dim + e] += u;
          }
        }
      }
  }
}

// -------------------------------------------------------------------------------------------------
// host side
// -------------------------------------------------------------------------------------------------
namespace {
bool aligned_view(const RowView& v) {
  return !v.base || ((reinterpret_cast<uintptr_t>(v.base) & 15u) == 0 && v.stride_b % 8 == 0 && v.stride_s % 8 == 0 && v.stride_h % 8 == 0);
}
// Do all rows come in 16-byte units?
bool in_units(const NormRopeParams& p) {
  if (p.D % 8 || p.D > nr::kMaxNormDim || p.rope_start % 8 || p.R % (p.interleaved ? 8 : 16) || p.norm_dim % 8 || p.R / 2 > nr::kMaxPairs) return false;
  for (const RopeSide& sd : p.side) {
    if (!sd.H) continue;
    if (!aligned_view(sd.x) || !aligned_view(sd.dy) || sd.split % 8) return false;
    if ((reinterpret_cast<uintptr_t>(sd.y) | reinterpret_cast<uintptr_t>(sd.y_tail)) & 15u) return false;
  }
  return true;
}
// Tokens x heads of a block: at most `rows` rows; one token's heads first (they share its angles).
void tile(NormRopeParams* p, int which, int rows) {
  RopeSide& sd = p->side[which];
  if (!sd.H) { sd.blocks = 0; sd.tile_heads = sd.tile_tokens = 1; return; }
  sd.tile_heads = sd.H < rows ? sd.H : rows;
  int tokens = rows / sd.tile_heads;
  const int most = nr::kMaxPairs / (p->R / 2);
  if (tokens > most) tokens = most;
  if (tokens > p->tokens) tokens = p->tokens;
  sd.tile_tokens = tokens < 1 ? 1 : tokens;
  sd.blocks = ((p->tokens + sd.tile_tokens - 1) / sd.tile_tokens) * ((sd.H + sd.tile_heads - 1) / sd.tile_heads);
}
// Rows per block: about 32 KB of them, which amortises a block's angles and weights (when the prefill call above took 194 us with 32 rows of
// 576 dims, 128 rows took 198; rows of 128 dims, forward + backward, 115 us with 32 rows, 103 with 128); calls whose blocks all fit the
// chip at once (three per SM) take shorter ones as long as they do (64 tokens x 129 rows of 576 dims: 32 rows 10.4 us, 16 rows -- more blocks than fit -- 14.4).
void tiles(NormRopeParams* p, int sms) {
  int rows = 256;
  while (rows > 32 && rows * p->D > 16384) rows >>= 1;
  for (;; rows >>= 1) {
    tile(p, 0, rows);
    tile(p, 1, rows);
    if (rows <= 8 || 2 * (p->side[0].blocks + p->side[1].blocks) > 3 * sms) return;
  }
}
int tile_smem(const NormRopeParams& p) {
  int tokens = 1;
  for (const RopeSide& sd : p.side)
    if (sd.H && sd.tile_tokens > tokens) tokens = sd.tile_tokens;
  return tokens * (p.R / 2) * static_cast<int>(sizeof(float2));
}

template <typename T, int G, int NV>
int forward(NormRopeParams p, cudaStream_t stream) {
  // Halves: does a unit's partner sit in the same turn of another lane of its group, at a fixed lane distance?
  const int d = p.R / 16;
  p.partner_xor = !p.interleaved && 2 * d <= G && (d & (d - 1)) == 0 && p.rope_start % (16 * d) == 0 ? d : 0;
  norm_rope_kernel<T, G, NV><<<p.side[0].blocks + p.side[1].blocks, nr::kThreads, tile_smem(p), stream>>>(p);
  return static_cast<int>(cudaGetLastError());
}
template <typename T, int G, int NV>
int backward(const NormRopeParams& p, int grid, cudaStream_t stream) {
  norm_rope_bwd_kernel<T, G, NV><<<grid, nr::kThreads, tile_smem(p), stream>>>(p);
  return static_cast<int>(cudaGetLastError());
}
template <typename T>
int forward_units(const NormRopeParams& p, cudaStream_t stream) {
  if (p.D <= 64) return forward<T, 8, 1>(p, stream);
  if (p.D <= 128) return forward<T, 8, 2>(p, stream);
  if (p.D <= 192) return forward<T, 8, 3>(p, stream);
  if (p.D <= 256) return forward<T, 8, 4>(p, stream);
  if (p.D <= 512) return forward<T, 8, 8>(p, stream);
  if (p.D <= 576) return forward<T, 8, 9>(p, stream);
  return forward<T, 16, 8>(p, stream);
}
// (the sums for dweight and dbias take 16 registers per unit of a lane: up to 32 lanes per row)
template <typename T>
int backward_units(const NormRopeParams& p, int grid, cudaStream_t stream) {
  if (p.D <= 64) return backward<T, 8, 1>(p, grid, stream);
  if (p.D <= 128) return backward<T, 16, 1>(p, grid, stream);
  if (p.D <= 256) return backward<T, 32, 1>(p, grid, stream);
  if (p.D <= 512) return backward<T, 32, 2>(p, grid, stream);
  if (p.D <= 768) return backward<T, 32, 3>(p, grid, stream);
  return backward<T, 32, 4>(p, grid, stream);
}
// Blocks of a backward with a norm: every block leaves one line of sums.
int norm_lines(int sms) { return 2 * sms; }
}  // namespace

int launch_norm_rope(NormRopeParams p, bool bf16, cudaStream_t stream) {
  int dev = 0, sms = 0;
  cudaError_t e = current_device_sms(&dev, &sms);
  if (e != cudaSuccess) return static_cast<int>(e);
  if (!in_units(p)) {
    const long long rows = static_cast<long long>(p.tokens) * (p.side[0].H + p.side[1].H), want = (rows + 7) / 8;
    const int grid = static_cast<int>(want < 8LL * sms ? want : 8LL * sms);
    if (bf16) norm_rope_any_kernel<__nv_bfloat16, false><<<grid, nr::kThreads, 0, stream>>>(p);
    else norm_rope_any_kernel<__half, false><<<grid, nr::kThreads, 0, stream>>>(p);
    return static_cast<int>(cudaGetLastError());
  }
  tiles(&p, sms);
  return bf16 ? forward_units<__nv_bfloat16>(p, stream) : forward_units<__half>(p, stream);
}

size_t norm_rope_bwd_workspace_bytes(int norm_dim) {
  int dev = 0, sms = 0;
  if (current_device_sms(&dev, &sms) != cudaSuccess) return 0;
  return static_cast<size_t>(norm_lines(sms)) * 2 * norm_dim * sizeof(float);
}

// Sides with x (norm only), dy, y = dx; d_weight / d_bias with the side's partials in the workspace, or null.
int launch_norm_rope_bwd(NormRopeParams p, void* const d_weight[2], void* const d_bias[2], bool bf16, cudaStream_t stream) {
  int dev = 0, sms = 0;
  cudaError_t e = current_device_sms(&dev, &sms);
  if (e != cudaSuccess) return static_cast<int>(e);
  p.back = 1;
  // sides without a norm: the forward with the angles turned round, both in one launch
  NormRopeParams turned = p;
  for (RopeSide& sd : turned.side) {
    if (sd.norm) sd.H = 0;
    sd.x = sd.dy;
  }
  if (turned.side[0].H || turned.side[1].H) {
    const int err = launch_norm_rope(turned, bf16, stream);
    if (err) return err;
  }
  for (int i = 0; i < 2; ++i) {
    if (!p.side[i].H || !p.side[i].norm) continue;
    NormRopeParams one = p;
    one.side[0] = p.side[i];
    one.side[1].H = 0;
    int grid, err;
    if (!in_units(one)) {
      const long long want = (static_cast<long long>(one.tokens) * one.side[0].H + 7) / 8;
      grid = static_cast<int>(want < norm_lines(sms) ? want : norm_lines(sms));
      if (bf16) norm_rope_any_kernel<__nv_bfloat16, true><<<grid, nr::kThreads, 0, stream>>>(one);
      else norm_rope_any_kernel<__half, true><<<grid, nr::kThreads, 0, stream>>>(one);
      err = static_cast<int>(cudaGetLastError());
    } else {
      tiles(&one, sms);
      grid = one.side[0].blocks > norm_lines(sms) ? norm_lines(sms) : one.side[0].blocks;
      err = bf16 ? backward_units<__nv_bfloat16>(one, grid, stream) : backward_units<__half>(one, grid, stream);
    }
    if (err) return err;
    if (!one.side[0].partials) continue;
    const int cols = (2 * p.norm_dim + 31) / 32;
    if (bf16)
      norm_rope_param_grad_kernel<__nv_bfloat16><<<cols, 1024, 0, stream>>>(one.side[0].partials, grid, p.norm_dim, d_weight[i], d_bias[i], one.side[0].param_fp32);
    else
      norm_rope_param_grad_kernel<__half><<<cols, 1024, 0, stream>>>(one.side[0].partials, grid, p.norm_dim, d_weight[i], d_bias[i], one.side[0].param_fp32);
    if ((err = static_cast<int>(cudaGetLastError()))) return err;
  }
  return 0;
}

}  // namespace dsa
