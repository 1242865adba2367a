// Parameter blocks of the norm + rotation kernels (norm_rope.cu).
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace dsa {

enum : int { kNormNone = 0, kNormRms = 1, kNormLayer = 2 };

// A [B, S, H, D] tensor with unit inner stride; strides in elements.
struct RowView {
  const void* base;
  long long stride_b, stride_s, stride_h;
};

// Queries or keys of a call.
struct RopeSide {
  RowView x;
  RowView dy;             // backward only
  int H;                  // 0: this side is not there
  int norm;               // kNorm*
  const void* weight;     // [norm_dim], nullable
  const void* bias;       // [norm_dim], nullable
  int param_fp32;         // weight and bias are fp32, else the rows' type
  // output rows: dims [0, split) in y, the rest in y_tail (split = D: all in y).  Row (token, head) is row token * H + head, or with
  // slots row slots[token] * H + head of y_slots * H rows; other slots are not written.
  void* y;
  void* y_tail;
  int split;
  const void* slots;
  int slots64;
  long long y_slots;
  float* partials;        // backward: one line [2, norm_dim] per block, nullable
  int blocks, tile_tokens, tile_heads;   // set by the launcher
};

struct NormRopeParams {
  RopeSide side[2];
  const void* positions;  // [tokens]
  int positions64;
  const float* inv_freq;  // [R / 2]
  int tokens, S, D, R, rope_start, norm_dim, interleaved;
  float rope_scale, eps, inv_norm_dim;
  int back;               // 1: the transposed rotation
  int partner_xor;        // set by the launcher
};

int launch_norm_rope(NormRopeParams p, bool bf16, cudaStream_t stream);
size_t norm_rope_bwd_workspace_bytes(int norm_dim);
int launch_norm_rope_bwd(NormRopeParams p, void* const d_weight[2], void* const d_bias[2], bool bf16, cudaStream_t stream);

}  // namespace dsa
