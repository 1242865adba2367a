// Parameter block of the distillation kernels (distill.cu).
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace dsa {

enum : int { kTypeBf16 = 0, kTypeF16 = 1, kTypeF32 = 2 };

struct DistillParams {
  const void* student;      // [rows, V], unit inner stride, rows row_stride elements apart
  const void* teacher;      // [rows, K]
  const int32_t* indices;   // [rows, K] columns of the entries, nullable (K = V: entry j is column j)
  float* loss;              // [rows]
  float* stats;             // [rows, 4], 16-byte aligned
  float* partials;          // forward: workspace of distill_workspace_bytes, null when that is 0
  const float* grad;        // backward: [rows]
  void* d_student;          // backward: [rows, V], the student's type
  int64_t rows, row_stride;
  int V, K;
  int student_type, teacher_type, teacher_logits, over_row;
  int quads;                // set by the launcher: lists in aligned fours
  float inv_T, exp_scale;   // 1 / T, log2(e) / T
};

size_t distill_workspace_bytes(int64_t rows, int V, int over_row, bool listed);
int launch_distill_fwd(DistillParams p, cudaStream_t stream);
int launch_distill_bwd(DistillParams p, cudaStream_t stream);

}  // namespace dsa
