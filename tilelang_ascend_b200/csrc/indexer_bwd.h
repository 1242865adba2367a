// Parameter block of the indexer's backward (indexer_bwd.cu).
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace dsa {

// All tensors contiguous row-major.
struct IndexerBwdParams {
  const void* q;            // [B, S1, N1, D]  bf16 / fp16
  const void* k;            // [B, S2, 1, D]
  const float* w;           // [B, S1, N1]
  const int32_t* indices;   // [B, S1, 1, K]; entries outside [0, S2) take no part
  const float* grad;        // [B, S1, 1, K]  of the scores at the listed keys; not looked at where the index takes no part
  void* d_q;                // as q, the inputs' type
  float* d_k;               // [B, S2, 1, D] fp32, added to
  float* d_w;               // [B, S1, N1]
  int B, S1, S2, N1, D, K;
  int* status;
  const int* only_if;       // not null: launch_indexer_bwd's kernel does nothing unless this holds something else than 0
};

size_t indexer_bwd_workspace_bytes(const IndexerBwdParams& p, bool bf16);
bool indexer_bwd_dense_fits(const IndexerBwdParams& p, bool bf16);
int launch_indexer_bwd_dense(const IndexerBwdParams& p, void* workspace, const int** dirty_out, cudaStream_t stream);
bool indexer_bwd_supported(const IndexerBwdParams& p);
int launch_indexer_bwd(const IndexerBwdParams& p, bool bf16, cudaStream_t stream);

}  // namespace dsa
