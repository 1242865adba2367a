// Distillation of rows of logits from a teacher's top entries (sm_100a).
//
//   A row has V student logits and a list of K teacher entries at columns c_j (without indices: c_j = j).  An entry takes part
//   when its column exists and the student's logit there is not -inf.  With z = student / T, p = the teacher's entries (weights,
//   or exp(logit / T)) normalised over the participating ones, and s = softmax(z) over the list or over the whole row:
//     loss = sum_j p_j (log p_j - log s_j)             d student_c = g / T (s_c - sum of the p_j at c)
//   A row without participating entries, or whose teacher holds nothing there, has loss 0 and gradient 0.
//
// Bound by memory: the forward reads the row once (online maximum and sum when it is normalised over the whole row), the backward reads it
// once more and writes the gradient.  The logarithm of a probability is taken as a difference to the row's maximum; all sums in fp32.  Backward with indices: a block owns 8192 columns of a row, adds the listed
// entries of its columns up in shared memory (a column may be listed more than once) and then streams the columns.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "distill.h"
#include "launch_util.h"

namespace dsa {

namespace dt {
constexpr float kLowest = -3.402823466e38f;
constexpr int kChunk = 8192;   // columns of a backward block: 32 KB of sums

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// exp((x - m) / T) with c = log2(e) / T: the difference is taken before anything is rounded, so rows far from zero keep their
// digits; x = -inf gives 0 for any finite m
__device__ __forceinline__ float exp_from(float x, float m, float c) { return ex2((x - m) * c); }

template <typename T>
__device__ __forceinline__ float to_f(T v) { return static_cast<float>(v); }
template <typename T>
__device__ __forceinline__ T from_f(float v) { return static_cast<T>(v); }

template <typename T>
struct Vec {
  static constexpr int kN = 16 / sizeof(T);
  uint4 raw;
  __device__ __forceinline__ void load(const T* p) { raw = __ldg(reinterpret_cast<const uint4*>(p)); }
  __device__ __forceinline__ float get(int i) const { return to_f(reinterpret_cast<const T*>(&raw)[i]); }
  __device__ __forceinline__ void set(int i, float v) { reinterpret_cast<T*>(&raw)[i] = from_f<T>(v); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<uint4*>(p) = raw; }
};

__device__ __forceinline__ float teacher_at(const DistillParams& p, int64_t i) {
  if (p.teacher_type == kTypeF32) return __ldg(static_cast<const float*>(p.teacher) + i);
  if (p.teacher_type == kTypeBf16) return to_f(static_cast<const __nv_bfloat16*>(p.teacher)[i]);
  return to_f(static_cast<const __half*>(p.teacher)[i]);
}

struct Entry {
  float z;   // student's logit
  float t;   // teacher's weight (not below 0) or logit
  bool in;
};
// Entry j of row r; its column goes to *column.
template <typename T>
__device__ __forceinline__ Entry entry_at(const DistillParams& p, int64_t r, const T* row, int j, int* column) {
  Entry e{0.f, 0.f, false};
  const int c = p.indices ? __ldg(p.indices + r * p.K + j) : j;
  *column = c;
  if (c < 0 || c >= p.V) return e;
  const float raw = to_f(row[c]);
  e.in = !(raw == -INFINITY);
  if (!e.in) return e;
  const float t = teacher_at(p, r * p.K + j);
  e.z = raw;
  e.t = p.teacher_logits ? t : (t < 0.f ? 0.f : t);   // (NaN stays NaN)
  return e;
}

enum { kMax, kSum };
// Reduction of two values over the block; every thread gets both.
template <int kThreads, int kOp>
__device__ __forceinline__ float2 block_reduce(float2 v, float2* scratch) {
  auto op = [](float a, float b) { return kOp == kMax ? fmaxf(a, b) : a + b; };
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    v.x = op(v.x, __shfl_xor_sync(0xffffffffu, v.x, o));
    v.y = op(v.y, __shfl_xor_sync(0xffffffffu, v.y, o));
  }
  constexpr int kWarps = kThreads / 32;
  __syncthreads();
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  v = scratch[threadIdx.x & (kWarps - 1)];
#pragma unroll
  for (int o = kWarps / 2; o > 0; o >>= 1) {
    v.x = op(v.x, __shfl_xor_sync(0xffffffffu, v.x, o));
    v.y = op(v.y, __shfl_xor_sync(0xffffffffu, v.y, o));
  }
  return v;
}

// Running maximum and sum of exponentials relative to it.
struct Online {
  float m = kLowest, s = 0.f;
  template <int N>
  __device__ __forceinline__ void add(const float (&z)[N], float c) {
    float top = z[0];
#pragma unroll
    for (int i = 1; i < N; ++i) top = fmaxf(top, z[i]);
    if (top > m) { s *= exp_from(m, top, c); m = top; }
#pragma unroll
    for (int i = 0; i < N; ++i) s += exp_from(z[i], m, c);
  }
};

// The row's columns in 16-byte units from the first aligned one on; `one` takes a single column, `unit` a whole unit's first column.
template <typename T, typename One, typename Unit>
__device__ __forceinline__ void for_columns(const T* row, int n, int tid, int threads, One one, Unit unit) {
  constexpr int kN = Vec<T>::kN;
  int head = static_cast<int>((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / static_cast<int>(sizeof(T));
  if (head > n) head = n;
  const int units = (n - head) / kN, tail = head + units * kN;
  if (tid < head) one(tid);
  for (int u = tid; u < units; u += threads) unit(head + u * kN);
  if (tail + tid < n) one(tail + tid);
}
}  // namespace dt

// -------------------------------------------------------------------------------------------------
// forward: a block per row.  Each thread keeps kItems list entries in registers (0: they are read again for every pass).
// -------------------------------------------------------------------------------------------------
template <typename T, int kThreads, int kItems>
__global__ void __launch_bounds__(kThreads) distill_fwd_kernel(const __grid_constant__ DistillParams p) {
  using namespace dt;
  __shared__ float2 scratch[32];
  const int64_t r = blockIdx.x;
  const int tid = threadIdx.x;
  const T* row = static_cast<const T*>(p.student) + r * p.row_stride;

  Entry keep[kItems ? kItems : 1];
  auto entries = [&](auto f) {
    if constexpr (kItems) {
#pragma unroll
      for (int i = 0; i < kItems; ++i)
        if (keep[i].in) f(keep[i]);
    } else {
      int c;
      for (int j = tid; j < p.K; j += kThreads) {
        const Entry e = entry_at<T>(p, r, row, j, &c);
        if (e.in) f(e);
      }
    }
  };
  if constexpr (kItems) {
    int c;
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const int j = tid + i * kThreads;
      keep[i] = j < p.K ? entry_at<T>(p, r, row, j, &c) : Entry{0.f, 0.f, false};
    }
  }
  // maxima of the student's list (or, online, of the whole row) and of the teacher's logits
  float2 top = make_float2(kLowest, kLowest), sum = make_float2(0.f, 0.f);
  Online all;
  if (p.over_row) {
    constexpr int kN = Vec<T>::kN;
    // four units in flight per thread
    int head = static_cast<int>((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / static_cast<int>(sizeof(T));
    if (head > p.V) head = p.V;
    const int units = (p.V - head) / kN, tail = head + units * kN;
    int u = tid;
    for (; u + 3 * kThreads < units; u += 4 * kThreads) {
      Vec<T> v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i].load(row + head + (u + i * kThreads) * kN);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float z[kN];
#pragma unroll
        for (int k = 0; k < kN; ++k) z[k] = v[i].get(k);
        all.add(z, p.exp_scale);
      }
    }
    for (; u < units; u += kThreads) {
      Vec<T> v;
      v.load(row + head + u * kN);
      float z[kN];
#pragma unroll
      for (int k = 0; k < kN; ++k) z[k] = v.get(k);
      all.add(z, p.exp_scale);
    }
    for (int side = 0; side < 2; ++side) {
      const int c = side ? tail + tid : tid;
      if (c < (side ? p.V : head)) {
        float z[1] = {to_f(row[c])};
        all.add(z, p.exp_scale);
      }
    }
    top.x = all.m;
  }
  entries([&](const Entry& e) {
    if (!p.over_row) top.x = fmaxf(top.x, e.z);
    if (p.teacher_logits) top.y = fmaxf(top.y, e.t);
  });
  top = block_reduce<kThreads, kMax>(top, scratch);
  if (p.over_row) sum.x = all.s * exp_from(all.m, top.x, p.exp_scale);
  entries([&](const Entry& e) {
    if (!p.over_row) sum.x += exp_from(e.z, top.x, p.exp_scale);
    sum.y += p.teacher_logits ? exp_from(e.t, top.y, p.exp_scale) : e.t;
  });
  sum = block_reduce<kThreads, kSum>(sum, scratch);
  const bool active = !(sum.y == 0.f);   // (NaN: the loss says so)
  const float log_s = logf(sum.x), log_w = logf(sum.y);
  float2 loss = make_float2(0.f, 0.f);
  if (active)
    entries([&](const Entry& e) {
      const float w = p.teacher_logits ? exp_from(e.t, top.y, p.exp_scale) : e.t;
      if (!(w == 0.f)) loss.x += w / sum.y * ((p.teacher_logits ? (e.t - top.y) * p.inv_T : logf(w)) - log_w + (top.x - e.z) * p.inv_T + log_s);
    });
  loss = block_reduce<kThreads, kSum>(loss, scratch);
  if (tid == 0) {
    p.loss[r] = loss.x;
    // for the backward: maximum and reciprocal sum of the student, maximum and sum of the teacher (sum 0: no gradient)
    reinterpret_cast<float4*>(p.stats)[r] = make_float4(top.x, 1.f / sum.x, top.y, sum.y);
  }
}

namespace dt {
__device__ __forceinline__ float teacher_p(const DistillParams& p, const float4& st, float t) {
  return (p.teacher_logits ? exp_from(t, st.z, p.exp_scale) : t) / st.w;
}
}  // namespace dt

// -------------------------------------------------------------------------------------------------
// backward without indices: element by element; block = (row, part of its columns)
// -------------------------------------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(256) distill_bwd_kernel(const __grid_constant__ DistillParams p, const int parts) {
  using namespace dt;
  const int64_t r = blockIdx.x / parts;
  const int part = static_cast<int>(blockIdx.x - r * parts);
  const T* row = static_cast<const T*>(p.student) + r * p.row_stride;
  T* out = static_cast<T*>(p.d_student) + r * p.V;
  const float4 st = __ldg(reinterpret_cast<const float4*>(p.stats) + r);
  const float g = st.w == 0.f ? 0.f : __ldg(p.grad + r) * p.inv_T;
  const int n = min(p.V, (part + 1) * kChunk);
#pragma unroll 4
  for (int c = part * kChunk + static_cast<int>(threadIdx.x); c < n; c += 256) {
    int column;
    const Entry e = entry_at<T>(p, r, row, c, &column);
    const float d = e.in && !(st.w == 0.f) ? g * (exp_from(e.z, st.x, p.exp_scale) * st.y - teacher_p(p, st, e.t)) : 0.f;
    out[c] = from_f<T>(d);
  }
}

// -------------------------------------------------------------------------------------------------
// backward with indices: block = (row, kChunk of its columns)
// -------------------------------------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(512) distill_bwd_listed_kernel(const __grid_constant__ DistillParams p, const int parts) {
  using namespace dt;
  __shared__ float acc[kChunk];
  const int64_t r = blockIdx.x / parts;
  const int c0 = static_cast<int>(blockIdx.x - r * parts) * kChunk, n = min(p.V - c0, kChunk);
  const int tid = threadIdx.x;
  const T* row = static_cast<const T*>(p.student) + r * p.row_stride;
  T* out = static_cast<T*>(p.d_student) + r * p.V + c0;
  const float4 st = __ldg(reinterpret_cast<const float4*>(p.stats) + r);
  const bool active = !(st.w == 0.f);
  const float g = active ? __ldg(p.grad + r) * p.inv_T : 0.f;
  for (int i = tid; i < n; i += 512) acc[i] = 0.f;
  __syncthreads();
  if (active)
    for (int j = tid; j < p.K; j += 512) {
      const int c = __ldg(p.indices + r * p.K + j) - c0;
      if (c < 0 || c >= n) continue;
      int column;
      const Entry e = entry_at<T>(p, r, row, j, &column);
      if (!e.in) continue;
      const float soft = p.over_row ? 0.f : exp_from(e.z, st.x, p.exp_scale) * st.y;
      atomicAdd(&acc[c], g * (soft - teacher_p(p, st, e.t)));
    }
  __syncthreads();
  const T* src = row + c0;
  const float scale = p.over_row ? g * st.y : 0.f;
  auto value = [&](float raw, int c) {
    return p.over_row && active ? fmaf(scale, exp_from(raw, st.x, p.exp_scale), acc[c]) : acc[c];
  };
  if (((reinterpret_cast<uintptr_t>(src) ^ reinterpret_cast<uintptr_t>(out)) & 15u) == 0) {
    for_columns(src, n, tid, 512, [&](int c) { out[c] = from_f<T>(value(p.over_row ? to_f(src[c]) : 0.f, c)); },
                [&](int c) {
                  Vec<T> v, o;
                  if (p.over_row) v.load(src + c);
#pragma unroll
                  for (int k = 0; k < Vec<T>::kN; ++k) o.set(k, value(p.over_row ? v.get(k) : 0.f, c + k));
                  o.store(out + c);
                });
  } else {
    for (int c = tid; c < n; c += 512) out[c] = from_f<T>(value(p.over_row ? to_f(src[c]) : 0.f, c));
  }
}

// -------------------------------------------------------------------------------------------------
// host side
// -------------------------------------------------------------------------------------------------
namespace {
template <typename T>
int forward(const DistillParams& p, cudaStream_t stream) {
  const unsigned rows = static_cast<unsigned>(p.rows);
  // a whole row of many columns is worth more threads; a list stays in registers where it fits
  if (p.over_row && p.V > 4096) {
    if (p.K <= 2048) distill_fwd_kernel<T, 512, 4><<<rows, 512, 0, stream>>>(p);
    else if (p.K <= 8192) distill_fwd_kernel<T, 512, 16><<<rows, 512, 0, stream>>>(p);
    else distill_fwd_kernel<T, 512, 0><<<rows, 512, 0, stream>>>(p);
  } else if (p.K <= 1024) distill_fwd_kernel<T, 256, 4><<<rows, 256, 0, stream>>>(p);
  else if (p.K <= 4096) distill_fwd_kernel<T, 256, 16><<<rows, 256, 0, stream>>>(p);
  else distill_fwd_kernel<T, 256, 0><<<rows, 256, 0, stream>>>(p);
  return static_cast<int>(cudaGetLastError());
}
template <typename T>
int backward(const DistillParams& p, cudaStream_t stream) {
  const int parts = (p.V + dt::kChunk - 1) / dt::kChunk;
  const int64_t blocks = p.rows * parts;
  if (blocks > 0x7fffffffLL) return static_cast<int>(cudaErrorInvalidValue);
  if (p.indices) distill_bwd_listed_kernel<T><<<static_cast<unsigned>(blocks), 512, 0, stream>>>(p, parts);
  else distill_bwd_kernel<T><<<static_cast<unsigned>(blocks), 256, 0, stream>>>(p, parts);
  return static_cast<int>(cudaGetLastError());
}
}  // namespace

int launch_distill_fwd(DistillParams p, cudaStream_t stream) {
  if (!p.indices) p.over_row = 0;   // the list is the row
  if (p.student_type == kTypeF32) return forward<float>(p, stream);
  return p.student_type == kTypeBf16 ? forward<__nv_bfloat16>(p, stream) : forward<__half>(p, stream);
}
int launch_distill_bwd(DistillParams p, cudaStream_t stream) {
  if (!p.indices) p.over_row = 0;
  if (p.student_type == kTypeF32) return backward<float>(p, stream);
  return p.student_type == kTypeBf16 ? backward<__nv_bfloat16>(p, stream) : backward<__half>(p, stream);
}

}  // namespace dsa
