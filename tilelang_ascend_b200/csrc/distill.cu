// Distillation of rows of logits from a teacher's top entries (sm_100a).
//
//   A row has V student logits and a list of K teacher entries at columns c_j (without indices: c_j = j).  An entry takes part
//   when its column exists and the student's logit there is not -inf.  With z = student / T, p = the teacher's entries (weights,
//   or exp(logit / T)) normalised over the participating ones, and s = softmax(z) over the list or over the whole row:
//     loss = sum_j p_j (log p_j - log s_j)             d student_c = g / T (s_c - sum of the p_j at c)
//   A row without participating entries, or whose teacher holds nothing there, has loss 0 and gradient 0.
//
// Bound by memory: the forward reads the row and the list once -- every thread carries running maxima and the sums relative to
// them (softmax normaliser S, teacher weight W, A = sum w (log w - z)), joined over the block at the end: loss = A / W - log W + log S --,
// the backward reads them once more and writes the gradient.  Everything is taken relative to the maxima, so rows far from zero keep
// their digits; all sums in fp32.  (Entries kept in registers and three passes over them: 4096 lists of 2048 forward 87 us; exact
// logarithms and divisions per entry were half of that.)  Backward with indices: a block owns 8192 columns of a row, asks for them,
// adds the listed entries of its columns up in shared memory meanwhile (a column may be listed more than once) and writes the columns.
// Measured, fp32: 1024 rows of 131072 with 2048 entries: forward 107 to 111 us (4.9 TB/s), backward 194 (5.5 TB/s); 4096 lists of 2048: 20 and 13 us
// (out of L2 in part).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "distill.h"
#include "launch_util.h"
#include "ptx.cuh"

namespace dsa {

namespace dt {
constexpr float kLowest = -3.402823466e38f, kLn2 = 0.6931471805599453f;
constexpr int kChunk = 8192;         // columns of a backward block with indices: 32 KB of sums
constexpr int kListedThreads = 512;
constexpr int kPartChunks = 4;       // chunks of a part of the forward
constexpr int kPerThread = kChunk / kListedThreads;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// ln of a weight: lg2 within 2^-22 (relative, or absolute next to 1)
__device__ __forceinline__ float ln_of(float x) {
  float y;
  asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y * kLn2;
}
// exp((x - m) / T) with c = log2(e) / T: the difference is taken before anything is rounded, so rows far from zero keep their
// digits; x = -inf gives 0 for any finite m
__device__ __forceinline__ float exp_from(float x, float m, float c) { return ex2((x - m) * c); }

template <typename T>
__device__ __forceinline__ float to_f(T v) { return static_cast<float>(v); }

// Four consecutive values (at a multiple of four elements).
template <typename T>
__device__ __forceinline__ void load4(const T* p, float (&v)[4]) {
  if constexpr (sizeof(T) == 4) {
    const float4 w = __ldg(reinterpret_cast<const float4*>(p));
    v[0] = w.x; v[1] = w.y; v[2] = w.z; v[3] = w.w;
  } else {
    const uint2 w = __ldg(reinterpret_cast<const uint2*>(p));
    const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = to_f(e[i]);
  }
}
template <typename T>
__device__ __forceinline__ void store4(T* p, const float (&v)[4]) {
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
    uint2 w;
    T* e = reinterpret_cast<T*>(&w);
#pragma unroll
    for (int i = 0; i < 4; ++i) e[i] = static_cast<T>(v[i]);
    *reinterpret_cast<uint2*>(p) = w;
  }
}
template <typename T>
struct Vec {   // 16 bytes
  static constexpr int kN = 16 / sizeof(T);
  uint4 raw;
  __device__ __forceinline__ void load(const T* p) { raw = __ldg(reinterpret_cast<const uint4*>(p)); }
  __device__ __forceinline__ float get(int i) const { return to_f(reinterpret_cast<const T*>(&raw)[i]); }
  __device__ __forceinline__ void set(int i, float v) { reinterpret_cast<T*>(&raw)[i] = static_cast<T>(v); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<uint4*>(p) = raw; }
};

__device__ __forceinline__ void teacher4(const DistillParams& p, int64_t i, float (&t)[4]) {
  if (p.teacher_type == kTypeF32) load4(static_cast<const float*>(p.teacher) + i, t);
  else if (p.teacher_type == kTypeBf16) load4(static_cast<const __nv_bfloat16*>(p.teacher) + i, t);
  else load4(static_cast<const __half*>(p.teacher) + i, t);
}
__device__ __forceinline__ float teacher_at(const DistillParams& p, int64_t i) {
  if (p.teacher_type == kTypeF32) return __ldg(static_cast<const float*>(p.teacher) + i);
  if (p.teacher_type == kTypeBf16) return to_f(static_cast<const __nv_bfloat16*>(p.teacher)[i]);
  return to_f(static_cast<const __half*>(p.teacher)[i]);
}
// The student's logit of an entry in column c (-inf: it takes no part).
template <typename T>
__device__ __forceinline__ float student_at(const DistillParams& p, const T* row, int c) {
  return c >= 0 && c < p.V ? to_f(row[c]) : -INFINITY;
}
// Entries j0 .. j0 + 3 of row r: z the student's logit, -inf where the entry takes no part, t the teacher's (0 there).  p.quads: lists
// come in aligned fours.
template <typename T>
__device__ __forceinline__ void entries4(const DistillParams& p, int64_t r, const T* row, int j0, float (&z)[4], float (&t)[4]) {
  if (p.quads) {
    if (p.indices) {
      const int4 c = __ldg(reinterpret_cast<const int4*>(p.indices + r * p.K + j0));
      z[0] = student_at(p, row, c.x); z[1] = student_at(p, row, c.y); z[2] = student_at(p, row, c.z); z[3] = student_at(p, row, c.w);
    } else {
      load4(row + j0, z);
    }
    teacher4(p, r * p.K + j0, t);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int j = j0 + i;
      z[i] = -INFINITY;
      t[i] = 0.f;
      if (j < p.K) {
        z[i] = student_at(p, row, p.indices ? __ldg(p.indices + r * p.K + j) : j);
        t[i] = teacher_at(p, r * p.K + j);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (z[i] == -INFINITY) t[i] = p.teacher_logits ? -INFINITY : 0.f;   // (whatever the teacher holds there)
    else if (!p.teacher_logits && t[i] < 0.f) t[i] = 0.f;
  }
}

struct Max { __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); } };
struct Sum { __device__ __forceinline__ float operator()(float a, float b) const { return a + b; } };
// Reduction over the block; every thread gets the result.  scratch: kThreads / 32 values of its own for every call.
template <int kThreads, int kN, typename Op>
__device__ __forceinline__ void block_reduce(float (&v)[kN], float (*scratch)[kN], Op op) {
  constexpr int kWarps = kThreads / 32;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
#pragma unroll
    for (int i = 0; i < kN; ++i) v[i] = op(v[i], __shfl_xor_sync(0xffffffffu, v[i], o));
  }
  if ((threadIdx.x & 31) == 0) {
#pragma unroll
    for (int i = 0; i < kN; ++i) scratch[threadIdx.x >> 5][i] = v[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kN; ++i) v[i] = scratch[threadIdx.x & (kWarps - 1)][i];
#pragma unroll
  for (int o = kWarps / 2; o > 0; o >>= 1) {
#pragma unroll
    for (int i = 0; i < kN; ++i) v[i] = op(v[i], __shfl_xor_sync(0xffffffffu, v[i], o));
  }
}

// Running maximum m and sum s of exp((x - m) / T).
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

// What a thread knows of its entries: zm, s as above over the entries; tm the teacher's largest logit (weights: unused), W = sum w,
// A = sum w (log w - (z - zm) / T), with w = weight or exp((t - tm) / T).
struct List {
  Online z;
  float tm = kLowest, W = 0.f, A = 0.f;
  template <int N>
  __device__ __forceinline__ void add(const DistillParams& p, const float (&zs)[N], const float (&ts)[N]) {
    const float before = z.m;
    z.add(zs, p.exp_scale);
    if (z.m > before && W != 0.f) A += W * ((z.m - before) * p.inv_T);
    if (p.teacher_logits) {
      float top = ts[0];
#pragma unroll
      for (int i = 1; i < N; ++i) top = fmaxf(top, ts[i]);
      if (top > tm) {
        if (W != 0.f) {
          const float f = exp_from(tm, top, p.exp_scale);
          A = f > 0.f ? f * (A + W * ((tm - top) * p.inv_T)) : 0.f;
          W *= f;
        }
        tm = top;
      }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float w = p.teacher_logits ? exp_from(ts[i], tm, p.exp_scale) : ts[i];
      if (w != 0.f) {   // (also keeps -inf out of a product with 0)
        const float log_w = p.teacher_logits ? (ts[i] - tm) * p.inv_T : ln_of(w);
        W += w;
        A += w * (log_w + (z.m - zs[i]) * p.inv_T);
      }
    }
  }
};

// sum = {S, W, A} of a thread or part with the row maximum m, A relative to the list maximum zm and teacher maximum tm: made relative
// to the maxima `top` = {row, teacher} instead.
__device__ __forceinline__ void rebase(const DistillParams& p, float (&sum)[3], float m, float zm, float tm, const float (&top)[2]) {
  sum[0] *= exp_from(m, top[0], p.exp_scale);
  if (sum[1] != 0.f) {
    sum[2] += sum[1] * ((top[0] - zm) * p.inv_T);
    if (p.teacher_logits) {
      const float f = exp_from(tm, top[1], p.exp_scale);
      sum[2] = f > 0.f ? f * (sum[2] + sum[1] * ((tm - top[1]) * p.inv_T)) : 0.f;
      sum[1] *= f;
    }
  }
}
// Loss of a row from its joined sums, and what the backward needs of it.
__device__ __forceinline__ void finish_row(const DistillParams& p, int64_t r, const float (&top)[2], const float (&sum)[3]) {
  const float W = sum[1];
  const bool active = !(W == 0.f);   // (NaN: the loss says so)
  p.loss[r] = active ? sum[2] / W - logf(W) + logf(sum[0]) : 0.f;
  // for the backward: maximum and reciprocal sum of the student; of the teacher the maximum of the logits, or a factor that keeps
  // the weights' reciprocal sum finite, and that reciprocal (0: no gradient; an infinite sum has none: NaN, as the loss)
  const float factor = p.teacher_logits ? 1.f : (W < 0x1p-100f ? 0x1p100f : 1.f);
  const float inv_W = W < INFINITY ? 1.f / (W * factor) : NAN;
  reinterpret_cast<float4*>(p.stats)[r] =
      make_float4(top[0], active ? 1.f / sum[0] : 0.f, p.teacher_logits ? top[1] : factor, active ? inv_W : 0.f);
}

// A block's kChunk columns in registers: 16-byte units (kWide) or single elements, kListedThreads apart.
template <typename T, bool kWide>
struct Columns {
  static constexpr int kN = kWide ? Vec<T>::kN : 1, kUnits = kPerThread / kN;
  Vec<T> wide[kWide ? kUnits : 1];
  float narrow[kWide ? 1 : kUnits];
  __device__ __forceinline__ void load(const T* src, int n, int tid) {
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const int c = (tid + u * kListedThreads) * kN;
      if (c < n) {
        if constexpr (kWide) wide[u].load(src + c);
        else narrow[u] = to_f(src[c]);
      }
    }
  }
  __device__ __forceinline__ float get(int u, int k) const {
    if constexpr (kWide) return wide[u].get(k);
    else return narrow[u];
  }
};

// A thread's first kAhead indices of a list, asked for before anything else; then f(column - c0, j) for those of its entries whose column
// lies in [c0, c0 + n).
constexpr int kAhead = 4;
__device__ __forceinline__ void first_indices(const DistillParams& p, int64_t r, int tid, int (&idx)[kAhead]) {
#pragma unroll
  for (int i = 0; i < kAhead; ++i) {
    const int j = tid + i * kListedThreads;
    idx[i] = j < p.K ? __ldg(p.indices + r * p.K + j) : -1;
  }
}
template <typename F>
__device__ __forceinline__ void for_listed(const DistillParams& p, int64_t r, int tid, const int (&idx)[kAhead], int c0, int n, F f) {
#pragma unroll
  for (int i = 0; i < kAhead; ++i) {
    const int c = idx[i] - c0;
    if (idx[i] >= 0 && c >= 0 && c < n) f(c, tid + i * kListedThreads);
  }
  for (int j = tid + kAhead * kListedThreads; j < p.K; j += kListedThreads) {
    const int k = __ldg(p.indices + r * p.K + j), c = k - c0;
    if (k >= 0 && c >= 0 && c < n) f(c, j);
  }
}
constexpr int kPartial = 5;   // floats a part leaves for the join
}  // namespace dt

// -------------------------------------------------------------------------------------------------
// forward: a block per row
// -------------------------------------------------------------------------------------------------
template <typename T, int kThreads, int kBlocks>
__global__ void __launch_bounds__(kThreads, kBlocks) distill_fwd_kernel(const __grid_constant__ DistillParams p) {
  using namespace dt;
  __shared__ float s_max[kThreads / 32][2], s_sum[kThreads / 32][3];
  const int64_t r = blockIdx.x;
  const int tid = threadIdx.x;
  const T* row = static_cast<const T*>(p.student) + r * p.row_stride;

  List list;
  for (int j0 = tid * 4; j0 < p.K; j0 += kThreads * 4) {
    float z[4], t[4];
    entries4<T>(p, r, row, j0, z, t);
    list.add(p, z, t);
  }
  Online all = list.z;
  if (p.over_row) {
    // the whole row, in 16-byte units from the first aligned one on, kUnroll of them on their way per thread
    constexpr int kN = Vec<T>::kN, kUnroll = 2;
    all = Online{};
    int head = static_cast<int>((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / static_cast<int>(sizeof(T));
    if (head > p.V) head = p.V;
    const int units = (p.V - head) / kN, tail = head + units * kN;
    const T* body = row + head;
    int u = tid;
    for (; u + (kUnroll - 1) * kThreads < units; u += kUnroll * kThreads) {
      Vec<T> v[kUnroll];
#pragma unroll
      for (int i = 0; i < kUnroll; ++i) v[i].load(body + static_cast<int64_t>(u + i * kThreads) * kN);
#pragma unroll
      for (int i = 0; i < kUnroll; ++i) {
        float z[kN];
#pragma unroll
        for (int k = 0; k < kN; ++k) z[k] = v[i].get(k);
        all.add(z, p.exp_scale);
      }
    }
    for (; u < units; u += kThreads) {
      Vec<T> v;
      v.load(body + static_cast<int64_t>(u) * kN);
      float z[kN];
#pragma unroll
      for (int k = 0; k < kN; ++k) z[k] = v.get(k);
      all.add(z, p.exp_scale);
    }
    if (tid < head) { const float z[1] = {to_f(row[tid])}; all.add(z, p.exp_scale); }
    if (tail + tid < p.V) { const float z[1] = {to_f(row[tail + tid])}; all.add(z, p.exp_scale); }
  }
  float top[2] = {all.m, list.tm};
  block_reduce<kThreads>(top, s_max, Max());
  float sum[3] = {all.s, list.W, list.A};
  rebase(p, sum, all.m, list.z.m, list.tm, top);
  block_reduce<kThreads>(sum, s_sum, Sum());
  if (tid == 0) finish_row(p, r, top, sum);
}

// -------------------------------------------------------------------------------------------------
// forward of wide rows, in parts: block = (row, kPartChunks chunks of its columns).  A chunk passes through one of two shared-memory
// buffers, the next one on its way meanwhile, and the listed entries of its columns are looked up there: gathered from global memory,
// 2048 entries of a row of 131072 cost as much as half of the row (1024 such rows: 141 us; one chunk per block: 147 us).
// A thread holds the first 2048 entries' columns; what a list has behind them is read again for every chunk.  In parts / a row per block, fp32,
// out of HBM, us: 1024 rows of 131072: 64 entries 104 / 107, 2048: 119 / 156, 4096: 168 / 205, 16384: 440 / 459, 65536: 1516 / 1409; 4 such
// rows: 2048: 16 / 18, 4096: 21 / 18, 16384: 51 / 25; 1024 rows of 20000: 64: 35 / 27, 2048: 47 / 41, 8192: 102 / 68.  So parts are taken for their gain on
// many wide rows with lists up to 16384, and lose on rows of a few parts and on few rows with long lists.
// kWide: rows in aligned 16-byte units, copied asynchronously; else element by element.
// -------------------------------------------------------------------------------------------------
template <typename T, bool kWide>
__global__ void __launch_bounds__(dt::kListedThreads) distill_fwd_part_kernel(const __grid_constant__ DistillParams p, const int parts) {
  using namespace dt;
  extern __shared__ __align__(16) uint8_t buffers[];   // T [2][kChunk]
  __shared__ float s_max[kListedThreads / 32][2], s_sum[kListedThreads / 32][3];
  constexpr int kN = kWide ? Vec<T>::kN : 1;
  const int64_t r = blockIdx.x / parts;
  const int first = static_cast<int>(blockIdx.x - r * parts) * kPartChunks * kChunk, cols = min(p.V - first, kPartChunks * kChunk);
  const int tid = threadIdx.x;
  const T* src = static_cast<const T*>(p.student) + r * p.row_stride + first;
  int idx[kAhead];
  first_indices(p, r, tid, idx);
  auto buffer = [&](int i) { return reinterpret_cast<T*>(buffers) + (i & 1) * kChunk; };
  auto fetch = [&](int i) {
    T* to = buffer(i);
    const T* from = src + i * kChunk;
    const int n = min(cols - i * kChunk, kChunk);
    for (int c = tid * kN; c < n; c += kListedThreads * kN) {
      if constexpr (kWide) cp_async16(smem_u32(to + c), from + c, 16u);
      else to[c] = from[c];
    }
    cp_async_commit();
  };
  Online all;
  List list;
  const int chunks = (cols + kChunk - 1) / kChunk;
  fetch(0);
  for (int i = 0; i < chunks; ++i) {
    if (i + 1 < chunks) {
      fetch(i + 1);
      cp_async_wait<1>();
    } else {
      cp_async_wait<0>();
    }
    __syncthreads();
    const T* zs = buffer(i);
    const int n = min(cols - i * kChunk, kChunk);
    for (int c = tid * kN; c < n; c += kListedThreads * kN) {
      float z[kN];
      if constexpr (kWide) {
        Vec<T> v;
        v.raw = *reinterpret_cast<const uint4*>(zs + c);
#pragma unroll
        for (int k = 0; k < kN; ++k) z[k] = v.get(k);
      } else {
        z[0] = to_f(zs[c]);
      }
      all.add(z, p.exp_scale);
    }
    for_listed(p, r, tid, idx, first + i * kChunk, n, [&](int c, int j) {
      const float z[1] = {to_f(zs[c])};
      if (z[0] == -INFINITY) return;
      float t[1] = {teacher_at(p, r * p.K + j)};
      if (!p.teacher_logits && t[0] < 0.f) t[0] = 0.f;
      list.add(p, z, t);
    });
    __syncthreads();   // the buffer may be filled again
  }
  float top[2] = {all.m, list.tm};
  block_reduce<kListedThreads>(top, s_max, Max());
  float sum[3] = {all.s, list.W, list.A};
  rebase(p, sum, all.m, list.z.m, list.tm, top);
  block_reduce<kListedThreads>(sum, s_sum, Sum());
  if (tid == 0) {
    float* out = p.partials + static_cast<int64_t>(blockIdx.x) * kPartial;
    out[0] = top[0]; out[1] = top[1]; out[2] = sum[0]; out[3] = sum[1]; out[4] = sum[2];
  }
}

// The parts of a row together: a warp per row.
__global__ void __launch_bounds__(128) distill_fwd_join_kernel(const __grid_constant__ DistillParams p, const int parts) {
  using namespace dt;
  const int64_t r = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (r >= p.rows) return;
  const float* in = p.partials + r * parts * kPartial;
  float top[2] = {kLowest, kLowest};
  for (int i = lane; i < parts; i += 32) {
    top[0] = fmaxf(top[0], in[i * kPartial]);
    top[1] = fmaxf(top[1], in[i * kPartial + 1]);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    top[0] = fmaxf(top[0], __shfl_xor_sync(0xffffffffu, top[0], o));
    top[1] = fmaxf(top[1], __shfl_xor_sync(0xffffffffu, top[1], o));
  }
  float sum[3] = {0.f, 0.f, 0.f};
  for (int i = lane; i < parts; i += 32) {
    const float* q = in + i * kPartial;
    float s[3] = {q[2], q[3], q[4]};
    rebase(p, s, q[0], q[0], q[1], top);
#pragma unroll
    for (int k = 0; k < 3; ++k) sum[k] += s[k];
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
#pragma unroll
    for (int k = 0; k < 3; ++k) sum[k] += __shfl_xor_sync(0xffffffffu, sum[k], o);
  }
  if (lane == 0) finish_row(p, r, top, sum);
}

namespace dt {
// The teacher's probability of an entry that takes part.
__device__ __forceinline__ float teacher_p(const DistillParams& p, const float4& st, float t) {
  return (p.teacher_logits ? exp_from(t, st.z, p.exp_scale) : t * st.z) * st.w;
}
}  // namespace dt

// -------------------------------------------------------------------------------------------------
// backward without indices: four entries per thread and step; block = (row, part of its columns)
// -------------------------------------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(256) distill_bwd_kernel(const __grid_constant__ DistillParams p, const int parts) {
  using namespace dt;
  const int64_t r = blockIdx.x / parts;
  const int part = static_cast<int>(blockIdx.x - r * parts);
  const T* row = static_cast<const T*>(p.student) + r * p.row_stride;
  T* out = static_cast<T*>(p.d_student) + r * p.V;
  const float4 st = __ldg(reinterpret_cast<const float4*>(p.stats) + r);
  const bool active = !(st.w == 0.f);
  const float g = active ? __ldg(p.grad + r) * p.inv_T : 0.f;
  const int n = min(p.V, (part + 1) * kChunk);
#pragma unroll 2
  for (int c = part * kChunk + static_cast<int>(threadIdx.x) * 4; c < n; c += 256 * 4) {
    float z[4], t[4], d[4];
    entries4<T>(p, r, row, c, z, t);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      d[i] = active && !(z[i] == -INFINITY) ? g * (exp_from(z[i], st.x, p.exp_scale) * st.y - teacher_p(p, st, t[i])) : 0.f;
    if (p.quads) store4(out + c, d);
    else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (c + i < n) out[c + i] = static_cast<T>(d[i]);
    }
  }
}

// -------------------------------------------------------------------------------------------------
// backward with indices: block = (row, kChunk of its columns).  kWide: rows in aligned 16-byte units, else element by element.
// Last rows first: those are still in L2 when the forward has just read them (1024 rows of 131072 fp32: 198 -> 194 us, and the next
// forward finds the first rows: 111 -> 107).
// -------------------------------------------------------------------------------------------------
template <typename T, bool kWide>
__global__ void __launch_bounds__(dt::kListedThreads) distill_bwd_listed_kernel(const __grid_constant__ DistillParams p, const int parts) {
  using namespace dt;
  __shared__ __align__(16) float acc[kChunk];
  constexpr int kN = kWide ? Vec<T>::kN : 1, kUnits = kPerThread / kN;
  const int64_t block = gridDim.x - 1 - blockIdx.x, r = block / parts;
  const int c0 = static_cast<int>(block - r * parts) * kChunk, n = min(p.V - c0, kChunk);
  const int tid = threadIdx.x;
  const T* src = static_cast<const T*>(p.student) + r * p.row_stride + c0;
  T* out = static_cast<T*>(p.d_student) + r * p.V + c0;
  int idx[kAhead];
  first_indices(p, r, tid, idx);
  const float4 st = __ldg(reinterpret_cast<const float4*>(p.stats) + r);
  const float grad = __ldg(p.grad + r);
  Columns<T, kWide> cols;
  if (p.over_row) cols.load(src, n, tid);   // the block's columns travel while the list is looked through
  const bool active = !(st.w == 0.f);
  const float g = active ? grad * p.inv_T : 0.f;
#pragma unroll
  for (int i = 0; i < kChunk; i += kListedThreads * 4) *reinterpret_cast<float4*>(acc + i + tid * 4) = make_float4(0.f, 0.f, 0.f, 0.f);
  __syncthreads();
  if (active)
    for_listed(p, r, tid, idx, c0, n, [&](int c, int j) {
      const float z = to_f(src[c]);
      if (z == -INFINITY) return;
      float t = teacher_at(p, r * p.K + j);
      if (!p.teacher_logits && t < 0.f) t = 0.f;
      const float soft = p.over_row ? 0.f : exp_from(z, st.x, p.exp_scale) * st.y;
      atomicAdd(&acc[c], g * (soft - teacher_p(p, st, t)));
    });
  __syncthreads();
  const float scale = g * st.y;
  auto value = [&](float z, int c) { return p.over_row && active ? fmaf(scale, exp_from(z, st.x, p.exp_scale), acc[c]) : acc[c]; };
#pragma unroll
  for (int u = 0; u < kUnits; ++u) {
    const int c = (tid + u * kListedThreads) * kN;
    if (c < n) {
      if constexpr (kWide) {
        Vec<T> o;
#pragma unroll
        for (int k = 0; k < kN; ++k) o.set(k, value(cols.get(u, k), c + k));
        o.store(out + c);
      } else {
        out[c] = static_cast<T>(value(cols.get(u, 0), c));
      }
    }
  }
}

// -------------------------------------------------------------------------------------------------
// host side
// -------------------------------------------------------------------------------------------------
namespace {
bool aligned(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
size_t type_bytes(int type) { return type == kTypeF32 ? 4 : 2; }

int distill_parts(int V) { return (V + dt::kChunk - 1) / dt::kChunk; }
int forward_parts(int V) { return (distill_parts(V) + dt::kPartChunks - 1) / dt::kPartChunks; }
// Do all rows (and those of the gradient) come in aligned 16-byte units?
template <typename T>
bool wide_rows(const DistillParams& p) {
  const int n = dt::Vec<T>::kN;
  return p.V % n == 0 && p.row_stride % n == 0 && aligned(p.student, 16) && (!p.d_student || aligned(p.d_student, 16));
}

template <typename T>
int forward(const DistillParams& p, int dev, int sms, cudaStream_t stream) {
  const unsigned rows = static_cast<unsigned>(p.rows);
  // Wide rows go in parts.  Other rows: many of them run side by side in blocks of 256 threads, eight to an SM; few rows take 1024
  // threads each.  Lists: 256 threads, 64 where that is four entries each.
  if (p.partials) {
    const int parts = forward_parts(p.V), smem = 2 * dt::kChunk * static_cast<int>(sizeof(T));
    if (p.rows * parts > 0x7fffffffLL) return static_cast<int>(cudaErrorInvalidValue);
    const unsigned grid = rows * static_cast<unsigned>(parts);
    auto kern = wide_rows<T>(p) ? distill_fwd_part_kernel<T, true> : distill_fwd_part_kernel<T, false>;
    const cudaError_t e = ensure_dynamic_smem(kern, dev, smem);
    if (e != cudaSuccess) return static_cast<int>(e);
    kern<<<grid, dt::kListedThreads, smem, stream>>>(p, parts);
    distill_fwd_join_kernel<<<(rows + 3) / 4, 128, 0, stream>>>(p, parts);
  } else if (p.over_row && p.V > 4096 && p.rows < 2 * sms) distill_fwd_kernel<T, 1024, 1><<<rows, 1024, 0, stream>>>(p);
  else if (!p.over_row && p.K <= 256) distill_fwd_kernel<T, 64, 1><<<rows, 64, 0, stream>>>(p);
  else distill_fwd_kernel<T, 256, 8><<<rows, 256, 0, stream>>>(p);
  return static_cast<int>(cudaGetLastError());
}
template <typename T>
int backward(const DistillParams& p, cudaStream_t stream) {
  const int parts = distill_parts(p.V);
  const int64_t blocks = p.rows * parts;
  if (blocks > 0x7fffffffLL) return static_cast<int>(cudaErrorInvalidValue);
  const unsigned grid = static_cast<unsigned>(blocks);
  if (!p.indices) distill_bwd_kernel<T><<<grid, 256, 0, stream>>>(p, parts);
  else if (wide_rows<T>(p))
    distill_bwd_listed_kernel<T, true><<<grid, dt::kListedThreads, 0, stream>>>(p, parts);
  else
    distill_bwd_listed_kernel<T, false><<<grid, dt::kListedThreads, 0, stream>>>(p, parts);
  return static_cast<int>(cudaGetLastError());
}
void finish(DistillParams* p) {
  if (!p->indices) p->over_row = 0;   // the list is the row
  // fours of a list: the indices, or without them the student's row (and its gradient), and the teacher's entries
  const size_t own = type_bytes(p->student_type);
  p->quads = p->K % 4 == 0 && aligned(p->teacher, 4 * type_bytes(p->teacher_type)) &&
             (p->indices ? aligned(p->indices, 16)
                         : p->row_stride % 4 == 0 && aligned(p->student, 4 * own) && (!p->d_student || aligned(p->d_student, 4 * own)));
}
}  // namespace

// Rows normalised as a whole, wide enough for several parts.
size_t distill_workspace_bytes(int64_t rows, int V, int over_row, bool listed) {
  return over_row && listed && V > 2 * dt::kChunk ? static_cast<size_t>(rows) * forward_parts(V) * dt::kPartial * sizeof(float) : 0;
}

int launch_distill_fwd(DistillParams p, cudaStream_t stream) {
  int dev = 0, sms = 0;
  cudaError_t e = current_device_sms(&dev, &sms);
  if (e != cudaSuccess) return static_cast<int>(e);
  finish(&p);
  if (p.student_type == kTypeF32) return forward<float>(p, dev, sms, stream);
  return p.student_type == kTypeBf16 ? forward<__nv_bfloat16>(p, dev, sms, stream) : forward<__half>(p, dev, sms, stream);
}
int launch_distill_bwd(DistillParams p, cudaStream_t stream) {
  finish(&p);
  if (p.student_type == kTypeF32) return backward<float>(p, stream);
  return p.student_type == kTypeBf16 ? backward<__nv_bfloat16>(p, stream) : backward<__half>(p, stream);
}

}  // namespace dsa
