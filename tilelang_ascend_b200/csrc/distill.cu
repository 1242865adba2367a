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
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "distill.h"
#include "launch_util.h"

namespace dsa {

namespace dt {
constexpr float kLowest = -3.402823466e38f, kLn2 = 0.6931471805599453f;
constexpr int kChunk = 8192;         // columns of a backward block with indices: 32 KB of sums
constexpr int kListedThreads = 512;
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
  __device__ __forceinline__ void add(const DistillParams& p, const float (&zs)[4], const float (&ts)[4]) {
    const float before = z.m;
    z.add(zs, p.exp_scale);
    if (z.m > before && W != 0.f) A += W * ((z.m - before) * p.inv_T);
    if (p.teacher_logits) {
      const float top = fmaxf(fmaxf(ts[0], ts[1]), fmaxf(ts[2], ts[3]));
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
    for (int i = 0; i < 4; ++i) {
      const float w = p.teacher_logits ? exp_from(ts[i], tm, p.exp_scale) : ts[i];
      if (w != 0.f) {   // (also keeps -inf out of a product with 0)
        const float log_w = p.teacher_logits ? (ts[i] - tm) * p.inv_T : ln_of(w);
        W += w;
        A += w * (log_w + (z.m - zs[i]) * p.inv_T);
      }
    }
  }
};
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
  // to the block's maxima
  float sum[3] = {all.s * exp_from(all.m, top[0], p.exp_scale), list.W, list.A};
  if (list.W != 0.f) {
    sum[2] += list.W * ((top[0] - list.z.m) * p.inv_T);
    if (p.teacher_logits) {
      const float f = exp_from(list.tm, top[1], p.exp_scale);
      sum[2] = f > 0.f ? f * (sum[2] + list.W * ((list.tm - top[1]) * p.inv_T)) : 0.f;
      sum[1] *= f;
    }
  }
  block_reduce<kThreads>(sum, s_sum, Sum());
  if (tid == 0) {
    const float W = sum[1];
    const bool active = !(W == 0.f);   // (NaN: the loss says so)
    p.loss[r] = active ? sum[2] / W - logf(W) + logf(sum[0]) : 0.f;
    // for the backward: maximum and reciprocal sum of the student; of the teacher the maximum of the logits, or a factor that keeps
    // the weights' reciprocal sum finite, and that reciprocal (0: no gradient)
    const float factor = p.teacher_logits ? 1.f : (W < 0x1p-100f ? 0x1p100f : 1.f);
    reinterpret_cast<float4*>(p.stats)[r] =
        make_float4(top[0], active ? 1.f / sum[0] : 0.f, p.teacher_logits ? top[1] : factor, active ? 1.f / (W * factor) : 0.f);
  }
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
// -------------------------------------------------------------------------------------------------
template <typename T, bool kWide>
__global__ void __launch_bounds__(dt::kListedThreads) distill_bwd_listed_kernel(const __grid_constant__ DistillParams p, const int parts) {
  using namespace dt;
  __shared__ float acc[kChunk];
  constexpr int kN = kWide ? Vec<T>::kN : 1, kUnits = kPerThread / kN;
  const int64_t r = blockIdx.x / parts;
  const int c0 = static_cast<int>(blockIdx.x - r * parts) * kChunk, n = min(p.V - c0, kChunk);
  const int tid = threadIdx.x;
  const T* row = static_cast<const T*>(p.student) + r * p.row_stride;
  const T* src = row + c0;
  T* out = static_cast<T*>(p.d_student) + r * p.V + c0;
  // the block's columns travel while the list is looked through
  Vec<T> wide[kWide ? kUnits : 1];
  float narrow[kWide ? 1 : kUnits];
  if (p.over_row) {
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const int c = (tid + u * kListedThreads) * kN;
      if (c < n) {
        if constexpr (kWide) wide[u].load(src + c);
        else narrow[u] = to_f(src[c]);
      }
    }
  }
  const float4 st = __ldg(reinterpret_cast<const float4*>(p.stats) + r);
  const bool active = !(st.w == 0.f);
  const float g = active ? __ldg(p.grad + r) * p.inv_T : 0.f;
#pragma unroll
  for (int i = 0; i < kChunk; i += kListedThreads * 4) *reinterpret_cast<float4*>(acc + i + tid * 4) = make_float4(0.f, 0.f, 0.f, 0.f);
  __syncthreads();
  if (active) {
#pragma unroll 4
    for (int j = tid; j < p.K; j += kListedThreads) {
      const int c = __ldg(p.indices + r * p.K + j) - c0;
      if (c < 0 || c >= n) continue;
      const float z = to_f(src[c]);
      if (z == -INFINITY) continue;
      float t = teacher_at(p, r * p.K + j);
      if (!p.teacher_logits && t < 0.f) t = 0.f;
      const float soft = p.over_row ? 0.f : exp_from(z, st.x, p.exp_scale) * st.y;
      atomicAdd(&acc[c], g * (soft - teacher_p(p, st, t)));
    }
  }
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
        for (int k = 0; k < kN; ++k) o.set(k, value(wide[u].get(k), c + k));
        o.store(out + c);
      } else {
        out[c] = static_cast<T>(value(narrow[u], c));
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

template <typename T>
int forward(const DistillParams& p, int sms, cudaStream_t stream) {
  const unsigned rows = static_cast<unsigned>(p.rows);
  // Whole rows: many of them run side by side in blocks of 256 threads, eight to an SM (1024 rows in blocks of 512 are 1.7 rounds of
  // the chip); few rows take 1024 threads each.  Lists: 256 threads, 64 where that is four entries each.
  if (p.over_row && p.V > 4096 && p.rows < 2 * sms) distill_fwd_kernel<T, 1024, 1><<<rows, 1024, 0, stream>>>(p);
  else if (!p.over_row && p.K <= 256) distill_fwd_kernel<T, 64, 1><<<rows, 64, 0, stream>>>(p);
  else distill_fwd_kernel<T, 256, 8><<<rows, 256, 0, stream>>>(p);
  return static_cast<int>(cudaGetLastError());
}
template <typename T>
int backward(const DistillParams& p, cudaStream_t stream) {
  const int parts = (p.V + dt::kChunk - 1) / dt::kChunk;
  const int64_t blocks = p.rows * parts;
  if (blocks > 0x7fffffffLL) return static_cast<int>(cudaErrorInvalidValue);
  const unsigned grid = static_cast<unsigned>(blocks);
  const int n = dt::Vec<T>::kN;
  if (!p.indices) distill_bwd_kernel<T><<<grid, 256, 0, stream>>>(p, parts);
  else if (p.V % n == 0 && p.row_stride % n == 0 && aligned(p.student, 16) && aligned(p.d_student, 16))
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

int launch_distill_fwd(DistillParams p, cudaStream_t stream) {
  int dev = 0, sms = 0;
  cudaError_t e = current_device_sms(&dev, &sms);
  if (e != cudaSuccess) return static_cast<int>(e);
  finish(&p);
  if (p.student_type == kTypeF32) return forward<float>(p, sms, stream);
  return p.student_type == kTypeBf16 ? forward<__nv_bfloat16>(p, sms, stream) : forward<__half>(p, sms, stream);
}
int launch_distill_bwd(DistillParams p, cudaStream_t stream) {
  finish(&p);
  if (p.student_type == kTypeF32) return backward<float>(p, stream);
  return p.student_type == kTypeBf16 ? backward<__nv_bfloat16>(p, stream) : backward<__half>(p, stream);
}

}  // namespace dsa
