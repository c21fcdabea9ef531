// Distillation from a teacher of whom the top logits are known: loss and gradient for rows of student logits z [N, V] against K teacher logits t [N, K]
// at classes i [N, K].
//
//   p = softmax(t / T) over the entries that are there,  q = softmax(z / T)
//   loss_n = T^2 sum_k p_k (log p_k - log q_{i_k}),      dloss_n / dz_j = T (q_j - sum of the p_k with i_k = j)
//
// An entry is there if its class lies in [0, V) and its logit is not -inf; a row without any has loss 0, gradient 0 and does not count in a mean.
#include "lt_cuda.h"

#include <algorithm>

#include "common/elem.cuh"
#include "common/host.h"
#include "common/ptx.cuh"

namespace lt {

constexpr int kDistillThreads = 512, kDistillWarps = kDistillThreads / 32, kDistillTop = 1024;
constexpr float kLog2e = 1.4426950408889634f;

struct DistillArgs {
  const void* z;
  long long ldz;
  const void* t;                 // [N, K] of type t_type
  int t_type;
  const long long* idx;          // [N, K]
  int N, V, K;
  float temperature;
  const unsigned char* flags;    // which rows have a teacher, for a mean; else null
  const float* up;               // upstream gradient: one (up_rows 0) or one for every row; null: 1
  int up_rows;
  int skip_one;                  // with one upstream gradient: return where it is 1 (the gradient is there)
  float2* stats;                 // [N] maximum of z, and sum of e^((z - maximum) / T)
  int have_stats;
  float* loss;                   // [N] or null
  void* grad;                    // [N, V] or null
};

__device__ __forceinline__ float load_as(int type, const void* p, long long i) {
  if (type == kElemF32) return static_cast<const float*>(p)[i];
  return type == kElemBf16 ? to_f32(static_cast<const __nv_bfloat16*>(p)[i]) : to_f32(static_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ bool entry_there(float t, long long i, int V) { return i >= 0 && i < V && t != -INFINITY; }

__global__ void __launch_bounds__(256) distill_flags_kernel(const void* t, int t_type, const long long* idx, int N, int V, int K, unsigned char* flags) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  for (long long r = blockIdx.x * 8ll + (threadIdx.x >> 5); r < N; r += gridDim.x * 8ll) {
    bool any = false;
    for (int k = lane; k < K && !any; k += 32) any = entry_there(load_as(t_type, t, r * K + k), idx[r * K + k], V);
    any = __any_sync(0xffffffffu, any);
    if (lane == 0) flags[r] = any;
  }
}

__device__ __forceinline__ int count_flags(const unsigned char* flags, int N, int* red) {
  int n = 0;
  for (int i = threadIdx.x; i < N; i += blockDim.x) n += flags[i];
  n = __reduce_add_sync(0xffffffffu, n);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = n;
  __syncthreads();
  n = 0;
  for (int w = 0; w < int(blockDim.x >> 5); ++w) n += red[w];
  __syncthreads();
  return n;
}

// (maximum, sum of 2^(c (. - maximum))) of two parts.  Differences are taken before the factor: next to the maximum they are exact.
__device__ __forceinline__ void join_max_sum(float& m, float& s, float om, float os, float c) {
  const float nm = fmaxf(m, om);
  s = (m == -INFINITY ? s : s * exp2f((m - nm) * c)) + (om == -INFINITY ? os : os * exp2f((om - nm) * c));
  m = nm;
}
__device__ __forceinline__ void block_max_sum(float& m, float& s, float c, float2* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float om = __shfl_xor_sync(0xffffffffu, m, o), os = __shfl_xor_sync(0xffffffffu, s, o);
    join_max_sum(m, s, om, os, c);
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __syncthreads();
  if (lane == 0) red[warp] = make_float2(m, s);
  __syncthreads();
  const float2 v = lane < kDistillWarps ? red[lane] : make_float2(-INFINITY, 0.f);
  m = v.x;
  s = v.y;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float om = __shfl_xor_sync(0xffffffffu, m, o), os = __shfl_xor_sync(0xffffffffu, s, o);
    join_max_sum(m, s, om, os, c);
  }
}

template <typename T>
__global__ void __launch_bounds__(kDistillThreads) distill_kernel(DistillArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int VEC = kVec<T>;
  __shared__ float2 red[32];
  __shared__ float top_p[kDistillTop];
  __shared__ int top_i[kDistillTop];
  __shared__ float fsum[32];
  __shared__ int isum[32];
  if (a.skip_one && a.up && a.up[0] == 1.f) return;
  float mean = 1.f;
  if (a.flags) mean = 1.f / float(max(1, count_flags(a.flags, a.N, isum)));
  const float c = kLog2e / a.temperature;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int row = blockIdx.x; row < a.N; row += gridDim.x) {
    const T* z = static_cast<const T*>(a.z) + row * a.ldz;
    T* g = a.grad ? static_cast<T*>(a.grad) + (long long)row * a.V : nullptr;
    // teacher: entries to shared memory, p over those that are there
    float tm = -INFINITY, ts = 0.f;
    for (int k = threadIdx.x; k < a.K; k += kDistillThreads) {
      const float t = load_as(a.t_type, a.t, (long long)row * a.K + k);
      const long long i = a.idx[(long long)row * a.K + k];
      const bool there = entry_there(t, i, a.V);
      top_i[k] = there ? int(i) : -1;
      top_p[k] = t;
      if (there) join_max_sum(tm, ts, t, 1.f, c);
    }
    block_max_sum(tm, ts, c, red);
    const bool empty = tm == -INFINITY && ts == 0.f;
    const int head = min(a.V, int((16 - (reinterpret_cast<uintptr_t>(z) & 15)) & 15) / int(sizeof(T)));
    const int vecs = (a.V - head) / VEC, tail = head + vecs * VEC;
    float m = -INFINITY, s = 0.f;
    if (a.have_stats) {
      m = a.stats[row].x;
      s = a.stats[row].y;
    } else if (!empty) {
      for (int i = threadIdx.x; i < vecs; i += kDistillThreads) {
        float f[VEC];
        unpack16<T>(*reinterpret_cast<const uint4*>(z + head + i * VEC), f);
        float vm = f[0];
#pragma unroll
        for (int j = 1; j < VEC; ++j) vm = fmaxf(vm, f[j]);
        float vs = 0.f;
#pragma unroll
        for (int j = 0; j < VEC; ++j) vs += f[j] == -INFINITY ? 0.f : exp2f((f[j] - vm) * c);
        join_max_sum(m, s, vm, vs, c);
      }
      for (int i = threadIdx.x; i < head + (a.V - tail); i += kDistillThreads) {
        const float f = to_f32(z[i < head ? i : tail + i - head]);
        if (f != -INFINITY) join_max_sum(m, s, f, 1.f, c);
      }
      block_max_sum(m, s, c, red);
      if (a.stats && threadIdx.x == 0) a.stats[row] = make_float2(m, s);
    }
    const float ln2 = 0.6931471805599453f;
    if (a.loss) {
      float part = 0.f;
      if (!empty)
        for (int k = threadIdx.x; k < a.K; k += kDistillThreads) {
          if (top_i[k] < 0) continue;
          const float lp = (top_p[k] - tm) * c - log2f(ts), p = exp2f(lp);
          const float lq = (to_f32(z[top_i[k]]) - m) * c - log2f(s);
          if (p > 0.f || p != p) part += p * (lp - lq);
        }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
      if (lane == 0) fsum[warp] = part;
      __syncthreads();
      if (threadIdx.x == 0) {
        part = 0.f;
        for (int w = 0; w < kDistillWarps; ++w) part += fsum[w];
        a.loss[row] = part * ln2 * a.temperature * a.temperature;
      }
    }
    if (g) {
      const float w = a.temperature * mean * (a.up ? a.up[a.up_rows ? row : 0] : 1.f);
      if (empty) {
        for (int i = threadIdx.x; i < a.V; i += kDistillThreads) g[i] = from_f32<T>(0.f);
      } else {
        const float k = w / s;
        const bool side = ((reinterpret_cast<uintptr_t>(g) ^ reinterpret_cast<uintptr_t>(z)) & 15) == 0;
        for (int i = threadIdx.x; i < vecs; i += kDistillThreads) {
          float f[VEC];
          unpack16<T>(*reinterpret_cast<const uint4*>(z + head + i * VEC), f);
#pragma unroll
          for (int j = 0; j < VEC; ++j) f[j] = exp2f((f[j] - m) * c) * k;
          if (side) *reinterpret_cast<uint4*>(g + head + i * VEC) = pack16<T>(f);
          else {
#pragma unroll
            for (int j = 0; j < VEC; ++j) g[head + i * VEC + j] = from_f32<T>(f[j]);
          }
        }
        for (int i = threadIdx.x; i < head + (a.V - tail); i += kDistillThreads) {
          const int at = i < head ? i : tail + i - head;
          g[at] = from_f32<T>(exp2f((to_f32(z[at]) - m) * c) * k);
        }
        __syncthreads();
        // the teacher's classes again, from the 32-bit values; a class that comes several times is written by its first entry
        for (int e = threadIdx.x; e < a.K; e += kDistillThreads) {
          const int at = top_i[e];
          if (at < 0) continue;
          float p = 0.f;
          bool first = true;
          for (int o = 0; o < a.K; ++o)
            if (top_i[o] == at) {
              if (o < e) first = false;
              p += exp2f((top_p[o] - tm) * c - log2f(ts));
            }
          if (first) g[at] = from_f32<T>((exp2f((to_f32(z[at]) - m) * c) / s - p) * w);
        }
      }
    }
    __syncthreads();
  }
}

// The mean over the rows that have a teacher, or the sum.
__global__ void __launch_bounds__(1024) distill_reduce_kernel(const float* rows, const unsigned char* flags, int N, float* out) {
  pdl_launch_dependents();
  pdl_wait();
  __shared__ double red[32];
  __shared__ int isum[32];
  double v = 0.0;
  for (int i = threadIdx.x; i < N; i += 1024) v += rows[i];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  const int n = flags ? max(1, count_flags(flags, N, isum)) : 1;
  __syncthreads();
  if (threadIdx.x == 0) {
    v = 0.0;
    for (int w = 0; w < 32; ++w) v += red[w];
    *out = float(v / n);
  }
}

template <typename T>
int distill(DistillArgs a, unsigned char* flags, int fill_flags, float* out, cudaStream_t st) {
  if (flags && fill_flags) {
    const int grid = int(std::min<long long>((a.N + 7) / 8, 8ll * sm_count()));
    LT_RETURN_IF_CUDA(launch_chained(distill_flags_kernel, grid, 256, 0, st, a.t, a.t_type, a.idx, a.N, a.V, a.K, flags));
  }
  a.flags = flags;
  const int grid = std::min(a.N, 4 * sm_count());
  LT_RETURN_IF_CUDA(launch_chained(distill_kernel<T>, grid, kDistillThreads, 0, st, a));
  if (out) LT_RETURN_IF_CUDA(launch_chained(distill_reduce_kernel, 1, 1024, 0, st, static_cast<const float*>(a.loss), static_cast<const unsigned char*>(flags), a.N, out));
  return 0;
}

}  // namespace lt

extern "C" {

// Distillation of student logits z [N, V] (pitch ldz; fp32, bf16 or fp16: type 0, 1, 2) from teacher logits t [N, K] (type t_type) at classes idx [N, K].
//   flags [N] bytes: the loss is a mean over the rows that have a teacher (fill_flags: find them first); null: no mean
//   loss [N] or null; out: their sum or mean, or null; stats [N, 2]: written, or read (have_stats: z is not searched for its maximum again)
//   grad [N, V] or null: times up, which is null (1), one number, or (up_rows) one for every row; skip_one: nothing is done where up is one number and it is 1
int lt_distill(int type, const void* z, long long ldz, int t_type, const void* t, const long long* idx, int N, int V, int K, float temperature, unsigned char* flags, int fill_flags,
               const float* up, int up_rows, int skip_one, float* stats, int have_stats, float* loss, float* out, void* grad, void* stream) {
  using namespace lt;
  if (type < 0 || type > 2 || t_type < 0 || t_type > 2 || N < 0 || V < 1 || K < 1 || K > kDistillTop || !(temperature > 0.f) || (out && !loss)) return -int(kStatusBadArgument);
  if (N == 0) return 0;
  DistillArgs a{z, ldz, t, t_type, idx, N, V, K, temperature, nullptr, up, up_rows, skip_one, reinterpret_cast<float2*>(stats), have_stats, loss, grad};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (type == kElemF32) return distill<float>(a, flags, fill_flags, out, st);
  if (type == kElemBf16) return distill<__nv_bfloat16>(a, flags, fill_flags, out, st);
  return distill<__half>(a, flags, fill_flags, out, st);
}

}  // extern "C"
