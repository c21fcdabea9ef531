// Tokens drawn from rows of logits with temperature, top-k, top-p and min-p, by one given random number a row.
//
//   w_j = e^((z_j - max z) / tau);  tokens stand in order of their logit, of equals the lowest index first
//   top-k: the first k stay;  top-p: those stay whose predecessors' mass is below p times the mass of what stayed;  min-p: those stay with w_j >= min_p
//   token = the first index at which the cumulated mass of what stays (in index order) exceeds u times all of it
//
// The result is a choice, so it must not depend on the order in which the GPU adds.  Weights are whole numbers of 2^-44 (from 64-bit exponentials):
// their sums are exact in 64 bits for up to 2^19 tokens, in any order, and the masses next to a border are off by less than 2^-45 for each token before it.
//
// A cluster of CTAs takes a row.  Limits in the order are found by radix selection on order-preserving keys of the logits: a histogram of counts
// (top-k) or of masses (top-p) over the next 11 bits of the keys that share the bits found so far.
#include "lt_cuda.h"

#include "common/elem.cuh"
#include "common/host.h"
#include "common/ptx.cuh"

namespace lt {

constexpr int kSampleThreads = 512, kSampleWarps = kSampleThreads / 32, kSampleBins = 2048, kSampleCluster = 8;
constexpr double kMassOne = 17592186044416.0;                 // 2^44

struct SampleArgs {
  const void* z;
  long long ldz;
  const void* u;                // [rows] fp32 or fp64
  int u64bit;
  const float *tau, *top_p, *min_p;      // [rows], or null: the numbers below
  const int* top_k;
  double tau1, top_p1, min_p1;
  int top_k1;
  int rows, V, ctas;
  long long* tokens;
  float* logprobs;              // or null
};

// Keys in the order of the values; NaN stands with -inf, -0 with 0.
template <typename T> struct Key {
  static constexpr int kBits = 32;
  static __device__ __forceinline__ uint32_t of(float f) {
    const uint32_t b = __float_as_uint(f == 0.f ? 0.f : f);
    return (b & 0x80000000u) ? ~b : b | 0x80000000u;
  }
  static __device__ __forceinline__ float value(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? k & 0x7fffffffu : ~k); }
};
template <> struct Key<__nv_bfloat16> {
  static constexpr int kBits = 16;
  static __device__ __forceinline__ uint32_t of(float f) { return Key<float>::of(f) >> 16; }
  static __device__ __forceinline__ float value(uint32_t k) {
    const uint32_t b = (k & 0x8000u) ? k & 0x7fffu : ~k & 0xffffu;
    return __uint_as_float(b << 16);
  }
};
template <> struct Key<__half> {
  static constexpr int kBits = 16;
  static __device__ __forceinline__ uint32_t of(float f) {
    const uint32_t b = f == 0.f ? 0u : __half_as_ushort(__float2half_rn(f));
    return (b & 0x8000u) ? ~b & 0xffffu : b | 0x8000u;
  }
  static __device__ __forceinline__ float value(uint32_t k) { return __half2float(__ushort_as_half((unsigned short)((k & 0x8000u) ? k & 0x7fffu : ~k & 0xffffu))); }
};

typedef unsigned long long u64;

__device__ __forceinline__ u64 mass_of(float z, float m, double inv_tau) {
  if (!(z > -INFINITY)) return 0ull;
  if (z == m) return u64(kMassOne);
  const double x = (double(z) - double(m)) * inv_tau;
  return x > -31.5 ? u64(rint(exp(x) * kMassOne)) : 0ull;     // (e^-31.5 is below half of 2^-44)
}
__device__ __forceinline__ u64 warp_add64(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <typename T>
__global__ void __launch_bounds__(kSampleThreads) sample_kernel(SampleArgs a) {
  constexpr int VEC = kVec<T>;
  __shared__ uint32_t hist[kSampleBins];
  __shared__ u64 mass[kSampleBins];
  __shared__ u64 part[2];                                     // what the other CTAs of the cluster read
  __shared__ u64 wsum[kSampleWarps];
  __shared__ uint32_t wcnt[kSampleWarps];
  __shared__ u64 found[3];
  pdl_launch_dependents();
  pdl_wait();
  const int C = a.ctas, rank = C > 1 ? int(cluster_ctarank()) : 0;
  const int row = blockIdx.x / C;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const T* z = static_cast<const T*>(a.z) + row * a.ldz;
  auto everywhere = [&] {                                     // all CTAs of the row are here, and see what was written before
    if (C > 1) cluster_sync_all();
    else __syncthreads();
  };

  double tau = a.tau ? double(a.tau[row]) : a.tau1;
  double p = a.top_p ? double(a.top_p[row]) : a.top_p1;
  const double low = a.min_p ? double(a.min_p[row]) : a.min_p1;
  int k = a.top_k ? a.top_k[row] : a.top_k1;
  if (!(tau > 0.0)) { k = 1; tau = 1.0; }
  if (k == 1) p = 1.0;
  const double inv_tau = 1.0 / tau;
  const u64 least = low > 0.0 ? u64(ceil(fmin(low, 1.0) * kMassOne)) : 0ull;

  // vectors of the row: [vlo, vhi) are this warp's, and of all warps of all CTAs in index order
  const int shift = int(reinterpret_cast<uintptr_t>(z) & 15) / int(sizeof(T));
  const int vecs = (a.V + shift + VEC - 1) / VEC;
  const int vcta = (vecs + C - 1) / C, vwarp = (vcta + kSampleWarps - 1) / kSampleWarps;
  const int cend = min(vecs, (rank + 1) * vcta);
  const int vlo = min(cend, rank * vcta + warp * vwarp), vhi = min(cend, vlo + vwarp);
  auto load = [&](int v, float (&f)[VEC]) {
    const int lo = v * VEC - shift;
    if (lo >= 0 && lo + VEC <= a.V) {
      unpack16<T>(*reinterpret_cast<const uint4*>(z + lo), f);
#pragma unroll
      for (int j = 0; j < VEC; ++j) f[j] = f[j] == f[j] ? f[j] : -INFINITY;
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        f[j] = lo + j >= 0 && lo + j < a.V ? to_f32(z[lo + j]) : -INFINITY;
        f[j] = f[j] == f[j] ? f[j] : -INFINITY;
      }
    }
  };

  // ---- the maximum
  float m = -INFINITY;
  for (int v = vlo + lane; v < vhi; v += 32) {
    float f[VEC];
    load(v, f);
#pragma unroll
    for (int j = 0; j < VEC; ++j) m = fmaxf(m, f[j]);
  }
  uint32_t top = __reduce_max_sync(0xffffffffu, Key<float>::of(m));
  if (lane == 0) wcnt[warp] = top;
  __syncthreads();
  for (int w = 0; w < kSampleWarps; ++w) top = max(top, wcnt[w]);
  if (C > 1) {
    if (threadIdx.x == 0) part[0] = top;
    cluster_sync_all();
    for (int c = 0; c < C; ++c) top = max(top, uint32_t(*cluster_peer(part, c)));
    cluster_sync_all();
  }
  m = Key<float>::value(top);
  if (m == -INFINITY) {
    if (rank == 0 && threadIdx.x == 0) {
      a.tokens[row] = -1;
      if (a.logprobs) a.logprobs[row] = -INFINITY;
    }
    return;
  }

  // Sum of v over the threads of all CTAs, for all of them.
  auto sum_all = [&](u64 v) {
    v = warp_add64(v);
    __syncthreads();
    if (lane == 0) wsum[warp] = v;
    __syncthreads();
    v = 0;
    for (int w = 0; w < kSampleWarps; ++w) v += wsum[w];
    if (C > 1) {
      if (threadIdx.x == 0) part[0] = v;
      cluster_sync_all();
      v = 0;
      for (int c = 0; c < C; ++c) v += *cluster_peer(part, c);
      cluster_sync_all();
    }
    return v;
  };

  // What stays: keys above `limit`, and the first `ties` of those at it.
  uint32_t limit = 0;
  u64 ties = ~0ull, all = 0;                                  // all: mass of what stays after top-k
  constexpr int kBits = Key<T>::kBits;
  constexpr int kDigit = 11;
  // The key at which the running sum over keys from the top (counts, or masses with the first `ties` of those at `limit`) reaches `want`, and the sum above it.
  auto select = [&](bool by_mass, u64 want, u64& above) {
    uint32_t prefix = 0;
    above = 0;
    for (int left = kBits; left > 0;) {
      const int bits = min(kDigit, left), sh = left - bits;
      const uint32_t low_mask = (1u << bits) - 1u;
      for (int i = threadIdx.x; i < kSampleBins; i += kSampleThreads) {
        hist[i] = 0u;
        if (by_mass) mass[i] = 0ull;
      }
      __syncthreads();
      for (int v = vlo + lane; v < vhi; v += 32) {
        float f[VEC];
        load(v, f);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const uint32_t key = Key<T>::of(f[j]);
          if (f[j] == -INFINITY || (left < 32 && (key >> (left & 31)) != prefix)) continue;
          if (!by_mass) atomicAdd(&hist[(key >> sh) & low_mask], 1u);
          else if (key > limit || (key == limit && ties == ~0ull)) {
            const u64 w = mass_of(f[j], m, inv_tau);
            if (w) atomicAdd(&mass[(key >> sh) & low_mask], w);
          }
        }
      }
      if (by_mass && ties != ~0ull && rank == 0 && threadIdx.x == 0 && (left >= 32 || (limit >> (left & 31)) == prefix))
        atomicAdd(&mass[(limit >> sh) & low_mask], ties * mass_of(Key<T>::value(limit), m, inv_tau));
      everywhere();
      // bins from the top, 2048 / threads to a thread
      constexpr int PER = kSampleBins / kSampleThreads;
      u64 v[PER], own = 0;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int bin = kSampleBins - 1 - (int(threadIdx.x) * PER + i);
        v[i] = 0;
        for (int c = 0; c < C; ++c) v[i] += by_mass ? (C > 1 ? *cluster_peer(mass + bin, c) : mass[bin]) : u64(C > 1 ? *cluster_peer(hist + bin, c) : hist[bin]);
        own += v[i];
      }
      u64 incl = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const u64 x = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += x;
      }
      if (lane == 31) wsum[warp] = incl;
      __syncthreads();
      u64 before = above + incl - own;
      for (int w = 0; w < warp; ++w) before += wsum[w];
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        if (before < want && want <= before + v[i]) {
          found[0] = u64(kSampleBins - 1 - (int(threadIdx.x) * PER + i));
          found[1] = before;
        }
        before += v[i];
      }
      everywhere();
      prefix = (prefix << bits) | uint32_t(found[0]);
      above = found[1];
      left = sh;
      __syncthreads();
    }
    return prefix;
  };

  // ---- top-k
  if (k > 0 && k < a.V) {
    u64 have = 0;
    if (k == 1) {
      limit = Key<T>::of(m);
      ties = 1;
    } else {
      for (int v = vlo + lane; v < vhi; v += 32) {
        float f[VEC];
        load(v, f);
#pragma unroll
        for (int j = 0; j < VEC; ++j) have += f[j] != -INFINITY;
      }
      if (sum_all(have) > u64(k)) {
        u64 above;
        limit = select(false, u64(k), above);
        ties = u64(k) - above;
      }
    }
  }
  // ---- top-p
  if (p < 1.0) {
    u64 own = 0;
    for (int v = vlo + lane; v < vhi; v += 32) {
      float f[VEC];
      load(v, f);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const uint32_t key = Key<T>::of(f[j]);
        if (key > limit || (key == limit && ties == ~0ull)) own += mass_of(f[j], m, inv_tau);
      }
    }
    if (ties != ~0ull && rank == 0 && threadIdx.x == 0) own += ties * mass_of(Key<T>::value(limit), m, inv_tau);
    all = sum_all(own);
    const u64 want = max(1ull, u64(ceil(fmax(p, 0.0) * double(all))));     // (the first always stays)
    u64 above;
    const uint32_t key = select(true, min(want, all), above);
    const u64 w = mass_of(Key<T>::value(key), m, inv_tau);
    limit = key;
    ties = (min(want, all) - above + w - 1) / w;
  }

  // ---- the draw
  const u64 tie_w = ties == ~0ull ? 0ull : mass_of(Key<T>::value(limit), m, inv_tau);
  const bool tie_in = tie_w >= least && tie_w > 0;
  auto stays = [&](float f, uint32_t key) -> u64 {            // mass of an element that stays whatever its place among equals
    if (!(key > limit || (key == limit && ties == ~0ull))) return 0ull;
    const u64 w = mass_of(f, m, inv_tau);
    return w >= least ? w : 0ull;
  };
  u64 sum = 0;
  uint32_t tied = 0;
  for (int v = vlo + lane; v < vhi; v += 32) {
    float f[VEC];
    load(v, f);
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const uint32_t key = Key<T>::of(f[j]);
      sum += stays(f[j], key);
      tied += tie_in && key == limit;
    }
  }
  sum = warp_add64(sum);
  tied = __reduce_add_sync(0xffffffffu, tied);
  __syncthreads();
  if (lane == 0) { wsum[warp] = sum; wcnt[warp] = tied; }
  __syncthreads();
  u64 csum = 0, ctied = 0;
  for (int w = 0; w < kSampleWarps; ++w) { csum += wsum[w]; ctied += wcnt[w]; }
  if (threadIdx.x == 0) { part[0] = csum; part[1] = ctied; }
  everywhere();
  u64 before = 0, ties_before = 0, total = 0, seen = 0;
  for (int c = 0; c < C; ++c) {
    const u64* q = C > 1 ? cluster_peer(part, c) : part;
    const u64 t = q[1], kept = tie_in ? min(t, ties > seen ? ties - seen : 0ull) : 0ull;
    const u64 x = q[0] + kept * tie_w;
    if (c < rank) { before += x; ties_before += t; }
    total += x;
    seen += t;
  }
  if (C > 1) cluster_sync_all();                              // a CTA's shared memory is read until here
  double u = a.u64bit ? static_cast<const double*>(a.u)[row] : double(static_cast<const float*>(a.u)[row]);
  u = u > 0.0 ? fmin(u, 1.0) : 0.0;
  const u64 target = min(u64(u * double(total)), total - 1);
  // this warp's mass
  for (int w = 0; w < warp; ++w) {
    const u64 t = wcnt[w], kept = tie_in ? min(t, ties > ties_before ? ties - ties_before : 0ull) : 0ull;
    before += wsum[w] + kept * tie_w;
    ties_before += t;
  }
  {
    const u64 kept = tie_in ? min(u64(tied), ties > ties_before ? ties - ties_before : 0ull) : 0ull;
    if (target < before || target >= before + sum + kept * tie_w) return;
  }
  for (int v0 = vlo; v0 < vhi; v0 += 32) {
    const int v = v0 + lane;
    float f[VEC];
    u64 w[VEC], own = 0;
    uint32_t eq = 0;
    if (v < vhi) load(v, f);
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const uint32_t key = v < vhi ? Key<T>::of(f[j]) : 0u;
      w[j] = v < vhi ? stays(f[j], key) : 0ull;
      eq += v < vhi && tie_in && key == limit;
    }
    uint32_t eq_incl = eq;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t x = __shfl_up_sync(0xffffffffu, eq_incl, o);
      if (lane >= o) eq_incl += x;
    }
    u64 nth = ties_before + eq_incl - eq;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      if (v < vhi && tie_in && Key<T>::of(f[j]) == limit) {
        if (nth < ties) w[j] = tie_w;
        ++nth;
      }
      own += w[j];
    }
    u64 incl = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 x = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += x;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, before + incl > target);
    if (hit) {
      if (lane == __ffs(hit) - 1) {
        u64 at = before + incl - own;
        bool done = false;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          at += w[j];
          if (!done && at > target) {
            done = true;
            a.tokens[row] = (long long)v * VEC - shift + j;
            if (a.logprobs) a.logprobs[row] = float((f[j] == m ? 0.0 : (double(f[j]) - double(m)) * inv_tau) - log(double(total) / kMassOne));
          }
        }
      }
      return;
    }
    before += __shfl_sync(0xffffffffu, incl, 31);
    ties_before += __shfl_sync(0xffffffffu, eq_incl, 31);
  }
}

}  // namespace lt

extern "C" {

// tokens[rows] (64-bit) and, if not null, logprobs[rows] of logits z [rows, V] (pitch ldz; fp32, bf16 or fp16: type 0, 1, 2) by the random numbers u [rows]
// (fp32, or fp64: u64bit), with a temperature, top_k, top_p and min_p for every row or (null) one for all.  tau <= 0: the largest; top_k <= 0, top_p >= 1 and
// min_p <= 0: off.  A row without any finite logit gets -1.  NaN counts as -inf.
int lt_sample_tokens(int type, const void* z, long long ldz, const void* u, int u64bit, const float* tau, const int* top_k, const float* top_p, const float* min_p,
                     double tau1, int top_k1, double top_p1, double min_p1, int rows, int V, long long* tokens, float* logprobs, void* stream) {
  using namespace lt;
  if (type < 0 || type > 2 || rows < 0 || V < 1 || V > (1 << 19)) return -int(kStatusBadArgument);
  if (rows == 0) return 0;
  int ctas = 1;
  while (ctas < kSampleCluster && (long long)rows * ctas * 2 <= 2 * sm_count() && V / ctas >= 8192) ctas *= 2;
  if ((long long)rows * ctas > 0x7fffffffll) return -int(kStatusBadArgument);
  SampleArgs a{z, ldz, u, u64bit, tau, top_p, min_p, top_k, tau1, top_p1, min_p1, top_k1, rows, V, ctas, tokens, logprobs};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto kernel = type == kElemF32 ? sample_kernel<float> : type == kElemBf16 ? sample_kernel<__nv_bfloat16> : sample_kernel<__half>;
  if (ctas > 1) LT_RETURN_IF_CUDA(launch_chained_clusters(kernel, rows * ctas, kSampleThreads, 0, ctas, st, a));
  else LT_RETURN_IF_CUDA(launch_chained(kernel, rows, kSampleThreads, 0, st, a));
  return 0;
}

}  // extern "C"
