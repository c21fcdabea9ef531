// Tokens drawn from rows of logits with temperature, top-k, top-p and min-p, by one given random number a row.
//
//   w_j = e^((z_j - max z) / tau);  tokens stand in order of their logit, of equals the lowest index first
//   top-k: the first k stay;  top-p: those stay whose predecessors' mass is below p times the mass of what stayed;  min-p: those stay with w_j >= min_p
//   token = the first index at which the cumulated mass of what stays (in index order) exceeds u times all of it
//
// The result is a choice, so it must not depend on the order in which the GPU adds.  Weights are whole numbers of 2^-44, so that their sums are exact in 64 bits for up
// to 2^19 tokens, in any order.  Each is off by up to 2^-42.6 of itself (the series of its exponential, always too small) and by half of 2^-44: what weighs less than 2^-45 of
// the largest weighs nothing, and a border lies within 2^-42.6 of the mass before it and 2^-45 for each token there of where exact weights would have it.
//
// A cluster of CTAs takes a row.  Limits in the order are found by selection on order-preserving keys of the logits: a histogram of counts
// (top-k) or of masses (top-p) over up to 1024 equal pieces of the interval of keys that is left, until pieces are single keys.
#include "lt_cuda.h"

#include "common/elem.cuh"
#include "common/host.h"
#include "common/ptx.cuh"

namespace lt {

constexpr int kSampleThreads = 512, kSampleWarps = kSampleThreads / 32, kSampleBins = 1024, kSampleCluster = 8;
constexpr int kSampleHold = 80 * 1024;                        // bytes of a row that a CTA holds at most: two share an SM
constexpr int kSampleFew = 256;                               // tokens that are compared each with each
constexpr int kSampleGroups = 512;                            // maxima of groups of tokens
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
  int rows, V, ctas, held;
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

// What the weights of a row go by.
struct Weigh {
  float m, cut;                 // the largest logit; below the other one weights are nothing (-45.5 powers of two)
  double md, k;                 // the largest logit, log2(e) / tau
};
// 2^44 times the weight of a logit, to the nearest whole number: 2^y with y = 16ths + r, |r| <= 1/32, the 16ths from a table, 2^r by the exponential series up to the
// fifth power (the next term is below 2^-42.6).  Adding 256 to the weight leaves the whole number in the low bits of the sum.  No branches: the compiler works at
// several at once, each of which is a long chain.  Of an infinite largest logit only its equals weigh anything.
__device__ __forceinline__ u64 mass_of(float z, const Weigh& q, const double* table) {
  const double y = (double(z) - q.md) * q.k;                  // (the difference first: it is exact, and 0 for the largest)
  const double shifted = fma(y, 16.0, 6755399441055744.0);    // (1.5 2^52: the sum's low bits are 16 y rounded)
  const int n = __double2loint(shifted);
  const double r = fma(shifted - 6755399441055744.0, -0.0625, y), t = table[n & 15];
  constexpr double L = 0.693147180559945309417232121458;
  double p = fma(r, L * L * L * L * L / 120.0, L * L * L * L / 24.0);
  p = fma(p, r, L * L * L / 6.0);
  p = fma(p, r, L * L / 2.0);
  p = fma(p, r, L);
  p = fma(fma(p, r, 1.0), __hiloint2double(__double2hiint(t) + (n & ~15) * 65536, __double2loint(t)), 256.0);
  const u64 w = u64(__double_as_longlong(p)) & 0xfffffffffffffull;
  return z >= q.cut ? q.m == INFINITY ? u64(kMassOne) : w : 0ull;
}
__device__ __forceinline__ u64 warp_add64(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ u64 warp_scan64(u64 v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 x = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += x;
  }
  return v;
}
// Logits with -inf in the place of NaN.
template <typename T> __device__ __forceinline__ uint4 no_nan(uint4 u) {
  if constexpr (sizeof(T) == 4) {
    return make_uint4(__float_as_uint(fmaxf(__uint_as_float(u.x), -INFINITY)), __float_as_uint(fmaxf(__uint_as_float(u.y), -INFINITY)),
                      __float_as_uint(fmaxf(__uint_as_float(u.z), -INFINITY)), __float_as_uint(fmaxf(__uint_as_float(u.w), -INFINITY)));
  } else {
    uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (__is_same(T, __nv_bfloat16)) {
        const __nv_bfloat162 h = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&w[i]), __floats2bfloat162_rn(-INFINITY, -INFINITY));
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __half2 h = __hmax2(*reinterpret_cast<const __half2*>(&w[i]), __floats2half2_rn(-INFINITY, -INFINITY));
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
}

struct SampleShared {
  uint32_t hist[kSampleBins];
  // of the general way: sums over the cluster, and a CTA's histograms (counts, or 15 bits of the masses each; 64-bit atomics are loops)
  u64 sums[kSampleBins];        // the short list's tokens and weights lie in the same place
  uint32_t mid[kSampleBins], high[kSampleBins];
  u64 part[2];                  // what the other CTAs of the cluster read
  u64 wsum[kSampleWarps];
  uint32_t wcnt[kSampleWarps];
  u64 found[2];
  double table[16];
  double k, top_p, low;         // log2(e) / tau and limits of the row
  u64 least;
  float from[2];                // what lies below does not stay for the limits in the order, or for min-p either
  double tau;
  uint32_t groups[kSampleGroups];
  uint32_t count;               // of the short list (the first CTA's)
};

// A row of a cluster of CTAs: where its vectors lie.  [vlo, vhi) are this warp's, and of all warps of all CTAs in index order.
template <typename T>
struct SampleRow {
  static constexpr int VEC = kVec<T>;
  const T* z;
  const uint4* held;            // vector 0 of the row, if it were in this CTA's shared memory as the CTA's own vectors are; null: they are read from z again
  int shift, V, vlo, vhi;
  __device__ __forceinline__ bool whole(int v) const { return v * VEC >= shift && v * VEC - shift + VEC <= V; }
  __device__ __forceinline__ uint4 fetch(int v) const {
    const int lo = v * VEC - shift;
    if (whole(v)) return *reinterpret_cast<const uint4*>(z + lo);
    float f[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) f[j] = lo + j >= 0 && lo + j < V ? to_f32(z[lo + j]) : -INFINITY;
    return pack16<T>(f);
  }
  __device__ __forceinline__ uint4 raw(int v) const { return held ? held[v] : fetch(v); }
  __device__ __forceinline__ uint4 load(int v) const { return no_nan<T>(raw(v)); }
  // f(logits, vector) for this warp's vectors
  template <class F>
  __device__ __forceinline__ void each(int lane, F f) const {
#pragma unroll 2
    for (int v = vlo + lane; v < vhi; v += 32) {
      float x[VEC];
      unpack16<T>(load(v), x);
      f(x, v);
    }
  }
};

struct Filters {
  int k;
  double p;
  u64 least;
};

// The cumulated mass that the drawn token's exceeds.
__device__ __forceinline__ u64 draw_target(const SampleArgs& a, int row, u64 total) {
  double u = a.u64bit ? static_cast<const double*>(a.u)[row] : double(static_cast<const float*>(a.u)[row]);
  u = u > 0.0 ? fmin(u, 1.0) : 0.0;
  return min(u64(u * double(total)), total - 1);
}
__device__ __forceinline__ void write_token(const SampleArgs& a, int row, int token, float z, const Weigh& q, u64 total) {
  a.tokens[row] = token;
  if (a.logprobs) a.logprobs[row] = float(((z == q.m ? 0.0 : (double(z) - q.md) * q.k) - log2(double(total) / kMassOne)) * 0.693147180559945309417232121458);
}

// n tokens in list (key and token): who stays, and which of them is drawn.
template <typename T>
__device__ __forceinline__ void short_list(const SampleArgs& a, int row, const Weigh& q, const Filters& by, int n, u64* list, SampleShared& sh) {
  u64* weight = list + kSampleFew;
  u64* mass_before = weight + kSampleFew;
  const int lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < n; i += blockDim.x) weight[i] = mass_of(Key<T>::value(uint32_t(list[i] >> 32)), q, sh.table);
  __syncthreads();
  // a quarter of a warp to a token: its place in the order, and the mass of those in front of it
  for (int i0 = threadIdx.x >> 3; i0 - (lane >> 3) < n; i0 += blockDim.x >> 3) {
    const int i = min(i0, n - 1);
    const u64 mine = list[i];
    uint32_t place = 0;
    u64 before = 0;
    for (int o = lane & 7; o < n; o += 8) {
      const u64 other = list[o];
      // greater key, or the same and a lower token
      const bool ahead = (other >> 32) > (mine >> 32) || ((other >> 32) == (mine >> 32) && uint32_t(other) < uint32_t(mine));
      place += ahead;
      before += ahead ? weight[o] : 0ull;
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
      place += __shfl_xor_sync(0xffffffffu, place, o);
      before += __shfl_xor_sync(0xffffffffu, before, o);
    }
    if (i0 < n && (lane & 7) == 0) {
      mass_before[i] = by.k <= 0 || place < uint32_t(by.k) ? before : ~0ull;       // (~0: does not stay)
      if (by.k > 0 && place + 1 == uint32_t(min(by.k, n))) sh.found[0] = before + weight[i];       // the mass of the first k
    }
  }
  __syncthreads();
  u64 want = ~0ull;
  if (by.p < 1.0) {
    const u64 all = by.k > 0 ? sh.found[0] : sh.found[1];
    want = max(1ull, u64(ceil(fmax(by.p, 0.0) * double(all))));
  }
  for (int i = threadIdx.x; i < n; i += blockDim.x)
    if (!(mass_before[i] < want) || weight[i] < by.least) weight[i] = 0;
  __syncthreads();
  // cumulated masses in the order of the tokens' numbers
  u64 total = 0;
  for (int i = lane; i < n; i += 32) total += weight[i];
  total = warp_add64(total);
  const u64 target = draw_target(a, row, total);
  for (int i0 = threadIdx.x >> 3; i0 - (lane >> 3) < n; i0 += blockDim.x >> 3) {
    const int i = min(i0, n - 1);
    const uint32_t token = uint32_t(list[i]);
    u64 before = 0;
    for (int o = lane & 7; o < n; o += 8) before += uint32_t(list[o]) < token ? weight[o] : 0ull;
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
    if (i0 < n && (lane & 7) == 0 && before <= target && target < before + weight[i]) write_token(a, row, int(token), Key<T>::value(uint32_t(list[i] >> 32)), q, total);
  }
}

// The general way, for filters that leave many tokens: every step goes over the row again (in L2).
// `bound`: tokens below it do not stay for top-k and top-p.  mass: that of all tokens, if top-p is the only limit.
template <typename T>
__device__ __noinline__ void sample_general(const SampleArgs& a, const SampleRow<T>& r, const Weigh& q, const Filters& by, float bound, u64 mass, int row, int rank,
                                            SampleShared& sh) {
  constexpr int VEC = kVec<T>;
  const int C = a.ctas, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = blockDim.x >> 5;
  auto everywhere = [&] {                                     // all CTAs of the row are here, and see what was written before
    if (C > 1) cluster_sync_all();
    else __syncthreads();
  };
  // Sum of v over the threads of all CTAs, for all of them.
  auto sum_all = [&](u64 v) {
    v = warp_add64(v);
    __syncthreads();
    if (lane == 0) sh.wsum[warp] = v;
    __syncthreads();
    v = 0;
    for (int w = 0; w < nw; ++w) v += sh.wsum[w];
    if (C > 1) {
      if (threadIdx.x == 0) sh.part[0] = v;
      cluster_sync_all();
      v = 0;
      for (int c = 0; c < C; ++c) v += *cluster_peer(sh.part, c);
      cluster_sync_all();
    }
    return v;
  };
  // What stays: keys above `limit`, and the first `ties` of those at it.
  uint32_t limit = 0;
  u64 ties = ~0ull;
  const uint32_t key_lo = Key<T>::of(bound), key_hi = Key<T>::of(q.m);
  // The key at which the running sum over keys from the top (counts, or masses with the first `ties` of those at `limit`) reaches `want`, and the sum above it:
  // the interval of the keys is cut into up to 1024 pieces until they are single keys.
  auto select = [&](bool by_mass, u64 want, u64& above) {
    uint32_t lo = key_lo, hi = key_hi;
    above = 0;
    for (;;) {
      const int width = 32 - __clz(int(hi - lo)), cut = max(0, width - 10);
      for (int i = threadIdx.x; i < kSampleBins; i += blockDim.x) {
        sh.hist[i] = sh.mid[i] = sh.high[i] = 0u;
      }
      __syncthreads();
      r.each(lane, [&](const float (&z)[VEC], int) {
        uint32_t key[VEC];
        bool in[VEC], any = false;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          key[j] = Key<T>::of(z[j]);
          in[j] = z[j] != -INFINITY && key[j] >= lo && key[j] <= hi && (!by_mass || key[j] > limit || (key[j] == limit && ties == ~0ull));
          any = any || in[j];
        }
        if (!any) return;
        if (by_mass && cut > 0) {
          u64 w[VEC];
#pragma unroll
          for (int j = 0; j < VEC; ++j) w[j] = mass_of(z[j], q, sh.table);
#pragma unroll
          for (int j = 0; j < VEC; ++j)
            if (in[j] && w[j]) {
              const uint32_t at = (key[j] - lo) >> cut;
              atomicAdd(&sh.hist[at], uint32_t(w[j]) & 0x7fffu);
              atomicAdd(&sh.mid[at], uint32_t(w[j] >> 15) & 0x7fffu);
              if (w[j] >> 30) atomicAdd(&sh.high[at], uint32_t(w[j] >> 30));
            }
        } else {
#pragma unroll
          for (int j = 0; j < VEC; ++j)
            if (in[j]) atomicAdd(&sh.hist[(key[j] - lo) >> cut], 1u);
        }
      });
      everywhere();
      // every CTA adds up its share of the bins over the cluster, and gives the sums to all
      {
        const int share = kSampleBins / C;
        for (int i = threadIdx.x; i < share; i += blockDim.x) {
          const int at = rank * share + i;
          u64 v[kSampleCluster], sum = 0;
#pragma unroll
          for (int c = 0; c < kSampleCluster; ++c) {
            v[c] = 0;
            if (c < C) {
              v[c] = C > 1 ? *cluster_peer(sh.hist + at, c) : sh.hist[at];
              if (by_mass && cut > 0) v[c] += (u64(C > 1 ? *cluster_peer(sh.mid + at, c) : sh.mid[at]) << 15) + (u64(C > 1 ? *cluster_peer(sh.high + at, c) : sh.high[at]) << 30);
            }
          }
#pragma unroll
          for (int c = 0; c < kSampleCluster; ++c) sum += v[c];
          if (by_mass) {
            const bool at_limit = ties != ~0ull && limit >= lo && limit <= hi && (limit - lo) >> cut == uint32_t(at);
            if (cut == 0 && sum) sum *= mass_of(Key<T>::value(lo + uint32_t(at)), q, sh.table);       // equal logits
            if (at_limit) sum += ties * mass_of(Key<T>::value(limit), q, sh.table);
          }
#pragma unroll
          for (int c = 0; c < kSampleCluster; ++c)
            if (c < C) *(C > 1 ? cluster_peer(sh.sums + at, c) : sh.sums + at) = sum;
        }
      }
      everywhere();
      // bins from the top, 1024 / threads to a thread
      const int per = kSampleBins / int(blockDim.x);
      auto bin = [&](int i) {
        const int at = kSampleBins - 1 - (int(threadIdx.x) * per + i);
        return sh.sums[at];
      };
      u64 own = 0;
      for (int i = 0; i < per; ++i) own += bin(i);
      const u64 incl = warp_scan64(own, lane);
      if (lane == 31) sh.wsum[warp] = incl;
      if (threadIdx.x == 0) { sh.found[0] = 0; sh.found[1] = above; }        // (always found below; whatever the sums say, the interval becomes shorter)
      __syncthreads();
      u64 before = above + incl - own;
      for (int w = 0; w < warp; ++w) before += sh.wsum[w];
      if (before < want && want <= before + own)
        for (int i = 0; i < per; ++i) {
          const u64 v = bin(i);
          if (before < want && want <= before + v) {
            sh.found[0] = u64(kSampleBins - 1 - (int(threadIdx.x) * per + i));
            sh.found[1] = before;
          }
          before += v;
        }
      __syncthreads();
      lo += uint32_t(sh.found[0]) << cut;
      above = sh.found[1];
      __syncthreads();
      if (cut == 0) return lo;
      hi = min(hi, lo + ((1u << cut) - 1u));
    }
  };

  if (by.k > 0 && by.k < a.V) {
    u64 have = 0;
    r.each(lane, [&](const float (&z)[VEC], int) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) have += z[j] != -INFINITY;
    });
    if (sum_all(have) > u64(by.k)) {
      u64 above;
      limit = select(false, u64(by.k), above);
      ties = u64(by.k) - above;
    }
  }
  if (by.p < 1.0) {
    u64 all = mass;
    if (by.k > 0) {
      u64 own = 0;
      r.each(lane, [&](const float (&z)[VEC], int) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const uint32_t key = Key<T>::of(z[j]);
          const u64 w = mass_of(z[j], q, sh.table);
          own += key > limit || (key == limit && ties == ~0ull) ? w : 0ull;
        }
      });
      if (ties != ~0ull && rank == 0 && threadIdx.x == 0) own += ties * mass_of(Key<T>::value(limit), q, sh.table);
      all = sum_all(own);
    }
    const u64 want = min(all, max(1ull, u64(ceil(fmax(by.p, 0.0) * double(all)))));       // (the first always stays)
    u64 above;
    limit = select(true, want, above);
    const u64 w = mass_of(Key<T>::value(limit), q, sh.table);
    ties = (want - above + w - 1) / w;
  }

  // the draw
  const u64 tie_w = ties == ~0ull ? 0ull : mass_of(Key<T>::value(limit), q, sh.table);
  const bool tie_in = tie_w >= by.least && tie_w > 0;
  auto stays = [&](float f, uint32_t key) -> u64 {            // mass of an element that stays whatever its place among equals
    const u64 w = mass_of(f, q, sh.table);
    return w >= by.least && (key > limit || (key == limit && ties == ~0ull)) ? w : 0ull;
  };
  u64 sum = 0;
  uint32_t tied = 0;
  r.each(lane, [&](const float (&z)[VEC], int) {
    bool any = false;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const uint32_t key = Key<T>::of(z[j]);
      any = any || key > limit || (key == limit && ties == ~0ull);
      tied += tie_in && key == limit;
    }
    if (!any) return;
#pragma unroll
    for (int j = 0; j < VEC; ++j) sum += stays(z[j], Key<T>::of(z[j]));
  });
  sum = warp_add64(sum);
  tied = __reduce_add_sync(0xffffffffu, tied);
  __syncthreads();
  if (lane == 0) { sh.wsum[warp] = sum; sh.wcnt[warp] = tied; }
  __syncthreads();
  u64 csum = 0, ctied = 0;
  for (int w = 0; w < nw; ++w) { csum += sh.wsum[w]; ctied += sh.wcnt[w]; }
  if (threadIdx.x == 0) { sh.part[0] = csum; sh.part[1] = ctied; }
  everywhere();
  u64 before = 0, ties_before = 0, total = 0, seen = 0;
  for (int c = 0; c < C; ++c) {
    const u64* o = C > 1 ? cluster_peer(sh.part, c) : sh.part;
    const u64 t = o[1], kept = tie_in ? min(t, ties > seen ? ties - seen : 0ull) : 0ull;
    const u64 x = o[0] + kept * tie_w;
    if (c < rank) { before += x; ties_before += t; }
    total += x;
    seen += t;
  }
  if (C > 1) cluster_sync_all();                              // a CTA's shared memory is read until here
  const u64 target = draw_target(a, row, total);
  for (int w = 0; w < warp; ++w) {
    const u64 t = sh.wcnt[w], kept = tie_in ? min(t, ties > ties_before ? ties - ties_before : 0ull) : 0ull;
    before += sh.wsum[w] + kept * tie_w;
    ties_before += t;
  }
  {
    const u64 kept = tie_in ? min(u64(tied), ties > ties_before ? ties - ties_before : 0ull) : 0ull;
    if (target < before || target >= before + sum + kept * tie_w) return;
  }
  for (int v0 = r.vlo; v0 < r.vhi; v0 += 32) {
    const int v = v0 + lane;
    float f[VEC];
    u64 w[VEC], own = 0;
    uint32_t eq = 0;
    if (v < r.vhi) unpack16<T>(r.load(v), f);
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const uint32_t key = v < r.vhi ? Key<T>::of(f[j]) : 0u;
      w[j] = v < r.vhi ? stays(f[j], key) : 0ull;
      eq += v < r.vhi && tie_in && key == limit;
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
      if (v < r.vhi && tie_in && Key<T>::of(f[j]) == limit) {
        if (nth < ties) w[j] = tie_w;
        ++nth;
      }
      own += w[j];
    }
    const u64 incl = warp_scan64(own, lane);
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
            write_token(a, row, v * VEC - r.shift + j, f[j], q, total);
          }
        }
      }
      return;
    }
    before += __shfl_sync(0xffffffffu, incl, 31);
    ties_before += __shfl_sync(0xffffffffu, eq_incl, 31);
  }
}

__constant__ double kSixteenths[16] = {1.0, 1.0442737824274138403, 1.0905077326652576592, 1.1387886347566916537, 1.1892071150027210667, 1.2418578120734840486,
                                       1.2968395546510096659, 1.3542555469368927283, 1.4142135623730950488, 1.4768261459394993114, 1.5422108254079408236,
                                       1.6104903319492543082, 1.6817928305074290861, 1.7562521603732994831, 1.8340080864093424635, 1.9152065613971472939};

// A cluster takes a row, and holds it in its shared memory if it fits.  Three ways lead to a token:
//   no limit in the order  the masses of all tokens are summed by warp; the warp that holds u times the total goes over its tokens again
//   a short list           a lower bound of what may stay is known: for top-k the k-th largest of the maxima of groups of tokens, for top-p the weight (1 - p) S / V
//                          (all tokens below it together weigh less than (1 - p) S), for min-p itself.  The tokens from there on go to the first CTA's list, where
//                          each is compared with each: its place in the order and the mass before it
//   the general way        where that list would be long
//
// What it takes: one row is a chain of exchanges (1 x 32000 bf16 with top-p: 12 us replayed; read in 0.01).  A short list needs one pass over keys: 256 x 50257 bf16, top-k
// and min-p, 25 us at 1.1 TB/s, in two waves of CTAs.  Masses of all tokens take eleven 64-bit operations and a table entry each: 512 x 128256 bf16 from the whole
// distribution 189 to 198 us, where nothing is full (with 16 warps an SM the pipe for them 21 % busy and 37 % of issue slots taken): too little is under way at once.  CTAs
// of 256 threads, four an SM, whose rows lie in L2 instead of shared memory take 197 as well (and 64 x 128256 fp32 160).
template <typename T, int THREADS>                            // up to so many
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) sample_kernel(SampleArgs a) {
  constexpr int VEC = kVec<T>;
  extern __shared__ uint4 slice[];                            // this CTA's vectors of the row
  __shared__ SampleShared sh;
  __shared__ uint32_t all_groups[kSampleGroups];
  pdl_launch_dependents();
  pdl_wait();
  const int C = a.ctas, rank = C > 1 ? int(cluster_ctarank()) : 0;
  const int row = blockIdx.x / C;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = blockDim.x >> 5;
  auto everywhere = [&] {
    if (C > 1) cluster_sync_all();
    else __syncthreads();
  };
  SampleRow<T> r;
  r.z = static_cast<const T*>(a.z) + row * a.ldz;
  r.V = a.V;
  r.shift = int(reinterpret_cast<uintptr_t>(r.z) & 15) / int(sizeof(T));
  const int vecs = (a.V + r.shift + VEC - 1) / VEC, vcta = (vecs + C - 1) / C, vwarp = (vcta + nw - 1) / nw;
  const int cend = min(vecs, (rank + 1) * vcta);
  r.vlo = min(cend, rank * vcta + warp * vwarp);
  r.vhi = min(cend, r.vlo + vwarp);
  r.held = nullptr;
  if (a.held) {                                               // (every thread reads the vectors that it fetches here)
    r.held = slice - rank * vcta;
    for (int v = r.vlo + lane; v < r.vhi; v += 32) {
      if (r.whole(v)) copy_async16(smem_u32(slice + (v - rank * vcta)), r.z + v * VEC - r.shift);
      else slice[v - rank * vcta] = r.fetch(v);
    }
  }
  if (threadIdx.x < 16) sh.table[threadIdx.x] = kSixteenths[threadIdx.x];
  if (threadIdx.x == 0) sh.count = 0;

  Filters by;
  by.k = a.top_k ? a.top_k[row] : a.top_k1;
  {
    const double tau = a.tau ? double(a.tau[row]) : a.tau1;
    if (!(tau > 0.0)) by.k = 1;
    if (by.k >= a.V && a.V > 1) by.k = 0;
    if (threadIdx.x == 32) {                                  // (divisions of 64 bits are long: one thread does them for all)
      const double low = a.min_p ? double(a.min_p[row]) : a.min_p1;
      sh.top_p = by.k == 1 ? 1.0 : a.top_p ? double(a.top_p[row]) : a.top_p1;
      sh.low = low;
      sh.tau = tau > 0.0 ? tau : 1.0;
      sh.k = fmin(1.4426950408889634074 / sh.tau, 1e300);
      sh.least = low > 0.0 ? u64(ceil(fmin(low, 1.0) * kMassOne)) : 0ull;
    }
  }

  // ---- maxima of groups of 32 / 2^per lanes, as many groups as top-k takes; the largest of them
  int per = 0;
  if (by.k > 1)
    while (per < 5 && (nw * C << per) < 2 * by.k && (nw * C << (per + 1)) <= kSampleGroups) ++per;
  const int own_groups = nw << per, groups = own_groups * C;
  asm volatile("cp.async.wait_all;" ::: "memory");
  {
    float m = -INFINITY;
#pragma unroll 4
    for (int v = r.vlo + lane; v < r.vhi; v += 32) m = fmaxf(m, max16<T>(r.raw(v)));
    uint32_t key = Key<T>::of(m);
    for (int o = 1; o < 32 >> per; o <<= 1) key = max(key, __shfl_xor_sync(0xffffffffu, key, o));
    if ((lane & ((32 >> per) - 1)) == 0) sh.groups[(warp << per) + lane / (32 >> per)] = key;
  }
  everywhere();
  uint32_t top = 0;
  for (int g = threadIdx.x; g < groups; g += blockDim.x) {
    const uint32_t key = C > 1 ? cluster_peer(sh.groups, g / own_groups)[g % own_groups] : sh.groups[g];
    all_groups[g] = key;
    top = max(top, key);
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if (lane == 0) sh.wcnt[warp] = top;
  __syncthreads();
  for (int w = 0; w < nw; ++w) top = max(top, sh.wcnt[w]);
  Weigh q;
  q.m = Key<T>::value(top);
  q.k = sh.k;
  q.md = double(q.m);
  by.p = sh.top_p;
  by.least = sh.least;
  if (q.m == -INFINITY) {
    if (rank == 0 && threadIdx.x == 0) {
      a.tokens[row] = -1;
      if (a.logprobs) a.logprobs[row] = -INFINITY;
    }
    if (C > 1) cluster_sync_all();                            // a CTA's shared memory is read until here
    return;
  }

  // (infinite factors, of tiny or huge temperatures and logits, leave the largest alone, or all that are finite, in their places)
  {
    const double cut = q.md - 45.5 / q.k;
    q.cut = cut == cut ? fminf(__double2float_ru(cut), q.m) : q.m;
    if (q.m == INFINITY) q.cut = q.m;
    q.cut = fmaxf(q.cut, -3.4028234663852886e38f);
  }
  const bool ordered = by.k > 0 || by.p < 1.0;                // a limit in the order
  float bound = -INFINITY, from = -INFINITY;                  // what lies below does not stay for the limits in the order, or for min-p either
  u64 mass = 0;
  bool listed = false;
  if (ordered || by.least > 0) {
    if (by.k == 1) {
      bound = q.m;
      listed = true;
    } else if (by.k > 0) {
      if (by.k <= groups) {
        // the k-th largest of the groups' maxima: the one with fewer than k above it, and k or more from it on
        for (int g = threadIdx.x; g < groups; g += blockDim.x) {
          const uint32_t key = all_groups[g];
          int above = 0, same = 0;
#pragma unroll 8
          for (int o = 0; o < groups; ++o) {
            above += all_groups[o] > key;
            same += all_groups[o] == key;
          }
          if (above < by.k && by.k <= above + same) sh.found[0] = key;
        }
        __syncthreads();
        bound = Key<T>::value(uint32_t(sh.found[0]));
        listed = true;
      }
    } else if (by.p < 1.0) {
      r.each(lane, [&](const float (&z)[VEC], int) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) mass += mass_of(z[j], q, sh.table);
      });
      mass = warp_add64(mass);
      if (lane == 0) sh.wsum[warp] = mass;
      __syncthreads();
      mass = 0;
      for (int w = 0; w < nw; ++w) mass += sh.wsum[w];
      if (C > 1) {
        if (threadIdx.x == 0) sh.part[0] = mass;
        cluster_sync_all();
        mass = 0;
        for (int c = 0; c < C; ++c) mass += *cluster_peer(sh.part, c);
      }
      // (NaN, of infinite logits and temperature, becomes the largest: nothing else weighs)
      if (threadIdx.x == 0) {
        const double least = (1.0 - fmax(by.p, 0.0)) * double(mass) / kMassOne / double(a.V) * (1.0 - 1e-9) - 1e-13;
        sh.from[0] = least > 0.0 ? fminf(__double2float_rd(q.md + sh.tau * log(least) * (1.0 + 1e-12) - 1e-30), q.m) : -INFINITY;
      }
      __syncthreads();
      bound = sh.from[0];
      listed = true;
    }
    // (with top-k and top-p the mass of the first k counts those that min-p leaves out)
    if (by.least > 0 && !(by.k > 0 && by.p < 1.0)) {
      if (threadIdx.x == 0)
        sh.from[1] = sh.low > 1e-12 ? __double2float_rd(q.md + sh.tau * log(fmin(sh.low, 1.0) - 1e-13) * (1.0 + 1e-12) - 1e-30) : -INFINITY;
      __syncthreads();
      from = sh.from[1];
      listed = listed || (!ordered && sh.low > 1e-12);
    }
    from = fminf(fmaxf(from, bound), q.m);
  }
  if (listed) {
    // ---- the short list
    u64* list = sh.sums;                                      // [256] key and token, then [256] weights and [256] masses
    u64* to = C > 1 ? cluster_peer(list, 0) : list;
    uint32_t* count = C > 1 ? cluster_peer(&sh.count, 0) : &sh.count;
    for (int v = r.vlo + lane; v < r.vhi; v += 32) {
      const uint4 u = r.raw(v);
      const float largest = max16<T>(u);
      if (!(largest >= from) || largest == -INFINITY) continue;
      float f[VEC];
      unpack16<T>(no_nan<T>(u), f);
      uint32_t n = 0;
#pragma unroll
      for (int j = 0; j < VEC; ++j) n += f[j] >= from && f[j] != -INFINITY;
      if (n) {
        uint32_t at = atomicAdd(count, n);
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          if (f[j] >= from && f[j] != -INFINITY) {
            if (at < kSampleFew) to[at] = u64(Key<T>::of(f[j])) << 32 | uint32_t(v * VEC - r.shift + j);
            ++at;
          }
      }
    }
    everywhere();
    const int n = int(*count);
    if (n <= kSampleFew) {
      if (C > 1) {
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        if (rank != 0) {
          asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
          return;
        }
      }
      if (threadIdx.x == 0) sh.found[1] = mass;
      short_list<T>(a, row, q, by, n, list, sh);
      if (C > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
      return;
    }
    everywhere();                                             // (the list's place is used again)
  }
  if (ordered) {
    sample_general<T>(a, r, q, by, bound, mass, row, rank, sh);
    return;
  }

  // ---- no limit in the order
  u64 sum = 0;
  if (by.least == 0)
    r.each(lane, [&](const float (&z)[VEC], int) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) sum += mass_of(z[j], q, sh.table);
    });
  else
    r.each(lane, [&](const float (&z)[VEC], int) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const u64 w = mass_of(z[j], q, sh.table);
        sum += w >= by.least ? w : 0ull;
      }
    });
  sum = warp_add64(sum);
  if (lane == 0) sh.wsum[warp] = sum;
  __syncthreads();
  u64 csum = 0, before = 0, total = 0;
  for (int w = 0; w < nw; ++w) {
    if (w < warp) before += sh.wsum[w];
    csum += sh.wsum[w];
  }
  if (C > 1) {
    if (threadIdx.x == 0) sh.part[0] = csum;
    cluster_sync_all();
    for (int c = 0; c < C; ++c) {
      const u64 x = *cluster_peer(sh.part, c);
      if (c < rank) before += x;
      total += x;
    }
    cluster_sync_all();                                       // a CTA's shared memory is read until here
  } else {
    total = csum;
  }
  const u64 target = draw_target(a, row, total);
  if (target < before || target >= before + sum) return;
  for (int v0 = r.vlo; v0 < r.vhi; v0 += 32) {
    const int v = v0 + lane;
    float f[VEC];
    u64 w[VEC], own = 0;
    if (v < r.vhi) unpack16<T>(r.load(v), f);
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      w[j] = v < r.vhi ? mass_of(f[j], q, sh.table) : 0ull;
      w[j] = w[j] >= by.least ? w[j] : 0ull;
      own += w[j];
    }
    const u64 incl = warp_scan64(own, lane);
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
            write_token(a, row, v * VEC - r.shift + j, f[j], q, total);
          }
        }
      }
      return;
    }
    before += __shfl_sync(0xffffffffu, incl, 31);
  }
}

template <typename T>
int sample(const SampleArgs& a, int threads, int smem, cudaStream_t st) {
  static OncePerDevice once;
  if (once.pending()) {
    LT_RETURN_IF_CUDA(cudaFuncSetAttribute(sample_kernel<T, kSampleThreads / 2>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSampleHold));
    LT_RETURN_IF_CUDA(cudaFuncSetAttribute(sample_kernel<T, kSampleThreads>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSampleHold));
    once.finish();
  }
  auto kernel = threads > kSampleThreads / 2 ? sample_kernel<T, kSampleThreads> : sample_kernel<T, kSampleThreads / 2>;
  if (a.ctas > 1) LT_RETURN_IF_CUDA(launch_chained_clusters(kernel, a.rows * a.ctas, threads, smem, a.ctas, st, a));
  else LT_RETURN_IF_CUDA(launch_chained(kernel, a.rows, threads, smem, st, a));
  return 0;
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
  const int vecs = V / (type == kElemF32 ? 4 : 8) + 2;
  auto bytes = [&](int n) { return (vecs / n + 1) * 16; };
  // as many CTAs as hold the row, and for few rows as many as two an SM with 8192 tokens or more each
  int ctas = 1, threads = kSampleThreads;
  while (ctas < kSampleCluster && bytes(ctas) > kSampleHold) ctas *= 2;
  while (ctas < kSampleCluster && (long long)rows * ctas * 2 <= 2 * sm_count() && V / ctas >= 8192) ctas *= 2;
  if ((long long)rows * ctas > 0x7fffffffll) return -int(kStatusBadArgument);
  const bool many = (long long)rows * ctas > 2 * sm_count();
  // (rows whose part takes so much memory that few CTAs share an SM: 512 threads; 64 x 128256 fp32 106 us, with 256 threads 121, 512 x 128256 bf16 197 and 205, in one run)
  while (threads > (many && bytes(ctas) > 48 * 1024 ? 512 : 128) && (many || vecs / ctas + 1 <= threads / 2)) threads /= 2;
  const bool held = (vecs / ctas + 1) * 16 <= kSampleHold;
  const int smem = held ? (vecs / ctas + 1) * 16 : 0;
  SampleArgs a{z, ldz, u, u64bit, tau, top_p, min_p, top_k, tau1, top_p1, min_p1, top_k1, rows, V, ctas, held, tokens, logprobs};
  if (type == kElemF32) return sample<float>(a, threads, smem, static_cast<cudaStream_t>(stream));
  if (type == kElemBf16) return sample<__nv_bfloat16>(a, threads, smem, static_cast<cudaStream_t>(stream));
  return sample<__half>(a, threads, smem, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
