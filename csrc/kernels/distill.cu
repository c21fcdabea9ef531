// Distillation from a teacher of whom the top logits are known: loss and gradient for rows of student logits z [N, V] against K teacher logits t [N, K]
// at classes i [N, K].
//
//   p = softmax(t / T) over the entries that are there,  q = softmax(z / T)
//   loss_n = T^2 sum_k p_k (log p_k - log q_{i_k}),      dloss_n / dz_j = T (q_j - sum of the p_k with i_k = j)
//
// An entry is there if its class lies in [0, V) and its logit is not -inf; a row without any has loss 0, gradient 0 and does not count in a mean.
#include "lt_cuda.h"

#include <algorithm>
#include <atomic>

#include "common/elem.cuh"
#include "common/host.h"
#include "common/ptx.cuh"

namespace lt {

constexpr int kDistillThreads = 512, kDistillWarps = kDistillThreads / 32, kDistillTop = 1024, kDistillCluster = 8;
constexpr int kLongThreads = 512, kLongWarps = kLongThreads / 32;
constexpr float kLog2e = 1.4426950408889634f;

struct DistillArgs {
  const void* z;
  long long ldz;
  float2* entries;               // [N, K]: log2 p of the teacher's entries and their class (its bits); -1: not there, -2: none of the row is
  int N, V, K;
  float temperature, c;          // c: log2(e) / temperature
  const unsigned char* flags;    // which rows have a teacher, for a mean; else null
  const float* up;               // upstream gradient: one (up_rows 0) or one for every row; null: 1
  int up_rows;
  int skip_one;                  // with one upstream gradient: return where it is 1 (the gradient is there)
  float2* stats;                 // [N] maximum of z, and the sum of 2^(z log2(e) / T - reference) with the maximum's reference
  int have_stats;
  float* loss;                   // [N] or null
  void* grad;                    // [N, V] (pitch ldg, rows where those of z lie within 16 bytes) or null
  long long ldg;
  int cluster_log, vpt;          // log2 of the CTAs of a cluster, vectors of a thread
  int* status;
};

__device__ __forceinline__ float load_as(int type, const void* p, long long i) {
  if (type == kElemF32) return static_cast<const float*>(p)[i];
  return type == kElemBf16 ? to_f32(static_cast<const __nv_bfloat16*>(p)[i]) : to_f32(static_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ bool entry_there(float t, long long i, int V) { return i >= 0 && i < V && t != -INFINITY; }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The teacher's side, a warp to a row: log2 of its probabilities, and whether it is there at all.
__global__ void __launch_bounds__(256) distill_teacher_kernel(const void* t, int t_type, const long long* idx, int N, int V, int K, float c, float2* entries,
                                                              unsigned char* flags, unsigned* finished) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  if (blockIdx.x == 0 && threadIdx.x == 0) *finished = 0u;
  for (long long r = blockIdx.x * 8ll + (threadIdx.x >> 5); r < N; r += gridDim.x * 8ll) {
    float m = -INFINITY, s = 0.f;
    bool any = false;
    for (int k = lane; k < K; k += 32) {
      const float x = load_as(t_type, t, r * K + k);
      if (!entry_there(x, idx[r * K + k], V)) continue;
      any = true;
      m = fmaxf(m, x);
    }
    any = __any_sync(0xffffffffu, any);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    for (int k = lane; k < K; k += 32) {
      const float x = load_as(t_type, t, r * K + k);
      if (entry_there(x, idx[r * K + k], V)) s += ex2((x - m) * c);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    const float ls = log2f(s);
    for (int k = lane; k < K; k += 32) {
      const float x = load_as(t_type, t, r * K + k);
      const long long i = idx[r * K + k];
      entries[r * K + k] = make_float2((x - m) * c - ls, __int_as_float(entry_there(x, i, V) ? int(i) : any ? -1 : -2));
    }
    if (flags && lane == 0) flags[r] = any;
  }
}

__device__ __forceinline__ int count_flags(const unsigned char* flags, int N, int* red) {
  int n = 0;                                                  // (flags are 0 or 1, and lie at 16 bytes)
  for (int i = threadIdx.x; i < N / 16; i += blockDim.x) {
    const uint4 u = reinterpret_cast<const uint4*>(flags)[i];
    n += __popc(u.x) + __popc(u.y) + __popc(u.z) + __popc(u.w);
  }
  for (int i = N / 16 * 16 + threadIdx.x; i < N; i += blockDim.x) n += flags[i];
  n = __reduce_add_sync(0xffffffffu, n);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = n;
  __syncthreads();
  n = 0;
  for (int w = 0; w < int(blockDim.x >> 5); ++w) n += red[w];
  __syncthreads();
  return n;
}

__device__ __forceinline__ float warp_max(float v) {
  float y;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(v));
  return y;
}
// Powers of two are taken of z c - ref, with ref = c times the largest logit m: z enters as fma(z, c, -ref), so that the reference is exact whatever its own
// rounding (which scales all of a row's powers alike, by up to 2^64 here).  From |ref| = 2^31 on (masks of the type's lowest value everywhere, say) what lies
// below m lies 128 or more below it: such a row is far out, and nothing but the equals of m weighs anything.
__device__ __forceinline__ bool far_out(float m, float ref) { return fabsf(ref) >= 0x1p31f && fabsf(m) != INFINITY; }
// The weight of a logit of a row that is far out (NaN stays).
__device__ __forceinline__ float far_weight(float f, float m) { return f == m ? 1.f : f != f ? f : 0.f; }
// A sum that belongs to the maximum `own` as one that belongs to m.
__device__ __forceinline__ float moved(float s, float own, float m, float c) {
  const float ref = __fmul_rn(m, c);                          // (not contracted: all round it alike)
  if (own == -INFINITY) return s;
  if (far_out(m, ref)) return own == m ? s : s * 0.f;
  return s * ex2(__fmul_rn(own, c) - ref);
}
template <typename T>
__device__ __noinline__ float far_sum(const uint4* mine, int vpt, float m) {
  float s = 0.f;
  for (int k = 0; k < vpt; ++k) {
    float f[kVec<T>];
    unpack16<T>(mine[k * 32], f);
#pragma unroll
    for (int j = 0; j < kVec<T>; ++j) s += far_weight(f[j], m);
  }
  return s;
}
template <typename T>
__device__ __noinline__ uint4 far_gradient(uint4 u, float m, float scale) {
  float f[kVec<T>];
  unpack16<T>(u, f);
#pragma unroll
  for (int j = 0; j < kVec<T>; ++j) f[j] = far_weight(f[j], m) * scale;
  return pack16<T>(f);
}
// A vector that begins with element i0 of a row of V, of which some lie outside.  (By elements from registers: warps are rows apart, and the last vector of
// neighbouring rows may be another warp's, so that they can share no memory for it.)
template <typename T>
__device__ __noinline__ void store_cut(T* row, int i0, int V, uint4 u) {
  float f[kVec<T>];
  unpack16<T>(u, f);
#pragma unroll
  for (int j = 0; j < kVec<T>; ++j)
    if (i0 + j >= 0 && i0 + j < V) row[i0 + j] = from_f32<T>(f[j]);
}
// (maximum, sum) over the warp.
__device__ __forceinline__ void warp_max_sum(float& m, float& s, float c) {
  const float own = m;
  m = warp_max(m);
  s = moved(s, own, m, c);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
}
// The first `bytes` of 16 (all that is read); the rest becomes zero.
__device__ __forceinline__ void copy_async16_part(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_async8(uint32_t dst, const void* src) { asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory"); }
// p[i] (bytes or 16-bit numbers) becomes v; returns what it was.
template <typename LINK>
__device__ __forceinline__ uint32_t exchange_small(LINK* p, int i, uint32_t v) {
  constexpr int BITS = 8 * sizeof(LINK), PER = 4 / sizeof(LINK);
  uint32_t* word = reinterpret_cast<uint32_t*>(p) + i / PER;
  const int sh = i % PER * BITS;
  const uint32_t mask = ((1u << BITS) - 1u) << sh;
  uint32_t old = *reinterpret_cast<volatile uint32_t*>(word);
  for (;;) {
    const uint32_t seen = atomicCAS(word, old, (old & ~mask) | v << sh);
    if (seen == old) return (old & mask) >> sh;
    old = seen;
  }
}
// The chains of a thread's eight vectors at once.
template <typename LINK> struct Heads;
template <> struct Heads<uint8_t> { typedef uint2 type; };
template <> struct Heads<uint16_t> { typedef uint4 type; };
__device__ __forceinline__ bool any(const uint2& h) { return (h.x | h.y) != 0u; }
__device__ __forceinline__ bool any(const uint4& h) { return (h.x | h.y | h.z | h.w) != 0u; }
__device__ __forceinline__ void clear(uint2& h) { h = make_uint2(0u, 0u); }
__device__ __forceinline__ void clear(uint4& h) { h = make_uint4(0u, 0u, 0u, 0u); }
// The number of the first chain from v on (8: there is none), and its first entry + 1.
__device__ __forceinline__ int first_head(const uint2& h, int v) {
  const unsigned long long x = v < 8 ? ((unsigned long long)h.y << 32 | h.x) >> (8 * v) : 0ull;
  return x ? v + (__ffsll(x) - 1) / 8 : 8;
}
__device__ __forceinline__ int head_of(const uint2& h, int v) { return ((v < 4 ? h.x : h.y) >> (8 * (v & 3))) & 0xff; }
__device__ __forceinline__ int head_of(const uint4& h, int v) { return ((v < 4 ? v < 2 ? h.x : h.y : v < 6 ? h.z : h.w) >> (16 * (v & 1))) & 0xffff; }
__device__ __forceinline__ int first_head(const uint4& h, int v) {
  while (v < 8 && head_of(h, v) == 0) ++v;
  return v;
}
// The teacher's probability of entry e's class (p by that entry alone) with those of the entries chained behind it that have the same.  Their sum is taken in
// whole numbers of 2^-62: it must not depend on the chain's order.
template <typename LINK>
__device__ __noinline__ float chained_p(const float2* entries, const LINK* link, int e, float p) {
  const int i = __float_as_int(entries[e - 1].y);
  unsigned long long sum = 0;
  int n = 0;
  for (int o = e; o; o = link[o - 1])
    if (__float_as_int(entries[o - 1].y) == i) {
      const float x = ex2(entries[o - 1].x);
      if (x != x) return x;
      sum += (unsigned long long)(x * 4611686018427387904.f);
      ++n;
    }
  return n > 1 ? float(double(sum) * (1.0 / 4611686018427387904.0)) : p;
}
// -inf in every element.
template <typename T> __device__ __forceinline__ uint32_t minus_inf() { return 0xff800000u; }
template <> __device__ __forceinline__ uint32_t minus_inf<__nv_bfloat16>() { return 0xff80ff80u; }
template <> __device__ __forceinline__ uint32_t minus_inf<__half>() { return 0xfc00fc00u; }
// An 8-byte store to the place `dst` of CTA `cta`'s shared memory that is counted on the barrier `bar` there.
__device__ __forceinline__ void send8(uint32_t dst, uint32_t bar, uint32_t cta, float2 v) {
  asm volatile(
      "{\n\t.reg .b32 rd, rb;\n\t.reg .b64 v;\n\t"
      "mapa.shared::cluster.u32 rd, %0, %2;\n\tmapa.shared::cluster.u32 rb, %1, %2;\n\t"
      "mov.b64 v, {%3, %4};\n\t"
      "st.async.shared::cluster.mbarrier::complete_tx::bytes.b64 [rd], v, [rb];\n\t}"
      ::"r"(dst), "r"(bar), "r"(cta), "f"(v.x), "f"(v.y)
      : "memory");
}

// Shared memory of a CTA of so many threads, 32 times a power of two.
template <typename LINK>
struct DistillSmem {
  static constexpr int kTop = sizeof(LINK) == 1 ? 255 : kDistillTop;      // entries that a LINK numbers
  static constexpr int kVectors = 3, kEntries = 5, kChains = 4, kPeers = 4;           // rows in turn
  // vpt: vectors of a thread.  Chains begin at 16 bytes (a thread takes its eight at once), which an odd K does not see to by itself.
  static __host__ __device__ int entries(int nt, int vpt) { return kVectors * vpt * nt * 16; }
  static __host__ __device__ int peers(int nt, int vpt, int K) { return entries(nt, vpt) + kEntries * K * 8; }
  static __host__ __device__ int heads(int nt, int vpt, int K) { return (peers(nt, vpt, K) + kPeers * kDistillCluster * (nt / 32) * 8 + 15) / 16 * 16; }
  static __host__ __device__ int links(int nt, int vpt, int K) { return heads(nt, vpt, K) + kChains * nt * 8 * int(sizeof(LINK)); }
  static __host__ __device__ int bytes(int nt, int vpt, int K) { return links(nt, vpt, K) + kChains * K * int(sizeof(LINK)); }
};

// A CTA, or for few rows a cluster of them, holds a row, every thread up to VPT vectors of 16 bytes: a row is read from global memory once.  The threads go over their vectors twice, first
// for the warps' maxima and sums, which go to all warps of the cluster, and then for the gradient; between the two they do the first pass over the
// next row, so that nobody waits for the exchange, and the rows after that are on their way into shared memory.  There is no barrier of all threads:
// a thread reads the vectors that it fetched itself, and one mbarrier a row counts the pairs that arrive and this CTA's warps.  A warp arrives there after its first pass
// over the row, that is, after its second pass over the row two before.  One in its first pass over row i has passed the barrier of row i - 2, so that the slowest may be in its
// second pass over row i - 3: pairs and chains lie in four places.  One that fetches row i + 2 has passed that of row i - 1, and the slowest may be in its second
// pass over row i - 2: entries lie in five.
// The teacher's classes are chained by the vector they lie in; the thread that writes the vector writes them again, from the 32-bit values.
// EVEN: all rows begin and end with a vector.  LINK: the type that numbers entries.
template <typename T, bool EVEN, typename LINK, int VPT>
__global__ void __launch_bounds__(kDistillThreads, 1) distill_kernel(DistillArgs a) {
  constexpr int VEC = kVec<T>;
  typedef DistillSmem<LINK> S;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ __align__(8) uint64_t bars[S::kPeers];
  __shared__ int isum[kDistillWarps];
  __shared__ int abort_flag;
  pdl_wait();
  if (a.skip_one && a.up && a.up[0] == 1.f) return;
  const float c = a.c;
  const uint64_t c2 = pack_f32x2(c, c);
  const int tid = threadIdx.x, lane = tid & 31, nt = blockDim.x, nw = nt >> 5;
  const int clog = a.cluster_log, rank = clog ? int(cluster_ctarank()) : 0;
  const int vpt = a.vpt, room = vpt * nt;
  const int first = (tid >> 5) * vpt * 32 + lane;             // this thread's vectors: first, first + 32, ... of the CTA's
  uint4* vectors = reinterpret_cast<uint4*>(smem) + first;    // [3][vpt nt]
  float2* entry_buf = reinterpret_cast<float2*>(smem + S::entries(nt, vpt));   // [5][K]
  float2* peers = reinterpret_cast<float2*>(smem + S::peers(nt, vpt, a.K));    // [4][CTAs][warps]: (maximum, sum)
  LINK* heads = reinterpret_cast<LINK*>(smem + S::heads(nt, vpt, a.K));        // [4][nt][8]: number of a vector's first entry + 1
  LINK* links = reinterpret_cast<LINK*>(smem + S::links(nt, vpt, a.K));        // [4][K]: that of an entry's next
  const int pairs = nw << clog;
  const uint32_t bar0 = smem_u32(bars);
  if (tid == 0) {
    abort_flag = 0;
    for (int i = 0; i < S::kPeers; ++i) mbar_init(bar0 + 8 * i, nw);
    fence_barrier_init();
  }
  for (int i = tid; i < S::kChains * nt * 2 * int(sizeof(LINK)); i += nt) reinterpret_cast<uint32_t*>(heads)[i] = 0u;
  const uint4 none = make_uint4(minus_inf<T>(), minus_inf<T>(), minus_inf<T>(), minus_inf<T>());
#pragma unroll
  for (int i = 0; i < S::kVectors; ++i)
#pragma unroll
    for (int k = 0; k < VPT; ++k)
      if (k < vpt) vectors[i * room + k * 32] = none;

  // Vector v of a row holds its elements [v VEC - shift, v VEC - shift + VEC): vectors are aligned, the first and the last may be cut.
  struct Row {
    int shift, lo, end, vecs;                                 // vectors [lo, end) are this CTA's
  };
  auto row_of = [&](const T* z) {
    Row r;
    r.shift = EVEN ? 0 : int(reinterpret_cast<uintptr_t>(z) & 15) / int(sizeof(T));
    r.vecs = (a.V + r.shift + VEC - 1) / VEC;
    const int part = (r.vecs + (1 << clog) - 1) >> clog;
    r.lo = min(r.vecs, rank * part);
    r.end = min(r.vecs, r.lo + part);
    return r;
  };
  // every thread of the warp has VPT vectors, none of which is cut
  auto full = [&](const Row& r) { return vpt == VPT && r.lo + first - lane + 32 * VPT <= r.end && (EVEN || (r.lo + first - lane > 0 && r.lo + first - lane + 32 * VPT < r.vecs)); };
  const int stride = gridDim.x >> clog;
  int row = blockIdx.x >> clog;
  const long long step = (long long)stride * a.ldz;
  const T* z = static_cast<const T*>(a.z) + (long long)row * a.ldz;      // the row of the first pass
  int to_fetch = row;
  const T* z_fetch = z;
  // (what lies in front of the row in its first 16 bytes belongs to the same tensor's memory; behind its last element nothing is read)
  auto fetch = [&](int buf, int entry_turn) {
    if (to_fetch < a.N) {
      const Row r = row_of(z_fetch);
      uint4* mine = vectors + buf * room;
      const T* from = z_fetch - r.shift + (r.lo + first) * VEC;
      const uint32_t to = smem_u32(mine);
      const int end = r.end - r.lo - first, last = r.vecs - 1 - r.lo - first;
      if (full(r)) {
#pragma unroll
        for (int k = 0; k < VPT; ++k) copy_async16(to + k * 512, from + k * 32 * VEC);
      } else
#pragma unroll
      for (int k = 0; k < VPT; ++k) {
        if (k >= vpt) break;
        if (k * 32 < end) {
          if (EVEN || k * 32 != last) copy_async16(to + k * 512, from + k * 32 * VEC);
          else copy_async16_part(to + k * 512, from + k * 32 * VEC, (a.V + r.shift - (r.vecs - 1) * VEC) * int(sizeof(T)));
        } else if (!EVEN) {                                   // (rows may differ by a vector)
          mine[k * 32] = none;
        }
      }
      if (a.grad)
        for (int k = tid; k < a.K; k += nt) copy_async8(smem_u32(entry_buf + entry_turn * a.K + k), a.entries + (long long)to_fetch * a.K + k);
    }
    to_fetch += stride;
    z_fetch += step;
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  __syncthreads();
  for (int i = 0; i < S::kVectors; ++i) fetch(i, i);
  float weight = a.temperature;
  if (a.flags) weight /= float(max(1, count_flags(a.flags, a.N, isum)));
  if (a.up && !a.up_rows) weight *= a.up[0];
  if (clog) cluster_sync_all();                               // every CTA is there to be written to
  int cur = 0, prev = 2;                                      // places of the first pass's vectors and of the second's
  int entry_cur = 0;                                          // place of the first pass's entries
  bool ok = true;
  for (int it = 0; row - stride < a.N; row += stride, z += step, ++it) {
    if (row < a.N) {
      // ---- first pass over this row
      asm volatile("cp.async.wait_group 1;" ::: "memory");
      const Row r = row_of(z);
      const int turn = it % S::kPeers;
      uint4* mine = vectors + cur * room;
      if (a.grad) {
        const float2* entries = entry_buf + entry_cur * a.K;
        const int elo = r.lo * VEC - r.shift, ehi = r.end * VEC - r.shift;
        for (int k = tid; k < a.K; k += nt) {
          const int i = __float_as_int(entries[k].y);
          if (i >= max(elo, 0) && i < ehi) {
            const int v = (i - elo) / VEC, w = v / (32 * vpt), owner = w * 32 + v % 32;
            links[turn * a.K + k] = LINK(exchange_small(heads, (turn * nt + owner) * 8 + (v / 32 - w * vpt), uint32_t(k + 1)));
          }
        }
      }
      if (!EVEN) {                                            // what a cut vector holds of others
        if (rank == 0 && tid == 0)
          for (int j = 0; j < r.shift; ++j) reinterpret_cast<T*>(mine)[j] = from_f32<T>(-INFINITY);
        const int last = r.vecs - 1 - r.lo - first;
        if (r.vecs == r.end && last >= 0 && last < 32 * vpt && last % 32 == 0)
          for (int j = a.V + r.shift - (r.vecs - 1) * VEC; j < VEC; ++j) reinterpret_cast<T*>(mine + last)[j] = from_f32<T>(-INFINITY);
      }
      if (!a.have_stats) {
        uint4 u[VPT];
        if (full(r)) {
#pragma unroll
          for (int k = 0; k < VPT; ++k) u[k] = mine[k * 32];
        } else {
#pragma unroll
          for (int k = 0; k < VPT; ++k) u[k] = k < vpt ? mine[k * 32] : none;
        }
        float m = -INFINITY;
#pragma unroll
        for (int k = 0; k < VPT; ++k) m = fmaxf(m, max16<T>(u[k]));
        const float ref = __fmul_rn(m, c), from = m == -INFINITY ? 0.f : -ref;
        uint64_t part[VEC / 2];
        const uint64_t from2 = pack_f32x2(from, from);
#pragma unroll
        for (int j = 0; j < VEC / 2; ++j) part[j] = 0ull;
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
          float f[VEC];
          unpack16<T>(u[k], f);
#pragma unroll
          for (int j = 0; j < VEC / 2; ++j) {
            float x, y;
            unpack_f32x2(fma_f32x2(pack_f32x2(f[2 * j], f[2 * j + 1]), c2, from2), x, y);
            part[j] = add_f32x2(part[j], pack_f32x2(ex2(x), ex2(y)));
          }
        }
#pragma unroll
        for (int j = VEC / 4; j > 0; j /= 2)
#pragma unroll
          for (int i = 0; i < j; ++i) part[i] = add_f32x2(part[i], part[i + j]);
        float s, s1;
        unpack_f32x2(part[0], s, s1);
        s += s1;
        if (far_out(m, ref)) s = far_sum<T>(mine, vpt, m);
        warp_max_sum(m, s, c);
        const int at = (turn * kDistillCluster + rank) * nw + (tid >> 5);
        if (clog) {
          if (lane >> clog == 0) send8(smem_u32(peers + at), bar0 + 8 * turn, lane, make_float2(m, s));
        } else if (lane == 0) {
          peers[at] = make_float2(m, s);
        }
      }
      __syncwarp();
      if (lane == 0) {
        if (tid == 0 && clog && !a.have_stats) mbar_expect_tx(bar0 + 8 * turn, pairs * 8);
        else mbar_arrive(bar0 + 8 * turn);
      }
    }
    if (it > 0) {
      // ---- second pass over the row before
      const int was = it - 1, old = row - stride, turn = was % S::kPeers;
      const Row r = row_of(z - step);
      uint4* mine = vectors + prev * room;
      const float2* entries = entry_buf + (entry_cur == 0 ? S::kEntries - 1 : entry_cur - 1) * a.K;
      // (A warp whose wait runs out sends and arrives no more, since what belongs to a later row would be counted into a phase of which nobody has seen the end.
      // It was there for this row and the next; the phase after them does not end, so that the waits of all other warps run out at that one at the latest.)
      ok = __all_sync(0xffffffffu, mbar_wait(bar0 + 8 * turn, (was / S::kPeers) & 1, &abort_flag, a.status, kStatusTimeoutLocalFlag));
      if (!ok) break;
      const bool empty = __float_as_int(entries[0].y) == -2;
      float m, s;
      if (a.have_stats) {
        const float2 q = a.stats[old];
        m = q.x;
        s = q.y;
      } else {
        m = -INFINITY;
        s = 0.f;
        const float2* all = peers + turn * kDistillCluster * nw;
        float2 q[kDistillCluster * kDistillWarps / 32];
#pragma unroll
        for (int i = 0; i < kDistillCluster * kDistillWarps / 32; ++i) {
          q[i] = make_float2(-INFINITY, 0.f);
          if (i * 32 < pairs) {
            if (i * 32 + lane < pairs) q[i] = all[i * 32 + lane];
            m = fmaxf(m, q[i].x);
          }
        }
        m = warp_max(m);
        const float ref = __fmul_rn(m, c);
        if (!far_out(m, ref)) {
#pragma unroll
          for (int i = 0; i < kDistillCluster * kDistillWarps / 32; ++i)
            if (i * 32 < pairs) s += q[i].y * ex2(__fmul_rn(q[i].x, c) - ref);
        } else {
#pragma unroll
          for (int i = 0; i < kDistillCluster * kDistillWarps / 32; ++i) s += q[i].x == m ? q[i].y : q[i].y * 0.f;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (a.stats && rank == 0 && tid == 0) a.stats[old] = make_float2(m, s);
      }
      if (a.grad) {
        T* g = static_cast<T*>(a.grad) + (long long)old * a.ldg;
        const float w = a.up_rows ? weight * a.up[old] : weight, scale = __fdividef(w, s), ref = __fmul_rn(m, c);
        const bool far = far_out(m, ref);
        T* to = g - r.shift + (r.lo + first) * VEC;
        const int end = r.end - r.lo - first;
        const bool cuts = !EVEN && (r.shift != 0 || r.vecs * VEC != a.V);
        const int head = cuts ? -r.lo - first : -1, last = cuts ? r.vecs - 1 - r.lo - first : -1;
        auto store = [&](int k, uint4 u) {
          if (!EVEN && (k * 32 == head || k * 32 == last)) store_cut<T>(g, (r.lo + first + k * 32) * VEC - r.shift, a.V, u);
          else *reinterpret_cast<uint4*>(to + k * 32 * VEC) = u;
        };
        auto gradient = [&](uint4 u) {
          float f[VEC];
          unpack16<T>(u, f);
#pragma unroll
          for (int j = 0; j < VEC / 2; ++j) {
            float x, y;
            unpack_f32x2(fma_f32x2(pack_f32x2(f[2 * j], f[2 * j + 1]), c2, pack_f32x2(-ref, -ref)), x, y);
            unpack_f32x2(mul_f32x2(pack_f32x2(ex2(x), ex2(y)), pack_f32x2(scale, scale)), f[2 * j], f[2 * j + 1]);
          }
          return pack16<T>(f);
        };
        if (!empty && !far && full(r)) {
          uint4 u[VPT];
#pragma unroll
          for (int k = 0; k < VPT; ++k) u[k] = mine[k * 32];
#pragma unroll
          for (int k = 0; k < VPT; ++k) *reinterpret_cast<uint4*>(to + k * 32 * VEC) = gradient(u[k]);
        } else if (!empty && !far) {
#pragma unroll 1
          for (int k = 0; k < vpt; ++k) {
            if (k * 32 < end) {
              store(k, gradient(mine[k * 32]));
            }
          }
        } else {
#pragma unroll 1
          for (int k = 0; k < vpt; ++k)
            if (k * 32 < end) store(k, empty ? make_uint4(0u, 0u, 0u, 0u) : far_gradient<T>(mine[k * 32], m, scale));
        }
        // chains of this thread's vectors
        typedef typename Heads<LINK>::type heads_t;
        heads_t& chains = *reinterpret_cast<heads_t*>(heads + (turn * nt + tid) * 8);
        if (any(chains)) {
          if (!empty) {
            const LINK* link = links + turn * a.K;
            const heads_t h = chains;
            for (int v = first_head(h, 0); v < 8; v = first_head(h, v + 1)) {
              uint32_t done = 0;
              for (int e = head_of(h, v); e; e = link[e - 1]) {
                const int i = __float_as_int(entries[e - 1].y), j = (i + r.shift) & (VEC - 1);
                if (done >> j & 1u) continue;
                done |= 1u << j;
                float p = ex2(entries[e - 1].x);
                if (link[e - 1]) p = chained_p(entries, link, e, p);
                const float x = to_f32(reinterpret_cast<const T*>(mine + v * 32)[j]);
                g[i] = from_f32<T>((__fdividef(far ? far_weight(x, m) : ex2(fmaf(x, c, -ref)), s) - p) * w);
              }
            }
          }
          clear(chains);
        }
      }
      fetch(prev, entry_cur < S::kEntries - 2 ? entry_cur + 2 : entry_cur + 2 - S::kEntries);
    }
    prev = cur;
    cur = cur == S::kVectors - 1 ? 0 : cur + 1;
    entry_cur = entry_cur == S::kEntries - 1 ? 0 : entry_cur + 1;
  }
  // (not earlier: CTAs of the next launch, which a CTA of this one leaves no registers, would gather on the few SMs that end first, and the losses then
  // take 24 us instead of 9, 2048 x 32000 with 128 entries a row)
  pdl_launch_dependents();
  asm volatile("cp.async.wait_all;" ::: "memory");
  if (clog) cluster_sync_all();                               // a CTA's shared memory is written until here
  if (!ok)                                                    // (and, where phases were not waited for, until what was sent has arrived)
    for (const long long t0 = clock64(); clock64() - t0 < 1 << 15;) {
    }
}

// Many long rows: a CTA goes over a row twice, the second time mostly out of L2 (of rows of 256 KB 296 are under way: 76 MB), and writes past it.  Nothing is
// exchanged between CTAs, and two an SM with up to 63 registers a thread fill all 148; the clusters above find places for 132.  It moves the 2.1 GB of 4096 x 128256 bf16
// logits and their gradient in 450 to 470 us with teacher and losses (cluster kernel: 506; the copy rate would allow 326), 1000 x 50257 fp32 in 97 us (127); losses
// alone read 1.05 GB in 195 us (348).  Nothing is full (DRAM 61 %, exponentials 55 %, issue 41 %): loads go to registers and stop at the end of each pass and row, and
// a CTA's two passes do not overlap with each other.  Three CTAs an SM of 40 registers spill (500 us), 1024 threads in one CTA wait for each other (509 us).
template <typename T>
__global__ void __launch_bounds__(kLongThreads) distill_long_kernel(DistillArgs a) {
  constexpr int VEC = kVec<T>, U = 4;
  __shared__ float2 red[kLongWarps];
  __shared__ int isum[kLongWarps];
  // the teacher's entries by the low bits of their class: a bucket's last entry + 1, and an entry's next
  __shared__ int classes[kDistillTop], bucket[kDistillTop], next[kDistillTop];
  pdl_launch_dependents();
  pdl_wait();
  if (a.skip_one && a.up && a.up[0] == 1.f) return;
  float weight = a.temperature;
  if (a.flags && a.grad) weight /= float(max(1, count_flags(a.flags, a.N, isum)));
  if (a.up && !a.up_rows) weight *= a.up[0];
  const float c = a.c;
  const uint64_t c2 = pack_f32x2(c, c);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  for (int row = blockIdx.x; row < a.N; row += gridDim.x) {
    const T* z = static_cast<const T*>(a.z) + (long long)row * a.ldz;
    T* g = a.grad ? static_cast<T*>(a.grad) + (long long)row * a.ldg : nullptr;
    const int head = min(a.V, int((16 - (reinterpret_cast<uintptr_t>(z) & 15)) & 15) / int(sizeof(T)));
    const int vecs = (a.V - head) / VEC, tail = head + vecs * VEC, rest = head + (a.V - tail);
    const uint4* from = reinterpret_cast<const uint4*>(z + head);
    auto edge = [&](int i) { return i < head ? i : tail + i - head; };
    float m = -INFINITY, s = 0.f;
    if (g)
      for (int i = tid; i < kDistillTop; i += kLongThreads) bucket[i] = 0;
    if (a.have_stats) {
      m = a.stats[row].x;
      s = a.stats[row].y;
      __syncthreads();
    } else {
      for (int i0 = tid; i0 < vecs; i0 += U * kLongThreads) {
        uint4 u[U];
#pragma unroll
        for (int k = 0; k < U; ++k)
          u[k] = i0 + k * kLongThreads < vecs ? __ldcg(from + i0 + k * kLongThreads) : make_uint4(minus_inf<T>(), minus_inf<T>(), minus_inf<T>(), minus_inf<T>());
        float vm = m;
#pragma unroll
        for (int k = 0; k < U; ++k) vm = fmaxf(vm, max16<T>(u[k]));
        s = moved(s, m, vm, c);
        m = vm;
        const float ref = __fmul_rn(m, c), below = m == -INFINITY ? 0.f : -ref;
        if (!far_out(m, ref)) {
          uint64_t sum[VEC / 2];
#pragma unroll
          for (int j = 0; j < VEC / 2; ++j) sum[j] = 0ull;
#pragma unroll
          for (int k = 0; k < U; ++k) {
            float f[VEC];
            unpack16<T>(u[k], f);
#pragma unroll
            for (int j = 0; j < VEC / 2; ++j) {
              float x, y;
              unpack_f32x2(fma_f32x2(pack_f32x2(f[2 * j], f[2 * j + 1]), c2, pack_f32x2(below, below)), x, y);
              sum[j] = add_f32x2(sum[j], pack_f32x2(ex2(x), ex2(y)));
            }
          }
#pragma unroll
          for (int j = 0; j < VEC / 2; ++j) {
            float x, y;
            unpack_f32x2(sum[j], x, y);
            s += x + y;
          }
        } else {
#pragma unroll
          for (int k = 0; k < U; ++k) {
            float f[VEC];
            unpack16<T>(u[k], f);
#pragma unroll
            for (int j = 0; j < VEC; ++j) s += far_weight(f[j], m);
          }
        }
      }
      for (int i = tid; i < rest; i += kLongThreads) {
        const float f = to_f32(z[edge(i)]), vm = fmaxf(m, f), ref = __fmul_rn(vm, c);
        s = moved(s, m, vm, c) + (far_out(vm, ref) ? far_weight(f, vm) : ex2(fmaf(f, c, vm == -INFINITY ? 0.f : -ref)));
        m = vm;
      }
      warp_max_sum(m, s, c);
      if (lane == 0) red[warp] = make_float2(m, s);
      __syncthreads();
      m = lane < kLongWarps ? red[lane].x : -INFINITY;
      s = lane < kLongWarps ? red[lane].y : 0.f;
      warp_max_sum(m, s, c);
      if (a.stats && tid == 0) a.stats[row] = make_float2(m, s);
    }
    if (g) {
      const float2* entries = a.entries + (long long)row * a.K;
      for (int k = tid; k < a.K; k += kLongThreads) {
        const int i = classes[k] = __float_as_int(entries[k].y);
        if (i >= 0) next[k] = atomicExch(&bucket[i & (kDistillTop - 1)], k + 1);
      }
      const bool empty = __float_as_int(entries[0].y) == -2;
      const float w = a.up_rows ? weight * a.up[row] : weight, scale = w / s, ref = __fmul_rn(m, c);
      const bool far = far_out(m, ref);
      uint4* to = reinterpret_cast<uint4*>(g + head);
      for (int i0 = tid; i0 < vecs; i0 += U * kLongThreads) {
        uint4 u[U];
#pragma unroll
        for (int k = 0; k < U; ++k)
          if (i0 + k * kLongThreads < vecs) u[k] = __ldcs(from + i0 + k * kLongThreads);
#pragma unroll
        for (int k = 0; k < U; ++k) {
          if (i0 + k * kLongThreads >= vecs) break;
          float f[VEC];
          unpack16<T>(u[k], f);
          if (!empty && !far) {
#pragma unroll
            for (int j = 0; j < VEC / 2; ++j) {
              float x, y;
              unpack_f32x2(fma_f32x2(pack_f32x2(f[2 * j], f[2 * j + 1]), c2, pack_f32x2(-ref, -ref)), x, y);
              unpack_f32x2(mul_f32x2(pack_f32x2(ex2(x), ex2(y)), pack_f32x2(scale, scale)), f[2 * j], f[2 * j + 1]);
            }
          } else {
#pragma unroll
            for (int j = 0; j < VEC; ++j) f[j] = empty ? 0.f : far_weight(f[j], m) * scale;
          }
          __stcs(to + i0 + k * kLongThreads, pack16<T>(f));
        }
      }
      for (int i = tid; i < rest; i += kLongThreads) {
        const float f = to_f32(z[edge(i)]);
        g[edge(i)] = from_f32<T>(empty ? 0.f : (far ? far_weight(f, m) : ex2(fmaf(f, c, -ref))) * scale);
      }
      __syncthreads();
      // the classes of the teacher's entries once more, one that comes again by its first entry
      for (int k = tid; k < a.K; k += kLongThreads) {
        const int i = classes[k];
        if (i < 0) continue;
        // (the sum in whole numbers of 2^-62: it must not depend on the chain's order)
        float p = ex2(entries[k].x);
        unsigned long long sum = 0;
        bool first = true, again = false;
        for (int o = bucket[i & (kDistillTop - 1)]; o; o = next[o - 1])
          if (classes[o - 1] == i) {
            first = first && o - 1 >= k;
            again = again || o - 1 != k;
            sum += (unsigned long long)(ex2(entries[o - 1].x) * 4611686018427387904.f);
          }
        if (again && p == p) p = float(double(sum) * (1.0 / 4611686018427387904.0));
        const float f = to_f32(z[i]);
        if (first) g[i] = from_f32<T>(((far ? far_weight(f, m) : ex2(fmaf(f, c, -ref))) / s - p) * w);
      }
    }
    __syncthreads();
  }
}

// The losses, a warp to a row, from the rows' maxima m and sums: log q = (z - m) / T - log sum e^((z' - m) / T), where what the reference's rounding took from the
// sum's exponents is put back (logits of a type's lowest value stay finite so); the last CTA to finish makes their mean over the rows that have a teacher, or their sum.
template <typename T>
__global__ void __launch_bounds__(256) distill_loss_kernel(DistillArgs a, float* out, unsigned* finished) {
  pdl_launch_dependents();
  pdl_wait();
  __shared__ double red[8];
  __shared__ int isum[8];
  __shared__ bool last;
  const int lane = threadIdx.x & 31;
  for (int row = blockIdx.x * 8 + (threadIdx.x >> 5); row < a.N; row += gridDim.x * 8) {
    const T* z = static_cast<const T*>(a.z) + (long long)row * a.ldz;
    const float2* entries = a.entries + (long long)row * a.K;
    const float2 q = a.stats[row];
    constexpr float kLn2 = 0.6931471805599453f;
    const float ref = __fmul_rn(q.x, a.c);
    const float base = kLn2 * (log2f(q.y) - (far_out(q.x, ref) ? 0.f : fmaf(q.x, a.c, -ref))), inv = 1.f / a.temperature;
    float part = 0.f;
    constexpr int U = 4;                                      // entries of a lane at once: their logits come from anywhere
    for (int k0 = lane; k0 < a.K; k0 += 32 * U) {
      float2 e[U];
      float x[U];
#pragma unroll
      for (int j = 0; j < U; ++j) e[j] = k0 + 32 * j < a.K ? entries[k0 + 32 * j] : make_float2(0.f, __int_as_float(-1));
#pragma unroll
      for (int j = 0; j < U; ++j) x[j] = __float_as_int(e[j].y) >= 0 ? to_f32(z[__float_as_int(e[j].y)]) : 0.f;
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const float p = ex2(e[j].x);
        if (__float_as_int(e[j].y) >= 0 && !(p == 0.f)) part += p * (fmaf(kLn2, e[j].x, base) - (x[j] - q.x) * inv);
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
    if (lane == 0) a.loss[row] = part * a.temperature * a.temperature;
  }
  if (!out) return;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(finished, 1u) == gridDim.x - 1;
  __syncthreads();
  if (!last) return;
  __threadfence();
  double v = 0.0;
#pragma unroll 4
  for (int i = threadIdx.x; i < a.N / 4; i += 256) {
    const float4 l = __ldcg(reinterpret_cast<const float4*>(a.loss) + i);
    v += (double(l.x) + double(l.y)) + (double(l.z) + double(l.w));
  }
  if (threadIdx.x < a.N % 4) v += __ldcg(a.loss + a.N / 4 * 4 + threadIdx.x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (lane == 0) red[threadIdx.x >> 5] = v;
  const int n = a.flags ? max(1, count_flags(a.flags, a.N, isum)) : 1;
  __syncthreads();
  if (threadIdx.x == 0) {
    v = 0.0;
    for (int w = 0; w < 8; ++w) v += red[w];
    *out = float(v / n);
  }
}

// How many clusters of 2^cluster_log CTAs of nt threads the GPU holds at once.
template <typename T, bool EVEN, typename LINK, int VPT>
cudaError_t cluster_places(int cluster_log, int nt, int vpt, int K, int* places) {
  auto kernel = distill_kernel<T, EVEN, LINK, VPT>;
  typedef DistillSmem<LINK> S;
  static std::atomic<int> known[64][4][5][VPT + 1][3];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  int size = 0;
  while (32 << size < nt) ++size;
  const int many = K > 128 ? 2 : K > 32 ? 1 : 0;              // (as if there were as many entries as that takes)
  std::atomic<int>& slot = known[dev & 63][cluster_log][size][vpt][many];
  *places = dev < 64 ? slot.load(std::memory_order_acquire) : 0;
  if (*places > 0) return cudaSuccess;
  if ((e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::bytes(kDistillThreads, VPT, S::kTop))) != cudaSuccess) return e;
  const int smem = S::bytes(nt, vpt, std::min(S::kTop, many == 2 ? kDistillTop : many == 1 ? 128 : 32));
  if (cluster_log == 0) {
    int per_sm = 0;
    if ((e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, nt, smem)) != cudaSuccess) return e;
    *places = per_sm * sm_count();
  } else {
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = 1 << cluster_log;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = 1 << cluster_log;
    cfg.blockDim = nt;
    cfg.dynamicSmemBytes = smem;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    if ((e = cudaOccupancyMaxActiveClusters(places, kernel, &cfg)) != cudaSuccess) return e;
  }
  if (*places < 1) return cudaErrorInvalidConfiguration;
  if (dev < 64) slot.store(*places, std::memory_order_release);
  return cudaSuccess;
}

template <typename T, bool EVEN, typename LINK, int VPT>
int distill_clusters(const DistillArgs& a, int nt, cudaStream_t st) {
  int places = 0;
  LT_RETURN_IF_CUDA((cluster_places<T, EVEN, LINK, VPT>(a.cluster_log, nt, a.vpt, a.K, &places)));
  const int ctas = 1 << a.cluster_log, clusters = std::min(a.N, places), smem = DistillSmem<LINK>::bytes(nt, a.vpt, a.K);
  auto kernel = distill_kernel<T, EVEN, LINK, VPT>;
  if (ctas > 1) LT_RETURN_IF_CUDA(launch_chained_clusters(kernel, clusters * ctas, nt, smem, ctas, st, a));
  else LT_RETURN_IF_CUDA(launch_chained(kernel, clusters, nt, smem, st, a));
  return 0;
}

template <typename T>
int distill(DistillArgs a, float* out, unsigned* finished, cudaStream_t st) {
  const bool even = a.V % kVec<T> == 0 && (a.N == 1 || a.ldz % kVec<T> == 0) && (reinterpret_cast<uintptr_t>(a.z) & 15) == 0;
  const int vecs = even ? a.V / kVec<T> : a.V / kVec<T> + 2;  // (a row may begin and end inside a vector)
  const bool few = a.K <= DistillSmem<uint8_t>::kTop;
  const int per = few ? 8 : 5;
  a.cluster_log = 0;
  while ((1 << a.cluster_log) < kDistillCluster && vecs > (per * kDistillThreads) << a.cluster_log) ++a.cluster_log;
  // rows that a CTA holds are read once (2048 x 32000 fp16, 128 entries: 82 us, twice 93; losses alone 47 and 43); few rows: clusters, so that all SMs have work
  // Many entries in a short row make chains whose threads the others wait for.  Loss and gradient / gradient alone, us, held and as a long row: 8192 x 1003 bf16 with 128
  // entries 73 / 50 and 107 / 67, 224: 117 / 89 and 115 / 69, 255: 148 / 109 and 122 / 70, 256 (whose chains are twice as wide, of fewer vectors a thread): 372 / 314 and
  // 117 / 70; 8192 x 4001 fp32 with 128: 126 / 81 and 147 / 95, 224: 147 / 98 and 156 / 101, 255: 165 / 106 and 161 / 100, 256: 270 / 179 and 157 / 100.
  const bool dense = a.grad && a.K > 224 && 8ll * a.K >= vecs;
  if (vecs <= (per * kDistillThreads) << a.cluster_log && ((a.cluster_log == 0 && !dense) || a.N < 2 * sm_count())) {
    // few rows: more CTAs for each
    while ((1 << a.cluster_log) < kDistillCluster && (long long)a.N << (a.cluster_log + 1) <= sm_count() && vecs >> a.cluster_log >= 512) ++a.cluster_log;
    const int own = (vecs + (1 << a.cluster_log) - 1) >> a.cluster_log;
    int nt = 32;
    while (nt < kDistillThreads && own > per * nt) nt *= 2;
    a.vpt = (own + nt - 1) / nt;
    int rc;
    if (few) rc = even ? distill_clusters<T, true, uint8_t, 8>(a, nt, st) : distill_clusters<T, false, uint8_t, 8>(a, nt, st);
    else rc = even ? distill_clusters<T, true, uint16_t, 5>(a, nt, st) : distill_clusters<T, false, uint16_t, 5>(a, nt, st);
    if (rc) return rc;
  } else {
    LT_RETURN_IF_CUDA(launch_chained(distill_long_kernel<T>, std::min(a.N, 4 * sm_count()), kLongThreads, 0, st, a));
  }
  if (a.loss) LT_RETURN_IF_CUDA(launch_chained(distill_loss_kernel<T>, std::min((a.N + 7) / 8, 8 * sm_count()), 256, 0, st, a, out, finished));
  return 0;
}

}  // namespace lt

extern "C" {

// Distillation of student logits z [N, V] (pitch ldz; fp32, bf16 or fp16: type 0, 1, 2) from teacher logits t [N, K] (type t_type) at classes idx [N, K].
//   entries [N, K, 2] floats and one more: written from t and idx; read if t is null
//   flags [N] bytes at 16 bytes: the loss is a mean over the rows that have a teacher (written or read likewise); null: no mean
//   loss [N] (with out: at 16 bytes) or null; out: their sum or mean, or null; stats [N, 2]: written, or read (have_stats: z is not searched for its maximum again)
//   grad [N, V] (pitch ldg; every row as far behind a multiple of 16 bytes as z's) or null: times up, which is null (1), one number, or (up_rows) one for every row; skip_one: nothing is done where up is one number and it is 1
int lt_distill(int type, const void* z, long long ldz, int t_type, const void* t, const long long* idx, float* entries, int N, int V, int K, float temperature,
               unsigned char* flags, const float* up, int up_rows, int skip_one, float* stats, int have_stats, float* loss, float* out, void* grad, long long ldg,
               void* stream) {
  using namespace lt;
  if (type < 0 || type > 2 || t_type < 0 || t_type > 2 || N < 0 || N >= 1 << 30 || V < 1 || V >= 1 << 30 || K < 1 || K > kDistillTop || !(temperature >= 0x1p-60f && temperature <= 0x1p60f) || (out && !loss) || (loss && (!stats || !t)) ||
      (reinterpret_cast<uintptr_t>(entries) & 7) != 0 || (reinterpret_cast<uintptr_t>(flags) & 15) != 0 || (out && (reinterpret_cast<uintptr_t>(loss) & 15) != 0))
    return -int(kStatusBadArgument);
  if (N == 0) return 0;
  const int bytes = type == kElemF32 ? 4 : 2;
  if (grad && (((reinterpret_cast<uintptr_t>(grad) ^ reinterpret_cast<uintptr_t>(z)) & 15) != 0 || (N > 1 && (ldg - ldz) * bytes % 16 != 0))) return -int(kStatusBadArgument);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  float2* pairs = reinterpret_cast<float2*>(entries);
  unsigned* finished = reinterpret_cast<unsigned*>(entries + 2ll * N * K);
  if (t) {
    const int grid = int(std::min<long long>((N + 7) / 8, 8ll * sm_count()));
    LT_RETURN_IF_CUDA(launch_chained(distill_teacher_kernel, grid, 256, 0, st, t, t_type, idx, N, V, K, kLog2e / temperature, pairs, flags, finished));
  }
  DistillArgs a{z, ldz, pairs, N, V, K, temperature, kLog2e / temperature, flags, up, up_rows, skip_one, reinterpret_cast<float2*>(stats), have_stats, loss, grad, ldg, 0, 0, device_status_word()};
  if (type == kElemF32) return distill<float>(a, out, finished, st);
  if (type == kElemBf16) return distill<__nv_bfloat16>(a, out, finished, st);
  return distill<__half>(a, out, finished, st);
}

// Where the parts of a CTA's shared memory lie for K entries, `threads` threads and `vectors` vectors a thread: entries, (maximum, sum) pairs, chains, links, the end.
int lt_distill_places(int K, int threads, int vectors, int* places) {
  using namespace lt;
  if (K < 1 || K > kDistillTop || threads < 32 || threads > kDistillThreads || vectors < 1 || vectors > 8) return -int(kStatusBadArgument);
  auto write = [&](auto s) {
    typedef decltype(s) S;
    const int at[5] = {S::entries(threads, vectors), S::peers(threads, vectors, K), S::heads(threads, vectors, K), S::links(threads, vectors, K), S::bytes(threads, vectors, K)};
    std::copy(at, at + 5, places);
  };
  if (K <= DistillSmem<uint8_t>::kTop) write(DistillSmem<uint8_t>());
  else write(DistillSmem<uint16_t>());
  return 0;
}

}  // extern "C"
