// Rows of an embedding table times a scale, and the gradient of the table by sorted tokens.
//
//   y[n] = scale * W[i_n]            dW[v] = scale * sum of dy[n] over the n with i_n = v, v != padding token
//
// A token outside the table gives a row of zeros and no gradient.  The sums are taken in fp32 in the order of the tokens and rounded
// once, so that results do not change from run to run (bf16 atomics, as in lt_embedding_bwd, round every addition and add in
// any order).
//
// The gradient takes three steps:
//   sort   one cluster of CTAs sorts (token, place) by token with a stable counting sort of 9 bits a pass: within a token the places stay in order
//   sum    a CTA takes `tile` neighbours of the sorted list and adds their rows; what begins and ends inside goes to the table, what goes
//          on in a neighbouring tile to a workspace
//   join   adds the pieces of a token that several tiles share, in order
#include "lt_cuda.h"

#include "common/elem.cuh"
#include "common/host.h"
#include "common/ptx.cuh"

namespace lt {

constexpr int kSortThreads = 1024, kSortWarps = kSortThreads / 32, kSortBits = 9, kSortBins = 1 << kSortBits;
constexpr int kMaxTile = 256;

// ---------------------------------------------------------------------------------------------- forward
template <typename T, typename IDX, int VEC>
__global__ void __launch_bounds__(256) token_embedding_fwd_kernel(const IDX* idx, const T* table, T* out, long long n, int D, int V, float scale) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int U = 4;
  const int vpr = D / VEC;
  const long long first = (long long)blockIdx.x * (256 * U);
  const long long row0 = first / vpr;
  const int rem = int(first - row0 * vpr);
  long long row[U], tok[U];
  int col[U];
#pragma unroll
  for (int k = 0; k < U; ++k) {
    const unsigned at = unsigned(rem + k * 256 + int(threadIdx.x));
    row[k] = row0 + at / unsigned(vpr);
    col[k] = int(at % unsigned(vpr)) * VEC;
    tok[k] = row[k] < n ? (long long)idx[row[k]] : -1;
  }
  if constexpr (VEC == 1) {
#pragma unroll
    for (int k = 0; k < U; ++k)
      if (row[k] < n) out[row[k] * D + col[k]] = from_f32<T>(tok[k] >= 0 && tok[k] < V ? to_f32(table[tok[k] * D + col[k]]) * scale : 0.f);
  } else {
    uint4 u[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      u[k] = make_uint4(0u, 0u, 0u, 0u);
      if (tok[k] >= 0 && tok[k] < V) u[k] = *reinterpret_cast<const uint4*>(table + tok[k] * D + col[k]);
    }
#pragma unroll
    for (int k = 0; k < U; ++k) {
      if (row[k] >= n) continue;
      float f[VEC];
      unpack16<T>(u[k], f);
#pragma unroll
      for (int j = 0; j < VEC; ++j) f[j] = tok[k] >= 0 && tok[k] < V ? f[j] * scale : 0.f;
      *reinterpret_cast<uint4*>(out + row[k] * D + col[k]) = pack16<T>(f);
    }
  }
}

// ---------------------------------------------------------------------------------------------- sort
// Sorted list of (token, place); tokens without a gradient get V and come last.  One cluster; every CTA holds the list's next n / CTAs entries, every warp
// the next part of those, so that entries of one digit stay in order.  Lists between two passes lie in global memory (in L2).
template <typename IDX>
__global__ void __launch_bounds__(kSortThreads) embed_sort_kernel(const IDX* idx, int n, int V, long long pad, uint2* buf0, uint2* buf1, int passes, int ctas) {
  extern __shared__ uint32_t sort_smem[];
  uint32_t(*cnt)[kSortBins] = reinterpret_cast<uint32_t(*)[kSortBins]>(sort_smem);        // [warp][digit]: how many, then places within the CTA
  uint32_t* total = sort_smem + kSortWarps * kSortBins;
  uint32_t* start = total + kSortBins;
  __shared__ uint32_t scan[32];
  pdl_launch_dependents();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = int(cluster_ctarank());
  const int part = (n + ctas - 1) / ctas;
  const int lo = min(n, rank * part), hi = min(n, lo + part);
  const int wpart = ((hi - lo + kSortWarps - 1) / kSortWarps + 31) / 32 * 32;
  const int wlo = min(hi, lo + warp * wpart), whi = min(hi, wlo + wpart);
  for (int p = 0; p < passes; ++p) {
    const uint2* src = (p & 1) ? buf0 : buf1;
    uint2* dst = (p & 1) ? buf1 : buf0;
    const int shift = p * kSortBits;
    auto entry = [&](int i) {
      if (p > 0) return __ldcg(src + i);
      const long long t = (long long)idx[i];
      return make_uint2(t >= 0 && t < V && t != pad ? uint32_t(t) : uint32_t(V), uint32_t(i));
    };
    for (int i = threadIdx.x; i < kSortWarps * kSortBins; i += kSortThreads) sort_smem[i] = 0u;
    __syncthreads();
    for (int i = wlo + lane; i < whi; i += 32) atomicAdd(&cnt[warp][(entry(i).x >> shift) & (kSortBins - 1)], 1u);
    __syncthreads();
    uint32_t mine = 0;
    if (threadIdx.x < kSortBins) {
#pragma unroll 8
      for (int w = 0; w < kSortWarps; ++w) {
        const uint32_t c = cnt[w][threadIdx.x];
        cnt[w][threadIdx.x] = mine;
        mine += c;
      }
      total[threadIdx.x] = mine;
    }
    if (ctas > 1) cluster_sync_all();
    else __syncthreads();
    uint32_t before = 0, all = 0;
    if (threadIdx.x < kSortBins) {
      for (int c = 0; c < ctas; ++c) {
        const uint32_t v = ctas > 1 ? *cluster_peer(total + threadIdx.x, c) : mine;
        before += c < rank ? v : 0u;
        all += v;
      }
    }
    uint32_t incl = all;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) scan[warp] = incl;
    __syncthreads();
    if (threadIdx.x < kSortBins) {
      uint32_t base = incl - all + before;
      for (int w = 0; w < warp; ++w) base += scan[w];
      start[threadIdx.x] = base;
    }
    __syncthreads();
    for (int i0 = wlo; i0 < whi; i0 += 32) {
      const int i = i0 + lane;
      const unsigned live = __ballot_sync(0xffffffffu, i < whi);
      if (i < whi) {
        const uint2 e = entry(i);
        const uint32_t d = (e.x >> shift) & (kSortBins - 1);
        const unsigned peers = __match_any_sync(live, d);
        const uint32_t at = start[d] + cnt[warp][d];
        dst[at + __popc(peers & ((1u << lane) - 1u))] = e;
        __syncwarp(live);
        if ((peers >> lane) == 1u) cnt[warp][d] += __popc(peers);         // the last of its digit
      }
      __syncwarp();
    }
    if (ctas > 1) cluster_sync_all();
    else __syncthreads();
  }
}

// ---------------------------------------------------------------------------------------------- sum
template <typename T, int VEC>
__device__ __forceinline__ void store_row(T* p, const float (&acc)[VEC], float scale) {
  if constexpr (VEC == 1) *p = from_f32<T>(acc[0] * scale);
  else {
    float f[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) f[j] = acc[j] * scale;
    *reinterpret_cast<uint4*>(p) = pack16<T>(f);
  }
}

// part[tile][0]: the sum of a segment that began before the tile; part[tile][1]: of one that begins in it and goes on behind it.
template <typename T, int VEC>
__global__ void __launch_bounds__(256) embed_sum_kernel(const uint2* order, const T* dout, long long ldd, T* grad, float* part, int n, int D, int V,
                                                        float scale, int tile, int chunks) {
  __shared__ uint2 s[kMaxTile + 2];                            // the tile with a neighbour on either side
  pdl_launch_dependents();
  pdl_wait();
  const int t = blockIdx.x / chunks, chunk = blockIdx.x % chunks;
  const int first = t * tile, cnt = min(tile, n - first);
  for (int i = threadIdx.x; i < cnt + 2; i += blockDim.x) {
    const int at = first - 1 + i;
    s[i] = at >= 0 && at < n ? order[at] : make_uint2(0xffffffffu, 0u);
  }
  __syncthreads();
  const int c = (chunk * int(blockDim.x) + int(threadIdx.x)) * VEC;
  if (c >= D) return;
  constexpr int U = 8;
  float acc[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
  for (int e0 = 0; e0 < cnt; e0 += U) {
    uint4 u[U];
    T one[U];
#pragma unroll
    for (int k = 0; k < U; ++k)
      if (e0 + k < cnt && s[e0 + k + 1].x < uint32_t(V)) {
        const T* p = dout + (long long)s[e0 + k + 1].y * ldd + c;
        if constexpr (VEC == 1) one[k] = *p;
        else u[k] = *reinterpret_cast<const uint4*>(p);
      }
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int e = e0 + k;
      if (e >= cnt || s[e + 1].x >= uint32_t(V)) break;
      const uint32_t key = s[e + 1].x;
      if constexpr (VEC == 1) acc[0] += to_f32(one[k]);
      else {
        float f[VEC];
        unpack16<T>(u[k], f);
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[j] += f[j];
      }
      const bool ends = s[e + 2].x != key, began = s[0].x != key;
      if (ends || e == cnt - 1) {
        if (ends && began) store_row<T, VEC>(grad + (long long)key * D + c, acc, scale);
        else {
          float* p = part + ((long long)t * 2 + (began ? 1 : 0)) * D + c;
#pragma unroll
          for (int j = 0; j < VEC; ++j) p[j] = acc[j];
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
      }
    }
  }
}

// The tile in which a token begins that goes on behind it adds the pieces.
template <typename T, int VEC>
__global__ void __launch_bounds__(256) embed_join_kernel(const uint2* order, const float* part, T* grad, int n, int D, int V, float scale, int tile, int chunks) {
  pdl_launch_dependents();
  pdl_wait();
  const int t = blockIdx.x / chunks, chunk = blockIdx.x % chunks;
  const int first = t * tile, last = min(n, first + tile) - 1;
  if (last + 1 >= n) return;
  const uint32_t key = order[last].x;
  if (key >= uint32_t(V) || order[last + 1].x != key || (first > 0 && order[first - 1].x == key)) return;
  int lo = last + 1, hi = n;                                   // first place behind the token
  while (lo < hi) {
    const int mid = lo + (hi - lo) / 2;
    if (order[mid].x == key) lo = mid + 1;
    else hi = mid;
  }
  const int end = (lo - 1) / tile;
  const int c = (chunk * int(blockDim.x) + int(threadIdx.x)) * VEC;
  if (c >= D) return;
  float acc[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) acc[j] = part[((long long)t * 2 + 1) * D + c + j];
#pragma unroll 4
  for (int k = t + 1; k <= end; ++k)
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[j] += part[(long long)k * 2 * D + c + j];
  store_row<T, VEC>(grad + (long long)key * D + c, acc, scale);
}

template <typename T, typename IDX>
int embedding_fwd(const void* idx, const void* table, void* out, long long n, int D, int V, float scale, cudaStream_t st) {
  const bool vec = D % kVec<T> == 0 && ((reinterpret_cast<uintptr_t>(table) | reinterpret_cast<uintptr_t>(out)) & 15) == 0;
  const long long items = n * (vec ? D / kVec<T> : D);
  const unsigned grid = unsigned((items + 1023) / 1024);
  auto kernel = vec ? token_embedding_fwd_kernel<T, IDX, kVec<T>> : token_embedding_fwd_kernel<T, IDX, 1>;
  LT_RETURN_IF_CUDA(launch_chained(kernel, grid, 256, 0, st, static_cast<const IDX*>(idx), static_cast<const T*>(table), static_cast<T*>(out), n, D, V, scale));
  return 0;
}

template <typename T, typename IDX>
int embedding_bwd(const void* idx, const void* dout, long long ldd, void* grad, int n, int D, int V, float scale, long long pad, void* order, float* part,
                  int tile, cudaStream_t st) {
  LT_RETURN_IF_CUDA(cudaMemsetAsync(grad, 0, size_t(V) * D * sizeof(T), st));
  if (n == 0) return 0;
  constexpr int smem = (kSortWarps * kSortBins + 2 * kSortBins) * 4;
  static OncePerDevice once;
  if (once.pending()) {
    LT_RETURN_IF_CUDA(cudaFuncSetAttribute(embed_sort_kernel<IDX>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    once.finish();
  }
  int passes = 1, ctas = 1;
  while (passes * kSortBits < 32 && (V >> (passes * kSortBits)) != 0) ++passes;
  while (ctas < 8 && n > ctas * 2048) ctas *= 2;
  uint2* buf0 = static_cast<uint2*>(order);
  uint2* buf1 = buf0 + n;
  const uint2* sorted = (passes & 1) ? buf0 : buf1;
  LT_RETURN_IF_CUDA(launch_chained_clusters(embed_sort_kernel<IDX>, ctas, kSortThreads, smem, ctas, st, static_cast<const IDX*>(idx), n, V, pad, buf0, buf1, passes, ctas));
  const bool vec = D % kVec<T> == 0 && ldd % kVec<T> == 0 && ((reinterpret_cast<uintptr_t>(dout) | reinterpret_cast<uintptr_t>(grad)) & 15) == 0;
  const int per = vec ? D / kVec<T> : D;
  const int threads = per >= 256 ? 256 : (per + 31) / 32 * 32;
  const int chunks = (per + threads - 1) / threads, tiles = (n + tile - 1) / tile;
  if ((long long)tiles * chunks > 0x7fffffffll) return -int(kStatusBadArgument);
  auto sum = vec ? embed_sum_kernel<T, kVec<T>> : embed_sum_kernel<T, 1>;
  auto join = vec ? embed_join_kernel<T, kVec<T>> : embed_join_kernel<T, 1>;
  LT_RETURN_IF_CUDA(launch_chained(sum, tiles * chunks, threads, 0, st, sorted, static_cast<const T*>(dout), ldd, static_cast<T*>(grad), part, n, D, V, scale, tile, chunks));
  if (tiles > 1)
    LT_RETURN_IF_CUDA(launch_chained(join, tiles * chunks, threads, 0, st, sorted, static_cast<const float*>(part), static_cast<T*>(grad), n, D, V, scale, tile, chunks));
  return 0;
}

}  // namespace lt

extern "C" {

// out[n, D] = scale * table[idx] of fp32 (type 0), bf16 (1) or fp16 (2) elements; zeros where a token is outside [0, V).  idx32: the tokens are 32-bit.
int lt_token_embedding_fwd(int type, const void* idx, int idx32, const void* table, void* out, long long n, int D, int V, float scale, void* stream) {
  using namespace lt;
  if (type < 0 || type > 2 || n < 0 || D < 0 || V < 1) return -int(kStatusBadArgument);
  if (n == 0 || D == 0) return 0;
  if (n > (0x7fffffffll * 1024) / D) return -int(kStatusBadArgument);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (type == kElemF32) return idx32 ? embedding_fwd<float, int>(idx, table, out, n, D, V, scale, st) : embedding_fwd<float, long long>(idx, table, out, n, D, V, scale, st);
  if (type == kElemBf16)
    return idx32 ? embedding_fwd<__nv_bfloat16, int>(idx, table, out, n, D, V, scale, st) : embedding_fwd<__nv_bfloat16, long long>(idx, table, out, n, D, V, scale, st);
  return idx32 ? embedding_fwd<__half, int>(idx, table, out, n, D, V, scale, st) : embedding_fwd<__half, long long>(idx, table, out, n, D, V, scale, st);
}

// grad[V, D] = scale * sums of dout's rows (pitch ldd) by token; tokens outside [0, V) and `pad` give nothing (pad < 0: there is none).  All of grad is written.
// order: 2 n entries of 8 bytes; part: 2 ceil(n / tile) rows of D floats; tile: up to 256 sorted rows a CTA.
int lt_token_embedding_bwd(int type, const void* idx, int idx32, const void* dout, long long ldd, void* grad, long long n, int D, int V, float scale, long long pad,
                           void* order, float* part, int tile, void* stream) {
  using namespace lt;
  if (type < 0 || type > 2 || n < 0 || n > 0x7fffffffll - 4096 || D < 0 || V < 1 || V == 0x7fffffff || tile < 1 || tile > kMaxTile) return -int(kStatusBadArgument);
  if (D == 0) return 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int m = int(n);
#define LT_EMBED_BWD(T)                                                                                                         \
  return idx32 ? embedding_bwd<T, int>(idx, dout, ldd, grad, m, D, V, scale, pad, order, part, tile, st)                        \
               : embedding_bwd<T, long long>(idx, dout, ldd, grad, m, D, V, scale, pad, order, part, tile, st)
  if (type == kElemF32) LT_EMBED_BWD(float);
  if (type == kElemBf16) LT_EMBED_BWD(__nv_bfloat16);
  LT_EMBED_BWD(__half);
#undef LT_EMBED_BWD
}

}  // extern "C"
