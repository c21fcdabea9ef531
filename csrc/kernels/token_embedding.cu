// Rows of an embedding table times a scale, and the gradient of the table by sorted tokens.
//
//   y[n] = scale * W[i_n]            dW[v] = scale * sum of dy[n] over the n with i_n = v, v != padding token
//
// A token outside the table gives a row of zeros and no gradient.  The sums are taken in fp32 in the order of the tokens and rounded
// once, so that results do not change from run to run (bf16 atomics, as in lt_embedding_bwd, round every addition and add in
// any order).
//
// The gradient of a small table by few tokens takes one launch (`embed_few_kernel`: 128 tokens, 8192 x 512 bf16 5.5 us, of which the write of 8 MB takes 1.3 at the copy rate), any
// other four:
//   sort   one cluster of CTAs sorts (token, place) by token with a stable counting sort of up to 9 bits a pass: within a token the places stay in order
//   clear  the table becomes zero, beside the sort
//   sum    a CTA takes `tile` neighbours of the sorted list and adds their rows.  A token with up to 64 places is summed where it begins; of one with more,
//          each tile leaves its piece in a workspace
//   join   adds the pieces, in order
//
// What bounds it: the bytes of the table's gradient where they are many (8192 tokens, 128256 x 4096 bf16: rows and gradient 191 us, 96 % of the copy rate; the clear
// alone writes 1.05 GB in 141 us and hides the sort), else launches one behind the other (2048 tokens, 32000 x 2048 bf16: 37 us replayed from a graph, of which the
// sort takes 17 and the join 11).  Rows that do not begin at 16 bytes are moved element by element: 40001 x 1027 fp32
// 145 us, where the bytes take 82.
#include "lt_cuda.h"

#include <algorithm>

#include "common/elem.cuh"
#include "common/host.h"
#include "common/ptx.cuh"

namespace lt {

constexpr int kSortThreads = 1024, kSortBits = 9, kSortBins = 1 << kSortBits;
constexpr int kMaxTile = 64, kShort = 64;                     // places of a token that are summed at once
constexpr int kFewThreads = 256, kFewLog = 3, kFewTokens = 2048;        // of one launch: threads, the smallest group (power of two), the most tokens
constexpr int kJoinTiles = 4;                                 // tiles that a CTA looks through

// ---------------------------------------------------------------------------------------------- forward
// 2^log threads to a row, each with every 2^log-th of its vectors, of four rows at once: a row alone keeps an SM waiting most of the time.
template <typename T, typename IDX>
__global__ void __launch_bounds__(256) token_embedding_fwd_kernel(const IDX* idx, const T* table, T* out, long long n, int D, int V, float scale, int log) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int VEC = kVec<T>, R = 4, U = 2;
  const int rows = 256 >> log;
  const long long first = (long long)blockIdx.x * (rows * R) + (threadIdx.x >> log);
  const T* from[R];
  bool in[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const long long row = first + r * rows, tok = row < n ? (long long)idx[row] : -1;
    in[r] = tok >= 0 && tok < V;
    from[r] = table + (in[r] ? tok : 0) * D;
  }
  const int step = VEC << log;
  for (int c0 = (threadIdx.x & ((1 << log) - 1)) * VEC; c0 < D; c0 += U * step) {
    uint4 u[R][U];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int k = 0; k < U; ++k)
        if (in[r] && c0 + k * step < D) u[r][k] = *reinterpret_cast<const uint4*>(from[r] + c0 + k * step);
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int k = 0; k < U; ++k) {
        if (first + r * rows >= n || c0 + k * step >= D) continue;
        float f[VEC];
        unpack16<T>(u[r][k], f);
#pragma unroll
        for (int j = 0; j < VEC; ++j) f[j] = in[r] ? f[j] * scale : 0.f;
        *reinterpret_cast<uint4*>(out + (first + r * rows) * D + c0 + k * step) = pack16<T>(f);
      }
  }
}

// Rows that do not begin at 16 bytes: four at once again, elements a CTA's width apart.  (Loads behind the end of a row take its last element.)
template <typename T, typename IDX>
__global__ void __launch_bounds__(256) token_embedding_odd_kernel(const IDX* idx, const T* table, T* out, long long n, int D, int V, float scale) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int R = 4, U = 4;
  const long long first = (long long)blockIdx.x * R;
  const T* from[R];
  bool in[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const long long tok = first + r < n ? (long long)idx[first + r] : -1;
    in[r] = tok >= 0 && tok < V;
    from[r] = table + (in[r] ? tok : 0) * D;
  }
  for (int c0 = threadIdx.x; c0 < D; c0 += U * 256) {
    T one[R][U];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int k = 0; k < U; ++k) one[r][k] = from[r][min(c0 + k * 256, D - 1)];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int k = 0; k < U; ++k)
        if (first + r < n && c0 + k * 256 < D) out[(first + r) * D + c0 + k * 256] = from_f32<T>(in[r] ? to_f32(one[r][k]) * scale : 0.f);
  }
}

// ---------------------------------------------------------------------------------------------- sort
// Sorted list of (token, place); tokens without a gradient get V and come last.  One cluster; every CTA holds the list's next n / CTAs entries, every warp
// the next part of those, so that entries of one digit stay in order.  Lists between two passes lie in global memory (in L2).
template <typename IDX>
__global__ void __launch_bounds__(kSortThreads) embed_sort_kernel(const IDX* idx, int n, int V, long long pad, uint2* buf0, uint2* buf1, int passes, int bits, int ctas) {
  extern __shared__ uint32_t sort_smem[];
  __shared__ uint32_t scan[32];
  pdl_wait();
  pdl_launch_dependents();                                    // (behind the wait: what starts now may write at once)
  const int bins = 1 << bits, nt = blockDim.x, nw = nt >> 5;
  uint32_t* cnt = sort_smem;                                  // [warp][digit]: how many, then places within the CTA
  uint32_t* total = sort_smem + nw * bins;
  uint32_t* start = total + bins;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = ctas > 1 ? int(cluster_ctarank()) : 0;
  const int part = (n + ctas - 1) / ctas;
  const int lo = min(n, rank * part), hi = min(n, lo + part);
  const int wpart = ((hi - lo + nw - 1) / nw + 31) / 32 * 32;
  const int wlo = min(hi, lo + warp * wpart), whi = min(hi, wlo + wpart);
  for (int p = 0; p < passes; ++p) {
    const uint2* src = (p & 1) ? buf0 : buf1;
    uint2* dst = (p & 1) ? buf1 : buf0;
    const int shift = p * bits;
    auto entry = [&](int i) {
      if (p > 0) return __ldcg(src + i);
      const long long t = (long long)idx[i];
      return make_uint2(t >= 0 && t < V && t != pad ? uint32_t(t) : uint32_t(V), uint32_t(i));
    };
    for (int i = threadIdx.x; i < nw * bins; i += nt) cnt[i] = 0u;
    __syncthreads();
#pragma unroll 4
    for (int i = wlo + lane; i < whi; i += 32) atomicAdd(&cnt[warp * bins + ((entry(i).x >> shift) & (bins - 1))], 1u);
    __syncthreads();
    for (int d = threadIdx.x; d < bins; d += nt) {
      uint32_t sum = 0;
#pragma unroll 8
      for (int w = 0; w < nw; ++w) {
        const uint32_t c = cnt[w * bins + d];
        cnt[w * bins + d] = sum;
        sum += c;
      }
      total[d] = sum;
    }
    if (ctas > 1) cluster_sync_all();
    else __syncthreads();
    uint32_t carry = 0;                                       // entries of the digits before
    for (int d0 = 0; d0 < bins; d0 += nt) {
      const int d = d0 + threadIdx.x;
      uint32_t before = 0, all = 0;
      if (d < bins)
        for (int c = 0; c < ctas; ++c) {
          const uint32_t v = ctas > 1 ? *cluster_peer(total + d, c) : total[d];
          before += c < rank ? v : 0u;
          all += v;
        }
      uint32_t incl = all;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
      if (lane == 31) scan[warp] = incl;
      __syncthreads();
      uint32_t base = carry + incl - all + before;
      for (int w = 0; w < nw; ++w) {
        if (w < warp) base += scan[w];
        carry += scan[w];
      }
      if (d < bins) start[d] = base;
      __syncthreads();
    }
    for (int i0 = wlo; i0 < whi; i0 += 32) {
      const int i = i0 + lane;
      const unsigned live = __ballot_sync(0xffffffffu, i < whi);
      if (i < whi) {
        const uint2 e = entry(i);
        const uint32_t d = (e.x >> shift) & (bins - 1);
        const unsigned peers = __match_any_sync(live, d);
        const uint32_t at = start[d] + cnt[warp * bins + d];
        dst[at + __popc(peers & ((1u << lane) - 1u))] = e;
        __syncwarp(live);
        if ((peers >> lane) == 1u) cnt[warp * bins + d] += __popc(peers);         // the last of its digit
      }
      __syncwarp();
    }
    if (ctas > 1) cluster_sync_all();
    else __syncthreads();
  }
}

// Zeros, 16 KB a CTA (1.05 GB: 65536 CTAs 7.4 TB/s, a few that stay 6.2).  Starts when the sort has begun (everything before that is complete) and runs beside it; the
// last CTA waits for the sort's end, so that the end of this launch is the end of both.
constexpr int kClear = 16384;
__global__ void __launch_bounds__(512) embed_clear_kernel(unsigned char* grad, long long bytes) {
  pdl_launch_dependents();
  const long long at = (long long)blockIdx.x * kClear;
  const int size = int(min((long long)kClear, bytes - at));
  if ((reinterpret_cast<uintptr_t>(grad) & 15) == 0) {
    for (int i = threadIdx.x; i < size / 16; i += 512) reinterpret_cast<uint4*>(grad + at)[i] = make_uint4(0u, 0u, 0u, 0u);
    if (threadIdx.x < size % 16) grad[at + size / 16 * 16 + threadIdx.x] = 0;
  } else {
    for (int i = threadIdx.x; i < size; i += 512) grad[at + i] = 0;
  }
  if (blockIdx.x == gridDim.x - 1) pdl_wait();
}

// ---------------------------------------------------------------------------------------------- sum
// Columns of a thread: a vector of 16 bytes, or (where rows do not begin at 16 bytes) four that lie a CTA's width apart.
template <typename T, bool WIDE> constexpr int kCols = WIDE ? kVec<T> : 4;

// apart: how far the columns of a thread lie apart.
template <typename T, bool WIDE>
__device__ __forceinline__ void store_row(T* row, int c, int D, const float (&acc)[kCols<T, WIDE>], float scale, int apart) {
  if constexpr (WIDE) {
    float f[kCols<T, WIDE>];
#pragma unroll
    for (int j = 0; j < kCols<T, WIDE>; ++j) f[j] = acc[j] * scale;
    *reinterpret_cast<uint4*>(row + c) = pack16<T>(f);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (c + j * apart < D) row[c + j * apart] = from_f32<T>(acc[j] * scale);
  }
}

// How many of the entries at s[from], s[from + dir], ... have the key, up to `most`; the whole warp.
__device__ __forceinline__ int run_length(const uint2* s, int from, int dir, uint32_t key, int most, int lane) {
  int n = 0;
  while (n < most) {
    const bool same = n + lane < most && s[from + dir * (n + lane)].x == key;
    const unsigned m = __ballot_sync(0xffffffffu, same);
    if (m != 0xffffffffu) return n + __ffs(~m) - 1;
    n += 32;
  }
  return n;
}

// part[tile][0]: the piece of a long segment that began before the tile; part[tile][1]: of one that begins in it.
template <typename T, bool WIDE>
__global__ void __launch_bounds__(256) embed_sum_kernel(const uint2* order, const T* dout, long long ldd, T* grad, float* part, int n, int D, int V,
                                                        float scale, int tile, int chunks) {
  __shared__ uint2 all[kShort + kMaxTile + kShort + 1];        // the tile with its neighbours on either side
  pdl_launch_dependents();
  pdl_wait();
  const int t = blockIdx.x / chunks, chunk = blockIdx.x % chunks, lane = threadIdx.x & 31;
  const int first = t * tile, cnt = min(tile, n - first);
  for (int i = threadIdx.x; i < kShort + cnt + kShort + 1; i += blockDim.x) {
    const long long at = (long long)first - kShort + i;
    all[i] = at >= 0 && at < n ? order[at] : make_uint2(0xffffffffu, 0u);
  }
  __syncthreads();
  const uint2* s = all + kShort;
  // the segment that comes from the tile before, and the one that goes on in the next
  const uint32_t head = s[0].x, tail = s[cnt - 1].x;
  if (head >= uint32_t(V)) return;
  int begin = 0, end = cnt;
  bool head_long = false, tail_long = false;
  const int back = run_length(s, -1, -1, head, kShort, lane);
  if (back > 0) {
    const int ahead = run_length(s, 0, 1, head, cnt + kShort, lane);
    head_long = back + ahead > kShort;
    if (!head_long) begin = min(ahead, cnt);                  // summed where it began
  }
  if (begin < cnt && tail < uint32_t(V)) {
    const int ahead = run_length(s, cnt, 1, tail, kShort, lane);
    if (ahead > 0) {
      const int own = run_length(s, cnt - 1, -1, tail, cnt, lane);
      tail_long = (own == cnt && back > 0 && head_long) || own + ahead > kShort;
      if (!tail_long) end = cnt + ahead;
    }
  }
  constexpr int NC = kCols<T, WIDE>;
  const int c = WIDE ? (chunk * int(blockDim.x) + int(threadIdx.x)) * NC : chunk * int(blockDim.x) * NC + int(threadIdx.x);
  if (c >= D) return;
  constexpr int U = 8;
  float acc[NC];
#pragma unroll
  for (int j = 0; j < NC; ++j) acc[j] = 0.f;
  for (int e0 = begin; e0 < end; e0 += U) {
    uint4 u[U];
    T one[U][4];
#pragma unroll
    for (int k = 0; k < U; ++k)
      if (e0 + k < end && s[e0 + k].x < uint32_t(V)) {
        const T* p = dout + (long long)s[e0 + k].y * ldd + c;
        if constexpr (WIDE) u[k] = *reinterpret_cast<const uint4*>(p);
        else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (c + j * int(blockDim.x) < D) one[k][j] = p[j * blockDim.x];
        }
      }
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int e = e0 + k;
      if (e >= end || s[e].x >= uint32_t(V)) break;
      const uint32_t key = s[e].x;
      if constexpr (!WIDE) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (c + j * int(blockDim.x) < D) acc[j] += to_f32(one[k][j]);
      } else {
        float f[NC];
        unpack16<T>(u[k], f);
#pragma unroll
        for (int j = 0; j < NC; ++j) acc[j] += f[j];
      }
      if (e == end - 1 || s[e + 1].x != key) {
        const bool from_before = head_long && key == head;
        if (!from_before && !(tail_long && key == tail)) store_row<T, WIDE>(grad + (long long)key * D, c, D, acc, scale, blockDim.x);
        else {
          float* p = part + ((long long)t * 2 + (from_before ? 0 : 1)) * D + c;
          if constexpr (WIDE) {
#pragma unroll
            for (int j = 0; j < NC; j += 4) *reinterpret_cast<float4*>(p + j) = make_float4(acc[j], acc[j + 1], acc[j + 2], acc[j + 3]);
          } else {
#pragma unroll
            for (int j = 0; j < NC; ++j)
              if (c + j * int(blockDim.x) < D) p[j * blockDim.x] = acc[j];
          }
        }
#pragma unroll
        for (int j = 0; j < NC; ++j) acc[j] = 0.f;
      }
    }
  }
}

// The pieces of long segments.  A CTA takes those that begin in its tiles; a long segment goes on behind the tile in which it begins, or fills it.
template <typename T, bool WIDE>
__global__ void __launch_bounds__(256) embed_join_kernel(const uint2* order, const float* part, T* grad, int n, int D, int V, float scale, int tile, int chunks) {
  __shared__ int until[kJoinTiles];                           // the last tile of the segment that begins in a tile, or -1
  pdl_launch_dependents();
  pdl_wait();
  const int group = blockIdx.x / chunks, chunk = blockIdx.x % chunks, lane = threadIdx.x & 31;
  const int tiles = (n + tile - 1) / tile;
  for (int w = threadIdx.x >> 5; w < kJoinTiles; w += blockDim.x >> 5) {
    const int t = group * kJoinTiles + w;
    int end = -1;
    if (t < tiles - 1) {
      const int first = t * tile, next = first + tile;
      const uint32_t key = order[next].x;
      // places of the token in this tile (of up to 64 places, two to a lane), if it is not in the one before too
      const bool a = lane < tile && order[first + lane].x == key, b = lane + 32 < tile && order[first + lane + 32].x == key;
      const int own = __popc(__ballot_sync(0xffffffffu, a)) + __popc(__ballot_sync(0xffffffffu, b));
      const bool begins = key < uint32_t(V) && own > 0 && (first == 0 || order[first - 1].x != key);
      if (begins && (long long)next - own + kShort < n && order[next - own + kShort].x == key) {
        for (int o = t + 1; end < 0; o += 32) {               // the first tile that does not end with it
          const long long last = min((long long)n, (long long)(o + lane + 1) * tile) - 1;
          const bool goes_on = o + lane < tiles - 1 && order[last].x == key;
          const unsigned m = __ballot_sync(0xffffffffu, !goes_on);
          if (m) {
            end = o + __ffs(m) - 1;
            if (order[(long long)end * tile].x != key) --end;
          }
        }
      }
    }
    if (lane == 0) until[w] = end;
  }
  __syncthreads();
  constexpr int NC = kCols<T, WIDE>;
  const int c = WIDE ? (chunk * int(blockDim.x) + int(threadIdx.x)) * NC : chunk * int(blockDim.x) * NC + int(threadIdx.x);
  if (c >= D) return;
  for (int i = 0; i < kJoinTiles; ++i) {
    const int t = group * kJoinTiles + i;
    if (until[i] < 0) continue;
    float acc[NC];
#pragma unroll
    for (int j = 0; j < NC; ++j) acc[j] = 0.f;
#pragma unroll 4
    for (int k = t; k <= until[i]; ++k) {
      const float* p = part + ((long long)k * 2 + (k == t ? 1 : 0)) * D + c;
      if constexpr (WIDE) {
#pragma unroll
        for (int j = 0; j < NC; j += 4) {
          const float4 v = *reinterpret_cast<const float4*>(p + j);
          acc[j] += v.x; acc[j + 1] += v.y; acc[j + 2] += v.z; acc[j + 3] += v.w;
        }
      } else {
#pragma unroll
        for (int j = 0; j < NC; ++j)
          if (c + j * int(blockDim.x) < D) acc[j] += p[j * blockDim.x];
      }
    }
    store_row<T, WIDE>(grad + (long long)order[min(n, t * tile + tile) - 1].x * D, c, D, acc, scale, blockDim.x);
  }
}

// ---------------------------------------------------------------------------------------------- few tokens
// One launch: a CTA takes 4 rows of the table a thread group, 16 KB of it, sets them to zero, looks through all tokens for those of its rows and adds theirs up.  Every CTA
// reads all tokens (out of L2), which a program with few of them can afford for the three launches less.  A token's rows are added in fp32 in the order of their
// places, by the group that has its row; those of a token with more than 64 places in as many pieces as there are groups, which are added in order.
template <typename T, bool WIDE, typename IDX>
__global__ void __launch_bounds__(kFewThreads) embed_few_kernel(const IDX* idx, const T* dout, long long ldd, T* grad, int n, int D, int V, float scale, long long pad, int log,
                                                                int chunks) {
  constexpr int NC = kCols<T, WIDE>, W = kFewThreads / 32, MAXR = kFewThreads / (1 << kFewLog) * 4, U = 8;
  extern __shared__ uint16_t few_list[];                      // places of this CTA's tokens by row
  __shared__ uint32_t cnt[W * MAXR], start[MAXR + 1], carry[W];
  __shared__ float pieces[kFewThreads * NC];
  pdl_launch_dependents();
  pdl_wait();
  const int G = 1 << log, groups = kFewThreads >> log, R = groups * 4;
  const int chunk = int(blockIdx.x) % chunks, v0 = int(blockIdx.x) / chunks * R, rows = min(R, V - v0);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, own = tid & (G - 1), g = tid >> log;
  const int c = WIDE ? (chunk * G + own) * NC : chunk * G * NC + own;
  float acc[NC];
#pragma unroll
  for (int j = 0; j < NC; ++j) acc[j] = 0.f;
  if (c < D)
    for (int r = g; r < rows; r += groups) store_row<T, WIDE>(grad + (long long)(v0 + r) * D, c, D, acc, 0.f, G);
  for (int i = tid; i < W * R; i += kFewThreads) cnt[i] = 0u;
  __syncthreads();
  const int wpart = ((n + W - 1) / W + 31) / 32 * 32, wlo = min(n, warp * wpart), whi = min(n, wlo + wpart);
  auto row_of = [&](int i) {                                  // -1: not this CTA's
    const long long t = i < whi ? (long long)idx[i] : -1;
    return t >= v0 && t < v0 + rows && t != pad ? int(t - v0) : -1;
  };
  bool any = false;
#pragma unroll 8
  for (int i = wlo + lane; i < whi; i += 32) {
    const int r = row_of(i);
    if (r >= 0) {
      atomicAdd(&cnt[warp * R + r], 1u);
      any = true;
    }
  }
  any = __syncthreads_or(any);
  if (!any) return;
  // where the tokens of a row begin in the list, and those of a warp among them
  {
    uint32_t sum = 0;
    if (tid < R)
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const uint32_t k = cnt[w * R + tid];
        cnt[w * R + tid] = sum;
        sum += k;
      }
    uint32_t incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t k = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += k;
    }
    if (lane == 31) carry[warp] = incl;
    __syncthreads();
    for (int w = 0; w < warp; ++w) incl += carry[w];
    if (tid < R) {
      start[tid + 1] = incl;
      if (tid == 0) start[0] = 0u;
#pragma unroll
      for (int w = 0; w < W; ++w) cnt[w * R + tid] += incl - sum;
    }
    __syncthreads();
  }
  for (int i0 = wlo; i0 < whi; i0 += 32) {
    const int r = row_of(i0 + lane);
    const unsigned with = __ballot_sync(0xffffffffu, r >= 0);
    if (r >= 0) {
      const unsigned peers = __match_any_sync(with, r);
      few_list[cnt[warp * R + r] + __popc(peers & ((1u << lane) - 1u))] = uint16_t(i0 + lane);
      __syncwarp(with);
      if ((peers >> lane) == 1u) cnt[warp * R + r] += __popc(peers);         // the last of its row
    }
    __syncwarp();
  }
  __syncthreads();
  // acc = sum of the rows of the places [lo, hi) of the list
  auto add = [&](uint32_t lo, uint32_t hi) {
#pragma unroll
    for (int j = 0; j < NC; ++j) acc[j] = 0.f;
    for (uint32_t e0 = lo; e0 < hi; e0 += U) {
      uint4 u[U];
      T one[U][4];
#pragma unroll
      for (int k = 0; k < U; ++k)
        if (e0 + k < hi) {
          const T* p = dout + (long long)few_list[e0 + k] * ldd + c;
          if constexpr (WIDE) u[k] = *reinterpret_cast<const uint4*>(p);
          else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (c + j * G < D) one[k][j] = p[j * G];
          }
        }
#pragma unroll
      for (int k = 0; k < U; ++k) {
        if (e0 + k >= hi) break;
        if constexpr (WIDE) {
          float f[NC];
          unpack16<T>(u[k], f);
#pragma unroll
          for (int j = 0; j < NC; ++j) acc[j] += f[j];
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (c + j * G < D) acc[j] += to_f32(one[k][j]);
        }
      }
    }
  };
  bool many = false;
  for (int r = g; r < rows; r += groups) {
    const uint32_t lo = start[r], hi = start[r + 1];
    many = many || hi - lo > uint32_t(kShort);
    if (hi == lo || hi - lo > uint32_t(kShort) || c >= D) continue;
    add(lo, hi);
    store_row<T, WIDE>(grad + (long long)(v0 + r) * D, c, D, acc, scale, G);
  }
  if (!__syncthreads_or(many)) return;
  for (int r = 0; r < rows; ++r) {
    const uint32_t lo = start[r], m = start[r + 1] - lo;
    if (m <= uint32_t(kShort)) continue;
    const uint32_t part = (m + groups - 1) / groups, from = min(m, g * part);
    if (c < D) {
      add(lo + from, lo + min(m, from + part));
#pragma unroll
      for (int j = 0; j < NC; ++j) pieces[tid * NC + j] = acc[j];
    }
    __syncthreads();
    if (g == 0 && c < D) {
      for (int o = 1; o < groups; ++o)
#pragma unroll
        for (int j = 0; j < NC; ++j) acc[j] += pieces[((o << log) + own) * NC + j];
      store_row<T, WIDE>(grad + (long long)(v0 + r) * D, c, D, acc, scale, G);
    }
    __syncthreads();
  }
}

template <typename T, typename IDX>
int embedding_fwd(const void* idx, const void* table, void* out, long long n, int D, int V, float scale, cudaStream_t st) {
  const bool vec = D % kVec<T> == 0 && ((reinterpret_cast<uintptr_t>(table) | reinterpret_cast<uintptr_t>(out)) & 15) == 0;
  auto i = static_cast<const IDX*>(idx);
  auto w = static_cast<const T*>(table);
  auto y = static_cast<T*>(out);
  if (vec) {
    int log = 0;
    while (log < 8 && (1 << log) < D / kVec<T>) ++log;
    const int rows = 1024 >> log;                             // of a CTA
    LT_RETURN_IF_CUDA(launch_chained(token_embedding_fwd_kernel<T, IDX>, unsigned((n + rows - 1) / rows), 256, 0, st, i, w, y, n, D, V, scale, log));
  } else {
    LT_RETURN_IF_CUDA(launch_chained(token_embedding_odd_kernel<T, IDX>, unsigned((n + 3) / 4), 256, 0, st, i, w, y, n, D, V, scale));
  }
  return 0;
}

template <typename T, typename IDX>
int embedding_bwd(const void* idx, const void* dout, long long ldd, void* grad, int n, int D, int V, float scale, long long pad, void* order, float* part,
                  int tile, cudaStream_t st) {
  const size_t bytes = size_t(V) * D * sizeof(T);
  if (n == 0) {
    LT_RETURN_IF_CUDA(cudaMemsetAsync(grad, 0, bytes, st));
    return 0;
  }
  const bool vec = D % kVec<T> == 0 && ldd % kVec<T> == 0 && ((reinterpret_cast<uintptr_t>(dout) | reinterpret_cast<uintptr_t>(grad) | reinterpret_cast<uintptr_t>(part)) & 15) == 0;
  if (order == nullptr) {
    const int per = vec ? D / kVec<T> : (D + 3) / 4;
    int log = kFewLog;
    while (log < 6 && (1 << log) < per) ++log;
    const long long rows = (kFewThreads >> log) * 4, chunks = (per + (1 << log) - 1) >> log, ctas = (V + rows - 1) / rows * chunks;
    if (n > kFewTokens || ctas > 0x7fffffffll) return -int(kStatusBadArgument);
    auto few = vec ? embed_few_kernel<T, true, IDX> : embed_few_kernel<T, false, IDX>;
    LT_RETURN_IF_CUDA(launch_chained(few, unsigned(ctas), kFewThreads, n * 2, st, static_cast<const IDX*>(idx), static_cast<const T*>(dout), ldd, static_cast<T*>(grad), n, D, V, scale, pad, log, int(chunks)));
    return 0;
  }
  static OncePerDevice once;
  if (once.pending()) {
    LT_RETURN_IF_CUDA(cudaFuncSetAttribute(embed_sort_kernel<IDX>, cudaFuncAttributeMaxDynamicSharedMemorySize, (kSortThreads / 32 + 2) * kSortBins * 4));
    once.finish();
  }
  int width = 1, passes = 1, ctas = 1, nt = kSortThreads;
  while (width < 31 && (V >> width) != 0) ++width;
  while (passes * kSortBits < width) ++passes;
  const int bits = (width + passes - 1) / passes;
  while (ctas < 8 && n > ctas * 1024) ctas *= 2;
  while (nt > 128 && n <= ctas * nt / 2) nt /= 2;
  uint2* buf0 = static_cast<uint2*>(order);
  uint2* buf1 = buf0 + n;
  const uint2* sorted = (passes & 1) ? buf0 : buf1;
  const int smem = (nt / 32 + 2) * (1 << bits) * 4;
  LT_RETURN_IF_CUDA(launch_chained_clusters(embed_sort_kernel<IDX>, ctas, nt, smem, ctas, st, static_cast<const IDX*>(idx), n, V, pad, buf0, buf1, passes, bits, ctas));
  if (bytes > size_t(kClear) * 0x7fffffff) return -int(kStatusBadArgument);
  LT_RETURN_IF_CUDA(launch_chained(embed_clear_kernel, unsigned((bytes + kClear - 1) / kClear), 512, 0, st, static_cast<unsigned char*>(grad), (long long)bytes));
  const int per = vec ? D / kVec<T> : (D + 3) / 4;
  const int threads = per >= 256 ? 256 : (per + 31) / 32 * 32;
  const int chunks = (per + threads - 1) / threads, tiles = (n + tile - 1) / tile;
  if ((long long)tiles * chunks > 0x7fffffffll) return -int(kStatusBadArgument);
  auto sum = vec ? embed_sum_kernel<T, true> : embed_sum_kernel<T, false>;
  auto join = vec ? embed_join_kernel<T, true> : embed_join_kernel<T, false>;
  LT_RETURN_IF_CUDA(launch_chained(sum, tiles * chunks, threads, 0, st, sorted, static_cast<const T*>(dout), ldd, static_cast<T*>(grad), part, n, D, V, scale, tile, chunks));
  if (n > kShort)
    LT_RETURN_IF_CUDA(launch_chained(join, (tiles + kJoinTiles - 1) / kJoinTiles * chunks, threads, 0, st, sorted, static_cast<const float*>(part), static_cast<T*>(grad), n, D, V, scale, tile, chunks));
  return 0;
}

}  // namespace lt

extern "C" {

// out[n, D] = scale * table[idx] of fp32 (type 0), bf16 (1) or fp16 (2) elements; zeros where a token is outside [0, V).  idx32: the tokens are 32-bit.
int lt_token_embedding_fwd(int type, const void* idx, int idx32, const void* table, void* out, long long n, int D, int V, float scale, void* stream) {
  using namespace lt;
  if (type < 0 || type > 2 || n < 0 || D < 0 || D > 1 << 30 || V < 1) return -int(kStatusBadArgument);
  if (n == 0 || D == 0) return 0;
  if (n > 0x7fffffffll) return -int(kStatusBadArgument);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (type == kElemF32) return idx32 ? embedding_fwd<float, int>(idx, table, out, n, D, V, scale, st) : embedding_fwd<float, long long>(idx, table, out, n, D, V, scale, st);
  if (type == kElemBf16)
    return idx32 ? embedding_fwd<__nv_bfloat16, int>(idx, table, out, n, D, V, scale, st) : embedding_fwd<__nv_bfloat16, long long>(idx, table, out, n, D, V, scale, st);
  return idx32 ? embedding_fwd<__half, int>(idx, table, out, n, D, V, scale, st) : embedding_fwd<__half, long long>(idx, table, out, n, D, V, scale, st);
}

// grad[V, D] = scale * sums of dout's rows (pitch ldd) by token; tokens outside [0, V) and `pad` give nothing (pad < 0: there is none).  All of grad is written.
// order: 2 n entries of 8 bytes, or null: all by one launch (up to 2048 tokens); part: 2 ceil(n / tile) rows of D floats; tile: up to 64 sorted rows a CTA.
int lt_token_embedding_bwd(int type, const void* idx, int idx32, const void* dout, long long ldd, void* grad, long long n, int D, int V, float scale, long long pad,
                           void* order, float* part, int tile, void* stream) {
  using namespace lt;
  if (type < 0 || type > 2 || n < 0 || n > 0x7fffffffll - 4096 || D < 0 || D > 1 << 30 || V < 1 || V == 0x7fffffff || tile < 1 || tile > kMaxTile) return -int(kStatusBadArgument);
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
