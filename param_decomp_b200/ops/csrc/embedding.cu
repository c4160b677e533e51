// Token embedding: y[n] = scale E[t_n], and its gradient dE[v] = scale sum over n with t_n = v of dy[n].
// Both are bound by HBM: the lookup reads a table row and writes an output row a token, the gradient reads the tokens'
// rows once and writes every row of the table (most of them zeros).
//
// The gradient sums each row in fp32 over its tokens in ascending order and rounds once, with two launches and no float
// atomics. First kernel: block b owns a span of the vocabulary. Its 32 warps walk all tokens, each its own consecutive
// part: once to count the block's tokens by id and warp (and the valid tokens of lower ids, which gives the block's place
// in the sorted order without asking the other blocks), once more to write each token's place in that order (a stable
// counting sort: id, then warp, then position). All blocks read all tokens, from L2. The block then writes the zero rows
// of its span and sums the rows of ids with up to kSlab tokens. Second kernel: ids with more tokens, in slabs of kSlab
// places of the sorted order, so a token that fills a tenth of the batch is shared by many blocks; a slab's sum goes to
// scratch and the block that finishes a run last adds its slabs in their order.
#include <algorithm>

#include "rows.cuh"

namespace {

using namespace pd;

constexpr int kSlab = 32;
constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kMaxSpan = 1280;  // ids a block: 32 counts of 4 bytes each in shared memory

__device__ __forceinline__ long long token_at(const void* tokens, int wide, long long i) {
  return wide ? static_cast<const long long*>(tokens)[i] : static_cast<const int*>(tokens)[i];
}

// ---- lookup ------------------------------------------------------------------------------------------------------
// A warp takes kRowsAhead tokens at a time, so that many loads are in flight before the first is needed.
template <typename P, typename T, bool kVec>
__global__ void __launch_bounds__(256) embedding_lookup_kernel(const void* __restrict__ tokens, int wide,
                                                               const P* __restrict__ table, T* __restrict__ y,
                                                               long long n, long long V, int d, float scale,
                                                               int* __restrict__ status, int* __restrict__ refused) {
  constexpr int kRowsAhead = 4;
  const int lane = threadIdx.x & 31;
  const long long warps = static_cast<long long>(gridDim.x) * (blockDim.x / 32);
  for (long long r0 = (blockIdx.x * (blockDim.x / 32ll) + threadIdx.x / 32) * kRowsAhead; r0 < n; r0 += warps * kRowsAhead) {
    const P* src[kRowsAhead];
    bool bad = false;
#pragma unroll
    for (int k = 0; k < kRowsAhead; ++k) {
      const long long t = r0 + k < n ? token_at(tokens, wide, r0 + k) : -1;
      const bool known = t >= 0 && t < V;
      bad |= !known && r0 + k < n;
      src[k] = known ? table + t * d : nullptr;
    }
    if (bad && lane == 0) {
      atomicCAS(status, 0, kBadToken);
      *static_cast<volatile int*>(refused) = 1;
    }
    for (int c = kVec ? 8 * lane : lane; c < d; c += kVec ? 256 : 32) {
      if (kVec) {
        Raw8<P> raw[kRowsAhead];
#pragma unroll
        for (int k = 0; k < kRowsAhead; ++k)
          if (src[k] != nullptr) raw[k] = load8(src[k] + c);
#pragma unroll
        for (int k = 0; k < kRowsAhead; ++k) {
          if (r0 + k >= n) break;
          float v[8];
          if (src[k] != nullptr) {
            unpack8(raw[k], v);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] *= scale;
          } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = 0.0f;
          }
          store8(y + (r0 + k) * d + c, v);
        }
      } else {
        float v[kRowsAhead];
#pragma unroll
        for (int k = 0; k < kRowsAhead; ++k) v[k] = src[k] != nullptr ? as_float(src[k][c]) : 0.0f;
#pragma unroll
        for (int k = 0; k < kRowsAhead; ++k)
          if (r0 + k < n) store1(y + (r0 + k) * d + c, v[k] * scale);
      }
    }
  }
}

// ---- gradient ----------------------------------------------------------------------------------------------------
struct Runs {        // what the first kernel tells the second
  int* order;        // [n] position of the token at each place of the sorted order
  int* run_start;    // [n] place where the run of an id with more than kSlab tokens starts, at each of its places; else -1
  int* id;           // [slabs] of the run that starts in the slab (a longer run than a slab: at most one does)
  int* end;          // [slabs] place behind it
  int* done;         // [slabs] slabs of it that are summed
};

template <typename T, typename P, bool kVec>
__global__ void __launch_bounds__(kSortThreads, 1) embedding_sort_kernel(const void* __restrict__ tokens, int wide,
                                                                      const T* __restrict__ dy, P* __restrict__ dE,
                                                                      int n, long long V, int d, float scale, int span,
                                                                      Runs runs) {
  extern __shared__ int hist[];  // [kSortWarps][span] counts, then next places; behind it [span] counts of the ids
  int* count = hist + kSortWarps * span;
  __shared__ int warp_total[kSortWarps], below_of[kSortWarps];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const long long lo = static_cast<long long>(blockIdx.x) * span;
  const int ids = static_cast<int>(min(static_cast<long long>(span), V - lo));
  for (int i = tid; i < kSortWarps * span; i += kSortThreads) hist[i] = 0;
  __syncthreads();
  const int part = (n + kSortThreads - 1) / kSortThreads * 32;  // tokens a warp
  const int from = min(n, warp * part), to = min(n, from + part);
  int* mine = hist + warp * span;
  int below = 0;
#pragma unroll 8
  for (int i = from + lane; i < to; i += 32) {
    const long long t = token_at(tokens, wide, i);
    below += t >= 0 && t < lo;
    if (t >= lo && t < lo + ids) atomicAdd(mine + (t - lo), 1);
  }
  below = __reduce_add_sync(0xffffffffu, below);
  if (lane == 0) below_of[warp] = below;
  __syncthreads();
  // exclusive sums over (id, warp); a thread takes two neighbouring ids
  int c[2] = {0, 0};
#pragma unroll
  for (int k = 0; k < 2; ++k)
    if (2 * tid + k < ids)
      for (int w = 0; w < kSortWarps; ++w) c[k] += hist[w * span + 2 * tid + k];
  int incl = c[0] + c[1];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) warp_total[warp] = incl;
  __syncthreads();
  int at = incl - c[0] - c[1];
  for (int w = 0; w < kSortWarps; ++w) {
    at += below_of[w];
    if (w < warp) at += warp_total[w];
  }
#pragma unroll
  for (int k = 0; k < 2; ++k)
    if (2 * tid + k < ids) {
      const int i = 2 * tid + k;
      count[i] = c[k];
      if (c[k] > kSlab) {
        const int slab = at / kSlab;
        runs.id[slab] = static_cast<int>(lo) + i;
        runs.end[slab] = at + c[k];
        runs.done[slab] = 0;
      }
      for (int w = 0; w < kSortWarps; ++w) {
        const int v = hist[w * span + i];
        hist[w * span + i] = at;
        at += v;
      }
    }
  __syncthreads();
  // zero rows first: the stores drain while the tokens are placed
  const int step = kVec ? 8 : 1;
  for (int i = warp; i < ids; i += kSortWarps) {
    if (count[i] != 0) continue;
    P* out = dE + (lo + i) * d;
    const float zero[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    for (int col = step * lane; col < d; col += 32 * step) {
      if (kVec)
        store8(out + col, zero);
      else
        store1(out + col, 0.0f);
    }
  }
#pragma unroll 4
  for (int i = from + lane; i - lane < to; i += 32) {
    const long long t = i < to ? token_at(tokens, wide, i) : -1;
    const bool own = t >= lo && t < lo + ids;
    const unsigned all = __ballot_sync(0xffffffffu, own);
    if (own) {
      const int bin = static_cast<int>(t - lo);
      const unsigned same = __match_any_sync(all, bin);
      const int first = mine[bin], rank = __popc(same & ((1u << lane) - 1));
      __syncwarp(all);
      if (rank == 0) mine[bin] = first + __popc(same);
      runs.order[first + rank] = i;
    }
    __syncwarp();
  }
  __syncthreads();
  let_next_start();
  // place of an id's first token: where the last warp's part of the id before it ended
  int base = 0;
  for (int w = 0; w < kSortWarps; ++w) base += below_of[w];
  const int* ends = hist + (kSortWarps - 1) * span;
  if (lo + ids == V)  // places behind the last valid token
    for (int i = ends[ids - 1] + tid; i < n; i += kSortThreads) runs.run_start[i] = -1;
  for (int i = warp; i < ids; i += kSortWarps) {
    const int k = count[i], start = i == 0 ? base : ends[i - 1];
    for (int j = lane; j < k; j += 32) runs.run_start[start + j] = k > kSlab ? start : -1;
    if (k == 0 || k > kSlab) continue;
    const int row_of = lane < k ? runs.order[start + lane] : 0;
    P* out = dE + (lo + i) * d;
    if (kVec) {
      constexpr int kCh = 3;
      for (int c0 = 8 * lane; c0 - 8 * lane < d; c0 += 256 * kCh) {
        float acc[kCh][8] = {};
        for (int r = 0; r < k; ++r) {
          const T* row = dy + static_cast<long long>(__shfl_sync(0xffffffffu, row_of, r)) * d;
          Raw8<T> raw[kCh];
#pragma unroll
          for (int h = 0; h < kCh; ++h)
            if (c0 + 256 * h < d) raw[h] = load8(row + c0 + 256 * h);
#pragma unroll
          for (int h = 0; h < kCh; ++h)
            if (c0 + 256 * h < d) {
              float v[8];
              unpack8(raw[h], v);
#pragma unroll
              for (int j = 0; j < 8; ++j) acc[h][j] += v[j];
            }
        }
#pragma unroll
        for (int h = 0; h < kCh; ++h)
          if (c0 + 256 * h < d) {
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[h][j] *= scale;
            store8(out + c0 + 256 * h, acc[h]);
          }
      }
    } else {
      constexpr int kCh = 8;
      for (int c0 = lane; c0 - lane < d; c0 += 32 * kCh) {
        float acc[kCh] = {};
        for (int r = 0; r < k; ++r) {
          const T* row = dy + static_cast<long long>(__shfl_sync(0xffffffffu, row_of, r)) * d;
#pragma unroll
          for (int h = 0; h < kCh; ++h)
            if (c0 + 32 * h < d) acc[h] += as_float(row[c0 + 32 * h]);
        }
#pragma unroll
        for (int h = 0; h < kCh; ++h)
          if (c0 + 32 * h < d) store1(out + c0 + 32 * h, acc[h] * scale);
      }
    }
  }
}

// Sums that other blocks wrote in this launch are read past L1, which may hold their lines from before.
__device__ __forceinline__ float value(const float* p, bool fresh) { return fresh ? __ldcg(p) : *p; }
__device__ __forceinline__ float value(const __nv_bfloat16* p, bool) { return as_float(*p); }
__device__ __forceinline__ void values8(const float* p, bool fresh, float (&v)[8]) {
  const float4* q = reinterpret_cast<const float4*>(p);
  const float4 a = fresh ? __ldcg(q) : q[0], b = fresh ? __ldcg(q + 1) : q[1];
  v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}
__device__ __forceinline__ void values8(const __nv_bfloat16* p, bool, float (&v)[8]) { unpack8(load8(p), v); }

// Sum over `rows` rows, row r at `row(r)`, of this thread's columns; the block's threads are `groups` groups of `width`
// that take every groups-th row, and group 0 adds the groups' sums in order and hands them to `put(column, values)`.
template <bool kVec, bool kFresh, typename Row, typename Put>
__device__ __forceinline__ void block_row_sum(int rows, int d, int width, float* red, Row row, Put put) {
  constexpr int kPer = kVec ? 8 : 1;
  const int groups = blockDim.x / width, g = threadIdx.x / width, c = threadIdx.x % width;
  for (int c0 = 0; c0 < d; c0 += width * kPer) {
    const int col = c0 + c * kPer;
    float acc[kPer] = {};
    if (col < d) {
#pragma unroll 8
      for (int r = g; r < rows; r += groups) {
        const auto* p = row(r) + col;
        if (kVec) {
          float v[8];
          values8(p, kFresh, v);
#pragma unroll
          for (int j = 0; j < kPer; ++j) acc[j] += v[j];
        } else {
          acc[0] += value(p, kFresh);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < kPer; ++j) red[j * blockDim.x + threadIdx.x] = acc[j];
    __syncthreads();
    if (g == 0 && col < d) {
      for (int h = 1; h < groups; ++h)
#pragma unroll
        for (int j = 0; j < kPer; ++j) acc[j] += red[j * blockDim.x + h * width + c];
      put(col, acc);
    }
    __syncthreads();
  }
}

template <typename T, typename P, bool kVec>
__global__ void __launch_bounds__(256) embedding_runs_kernel(const T* __restrict__ dy, P* __restrict__ dE, int n, int d,
                                                             float scale, Runs runs, float* __restrict__ partial) {
  __shared__ int where[kSlab], place[kSlab], last;
  __shared__ float red[256 * 8];
  wait_for_previous();
  const int slab = blockIdx.x, begin = slab * kSlab, stop = min(n, begin + kSlab);
  if (threadIdx.x < kSlab) {
    const bool in = begin + static_cast<int>(threadIdx.x) < stop;
    where[threadIdx.x] = in ? runs.run_start[begin + threadIdx.x] : -1;
    place[threadIdx.x] = in ? runs.order[begin + threadIdx.x] : 0;
  }
  __syncthreads();
  constexpr int kPer = kVec ? 8 : 1;
  int width = 32;
  while (width < 256 && width * kPer < d) width *= 2;
  // Two runs at most: one that comes in over the slab's beginning, one that starts in it.
  for (int which = 0; which < 2; ++which) {
    int a = 0, b;
    if (which == 0) {
      if (where[0] < 0 || where[0] >= begin) continue;
    } else {
      while (a < kSlab && (where[a] < 0 || where[a] < begin)) ++a;
      if (a == kSlab) continue;
    }
    const int start = where[a], slot = start / kSlab, end = runs.end[slot], id = runs.id[slot];
    b = min(kSlab, end - begin);
    float* mine = partial + (2ll * slab + which) * d;
    block_row_sum<kVec, false>(
        b - a, d, width, red, [&](int r) { return dy + static_cast<long long>(place[a + r]) * d; },
        [&](int col, const float(&v)[kPer]) {
#pragma unroll
          for (int j = 0; j < kPer; ++j) mine[col + j] = v[j];
        });
    __threadfence();
    __syncthreads();
    const int slabs = (end - 1) / kSlab - slot + 1;
    if (threadIdx.x == 0) last = atomicAdd(runs.done + slot, 1) == slabs - 1;
    __syncthreads();
    if (last) {
      __threadfence();
      const float* parts = partial;
      P* out = dE + static_cast<long long>(id) * d;
      block_row_sum<kVec, true>(
          slabs, d, width, red, [&](int r) { return parts + (2ll * (slot + r) + (r == 0 ? 1 : 0)) * d; },
          [&](int col, const float(&v)[kPer]) {
            float o[kPer];
#pragma unroll
            for (int j = 0; j < kPer; ++j) o[j] = v[j] * scale;
            if constexpr (kVec)
              store8(out + col, o);
            else
              store1(out + col, o[0]);
          });
    }
    __syncthreads();
  }
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <typename P, typename T, bool kVec>
int lookup(const void* tokens, int wide, const void* table, void* y, long long n, long long V, int d, float scale,
           int* status, int* refused, cudaStream_t st) {
  const int blocks = static_cast<int>(std::min<long long>((n + 31) / 32, 148 * 8));
  embedding_lookup_kernel<P, T, kVec><<<blocks, 256, 0, st>>>(tokens, wide, static_cast<const P*>(table),
                                                              static_cast<T*>(y), n, V, d, scale, status, refused);
  return cudaGetLastError() == cudaSuccess ? 0 : 1;
}

template <typename T, typename P, bool kVec>
int grad(const void* tokens, int wide, const void* dy, void* dE, int n, long long V, int d, float scale, int* ints,
         float* partial, cudaStream_t st) {
  const long long blocks_min = (V + kMaxSpan - 1) / kMaxSpan;
  const int span = static_cast<int>((V + std::max(148ll, blocks_min) - 1) / std::max(148ll, blocks_min));
  const int blocks = static_cast<int>((V + span - 1) / span);
  const int slabs = (n + kSlab - 1) / kSlab;
  const Runs runs{ints, ints + n, ints + 2ll * n, ints + 2ll * n + slabs, ints + 2ll * n + 2ll * slabs};
  const size_t smem = static_cast<size_t>(span) * (kSortWarps + 1) * sizeof(int);
  auto kern = embedding_sort_kernel<T, P, kVec>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSpan * (kSortWarps + 1) * 4) !=
      cudaSuccess)
    return 2;
  kern<<<blocks, kSortThreads, smem, st>>>(tokens, wide, static_cast<const T*>(dy), static_cast<P*>(dE), n, V, d, scale,
                                           span, runs);
  if (cudaGetLastError() != cudaSuccess) return 1;
  if (n <= kSlab) return 0;  // no id has more tokens than a slab
  return launch_after(embedding_runs_kernel<T, P, kVec>, dim3(slabs), dim3(256), 0, st, static_cast<const T*>(dy),
                      static_cast<P*>(dE), n, d, scale, runs, partial) == cudaSuccess
             ? 0
             : 1;
}

}  // namespace

// y [n, d] = scale table[tokens]; a token outside [0, V) is reported and gives a zero row. tokens int64 (wide) or int32.
extern "C" int pd_embedding(const void* tokens, int wide, const void* table, void* y, long long n, long long V, int d,
                            float scale, int table_fp32, int y_fp32, int* status, int* refused, void* stream) {
  if (n <= 0 || V <= 0 || d <= 0) return 5;
  const bool vec = d % 8 == 0 && aligned16(table) && aligned16(y);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto go = [&](auto p, auto t) {
    using P = decltype(p);
    using T = decltype(t);
    return vec ? lookup<P, T, true>(tokens, wide, table, y, n, V, d, scale, status, refused, st)
               : lookup<P, T, false>(tokens, wide, table, y, n, V, d, scale, status, refused, st);
  };
  using B = __nv_bfloat16;
  if (table_fp32) return y_fp32 ? go(float(), float()) : go(float(), B());
  return y_fp32 ? go(B(), float()) : go(B(), B());
}

// Scratch of the gradient, in ints and in floats.
extern "C" long long pd_embedding_grad_ints(long long n) { return 2 * n + 3 * ((n + kSlab - 1) / kSlab); }
extern "C" long long pd_embedding_grad_floats(long long n, int d) { return 2 * ((n + kSlab - 1) / kSlab) * d; }

// dE [V, d], every row of it; tokens outside [0, V) take no part.
extern "C" int pd_embedding_grad(const void* tokens, int wide, const void* dy, void* dE, long long n, long long V, int d,
                                 float scale, int dy_fp32, int table_fp32, int* ints, float* partial, void* stream) {
  if (n < 0 || n >= (1ll << 30) || V <= 0 || V >= (1ll << 31) || d <= 0) return 5;
  const bool vec = d % 8 == 0 && aligned16(dy) && aligned16(dE) && aligned16(partial);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto go = [&](auto t, auto p) {
    using T = decltype(t);
    using P = decltype(p);
    return vec ? grad<T, P, true>(tokens, wide, dy, dE, static_cast<int>(n), V, d, scale, ints, partial, st)
               : grad<T, P, false>(tokens, wide, dy, dE, static_cast<int>(n), V, d, scale, ints, partial, st);
  };
  using B = __nv_bfloat16;
  if (dy_fp32) return table_fp32 ? go(float(), float()) : go(float(), B());
  return table_fp32 ? go(B(), float()) : go(B(), B());
}
