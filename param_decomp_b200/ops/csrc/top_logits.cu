// The k largest logits of every row (descending, equal logits in the order of their columns), their columns, and the
// logarithm of the sum of exp(z / T) over the rest of the row.
//
// One block a row, two passes. First: every thread keeps the maximum of its own columns; the k-th largest T_0 of those
// maxima is a lower bound of the k-th largest logit, and a tight one (k = 64 of 512 threads: about 68 logits reach it).
// Second, out of L2: logits that reach T_0 are collected with their columns, all others go into the sum of
// exponentials relative to T_0. The collected ones are ranked by counting, with (logit, column) as one number, so the
// order in which they arrived does not matter. A row that defeats the bound (fewer than 2 k groups of 16 bytes, ties in
// masses, rows of -inf) is selected by its keys' digits instead, exactly and at any number of ties.
// HBM is read once; what bounds a row is its first pass.
#include <algorithm>

#include "rows.cuh"

namespace {

using namespace pd;

constexpr int kMaxK = 256;
constexpr int kRoom = 512;  // logits collected
constexpr float kLog2E = 1.4426950408889634f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Whole numbers in the order of the values: -0 equals +0, NaN above everything.
__device__ __forceinline__ uint32_t key_of(float v) {
  if (v != v) return 0xFFFFFFFFu;
  const uint32_t u = __float_as_uint(v + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}
// (logit, column) as one number: larger logits first, then lower columns.
__device__ __forceinline__ unsigned long long place_of(float v, int col) {
  return (static_cast<unsigned long long>(key_of(v)) << 32) | (0xFFFFFFFFu - static_cast<uint32_t>(col));
}

// 16 bytes of a row at a time, at 16-byte addresses wherever the row starts: group g holds columns g kE - shift + j.
template <typename T>
struct Row {
  static constexpr int kE = 16 / sizeof(T);
  const T* base;  // column 0
  int V, shift, groups;
  __device__ __forceinline__ Row(const T* p, int V_) : base(p), V(V_) {
    shift = static_cast<int>((reinterpret_cast<uintptr_t>(p) & 15) / sizeof(T));
    groups = (shift + V + kE - 1) / kE;
  }
  // The group's values; columns outside the row hold -inf.
  __device__ __forceinline__ void load(int g, float (&v)[kE]) const {
    const int c0 = g * kE - shift;
    if (c0 >= 0 && c0 + kE <= V) {
      const uint4 q = *reinterpret_cast<const uint4*>(base + c0);
      const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (sizeof(T) == 2) {
          v[2 * j] = __uint_as_float(w[j] << 16);
          v[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
        } else {
          v[j] = __uint_as_float(w[j]);
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < kE; ++j) v[j] = c0 + j >= 0 && c0 + j < V ? as_float(base[c0 + j]) : -INFINITY;
    }
  }
  __device__ __forceinline__ bool inside(int col) const { return col >= 0 && col < V; }
};

// log of the sum of exp(z / T) over the columns behind the place `last` of the k-th, relative to their own maximum.
template <typename T>
__device__ float rest_logsumexp(const Row<T>& row, unsigned long long last, float inv_t, float (*red)[32]) {
  constexpr int kE = Row<T>::kE;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  float m = -INFINITY;
  bool nan = false;
  for (int g = threadIdx.x; g < row.groups; g += blockDim.x) {
    float v[kE];
    row.load(g, v);
#pragma unroll
    for (int j = 0; j < kE; ++j) {
      const int col = g * kE - row.shift + j;
      if (row.inside(col) && place_of(v[j], col) < last) {
        m = fmaxf(m, v[j]);
        nan |= v[j] != v[j];
      }
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  nan = __syncthreads_or(nan);
  if (lane == 0) red[0][warp] = m;
  __syncthreads();
  for (int w = 0; w < warps; ++w) m = fmaxf(m, red[0][w]);
  float s = 0.0f;
  if (m > -INFINITY && m < INFINITY) {
    for (int g = threadIdx.x; g < row.groups; g += blockDim.x) {
      float v[kE];
      row.load(g, v);
#pragma unroll
      for (int j = 0; j < kE; ++j) {
        const int col = g * kE - row.shift + j;
        if (row.inside(col) && place_of(v[j], col) < last) s += ex2((v[j] - m) * (inv_t * kLog2E));
      }
    }
  }
  s = warp_sum(s);
  if (lane == 0) red[1][warp] = s;
  __syncthreads();
  s = 0.0f;
  for (int w = 0; w < warps; ++w) s += red[1][w];
  __syncthreads();
  if (nan) return NAN;
  return m > -INFINITY && m < INFINITY ? m * inv_t + logf(s) : m;
}

// The k-th largest (value, column) place by the keys' digits from the top; leaves the k best in `kept` (any order).
template <typename T>
__device__ void select_by_digits(const Row<T>& row, int k, unsigned long long* kept, int* hist, int* shared) {
  constexpr int kE = Row<T>::kE;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint32_t prefix = 0;
  int need = k;
  constexpr int kDigits = sizeof(T);  // bf16 keys are settled by their upper 16 bits
#pragma unroll 1
  for (int digit = 0; digit < kDigits; ++digit) {
    const int down = 24 - 8 * digit;
    for (int i = tid; i < 256; i += blockDim.x) hist[i] = 0;
    __syncthreads();
    for (int g = tid; g < row.groups; g += blockDim.x) {
      float v[kE];
      row.load(g, v);
#pragma unroll
      for (int j = 0; j < kE; ++j) {
        const uint32_t key = key_of(v[j]);
        if (row.inside(g * kE - row.shift + j) && (digit == 0 || key >> (down + 8) == prefix))
          atomicAdd(hist + ((key >> down) & 255), 1);
      }
    }
    __syncthreads();
    if (warp == 0) {  // lane l holds the eight bins 255 - 8 l and below: from the largest digit down
      int sum = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) sum += hist[255 - 8 * lane - j];
      int upto = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
      }
      int before = upto - sum;
      if (before < need && need <= upto) {
        for (int j = 0; j < 8; ++j) {
          const int bin = 255 - 8 * lane - j, here = hist[bin];
          if (need <= before + here) {
            shared[0] = bin;
            shared[1] = need - before;
            break;
          }
          before += here;
        }
      }
    }
    __syncthreads();
    prefix = prefix << 8 | static_cast<uint32_t>(shared[0]);
    need = shared[1];
    __syncthreads();
  }
  // everything above the k-th key, and the first `need` columns that hold it
  if (tid == 0) shared[0] = shared[1] = 0;
  __syncthreads();
  constexpr int kDown = 32 - 8 * kDigits;
  for (int g0 = 0; g0 < row.groups; g0 += blockDim.x) {
    const int g = g0 + tid;
    float v[kE];
    int equal = 0;
    if (g < row.groups) {
      row.load(g, v);
#pragma unroll
      for (int j = 0; j < kE; ++j) {
        const int col = g * kE - row.shift + j;
        if (!row.inside(col)) continue;
        const uint32_t key = key_of(v[j]) >> kDown;
        if (key > prefix) kept[atomicAdd(shared, 1)] = place_of(v[j], col);
        equal += key == prefix;
      }
    }
    int upto = equal;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += u;
    }
    if (lane == 31) hist[warp] = upto;
    __syncthreads();
    int before = shared[1] + upto - equal, all = 0;
    for (int w = 0; w < static_cast<int>(blockDim.x) / 32; ++w) {
      if (w < warp) before += hist[w];
      all += hist[w];
    }
    if (g < row.groups && equal > 0) {
#pragma unroll
      for (int j = 0; j < kE; ++j) {
        const int col = g * kE - row.shift + j;
        if (!row.inside(col) || key_of(v[j]) >> kDown != prefix) continue;
        if (before < need) kept[k - need + before] = place_of(v[j], col);
        ++before;
      }
    }
    __syncthreads();
    if (tid == 0) shared[1] += all;
    __syncthreads();
  }
}

template <typename T>
__global__ void __launch_bounds__(512) top_logits_kernel(const T* __restrict__ z, long long ld, int V, int k, float inv_t,
                                                         T* __restrict__ values, int* __restrict__ indices,
                                                         float* __restrict__ tail) {
  constexpr int kE = Row<T>::kE;
  __shared__ unsigned long long kept[kRoom];
  __shared__ float red[2][32];
  __shared__ int hist[256], shared[2], found;
  __shared__ unsigned long long last;
  const int tid = threadIdx.x, nt = blockDim.x, lane = tid & 31, warp = tid >> 5;
  const long long r = blockIdx.x;
  const Row<T> row(z + r * ld, V);
  bool by_digits = min(nt, row.groups) < 2 * k;
  int n = 0;
  float low = 0.0f, sum = 0.0f;
  if (!by_digits) {
    float m = -INFINITY;
#pragma unroll 4
    for (int g = tid; g < row.groups; g += nt) {
      float v[kE];
      row.load(g, v);
#pragma unroll
      for (int j = 0; j < kE; ++j) m = fmaxf(m, v[j]);
    }
    if (tid == 0) found = 0;
    // the k-th largest of the threads' maxima, in the upper 16 bits of its key (rounded down: still a lower bound)
    const uint32_t mine = key_of(m) >> 16;
    uint32_t bound = 0;
#pragma unroll 1
    for (int bit = 15; bit >= 0; --bit) {
      const uint32_t trial = bound | 1u << bit;
      if (__syncthreads_count(mine >= trial) >= k) bound = trial;
    }
    low = value_of(bound << 16);
    by_digits = !(low > -INFINITY && low < INFINITY);
    if (!by_digits) {
      const float c = inv_t * kLog2E;
#pragma unroll 4
      for (int g = tid; g < row.groups; g += nt) {
        float v[kE];
        row.load(g, v);
#pragma unroll
        for (int j = 0; j < kE; ++j) {
          if (v[j] < low) {
            sum += ex2((v[j] - low) * c);
          } else {
            const int at = atomicAdd(&found, 1);
            if (at < kRoom) kept[at] = place_of(v[j], g * kE - row.shift + j);
          }
        }
      }
      sum = warp_sum(sum);
      if (lane == 0) red[0][warp] = sum;
      __syncthreads();
      sum = 0.0f;
      for (int w = 0; w < nt / 32; ++w) sum += red[0][w];
      n = found;
      by_digits = n > kRoom;
    }
    __syncthreads();
  }
  if (by_digits) {
    select_by_digits(row, k, kept, hist, shared);
    n = k;
  }
  // rank by counting; every place differs from every other
  float over = 0.0f;  // collected, but not among the k
  for (int i = tid; i < n; i += nt) {
    const unsigned long long own = kept[i];
    int rank = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) rank += kept[j] > own;
    const int col = static_cast<int>(0xFFFFFFFFu - static_cast<uint32_t>(own));
    if (rank < k) {
      values[r * k + rank] = row.base[col];
      indices[r * k + rank] = col;
      if (rank == k - 1) last = own;
    } else {
      over += ex2((as_float(row.base[col]) - low) * (inv_t * kLog2E));
    }
  }
  // What is left: the sum relative to the bound with the collected ones that did not make it. Sums that are tiny have lost
  // what lies far below the bound, and take the exact way; so do rows selected by digits.
  const bool exact = __syncthreads_or(by_digits || !(over < 1e30f));
  float result;
  if (!exact) {
    const float s = warp_sum(over);
    if (lane == 0) red[1][warp] = s;
    __syncthreads();
    for (int w = 0; w < nt / 32; ++w) sum += red[1][w];
    result = low * inv_t + logf(sum);
  }
  if (exact || !(sum > 1e-20f)) result = rest_logsumexp(row, last, inv_t, red);
  if (tid == 0) tail[r] = result;
}

template <typename T>
int top(const void* z, long long rows, int V, long long ld, int k, float inv_t, void* values, int* indices, float* tail,
        cudaStream_t st) {
  const int groups = (V + Row<T>::kE - 1) / Row<T>::kE;
  const int threads = groups > 1024 || k > 64 ? 512 : 256;
  top_logits_kernel<T><<<static_cast<unsigned>(rows), threads, 0, st>>>(static_cast<const T*>(z), ld, V, k, inv_t,
                                                                        static_cast<T*>(values), indices, tail);
  return cudaGetLastError() == cudaSuccess ? 0 : 1;
}

}  // namespace

// z [rows, V] in bf16 or fp32, rows ld elements apart; values, indices [rows, k], tail [rows].
extern "C" int pd_top_logits(const void* z, long long rows, int V, long long ld, int k, float inv_t, void* values,
                             int* indices, float* tail, int z_fp32, void* stream) {
  if (rows <= 0 || rows >= (1ll << 31) || V <= 0 || k <= 0 || k > kMaxK || k > V || !(inv_t > 0.0f)) return 5;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return z_fp32 ? top<float>(z, rows, V, ld, k, inv_t, values, indices, tail, st)
                : top<__nv_bfloat16>(z, rows, V, ld, k, inv_t, values, indices, tail, st);
}
