// Layer norm over rows of `d` columns:
//   mean = sum x / d, var = sum (x - mean)^2 / d, xh = (x - mean) rstd, rstd = 1 / sqrt(var + eps), y = xh w + b
//   dx = rstd (g - mean(g) - xh mean(g xh)) with g = dy w;  dw = sum over rows of dy xh;  db = sum over rows of dy
// Bound by HBM: 2 (forward) and 3 (backward) passes of the row data. A group of warps holds a few rows at a time in
// registers as they lie in memory, 8 columns a thread (up to 4096 columns; two or three times 8 beyond), so x and dy cross
// HBM once, and one barrier serves the sums of all those rows. The handfuls to come are copied into shared memory meanwhile
// (every thread's own columns, so no barrier but the thread's own wait): 60 to 90 KB an SM are on their way at any time,
// more than registers could wait for. The variance is summed around the mean that was just formed, not from sums of
// squares. All sums are in fp32; what is stored is rounded once.
// The weight gradients: every thread keeps the sums of its own columns over all rows that its group walks; blocks write
// those to scratch and a second kernel adds them in a fixed order, so a result does not change from run to run.
// Measured: 32,768 rows of 768 bf16: forward 24 us (4.1 TB/s, 0.64 of copy bandwidth), backward 35 (4.3), parameters 3; 6151
// rows of 2047 fp32: 33 and 38 us (3.1 and 4.0 TB/s). Of the 24 us a block is at work for 20, the first 4 of them until its
// first rows are there; 131,072 rows of 768 forward: 75 us, 5.4 TB/s, 0.83. Two to eight times as many blocks of fewer rows
// cost 3 to 10 us more, fewer rows a group at a time change nothing.
#include <algorithm>

#include "rows.cuh"

namespace {

using namespace pd;

constexpr int kMaxWarps = 16;  // of a row
constexpr int kMaxChunks = 3;  // of 8 columns a thread
constexpr int kMaxGroups = 8;  // of a block

// Eight elements as they lie in memory.
template <typename T>
struct Words {
  uint32_t w[2 * sizeof(T)];
  __device__ __forceinline__ f32x2 pair(int i) const {  // elements 2 i and 2 i + 1
    if constexpr (sizeof(T) == 2)
      return unpack_bf16_2(w[i]);
    else
      return pk2u(w[2 * i], w[2 * i + 1]);
  }
};

// Which column element j of chunk c is, for thread t of `tpr` that share a row. Rows of 16-byte pieces: eight
// neighbours a thread; any other row: threads side by side, one element each.
template <bool kVec>
__device__ __forceinline__ int column(int c, int j, int t, int tpr) {
  return kVec ? (c * tpr + t) * 8 + j : (c * 8 + j) * tpr + t;
}
// Columns outside the row read as zero.
template <typename T, bool kVec>
__device__ __forceinline__ Words<T> load_words(const T* __restrict__ row, int c, int d, int t, int tpr, bool there) {
  Words<T> r;
#pragma unroll
  for (int i = 0; i < static_cast<int>(2 * sizeof(T)); ++i) r.w[i] = 0u;
  if constexpr (kVec) {
    const int col = column<true>(c, 0, t, tpr);
    if (there && col < d) {
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) {
        const uint4 q = reinterpret_cast<const uint4*>(row + col)[i];
        r.w[4 * i] = q.x, r.w[4 * i + 1] = q.y, r.w[4 * i + 2] = q.z, r.w[4 * i + 3] = q.w;
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int col = column<false>(c, j, t, tpr);
      if (there && col < d) {
        if constexpr (sizeof(T) == 2)
          r.w[j / 2] |= static_cast<uint32_t>(reinterpret_cast<const unsigned short*>(row)[col]) << 16 * (j % 2);
        else
          r.w[j] = reinterpret_cast<const uint32_t*>(row)[col];
      }
    }
  }
  return r;
}
// Rows of 16-byte pieces are copied ahead; in pieces of 4 bytes that does not gain (35 and 42 us against 31 and 36 on 6151
// rows of 2047 fp32 columns), so other rows are loaded when their turn comes.
__device__ __forceinline__ void copy_async_16(uint32_t to, const void* from, bool there) {  // zeros where not
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");
}
// The handfuls of rows that a thread's group walks, kTensors rows of kCh chunks of 8 columns each.
template <typename T, int kCh, int kRows, int kTensors>
struct Ahead {
  static constexpr int kParts = sizeof(T) / 2;  // 16-byte pieces of 8 elements
  static constexpr int kPieces = kRows * kTensors * kCh * kParts;
  static constexpr int kStages = kPieces <= 4 ? 4 : kPieces <= 8 ? 3 : 2;  // up to 192 KB with 512 threads
  const T* from[kTensors];  // this thread's first column
  int rows, d, stride;      // columns between chunks
  int inside;               // chunks that lie in the row
  uint32_t slot;            // this thread's piece 0 of stage 0; pieces lie blockDim.x * 16 bytes apart

  // Ask for the handful at r0 (nothing but an empty group of copies past the last row).
  __device__ __forceinline__ void ask(int stage, int r0) const {
    uint32_t to = slot + stage * (kPieces * 16) * blockDim.x;
    if (r0 < rows) {
#pragma unroll
      for (int k = 0; k < kRows; ++k) {
        const bool row = r0 + k < rows;
        const long long at = static_cast<long long>(row ? r0 + k : r0) * d;
#pragma unroll
        for (int n = 0; n < kTensors; ++n)
#pragma unroll
          for (int c = 0; c < kCh; ++c) {
            const T* p = from[n] + (c < inside ? at + c * stride : 0);
#pragma unroll
            for (int part = 0; part < kParts; ++part, to += 16 * blockDim.x)
              copy_async_16(to, p + part * (16 / sizeof(T)), row && c < inside);
          }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  __device__ __forceinline__ Words<T> get(int stage, int k, int n, int c) const {
    Words<T> r;
#pragma unroll
    for (int part = 0; part < kParts; ++part) {
      const uint32_t at = slot + (stage * kPieces + ((k * kTensors + n) * kCh + c) * kParts + part) * 16 * blockDim.x;
      asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(r.w[4 * part]), "=r"(r.w[4 * part + 1]), "=r"(r.w[4 * part + 2]), "=r"(r.w[4 * part + 3])
                   : "r"(at)
                   : "memory");
    }
    return r;
  }
};
template <typename T, int kCh, int kRows, int kTensors>
__device__ __forceinline__ Ahead<T, kCh, kRows, kTensors> ahead_of(const T* a, const T* b, int rows, int d, int t, int tpr,
                                                                   void* slots) {
  Ahead<T, kCh, kRows, kTensors> r;
  int inside = 0;
  for (int c = 0; c < kCh; ++c) inside += column<true>(c, 0, t, tpr) < d;
  const int col = inside > 0 ? column<true>(0, 0, t, tpr) : 0;
  r.from[0] = a + col;
  if constexpr (kTensors > 1) r.from[1] = b + col;
  r.rows = rows, r.d = d, r.stride = 8 * tpr, r.inside = inside;
  r.slot = smem_u32(slots) + threadIdx.x * 16;
  return r;
}

template <typename T, bool kVec>
__device__ __forceinline__ void store_pairs(T* __restrict__ row, int c, int d, int t, int tpr, const f32x2 (&v)[4]) {
  if constexpr (kVec) {
    const int col = column<true>(c, 0, t, tpr);
    if (col >= d) return;
    if constexpr (sizeof(T) == 2) {
      *reinterpret_cast<uint4*>(row + col) = make_uint4(pack_bf16_2(v[0]), pack_bf16_2(v[1]), pack_bf16_2(v[2]), pack_bf16_2(v[3]));
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float2 a = unpack2(v[2 * i]), b = unpack2(v[2 * i + 1]);
        reinterpret_cast<float4*>(row + col)[i] = make_float4(a.x, a.y, b.x, b.y);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 a = unpack2(v[i]);
      const int c0 = column<false>(c, 2 * i, t, tpr), c1 = column<false>(c, 2 * i + 1, t, tpr);
      if (c0 < d) store1(row + c0, a.x);
      if (c1 < d) store1(row + c1, a.y);
    }
  }
}
// Eight parameters in either type (a branch every thread takes alike), `none` where there are none.
template <bool kVec>
__device__ __forceinline__ void load_params(const void* p, int fp32, float none, int c, int d, int t, int tpr, f32x2 (&v)[4]) {
  float x[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int col = column<kVec>(c, j, t, tpr);
    x[j] = p == nullptr ? none : 0.0f;
    if (p != nullptr && col < d)
      x[j] = fp32 ? static_cast<const float*>(p)[col] : as_float(static_cast<const __nv_bfloat16*>(p)[col]);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = pk2(x[2 * i], x[2 * i + 1]);
}
__device__ __forceinline__ float total_of(f32x2 v) {
  const float2 a = unpack2(v);
  return a.x + a.y;
}

// N sums over the 32 lanes with as few shuffles as there are halves to exchange; lane (j << (5 - log2 N)) ends with sum j.
template <int N>
__device__ __forceinline__ float lane_sums(float (&v)[N], int lane) {
  int o = 16;
#pragma unroll
  for (int n = N; n > 1; n /= 2, o /= 2) {
    const bool upper = lane & o;
#pragma unroll
    for (int i = 0; i < n / 2; ++i) {
      const float send = upper ? v[i] : v[i + n / 2], keep = upper ? v[i + n / 2] : v[i];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, send, o);
    }
  }
  float s = v[0];
#pragma unroll
  for (; o > 0; o /= 2) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}

// The threads that share rows: `wpr` warps, group `g` of the block.
struct Group {
  int wpr, g, t, tpr, lane, warp;  // warp: of the group
  float* red;                      // [2][wpr][8], used in turn, so one barrier a sum is enough
  int turn;
  // v[j] becomes its sum over the group's threads.
  template <int N>
  __device__ __forceinline__ void sum(float (&v)[N]) {
    constexpr int kShift = N == 8 ? 2 : N == 4 ? 3 : N == 2 ? 4 : 5;
    const float s = lane_sums(v, lane);
    if (wpr == 1) {
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] = __shfl_sync(0xffffffffu, s, j << kShift);
      return;
    }
    float* r = red + turn * wpr * 8;
    turn ^= 1;
    if ((lane & ((1 << kShift) - 1)) == 0) r[warp * 8 + (lane >> kShift)] = s;
    asm volatile("barrier.sync %0, %1;" ::"r"(g + 1), "r"(tpr) : "memory");
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = r[j];
    for (int w = 1; w < wpr; ++w) {
      float e[N];
      if constexpr (N >= 4) {
#pragma unroll
        for (int j = 0; j < N; j += 4) {
          const float4 q = *reinterpret_cast<const float4*>(r + w * 8 + j);
          e[j] = q.x, e[j + 1] = q.y, e[j + 2] = q.z, e[j + 3] = q.w;
        }
      } else {
#pragma unroll
        for (int j = 0; j < N; ++j) e[j] = r[w * 8 + j];
      }
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] += e[j];
    }
  }
};
__device__ __forceinline__ Group group_of(int wpr, float* red) {
  const int warp = threadIdx.x >> 5, g = warp / wpr;
  return Group{wpr, g, static_cast<int>(threadIdx.x) - g * 32 * wpr, 32 * wpr, static_cast<int>(threadIdx.x & 31), warp - g * wpr,
               red + g * 2 * wpr * 8, 0};
}

// kRows rows a group at a time.
template <typename T, int kCh, int kRows, bool kVec>
__global__ void __launch_bounds__(32 * kMaxWarps) layer_norm_fwd_kernel(
    const T* __restrict__ x, const void* __restrict__ w, const void* __restrict__ b, T* __restrict__ y,
    float* __restrict__ mean_out, float* __restrict__ rstd_out, int rows, int d, float eps, int wpr, int p_fp32) {
  extern __shared__ __align__(16) uint8_t slots[];
  __shared__ __align__(16) float red[kMaxWarps * 16];
  Group group = group_of(wpr, red);
  const int t = group.t, tpr = group.tpr, groups = blockDim.x / tpr;
  const float inv_d = 1.0f / static_cast<float>(d);
  const int first = (blockIdx.x * groups + group.g) * kRows, step = gridDim.x * groups * kRows;
  using Copies = Ahead<T, kCh, kRows, 1>;
  constexpr int kStages = Copies::kStages;
  const Copies ahead = ahead_of<T, kCh, kRows, 1>(x, nullptr, rows, d, t, tpr, slots);
  if constexpr (kVec)
    for (int i = 0; i < kStages - 1; ++i) ahead.ask(i, first + i * step);
  f32x2 scale[kCh][4], shift[kCh][4];
#pragma unroll
  for (int c = 0; c < kCh; ++c) {
    load_params<kVec>(w, p_fp32, 1.0f, c, d, t, tpr, scale[c]);
    load_params<kVec>(b, p_fp32, 0.0f, c, d, t, tpr, shift[c]);
  }
  int stage = 0;
  for (int r0 = first; r0 < rows; r0 += step) {
    f32x2 v[kRows][kCh][4];
    float s[kRows];
    if constexpr (kVec) asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      f32x2 a = 0ull;
#pragma unroll
      for (int c = 0; c < kCh; ++c) {
        const Words<T> words = kVec ? ahead.get(stage, k, 0, c)
                                    : load_words<T, kVec>(x + static_cast<long long>(r0 + k) * d, c, d, t, tpr, r0 + k < rows);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v[k][c][i] = words.pair(i);
          a = add2(a, v[k][c][i]);
        }
      }
      s[k] = total_of(a);
    }
    if constexpr (kVec) {
      ahead.ask((stage + kStages - 1) % kStages, r0 + (kStages - 1) * step);
      stage = (stage + 1) % kStages;
    }
    group.sum(s);
    float mean[kRows];
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      mean[k] = s[k] * inv_d;
      const f32x2 neg = pk2(-mean[k], -mean[k]);
      s[k] = 0.0f;
#pragma unroll
      for (int c = 0; c < kCh; ++c) {
        f32x2 a = 0ull;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v[k][c][i] = add2(v[k][c][i], neg);
          if constexpr (!kVec) {
            const float2 e = unpack2(v[k][c][i]);
            v[k][c][i] = pk2(column<kVec>(c, 2 * i, t, tpr) < d ? e.x : 0.0f, column<kVec>(c, 2 * i + 1, t, tpr) < d ? e.y : 0.0f);
          }
          a = fma2(v[k][c][i], v[k][c][i], a);
        }
        s[k] += !kVec || column<kVec>(c, 0, t, tpr) < d ? total_of(a) : 0.0f;
      }
    }
    group.sum(s);
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      if (r0 + k >= rows) break;
      const float rstd = rsqrtf(s[k] * inv_d + eps);
      if (t == 0 && mean_out != nullptr) {
        mean_out[r0 + k] = mean[k];
        rstd_out[r0 + k] = rstd;
      }
      const f32x2 r2 = pk2(rstd, rstd);
#pragma unroll
      for (int c = 0; c < kCh; ++c) {
        f32x2 o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = fma2(mul2(v[k][c][i], r2), scale[c][i], shift[c][i]);
        store_pairs<T, kVec>(y + static_cast<long long>(r0 + k) * d, c, d, t, tpr, o);
      }
    }
  }
}

template <typename T, int kCh, int kRows, bool kVec, bool kParams>
__global__ void __launch_bounds__(32 * kMaxWarps) layer_norm_bwd_kernel(
    const T* __restrict__ x, const void* __restrict__ w, const T* __restrict__ dy, const float* __restrict__ mean_in,
    const float* __restrict__ rstd_in, T* __restrict__ dx, float* __restrict__ partial, int rows, int d, int wpr, int p_fp32) {
  extern __shared__ __align__(16) uint8_t slots[];
  float* sums = reinterpret_cast<float*>(slots);  // at the end: [2][d], where groups of a block share columns
  __shared__ __align__(16) float red[kMaxWarps * 16];
  Group group = group_of(wpr, red);
  const int t = group.t, tpr = group.tpr, groups = blockDim.x / tpr;
  const float inv_d = 1.0f / static_cast<float>(d);
  const int first = (blockIdx.x * groups + group.g) * kRows, step = gridDim.x * groups * kRows;
  using Copies = Ahead<T, kCh, kRows, 2>;
  constexpr int kStages = Copies::kStages;
  const Copies ahead = ahead_of<T, kCh, kRows, 2>(x, dy, rows, d, t, tpr, slots);
  if constexpr (kVec)
    for (int i = 0; i < kStages - 1; ++i) ahead.ask(i, first + i * step);
  f32x2 scale[kCh][4], dw[kCh][4], db[kCh][4];
#pragma unroll
  for (int c = 0; c < kCh; ++c) {
    load_params<kVec>(w, p_fp32, 1.0f, c, d, t, tpr, scale[c]);
#pragma unroll
    for (int i = 0; i < 4; ++i) dw[c][i] = db[c][i] = 0ull;
  }
  int stage = 0;
  float next_mean[kRows], next_rstd[kRows];
  auto ask_stats = [&](int r0) {
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      next_mean[k] = r0 + k < rows ? mean_in[r0 + k] : 0.0f;
      next_rstd[k] = r0 + k < rows ? rstd_in[r0 + k] : 0.0f;
    }
  };
  ask_stats(first);
  for (int r0 = first; r0 < rows; r0 += step) {
    f32x2 xh[kRows][kCh][4], g[kRows][kCh][4];
    float rstd[kRows], s[2 * kRows];
    if constexpr (kVec) asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
    // outside the row dy reads as zero, and with it all that is summed
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      rstd[k] = next_rstd[k];
      const f32x2 neg = pk2(-next_mean[k], -next_mean[k]), r2 = pk2(rstd[k], rstd[k]);
      f32x2 s1 = 0ull, s2 = 0ull;
#pragma unroll
      for (int c = 0; c < kCh; ++c) {
        const long long at = static_cast<long long>(r0 + k) * d;
        const Words<T> vx = kVec ? ahead.get(stage, k, 0, c) : load_words<T, kVec>(x + at, c, d, t, tpr, r0 + k < rows);
        const Words<T> vy = kVec ? ahead.get(stage, k, 1, c) : load_words<T, kVec>(dy + at, c, d, t, tpr, r0 + k < rows);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const f32x2 e = vy.pair(i);
          xh[k][c][i] = mul2(add2(vx.pair(i), neg), r2);
          g[k][c][i] = mul2(e, scale[c][i]);
          if (kParams) {
            dw[c][i] = fma2(e, xh[k][c][i], dw[c][i]);
            db[c][i] = add2(db[c][i], e);
          }
          s1 = add2(s1, g[k][c][i]);
          s2 = fma2(g[k][c][i], xh[k][c][i], s2);
        }
      }
      s[2 * k] = total_of(s1);
      s[2 * k + 1] = total_of(s2);
    }
    ask_stats(r0 + step);
    if constexpr (kVec) {
      ahead.ask((stage + kStages - 1) % kStages, r0 + (kStages - 1) * step);
      stage = (stage + 1) % kStages;
    }
    if (dx == nullptr) continue;
    group.sum(s);
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      if (r0 + k >= rows) break;
      const float m1 = -s[2 * k] * inv_d, m2 = -s[2 * k + 1] * inv_d;
      const f32x2 r2 = pk2(rstd[k], rstd[k]), m1_2 = pk2(m1, m1), m2_2 = pk2(m2, m2);
#pragma unroll
      for (int c = 0; c < kCh; ++c) {
        f32x2 o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = mul2(r2, fma2(xh[k][c][i], m2_2, add2(g[k][c][i], m1_2)));
        store_pairs<T, kVec>(dx + static_cast<long long>(r0 + k) * d, c, d, t, tpr, o);
      }
    }
  }
  if (kParams) {
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();  // nothing is on its way to the slots, which the sums take over
    float* out = partial + static_cast<long long>(blockIdx.x) * 2 * d;
    float* to = groups > 1 ? sums : out;
    for (int turn = 0; turn < groups; ++turn) {  // the groups add their sums in order
      if (group.g == turn) {
#pragma unroll
        for (int c = 0; c < kCh; ++c)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 a = unpack2(dw[c][i]), e = unpack2(db[c][i]);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int col = column<kVec>(c, 2 * i + h, t, tpr);
              if (col < d) {
                to[col] = (turn ? to[col] : 0.0f) + (h ? a.y : a.x);
                to[d + col] = (turn ? to[d + col] : 0.0f) + (h ? e.y : e.x);
              }
            }
          }
      }
      if (groups > 1) __syncthreads();
    }
    if (groups > 1)
      for (int i = threadIdx.x; i < 2 * d; i += blockDim.x) out[i] = sums[i];
  }
}

// dw, db [d] from the blocks' sums [blocks][2][d]: 32 columns a block, its 32 warps take every 32nd partial row.
template <typename P>
__global__ void __launch_bounds__(1024) layer_norm_params_kernel(const float* __restrict__ partial, P* __restrict__ dw,
                                                                 P* __restrict__ db, int blocks, int d) {
  __shared__ float part[32][33];
  wait_for_previous();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int col = blockIdx.x * 32 + lane;  // of 2 d
  float s = 0.0f;
  if (col < 2 * d)
    for (int r = warp; r < blocks; r += 32) s += partial[static_cast<long long>(r) * 2 * d + col];
  part[warp][lane] = s;
  __syncthreads();
  s = warp_sum(part[lane][warp]);  // column `warp` of this block
  const int mine = blockIdx.x * 32 + warp;
  if (lane == 0 && mine < 2 * d) {
    P* out = mine < d ? dw : db;
    if (out != nullptr) store1(out + (mine < d ? mine : mine - d), s);
  }
}

// How rows are spread: the fewest warps whose threads hold a row of up to 4096 columns 8 a thread, or of up to 8192 and
// 12,288 in two and three chunks; as many groups as make 256 to 512 threads a block.
struct Shape {
  int wpr, ch, groups;
};
inline Shape shape_of(int d) {
  const int ch = (d + 256 * kMaxWarps - 1) / (256 * kMaxWarps);
  const int wpr = (d + 256 * ch - 1) / (256 * ch);
  return {wpr, ch, std::max(1, std::min(kMaxGroups, kMaxWarps / wpr))};
}
// Rows a group at a time: fewer where they would not fit registers or the room for copies, or with so many warps a row that
// their sums cost more than the barriers saved.
inline int rows_of(const Shape& s, bool fp32, bool backward) {
  return s.ch > 1 ? 1 : s.wpr > 8 || (fp32 && backward) ? 2 : 4;
}

// What is asked once about a kernel: its room, and how many blocks of a size fit an SM (0: not yet).
struct Fit {
  std::atomic<unsigned long long> asked{0};
  std::atomic<int> per_sm[kMaxWarps + 1] = {};
};

template <typename T, int kCh, int kRows, int kTensors, bool kVec>
inline size_t slots_bytes(int threads) {
  using Copies = Ahead<T, kCh, kRows, kTensors>;
  return kVec ? static_cast<size_t>(Copies::kStages) * Copies::kPieces * threads * 16 : 0;
}
// The blocks of a kernel that walks rows: as many as fit the machine at once, at most one a handful of rows. 0: none fits.
template <typename K>
inline int prepare(K kern, Fit& fit, int threads, size_t smem, long long rows, int rpb) {
  if (!make_room(fit.asked, reinterpret_cast<const void*>(kern), 216 * 1024)) return 0;
  int per_sm = fit.per_sm[threads / 32].load(std::memory_order_relaxed);
  if (per_sm == 0) {
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kern, threads, smem) != cudaSuccess || per_sm < 1) return 0;
    fit.per_sm[threads / 32].store(per_sm, std::memory_order_relaxed);
  }
  return static_cast<int>(std::min<long long>((rows + rpb - 1) / rpb, 148ll * per_sm));
}

template <typename T, int kCh, int kRows, bool kVec>
int fwd(const void* x, const void* w, const void* b, void* y, float* mean, float* rstd, long long rows, int d, float eps,
        Shape s, int p_fp32, cudaStream_t st) {
  const int threads = 32 * s.wpr * s.groups;
  const size_t smem = slots_bytes<T, kCh, kRows, 1, kVec>(threads);
  auto kern = layer_norm_fwd_kernel<T, kCh, kRows, kVec>;
  static Fit fit;
  const int grid = prepare(kern, fit, threads, smem, rows, kRows * s.groups);
  if (grid == 0) return 2;
  kern<<<grid, threads, smem, st>>>(static_cast<const T*>(x), w, b, static_cast<T*>(y), mean, rstd, static_cast<int>(rows), d, eps, s.wpr,
                                    p_fp32);
  return cudaGetLastError() == cudaSuccess ? 0 : 1;
}

template <typename T, int kCh, int kRows, bool kVec, bool kParams>
int bwd(const void* x, const void* w, const void* dy, const float* mean, const float* rstd, void* dx, void* dw, void* db,
        float* partial, int max_blocks, long long rows, int d, Shape s, int p_fp32, cudaStream_t st) {
  const int threads = 32 * s.wpr * s.groups;
  const size_t sums = kParams && s.groups > 1 ? static_cast<size_t>(16 * s.wpr * 256) : 0;  // 2 d floats and more
  const size_t smem = std::max(sums, slots_bytes<T, kCh, kRows, 2, kVec>(threads));
  auto kern = layer_norm_bwd_kernel<T, kCh, kRows, kVec, kParams>;
  static Fit fit;
  int grid = prepare(kern, fit, threads, smem, rows, kRows * s.groups);
  if (grid == 0) return 2;
  if (kParams) grid = std::min(grid, max_blocks);
  kern<<<grid, threads, smem, st>>>(static_cast<const T*>(x), w, static_cast<const T*>(dy), mean, rstd,
                                    static_cast<T*>(dx), partial, static_cast<int>(rows), d, s.wpr, p_fp32);
  if (cudaGetLastError() != cudaSuccess) return 1;
  if (!kParams) return 0;
  const dim3 blocks((2 * d + 31) / 32);
  const cudaError_t e =
      p_fp32 ? launch_after(layer_norm_params_kernel<float>, blocks, dim3(1024), 0, st, partial, static_cast<float*>(dw),
                            static_cast<float*>(db), grid, d)
             : launch_after(layer_norm_params_kernel<__nv_bfloat16>, blocks, dim3(1024), 0, st, partial,
                            static_cast<__nv_bfloat16*>(dw), static_cast<__nv_bfloat16*>(db), grid, d);
  return e == cudaSuccess ? 0 : 1;
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// The kernel for (chunks, rows at a time).
template <typename T, bool kVec, typename... A>
int fwd_rows(int ch, int n, A... a) {
  if (ch == 2) return fwd<T, 2, 1, kVec>(a...);
  if (ch == 3) return fwd<T, 3, 1, kVec>(a...);
  return n == 4 ? fwd<T, 1, 4, kVec>(a...) : fwd<T, 1, 2, kVec>(a...);
}
template <typename T, bool kVec, bool kParams, typename... A>
int bwd_rows(int ch, int n, A... a) {
  if (ch == 2) return bwd<T, 2, 1, kVec, kParams>(a...);
  if (ch == 3) return bwd<T, 3, 1, kVec, kParams>(a...);
  if constexpr (sizeof(T) == 2)
    if (n == 4) return bwd<T, 1, 4, kVec, kParams>(a...);
  return bwd<T, 1, 2, kVec, kParams>(a...);
}
template <typename T, typename... A>
int bwd_all(bool vec, bool params, int ch, int n, A... a) {
  if (params) return vec ? bwd_rows<T, true, true>(ch, n, a...) : bwd_rows<T, false, true>(ch, n, a...);
  return vec ? bwd_rows<T, true, false>(ch, n, a...) : bwd_rows<T, false, false>(ch, n, a...);
}

}  // namespace

// Widest row (columns) and the most blocks whose partial sums the backward writes.
extern "C" int pd_layer_norm_max_columns() { return 256 * kMaxWarps * kMaxChunks; }
extern "C" int pd_layer_norm_partial_rows(long long rows, int d) {
  const Shape s = shape_of(d);
  return static_cast<int>(std::min<long long>((rows + s.groups - 1) / s.groups, 148ll * 4));
}

// x, y [rows, d] contiguous in bf16 or fp32 (x_fp32); w, b [d] or null, of one type (p_fp32). mean, rstd [rows] or null.
extern "C" int pd_layer_norm_fwd(const void* x, const void* w, const void* b, void* y, float* mean, float* rstd,
                                 long long rows, int d, float eps, int x_fp32, int p_fp32, void* stream) {
  if (rows <= 0 || rows >= (1ll << 30) || d <= 0 || d > pd_layer_norm_max_columns() || (mean == nullptr) != (rstd == nullptr)) return 5;
  const Shape s = shape_of(d);
  const bool vec = d % 8 == 0 && aligned16(x) && aligned16(y);
  const int n = rows_of(s, x_fp32, false);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto go = [&](auto t) {
    using T = decltype(t);
    return vec ? fwd_rows<T, true>(s.ch, n, x, w, b, y, mean, rstd, rows, d, eps, s, p_fp32, st)
               : fwd_rows<T, false>(s.ch, n, x, w, b, y, mean, rstd, rows, d, eps, s, p_fp32, st);
  };
  return x_fp32 ? go(float()) : go(__nv_bfloat16());
}

// dx [rows, d] or null; dw, db [d] or null in the parameters' type; partial: pd_layer_norm_partial_rows x 2 x d floats
// (null where neither is asked for).
extern "C" int pd_layer_norm_bwd(const void* x, const void* w, const void* dy, const float* mean, const float* rstd,
                                 void* dx, void* dw, void* db, float* partial, long long rows, int d, int x_fp32,
                                 int p_fp32, void* stream) {
  if (rows <= 0 || rows >= (1ll << 30) || d <= 0 || d > pd_layer_norm_max_columns()) return 5;
  const bool params = dw != nullptr || db != nullptr;
  if (params && partial == nullptr) return 5;
  const Shape s = shape_of(d);
  const bool vec = d % 8 == 0 && aligned16(x) && aligned16(dy) && aligned16(dx);
  const int n = rows_of(s, x_fp32, true), blocks = pd_layer_norm_partial_rows(rows, d);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto go = [&](auto t) {
    return bwd_all<decltype(t)>(vec, params, s.ch, n, x, w, dy, mean, rstd, dx, dw, db, partial, blocks, rows, d, s, p_fp32, st);
  };
  return x_fp32 ? go(float()) : go(__nv_bfloat16());
}
