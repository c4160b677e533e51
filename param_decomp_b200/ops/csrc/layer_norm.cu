// Layer norm over rows of `d` columns:
//   mean = sum x / d, var = sum (x - mean)^2 / d, xh = (x - mean) rstd, rstd = 1 / sqrt(var + eps), y = xh w + b
//   dx = rstd (g - mean(g) - xh mean(g xh)) with g = dy w;  dw = sum over rows of dy xh;  db = sum over rows of dy
// A row is held in the registers of one warp (up to 768 columns) or of one block, so x (and dy) cross HBM once and the
// variance is summed around the mean that was just formed, not from sums of squares. All sums are in fp32; what is stored
// is rounded once. Bound by HBM: 2 (forward) and 3 (backward) passes of the row data.
// The weight gradients: every thread keeps the sums of its own columns over all rows that its block walks; blocks write
// those to scratch and a second kernel adds them in a fixed order, so a result does not change from run to run.
#include <algorithm>

#include "rows.cuh"

namespace {

using namespace pd;

constexpr int kMaxWarps = 16;  // of a row
constexpr int kMaxChunks = 3;  // of 8 columns a thread: the backward holds 4 x 8 values a chunk
constexpr int kWarpsPerBlock = 8;  // where a warp takes whole rows

// Which column element j of chunk c is, for thread t of `tpr` that share a row. Rows of 16-byte pieces: eight
// neighbours a thread; any other row: threads side by side, one element each.
template <bool kVec>
__device__ __forceinline__ int column(int c, int j, int t, int tpr) {
  return kVec ? (c * tpr + t) * 8 + j : (c * 8 + j) * tpr + t;
}

// Eight neighbouring parameters, or one, in either type (a branch every thread takes alike).
__device__ __forceinline__ void params8(const void* p, int fp32, int col, float (&v)[8]) {
  if (fp32)
    unpack8(load8(static_cast<const float*>(p) + col), v);
  else
    unpack8(load8(static_cast<const __nv_bfloat16*>(p) + col), v);
}
__device__ __forceinline__ float param1(const void* p, int fp32, int col) {
  return fp32 ? static_cast<const float*>(p)[col] : as_float(static_cast<const __nv_bfloat16*>(p)[col]);
}

template <typename T, int kCh, bool kVec>
__device__ __forceinline__ void load_row(const T* __restrict__ row, int d, int t, int tpr, float (&v)[kCh][8]) {
  if (kVec) {
    Raw8<T> raw[kCh];
#pragma unroll
    for (int c = 0; c < kCh; ++c)
      if (column<kVec>(c, 0, t, tpr) < d) raw[c] = load8(row + column<kVec>(c, 0, t, tpr));
#pragma unroll
    for (int c = 0; c < kCh; ++c) {
      if (column<kVec>(c, 0, t, tpr) < d) {
        unpack8(raw[c], v[c]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[c][j] = 0.0f;
      }
    }
  } else {
#pragma unroll
    for (int c = 0; c < kCh; ++c)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int col = column<kVec>(c, j, t, tpr);
        v[c][j] = col < d ? as_float(row[col]) : 0.0f;
      }
  }
}

template <typename T, int kCh, bool kVec>
__device__ __forceinline__ void store_row(T* __restrict__ row, int d, int t, int tpr, const float (&v)[kCh][8]) {
#pragma unroll
  for (int c = 0; c < kCh; ++c) {
    if (kVec) {
      if (column<kVec>(c, 0, t, tpr) < d) store8(row + column<kVec>(c, 0, t, tpr), v[c]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int col = column<kVec>(c, j, t, tpr);
        if (col < d) store1(row + col, v[c][j]);
      }
    }
  }
}

// Sums over the threads of a row; `red` is used in turn (two halves), so one barrier a sum is enough.
__device__ __forceinline__ float2 row_sum(float2 s, int wpr, float2 (*red)[32], int& turn) {
  s.x = warp_sum(s.x);
  s.y = warp_sum(s.y);
  if (wpr > 1) {
    float2* r = red[turn & 1];
    ++turn;
    if ((threadIdx.x & 31) == 0) r[threadIdx.x >> 5] = s;
    __syncthreads();
    s = r[0];
    for (int w = 1; w < wpr; ++w) {
      s.x += r[w].x;
      s.y += r[w].y;
    }
  }
  return s;
}

template <typename T, int kCh, bool kVec>
__global__ void __launch_bounds__(32 * kMaxWarps) layer_norm_fwd_kernel(const T* __restrict__ x, const void* __restrict__ w,
                                                              const void* __restrict__ b, T* __restrict__ y,
                                                              float* __restrict__ mean_out, float* __restrict__ rstd_out,
                                                              long long rows, int d, float eps, int wpr, int p_fp32) {
  __shared__ float2 red[2][32];
  const int tpr = 32 * wpr, rpb = blockDim.x / tpr, t = threadIdx.x % tpr;
  const float inv_d = 1.0f / static_cast<float>(d);
  int turn = 0;
  for (long long r = static_cast<long long>(blockIdx.x) * rpb + threadIdx.x / tpr; r < rows;
       r += static_cast<long long>(gridDim.x) * rpb) {
    float v[kCh][8];
    load_row<T, kCh, kVec>(x + r * d, d, t, tpr, v);
    float2 s = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int c = 0; c < kCh; ++c)
#pragma unroll
      for (int j = 0; j < 8; ++j) s.x += v[c][j];
    const float mean = row_sum(s, wpr, red, turn).x * inv_d;
    s = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int c = 0; c < kCh; ++c)
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (column<kVec>(c, j, t, tpr) < d) {
          v[c][j] -= mean;
          s.x += v[c][j] * v[c][j];
        }
    const float rstd = rsqrtf(row_sum(s, wpr, red, turn).x * inv_d + eps);
    if (t == 0 && mean_out != nullptr) {
      mean_out[r] = mean;
      rstd_out[r] = rstd;
    }
#pragma unroll
    for (int c = 0; c < kCh; ++c) {
      float wv[8], bv[8];
      // the parameters are read again for every row: they stay in L1
      if (kVec) {
        const int col = column<kVec>(c, 0, t, tpr);
        if (col < d) {
          if (w != nullptr) params8(w, p_fp32, col, wv);
          if (b != nullptr) params8(b, p_fp32, col, bv);
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int col = column<kVec>(c, j, t, tpr);
        if (col >= d) continue;
        const float scale = w == nullptr ? 1.0f : kVec ? wv[j] : param1(w, p_fp32, col);
        const float shift = b == nullptr ? 0.0f : kVec ? bv[j] : param1(b, p_fp32, col);
        v[c][j] = v[c][j] * rstd * scale + shift;
      }
    }
    store_row<T, kCh, kVec>(y + r * d, d, t, tpr, v);
  }
}

template <typename T, int kCh, bool kVec, bool kParams>
__global__ void __launch_bounds__(32 * kMaxWarps) layer_norm_bwd_kernel(
    const T* __restrict__ x, const void* __restrict__ w, const T* __restrict__ dy, const float* __restrict__ mean_in,
    const float* __restrict__ rstd_in, T* __restrict__ dx, float* __restrict__ partial, long long rows, int d, int wpr,
    int p_fp32) {
  extern __shared__ float sums[];  // [2][d], where warps of a block share columns
  __shared__ float2 red[2][32];
  const int tpr = 32 * wpr, rpb = blockDim.x / tpr, t = threadIdx.x % tpr;
  const float inv_d = 1.0f / static_cast<float>(d);
  float dw[kCh][8], db[kCh][8];
#pragma unroll
  for (int c = 0; c < kCh; ++c)
#pragma unroll
    for (int j = 0; j < 8; ++j) dw[c][j] = db[c][j] = 0.0f;
  int turn = 0;
  for (long long r = static_cast<long long>(blockIdx.x) * rpb + threadIdx.x / tpr; r < rows;
       r += static_cast<long long>(gridDim.x) * rpb) {
    float xh[kCh][8], g[kCh][8];
    load_row<T, kCh, kVec>(x + r * d, d, t, tpr, xh);
    load_row<T, kCh, kVec>(dy + r * d, d, t, tpr, g);
    const float mean = mean_in[r], rstd = rstd_in[r];
    float2 s = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int c = 0; c < kCh; ++c) {
      float wv[8];
      if (kVec && w != nullptr && column<kVec>(c, 0, t, tpr) < d) params8(w, p_fp32, column<kVec>(c, 0, t, tpr), wv);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int col = column<kVec>(c, j, t, tpr);
        if (col >= d) continue;
        xh[c][j] = (xh[c][j] - mean) * rstd;
        if (kParams) {
          dw[c][j] += g[c][j] * xh[c][j];
          db[c][j] += g[c][j];
        }
        g[c][j] *= w == nullptr ? 1.0f : kVec ? wv[j] : param1(w, p_fp32, col);
        s.x += g[c][j];
        s.y += g[c][j] * xh[c][j];
      }
    }
    s = row_sum(s, wpr, red, turn);
    if (dx != nullptr) {
      const float m1 = s.x * inv_d, m2 = s.y * inv_d;
#pragma unroll
      for (int c = 0; c < kCh; ++c)
#pragma unroll
        for (int j = 0; j < 8; ++j) g[c][j] = rstd * (g[c][j] - m1 - xh[c][j] * m2);
      store_row<T, kCh, kVec>(dx + r * d, d, t, tpr, g);
    }
  }
  if (kParams) {
    float* out = partial + static_cast<long long>(blockIdx.x) * 2 * d;
    if (wpr > 1) {
#pragma unroll
      for (int c = 0; c < kCh; ++c)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int col = column<kVec>(c, j, t, tpr);
          if (col < d) {
            out[col] = dw[c][j];
            out[d + col] = db[c][j];
          }
        }
    } else {
      for (int turn_of = 0; turn_of < rpb; ++turn_of) {  // the warps add their sums in order
        if (static_cast<int>(threadIdx.x >> 5) == turn_of) {
#pragma unroll
          for (int c = 0; c < kCh; ++c)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const int col = column<kVec>(c, j, t, tpr);
              if (col < d) {
                sums[col] = (turn_of ? sums[col] : 0.0f) + dw[c][j];
                sums[d + col] = (turn_of ? sums[d + col] : 0.0f) + db[c][j];
              }
            }
        }
        __syncthreads();
      }
      for (int i = threadIdx.x; i < 2 * d; i += blockDim.x) out[i] = sums[i];
    }
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

struct Shape {
  int wpr, ch;
};
// A warp a row up to 768 columns; then the fewest warps whose threads hold the row in two chunks, or three at the most warps.
inline Shape shape_of(int d) {
  int wpr = 1;
  if (d > 256 * kMaxChunks)
    while (wpr < kMaxWarps && d > 512 * wpr) wpr *= 2;
  return {wpr, (d + 256 * wpr - 1) / (256 * wpr)};
}

// Blocks that fit the machine at once, at most one a row (or a row group). What fits an SM is asked once a kernel and
// block size (`fit`, zero at first; the answer is the same whoever writes it).
template <typename K>
inline int grid_for(K kern, int* fit, int threads, size_t smem, long long rows, int rpb) {
  int& per_sm = fit[threads / 32];
  if (per_sm == 0 && (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kern, threads, smem) != cudaSuccess || per_sm < 1)) {
    per_sm = 0;
    return 0;
  }
  return static_cast<int>(std::min<long long>((rows + rpb - 1) / rpb, 148ll * per_sm));
}

template <typename T, int kCh, bool kVec>
int fwd(const void* x, const void* w, const void* b, void* y, float* mean, float* rstd, long long rows, int d, float eps,
        int wpr, int p_fp32, cudaStream_t st) {
  const int threads = wpr == 1 ? 32 * kWarpsPerBlock : 32 * wpr;
  auto kern = layer_norm_fwd_kernel<T, kCh, kVec>;
  static int fit[kMaxWarps + 1];
  const int grid = grid_for(kern, fit, threads, 0, rows, threads / (32 * wpr));
  if (grid == 0) return 2;
  kern<<<grid, threads, 0, st>>>(static_cast<const T*>(x), w, b, static_cast<T*>(y), mean, rstd, rows, d, eps, wpr, p_fp32);
  return cudaGetLastError() == cudaSuccess ? 0 : 1;
}

template <typename T, int kCh, bool kVec, bool kParams>
int bwd(const void* x, const void* w, const void* dy, const float* mean, const float* rstd, void* dx, void* dw, void* db,
        float* partial, int max_blocks, long long rows, int d, int wpr, int p_fp32, cudaStream_t st) {
  const int threads = wpr == 1 ? 32 * kWarpsPerBlock : 32 * wpr;
  const size_t smem = kParams && wpr == 1 ? static_cast<size_t>(2 * d) * sizeof(float) : 0;
  auto kern = layer_norm_bwd_kernel<T, kCh, kVec, kParams>;
  static int fit[kMaxWarps + 1];
  int grid = grid_for(kern, fit, threads, smem, rows, threads / (32 * wpr));
  if (grid == 0) return 2;
  grid = std::min(grid, max_blocks);
  kern<<<grid, threads, smem, st>>>(static_cast<const T*>(x), w, static_cast<const T*>(dy), mean, rstd,
                                    static_cast<T*>(dx), partial, rows, d, wpr, p_fp32);
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

template <typename T, bool kVec, typename... A>
int fwd_ch(int ch, A... a) {
  return ch == 1 ? fwd<T, 1, kVec>(a...) : ch == 2 ? fwd<T, 2, kVec>(a...) : fwd<T, 3, kVec>(a...);
}
template <typename T, bool kVec, bool kParams, typename... A>
int bwd_ch(int ch, A... a) {
  return ch == 1   ? bwd<T, 1, kVec, kParams>(a...)
         : ch == 2 ? bwd<T, 2, kVec, kParams>(a...)
                   : bwd<T, 3, kVec, kParams>(a...);
}
template <typename T, typename... A>
int bwd_all(bool vec, bool params, int ch, A... a) {
  if (params) return vec ? bwd_ch<T, true, true>(ch, a...) : bwd_ch<T, false, true>(ch, a...);
  return vec ? bwd_ch<T, true, false>(ch, a...) : bwd_ch<T, false, false>(ch, a...);
}

}  // namespace

// Widest row (columns) and the most blocks whose partial sums the backward writes.
extern "C" int pd_layer_norm_max_columns() { return 256 * kMaxWarps * kMaxChunks; }
extern "C" int pd_layer_norm_partial_rows(long long rows, int d) {
  const Shape s = shape_of(d);
  const int rpb = s.wpr == 1 ? kWarpsPerBlock : 1;
  return static_cast<int>(std::min<long long>((rows + rpb - 1) / rpb, 148ll * std::max(1, 16 / std::max(8, s.wpr))));
}

// x, y [rows, d] contiguous in bf16 or fp32 (x_fp32); w, b [d] or null, of one type (p_fp32). mean, rstd [rows] or null.
extern "C" int pd_layer_norm_fwd(const void* x, const void* w, const void* b, void* y, float* mean, float* rstd,
                                 long long rows, int d, float eps, int x_fp32, int p_fp32, void* stream) {
  if (rows <= 0 || d <= 0 || d > pd_layer_norm_max_columns() || (mean == nullptr) != (rstd == nullptr)) return 5;
  const Shape s = shape_of(d);
  const bool vec = d % 8 == 0 && aligned16(x) && aligned16(y) && aligned16(w) && aligned16(b);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto go = [&](auto t) {
    using T = decltype(t);
    return vec ? fwd_ch<T, true>(s.ch, x, w, b, y, mean, rstd, rows, d, eps, s.wpr, p_fp32, st)
               : fwd_ch<T, false>(s.ch, x, w, b, y, mean, rstd, rows, d, eps, s.wpr, p_fp32, st);
  };
  return x_fp32 ? go(float()) : go(__nv_bfloat16());
}

// dx [rows, d] or null; dw, db [d] or null in the parameters' type; partial: pd_layer_norm_partial_rows x 2 x d floats
// (null where neither is asked for).
extern "C" int pd_layer_norm_bwd(const void* x, const void* w, const void* dy, const float* mean, const float* rstd,
                                 void* dx, void* dw, void* db, float* partial, long long rows, int d, int x_fp32,
                                 int p_fp32, void* stream) {
  if (rows <= 0 || d <= 0 || d > pd_layer_norm_max_columns()) return 5;
  const bool params = dw != nullptr || db != nullptr;
  if (params && partial == nullptr) return 5;
  const Shape s = shape_of(d);
  const bool vec = d % 8 == 0 && aligned16(x) && aligned16(dy) && aligned16(dx) && aligned16(w);
  const int blocks = pd_layer_norm_partial_rows(rows, d);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto go = [&](auto t) {
    return bwd_all<decltype(t)>(vec, params, s.ch, x, w, dy, mean, rstd, dx, dw, db, partial, blocks, rows, d, s.wpr,
                                p_fp32, st);
  };
  return x_fp32 ? go(float()) : go(__nv_bfloat16());
}
