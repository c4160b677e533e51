// Distillation from a teacher's top logits. A teacher's row is K logits t_k at columns i_k and, as one more event, the
// logarithm of the sum of exponentials of all its other logits (`tail`); p_k and r are its softmax over these K + 1. With
// q the student's softmax over all V columns and R its sum over the columns that are not named,
//   loss = sum_k p_k (log p_k - log q_{i_k}) + r (log r - log R)
//   dloss / dz_j = (q_j - p_j) / T at a named column (p summed where a column is named twice), q_j (1 - r / R) / T elsewhere
// Without a tail r = 0: K = 1 is the cross entropy of one target. A slot with a negative column is unused; a row whose
// teacher has no mass counts zero with a zero gradient.
//
// Rows are held in the shared memory of a cluster of 1 to 8 blocks (each a slice of the row, brought in by bulk copies) and
// read there for the sums and again for the gradient, so a logit crosses HBM once, its gradient once: bound by HBM, beside
// two exponentials a logit (16 lanes a clock). The named columns are taken out of the row first and written as -inf, so
// that R is a sum of what it consists of, not a difference; named and other logits have maxima of their own, so a rest far
// below the named ones keeps its value. The few scalars of a row's loss are formed in 64 bits: it is a small difference of
// logarithms. Clusters walk the rows; a piece of the next row is requested as soon as the gradient pass has read the
// present one out of it.
#include <algorithm>

#include "rows.cuh"

namespace {

using namespace pd;

constexpr int kMaxK = 256;
constexpr int kMaxPieces = 32;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}
__device__ __forceinline__ void store_cluster_f32(uint32_t addr, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}

struct MaxSum {  // a maximum and the sum of exp((z - m) / T)
  float m, s;
};
__device__ __forceinline__ MaxSum merge(const MaxSum& x, const MaxSum& y, float c) {
  MaxSum r;
  r.m = fmaxf(x.m, y.m);
  // equal maxima, -inf on both sides among them, are not subtracted
  r.s = x.s * (x.m == r.m ? 1.0f : ex2((x.m - r.m) * c)) + y.s * (y.m == r.m ? 1.0f : ex2((y.m - r.m) * c));
  return r;
}
__device__ __forceinline__ MaxSum warp_merge(MaxSum t, float c) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    t = merge(t, MaxSum{__shfl_xor_sync(0xffffffffu, t.m, o), __shfl_xor_sync(0xffffffffu, t.s, o)}, c);
  return t;
}

// 16 bytes of shared memory as pairs of fp32.
template <typename T>
__device__ __forceinline__ void pairs_of(const uint4& q, f32x2 (&v)[8 / sizeof(T)]) {
  if constexpr (sizeof(T) == 2) {
    v[0] = unpack_bf16_2(q.x);
    v[1] = unpack_bf16_2(q.y);
    v[2] = unpack_bf16_2(q.z);
    v[3] = unpack_bf16_2(q.w);
  } else {
    v[0] = pk2u(q.x, q.y);
    v[1] = pk2u(q.z, q.w);
  }
}

struct Call {
  const void* z;
  long long rows, ld;
  int V;
  const void* indices;
  int wide;  // indices are int64, else int32
  const void* values;
  int values_fp32, K;
  const float* tail;  // or null
  double inv_t;
  float* loss;       // [rows] or null
  void* dz;          // [rows, V], rows ldo apart, each at z's row's address modulo 16; or null
  long long ldo;
  const float* scale;  // [rows]: the gradient's factor; or null
  int* status;
  int* refused;
};

template <typename T>
__global__ void __launch_bounds__(512) top_kl_kernel(const Call call, int slice, int cs) {
  constexpr int kE = 16 / sizeof(T), kP = kE / 2;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(8) unsigned long long bars[kMaxPieces];
  __shared__ MaxSum red[16], xch[2][8];
  __shared__ float named[2][kMaxK];  // student's logits at the columns, in the slots that speak for them
  __shared__ int column[kMaxK], owner[kMaxK];
  __shared__ float prob[kMaxK], prob_of_column[kMaxK];
  __shared__ float teacher[3];  // r, sum of p, 0 or 1: the row counts
  __shared__ double teacher_log[3];  // maximum (over T), log of the sum, log r
  __shared__ int abort_flag;
  const int tid = threadIdx.x, nt = blockDim.x, warp = tid >> 5, lane = tid & 31, warps = nt >> 5;
  const int rank = cs > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int V = call.V, K = call.K, g0 = rank * slice, pieces = (slice + nt - 1) / nt;
  const float c = static_cast<float>(call.inv_t * 1.4426950408889634);
  const T* z = static_cast<const T*>(call.z);
  T* buf = reinterpret_cast<T*>(smem);
  const uint32_t bar0 = smem_u32(bars);
  if (tid == 0) {
    for (int i = 0; i < pieces; ++i) mbar_init(bar0 + 8 * i, 1);
    abort_flag = 0;
    mbar_fence_init();
  }
  __syncthreads();
  auto shift_of = [&](long long row) {
    return static_cast<int>((reinterpret_cast<uintptr_t>(z + row * call.ld) & 15) / sizeof(T));
  };
  // Groups of 16 bytes at 16-byte addresses: those that lie in the row whole come by bulk copy, its ragged ends by loads.
  auto request = [&](long long row, int piece) {  // one thread; nothing new once a wait has run out
    if (*static_cast<volatile int*>(&abort_flag)) return;
    const int shift = shift_of(row);
    const int first = max(g0 + piece * nt, shift > 0 ? 1 : 0);
    const int stop = min(g0 + min((piece + 1) * nt, slice), (shift + V) / kE);
    const uint32_t bytes = stop > first ? 16u * (stop - first) : 0u;
    mbar_expect_tx(bar0 + 8 * piece, bytes);
    if (bytes > 0)
      bulk_load(smem_u32(smem + 16ll * (first - g0)), z + row * call.ld - shift + static_cast<long long>(first) * kE, bytes,
                bar0 + 8 * piece);
  };
  const long long first_row = blockIdx.x / cs, step = gridDim.x / cs;
  if (tid == 0 && first_row < call.rows)
    for (int i = 0; i < pieces; ++i) request(first_row, i);
  if (cs > 1) cluster_sync_all();  // every block of the cluster runs before another one stores to its shared memory
  int turn = 0;
  for (long long row = first_row; row < call.rows; row += step, ++turn) {
    const int shift = shift_of(row), half = turn & 1;
    const int groups = min(slice, max(0, (shift + V + kE - 1) / kE - g0));
    const T* zr = z + row * call.ld;
    // the ragged ends: thread j < kE an element of the row's first group, the next kE one of its last
    int end_at = -1;
    T end_value{};
    if (tid < 2 * kE) {
      const int g = tid < kE ? 0 : (shift + V) / kE, at = g * kE + tid % kE, col = at - shift;
      const bool ragged = tid < kE ? shift > 0 : (shift + V) % kE != 0;
      if (ragged && g >= g0 && g < g0 + groups) {
        end_at = at - g0 * kE;
        if (col >= 0 && col < V)
          end_value = zr[col];
        else
          store1(&end_value, -INFINITY);
      }
    }
    // the teacher's distribution, while the row is on its way
    if (tid < K) {
      long long i = call.wide ? static_cast<const long long*>(call.indices)[row * K + tid]
                              : static_cast<const int*>(call.indices)[row * K + tid];
      const float t = call.values_fp32 ? static_cast<const float*>(call.values)[row * K + tid]
                                       : as_float(static_cast<const __nv_bfloat16*>(call.values)[row * K + tid]);
      if (i >= V) {
        atomicCAS(call.status, 0, kBadColumn);
        *static_cast<volatile int*>(call.refused) = 1;
        i = -1;
      }
      column[tid] = i < 0 ? -1 : static_cast<int>(i);
      prob[tid] = i < 0 ? -INFINITY : t;
    }
    __syncthreads();
    if (warp == 0) {
      const float tl = call.tail != nullptr ? call.tail[row] : -INFINITY;  // already over T
      float m = -INFINITY;
      bool nan = tl != tl;
      for (int k = lane; k < K; k += 32) {
        m = fmaxf(m, prob[k]);
        nan |= prob[k] != prob[k];
      }
      nan = __any_sync(0xffffffffu, nan);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      const double top = fmax(static_cast<double>(m) * call.inv_t, static_cast<double>(tl));
      float s = 0.0f;
      for (int k = lane; k < K; k += 32) s += expf(static_cast<float>(prob[k] * call.inv_t - top));
      s = warp_sum(s);
      const float rest = expf(static_cast<float>(tl - top)), total = s + rest;
      if (lane == 0) {
        const bool live = nan || top > -INFINITY;
        teacher[0] = live ? rest / total : 0.0f;
        teacher[1] = live ? s / total : 0.0f;
        teacher[2] = live ? 1.0f : 0.0f;
        teacher_log[0] = top;
        teacher_log[1] = log(static_cast<double>(total));
        teacher_log[2] = tl - top - teacher_log[1];
      }
    }
    __syncthreads();
    // Every slot learns which slot speaks for its column (the first that names it) and the column's whole probability.
    const bool live = teacher[2] != 0.0f;
    if (tid < K) {
      const double top = teacher_log[0], log_total = teacher_log[1];
      const int mine = column[tid];
      int speaker = tid;
      float p = 0.0f;
      if (mine >= 0 && live)
        for (int k = 0; k < K; ++k)
          if (column[k] == mine) {
            speaker = min(speaker, k);
            p += expf(static_cast<float>(prob[k] * call.inv_t - top - log_total));
          }
      owner[tid] = speaker;
      prob_of_column[tid] = p;
    }
    for (int i = 0; i < pieces; ++i)
      if (!mbar_wait(bar0 + 8 * i, turn & 1, &abort_flag) && call.status != nullptr)
        atomicCAS(call.status, 0, kTimeoutProducer);
    if (end_at >= 0) buf[end_at] = end_value;
    __syncthreads();
    // Named columns leave the row: their logits go to every block of the cluster.
    const int at = tid < K && column[tid] >= 0 && owner[tid] == tid ? shift + column[tid] - g0 * kE : -1;
    const bool here = at >= 0 && at < groups * kE;
    if (here) {
      const float v = as_float(buf[at]);
      const uint32_t local = smem_u32(&named[half][tid]);
      if (cs > 1)
        for (int b = 0; b < cs; ++b) store_cluster_f32(mapa_shared(local, b), v);
      else
        named[half][tid] = v;
      store1(buf + at, -INFINITY);
    }
    fence_proxy_async_smem();  // before the next row's bulk copies write where this row's ends and marks are
    __syncthreads();
    float m = -INFINITY;
    for (int g = tid; g < groups; g += nt) {
      f32x2 v[kP];
      pairs_of<T>(*reinterpret_cast<const uint4*>(smem + 16 * g), v);
#pragma unroll
      for (int j = 0; j < kP; ++j) {
        const float2 x = unpack2(v[j]);
        m = fmaxf(m, fmaxf(x.x, x.y));
      }
    }
    MaxSum t{m, 0.0f};
    if (m > -INFINITY) {
      const f32x2 neg = pk2(-m, -m), c2 = pk2(c, c);
      f32x2 s = 0ull;
      for (int g = tid; g < groups; g += nt) {
        f32x2 v[kP];
        pairs_of<T>(*reinterpret_cast<const uint4*>(smem + 16 * g), v);
#pragma unroll
        for (int j = 0; j < kP; ++j) {
          const float2 x = unpack2(mul2(add2(v[j], neg), c2));
          s = add2(s, pk2(ex2(x.x), ex2(x.y)));
        }
      }
      const float2 s2 = unpack2(s);
      t.s = s2.x + s2.y;
    }
    t = warp_merge(t, c);
    if (lane == 0) red[warp] = t;
    __syncthreads();
    if (warp == 0) {
      t = lane < warps ? red[lane] : MaxSum{-INFINITY, 0.0f};
      t = warp_merge(t, c);
      if (lane < cs) {
        const uint32_t local = smem_u32(&xch[half][rank]);
        const uint32_t to = cs > 1 ? mapa_shared(local, lane) : local;
        store_cluster_f32(to, t.m);
        store_cluster_f32(to + 4, t.s);
      }
    }
    if (cs > 1)
      cluster_sync_all();
    else
      __syncthreads();
    MaxSum rest = xch[half][0];
    for (int b = 1; b < cs; ++b) rest = merge(rest, xch[half][b], c);
    MaxSum top{-INFINITY, 0.0f};  // of the named columns; every warp forms it for itself
    for (int k = lane; k < K; k += 32)
      if (column[k] >= 0 && owner[k] == k) top = merge(top, MaxSum{named[half][k], 1.0f}, c);
    top = warp_merge(top, c);
    const MaxSum all = merge(rest, top, c);
    const float r = teacher[0], p_named = teacher[1];
    if (warp == 0 && rank == 0 && call.loss != nullptr) {
      const double log_all = log(static_cast<double>(all.s)), inv_t = call.inv_t;
      double sum = 0.0;
      for (int k = lane; k < K; k += 32) {
        if (column[k] < 0) continue;
        const double log_p = prob[k] * inv_t - teacher_log[0] - teacher_log[1];
        const double log_q = (static_cast<double>(named[half][owner[k]]) - all.m) * inv_t - log_all;
        const float p = expf(static_cast<float>(log_p));
        if (!(p == 0.0f)) sum += p * (log_p - log_q);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (lane == 0) {
        if (!(r == 0.0f)) {
          const double log_rest = (static_cast<double>(rest.m) - all.m) * inv_t + log(static_cast<double>(rest.s)) - log_all;
          sum += r * (teacher_log[2] - log_rest);
        }
        call.loss[row] = live ? static_cast<float>(sum) : 0.0f;
      }
    }
    const bool more = row + step < call.rows;
    if (call.dz != nullptr) {
      const float up = (call.scale != nullptr ? call.scale[row] : 1.0f) * static_cast<float>(call.inv_t);
      // q of the named columns and of the rest; the difference R - r from whichever side is small
      const float q_top = top.s * (top.m == all.m ? 1.0f : ex2((top.m - all.m) * c)) / all.s;
      const float q_rest = rest.s * (rest.m == all.m ? 1.0f : ex2((rest.m - all.m) * c)) / all.s;
      const float gap = r > 0.5f ? p_named - q_top : q_rest - r;
      const float f = live && rest.s > 0.0f ? gap / rest.s * up : (rest.s == rest.s ? 0.0f : rest.s);
      const float ref = rest.m > -INFINITY ? rest.m : 0.0f;
      const f32x2 neg = pk2(-ref, -ref), c2 = pk2(c, c), f2 = pk2(f, f);
      T* out = static_cast<T*>(call.dz) + row * call.ldo;
      for (int i = 0; i < pieces; ++i) {
        const int g = i * nt + tid;
        if (g < groups) {
          f32x2 v[kP];
          pairs_of<T>(*reinterpret_cast<const uint4*>(smem + 16 * g), v);
#pragma unroll
          for (int j = 0; j < kP; ++j) {
            const float2 x = unpack2(mul2(add2(v[j], neg), c2));
            v[j] = live ? mul2(pk2(ex2(x.x), ex2(x.y)), f2) : 0ull;
          }
          const int col = (g0 + g) * kE - shift;
          if (col >= 0 && col + kE <= V) {
            uint4 q;
            if constexpr (sizeof(T) == 2) {
              q = make_uint4(pack_bf16_2(v[0]), pack_bf16_2(v[1]), pack_bf16_2(v[2]), pack_bf16_2(v[3]));
            } else {
              const float2 a = unpack2(v[0]), b = unpack2(v[1]);
              q = make_uint4(__float_as_uint(a.x), __float_as_uint(a.y), __float_as_uint(b.x), __float_as_uint(b.y));
            }
            *reinterpret_cast<uint4*>(out + col) = q;
          } else {
#pragma unroll
            for (int j = 0; j < kP; ++j) {
              const float2 a = unpack2(v[j]);
              if (col + 2 * j >= 0 && col + 2 * j < V) store1(out + col + 2 * j, a.x);
              if (col + 2 * j + 1 >= 0 && col + 2 * j + 1 < V) store1(out + col + 2 * j + 1, a.y);
            }
          }
        }
        __syncthreads();  // the piece has been read; behind the last one, the row's stores are in order before the named
        if (more && tid == 0) request(row + step, i);
      }
      if (here) {
        const float q = ex2((named[half][tid] - all.m) * c) / all.s;
        store1(out + column[tid], live ? (q - prob_of_column[tid]) * up : 0.0f);
      }
      __syncthreads();  // before the next row's slots overwrite this one's
    } else {
      __syncthreads();
      if (more && tid == 0)
        for (int i = 0; i < pieces; ++i) request(row + step, i);
    }
  }
}

// Slices (16-byte groups a block) and the cluster that holds a row of V columns; 0 where none does.
struct Plan {
  int cs, slice;
};
template <typename T>
Plan plan_for(long long V) {
  // the smallest cluster that leaves room for two blocks an SM; past that, up to one block an SM
  constexpr long long kHalfSm = 104 * 1024, kWholeSm = 216 * 1024, kE = 16 / sizeof(T);
  const long long groups = (V + 2 * kE - 2) / kE;  // wherever a row starts
  int cs = 1;
  while (cs < 8 && (groups + cs - 1) / cs * 16 > kHalfSm) cs *= 2;
  const long long slice = (groups + cs - 1) / cs;
  return slice * 16 > kWholeSm ? Plan{0, 0} : Plan{cs, static_cast<int>(slice)};
}

template <typename T>
int launch(const Call& call, cudaStream_t st) {
  const Plan plan = plan_for<T>(call.V);
  if (plan.cs == 0) return 5;
  const int smem = plan.slice * 16;
  // short rows: fewer threads, so that every thread has a group and more rows share an SM; a slot needs a thread
  const int nt = plan.slice >= 1024 ? 512 : 256;
  auto kern = top_kl_kernel<T>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 216 * 1024) != cudaSuccess) return 2;
  const int per_sm = std::max(1, std::min(1024 / nt, 227 * 1024 / (smem + 8 * 1024)));
  const long long clusters = std::min<long long>(call.rows, std::max(1, 148 * per_sm / plan.cs));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(clusters * plan.cs));
  cfg.blockDim = dim3(nt);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = plan.cs;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, call, plan.slice, plan.cs);
  return e == cudaSuccess && cudaGetLastError() == cudaSuccess ? 0 : 1;
}

}  // namespace

// Widest row that a cluster holds.
extern "C" long long pd_top_kl_max_columns(int z_fp32) { return 8ll * 216 * 1024 / (z_fp32 ? 4 : 2) - 16; }

extern "C" int pd_top_kl(const void* z, long long rows, int V, long long ld, const void* indices, int wide,
                         const void* values, int values_fp32, int K, const float* tail, double inv_t, float* loss, void* dz,
                         long long ldo, const float* scale, int z_fp32, int* status, int* refused, void* stream) {
  if (rows <= 0 || V <= 0 || K <= 0 || K > kMaxK || !(inv_t > 0.0)) return 5;
  const Call call{z, rows, ld, V, indices, wide, values, values_fp32, K, tail, inv_t, loss, dz, ldo, scale, status, refused};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return z_fp32 ? launch<float>(call, st) : launch<__nv_bfloat16>(call, st);
}
