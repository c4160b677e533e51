// Rows of logits held in the shared memory of a cluster: block b of a cluster holds the 16-byte groups
// [b slice, (b + 1) slice) of a row, and every warp of the block owns `per` neighbouring groups of them, with a bulk copy
// and a barrier of its own. A warp that has read its part for the last time asks for its part of the next row by itself,
// without waiting for the others.
// Groups lie at 16-byte addresses wherever a row starts: group g holds columns g kE - shift + j. Those that a row fills
// whole come by bulk copy; the up to two at its ragged ends are fetched element by element (`edge_*`).
#pragma once

#include <algorithm>

#include "rows.cuh"

namespace pd {

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
// A barrier of the block's first `threads` threads, whose warps may come to it in parts (the form without .aligned).
__device__ __forceinline__ void sync_first(int threads) {
  __syncwarp();
  asm volatile("barrier.sync 1, %0;" ::"r"(threads) : "memory");
}

// Bounded waits that count cycles (4e9: about two seconds): reading the global timer takes about a microsecond, which a
// wait that is over in less would pay each time. With kCluster, what other blocks stored before they arrived is seen.
// Lanes that wait may keep a lane of their warp that has not arrived yet from running: `if (lane == 0) arrive` is followed
// by __syncwarp().
template <bool kCluster>
__device__ __forceinline__ bool short_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  long long t0 = 0;
  for (uint32_t spins = 0;; ++spins) {
    uint32_t done;
    if constexpr (kCluster)
      asm volatile(
          "{\n\t.reg .pred p;\n\t"
          "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
          "selp.b32 %0, 1, 0, p;\n\t}\n"
          : "=r"(done)
          : "r"(bar), "r"(parity)
          : "memory");
    else
      done = mbar_try_wait(bar, parity);
    if (done) return true;
    if ((spins & 63) == 0) {
      const long long now = clock64();
      if (spins == 0) t0 = now;
      if (*abort_flag) return false;
      if (now - t0 > 4000000000ll) {
        *abort_flag = 1;
        return false;
      }
    }
  }
}

// 16 bytes as pairs of fp32.
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
__device__ __forceinline__ uint32_t max_bf16x2(uint32_t a, uint32_t b) {
  const __nv_bfloat162 r = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
// The largest of a thread's groups; NaN is passed over.
template <typename T>
struct GroupMax {
  uint32_t w = 0xFF80FF80u;  // bf16: a pair of maxima
  float m = -INFINITY;       // fp32
  __device__ __forceinline__ void add(const uint4& q) {
    if constexpr (sizeof(T) == 2)
      w = max_bf16x2(w, max_bf16x2(max_bf16x2(q.x, q.y), max_bf16x2(q.z, q.w)));
    else
      m = fmaxf(m, fmaxf(fmaxf(__uint_as_float(q.x), __uint_as_float(q.y)), fmaxf(__uint_as_float(q.z), __uint_as_float(q.w))));
  }
  __device__ __forceinline__ float value() const {
    if constexpr (sizeof(T) == 2)
      return fmaxf(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
    else
      return m;
  }
};

template <typename T>
struct RowSlice {
  static constexpr int kE = 16 / sizeof(T);
  const T* z;
  long long ld;
  int V, g0, slice, per;

  __device__ __forceinline__ const T* row(long long r) const { return z + r * ld; }
  __device__ __forceinline__ int shift(long long r) const {
    return static_cast<int>((reinterpret_cast<uintptr_t>(row(r)) & 15) / sizeof(T));
  }
  // Groups of this block that hold columns of the row.
  __device__ __forceinline__ int groups(int shift) const { return min(slice, max(0, (shift + V + kE - 1) / kE - g0)); }
  // Groups (of the whole row) that come by bulk copy.
  __device__ __forceinline__ int whole_first(int shift) const { return shift > 0 ? 1 : 0; }
  __device__ __forceinline__ int whole_stop(int shift) const { return (shift + V) / kE; }
  // One thread: this warp's part of a row; completes a phase of `bar`. Nothing is copied once a wait has run out.
  __device__ __forceinline__ void request(long long r, int warp, uint8_t* smem, uint32_t bar, bool aborted) const {
    const int s = shift(r);
    const int first = max(g0 + warp * per, whole_first(s));
    const int stop = min(g0 + min((warp + 1) * per, slice), whole_stop(s));
    const uint32_t bytes = stop > first && !aborted ? 16u * (stop - first) : 0u;
    mbar_expect_tx(bar, bytes);
    if (bytes > 0) bulk_load(smem_u32(smem + 16ll * (first - g0)), row(r) - s + static_cast<long long>(first) * kE, bytes, bar);
  }
  // Ragged element i (below 2 kE): its place in this block's slice, or -1; and its column, which may lie outside the row.
  __device__ __forceinline__ int edge_place(int i, int shift, int& col) const {
    const int g = i < kE ? 0 : (shift + V) / kE, at = g * kE + i % kE;
    col = at - shift;
    const bool ragged = i < kE ? shift > 0 : (shift + V) % kE != 0 && (g > 0 || shift == 0);
    return ragged && g >= g0 && g < g0 + groups(shift) ? at - g0 * kE : -1;
  }
};

// How rows of V columns are spread: the smallest cluster whose slices leave room for two blocks an SM (`half` bytes, of
// which `each` a block of the cluster are taken, where there is more than one); past 8 blocks, up to `whole` bytes.
// cs = 0: no cluster holds such a row.
struct SlicePlan {
  int cs, slice, per;
};
template <typename T>
inline SlicePlan slice_plan(long long V, int warps, long long half, long long whole, long long each = 0) {
  constexpr long long kE = 16 / sizeof(T);
  const long long groups = (V + 2 * kE - 2) / kE;  // wherever a row starts
  int cs = 1;
  while (cs < 8 && (groups + cs - 1) / cs * 16 + (cs > 1 ? cs * each : 0) > half) cs *= 2;
  const long long slice = (groups + cs - 1) / cs;
  if (slice * 16 > whole) return {0, 0, 0};
  return {cs, static_cast<int>(slice), static_cast<int>((slice + warps - 1) / warps)};
}

// Rows are dealt by the launch itself: one cluster a row, of which the first ones start, and a running cluster that wants
// more work cancels the start of a waiting one and takes its row (`clusterlaunchcontrol`). SMs differ by up to 40% in the
// bandwidth they get under full load, so equal shares would leave the fast ones waiting.
// One warp a block calls this; block 0 of the cluster asks, and tells the others, which may be up to three rows late: four
// barriers take turns, since one that has completed twice reads like one that has not.
struct RowQueue {
  uint4 answer;  // 16-byte aligned
  unsigned long long come, told[4];  // the answer has come; the next row is known here
  int next[4];

  // One thread, before the block's first barrier.
  __device__ __forceinline__ void init() {
    mbar_init(smem_u32(&come), 1);
    for (int i = 0; i < 4; ++i) mbar_init(smem_u32(told + i), 1);
  }
  // One thread of block 0: ask for the n-th row (n = 1, 2, ..), not after an answer that there is none.
  __device__ __forceinline__ void ask() {
    fence_proxy_async_smem();
    mbar_expect_tx(smem_u32(&come), 16);
    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
                     smem_u32(&answer)),
                 "r"(smem_u32(&come))
                 : "memory");
  }
  // The warp: the n-th row, or -1. Block 0 must have asked for it.
  __device__ __forceinline__ int take(int n, int rank, int cs, int lane, volatile int* abort_flag, bool& in_time) {
    if (rank == 0) {
      in_time &= short_wait<false>(smem_u32(&come), (n - 1) & 1, abort_flag);
      uint32_t got, x;
      asm volatile(
          "{\n\t.reg .b128 r;\n\t.reg .pred p;\n\t.reg .b64 lo, hi;\n\t"
          "ld.shared.v2.b64 {lo, hi}, [%2];\n\t"
          "mov.b128 r, {lo, hi};\n\t"
          "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n\t"
          "selp.b32 %0, 1, 0, p;\n\t"
          "mov.b32 %1, 0;\n\t"
          "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, r;\n\t}\n"
          : "=r"(got), "=r"(x)
          : "r"(smem_u32(&answer))
          : "memory");
      const int row = got && in_time ? static_cast<int>(x) / cs : -1;
      __syncwarp();
      if (cs == 1) return row;
      if (lane < cs) {
        const uint32_t to = mapa_shared(smem_u32(next + (n & 3)), lane);
        asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(to), "r"(row) : "memory");
        mbar_arrive_cluster(mapa_shared(smem_u32(told + ((n - 1) & 3)), lane));
      }
      __syncwarp();
    }
    in_time &= short_wait<true>(smem_u32(told + ((n - 1) & 3)), ((n - 1) >> 2) & 1, abort_flag);
    return in_time ? *static_cast<volatile int*>(next + (n & 3)) : -1;
  }
};

// One cluster of cs blocks a row.
template <typename K, typename... A>
inline int launch_clusters(K kern, long long rows, int cs, int threads, size_t smem, cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(rows * cs));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cs;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, args...) == cudaSuccess ? 0 : 1;
}

}  // namespace pd
