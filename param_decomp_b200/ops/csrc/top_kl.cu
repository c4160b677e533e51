// Distillation from a teacher's top logits. A teacher's row is K logits t_k at columns i_k and, as one more event, the
// logarithm of the sum of exponentials of all its other logits (`tail`); p_k and r are its softmax over these K + 1. With
// q the student's softmax over all V columns and R its sum over the columns that are not named,
//   loss = sum_k p_k (log p_k - log q_{i_k}) + r (log r - log R)
//   dloss / dz_j = (q_j - p_j) / T at a named column (p summed where a column is named twice), q_j (1 - r / R) / T elsewhere
// Without a tail r = 0: K = 1 is the cross entropy of one target. A slot with a negative column is unused; a row whose
// teacher has no mass counts zero with a zero gradient. The loss counts the slots of a column that is named twice one by one.
//
// Rows are held in the shared memory of a cluster of 1 to 8 blocks (`row_slice.cuh`) and read there for the sums and again
// for the gradient, so a logit crosses HBM once, its gradient once: bound by HBM, beside two exponentials a logit (16 lanes
// a clock). The named columns are taken out of the row first and written as -inf, so that R is a sum of what it consists
// of, not a difference, and relative to a logit that is in it: a rest far below the named logits keeps its value.
// The teacher's side is a chain of dependent steps on K numbers, and so is a loss, formed in 64 bits because it is a small
// difference of logarithms: a warp of its own does each, up to two rows ahead of the others and a row behind them.
// A gradient that is asked for by itself starts from the row's sums that an earlier call left (`known`): no sums, no exchange.
// Measured: loss and gradient of 8192 rows of 50,277 bf16, K = 64: 315 us, 5.2 TB/s, 0.81 of copy bandwidth. 1031 rows of
// 151,936 fp32, K = 32, a loss and then its gradient: 341 us for 1.88 GB, 5.5 TB/s, 0.85 of copy bandwidth (443 when the
// gradient formed the sums again; 367 when the blocks waited for the exchange of sums, 1.7 us a row, where no gradient is
// asked for and only the first block needs them). Rows to come asked for in L2 were slower (370 us for 315 at 50,277).
#include "row_slice.cuh"

namespace {

using namespace pd;

constexpr int kWarps = 8;  // that hold a row; as many threads as a row may have slots
constexpr int kMaxK = 32 * kWarps;

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
  float4* sums;        // [rows]: a row's sums, for a gradient that is asked for later; or null
  const float4* known; // [rows]: the sums of an earlier call with the same row and teacher; or null
  int* status;
  int* refused;
};

// A sum of exp(z / T) = 2^(c z) is kept as m, one of its z (the largest, or one that is not far below it), and s, the sum
// relative to a power of two near that z's own term: 2^k, k = c m to the nearest whole number. One fused multiply-add then
// gives an exponent, c z - k, without the rounding of c m in it, and a change of k is exact. (Where |c m| is so large that
// whole numbers are no closer than its rounding, as for logits masked with the type's lowest value, s is relative to
// exp(m / T) itself.)
struct MaxSum {
  float m, s;
};
constexpr float kLargest = 1.0e6f;
__device__ __forceinline__ float power_of(float m, float c) { return rintf(m * c); }
__device__ __forceinline__ bool moderate(float m, float c) { return fabsf(m * c) < kLargest; }
__device__ __forceinline__ float scaled(const MaxSum& x, float m, float c) {  // the sum as relative to m, not below x.m
  if (x.m == m) return x.s;  // -inf on both sides among them
  return x.s * ex2(moderate(x.m, c) && moderate(m, c) ? power_of(x.m, c) - power_of(m, c) : (x.m - m) * c);
}
// exp(z / T) as relative to m.
__device__ __forceinline__ float term(float z, float m, float c) {
  return ex2(moderate(m, c) ? fmaf(z, c, -power_of(m, c)) : (z - m) * c);
}
__device__ __forceinline__ MaxSum merge(const MaxSum& x, const MaxSum& y, float c) {
  const float m = fmaxf(x.m, y.m);
  return MaxSum{m, scaled(x, m, c) + scaled(y, m, c)};
}
// Logarithm of the sum over exp(m / T), in 64 bits.
constexpr double kLn2 = 0.6931471805599453;
__device__ __forceinline__ double log_of(const MaxSum& x, float m, float c) {
  const double at = moderate(x.m, c) ? power_of(x.m, c) - static_cast<double>(m) * c : (static_cast<double>(x.m) - m) * c;
  return at * kLn2 + log(static_cast<double>(x.s));
}

struct Row {  // sums over a row: the columns that are not named, and those that are
  MaxSum rest, top;
};
// Over the `n` (a power of two) neighbouring lanes.
__device__ __forceinline__ Row merge_lanes(const Row& x, int n, float c) {
  float m0 = x.rest.m, m1 = x.top.m;
  for (int o = n / 2; o > 0; o >>= 1) {
    m0 = fmaxf(m0, __shfl_xor_sync(0xffffffffu, m0, o));
    m1 = fmaxf(m1, __shfl_xor_sync(0xffffffffu, m1, o));
  }
  float s0 = scaled(x.rest, m0, c), s1 = scaled(x.top, m1, c);
  for (int o = n / 2; o > 0; o >>= 1) {
    s0 += __shfl_xor_sync(0xffffffffu, s0, o);
    s1 += __shfl_xor_sync(0xffffffffu, s1, o);
  }
  return Row{{m0, s0}, {m1, s1}};
}

struct Teacher {  // of a row
  int column[kMaxK];       // of the slots; -1 where a slot is unused, -2 - i where slot i has named the column already
  float of_column[kMaxK];  // probability of the slot's column, over all slots that name it
  float edge[16];          // elements at the row's ragged ends, named ones as -inf
  float r, named;          // probability of the tail; of all slots
  int row;                 // or -1: there is no further one
  float most;              // largest of the logits, or 0 where none is above -inf
  double most_at, tail_at; // it over T, and the tail, relative to the larger of the two
  bool live;
};

__device__ __forceinline__ float value_at(const Call& call, long long i) {
  return call.values_fp32 ? static_cast<const float*>(call.values)[i]
                          : as_float(static_cast<const __nv_bfloat16*>(call.values)[i]);
}

// One warp: the teacher's row, kPer slots a lane, and the row's ragged ends.
template <typename T, int kPer>
__device__ void prepare(const Call& call, const RowSlice<T>& rows, long long row, Teacher& t, int lane) {
  const int K = call.K;
  int col[kPer];
  float v[kPer];
  bool bad = false, nan = false;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int k = 32 * i + lane;
    col[i] = -1;
    v[i] = -INFINITY;
    if (k < K) {
      const long long at = row * K + k;
      const long long c = call.wide ? static_cast<const long long*>(call.indices)[at] : static_cast<const int*>(call.indices)[at];
      v[i] = value_at(call, at);
      bad |= c >= call.V;
      col[i] = c < 0 || c >= call.V ? -1 : static_cast<int>(c);
    }
  }
  const float tail = call.tail != nullptr ? call.tail[row] : -INFINITY;  // already over T
  const int shift = rows.shift(row);
  int edge_col = -1;
  const int edge_at = lane < 2 * RowSlice<T>::kE ? rows.edge_place(lane, shift, edge_col) : -1;
  float edge = edge_at >= 0 && edge_col >= 0 && edge_col < call.V ? as_float(rows.row(row)[edge_col]) : -INFINITY;
  if (bad) {
    atomicCAS(call.status, 0, kBadColumn);
    *static_cast<volatile int*>(call.refused) = 1;
  }
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    if (col[i] < 0) v[i] = -INFINITY;
    m = fmaxf(m, v[i]);
    nan |= v[i] != v[i];
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  nan = __any_sync(0xffffffffu, nan) || tail != tail;
  // The largest over T in 64 bits (in 32 a row of the type's lowest value would have no mass at T < 1), and rounded before
  // anything is taken off it: what a fused multiply-add keeps of the product is 10^22 there.
  const float inv_t = static_cast<float>(call.inv_t), most = m > -INFINITY ? m : 0.0f;
  const double over_t = __dmul_rn(m, call.inv_t), top = fmax(over_t, static_cast<double>(tail));
  const bool live = nan || top > -INFINITY;
  const double most_at = m > -INFINITY ? over_t - top : 0.0, tail_at = tail == -INFINITY ? tail : tail - top;
  const float below = static_cast<float>(most_at);
  float p[kPer], s = 0.0f;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    p[i] = v[i] == -INFINITY ? 0.0f : expf((v[i] - most) * inv_t + below);
    s += p[i];
  }
  s = warp_sum(s);
  const float rest = tail == -INFINITY ? 0.0f : expf(static_cast<float>(tail_at)), total = live ? s + rest : 1.0f, share = 1.0f / total;
  // does a column come twice?
  bool twice = false;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const unsigned same = __match_any_sync(0xffffffffu, col[i]);  // every lane, whether its slot is used or not
    twice |= col[i] >= 0 && __popc(same) > 1;
    if (32 * (i + 1) >= K) break;
#pragma unroll 4
    for (int o = 0; o < 32; ++o) {
      const int other = __shfl_sync(0xffffffffu, col[i], lane + o);
#pragma unroll
      for (int j = i + 1; j < kPer; ++j) twice |= col[j] == other && other >= 0;
    }
  }
  twice = __any_sync(0xffffffffu, twice);
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int k = 32 * i + lane;
    if (k < K) {
      t.column[k] = col[i];
      t.of_column[k] = p[i] * share;
    }
  }
  __syncwarp();
  if (twice) {
    float sum[kPer];
    int first[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int k = 32 * i + lane;
      sum[i] = 0.0f;
      first[i] = k;
      if (k < K && col[i] >= 0)
        for (int j = 0; j < K; ++j)
          if (t.column[j] == col[i]) {
            first[i] = min(first[i], j);
            sum[i] += t.of_column[j];
          }
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (32 * i + lane < K) {
        if (first[i] != 32 * i + lane) t.column[32 * i + lane] = -2 - first[i];
        t.of_column[32 * i + lane] = sum[i];
      }
  }
  if (edge_at >= 0)
    for (int k = 0; k < K; ++k)
      if (t.column[k] == edge_col) edge = -INFINITY;
  if (lane < 2 * RowSlice<T>::kE) t.edge[lane] = edge;
  if (lane == 0) {
    t.r = live ? rest * share : 0.0f;
    t.named = live ? s * share : 0.0f;
    t.live = live;
    t.most = most;
    t.most_at = most_at;
    t.tail_at = tail_at;
  }
}

// One warp: the loss of a row, sum_k p_k (a_k - b_k - log E + log Z) + r (log r - log R), with a and b the two sides' logits
// and E and Z their sums. At a small loss a rounding of E, Z or a p_k would count in full, so all that the slots add to
// them is formed in 64 bits; that of the student's other logits counts as R - r, which is small there, on the 32 bits of
// its sum. The student's side is taken relative to m, one of its larger logits.
__device__ float loss_of(const Call& call, long long row, const Teacher& t, const Row& sums, const float* named, float c,
                         int lane) {
  const double inv_t = call.inv_t, own_inv_t = static_cast<double>(c) * kLn2;  // the sums' own 1 / T
  const float larger = fmaxf(sums.rest.m, sums.top.m), m = larger > -INFINITY ? larger : 0.0f;
  double teacher = 0.0, weighted = 0.0, student = 0.0;  // sums over the slots: E's part, that of E p_k (a_k - b_k), Z's part
  for (int k = lane; k < call.K; k += 32) {
    const int column = t.column[k];
    if (column == -1) continue;
    const double a = (static_cast<double>(value_at(call, row * call.K + k)) - t.most) * inv_t + t.most_at;
    const double b = (static_cast<double>(named[column >= 0 ? k : -2 - column]) - m) * own_inv_t;
    const double e = exp(a);
    if (!(static_cast<float>(e) == 0.0f)) {  // what is nothing in 32 bits costs nothing where the student's is -inf
      teacher += e;
      weighted += e * (a - b);
    }
    if (column >= 0) student += exp(b);
  }
  __syncwarp();
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    teacher += __shfl_xor_sync(0xffffffffu, teacher, o);
    weighted += __shfl_xor_sync(0xffffffffu, weighted, o);
    student += __shfl_xor_sync(0xffffffffu, student, o);
  }
  const double a_rest = t.tail_at, e_rest = t.r == 0.0f ? 0.0 : exp(a_rest);
  const double log_rest = log_of(sums.rest, m, c), total = teacher + e_rest;
  const double log_ratio = log(exp(log_rest) + student) - log(total);
  double sum = 0.0;
  if (!(teacher == 0.0)) sum += weighted + teacher * log_ratio;
  if (!(t.r == 0.0f)) sum += e_rest * (a_rest - log_rest + log_ratio);
  return t.live ? static_cast<float>(sum / total) : 0.0f;
}

// One object: the address of its barriers goes to inline assembly, so the compiler takes every wait and barrier there for
// one that may change any part of it.
struct Shared {
  RowQueue queue;
  unsigned long long bars[kWarps + 12];
  Teacher teacher[3];
  float named[3][kMaxK];  // student's logits at the columns, in the slots that speak for them
  Row red[kWarps], xch[3][8], sums[3];  // of the last three rows, as `named`: blocks may be two rows apart
  float2 part[kWarps];
  int next;  // the row behind the present one, or -1
  int rows;  // this cluster has had, once there is no further one
  int abort_flag;
};

constexpr int kShared = 11264;
static_assert(sizeof(Shared) <= kShared);

template <typename T>
__global__ void __launch_bounds__(32 * (kWarps + 2), 3) top_kl_kernel(const Call call, const SlicePlan plan) {
  constexpr int kE = RowSlice<T>::kE, kP = kE / 2;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(16) Shared sh;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int cs = plan.cs, warps = kWarps, nt = 32 * kWarps;
  const int rank = cs > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const float c = static_cast<float>(call.inv_t * 1.4426950408889634);
  const RowSlice<T> rows{static_cast<const T*>(call.z), call.ld, call.V, rank * plan.slice, plan.slice, plan.per};
  T* buf = reinterpret_cast<T*>(smem);
  const uint32_t bar0 = smem_u32(sh.bars), ready = bar0 + 8 * kWarps, lost = ready + 16, summed = ready + 32, met = ready + 64;
  if (tid == 0) {
    for (int i = 0; i < warps; ++i) mbar_init(bar0 + 8 * i, 1);
    for (int i = 0; i < 8; ++i) mbar_init(ready + 8 * i, 1);
    for (int i = 0; i < 4; ++i) mbar_init(met + 8 * i, cs);
    sh.rows = -1;
    sh.queue.init();
    sh.abort_flag = 0;
    mbar_fence_init();
  }
  __syncthreads();
  if (cs > 1) cluster_sync_all();  // every block of the cluster runs before another one stores to its shared memory
  auto late = [&](bool in_time) {
    if (!in_time && call.status != nullptr) atomicCAS(call.status, 0, kTimeoutProducer);
  };
  // The n-th completion of a pair of barriers that take turns: one that is waited for late is not mistaken for the next.
  auto wait_pair = [&](uint32_t pair, int n) { return short_wait<false>(pair + 8 * (n & 1), (n >> 1) & 1, &sh.abort_flag); };
  // The n-th completion of four that take turns.
  auto wait_four = [&](uint32_t four, int n) { return short_wait<false>(four + 8 * (n & 3), (n >> 2) & 1, &sh.abort_flag); };
  auto wait_met = [&](int n) { return short_wait<true>(met + 8 * (n & 3), (n >> 2) & 1, &sh.abort_flag); };
  const bool losses = rank == 0 && call.loss != nullptr;
  const bool loose = cs > 1 && call.known != nullptr;  // nothing else keeps the cluster's blocks together
  const bool apart = cs > 1 && call.dz == nullptr;     // only the first block needs the cluster's sums, and not to go on
  auto send = [&](const Row& sums, int n, int block) {  // this block's part of a row's
    const uint32_t to = mapa_shared(smem_u32(&sh.xch[n % 3][rank]), block);
    store_cluster_f32(to, sums.rest.m);
    store_cluster_f32(to + 4, sums.rest.s);
    store_cluster_f32(to + 8, sums.top.m);
    store_cluster_f32(to + 12, sums.top.s);
  };
  auto met_sums = [&](int n) {  // the warp
    const Row none{{-INFINITY, 0.0f}, {-INFINITY, 0.0f}};
    return merge_lanes((lane & 7) < cs ? sh.xch[n % 3][lane & 7] : none, 8, c);
  };
  if (warp == warps) {  // the teacher's side, up to two rows ahead
    auto teach = [&](int row, int n) {
      Teacher& t = sh.teacher[n % 3];
      if (row < 0) {
      } else if (call.K <= 32) {
        prepare<T, 1>(call, rows, row, t, lane);
      } else if (call.K <= 64) {
        prepare<T, 2>(call, rows, row, t, lane);
      } else {
        prepare<T, kMaxK / 32>(call, rows, row, t, lane);
      }
      t.row = row;
      __syncwarp();
      if (lane == 0) mbar_arrive(ready + 8 * (n & 1));
      __syncwarp();
    };
    // The n-th row, while the one after it is asked for.
    bool more = true;
    auto next = [&](int n) {
      if (!more) return -1;
      bool in_time = true;
      const int row = sh.queue.take(n, rank, cs, lane, &sh.abort_flag, in_time);
      late(in_time);
      more = row >= 0;
      if (more && rank == 0 && lane == 0) sh.queue.ask();
      __syncwarp();
      return row;
    };
    if (rank == 0 && lane == 0) sh.queue.ask();
    __syncwarp();
    teach(blockIdx.x / cs, 0);
    teach(next(1), 1);
    int ahead = next(2);
    for (int n = 0; sh.teacher[n % 3].row >= 0; ++n) {
      late(wait_four(summed, n));  // the others are done with the row before,
      if (losses && n > 0) late(wait_pair(lost, n - 1));  // and so is the warp below
      if (loose && rank == 0 && n > 0) late(wait_met(n - 1));  // all blocks have begun the row before: none is left far behind
      teach(ahead, n + 2);
      if (apart && rank == 0) late(wait_pair(lost, n));  // all blocks have handed this row over: its places serve the third one on
      ahead = next(n + 3);
    }
  } else if (warp == warps + 1) {  // losses, a row behind
    // What a loss reads is written again by a row that is not told to any block before the teacher of the row behind is
    // there, which waits for this warp.
    for (int n = 0; losses || loose || apart; ++n) {
      late(wait_four(summed, n));
      if (n == *static_cast<volatile int*>(&sh.rows) || *static_cast<volatile int*>(&sh.abort_flag)) break;
      Row sums = sh.sums[n % 3];
      if (loose || apart) {
        if (lane == 0) {
          if (apart) send(sums, n, 0);
          mbar_arrive_cluster(mapa_shared(met + 8 * (n & 3), 0));  // with it, the named logits that were stored before the barriers
        }
        __syncwarp();
        if (loose || rank != 0) continue;
        late(wait_met(n));
        sums = met_sums(n);
      }
      const Teacher& t = sh.teacher[n % 3];
      if (call.sums != nullptr && lane == 0)
        call.sums[t.row] = make_float4(sums.rest.m, sums.rest.s, sums.top.m, sums.top.s);
      const float loss = loss_of(call, t.row, t, sums, sh.named[n % 3], c, lane);
      if (lane == 0) {
        call.loss[t.row] = loss;
        mbar_arrive(lost + 8 * (n & 1));
      }
      __syncwarp();
    }
  } else {
    if (lane == 0) rows.request(blockIdx.x / cs, warp, smem, bar0 + 8 * warp, false);
    __syncwarp();
    late(wait_pair(ready, 0));
    int n = 0;
    for (int row = blockIdx.x / cs; row >= 0; ++n) {
      const Teacher& t = sh.teacher[n % 3];
      const int shift = rows.shift(row), groups = rows.groups(shift);
      const int begin = warp * plan.per + lane, stop = min(groups, (warp + 1) * plan.per);
      float* zk = sh.named[n % 3];
      const float up =  // on its way while the row is waited for
          (call.scale != nullptr ? call.scale[row] : 1.0f) * static_cast<float>(call.inv_t);
      late(short_wait<false>(bar0 + 8 * warp, n & 1, &sh.abort_flag));
      if (tid < 2 * kE) {
        int col;
        const int at = rows.edge_place(tid, shift, col);
        if (at >= 0) store1(buf + at, t.edge[tid]);
      }
      int mine = -1, next;  // the column whose gradient this thread writes; the row behind this one
      float mine_logit = 0.0f;
      Row sums;
      const f32x2 c2 = pk2(c, c);
      if (call.known != nullptr) {  // the row's sums are there: a gradient is all that is left to do
        const float4 q = call.known[row];
        sums = Row{{q.x, q.y}, {q.z, q.w}};
        if (tid < call.K && t.column[tid] >= 0) {
          const int at = shift + t.column[tid] - rows.g0 * kE;
          if (at >= 0 && at < groups * kE) {
            mine = t.column[tid];
            mine_logit = as_float(rows.row(row)[mine]);
          }
        }
        if (warp == 0) late(wait_pair(ready, n + 1));
        if (tid == 0) sh.next = *static_cast<volatile int*>(&sh.abort_flag) ? -1 : sh.teacher[(n + 1) % 3].row;
        fence_proxy_async_smem();  // before bulk copies of the next row write where this row's ends are
        sync_first(nt);
        next = sh.next;
      } else {
        // Named columns leave the row: their logits go to the first block, for the loss. A warp with slots waits for all parts
        // of the slice, and as a whole: lanes that wait each for their own leave it split for the rest of the kernel.
        if (32 * warp < call.K)
          for (int w = 0; w < warps; ++w) late(short_wait<false>(bar0 + 8 * w, n & 1, &sh.abort_flag));
        if (tid < call.K && t.column[tid] >= 0 && t.column[tid] < call.V) {
          const int place = shift + t.column[tid], g = place / kE, at = place - rows.g0 * kE;
          if (at >= 0 && at < groups * kE) {
            mine = t.column[tid];
            if (g >= rows.whole_first(shift) && g < rows.whole_stop(shift)) {
              mine_logit = as_float(buf[at]);
              store1(buf + at, -INFINITY);
            } else {
              mine_logit = as_float(rows.row(row)[mine]);  // at a ragged end, which is already without it
            }
            if (cs > 1)
              store_cluster_f32(mapa_shared(smem_u32(zk + tid), 0), mine_logit);
            else
              zk[tid] = mine_logit;
          }
        }
        fence_proxy_async_smem();  // before bulk copies of the next row write where this row's ends and marks are
        sync_first(nt);
        // The slice's sums relative to one of its own logits: they serve as they are unless another one is larger by 2^100.
        GroupMax<T> gm;
        if (groups > 0) gm.add(*reinterpret_cast<const uint4*>(smem));
        if (groups > 1) gm.add(*reinterpret_cast<const uint4*>(smem + 16));
        const float ref = gm.value();
        auto add_up = [&](auto exponent) {  // of a pair of logits
          f32x2 s0 = 0ull, s1 = 0ull;
#pragma unroll 4
          for (int g = begin; g < stop; g += 32) {
            f32x2 v[kP];
            pairs_of<T>(*reinterpret_cast<const uint4*>(smem + 16 * g), v);
#pragma unroll
            for (int j = 0; j < kP; ++j) {
              const float2 x = unpack2(exponent(v[j]));
              const f32x2 e = pk2(ex2(x.x), ex2(x.y));
              if (j & 1)
                s1 = add2(s1, e);
              else
                s0 = add2(s0, e);
            }
          }
          const float2 a = unpack2(add2(s0, s1));
          return a.x + a.y;
        };
        float2 part = make_float2(INFINITY, 0.0f);
        if (moderate(ref, c)) {
          const float k = -power_of(ref, c);
          const f32x2 k2 = pk2(k, k);
          part = make_float2(add_up([&](f32x2 v) { return fma2(v, c2, k2); }), mine >= 0 ? term(mine_logit, ref, c) : 0.0f);
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) {
            part.x += __shfl_xor_sync(0xffffffffu, part.x, o);
            part.y += __shfl_xor_sync(0xffffffffu, part.y, o);
          }
        }
        if (lane == 0) sh.part[warp] = part;
        if (warp == 0) late(wait_pair(ready, n + 1));
        if (tid == 0) {  // all warps go on together, or none does: what the barrier below shows them decides
          sh.next = *static_cast<volatile int*>(&sh.abort_flag) ? -1 : sh.teacher[(n + 1) % 3].row;
        }
        sync_first(nt);
        next = sh.next;
        part = sh.part[lane & 7];
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) {
          part.x += __shfl_xor_sync(0xffffffffu, part.x, o);
          part.y += __shfl_xor_sync(0xffffffffu, part.y, o);
        }
        sums = Row{{ref, part.x}, {ref, part.y}};
        if (!(part.x < 1e30f && part.y < 1e30f)) {  // the same in every thread: sums relative to true maxima
          GroupMax<T> all;
          bool nan = false;
          for (int g = begin; g < stop; g += 32) {
            const uint4 q = *reinterpret_cast<const uint4*>(smem + 16 * g);
            all.add(q);
            f32x2 v[kP];
            pairs_of<T>(q, v);
#pragma unroll
            for (int j = 0; j < kP; ++j) {
              const float2 x = unpack2(v[j]);
              nan |= x.x != x.x || x.y != x.y;
            }
          }
          const float own = all.value();
          sums = Row{{own, 0.0f}, {-INFINITY, 0.0f}};
          if (mine >= 0 && mine_logit > -INFINITY) sums.top = MaxSum{mine_logit, term(mine_logit, mine_logit, c)};
          // a maximum passes NaN over: beside nothing but -inf it would be lost
          if (mine_logit != mine_logit) sums.top.s = NAN;
          if (nan) {
            sums.rest.s = NAN;
          } else if (moderate(own, c)) {
            const float k = -power_of(own, c);
            const f32x2 k2 = pk2(k, k);
            sums.rest.s = add_up([&](f32x2 v) { return fma2(v, c2, k2); });
          } else if (own > -INFINITY) {
            const f32x2 neg = pk2(-own, -own);
            sums.rest.s = add_up([&](f32x2 v) { return mul2(add2(v, neg), c2); });
          }
          sums = merge_lanes(sums, 32, c);
          if (lane == 0) sh.red[warp] = sums;
          sync_first(nt);
          sums = merge_lanes(sh.red[lane & 7], 8, c);
        }
        if (cs > 1 && !apart) {
          if (warp == 0 && lane < cs) {
            send(sums, n, lane);
            mbar_arrive_cluster(mapa_shared(met + 8 * (n & 3), lane));
          }
          __syncwarp();
          late(wait_met(n));
          sums = met_sums(n);
        }
      }
      if (tid == 0) {
        sh.sums[n % 3] = sums;
        mbar_arrive(summed + 8 * (n & 3));
      }
      __syncwarp();
      auto ask_for_next = [&] {  // the warp's part of it
        __syncwarp();
        if (lane == 0 && next >= 0) {
          fence_proxy_async_smem();
          rows.request(next, warp, smem, bar0 + 8 * warp, false);
        }
        __syncwarp();
      };
      if (call.dz != nullptr) {
        const MaxSum all = merge(sums.rest, sums.top, c), rest = sums.rest;
        const bool live = t.live;
        // the difference R - r from whichever side is small
        const float gap = t.r > 0.5f ? t.named - scaled(sums.top, all.m, c) / all.s : scaled(rest, all.m, c) / all.s - t.r;
        float f = rest.s == 0.0f ? 0.0f * all.s : gap / rest.s * up;  // of an exponential as relative to rest.m; NaN stays NaN
        T* const out = static_cast<T*>(call.dz) + static_cast<long long>(row) * call.ldo;  // column 0
        T* const slice_out = out + (rows.g0 * kE - shift);
        const int inner_first = rows.whole_first(shift) - rows.g0, inner_stop = rows.whole_stop(shift) - rows.g0;
        auto put = [&](auto gradient) {  // words of gradients from words of the row
          auto ragged = [&](int g) {
            const uint4 q = gradient(*reinterpret_cast<const uint4*>(smem + 16 * g));
            const T* each = reinterpret_cast<const T*>(&q);
            const int col = (rows.g0 + g) * kE - shift;
#pragma unroll
            for (int j = 0; j < kE; ++j)
              if (col + j >= 0 && col + j < call.V) out[col + j] = each[j];
          };
          int g = begin;
          if (g < inner_first && g < stop) {  // no more than the row's first group
            ragged(g);
            g += 32;
          }
          const int inner = min(stop, inner_stop);
          uint4* to = reinterpret_cast<uint4*>(slice_out + g * kE);
#pragma unroll 4
          for (; g < inner; g += 32, to += 32) *to = gradient(*reinterpret_cast<const uint4*>(smem + 16 * g));
          if (g < stop) ragged(g);  // no more than its last
        };
        if (!live || f == 0.0f) {
          put([&](const uint4&) { return make_uint4(0u, 0u, 0u, 0u); });
        } else if constexpr (sizeof(T) == 4) {
          const float k = moderate(rest.m, c) ? -power_of(rest.m, c) : 0.0f;
          const f32x2 k2 = pk2(k, k), neg = pk2(-rest.m, -rest.m), f2 = pk2(f, f);
          auto words = [&](const uint4& w, auto exponent) {
            f32x2 v[kP];
            pairs_of<T>(w, v);
#pragma unroll
            for (int j = 0; j < kP; ++j) {
              const float2 x = unpack2(exponent(v[j])), e = unpack2(mul2(pk2(ex2(x.x), ex2(x.y)), f2));
              v[j] = pk2(e.x, e.y);
            }
            const float2 a = unpack2(v[0]), b = unpack2(v[1]);
            return make_uint4(__float_as_uint(a.x), __float_as_uint(a.y), __float_as_uint(b.x), __float_as_uint(b.y));
          };
          if (moderate(rest.m, c))
            put([&](const uint4& w) { return words(w, [&](f32x2 v) { return fma2(v, c2, k2); }); });
          else
            put([&](const uint4& w) { return words(w, [&](f32x2 v) { return mul2(add2(v, neg), c2); }); });
        } else if (const float power = power_of(rest.m, c); moderate(rest.m, c) && fabsf(power) > 512.0f) {
          // far from zero the exponent has no bits left for the logarithm of f, which the next branch adds to it
          const f32x2 k2 = pk2(-power, -power), f2 = pk2(f, f);
          put([&](const uint4& w) {
            f32x2 v[kP];
            pairs_of<T>(w, v);
            uint32_t o[kP];
#pragma unroll
            for (int j = 0; j < kP; ++j) {
              const float2 x = unpack2(fma2(v[j], c2, k2));
              o[j] = pack_bf16_2(mul2(pk2(ex2(x.x), ex2(x.y)), f2));
            }
            return make_uint4(o[0], o[1], o[2], o[3]);
          });
        } else {
          // f goes into the exponent, its sign into the word: with it an exponent of up to 512 + 150 is rounded to 2^-15, so a
          // value is off by 2^-15.5 of itself at most, by 2^-17.5 where the exponent is below 128: far below its half step
          const float lf = log2f(fabsf(f)), k = moderate(rest.m, c) ? lf - power_of(rest.m, c) : 0.0f;
          const f32x2 k2 = pk2(k, k), neg = pk2(-rest.m, -rest.m), lf2 = pk2(lf, lf);
          const uint32_t sign = f < 0.0f ? 0x80008000u : 0u;
          auto words = [&](const uint4& w, auto exponent) {
            f32x2 v[kP];
            pairs_of<T>(w, v);
            uint32_t o[kP];
#pragma unroll
            for (int j = 0; j < kP; ++j) {
              const float2 x = unpack2(exponent(v[j]));
              o[j] = pack_bf16_2(pk2(ex2(x.x), ex2(x.y))) ^ sign;
            }
            return make_uint4(o[0], o[1], o[2], o[3]);
          };
          if (moderate(rest.m, c))
            put([&](const uint4& w) { return words(w, [&](f32x2 v) { return fma2(v, c2, k2); }); });
          else
            put([&](const uint4& w) { return words(w, [&](f32x2 v) { return fma2(add2(v, neg), c2, lf2); }); });
        }
        ask_for_next();
        sync_first(nt);  // the row's stores are in order before those of the named columns
        if (mine >= 0) {
          const float q = term(mine_logit, all.m, c) / all.s;
          store1(out + mine, live ? (q - t.of_column[tid]) * up : 0.0f);
        }
      } else {
        ask_for_next();
      }
      row = next;
    }
    if (tid == 0) {
      *static_cast<volatile int*>(&sh.rows) = n;
      mbar_arrive(summed + 8 * (n & 3));
    }
  }
  __syncwarp();
  if (cs > 1) cluster_sync_all();  // no block leaves while another one may still store to it
}

// A slice beside the fixed shared memory and 1 KB of the system's: two blocks an SM, or one.
constexpr long long kHalfSm = 113 * 1024 - kShared, kWholeSm = 227 * 1024 - kShared;

template <typename T>
int launch(const Call& call, cudaStream_t st) {
  const SlicePlan plan = slice_plan<T>(call.V, kWarps, kHalfSm, kWholeSm);
  if (plan.cs == 0) return 5;
  const int smem = plan.slice * 16, threads = 32 * (kWarps + 2);
  auto kern = top_kl_kernel<T>;
  static std::atomic<unsigned long long> asked{0};
  if (!make_room(asked, reinterpret_cast<const void*>(kern), kWholeSm)) return 2;
  return launch_clusters(kern, call.rows, plan.cs, threads, smem, st, call, plan);
}

}  // namespace

// Widest row that a cluster holds.
extern "C" long long pd_top_kl_max_columns(int z_fp32) { return 8 * kWholeSm / (z_fp32 ? 4 : 2) - 16; }

extern "C" int pd_top_kl(const void* z, long long rows, int V, long long ld, const void* indices, int wide,
                         const void* values, int values_fp32, int K, const float* tail, double inv_t, float* loss, void* dz,
                         long long ldo, const float* scale, float* sums, const float* known, int z_fp32, int* status,
                         int* refused, void* stream) {
  if (rows <= 0 || rows >= (1ll << 28) || V <= 0 || K <= 0 || K > kMaxK || !(inv_t > 0.0)) return 5;
  if ((dz == nullptr && loss == nullptr) || (known != nullptr && (dz == nullptr || loss != nullptr))) return 5;
  const Call call{z, rows, ld, V, indices, wide, values, values_fp32, K, tail, inv_t, loss, dz, ldo, scale,
                  reinterpret_cast<float4*>(sums), reinterpret_cast<const float4*>(known), status, refused};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return z_fp32 ? launch<float>(call, st) : launch<__nv_bfloat16>(call, st);
}
