// The k largest logits of every row (descending, equal logits in the order of their columns), their columns, and the
// logarithm of the sum of exp(z / T) over the rest of the row.
//
// Rows are held in the shared memory of a cluster of 1 to 8 blocks (`row_slice.cuh`) and read there twice, so a logit
// crosses HBM once, and that bounds it. First pass: every thread keeps the maxima of two halves of its own columns; the k-th
// largest T_0 of those (over the cluster's blocks, of the threads of one number taken together) is a lower bound of the k-th
// largest logit, and a tight one (k = 64 of 512 maxima: about 68 logits reach it). Second: logits that reach T_0 are
// collected with their columns, and exponentials are summed with every logit cut off at T_0, whose term is taken off again
// once a collected logit. Four more warps of the cluster's first block place the collected ones, sorted into 256 bins by key
// and counted within a bin, with (logit, column) as one number, so the order in which they arrived does not matter; the
// others read the next row meanwhile.
// A row that defeats the bound (fewer than 2 k groups of 16 bytes, ties in masses, rows of -inf) is selected out of global
// memory by its keys' digits instead, exactly and at any number of ties, and a rest that is small beside what was taken off
// is summed by itself. That costs 100 to 200 us a row in place of 7. Rows of normal logits about a mean that falls with the
// logarithm of the column do not need it at k = 64 (8192 rows of 50,277 bf16: 358 us, columns permuted 265) but at k = 256 they
// do when the columns are in that order (5.8 ms, permuted 0.45): the largest are neighbours then, and share their maxima.
// Groups dealt to the warps 32 at a time spread them (309 us) but take 25 bulk copies a warp: 240 us in place of 213 on level
// rows. Eight or four loads in flight in the selection did not pay: their registers cost the common case 10 to 40%.
// Measured: 8192 rows of 50,277 bf16, k = 64: 210 us, 3.9 TB/s (250 with the placing in the readers' path). A row takes a
// block 7.5 us, of which the sums are 2.9 (two blocks an SM share 16 exponentials a clock), the maxima 1.5, bound and
// collecting 2.3, waiting for the row 0.5. 1031 rows of 151,936 fp32, k = 256, clusters of 8: 216 us, 2.9 TB/s (390 with the
// placing in the path, and a warp that was split by a lane that waited alone): a row takes 6.8 us, of which 1 to 2 are the
// exchange of maxima. Asking for rows to come in L2 gained nothing (217 and 307 us), nor did maxima of half
// the row, a looser bound with twice as many to collect (217 us).
#include <algorithm>

#include "row_slice.cuh"

namespace {

using namespace pd;

constexpr int kMaxK = 256;
constexpr int kRoom = 512;  // logits collected
constexpr int kWarps = 8, kThreads = 32 * kWarps;  // that hold a row; one more warp deals rows,
constexpr int kSelWarps = 4, kSelThreads = 32 * kSelWarps;  // and these select, in a cluster's first block, a row behind
constexpr int kMaxima = 2 * kThreads;
constexpr int kBins = 512;
constexpr int kSelBins = 256;
constexpr float kLog2E = 1.4426950408889634f;

__device__ __forceinline__ uint32_t load_cluster_u32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ unsigned long long load_cluster_u64(uint32_t addr) {
  unsigned long long v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
  return v;
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
// (logit, column) as one number: larger logits first, then lower columns; the last bit keeps a zero's sign.
__device__ __forceinline__ unsigned long long place_of(float v, int col) {
  return (static_cast<unsigned long long>(key_of(v)) << 32) | ((0x7FFFFFFFu - static_cast<uint32_t>(col)) << 1) |
         (__float_as_uint(v) == 0x80000000u);
}
__device__ __forceinline__ int column_of(unsigned long long place) {
  return static_cast<int>(0x7FFFFFFFu - (static_cast<uint32_t>(place) >> 1));
}
__device__ __forceinline__ float logit_of(unsigned long long place) {
  const float v = value_of(static_cast<uint32_t>(place >> 32));
  return v == 0.0f && (place & 1) ? -0.0f : v;
}
// The larger of two words' values, NaN before everything; and a word cut off at `low`, NaN too.
template <typename T>
__device__ __forceinline__ uint32_t most(uint32_t a, uint32_t b) {
  if constexpr (sizeof(T) == 2) {
    const __nv_bfloat162 r =
        __hmax2_nan(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  } else {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(__uint_as_float(a)), "f"(__uint_as_float(b)));
    return __float_as_uint(r);
  }
}
template <typename T>
__device__ __forceinline__ uint32_t most(const uint4& q) {
  return most<T>(most<T>(q.x, q.y), most<T>(q.z, q.w));
}
template <typename T>
__device__ __forceinline__ bool below(uint32_t w, float low) {
  if constexpr (sizeof(T) == 2)
    return __uint_as_float(w << 16) < low && __uint_as_float(w & 0xFFFF0000u) < low;
  else
    return __uint_as_float(w) < low;
}
// One bit a value of the group that is not below `low`.
template <typename T>
__device__ __forceinline__ uint32_t reached(const uint4& q, float low) {
  f32x2 v[8 / sizeof(T)];
  pairs_of<T>(q, v);
  uint32_t bits = 0;
#pragma unroll
  for (int j = 0; j < static_cast<int>(8 / sizeof(T)); ++j) {
    const float2 x = unpack2(v[j]);
    bits |= (x.x < low ? 0u : 1u << 2 * j) | (x.y < low ? 0u : 2u << 2 * j);
  }
  return bits;
}
template <typename T>
__device__ __forceinline__ uint32_t cut_off(uint32_t w, uint32_t low) {
  if constexpr (sizeof(T) == 2) {
    const __nv_bfloat162 r = __hmin2(*reinterpret_cast<const __nv_bfloat162*>(&w), *reinterpret_cast<const __nv_bfloat162*>(&low));
    return *reinterpret_cast<const uint32_t*>(&r);
  } else {
    return __float_as_uint(fminf(__uint_as_float(w), __uint_as_float(low)));
  }
}

// A row in global memory, 16 bytes at a time, at 16-byte addresses wherever it starts: group g holds columns g kE - shift + j.
template <typename T>
struct Row {
  static constexpr int kE = 16 / sizeof(T);
  const T* base;  // column 0
  int V, shift, groups;
  __device__ __forceinline__ Row(const T* p, int V_) : base(p), V(V_) {
    shift = static_cast<int>((reinterpret_cast<uintptr_t>(p) & 15) / sizeof(T));
    groups = (shift + V + kE - 1) / kE;
  }
  // A group as it lies in memory; columns outside the row hold -inf.
  __device__ __forceinline__ uint4 load(int g) const {
    const int c0 = g * kE - shift;
    if (c0 >= 0 && c0 + kE <= V) return *reinterpret_cast<const uint4*>(base + c0);
    T each[kE];
#pragma unroll
    for (int j = 0; j < kE; ++j) {
      if (c0 + j >= 0 && c0 + j < V)
        each[j] = base[c0 + j];
      else
        store1(each + j, -INFINITY);
    }
    uint4 q;
    memcpy(&q, each, 16);
    return q;
  }
  __device__ __forceinline__ static void values(const uint4& q, float (&v)[kE]) {
    f32x2 pair[kE / 2];
    pairs_of<T>(q, pair);
#pragma unroll
    for (int j = 0; j < kE / 2; ++j) {
      const float2 x = unpack2(pair[j]);
      v[2 * j] = x.x;
      v[2 * j + 1] = x.y;
    }
  }
  __device__ __forceinline__ bool inside(int col) const { return col >= 0 && col < V; }
};

// The barrier of the warps that select.
__device__ __forceinline__ void sync_selectors() {
  __syncwarp();
  asm volatile("barrier.sync 2, %0;" ::"n"(kSelThreads) : "memory");
}

// The columns behind the place `last` of the k-th: their maximum m, and the sum of exp((z - m) / T).
template <typename T>
__device__ float2 rest_of(const Row<T>& row, unsigned long long last, float inv_t, int st, float (*red)[32]) {
  constexpr int kE = Row<T>::kE;
  const int lane = st & 31, warp = st >> 5, warps = kSelWarps;
  float m = -INFINITY;
  bool nan = false;
  for (int g = st; g < row.groups; g += kSelThreads) {
    float v[kE];
    Row<T>::values(row.load(g), v);
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
  nan = __any_sync(0xffffffffu, nan);
  sync_selectors();
  if (lane == 0) red[0][warp] = nan ? NAN : m;
  sync_selectors();
  nan = false;
  for (int w = 0; w < warps; ++w) {
    nan |= red[0][w] != red[0][w];
    m = fmaxf(m, red[0][w]);
  }
  float s = 0.0f;
  if (m > -INFINITY && m < INFINITY) {
    for (int g = st; g < row.groups; g += kSelThreads) {
      float v[kE];
      Row<T>::values(row.load(g), v);
#pragma unroll
      for (int j = 0; j < kE; ++j) {
        const int col = g * kE - row.shift + j;
        if (row.inside(col) && place_of(v[j], col) < last) s += ex2((v[j] - m) * (inv_t * kLog2E));
      }
    }
  }
  s = warp_sum(s);
  if (lane == 0) red[1][warp] = s;
  sync_selectors();
  s = 0.0f;
  for (int w = 0; w < warps; ++w) s += red[1][w];
  sync_selectors();
  if (nan) return make_float2(INFINITY, NAN);
  return make_float2(m, m == INFINITY ? 1.0f : s);
}

// The k-th largest (value, column) place by the keys' digits from the top; leaves the k best in `kept` (any order).
template <typename T>
__device__ void select_by_digits(const Row<T>& row, int k, int tid, unsigned long long* kept, int* hist, int* shared) {
  constexpr int kE = Row<T>::kE;
  const int lane = tid & 31, warp = tid >> 5;
  uint32_t prefix = 0;
  int need = k;
  constexpr int kDigits = sizeof(T);  // bf16 keys are settled by their upper 16 bits
#pragma unroll 1
  for (int digit = 0; digit < kDigits; ++digit) {
    const int down = 24 - 8 * digit;
    for (int i = tid; i < 256; i += kSelThreads) hist[i] = 0;
    sync_selectors();
    for (int g = tid; g < row.groups; g += kSelThreads) {
      float v[kE];
      Row<T>::values(row.load(g), v);
#pragma unroll
      for (int j = 0; j < kE; ++j) {
        const uint32_t key = key_of(v[j]);
        if (row.inside(g * kE - row.shift + j) && (digit == 0 || key >> (down + 8) == prefix))
          atomicAdd(hist + ((key >> down) & 255), 1);
      }
    }
    sync_selectors();
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
    sync_selectors();
    prefix = prefix << 8 | static_cast<uint32_t>(shared[0]);
    need = shared[1];
    sync_selectors();
  }
  // everything above the k-th key, and the first `need` columns that hold it
  if (tid == 0) shared[0] = shared[1] = 0;
  sync_selectors();
  constexpr int kDown = 32 - 8 * kDigits;
  for (int g0 = 0; g0 < row.groups; g0 += kSelThreads) {
    const int g = g0 + tid;
    float v[kE];
    int equal = 0;
    if (g < row.groups) {
      Row<T>::values(row.load(g), v);
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
    sync_selectors();
    int before = shared[1] + upto - equal, all = 0;
    for (int w = 0; w < kSelWarps; ++w) {
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
    sync_selectors();
    if (tid == 0) shared[1] += all;
    sync_selectors();
  }
}

// log of s exp(m / T); s = 0 for nothing, and for an infinite m whatever it is (NaN stays NaN).
__device__ __forceinline__ float log_sum(float2 r, float inv_t) { return r.x > -INFINITY && r.x < INFINITY ? r.x * inv_t + logf(r.y) : r.x + 0.0f * r.y; }

// One object, whose address inline assembly gets: waits there may change any part of it. What belongs to a row is there
// twice and taken in turns: warps of the block may be in neighbouring rows, and the selection of a row goes on while the
// next one is read.
struct Shared {
  RowQueue queue;
  unsigned long long bars[kWarps + 11];
  unsigned long long kept[2][kRoom], last;
  alignas(16) int hist[2][kBins];
  float sums[2][kWarps];
  uint32_t top[2];  // the largest key
  int found[2], next[2];
  struct {
    int row;  // or -1: there is no further one
    float low, power;
    bool by_digits;
  } work[2];
  struct {
    int row;
    float edge[16];
  } ahead[3];  // rows to come, with the elements at their ragged ends
  // the selecting warps'
  int bins[kSelBins + 1], pair[2], row;
  uint32_t ends[2][kSelWarps];
  float red[2][32];
  int abort_flag;
};
constexpr int kShared = 14848;
static_assert(sizeof(Shared) <= kShared);

// The selection of the rows that a cluster has read: its first block's selecting warps, thread st of them; one warp of the
// other blocks says when theirs have been. (An arrival at another block's barrier takes up to 2 us to get past what its
// thread has seen stored: not the warps that read rows do it.)
template <typename T>
__device__ void select_rows(Shared& sh, const RowSlice<T>& rows, int cs, int k, float inv_t, T* values, int* indices,
                            float* tail, int* status, uint32_t collected_bar, uint32_t selected_bar, uint32_t gathered_bar, int rank,
                            int st) {
  const int lane = st & 31, sw = st >> 5;
  const float c = inv_t * kLog2E;
  for (int n = 0;; ++n) {
    const int turn = n & 1;
    if (sw == 0) {  // all of them go on, or none does
      const uint32_t phase = (n >> 1) & 1;
      bool in_time = short_wait<false>(collected_bar + 8 * turn, phase, &sh.abort_flag);
      const int next = in_time ? sh.work[turn].row : -1;
      if (cs > 1) {
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(mapa_shared(gathered_bar + 8 * turn, 0));
        __syncwarp();
        if (rank == 0) in_time &= short_wait<true>(gathered_bar + 8 * turn, phase, &sh.abort_flag);
      }
      if (!in_time && status != nullptr) atomicCAS(status, 0, kTimeoutProducer);
      if (lane == 0) sh.row = in_time ? next : -1;
      __syncwarp();
      if (rank != 0 && next < 0) break;
    }
    if (rank != 0) continue;
    sync_selectors();
    const int r = sh.row;
    if (r < 0) break;
    const float low = sh.work[turn].low, power = sh.work[turn].power;
    bool by_digits = sh.work[turn].by_digits;
    const Row<T> row(rows.row(r), rows.V);
    unsigned long long* const kept = sh.kept[turn];
    float sum = 0.0f, over = 0.0f;
    int collected = 0;
    if (!by_digits) {
      if (cs == 1) {
        collected = sh.found[turn];
        for (int w = 0; w < kWarps; ++w) sum += sh.sums[turn][w];
      } else {
        // every warp reads all counts and sums for itself, then its share of the lists
        const uint32_t there = mapa_shared(smem_u32(&sh), lane & 7);  // of block lane, where there is one
        auto of = [&](const void* x) { return there + (smem_u32(x) - smem_u32(&sh)); };
        const int count = lane < cs ? static_cast<int>(load_cluster_u32(of(sh.found + turn))) : 0;
        if (lane < cs)
          for (int w = 0; w < kWarps; ++w) sum += __uint_as_float(load_cluster_u32(of(sh.sums[turn] + w)));
        sum = warp_sum(sum);
        int upto = count;
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) {
          const int v = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= o) upto += v;
        }
        collected = __shfl_sync(0xffffffffu, upto, 7);
        for (int b = 1 + sw; b < cs; b += kSelWarps) {
          const int mine = __shfl_sync(0xffffffffu, count, b), at = __shfl_sync(0xffffffffu, upto, b) - mine;
          const uint32_t list = mapa_shared(smem_u32(kept), b);
          for (int i = lane; i < mine && at + i < kRoom; i += 32) kept[at + i] = load_cluster_u64(list + 8 * i);
        }
        sync_selectors();
      }
    }
    by_digits |= collected > kRoom;
    if (by_digits) {
      select_by_digits(row, k, st, kept, sh.bins, sh.pair);
      collected = k;
    } else {
      const float taken = static_cast<float>(collected) * ex2(fmaf(low, c, -power));
      over = sum < 1.0625f * taken ? INFINITY : 0.0f;  // too little is left of it
      sum = (sum - taken) * ex2(fmaf(-low, c, power));  // relative to exp(low / T) from here on
    }
    // Places: sorted into 256 bins by key, each then counted within its bin. Every place differs from every other.
    constexpr int kOwn = kRoom / kSelThreads;
    unsigned long long own[kOwn];
    uint32_t hi = 0, lo = 0xFFFFFFFFu;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      const int at = st + i * kSelThreads;
      own[i] = at < collected ? kept[at] : 0ull;
      if (at < collected) {
        const uint32_t key = static_cast<uint32_t>(own[i] >> 32);
        hi = max(hi, key);
        lo = min(lo, key);
      }
    }
    hi = __reduce_max_sync(0xffffffffu, hi);
    lo = __reduce_min_sync(0xffffffffu, lo);
    if (lane == 0) {
      sh.ends[0][sw] = hi;
      sh.ends[1][sw] = lo;
    }
    for (int i = st; i < kSelBins; i += kSelThreads) sh.bins[i] = 0;
    sync_selectors();
#pragma unroll
    for (int w = 0; w < kSelWarps; ++w) {
      hi = max(hi, sh.ends[0][w]);
      lo = min(lo, sh.ends[1][w]);
    }
    const int down = max(0, 24 - __clz(hi - lo));
    int bin[kOwn], before[kOwn];
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      bin[i] = static_cast<int>((hi - static_cast<uint32_t>(own[i] >> 32)) >> down);
      before[i] = st + i * kSelThreads < collected ? atomicAdd(sh.bins + bin[i], 1) : 0;
    }
    sync_selectors();
    if (sw == 0) {  // counts become the places at which bins begin
      int count[kSelBins / 32], all = 0;
#pragma unroll
      for (int j = 0; j < kSelBins / 32; ++j) {
        count[j] = sh.bins[kSelBins / 32 * lane + j];
        all += count[j];
      }
      int upto = all;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
      }
      int begin = upto - all;
#pragma unroll
      for (int j = 0; j < kSelBins / 32; ++j) {
        sh.bins[kSelBins / 32 * lane + j] = begin;
        begin += count[j];
      }
      if (lane == 31) sh.bins[kSelBins] = begin;
    }
    sync_selectors();
#pragma unroll
    for (int i = 0; i < kOwn; ++i)
      if (st + i * kSelThreads < collected) kept[sh.bins[bin[i]] + before[i]] = own[i];
    sync_selectors();
    float more[kOwn];
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      more[i] = 0.0f;
      before[i] = 0;
      if (st + i * kSelThreads < collected) {
        const int from = sh.bins[bin[i]], to = sh.bins[bin[i] + 1];
        int place = from;
        for (int j = from; j < to; ++j) place += kept[j] > own[i];
        if (place < k) {
          const long long at = static_cast<long long>(r) * k + place;
          store1(values + at, logit_of(own[i]));
          indices[at] = column_of(own[i]);
          if (place == k - 1) sh.last = own[i];
        } else {
          more[i] = ex2((logit_of(own[i]) - low) * c);  // collected, but not among the k
        }
        before[i] = place;
      }
    }
    sync_selectors();
    // What is left: the sum relative to the bound with the collected ones that did not make it, added in the order of
    // their places, not of their arrival.
    float* const terms = reinterpret_cast<float*>(kept);
#pragma unroll
    for (int i = 0; i < kOwn; ++i)
      if (before[i] >= k) terms[before[i] - k] = more[i];
    sync_selectors();
    float added = 0.0f;
    for (int i = lane; i < collected - k; i += 32) added += terms[i];
    over += warp_sum(added);  // every warp for itself
    float2 result = make_float2(low, sum + over);
    if (by_digits || !(over < 1e30f)) result = rest_of(row, sh.last, inv_t, st, sh.red);
    if (st == 0) tail[r] = log_sum(result, inv_t);
    sync_selectors();
    if (st == 0) mbar_arrive(selected_bar + 8 * turn);
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads + 32 + kSelThreads, 2) top_logits_kernel(const T* __restrict__ z, long long ld, int V, int k,
                                                                      float inv_t, SlicePlan plan, T* __restrict__ values,
                                                                      int* __restrict__ indices, float* __restrict__ tail,
                                                                      int* __restrict__ status) {
  constexpr int kE = Row<T>::kE;
  extern __shared__ __align__(128) uint8_t smem[];  // the slice; behind it, in a cluster, [2][cs][kMaxima] maxima
  __shared__ __align__(16) Shared sh;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, cs = plan.cs;
  const int rank = cs > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const RowSlice<T> rows{z, ld, V, rank * plan.slice, plan.slice, plan.per};
  unsigned short* maxima = reinterpret_cast<unsigned short*>(smem + 16ll * plan.slice);
  T* buf = reinterpret_cast<T*>(smem);
  const float c = inv_t * kLog2E;
  const uint32_t bar0 = smem_u32(sh.bars), ready = bar0 + 8 * kWarps, done = ready + 16, selected = ready + 32,
                 collected = ready + 48, met = ready + 64;
  if (tid == 0) {
    for (int i = 0; i < kWarps + 6; ++i) mbar_init(bar0 + 8 * i, 1);
    for (int i = 0; i < 2; ++i) mbar_init(collected + 8 * i, kWarps);
    for (int i = 0; i < 3; ++i) mbar_init(met + 8 * i, cs);  // and `gathered`
    sh.queue.init();
    sh.abort_flag = 0;
    sh.top[0] = sh.top[1] = 0;
    mbar_fence_init();
  }
  __syncthreads();
  if (cs > 1) cluster_sync_all();  // every block of the cluster runs before another one stores to its shared memory
  auto late = [&](bool in_time) {
    if (!in_time && status != nullptr) atomicCAS(status, 0, kTimeoutProducer);
  };
  // The n-th completion of a pair of barriers that take turns.
  auto wait_pair = [&](uint32_t pair, int n) { return short_wait<false>(pair + 8 * (n & 1), (n >> 1) & 1, &sh.abort_flag); };
  if (warp > kWarps) {
    if (rank == 0 || warp == kWarps + 1)
      select_rows(sh, rows, cs, k, inv_t, values, indices, tail, status, collected, selected, met + 8, rank, tid - kThreads - 32);
  } else if (warp == kWarps) {  // rows to come, two ahead
    bool more = true;
    if (rank == 0 && lane == 0) sh.queue.ask();
    __syncwarp();
    for (int n = 0;; ++n) {
      int row = -1;
      if (n == 0) {
        row = blockIdx.x / cs;
      } else if (more) {
        bool in_time = true;
        row = sh.queue.take(n, rank, cs, lane, &sh.abort_flag, in_time);
        late(in_time);
        if (row >= 0 && rank == 0 && lane == 0) sh.queue.ask();
        __syncwarp();
      }
      more = row >= 0;
      float edge = -INFINITY;
      if (more && lane < 2 * kE) {
        int col;
        if (rows.edge_place(lane, rows.shift(row), col) >= 0 && col >= 0 && col < V) edge = as_float(rows.row(row)[col]);
      }
      if (n >= 2) late(wait_pair(done, n - 2));  // all warps have been past the first barrier of that row
      if (lane < 2 * kE) sh.ahead[n % 3].edge[lane] = edge;
      if (lane == 0) sh.ahead[n % 3].row = row;
      __syncwarp();
      if (lane == 0) mbar_arrive(ready + 8 * (n & 1));
      __syncwarp();
      if (!more) break;
    }
  } else {
    if (lane == 0) rows.request(blockIdx.x / cs, warp, smem, bar0 + 8 * warp, false);
    __syncwarp();
    late(wait_pair(ready, 0));
    auto hand_over = [&](int n) {  // the warp, to the selecting warps
      __syncwarp();
      if (lane == 0) mbar_arrive(collected + 8 * (n & 1));
      __syncwarp();
    };
    int n = 0;
    for (int r = blockIdx.x / cs; r >= 0; ++n) {
      const int turn = n & 1;
      const int shift = rows.shift(r), groups = rows.groups(shift);
      const int begin = warp * plan.per + lane, stop = min(groups, (warp + 1) * plan.per);
      late(short_wait<false>(bar0 + 8 * warp, n & 1, &sh.abort_flag));
      // a ragged end is written by the warp that reads it
      if (warp == 0 || stop == groups) {
        int col;
        const int at = lane < 2 * kE ? rows.edge_place(lane, shift, col) : -1;
        if (at >= 0 && at / kE >= warp * plan.per && at / kE < stop) store1(buf + at, sh.ahead[n % 3].edge[lane]);
        fence_proxy_async_smem();  // before bulk copies of the next row write there
        __syncwarp();
      }
      bool by_digits = min(kMaxima, (shift + V + kE - 1) / kE) < 2 * k;  // from sizes alone: the same in every block
      float low = 0.0f, power = 0.0f;
      uint32_t keys = 0;
      int* const hist = sh.hist[turn];
      if (!by_digits) {
        GroupMax<T> m0, m1;
        int g = begin;
#pragma unroll 4
        for (; g + 32 < stop; g += 64) {
          m0.add(*reinterpret_cast<const uint4*>(smem + 16 * g));
          m1.add(*reinterpret_cast<const uint4*>(smem + 16 * (g + 32)));
        }
        if (g < stop) m0.add(*reinterpret_cast<const uint4*>(smem + 16 * g));
        keys = key_of(m0.value()) >> 16 | (key_of(m1.value()) & 0xFFFF0000u);
        if (cs > 1) {
          const uint32_t local = smem_u32(maxima + (turn * cs + rank) * kMaxima + 2 * tid);
          for (int b = 0; b < cs; ++b)
            asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(mapa_shared(local, b)), "r"(keys) : "memory");
        } else {
          const uint32_t most = __reduce_max_sync(0xffffffffu, max(keys >> 16, keys & 0xFFFFu));
          if (lane == 0) atomicMax(sh.top + turn, most);
        }
        hist[tid] = hist[tid + kThreads] = 0;
      }
      if (warp == 0) {  // the whole of it: a lane that waits by itself leaves the warp split in two for the rest of the kernel
        late(wait_pair(ready, n + 1));
        if (rank == 0 && n >= 2) late(wait_pair(selected, n - 2));  // the list of two rows ago has been read
      }
      if (tid == 0) {  // all warps go on together, or none does: what the barrier below shows them decides
        if (cs == 1) sh.found[turn] = 0;
        sh.next[turn] = *static_cast<volatile int*>(&sh.abort_flag) ? -1 : sh.ahead[(n + 1) % 3].row;
      }
      sync_first(kThreads);
      const int next = sh.next[turn];
      if (tid == 0) sh.top[turn ^ 1] = 0;
      if (!by_digits) {
        if (cs > 1) {
          if (warp == 0 && lane < cs) mbar_arrive_cluster(mapa_shared(met, lane));
          __syncwarp();
          late(short_wait<true>(met, n & 1, &sh.abort_flag));
          for (int b = 0; b < cs; ++b) keys = __vmaxu2(keys, reinterpret_cast<const uint32_t*>(maxima + (turn * cs + b) * kMaxima)[tid]);
          const uint32_t most = __reduce_max_sync(0xffffffffu, max(keys >> 16, keys & 0xFFFFu));
          if (lane == 0) atomicMax(sh.top + turn, most);
          if (tid == 0) sh.found[turn] = 0;  // the first block has come to this row: it has read the list of two rows ago
          sync_first(kThreads);
        }
        // The k-th largest of the maxima in the upper 16 bits of its key, rounded down: by a histogram of their distances
        // from the largest, 512 of them (4 octaves); where that does not reach far enough (a bound near zero or below it, under
        // a positive maximum), by one of 128 distances a bin and another one of the distances in the bin that was found.
        const uint32_t top = sh.top[turn];
        uint32_t bound, from = 0;
        int need = k;
        for (int level = 0;; ++level) {
          const int down = level == 1 ? 7 : 0;
          const uint32_t stop_at = level == 2 ? 128u : 0x10000u;  // distances past `from` that count
          auto note = [&](uint32_t key) {
            const uint32_t past = top - key - from;  // wraps below `from`
            if (past < stop_at) atomicAdd(hist + min(kBins - 1u, past >> down), 1);
          };
          note(keys >> 16);
          note(keys & 0xFFFFu);
          sync_first(kThreads);
          int count[kBins / 32], total = 0;  // every warp for itself
#pragma unroll
          for (int i = 0; i < kBins / 128; ++i) {
            const int4 q = reinterpret_cast<const int4*>(hist)[kBins / 128 * lane + i];
            count[4 * i] = q.x, count[4 * i + 1] = q.y, count[4 * i + 2] = q.z, count[4 * i + 3] = q.w;
            total += q.x + q.y + q.z + q.w;
          }
          int upto = total;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
          }
          const int holder = __ffs(__ballot_sync(0xffffffffu, upto >= need)) - 1;  // kMaxima >= 2 k: there is one
          int before = upto - total, bin = 0;
#pragma unroll
          for (int i = 0; i < kBins / 32; ++i) {
            if (before + count[i] < need) {
              before += count[i];
              ++bin;
            } else {
              break;
            }
          }
          before = __shfl_sync(0xffffffffu, before, holder);
          bin = __shfl_sync(0xffffffffu, kBins / 32 * lane + min(bin, kBins / 32 - 1), holder);
          if (level == 2 || (level == 0 && bin < kBins - 1)) {
            const uint32_t reach = from + bin;
            bound = reach < top ? top - reach : 0;
            break;
          }
          if (level == 1) {
            from = static_cast<uint32_t>(bin) << 7;
            need -= before;
          }
          sync_first(kThreads);
          hist[tid] = hist[tid + kThreads] = 0;
          sync_first(kThreads);
        }
        low = value_of(bound << 16);
        if (sizeof(T) == 2) low = __uint_as_float(__float_as_uint(low) & 0xFFFF0000u);  // the bf16 number of that key
        // Sums are relative to 2^power, so that one fused multiply-add gives an exponent.
        power = rintf(low * c);
        by_digits = !(fabsf(power) < 1.0e6f);
        if (!by_digits) {
          const f32x2 c2 = pk2(c, c), k2 = pk2(-power, -power);
          const uint32_t low_bits = __float_as_uint(low), low_word = sizeof(T) == 2 ? low_bits >> 16 | low_bits : low_bits;
          f32x2 s0 = 0ull, s1 = 0ull;
          // groups that hold a logit to collect are noted, and looked into when the sums are done
          unsigned long long noted = 0ull, bit = 1ull;
#pragma unroll 4
          for (int g = begin; g < stop; g += 32) {
            const uint4 q = *reinterpret_cast<const uint4*>(smem + 16 * g);
            if (!below<T>(most<T>(q), low)) noted |= bit;
            bit <<= 1;
            f32x2 v[kE / 2];
            pairs_of<T>(make_uint4(cut_off<T>(q.x, low_word), cut_off<T>(q.y, low_word), cut_off<T>(q.z, low_word),
                                   cut_off<T>(q.w, low_word)),
                        v);
#pragma unroll
            for (int j = 0; j < kE / 2; ++j) {
              const float2 x = unpack2(fma2(v[j], c2, k2));
              const f32x2 e = pk2(ex2(x.x), ex2(x.y));
              if (j & 1)
                s1 = add2(s1, e);
              else
                s0 = add2(s0, e);
            }
          }
          for (; noted != 0; noted &= noted - 1) {
            const int g = begin + 32 * (__ffsll(noted) - 1);
            for (uint32_t bits = reached<T>(*reinterpret_cast<const uint4*>(smem + 16 * g), low); bits != 0; bits &= bits - 1) {
              const int j = __ffs(bits) - 1, col = (rows.g0 + g) * kE - shift + j;
              const int at = col >= 0 && col < V ? atomicAdd(sh.found + turn, 1) : kRoom;
              if (at < kRoom) sh.kept[turn][at] = place_of(as_float(buf[g * kE + j]), col);
            }
          }
          const float2 a = unpack2(add2(s0, s1));
          const float sum = warp_sum(a.x + a.y);
          if (lane == 0) sh.sums[turn][warp] = sum;
        }
      }
      __syncwarp();
      if (lane == 0 && next >= 0) {  // the warp's part of the next row
        fence_proxy_async_smem();
        rows.request(next, warp, smem, bar0 + 8 * warp, false);
      }
      __syncwarp();
      if (tid == 0) {
        sh.work[turn].row = r;
        sh.work[turn].low = low;
        sh.work[turn].power = power;
        sh.work[turn].by_digits = by_digits;
      }
      hand_over(n);
      if (tid == 0) mbar_arrive(done + 8 * (n & 1));
      __syncwarp();
      r = next;
    }
    // Before the end is written over the entry of two rows ago the cluster meets as it does in every row: the first block has
    // waited for that row's selection, so the warps that relay, and the barriers they arrive on, are past it in all blocks.
    if (warp == 0) {
      if (rank == 0 && n >= 2) late(wait_pair(selected, n - 2));
      if (cs > 1) {
        if (lane < cs) mbar_arrive_cluster(mapa_shared(met, lane));
        __syncwarp();
        late(short_wait<true>(met, n & 1, &sh.abort_flag));
      }
    }
    if (tid == 0) sh.work[n & 1].row = -1;
    hand_over(n);
  }
  __syncwarp();
  if (cs > 1) cluster_sync_all();  // no block leaves while another one may still read from it or store to it
}

// A slice beside the fixed shared memory and 1 KB of the system's: two blocks an SM; one, with a cluster's maxima beside it.
constexpr long long kMaximaBytes = 2 * 8 * kMaxima * 2;
constexpr long long kHalfSm = 113 * 1024 - kShared, kWholeSm = 227 * 1024 - kShared - kMaximaBytes;

template <typename T>
int top(const void* z, long long rows, int V, long long ld, int k, float inv_t, void* values, int* indices, float* tail,
        int* status, cudaStream_t st) {
  const SlicePlan plan = slice_plan<T>(V, kWarps, kHalfSm, kWholeSm, 2 * kMaxima * 2);
  if (plan.cs == 0) return 5;
  const int smem = plan.slice * 16 + (plan.cs > 1 ? 2 * plan.cs * kMaxima * 2 : 0);
  auto kern = top_logits_kernel<T>;
  static std::atomic<unsigned long long> asked{0};
  if (!make_room(asked, reinterpret_cast<const void*>(kern), kWholeSm + kMaximaBytes)) return 2;
  return launch_clusters(kern, rows, plan.cs, kThreads + 32 + kSelThreads, smem, st, static_cast<const T*>(z), ld, V, k, inv_t, plan,
                         static_cast<T*>(values), indices, tail, status);
}

}  // namespace

// Widest row that a cluster holds.
extern "C" long long pd_top_logits_max_columns(int z_fp32) { return 8 * kWholeSm / (z_fp32 ? 4 : 2) - 16; }

// z [rows, V] in bf16 or fp32, rows ld elements apart; values, indices [rows, k], tail [rows].
extern "C" int pd_top_logits(const void* z, long long rows, int V, long long ld, int k, float inv_t, void* values,
                             int* indices, float* tail, int z_fp32, int* status, void* stream) {
  if (rows <= 0 || rows >= (1ll << 28) || V <= 0 || k <= 0 || k > kMaxK || k > V || !(inv_t > 0.0f)) return 5;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return z_fp32 ? top<float>(z, rows, V, ld, k, inv_t, values, indices, tail, status, st)
                : top<__nv_bfloat16>(z, rows, V, ld, k, inv_t, values, indices, tail, status, st);
}
