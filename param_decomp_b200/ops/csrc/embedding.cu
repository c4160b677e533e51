// Token embedding: y[n] = scale E[t_n], and its gradient dE[v] = scale sum over n with t_n = v of dy[n].
// Both are bound by HBM: the lookup reads a table row and writes an output row a token, the gradient reads the tokens'
// rows once and writes every row of the table (most of them zeros).
//
// The gradient sums each row in fp32 over its tokens in a fixed order and rounds once, with two launches and no float
// atomics. First kernel: ids are dealt to the blocks like cards (id v is the v / blocks -th of block v % blocks), since
// vocabularies hold frequent tokens together: with a span of neighbouring ids a block, 32,768 tokens over 50,277 ids in
// order of frequency took 270 us, so 56 (58 with ids in no order, either way). A block's 32 warps read all tokens (from L2,
// as the lookup left them in 32 bits), each its own consecutive part, note those of the block and count those of the blocks
// before it, which gives the block's place in the sorted order without asking them. The noted ones are sorted by counting: id,
// then warp, then position, and rows of up to kSlab tokens are summed. Second kernel: ids with more tokens, in slabs of
// kSlab places of the sorted order, so a token that fills a tenth of the batch is shared by many blocks; a slab's sum goes
// to scratch and the block that finishes a run last adds its slabs in their order. Rows of dy come in no order that a cache
// could guess, so the block that finds a token asks for its row in L2 at once, long before it is summed. The rows without a
// token, most of the bytes, are written by blocks of the second kernel too: zeros at the full rate in the first one made the
// loads of its sums wait for several microseconds each (32,768 tokens in 50,277 rows of 768: 77 us).
// Measured there, bf16: lookup 15.6 us (6.4 TB/s by a row a token, most of them from L2), first kernel 34, second 25: 78 us with the launches. 6151
// tokens in 151,936 rows of 515 fp32: 11, 26 and 57. The first kernel is a chain of steps, each with its own latency, over
// all tokens in every block; what the second has to write takes 12 and 48 us of it.
#include <algorithm>

#include "rows.cuh"

namespace {

using namespace pd;

constexpr int kSlab = 32;
constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kMaxSpan = 1280;  // ids a block: 32 counts of 4 bytes each in shared memory
constexpr int kNoted = 128;     // tokens a warp notes; where there are more, it reads its part again
// Rows a warp asks for in L2 while it reads tokens, the first it finds: where a token fills a tenth of the batch, its block
// would be busy asking (30,000 cycles for 9,000; 32,768 tokens: 61 us without a limit, 58 at 32 and 16, 59 at 8).
constexpr int kAhead = 32;
constexpr int kRunThreads = 384;
constexpr int kMaxPer = 512;  // ids of a block that writes zeros

__device__ __forceinline__ long long token_at(const void* tokens, int wide, long long i) {
  return wide ? static_cast<const long long*>(tokens)[i] : static_cast<const int*>(tokens)[i];
}

// ---- lookup ------------------------------------------------------------------------------------------------------
// A warp takes kRowsAhead tokens at a time, so that many loads are in flight before the first is needed.
template <typename P, typename T, bool kVec>
__global__ void __launch_bounds__(256) embedding_lookup_kernel(const void* __restrict__ tokens, int wide,
                                                               const P* __restrict__ table, T* __restrict__ y,
                                                               int* __restrict__ ids, long long n, long long V, int d,
                                                               float scale, int* __restrict__ status,
                                                               int* __restrict__ refused) {
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
      if (lane == 0 && ids != nullptr && r0 + k < n) ids[r0 + k] = known ? static_cast<int>(t) : -1;
    }
    if (bad && lane == 0) {
      atomicCAS(status, 0, kBadToken);
      *static_cast<volatile int*>(refused) = 1;
    }
    constexpr int kColumns = kVec ? 1 : 4;  // of a lane, 32 apart, where it loads one at a time
    for (int c = kVec ? 8 * lane : lane; c < d; c += kVec ? 256 : 32 * kColumns) {
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
        float v[kRowsAhead][kColumns];
#pragma unroll
        for (int k = 0; k < kRowsAhead; ++k)
#pragma unroll
          for (int j = 0; j < kColumns; ++j)
            v[k][j] = src[k] != nullptr && c + 32 * j < d ? as_float(src[k][c + 32 * j]) : 0.0f;
#pragma unroll
        for (int k = 0; k < kRowsAhead; ++k)
#pragma unroll
          for (int j = 0; j < kColumns; ++j)
            if (r0 + k < n && c + 32 * j < d) store1(y + (r0 + k) * d + c + 32 * j, v[k][j] * scale);
      }
    }
  }
}

// ---- gradient ----------------------------------------------------------------------------------------------------
struct Runs {        // what the first kernel tells the second
  int* order;        // [n] position of the token at each place of the sorted order, where its id has more than kSlab
  int* run_start;    // [n] place where the run of an id with more than kSlab tokens starts, at each of its places; else -1
  int* id;           // [slabs] of the run that starts in the slab (a longer run than a slab: at most one does)
  int* end;          // [slabs] place behind it
  int* done;         // [slabs] slabs of it that are summed
  uint8_t* empty;    // [V] the id has no token
};

// A block: zeros in those rows [from, to) of the table's gradient that have no token. All of them as one stretch of 16-byte
// pieces, whatever the rows' own alignment: rows of 515 fp32 begin at any of them.
template <typename P>
__device__ void write_zeros(P* __restrict__ dE, int from, int to, int d, const uint8_t* __restrict__ is_empty,
                            uint8_t* empty) {
  constexpr int kE = 16 / sizeof(P);
  for (int i = threadIdx.x; i < to - from; i += kRunThreads) empty[i] = is_empty[from + i];
  __syncthreads();
  P* const base = dE + static_cast<long long>(from) * d;
  const long long total = static_cast<long long>(to - from) * d;
  const long long head = min(total, static_cast<long long>((16 - (reinterpret_cast<uintptr_t>(base) & 15)) % 16 / sizeof(P)));
  const long long pieces = (total - head) / kE, tail = head + pieces * kE;
  const long long edge = threadIdx.x < kE ? threadIdx.x : tail + threadIdx.x - kE;
  if (threadIdx.x < kE ? edge < head : edge < total && threadIdx.x < 2 * kE)
    if (empty[edge / d]) store1(base + edge, 0.0f);
  long long e = head + static_cast<long long>(kE) * threadIdx.x;
  constexpr int kStep = kE * kRunThreads;
  int row = static_cast<int>(e / d), rem = static_cast<int>(e % d);
  for (long long p = threadIdx.x; p < pieces; p += kRunThreads, e += kStep) {
    const bool inside = rem + kE <= d;
    if (inside || d >= kE ? empty[row] && (inside || empty[row + 1]) : false) {
      *reinterpret_cast<uint4*>(base + e) = make_uint4(0u, 0u, 0u, 0u);
    } else if (!inside) {
      for (int j = 0, r = row, m = rem; j < kE; ++j) {
        if (empty[r]) store1(base + e + j, 0.0f);
        if (++m == d) m = 0, ++r;
      }
    }
    row += kStep / d;
    rem += kStep % d;
    if (rem >= d) rem -= d, ++row;
  }
}

// One warp: scale times rows of dy, each in one piece of 256 columns; lane u names the u-th row, its place in the table and
// its first column (d: none). All of their loads are in flight together.
constexpr int kItems = 4;
template <typename T, typename P, bool kVec>
__device__ __forceinline__ void copy_rows(const T* __restrict__ dy, P* __restrict__ dE, int from, int to, int c0, int d,
                                          float scale, int lane) {
  Raw8<T> raw[kVec ? kItems : 1];
  float v[kVec ? 1 : kItems][8];
#pragma unroll
  for (int u = 0; u < kItems; ++u) {
    const T* row = dy + static_cast<long long>(__shfl_sync(0xffffffffu, from, u)) * d;
    const int col = __shfl_sync(0xffffffffu, c0, u) + (kVec ? 8 * lane : lane);
    if constexpr (kVec) {
      if (col < d) raw[u] = load8(row + col);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[u][j] = col + 32 * j < d ? as_float(row[col + 32 * j]) : 0.0f;
    }
  }
#pragma unroll
  for (int u = 0; u < kItems; ++u) {
    P* out = dE + static_cast<long long>(__shfl_sync(0xffffffffu, to, u)) * d;
    const int col = __shfl_sync(0xffffffffu, c0, u) + (kVec ? 8 * lane : lane);
    if constexpr (kVec) {
      float e[8];
      if (col < d) {
        unpack8(raw[u], e);
#pragma unroll
        for (int j = 0; j < 8; ++j) e[j] *= scale;
        store8(out + col, e);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (col + 32 * j < d) store1(out + col + 32 * j, v[u][j] * scale);
    }
  }
}

// One warp: scale times the sum of k rows of dy, the r-th at lane r's `row_of`, over 256 columns from c0; the loads of eight
// bf16 rows or four fp32 rows are in flight (two, element by element, where rows are not of 16-byte pieces).
template <typename T, typename P, bool kVec>
__device__ __forceinline__ void sum_rows(const T* __restrict__ dy, int row_of, int k, P* out, int c0, int d, float scale,
                                         int lane) {
  constexpr int kRows = kVec ? 16 / sizeof(T) : 2;
  const int col = kVec ? c0 + 8 * lane : c0 + lane;
  float acc[8] = {};
#pragma unroll 1
  for (int r = 0; r < k; r += kRows) {
    Raw8<T> raw[kVec ? kRows : 1];
    float v[kVec ? 1 : kRows][8];
#pragma unroll
    for (int u = 0; u < kRows; ++u) {
      const T* row = dy + static_cast<long long>(__shfl_sync(0xffffffffu, row_of, min(r + u, k - 1))) * d;
      if constexpr (kVec) {
        if (col < d && r + u < k) raw[u] = load8(row + col);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[u][j] = col + 32 * j < d && r + u < k ? as_float(row[col + 32 * j]) : 0.0f;
      }
    }
#pragma unroll
    for (int u = 0; u < kRows; ++u) {
      if constexpr (kVec) {
        if (col < d && r + u < k) {
          float e[8];
          unpack8(raw[u], e);
#pragma unroll
          for (int j = 0; j < 8; ++j) acc[j] += e[j];
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[j] += v[u][j];
      }
    }
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) acc[j] *= scale;
  if constexpr (kVec) {
    if (col < d) store8(out + col, acc);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (col + 32 * j < d) store1(out + col + 32 * j, acc[j]);
  }
}

// Asks for a row's whole 16-byte pieces in L2.
template <typename T>
__device__ __forceinline__ void fetch_to_l2(const T* row, int d) {
  const uintptr_t from = (reinterpret_cast<uintptr_t>(row) + 15) & ~static_cast<uintptr_t>(15);
  const uintptr_t to = reinterpret_cast<uintptr_t>(row + d) & ~static_cast<uintptr_t>(15);
  if (to > from)
    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(from), "r"(static_cast<uint32_t>(to - from)) : "memory");
}

template <typename T, typename P, bool kVec>
__global__ void __launch_bounds__(kSortThreads, 1) embedding_sort_kernel(const int* __restrict__ ids_of,
                                                                         const T* __restrict__ dy, P* __restrict__ dE,
                                                                         int n, int V, int d, float scale, int span,
                                                                         int ahead, Runs runs) {
  extern __shared__ __align__(16) uint8_t smem[];
  int* noted = reinterpret_cast<int*>(smem);  // [kSortWarps][kNoted] positions
  int* sorted = noted + kSortWarps * kNoted;               // [kSortWarps * kNoted] positions in the sorted order
  int* hist = sorted + kSortWarps * kNoted;                // [kSortWarps][span] counts, then next places
  int* count = hist + kSortWarps * span;                   // [span] of the ids
  int* listed = count + span;  // [span] from the front ids with 2 to kSlab tokens, from the back those with more, in any order
  int* single = listed + span;  // [span] ids with one token
  __shared__ int warp_total[kSortWarps], below_of[kSortWarps], n_few, n_many, n_single;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // id b + i blocks is block b's i-th
  const int blocks = gridDim.x, b = blockIdx.x, ids = (V - b + blocks - 1) / blocks;
  const unsigned inverse = 0xFFFFFFFFu / blocks;
  auto id_of = [&](int i) { return b + i * blocks; };
  auto owner_of = [&](int t, int& i) {  // the block of an id, its place there; no block, past all of them, for -1
    const unsigned u = static_cast<unsigned>(t), q = __umulhi(u, inverse), r = u - q * blocks;  // q or one less
    const bool one_less = r >= static_cast<unsigned>(blocks);
    i = static_cast<int>(one_less ? q + 1 : q);
    return t < 0 ? 0x7FFFFFFF : static_cast<int>(one_less ? r - blocks : r);
  };
  for (int i = tid; i < kSortWarps * span; i += kSortThreads) hist[i] = 0;
  if (tid == 0) n_few = n_many = n_single = 0;
  __syncthreads();
  const int part = (n + 128 * kSortWarps - 1) / (128 * kSortWarps) * 128;  // tokens a warp
  const int from = min(n, warp * part), to = min(n, from + part);
  int *mine = hist + warp * span, *my_noted = noted + warp * kNoted;
  int below = 0, found = 0;
  // four tokens a lane; f(position, in order over the lanes, belongs to the block) by every lane, or not at all
  auto scan = [&](auto f) {
    const int4* p = reinterpret_cast<const int4*>(ids_of + from) + lane;
#pragma unroll 4
    for (int i = from + 4 * lane; i - 4 * lane < to; i += 128, p += 32) {
      int4 q = make_int4(-1, -1, -1, -1);
      if (i + 3 < n)
        q = *p;
      else if (i < n)
        q = make_int4(ids_of[i], i + 1 < n ? ids_of[i + 1] : -1, i + 2 < n ? ids_of[i + 2] : -1, -1);
      f(i, q);
    }
  };
  scan([&](int i, const int4& q) {
    int i0, i1, i2, i3;
    const int r0 = owner_of(q.x, i0), r1 = owner_of(q.y, i1), r2 = owner_of(q.z, i2), r3 = owner_of(q.w, i3);
    below += (r0 < b) + (r1 < b) + (r2 < b) + (r3 < b);
    const bool o0 = r0 == b, o1 = r1 == b, o2 = r2 == b, o3 = r3 == b;
    if (!__any_sync(0xffffffffu, o0 | o1 | o2 | o3)) return;
    const unsigned b0 = __ballot_sync(0xffffffffu, o0), b1 = __ballot_sync(0xffffffffu, o1),
                   b2 = __ballot_sync(0xffffffffu, o2), b3 = __ballot_sync(0xffffffffu, o3), under = (1u << lane) - 1;
    int at = found + __popc(b0 & under) + __popc(b1 & under) + __popc(b2 & under) + __popc(b3 & under);
    auto note = [&](bool own, int bin, int position) {
      if (!own) return;
      atomicAdd(mine + bin, 1);
      if (ahead && at < kAhead) fetch_to_l2(dy + static_cast<long long>(position) * d, d);
      if (at < kNoted) my_noted[at] = position;
      ++at;
    };
    note(o0, i0, i), note(o1, i1, i + 1), note(o2, i2, i + 2), note(o3, i3, i + 3);
    found += __popc(b0) + __popc(b1) + __popc(b2) + __popc(b3);
  });
  below = __reduce_add_sync(0xffffffffu, below);
  if (lane == 0) below_of[warp] = below;
  __syncthreads();
  // exclusive sums over (id, warp); a thread takes an id, or two neighbouring ones
  const int each = ids <= kSortThreads ? 1 : 2;
  int totals[2] = {0, 0};
#pragma unroll
  for (int k = 0; k < 2; ++k)
    if (k < each && each * tid + k < ids) {
#pragma unroll 8
      for (int w = 0; w < kSortWarps; ++w) totals[k] += hist[w * span + each * tid + k];
    }
  int incl = totals[0] + totals[1];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) warp_total[warp] = incl;
  __syncthreads();
  const int base = __reduce_add_sync(0xffffffffu, below_of[lane]);
  const int block_total = __reduce_add_sync(0xffffffffu, warp_total[lane]);
  int at = base + __reduce_add_sync(0xffffffffu, lane < warp ? warp_total[lane] : 0) + incl - totals[0] - totals[1];
#pragma unroll
  for (int k = 0; k < 2; ++k)
    if (k < each && each * tid + k < ids) {
      const int i = each * tid + k;
      count[i] = totals[k];
      runs.empty[id_of(i)] = totals[k] == 0;
      if (totals[k] == 1) single[atomicAdd(&n_single, 1)] = i;
      if (totals[k] > 1 && totals[k] <= kSlab) listed[atomicAdd(&n_few, 1)] = i;
      if (totals[k] > kSlab) {
        listed[span - 1 - atomicAdd(&n_many, 1)] = i;
        const int slab = at / kSlab;
        runs.id[slab] = id_of(i);
        runs.end[slab] = at + totals[k];
        runs.done[slab] = 0;
      }
#pragma unroll 8
      for (int w = 0; w < kSortWarps; ++w) {
        const int v = hist[w * span + i];
        hist[w * span + i] = at;
        at += v;
      }
    }
  __syncthreads();
  const bool local = block_total <= kSortWarps * kNoted;  // the sorted order fits shared memory
  auto place = [&](bool own, int bin, int position) {     // by every lane of the warp, positions ascending with the lane
    const unsigned all = __ballot_sync(0xffffffffu, own);
    if (own) {
      const unsigned same = __match_any_sync(all, bin);
      const int first = mine[bin], rank = __popc(same & ((1u << lane) - 1));
      __syncwarp(all);
      if (rank == 0) mine[bin] = first + __popc(same);
      if (local) sorted[first + rank - base] = position;
      if (!local || count[bin] > kSlab) runs.order[first + rank] = position;
    }
    __syncwarp();
  };
  if (found <= kNoted) {
    for (int e = lane; e - lane < found; e += 32) {
      const int position = e < found ? my_noted[e] : -1;
      int bin = 0;
      if (e < found) owner_of(ids_of[position], bin);
      place(e < found, bin, position);
    }
  } else {
    for (int i = from + lane; i - lane < to; i += 32) {
      int bin;
      const bool own = owner_of(i < to ? ids_of[i] : -1, bin) == b;
      place(own, bin, i);
    }
  }
  __syncthreads();
  let_next_start();
  // place of an id's first token: where the last warp's part of the id before it ended
  auto start_of = [&](int i) { return i == 0 ? base : hist[(kSortWarps - 1) * span + i - 1]; };
  if (n > kSlab) {  // else the second kernel does not look for runs
    for (int i = base + tid; i < base + block_total; i += kSortThreads) runs.run_start[i] = -1;
    if (b == blocks - 1)  // places behind the last valid token
      for (int i = base + block_total + tid; i < n; i += kSortThreads) runs.run_start[i] = -1;
    __syncthreads();
    for (int m = warp; m < n_many; m += kSortWarps) {
      const int i = listed[span - 1 - m], start = start_of(i);
      for (int j = lane; j < count[i]; j += 32) runs.run_start[start + j] = start;
    }
  }
  // A warp takes a piece of 256 columns of an id's rows; what it waits for is a chain of lookups and one random access to
  // memory (2,000 to 4,000 cycles), so of ids with one token it takes four at a time.
  const int pieces = (d + 255) / 256;
  auto position_of = [&](int i, int r) { return local ? sorted[start_of(i) - base + r] : runs.order[start_of(i) + r]; };
#pragma unroll 1
  for (int item = warp * kItems; item < n_single * pieces; item += kSortWarps * kItems) {
    int from = 0, to = 0, c0 = d;  // lane u: the u-th item's
    if (lane < kItems && item + lane < n_single * pieces) {
      const int i = single[(item + lane) / pieces];
      from = position_of(i, 0), to = id_of(i), c0 = ((item + lane) % pieces) * 256;
    }
    copy_rows<T, P, kVec>(dy, dE, from, to, c0, d, scale, lane);
  }
#pragma unroll 1
  for (int item = warp; item < n_few * pieces; item += kSortWarps) {
    const int i = listed[item / pieces], piece = item % pieces;
    const int k = count[i], row_of = lane < k ? position_of(i, lane) : 0;
    sum_rows<T, P, kVec>(dy, row_of, k, dE + static_cast<long long>(id_of(i)) * d, 256 * piece, d, scale, lane);
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
  const int groups = blockDim.x / width, g = threadIdx.x / width, c = threadIdx.x - g * width;
  for (int c0 = 0; c0 < d; c0 += width * kPer) {
    const int col = c0 + c * kPer;
    float acc[kPer] = {};
    if (col < d && g < groups) {
#pragma unroll 4
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
__global__ void __launch_bounds__(kRunThreads, 4) embedding_runs_kernel(const T* __restrict__ dy, P* __restrict__ dE, int n, int V,
                                                                     int d, float scale, Runs runs,
                                                                     float* __restrict__ partial, int slabs, int per) {
  __shared__ int where[kSlab], place[kSlab], last;
  __shared__ float red[kRunThreads * 8];
  __shared__ uint8_t empty[kMaxPer + 1];
  wait_for_previous();
  // Blocks with a slab and blocks with `per` ids, whose rows without a token they write, take turns while there are both:
  // the former wait for loads, the latter do not.
  const int zero_blocks = gridDim.x - slabs, pairs = min(slabs, zero_blocks), b = blockIdx.x;
  const bool zeros = b < 2 * pairs ? b & 1 : slabs <= zero_blocks;
  const int mine = b < 2 * pairs ? b / 2 : b - pairs;
  if (zeros) {
    write_zeros(dE, mine * per, min(V, (mine + 1) * per), d, runs.empty, empty);
    return;
  }
  const int slab = mine, begin = slab * kSlab, stop = min(n, begin + kSlab);
  if (threadIdx.x < kSlab) {
    const bool in = begin + static_cast<int>(threadIdx.x) < stop;
    where[threadIdx.x] = in ? runs.run_start[begin + threadIdx.x] : -1;
    place[threadIdx.x] = in ? runs.order[begin + threadIdx.x] : 0;
  }
  __syncthreads();
  constexpr int kPer = kVec ? 8 : 1;
  const int width = min(kRunThreads, (d + kPer - 1) / kPer);  // as many groups of threads as the block has room for
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
    float* own_part = partial + (2ll * slab + which) * d;
    block_row_sum<kVec, false>(
        b - a, d, width, red, [&](int r) { return dy + static_cast<long long>(place[a + r]) * d; },
        [&](int col, const float(&v)[kPer]) {
#pragma unroll
          for (int j = 0; j < kPer; ++j) own_part[col + j] = v[j];
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
int lookup(const void* tokens, int wide, const void* table, void* y, int* ids, long long n, long long V, int d, float scale,
           int* status, int* refused, cudaStream_t st) {
  const int blocks = static_cast<int>(std::min<long long>((n + 31) / 32, 148 * 8));
  embedding_lookup_kernel<P, T, kVec><<<blocks, 256, 0, st>>>(tokens, wide, static_cast<const P*>(table),
                                                              static_cast<T*>(y), ids, n, V, d, scale, status, refused);
  return cudaGetLastError() == cudaSuccess ? 0 : 1;
}

template <typename T, typename P, bool kVec>
int grad(const int* ids, const void* dy, void* dE, int n, int V, int d, float scale, int* ints, float* partial,
         cudaStream_t st) {
  // a block an SM, or more where a span would not fit
  const int blocks_min = std::max(148, (V + kMaxSpan - 1) / kMaxSpan);
  const int span = (V + blocks_min - 1) / blocks_min, blocks = (V + span - 1) / span;
  const int slabs = n > kSlab ? (n + kSlab - 1) / kSlab : 0;  // else no id has more tokens than a slab
  const long long all = (n + kSlab - 1) / kSlab;
  const Runs runs{ints, ints + n, ints + 2ll * n, ints + 2ll * n + all, ints + 2ll * n + 2 * all,
                  reinterpret_cast<uint8_t*>(ints + 2ll * n + 3 * all)};
  const size_t smem = (static_cast<size_t>(span) * (kSortWarps + 3) + 2 * kSortWarps * kNoted) * sizeof(int);
  auto kern = embedding_sort_kernel<T, P, kVec>;
  static std::atomic<unsigned long long> asked{0};
  constexpr int kMostBytes = (kMaxSpan * (kSortWarps + 3) + 2 * kSortWarps * kNoted) * 4;
  if (!make_room(asked, reinterpret_cast<const void*>(kern), kMostBytes)) return 2;
  // half of L2 may hold the rows until they are summed
  const int ahead = static_cast<long long>(n) * d * static_cast<long long>(sizeof(T)) <= (64ll << 20);
  kern<<<blocks, kSortThreads, smem, st>>>(ids, static_cast<const T*>(dy), static_cast<P*>(dE), n, V, d, scale, span, ahead,
                                           runs);
  if (cudaGetLastError() != cudaSuccess) return 1;
  // Blocks that write zeros take about 32 KB each, so that those which run at one time write one stretch of the table: with
  // 592 blocks for all of it, a stretch each, 151,936 rows of 515 fp32 took 90 us, so 69.
  const int per = static_cast<int>(std::clamp<long long>(32768 / (static_cast<long long>(d) * sizeof(P)), 16, kMaxPer));
  const int zero_blocks = (V + per - 1) / per;
  return launch_after(embedding_runs_kernel<T, P, kVec>, dim3(slabs + zero_blocks), dim3(kRunThreads), 0, st,
                      static_cast<const T*>(dy), static_cast<P*>(dE), n, V, d, scale, runs, partial, slabs, per) == cudaSuccess
             ? 0
             : 1;
}

}  // namespace

// y [n, d] = scale table[tokens]; a token outside [0, V) is reported and gives a zero row. tokens int64 (wide) or int32.
// ids [n] (or null) receives them in 32 bits, unknown ones as -1.
extern "C" int pd_embedding(const void* tokens, int wide, const void* table, void* y, int* ids, long long n, long long V,
                            int d, float scale, int table_fp32, int y_fp32, int* status, int* refused, void* stream) {
  if (n <= 0 || V <= 0 || V >= (1ll << 30) || d <= 0) return 5;
  const bool vec = d % 8 == 0 && aligned16(table) && aligned16(y);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto go = [&](auto p, auto t) {
    using P = decltype(p);
    using T = decltype(t);
    return vec ? lookup<P, T, true>(tokens, wide, table, y, ids, n, V, d, scale, status, refused, st)
               : lookup<P, T, false>(tokens, wide, table, y, ids, n, V, d, scale, status, refused, st);
  };
  using B = __nv_bfloat16;
  if (table_fp32) return y_fp32 ? go(float(), float()) : go(float(), B());
  return y_fp32 ? go(B(), float()) : go(B(), B());
}

// Scratch of the gradient, in ints and in floats.
extern "C" long long pd_embedding_grad_ints(long long n, long long V) {
  return 2 * n + 3 * ((n + kSlab - 1) / kSlab) + (V + 3) / 4;
}
extern "C" long long pd_embedding_grad_floats(long long n, int d) { return 2 * ((n + kSlab - 1) / kSlab) * d; }

// dE [V, d], every row of it; ids as the lookup left them, 16-byte aligned: those outside [0, V) take no part.
extern "C" int pd_embedding_grad(const int* ids, const void* dy, void* dE, long long n, long long V, int d, float scale,
                                 int dy_fp32, int table_fp32, int* ints, float* partial, void* stream) {
  if (n < 0 || n >= (1ll << 30) || V <= 0 || V >= (1ll << 30) || d <= 0 || !aligned16(ids)) return 5;
  const bool vec = d % 8 == 0 && aligned16(dy) && aligned16(dE) && aligned16(partial);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int n32 = static_cast<int>(n), V32 = static_cast<int>(V);
  auto go = [&](auto t, auto p) {
    using T = decltype(t);
    using P = decltype(p);
    return vec ? grad<T, P, true>(ids, dy, dE, n32, V32, d, scale, ints, partial, st)
               : grad<T, P, false>(ids, dy, dE, n32, V32, d, scale, ints, partial, st);
  };
  using B = __nv_bfloat16;
  if (dy_fp32) return table_fp32 ? go(float(), float()) : go(float(), B());
  return table_fp32 ? go(B(), float()) : go(B(), B());
}
