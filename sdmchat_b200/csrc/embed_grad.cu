// The scaled token lookup and its gradient, the sum of dout's rows over the positions of each token.
//
// Gradient.  Up to kFewMax positions are done in one launch (few_kernel): blocks clear the rows that no id names, and the
// first position of each token adds up its others.  For more, the positions are sorted by token while the gradient is
// cleared: up to kSortMax positions by one cluster's radix sort in shared memory (sort_kernel; the other blocks clear),
// more by a counting sort over all SMs (group_kernel: every cluster reads all ids; 131,072 positions over 32,768 x 768
// 106 us, over 131,072 x 768, of which 61 us are the gradient's zeros, 194).  sum_kernel cuts the sorted order into pieces
// of kPiece positions, a warp each: a group inside a piece is added up and written, a group that crosses a cut leaves a
// partial sum on each side.  join_kernel adds the partial sums in order.  No float atomics, and every addition has its
// place: the result is a function of the inputs alone.
#include <algorithm>
#include "vocab.cuh"

namespace sdm {
namespace {

constexpr int kPiece = 16;       // positions summed by one warp (with its two neighbours at most 32)
constexpr int kFewMax = 1024;    // positions that one launch compares with one another: 16 to 24 us over a table of
                                 // 32,768 x 768, against 28 by sorting; at 2,048 it takes 40, and sorting 29
constexpr int kLong = 6;         // a group that goes on over so many more pieces is joined by blocks (65,536 x 768 by a
                                 // Zipf law 63 us, with 16 66; 5,000 x 330 24.7 and 26.9)
constexpr int kSortThreads = 1024, kSortWarps = kSortThreads / 32;
constexpr int kSortCluster = 16; // blocks of the sorting cluster at most (more than the portable 8)
constexpr int kSortEach = 4096;  // positions of one of them
constexpr int kSortMax = kSortCluster * kSortEach;
constexpr int kGroupThreads = 512, kGroupWarps = kGroupThreads / 32;
constexpr int kCluster = 8;      // blocks of a cluster
constexpr int kOwned = 1024;     // tokens of a counting cluster at most: 64 KB of counters
constexpr int kSteps = 64;       // of 32 ids: so many of a warp are remembered from the count to the placing
constexpr int kLookWords = 3;
constexpr int kSumThreads = 256, kSumWarps = kSumThreads / 32;

struct GroupWs {
  int32_t *order;    // (N) positions, grouped by token, in order within a group
  int32_t *token;    // (N) their tokens
  int32_t *crossing; // (pieces) the token whose group begins in the piece and goes on after it, or -1
  int32_t *hot;      // (pieces / kLong) the pieces in which a long group begins
  int32_t *hot_n;
  int32_t *total;    // grouped positions
  float *partial;    // (2 * pieces, ldp)
  int ldp;           // d rounded up to whole 16-byte words
};

__host__ int owner_bits(int V) {  // 32 clusters (256 blocks of two per SM), more where an owner would have too many tokens
  int b = 5;
  while (((int64_t)1 << b) * kOwned < V) ++b;
  return b;
}

size_t carve(GroupWs& w, void* base, int64_t N, int d) {
  size_t off = 0;
  auto take = [&](size_t bytes) {
    char* p = base ? static_cast<char*>(base) + off : nullptr;
    off += (bytes + 255) & ~(size_t)255;
    return p;
  };
  const int64_t pieces = ceil_div(N, kPiece);
  w.ldp = (d + 3) / 4 * 4;
  w.order = reinterpret_cast<int32_t*>(take(N * 4));
  w.token = reinterpret_cast<int32_t*>(take(N * 4));
  w.crossing = reinterpret_cast<int32_t*>(take(pieces * 4));
  w.hot = reinterpret_cast<int32_t*>(take((pieces / kLong + 1) * 4));
  w.hot_n = reinterpret_cast<int32_t*>(take(4));
  w.total = reinterpret_cast<int32_t*>(take(4));
  w.partial = reinterpret_cast<float*>(take((size_t)2 * pieces * w.ldp * 4));
  return off;
}

// Zeroes `bytes` bytes at `at`: thread t of `threads`.
__device__ __forceinline__ void clear_bytes(char* at, int64_t bytes, int64_t t, int64_t threads) {
  const int64_t head = min(bytes, (int64_t)(-reinterpret_cast<uintptr_t>(at) & 15)), words = (bytes - head) / 16;
  uint4* q = reinterpret_cast<uint4*>(at + head);
  const uint4 zero = make_uint4(0, 0, 0, 0);
#pragma unroll 4
  for (int64_t i = t; i < words; i += threads) q[i] = zero;
  if (t < head) at[t] = 0;
  if (t < bytes - head - words * 16) at[head + words * 16 + t] = 0;
}

// The lanes of the warp with this lane's digit, a ballot per bit (a digit has 9 at most).
__device__ __forceinline__ uint32_t same_digit(uint32_t digit) {
  uint32_t same = 0xffffffffu;
#pragma unroll
  for (int b = 0; b < 9; ++b) {
    const uint32_t set = __ballot_sync(0xffffffffu, (digit >> b) & 1);
    same &= (digit >> b) & 1 ? set : ~set;
  }
  return same;
}

// Cluster 0 sorts the positions by token, least significant digits first; the other clusters clear the gradient.  Block
// r of the sorting cluster holds positions [r * each, +each) of the present order in shared memory, each warp one
// stretch of them, as token << 16 | position.  A digit's counts by warp, block and cluster give every entry its place
// in the next order, where it is stored in the block that holds it.  An id to be skipped sorts behind all tokens.
__global__ void __launch_bounds__(kSortThreads, 1)
    sort_kernel(const int32_t* __restrict__ ids, int N, int V, int each, int digit_bits, int passes, int padding_id,
                GroupWs w, char* grad, int64_t grad_bytes) {
  pdl_enter();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  auto cluster = cooperative_groups::this_cluster();
  const int C = (int)cluster.num_blocks();
  if ((int)blockIdx.x >= C) {
    clear_bytes(grad, grad_bytes, (int64_t)(blockIdx.x - C) * kSortThreads + tid, (int64_t)(gridDim.x - C) * kSortThreads);
    return;
  }
  typedef unsigned long long u64;
  extern __shared__ u64 entry[];  // two orders of `each`, then the warps' counts of a digit
  __shared__ uint32_t sum[kSortWarps], sum_own[kSortWarps], here[512], base[512], base_own[512], valid_here;
  const int digits = 1 << digit_bits;
  uint32_t* count = reinterpret_cast<uint32_t*>(entry + 2 * each);
  const int rank = (int)cluster.block_rank();
  const int first = rank * each;                     // of this block's positions
  const int per_warp = each / kSortWarps, steps = per_warp / 32, e0 = warp * per_warp + lane;
  if (tid == 0) valid_here = 0;
  __syncthreads();
  uint32_t valid = 0;
#pragma unroll 8
  for (int i = tid; i < each; i += kSortThreads) {
    const int n = first + i;
    int id = n < N ? ids[n] : -1;
    const bool ok = id >= 0 && id < V && id != padding_id;
    valid += ok;
    entry[i] = (u64)(uint32_t)(ok ? id : V) << 16 | (uint32_t)(n & 0xffff);
  }
  valid = __reduce_add_sync(0xffffffffu, valid);
  if (lane == 0) atomicAdd(&valid_here, valid);
  u64* from = entry;
  u64* to = entry + each;
  uint32_t* mine = count + warp * digits;
  for (int pass = 0; pass < passes; ++pass) {
    const int shift = 16 + pass * digit_bits;
    for (int i = tid; i < kSortWarps * digits; i += kSortThreads) count[i] = 0;
    __syncthreads();
    constexpr int S = kSortEach / kSortThreads;
    uint32_t place[S];  // digit, and the place among the warp's entries of that digit
    u64 held[S];
#pragma unroll
    for (int s = 0; s < S; ++s) {
      if (s >= steps) break;
      held[s] = from[e0 + 32 * s];
      const uint32_t digit = (uint32_t)(held[s] >> shift) & (digits - 1);
      const uint32_t same = same_digit(digit);
      const uint32_t at = mine[digit];
      __syncwarp();
      if (lane == __ffs(same) - 1) mine[digit] = at + __popc(same);
      __syncwarp();
      place[s] = digit << 16 | (at + __popc(same & ((1u << lane) - 1)));
    }
    __syncthreads();
    // counts become sums over the warps before
    uint32_t own = 0;
    if (tid < digits) {
#pragma unroll 8
      for (int k = 0; k < kSortWarps; ++k) {
        const uint32_t c = count[k * digits + tid];
        count[k * digits + tid] = own;
        own += c;
      }
      here[tid] = own;
    }
    cluster.sync();
    uint32_t all = 0, ahead = 0;
    if (tid < digits) {
#pragma unroll 8
      for (int r = 0; r < C; ++r) {
        const uint32_t c = *cluster.map_shared_rank(&here[tid], r);
        all += c;
        if (r < rank) ahead += c;
      }
    }
    // where a digit begins in the cluster's next order (for this block's entries), and in this block's own
    uint32_t run = all, run_own = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t up = __shfl_up_sync(0xffffffffu, run, o), up_own = __shfl_up_sync(0xffffffffu, run_own, o);
      if (lane >= o) {
        run += up;
        run_own += up_own;
      }
    }
    if (lane == 31) {
      sum[warp] = run;
      sum_own[warp] = run_own;
    }
    __syncthreads();
    if (tid < digits) {
      uint32_t before = run - all + ahead, before_own = run_own - own;
      for (int k = 0; k < warp; ++k) {
        before += sum[k];
        before_own += sum_own[k];
      }
      base_own[tid] = before_own;
      base[tid] = before - before_own;
    }
    __syncthreads();
    // first within the block, so that what goes to another block leaves in whole lines
#pragma unroll
    for (int s = 0; s < S; ++s) {
      if (s >= steps) break;
      const uint32_t digit = place[s] >> 16;
      from[base_own[digit] + mine[digit] + (place[s] & 0xffffu)] = held[s];
    }
    __syncthreads();
#pragma unroll
    for (int s = 0; s < S; ++s) {
      if (s >= steps) break;
      const uint32_t i = s * kSortThreads + tid;
      const u64 e = from[i];
      const uint32_t at = base[(uint32_t)(e >> shift) & (digits - 1)] + i;
      const uint32_t r = at / each;
      *cluster.map_shared_rank(to + (at - r * each), r) = e;
    }
    cluster.sync();
    u64* t = from;
    from = to;
    to = t;
  }
  uint32_t total = 0;
  if (rank == 0 && tid < C) total = *cluster.map_shared_rank(&valid_here, tid);
  total = __reduce_add_sync(0xffffffffu, total);
  if (rank == 0 && tid == 0) {
    *w.total = (int32_t)total;
    *w.hot_n = 0;
  }
  for (int i = tid; i < each; i += kSortThreads) {
    if (first + i >= N) break;
    const u64 e = from[i];
    w.order[first + i] = (int32_t)(e & 0xffff);
    w.token[first + i] = (int32_t)(e >> 16);
  }
  cluster.sync();
}

// Cluster b owns the tokens v with v mod owners == b (v = local * owners + b).  Each warp counts and later places one
// stretch of the ids, so the sort is stable; a word of lanes per 32 ids tells it which of them to come back to.
__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kGroupThreads, 2)
    group_kernel(const int32_t* __restrict__ ids, int N, int V, int bits, int per, int padding_id, GroupWs w, char* grad,
                 int64_t grad_bytes) {
  pdl_enter();
  const uint32_t me = blockIdx.x / kCluster, low = (1u << bits) - 1;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  extern __shared__ uint32_t count[];  // (warps, per)
  __shared__ uint32_t size_here[kOwned];  // of each token in this block's ids
  __shared__ uint32_t warp_sum_[kGroupWarps], below_here;
  __shared__ uint32_t seen[kGroupWarps][kSteps];  // lanes of a step whose id is owned
  auto cluster = cooperative_groups::this_cluster();
  const int rank = (int)cluster.block_rank();
  for (int i = tid; i < kGroupWarps * per; i += kGroupThreads) count[i] = 0;
  clear_bytes(grad, grad_bytes, (int64_t)blockIdx.x * kGroupThreads + tid, (int64_t)gridDim.x * kGroupThreads);
  __syncthreads();
  const int seg = (int)(ceil_div(ceil_div(N, kGroupWarps * kCluster), 32) * 32);
  const int n0 = (int)min((int64_t)N, (int64_t)(rank * kGroupWarps + warp) * seg), n1 = (int)min((int64_t)N, (int64_t)n0 + seg);
  const int steps = (n1 - n0 + 31) / 32;
  uint32_t* mine = count + warp * per;
  uint32_t below = 0;
  constexpr int U = 8;
  for (int s0 = 0; s0 < steps; s0 += U) {
    int id[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int n = n0 + (s0 + u) * 32 + lane;
      id[u] = n < n1 ? ids[n] : -1;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool ok = id[u] >= 0 && id[u] < V && id[u] != padding_id;
      const uint32_t owner = (uint32_t)id[u] & low;
      below += ok && owner < me;
      const bool owned = ok && owner == me;
      const uint32_t lanes = __ballot_sync(0xffffffffu, owned);
      if (owned) atomicAdd(&mine[id[u] >> bits], 1u);
      if (lane == 0 && s0 + u < kSteps) seen[warp][s0 + u] = lanes;
    }
  }
  below = __reduce_add_sync(0xffffffffu, below);
  if (lane == 0) warp_sum_[warp] = below;
  __syncthreads();
  if (tid == 0) {
    uint32_t b = 0;
    for (int i = 0; i < kGroupWarps; ++i) b += warp_sum_[i];
    below_here = b;
  }
  for (int t = tid; t < per; t += kGroupThreads) {  // counts become offsets within the block's share of the token
    uint32_t size = 0;
#pragma unroll
    for (int i = 0; i < kGroupWarps; ++i) {
      const uint32_t c = count[i * per + t];
      count[i * per + t] = size;
      size += c;
    }
    size_here[t] = size;
  }
  cluster.sync();
  // two neighbouring tokens per thread: their sizes in the whole cluster and in the blocks before this one
  uint32_t size[2] = {0, 0}, ahead[2] = {0, 0}, base = 0;
#pragma unroll
  for (int r = 0; r < kCluster; ++r) {
    base += *cluster.map_shared_rank(&below_here, r);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const uint32_t c = 2 * tid + e < per ? *cluster.map_shared_rank(&size_here[2 * tid + e], r) : 0u;
      size[e] += c;
      if (r < rank) ahead[e] += c;
    }
  }
  cluster.barrier_arrive();  // this block reads no other one from here on
  const uint32_t both = size[0] + size[1];
  uint32_t run = both;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t up = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= o) run += up;
  }
  if (lane == 31) warp_sum_[warp] = run;
  __syncthreads();
  uint32_t first = base + run - both;
#pragma unroll
  for (int i = 0; i < kGroupWarps; ++i) first += i < warp ? warp_sum_[i] : 0u;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int t = 2 * tid + e;
    if (t < per) {
#pragma unroll
      for (int i = 0; i < kGroupWarps; ++i) count[i * per + t] += first + ahead[e];
    }
    first += size[e];
  }
  if (me == low && rank == 0 && tid == kGroupThreads - 1) {
    *w.total = (int32_t)first;
    *w.hot_n = 0;
  }
  __syncthreads();
  auto place = [&](int n, int id) {
    const bool owned = id >= 0 && id < V && id != padding_id && ((uint32_t)id & low) == me;
    if (!__any_sync(0xffffffffu, owned)) return;
    const int local = owned ? id >> bits : -1;
    const uint32_t same = __match_any_sync(0xffffffffu, local);
    const int rank_ = __popc(same & ((1u << lane) - 1));
    uint32_t at = 0;
    if (owned) at = mine[local] + rank_;
    __syncwarp();
    if (owned) {
      w.order[at] = n;
      w.token[at] = id;
      if (rank_ == 0) mine[local] += __popc(same);
    }
    __syncwarp();
  };
#pragma unroll 1
  for (int half = 0; half < kSteps; half += 32) {
    uint32_t todo = __ballot_sync(0xffffffffu, half + lane < steps && seen[warp][half + lane] != 0);
    while (todo) {  // eight steps' ids at a time
      int n[U], id[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        n[u] = todo ? n0 + (half + __ffs(todo) - 1) * 32 + lane : n1;
        todo &= todo - 1;
        id[u] = n[u] < n1 ? ids[n[u]] : -1;
      }
#pragma unroll
      for (int u = 0; u < U; ++u) place(n[u], id[u]);
    }
  }
#pragma unroll 1
  for (int s = kSteps; s < steps; s += U) {
    int id[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int n = n0 + (s + u) * 32 + lane;
      id[u] = n < n1 ? ids[n] : -1;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) place(n0 + (s + u) * 32 + lane, id[u]);
  }
  cluster.barrier_wait();
}

template <int BYTES> struct Word;
template <> struct Word<16> { typedef uint4 type; };
template <> struct Word<8> { typedef uint2 type; };
template <> struct Word<4> { typedef uint32_t type; };
template <> struct Word<2> { typedef uint16_t type; };

template <typename T, int VEC>
struct Pack {
  typename Word<VEC * sizeof(T)>::type u;
  __device__ float get(int e) const { return to_f32(reinterpret_cast<const T*>(&u)[e]); }
};

// VEC sums times scale (plus the old gradient) to `at`, aligned to their size or 16 bytes.
template <typename G, int VEC>
__device__ __forceinline__ void store_grad(G* at, const float* v, float scale, int accumulate) {
  constexpr int BYTES = VEC * sizeof(G) > 16 ? 16 : VEC * sizeof(G), N = BYTES / sizeof(G);
  typedef typename Word<BYTES>::type W;
#pragma unroll
  for (int k = 0; k < VEC; k += N) {
    union {
      W u;
      G g[N];
    } y;
    if (accumulate) y.u = *reinterpret_cast<const W*>(at + k);
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float s = v[k + e] * scale;
      y.g[e] = from_f32<G>(accumulate ? to_f32(y.g[e]) + s : s);
    }
    *reinterpret_cast<W*>(at + k) = y.u;
  }
}

// Warp (piece, 32 VEC NQ columns): the sums of the piece's groups.  A lane's columns are c + 32 VEC q + e.  As many rows
// as 64 registers hold are in flight together (all of the piece's for bfloat16): with fewer, and more warps in their
// stead, the same sums took longer.
template <typename T, typename G, int VEC, int NQ>
__global__ void __launch_bounds__(kSumThreads, 2) sum_kernel(const T* __restrict__ dout,
                                                              int64_t ld, int N, int d,
                                                              int col_blocks, int64_t items, float scale,
                                                              int accumulate, GroupWs w, G* __restrict__ grad) {
  pdl_enter();
  constexpr int kRowRegs = NQ * (VEC * sizeof(T) < 4 ? 1 : VEC * sizeof(T) / 4);
  constexpr int kRows = 64 / kRowRegs < kPiece ? 64 / kRowRegs : kPiece;
  typedef typename Word<VEC * sizeof(T)>::type W;
  const int64_t item = (int64_t)blockIdx.x * kSumWarps + (threadIdx.x >> 5);
  if (item >= items) return;
  const int lane = threadIdx.x & 31;
  const int piece = (int)(col_blocks == 1 ? item : item / col_blocks);
  const int c = (int)(item - (int64_t)piece * col_blocks) * (32 * VEC * NQ) + VEC * lane;
  const int j0 = piece * kPiece;
  // lane l: the position before the piece (l = 0), the piece's (1 .. n), and the one after it (n + 1); fetched before
  // `total` is known, and used below it
  const int j = j0 - 1 + lane;
  const bool inside = lane <= kPiece + 1 && j >= 0 && j < N;
  int pos = inside ? w.order[j] : -1, id = inside ? w.token[j] : -1;
  int later = j0 + kLong * kPiece < N ? w.token[j0 + kLong * kPiece] : -1;
  const int total = *w.total, n = min(kPiece, total - j0);
  if (n <= 0) {
    if (c == 0) w.crossing[piece] = -1;
    return;
  }
  if (lane > n + 1 || j >= total) pos = id = -1;
  if (j0 + kLong * kPiece >= total) later = -1;
  const int before = __shfl_sync(0xffffffffu, id, 0), after = __shfl_sync(0xffffffffu, id, n + 1);
  const uint32_t ends = __ballot_sync(0xffffffffu, id != __shfl_down_sync(0xffffffffu, id, 1) || lane == n) >> 1;
  float acc[NQ][VEC];
#pragma unroll
  for (int q = 0; q < NQ; ++q)
#pragma unroll
    for (int e = 0; e < VEC; ++e) acc[q][e] = 0.f;
  bool head = true;  // in the group that holds the piece's first position
#pragma unroll 1
  for (int i0 = 0; i0 < n; i0 += kRows) {
    Pack<T, VEC> p[kRows][NQ];
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      const int at = __shfl_sync(0xffffffffu, pos, min(i0 + k, n - 1) + 1);
      const T* r = dout + (int64_t)at * ld + c;
#pragma unroll
      for (int q = 0; q < NQ; ++q)
        if (c + 32 * VEC * q < d && i0 + k < n) p[k][q].u = __ldg(reinterpret_cast<const W*>(r + 32 * VEC * q));
    }
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      const int i = i0 + k;
      if (i >= n) break;
#pragma unroll
      for (int q = 0; q < NQ; ++q)
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[q][e] += p[k][q].get(e);
      if ((ends >> i) & 1) {
        const int v = __shfl_sync(0xffffffffu, id, i + 1);
        const bool came = head && v == before, goes = i == n - 1 && v == after, crosses = came || goes;
        if (i == n - 1 && c == 0) {
          const bool long_ = goes && !came && v == later;
          if (long_) w.hot[atomicAdd(w.hot_n, 1)] = piece;  // in any order: each is joined by itself
          w.crossing[piece] = goes && !came && !long_ ? v : -1;
        }
        if (crosses) {
          float* out = w.partial + (2 * (int64_t)piece + (head ? 0 : 1)) * w.ldp + c;
#pragma unroll
          for (int q = 0; q < NQ; ++q)
            if (c + 32 * VEC * q < d) store_grad<float, VEC>(out + 32 * VEC * q, acc[q], 1.f, 0);
        } else {
          G* out = grad + (int64_t)v * d + c;
#pragma unroll
          for (int q = 0; q < NQ; ++q)
            if (c + 32 * VEC * q < d) store_grad<G, VEC>(out + 32 * VEC * q, acc[q], scale, accumulate);
        }
#pragma unroll
        for (int q = 0; q < NQ; ++q)
#pragma unroll
          for (int e = 0; e < VEC; ++e) acc[q][e] = 0.f;
        head = false;
      }
    }
  }
}

// Few positions: warp (position, 32 VEC columns) passes on unless its position is the first of its token, else it adds up
// the token's rows in order; then block b zeroes its share of the table's rows but for those that an id names.
template <typename T, typename G, int VEC>
__global__ void __launch_bounds__(256) few_kernel(const int32_t* __restrict__ ids, const T* __restrict__ dout, int64_t ld,
                                                  int N, int d, int V, int col_blocks, int share, int zero_words,
                                                  float scale, int padding_id, int accumulate, G* __restrict__ grad) {
  pdl_enter();
  __shared__ int32_t id_[kFewMax];       // ids, -1 where skipped
  __shared__ uint16_t list[8][kFewMax];  // a warp's positions
  extern __shared__ unsigned char named[];  // a flag per row of the block's share
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint16_t* at = list[warp];
  const int64_t r0 = (int64_t)blockIdx.x * share, r1 = min((int64_t)V, r0 + share);
  if (!accumulate)
    for (int i = tid; i < share; i += 256) named[i] = 0;
  __syncthreads();
  for (int n = tid; n < N; n += 256) {
    int id = ids[n];
    if (id < 0 || id >= V || id == padding_id) id = -1;
    id_[n] = id;
    if (!accumulate && id >= r0 && id < r1) named[id - r0] = 1;
  }
  __syncthreads();
  for (int64_t item = (int64_t)blockIdx.x * 8 + warp; item < (int64_t)N * col_blocks; item += (int64_t)gridDim.x * 8) {
    const int n = (int)(item / col_blocks), c = (int)(item - (int64_t)n * col_blocks) * 32 * VEC + VEC * lane;
    const int v = id_[n];
    if (v < 0) continue;
    bool earlier = false;
    for (int i = lane; i < n; i += 32) earlier |= id_[i] == v;
    if (__any_sync(0xffffffffu, earlier)) continue;
    int m = 0;  // the token's positions, in order
    for (int i0 = n & ~31; i0 < N; i0 += 32) {
      const bool same = i0 + lane < N && id_[i0 + lane] == v;
      const uint32_t lanes = __ballot_sync(0xffffffffu, same);
      if (same) at[m + __popc(lanes & ((1u << lane) - 1))] = (uint16_t)(i0 + lane);
      m += __popc(lanes);
    }
    __syncwarp();
    float acc[VEC] = {};
    constexpr int R = 16;  // rows whose loads are in flight
    for (int i0 = 0; i0 < m; i0 += R) {
      Pack<T, VEC> p[R];
#pragma unroll
      for (int u = 0; u < R; ++u)
        if (i0 + u < m && c < d)
          p[u].u = __ldg(reinterpret_cast<const typename Word<VEC * sizeof(T)>::type*>(dout + (int64_t)at[i0 + u] * ld + c));
#pragma unroll
      for (int u = 0; u < R; ++u)
        if (i0 + u < m) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) acc[e] += p[u].get(e);
        }
    }
    __syncwarp();
    if (c < d) store_grad<G, VEC>(grad + (int64_t)v * d + c, acc, scale, accumulate);
  }
  if (!accumulate)
    for (int64_t r = r0 + warp; r < r1; r += 8) {
      if (named[r - r0]) continue;
      if (zero_words) {  // rows of whole 16-byte words
        uint4* row = reinterpret_cast<uint4*>(grad + r * d);
        for (int i = lane; i < zero_words; i += 32) row[i] = make_uint4(0, 0, 0, 0);
      } else {
        G* row = grad + r * d;
        const float none[VEC] = {};
        for (int c = VEC * lane; c < d; c += 32 * VEC) store_grad<G, VEC>(row + c, none, 0.f, 0);
      }
    }
}

template <typename G>
__device__ __forceinline__ void store_joined(G* row, int c, int d, float4 s, float scale, int accumulate) {
  const float v[4] = {s.x, s.y, s.z, s.w};
  if (d % 4 == 0 && (reinterpret_cast<uintptr_t>(row) & (4 * sizeof(G) - 1)) == 0) {
    store_grad<G, 4>(row + c, v, scale, accumulate);
  } else {
    for (int e = 0; e < 4 && c + e < d; ++e) store_grad<G, 1>(row + c + e, v + e, scale, accumulate);
  }
}

__device__ __forceinline__ void add4(float4& a, const float4& b) {
  a.x += b.x;
  a.y += b.y;
  a.z += b.z;
  a.w += b.w;
}

// The first hot_blocks * cols blocks: 128 columns of the long groups i, i + hot_blocks, ...; warp w takes every
// sixteenth piece, and the warps' sums are added in order.  The others, a warp per piece: the group that begins in the
// piece and goes on over fewer than kLong more.
constexpr int kJoinWarps = 16;
template <typename G>
__global__ void __launch_bounds__(32 * kJoinWarps, 2) join_kernel(int d, int pieces, int hot_blocks, int cols,
                                                                  float scale, int accumulate, GroupWs w,
                                                                  G* __restrict__ grad) {
  pdl_enter();
  __shared__ float4 part[kJoinWarps][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int total = *w.total;
  // a group's partial sums: slot 1 of the piece it begins in (slot 0 if it begins with the piece), slot 0 of the others
  if ((int)blockIdx.x >= hot_blocks * cols) {
    const int m = ((int)blockIdx.x - hot_blocks * cols) * kJoinWarps + warp;
    if (m >= pieces) return;
    const int v = w.crossing[m];
    // the tokens at the starts of this piece and the later ones (beyond `total` there is anything, and it is not used)
    const int k = min(m + lane, pieces - 1), t = w.token[k * kPiece];
    if (v < 0) return;
    const int t0 = __shfl_sync(0xffffffffu, t, 0);
    const uint32_t in = __ballot_sync(0xffffffffu, lane > 0 && lane <= kLong && k == m + lane && k * kPiece < total && t == v);
    const int more = __ffs(~(in >> 1)) - 1;
    const float* first = w.partial + (2 * (int64_t)m + (t0 != v ? 1 : 0)) * w.ldp;
    const float* rest = w.partial + 2 * (int64_t)(m + 1) * w.ldp;
    constexpr int NC = 6;  // 768 columns in flight
    for (int c0 = lane * 4; c0 < d; c0 += 128 * NC) {
      float4 sum[NC];
#pragma unroll
      for (int q = 0; q < NC; ++q)
        if (c0 + 128 * q < d) sum[q] = *reinterpret_cast<const float4*>(first + c0 + 128 * q);
#pragma unroll 2
      for (int k = 0; k < more; ++k) {
#pragma unroll
        for (int q = 0; q < NC; ++q)
          if (c0 + 128 * q < d) add4(sum[q], *reinterpret_cast<const float4*>(rest + (int64_t)2 * k * w.ldp + c0 + 128 * q));
      }
#pragma unroll
      for (int q = 0; q < NC; ++q)
        if (c0 + 128 * q < d) store_joined(grad + (int64_t)v * d, c0 + 128 * q, d, sum[q], scale, accumulate);
    }
    return;
  }
  const int c = ((int)blockIdx.x % cols) * 128 + lane * 4, hot_n = *w.hot_n;
  for (int i = (int)blockIdx.x / cols; i < hot_n; i += hot_blocks) {
    const int m = w.hot[i];
    const int v = w.token[(m + 1) * kPiece];
    int more = 0;  // the pieces after m that begin with v
    for (int k0 = m + 1; k0 < pieces; k0 += 32 * kJoinWarps) {
      const int k = k0 + (int)threadIdx.x;
      const int n = __syncthreads_count(k < pieces && k * kPiece < total && w.token[min(k * kPiece, total - 1)] == v);
      more += n;
      if (n < 32 * kJoinWarps) break;
    }
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    if (c < d) {
      const int slot = w.token[m * kPiece] != v ? 1 : 0;
#pragma unroll 8
      for (int k = warp; k <= more; k += kJoinWarps)
        add4(sum, *reinterpret_cast<const float4*>(w.partial + (2 * (int64_t)(m + k) + (k == 0 ? slot : 0)) * w.ldp + c));
    }
    part[warp][lane] = sum;
    __syncthreads();
    if (warp == 0 && c < d) {
#pragma unroll
      for (int k = 1; k < kJoinWarps; ++k) add4(sum, part[k][lane]);
      store_joined(grad + (int64_t)v * d, c, d, sum, scale, accumulate);
    }
    __syncthreads();
  }
}

// A warp per row, kLookWords of a lane's words in flight (65,536 rows of 768 bfloat16: 22 us; word by word 25).
template <typename T, int VEC>
__global__ void __launch_bounds__(256) lookup_kernel(const int32_t* __restrict__ ids, const T* __restrict__ emb,
                                                     int64_t N, int d, int V, float scale, T* __restrict__ out,
                                                     int* bad) {
  pdl_enter();
  typedef typename Word<VEC * sizeof(T)>::type W;
  const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= N) return;
  const int id = ids[row];
  const bool ok = id >= 0 && id < V;
  if (!ok && lane == 0 && bad) atomicExch(bad, 1);
  for (int c0 = VEC * lane; c0 < d; c0 += VEC * 32 * kLookWords) {
    union {
      W u;
      T t[VEC];
    } y[kLookWords];
#pragma unroll
    for (int q = 0; q < kLookWords; ++q) {
      const int c = c0 + 32 * VEC * q;
      y[q].u = W{};
      if (ok && c < d) y[q].u = __ldg(reinterpret_cast<const W*>(emb + (int64_t)id * d + c));
    }
#pragma unroll
    for (int q = 0; q < kLookWords; ++q) {
      const int c = c0 + 32 * VEC * q;
      if (c >= d) break;
      if (ok) {  // a row that is not there stays 0 whatever the scale
#pragma unroll
        for (int e = 0; e < VEC; ++e) y[q].t[e] = from_f32<T>(to_f32(y[q].t[e]) * scale);
      }
      *reinterpret_cast<W*>(out + row * d + c) = y[q].u;
    }
  }
}

// The widest vector (elements, at most `most`) that a row length, a stride and the pointers allow.
int vec_of(int most, int64_t d, int64_t ld, const void* a, int es_a, const void* b, int es_b) {
  for (int v = most; v > 1; v /= 2) {
    const uintptr_t am = (uintptr_t)v * es_a - 1, bm = (uintptr_t)(v * es_b > 16 ? 16 : v * es_b) - 1;
    if (d % v == 0 && ld % v == 0 && (reinterpret_cast<uintptr_t>(a) & am) == 0 &&
        (reinterpret_cast<uintptr_t>(b) & bm) == 0)
      return v;
  }
  return 1;
}

template <typename T>
cudaError_t lookup_t(const int32_t* ids, const T* emb, int64_t N, int d, int V, float scale, T* out, int* bad,
                     cudaStream_t st) {
  LaunchScope scope_("embed_scaled", st);
  const dim3 grid((unsigned)ceil_div(N, 8)), block(256);
  switch (vec_of(16 / sizeof(T), d, d, emb, sizeof(T), out, sizeof(T))) {
    case 8:
      if constexpr (sizeof(T) == 2) return launch_k(lookup_kernel<T, 8>, grid, block, 0, st, ids, emb, N, d, V, scale, out, bad);
      return cudaErrorInvalidValue;
    case 4: return launch_k(lookup_kernel<T, 4>, grid, block, 0, st, ids, emb, N, d, V, scale, out, bad);
    case 2: return launch_k(lookup_kernel<T, 2>, grid, block, 0, st, ids, emb, N, d, V, scale, out, bad);
    default: return launch_k(lookup_kernel<T, 1>, grid, block, 0, st, ids, emb, N, d, V, scale, out, bad);
  }
}

template <typename T, typename G, int VEC, int NQ>
cudaError_t launch_sum_q(const T* dout, int64_t ld, int64_t N, int d, float scale, int accumulate,
                         const GroupWs& w, G* grad, cudaStream_t st) {
  const int col_blocks = (int)ceil_div(d, 32 * VEC * NQ);
  const int64_t items = ceil_div(N, kPiece) * col_blocks, blocks = ceil_div(items, kSumWarps);
  if (blocks > 0x7fffffff) return cudaErrorInvalidValue;
  LaunchScope scope_("embed_grad_sum", st);
  return launch_next(sum_kernel<T, G, VEC, NQ>, (unsigned)blocks, kSumThreads, st, dout, ld, (int)N, d, col_blocks, items,
                     scale, accumulate, w, grad);
}
template <typename T, typename G, int VEC>
cudaError_t launch_sum(const T* dout, int64_t ld, int64_t N, int d, float scale, int accumulate,
                       const GroupWs& w, G* grad, cudaStream_t st) {
  // 256 columns per warp while that still gives the SMs a warp per scheduler slot, else as few as a lane loads at once
  if (VEC == 8 || ceil_div(N, kPiece) * ceil_div(d, 256) >= kSMs * 24)
    return launch_sum_q<T, G, VEC, 8 / VEC>(dout, ld, N, d, scale, accumulate, w, grad, st);
  return launch_sum_q<T, G, VEC, 1>(dout, ld, N, d, scale, accumulate, w, grad, st);
}

template <typename T, typename G, int VEC>
cudaError_t launch_few(const int32_t* ids, const T* dout, int64_t ld, int64_t N, int d, int V, float scale, int padding_id,
                       int accumulate, G* grad, cudaStream_t st) {
  const int col_blocks = (int)ceil_div(d, 32 * VEC);
  int64_t blocks = std::max(ceil_div(N * col_blocks, 8), accumulate ? (int64_t)1 : ceil_div(V, 8));
  blocks = std::min(blocks, (int64_t)kSMs * 8);  // eight blocks per SM
  const int share = (int)ceil_div(V, blocks);
  const bool whole = (int64_t)d * sizeof(G) % 16 == 0 && (reinterpret_cast<uintptr_t>(grad) & 15) == 0;
  LaunchScope scope_("embed_grad_few", st);
  return launch_k(few_kernel<T, G, VEC>, dim3((unsigned)blocks), dim3(256), accumulate ? 0 : (size_t)share, st, ids, dout, ld,
                  (int)N, d, V, col_blocks, share, whole ? (int)((int64_t)d * sizeof(G) / 16) : 0, scale, padding_id,
                  accumulate, grad);
}

template <typename T, typename G>
cudaError_t grad_t(const int32_t* ids, const T* dout, int64_t ld, int64_t N, int d, int V, float scale,
                   int padding_id, int accumulate, G* grad, void* ws, cudaStream_t st) {
  const int vec = vec_of(16 / sizeof(T), d, ld, dout, sizeof(T), grad, sizeof(G));
  if (N <= kFewMax) {
    switch (vec) {
      case 8:
        if constexpr (sizeof(T) == 2) return launch_few<T, G, 8>(ids, dout, ld, N, d, V, scale, padding_id, accumulate, grad, st);
        return cudaErrorInvalidValue;
      case 4: return launch_few<T, G, 4>(ids, dout, ld, N, d, V, scale, padding_id, accumulate, grad, st);
      case 2: return launch_few<T, G, 2>(ids, dout, ld, N, d, V, scale, padding_id, accumulate, grad, st);
      default: return launch_few<T, G, 1>(ids, dout, ld, N, d, V, scale, padding_id, accumulate, grad, st);
    }
  }
  GroupWs w;
  carve(w, ws, N, d);
  const int64_t bytes = accumulate ? 0 : (int64_t)V * d * sizeof(G);
  cudaError_t e;
  // One cluster sorts 65,536 positions in the time (20 us) in which the others clear a table of 100 MB; the counting
  // sort's cost grows with the table besides (the same two took 33 us, 5,000 positions of 50,021 tokens 31 against 14).
  if (N <= kSortMax) {
    int id_bits = 1;
    while (((int64_t)1 << id_bits) <= V) ++id_bits;  // V itself stands for an id to be skipped
    const int passes = (id_bits + 8) / 9, digit_bits = (id_bits + passes - 1) / passes;
    // 2,048 positions a block, or as many as 16 blocks leave it: fewer blocks exchange less (5,000 positions of 50,021 x 330
    // 22.5 us by 4, by 8 22.9, by 16 23.9; 2,048 positions 20.3 and 22.7)
    int C = 1;
    while (C < kSortCluster && N > C * 2048) C *= 2;
    const int each = (int)(ceil_div(std::max(N, (int64_t)1), C * kSortThreads) * kSortThreads);
    const size_t smem = (size_t)each * 16 + ((size_t)kSortWarps << digit_bits) * 4;
    e = cudaFuncSetAttribute(sort_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
    const int64_t clear = std::min((int64_t)2 * kSMs / C, ceil_div(bytes, 16 * kSortThreads * C));
    LaunchScope scope_("embed_grad_sort", st);
    e = launch_clusters(sort_kernel, (unsigned)((1 + clear) * C), C, kSortThreads, smem, st, ids,
                        (int)N, V, each, digit_bits, passes, padding_id, w, reinterpret_cast<char*>(grad), bytes);
  } else {
    const int bits = owner_bits(V), owners = 1 << bits, per = (int)ceil_div(V, owners);
    e = cudaFuncSetAttribute(group_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kGroupWarps * kOwned * 4);
    if (e != cudaSuccess) return e;
    LaunchScope scope_("embed_grad_group", st);
    e = launch_k(group_kernel, dim3((unsigned)(owners * kCluster)), dim3(kGroupThreads), (size_t)kGroupWarps * per * 4, st,
                 ids, (int)N, V, bits, per, padding_id, w, reinterpret_cast<char*>(grad), bytes);
  }
  if (e != cudaSuccess) return e;
  switch (vec) {
    case 8:
      if constexpr (sizeof(T) == 2) e = launch_sum<T, G, 8>(dout, ld, N, d, scale, accumulate, w, grad, st);
      else e = cudaErrorInvalidValue;
      break;
    case 4: e = launch_sum<T, G, 4>(dout, ld, N, d, scale, accumulate, w, grad, st); break;
    case 2: e = launch_sum<T, G, 2>(dout, ld, N, d, scale, accumulate, w, grad, st); break;
    default: e = launch_sum<T, G, 1>(dout, ld, N, d, scale, accumulate, w, grad, st); break;
  }
  if (e != cudaSuccess) return e;
  const int pieces = (int)ceil_div(N, kPiece), cols = (int)ceil_div(d, 128);
  const int hot_blocks = std::min(pieces / kLong + 1, kSMs);
  const int64_t blocks = (int64_t)hot_blocks * cols + ceil_div(pieces, kJoinWarps);
  if (blocks > 0x7fffffff) return cudaErrorInvalidValue;
  LaunchScope scope_("embed_grad_join", st);
  return launch_next(join_kernel<G>, (unsigned)blocks, 32 * kJoinWarps, st, d, pieces, hot_blocks, cols, scale, accumulate,
                     w, grad);
}

}  // namespace

size_t embed_grad_workspace_bytes(int64_t N, int d, int V) {
  (void)V;
  GroupWs w;
  return carve(w, nullptr, N, d);
}

cudaError_t launch_embed_scaled(const int32_t* ids, const void* emb, int64_t N, int d, int V, float scale, int dtype,
                                void* out, int* bad, cudaStream_t st) {
  if (N == 0) return cudaSuccess;
  if (dtype == SDM_BF16)
    return lookup_t<bf16_t>(ids, static_cast<const bf16_t*>(emb), N, d, V, scale, static_cast<bf16_t*>(out), bad, st);
  return lookup_t<float>(ids, static_cast<const float*>(emb), N, d, V, scale, static_cast<float*>(out), bad, st);
}

cudaError_t launch_embed_grad(const int32_t* ids, const void* dout, int64_t ld, int64_t N, int d, int V, float scale,
                              int padding_id, int dtype, int grad_dtype, int accumulate, void* grad, void* ws,
                              cudaStream_t st) {
#define SDM_GRAD(T, G)                                                                                             \
  grad_t<T, G>(ids, static_cast<const T*>(dout), ld, N, d, V, scale, padding_id, accumulate, static_cast<G*>(grad), \
               ws, st)
  if (dtype == SDM_BF16) return grad_dtype == SDM_BF16 ? SDM_GRAD(bf16_t, bf16_t) : SDM_GRAD(bf16_t, float);
  return grad_dtype == SDM_BF16 ? SDM_GRAD(float, bf16_t) : SDM_GRAD(float, float);
#undef SDM_GRAD
}

}  // namespace sdm
