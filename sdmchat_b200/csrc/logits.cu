// Rules on logits (penalties for repeated tokens, biases, grammar masks) and the choice of a token from them.
//
// Both kernels split a row over blocks, each block owning a slice of the vocabulary.  A block marks, in one shared
// word per token of its slice, what the row's history and biases say about the token; then it reads its logits once,
// 16 bytes per thread, and applies the rules where a word is set.
#include <float.h>
#include <math_constants.h>
#include "vocab.cuh"

namespace sdm {
namespace {

namespace cg = cooperative_groups;
typedef unsigned long long u64;

// A token's word: it occurs in the prompt; it has bias entries, and the number of the first; how often it was generated.
constexpr uint32_t kSeen = 0x80000000u, kBias = 0x40000000u, kTimes = kMaxHistory;
constexpr int kBiasAt = 20;
static_assert(kMaxBias <= 1024 && kMaxHistory < (1 << kBiasAt), "a token's word holds both");

struct RowRules {
  float repetition, frequency, presence;
  const uint32_t* mask;  // this row's mask words, or null
  int bias_n;
  bool marks;            // the row has history or biases
};

__device__ __forceinline__ RowRules row_rules(const sdm_logit_rules& r, int64_t row, int V) {
  RowRules q;
  q.repetition = r.repetition ? r.repetition[row] : r.repetition_all;
  q.frequency = r.frequency ? r.frequency[row] : r.frequency_all;
  q.presence = r.presence ? r.presence[row] : r.presence_all;
  q.mask = nullptr;
  if (r.mask) {
    const int64_t g = r.mask_row ? (int64_t)r.mask_row[row] : (r.mask_rows == 1 ? 0 : row);
    if (g >= 0 && g < r.mask_rows)
      q.mask = reinterpret_cast<const uint32_t*>(r.mask) + g * (((int64_t)V + 31) / 32);
  }
  q.bias_n = r.bias_ids ? r.bias_n : 0;
  q.marks = q.bias_n > 0 || (r.history && r.history_n > 0);
  return q;
}

// Shared memory of the marks: a word per token of the slice, then the bias entries (ids, sums).
inline size_t marks_bytes(const sdm_logit_rules& r, int slice) {
  return (size_t)slice * 4 + (r.bias_ids ? (size_t)r.bias_n * 8 : 0);
}

__device__ __forceinline__ int row_length(const sdm_logit_rules& r, int64_t row) {
  const int width = r.history ? r.history_n : 0;
  return width == 0 ? 0 : r.history_len ? max(0, min((int)r.history_len[row], width)) : width;
}

// Fills word[0 .. n) for tokens v0 .. v0 + n - 1 (v0 may be negative: a slice that starts before the row) from the
// row's history and biases, and bias[j] with the sum of the entries of entry j's token where entry j is the first of
// them.  Whole-number atomics: the words do not depend on their order.  Ends with a barrier.
template <int THREADS>
__device__ __forceinline__ void mark_tokens(const sdm_logit_rules& r, const RowRules& q, int64_t row, int v0, int n,
                                            int V, uint32_t* word, float* bias) {
  // the row's first history entries and its biases are on their way before its length is known
  constexpr int U = THREADS > 1024 ? 1 : 2048 / THREADS;
  const int tid = threadIdx.x;
  const int width = r.history ? r.history_n : 0;
  const int32_t* h = r.history + (width ? row * r.history_ld : 0);
  int32_t tok[U];
#pragma unroll
  for (int u = 0; u < U; ++u) tok[u] = u * THREADS + tid < width ? h[u * THREADS + tid] : -1;
  const int len = row_length(r, row);
  const int made = width > 0 && r.prompt_len ? max(0, min((int)r.prompt_len[row], len)) : 0;
  int32_t* bias_id = reinterpret_cast<int32_t*>(bias + q.bias_n);
  float* bias_value = bias;
  for (int j = tid; j < q.bias_n; j += THREADS) {
    bias_id[j] = r.bias_ids[row * q.bias_n + j];
    bias_value[j] = r.bias_values[row * q.bias_n + j];
  }
  for (int i = tid * 4; i < n; i += THREADS * 4) *reinterpret_cast<uint4*>(word + i) = make_uint4(0, 0, 0, 0);
  __syncthreads();
  for (int j0 = 0; j0 < len; j0 += U * THREADS) {
    if (j0 > 0) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int j = j0 + u * THREADS + tid;
        tok[u] = j < len ? h[j] : -1;
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = j0 + u * THREADS + tid, v = tok[u];
      if (j >= len || v < 0 || v >= V || v < v0 || v - v0 >= n) continue;
      if (j < made) atomicOr(&word[v - v0], kSeen);
      else atomicAdd(&word[v - v0], 1u);
    }
  }
  float sum[kMaxBias / THREADS] = {};
#pragma unroll
  for (int k = 0; k < kMaxBias / THREADS; ++k) {
    const int j = k * THREADS + tid;
    if (j >= q.bias_n) break;
    const int v = bias_id[j];
    if (v < 0 || v >= V || v < v0 || v - v0 >= n) continue;
    bool first = true;
    for (int i = 0; i < j; ++i) first &= bias_id[i] != v;
    for (int i = 0; i < q.bias_n; ++i)
      if (bias_id[i] == v) sum[k] = __fadd_rn(sum[k], bias_value[i]);
    if (first) atomicOr(&word[v - v0], kBias | (uint32_t)j << kBiasAt);
  }
  __syncthreads();
  if (q.bias_n > 0) {  // uniform over the block
#pragma unroll
    for (int k = 0; k < kMaxBias / THREADS; ++k)
      if (k * THREADS + tid < q.bias_n) bias[k * THREADS + tid] = sum[k];
    __syncthreads();
  }
}

// The rules of one marked token, in the plain form's order of operations (each rounded to float32, none fused), so
// that tokens the plain form ties are tied here too.
__device__ __forceinline__ float ruled(float x, uint32_t w, const RowRules& q, const float* bias) {
  if (w & (kSeen | kTimes)) x = x > 0.f ? __fdiv_rn(x, q.repetition) : __fmul_rn(x, q.repetition);
  const uint32_t g = w & kTimes;
  if (g) {
    x = __fsub_rn(x, __fmul_rn(q.frequency, (float)g));
    x = __fsub_rn(x, q.presence);
  }
  if (w & kBias) x = __fadd_rn(x, bias[(w >> kBiasAt) & (kMaxBias - 1)]);
  return x;
}

// The rules on a thread's E elements f, whose words are at `word`.  Marked tokens are few but for the commonest ones: most
// warps leave at the first test.
template <int E>
__device__ __forceinline__ void rule_chunk(float* f, const uint32_t* word, const RowRules& q, const float* bias) {
  uint4 w[E / 4];
  uint32_t any = 0;
#pragma unroll
  for (int k = 0; k < E / 4; ++k) {
    w[k] = *reinterpret_cast<const uint4*>(word + 4 * k);
    any |= w[k].x | w[k].y | w[k].z | w[k].w;
  }
  if (!any) return;
#pragma unroll
  for (int k = 0; k < E / 4; ++k) {
    if (w[k].x) f[4 * k] = ruled(f[4 * k], w[k].x, q, bias);
    if (w[k].y) f[4 * k + 1] = ruled(f[4 * k + 1], w[k].y, q, bias);
    if (w[k].z) f[4 * k + 2] = ruled(f[4 * k + 2], w[k].z, q, bias);
    if (w[k].w) f[4 * k + 3] = ruled(f[4 * k + 3], w[k].w, q, bias);
  }
}

// Mask bits of the E tokens from v on (v >= 0, v < V); the bits above them are set.
template <int E>
__device__ __forceinline__ uint32_t mask_bits(const uint32_t* mask, int v, int V) {
  const int w = v >> 5, s = v & 31;
  const uint32_t lo = __ldg(mask + w);
  const uint32_t hi = (s > 32 - E && ((int64_t)w + 1) * 32 < V) ? __ldg(mask + w + 1) : 0u;
  return __funnelshift_r(lo, hi, s) | ~((1u << E) - 1);
}

// ------------------------------------------------------------------------------------------------------- process
constexpr int kProcessThreads = 256;

// Block (slice, row): 256 x E x U positions of the row, U chunks per thread.  The loads are issued first, so that they
// are on their way while the history is marked.
template <typename T, int U>
__global__ void __launch_bounds__(kProcessThreads, 4) process_kernel(sdm_logit_rules r, const T* logits, int64_t ld,
                                                                  int V, int slices, T* out, int64_t ld_out) {
  pdl_enter();
  constexpr int E = Chunk<T>::E, tile = kProcessThreads * E * U;
  extern __shared__ __align__(16) uint32_t word[];
  float* bias = reinterpret_cast<float*>(word + tile);
  const int64_t row = blockIdx.x / slices;
  const int slice = blockIdx.x % slices;
  const T* x = logits + row * ld;
  T* y = out + row * ld_out;
  const int off = row_offset(x);
  const bool aligned_out = row_offset(y) == off;
  const int64_t p0 = (int64_t)slice * tile;
  const int v0 = (int)(p0 - off);  // the token of word[0]
  uint4 raw[U];
#pragma unroll
  for (int k = 0; k < U; ++k) {
    const int64_t v = (int64_t)v0 + (k * kProcessThreads + (int)threadIdx.x) * E;
    raw[k] = make_uint4(0, 0, 0, 0);
    if (v >= 0 && v + E <= V) raw[k] = *reinterpret_cast<const uint4*>(x + v);
  }
  const RowRules q = row_rules(r, row, V);
  uint32_t bits[U];
#pragma unroll
  for (int k = 0; k < U; ++k) {
    const int64_t v = (int64_t)v0 + (k * kProcessThreads + (int)threadIdx.x) * E;
    bits[k] = q.mask && v >= 0 && v + E <= V ? mask_bits<E>(q.mask, (int)v, V) : 0xffffffffu;
  }
  if (q.marks) mark_tokens<kProcessThreads>(r, q, row, v0, tile, V, word, bias);
#pragma unroll
  for (int k = 0; k < U; ++k) {
    const int i = (k * kProcessThreads + (int)threadIdx.x) * E;
    const int64_t v = (int64_t)v0 + i;
    if (v >= V) break;
    const bool whole = v >= 0 && v + E <= V;
    if (whole && aligned_out) {
      float f[E];
      Chunk<T>::unpack(raw[k], f);
      if (q.marks) rule_chunk<E>(f, word + i, q, bias);
      if (q.mask) {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (!((bits[k] >> e) & 1)) f[e] = -CUDART_INF_F;
      }
      *reinterpret_cast<uint4*>(y + v) = Chunk<T>::pack(f);
    } else {
      for (int e = 0; e < E; ++e) {
        const int64_t u = v + e;
        if (u < 0 || u >= V) continue;
        float f = to_f32(x[u]);
        if (q.marks && word[i + e]) f = ruled(f, word[i + e], q, bias);
        if (q.mask && !((q.mask[u >> 5] >> (u & 31)) & 1)) f = -CUDART_INF_F;
        y[u] = from_f32<T>(f);
      }
    }
  }
}

// -------------------------------------------------------------------------------------------------------- choose
constexpr int kMaxWarps = 32;      // a block has NT = 512 or 1,024 threads
constexpr int kBins = 512;         // at most one per thread when they are scanned
constexpr int kSplit = 256;        // parts of a key range
constexpr int kList = 1024;        // candidates that one block ranks
constexpr int kRank = 128;         // more candidates of one bin are thinned out before they are ranked
constexpr int kListK = 256;        // a top_k up to this, all blocks of a row together, is found among candidates

// float -> unsigned in the same order; -0 and +0 are one value (NaN has been made -infinity).
__device__ __forceinline__ uint32_t order_key(float y) {
  const uint32_t b = __float_as_uint(__fadd_rn(y, 0.f));
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// A token's mass: exp((y - m) / T) as a whole number of 2^-40 of the largest token's.  One float32 has 24 bits, so
// nothing is rounded off a token above 2^-16 of the largest; sums (at most 2^18 tokens of 2^40) are exact in 64 bits.
__device__ __forceinline__ float scaled_gap(float y, float m, float T) {
  return y == m ? 0.f : __fdiv_rn(__fsub_rn(y, m), T);
}

// The same mass, many tokens over one T: hi * 2^20 + lo with 0 <= hi <= 2^20 and |lo| <= 2^19, by adding and taking
// off powers of two whose last place is 1 (no conversions).  The quotient is div_rn_by's, correctly rounded as
// __fdiv_rn's while T and 1 / T are normal; other temperatures divide.  At 29 T below the largest a mass is 0.
struct Masses {
  float m, T, inv, floor_;
  bool plain;
  __device__ Masses(float m_, float T_) {
    m = m_;
    T = T_;
    inv = __frcp_rn(T_);
    floor_ = -29.f * T_;
    plain = !(T_ > 1e-30f && T_ < 1e30f);
  }
  __device__ __forceinline__ void get(float y, uint32_t& hi, int& lo) const {
    const float x = y == m ? 0.f : __fsub_rn(y, m);
    float e = 0.f;
    if (x > floor_ || plain) e = expf(plain ? __fdiv_rn(x, T) : div_rn_by(x, T, inv));
    const float h = __fmaf_rn(e, 1048576.f, 8388608.f);              // 2^23 + rint(e 2^20)
    const float r = __fmaf_rn(e, 1048576.f, -__fsub_rn(h, 8388608.f));  // exact, in [-1/2, 1/2]
    const float l = __fmaf_rn(r, 1048576.f, 12582912.f);             // 2^23 + 2^22 + rint(r 2^20)
    hi = __float_as_uint(h) - 0x4b000000u;
    lo = (int)(__float_as_uint(l) - 0x4b400000u);
  }
  __device__ __forceinline__ u64 operator()(float y) const {
    uint32_t hi;
    int lo;
    get(y, hi, lo);
    return ((u64)hi << 20) + (u64)(long long)lo;
  }
};

__device__ __forceinline__ u64 warp_sum64(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ u64 warp_scan64(u64 v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 up = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += up;
  }
  return v;
}

// kept: key > cut, and of the tokens with key == cut the first `ties` in index order
struct Cut {
  uint32_t key;
  uint32_t ties, tie_count;  // kept and all tokens of that key (tie_count 0: no token has it)
  u64 mass;                  // the kept tokens' (of a search by mass, or where masses were counted)
};

struct ChooseShared {
  u64 total[kMaxCluster];
  float top[kMaxCluster];
  uint32_t ties[kMaxCluster], listed[kMaxCluster];
  int first[kMaxCluster];
  union {
    // this block's histogram: tokens, and masses in three limbs of 14 bits (a slice's tokens, under 2^16, cannot overflow one;
    // 64-bit shared atomics: 43.8 us for 33 rows of 50,021 where these took 35.5)
    struct {
      uint32_t count[kBins], limb[3][kBins];
    };
    u64 sorted[kList];              // block 0's list in order, once the histogram is done with
  };
  u64 joined_mass[kBins];           // over the cluster, then summed over the bins before:
  uint32_t joined_count[kBins];
  u64 mass_before[kBins + 1];
  uint32_t count_before[kBins + 1];
  u64 split_mass[kSplit + 1];       // the same of a split key range
  uint32_t split_count[kSplit + 1];
  u64 warp64[kMaxWarps];
  uint32_t warp32[kMaxWarps];
  uint32_t list_n;
  int bin;
  uint32_t klo, khi;
  uint32_t lo[2][kMaxCluster], hi[2][kMaxCluster];
  Cut cut;
  u64 list[kList];                  // candidates: key << 32 | ~token
};

template <int NT, int N>
__device__ __forceinline__ void clear_bins(ChooseShared& s) {
  for (int b = threadIdx.x; b < N; b += NT) s.count[b] = s.limb[0][b] = s.limb[1][b] = s.limb[2][b] = 0;
}
__device__ __forceinline__ void add_mass(ChooseShared& s, int b, u64 w) {
  const uint32_t w0 = (uint32_t)w & 0x3fffu, w1 = (uint32_t)(w >> 14) & 0x3fffu, w2 = (uint32_t)(w >> 28);
  if (w0) atomicAdd(&s.limb[0][b], w0);
  if (w1) atomicAdd(&s.limb[1][b], w1);
  if (w2) atomicAdd(&s.limb[2][b], w2);
}

// Sums over the bins before each of N bins, from a count and a mass per thread (bin).
template <int N>
__device__ void scan_bins(ChooseShared& s, uint32_t c, u64 m, u64* mass_before, uint32_t* count_before) {
  const int b = threadIdx.x, lane = b & 31, warp = b >> 5;
  uint32_t ic = c;
  u64 im = m;
  if (b < N) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t up = __shfl_up_sync(0xffffffffu, ic, o);
      if (lane >= o) ic += up;
    }
    im = warp_scan64(m, lane);
    if (lane == 31) {
      s.warp64[warp] = im;
      s.warp32[warp] = ic;
    }
  }
  __syncthreads();
  if (b < N) {
    for (int w = 0; w < warp; ++w) {
      im += s.warp64[w];
      ic += s.warp32[w];
    }
    if (b == 0) {
      mass_before[0] = 0;
      count_before[0] = 0;
    }
    mass_before[b + 1] = im;
    count_before[b + 1] = ic;
  }
  __syncthreads();
}

// Sums the blocks' histograms over the cluster (each block a share of the bins, sent to all), and over the bins.
template <int NT, int N, typename Cluster>
__device__ void join_bins(Cluster& cluster, ChooseShared& s, bool masses, u64* mass_before, uint32_t* count_before) {
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), share = N / C;
  cluster.sync();
  // thread: a bin of the share and a block, whose part it fetches and to which it sends the sum
  if (threadIdx.x < N) {
    const int b = rank * share + (int)threadIdx.x / C, r = (int)threadIdx.x % C;
    uint32_t c = *cluster.map_shared_rank(&s.count[b], r);
    u64 m = 0;
    if (masses)
      m = (u64)*cluster.map_shared_rank(&s.limb[0][b], r) + ((u64)*cluster.map_shared_rank(&s.limb[1][b], r) << 14) +
          ((u64)*cluster.map_shared_rank(&s.limb[2][b], r) << 28);
    for (int o = 1; o < C; o <<= 1) {
      c += __shfl_xor_sync(0xffffffffu, c, o);
      m += __shfl_xor_sync(0xffffffffu, m, o);
    }
    *cluster.map_shared_rank(&s.joined_count[b], r) = c;
    if (masses) *cluster.map_shared_rank(&s.joined_mass[b], r) = m;
  }
  cluster.sync();
  const int b = threadIdx.x;
  scan_bins<N>(s, b < N ? s.joined_count[b] : 0u, b < N && masses ? s.joined_mass[b] : 0, mass_before, count_before);
}

// The first of N bins through which the running count (by_count) or mass reaches `target`; N - 1 if none does.
template <int N>
__device__ __forceinline__ int find_bin(ChooseShared& s, const u64* mass_before, const uint32_t* count_before,
                                        bool by_count, u64 target) {
  const int b = threadIdx.x;
  if (b == 0) s.bin = N - 1;
  __syncthreads();
  if (b < N) {
    const u64 before = by_count ? (u64)count_before[b] : mass_before[b];
    const u64 through = by_count ? (u64)count_before[b + 1] : mass_before[b + 1];
    if (before < target && target <= through) s.bin = b;
  }
  __syncthreads();
  return s.bin;
}

// Bin of a logit: linear in its distance from the largest, so that bins hold comparable numbers of tokens.
__device__ __forceinline__ int gap_bin(float v, float m, float scale) {
  return v == m ? 0 : min(kBins - 1, (int)((m - v) * scale));
}

// This block's list of tokens: emptied, filled, and its length told to the cluster, whose number of tokens is returned
// (lists are cut at kList, and the number is then above it).
__device__ __forceinline__ void begin_list(ChooseShared& s) {
  if (threadIdx.x == 0) s.list_n = 0;
  __syncthreads();
}
template <typename Cluster>
__device__ __forceinline__ uint32_t end_list(Cluster& cluster, ChooseShared& s) {
  __syncthreads();
  if (threadIdx.x < cluster.num_blocks()) *cluster.map_shared_rank(&s.listed[cluster.block_rank()], threadIdx.x) = s.list_n;
  cluster.sync();
  uint32_t n = 0;
  for (unsigned r = 0; r < cluster.num_blocks(); ++r) n += s.listed[r];
  return n;
}
// Of the four positions from i on, those in [lo, hi) for which `take` holds.
template <typename F>
__device__ __forceinline__ void list_four(ChooseShared& s, const float* y, int i, int lo, int hi, int v0, F take) {
  const float4 q = *reinterpret_cast<const float4*>(y + i);
  const float v[4] = {q.x, q.y, q.z, q.w};
  uint32_t in = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) in |= (uint32_t)take(v[e]) << e;
  if (!in) return;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (((in >> e) & 1) && i + e >= lo && i + e < hi) {
      const uint32_t at = atomicAdd(&s.list_n, 1u);
      if (at < kList) s.list[at] = (u64)order_key(v[e]) << 32 | (0xffffffffu - (uint32_t)(v0 + i + e));
    }
  }
}

// Block 0: brings the cluster's lists (n tokens, n <= kList) together in s.list.
template <int NT, typename Cluster>
__device__ void join_lists(Cluster& cluster, ChooseShared& s) {
  uint32_t at = s.listed[0];
  for (unsigned r = 1; r < cluster.num_blocks(); ++r) {
    const uint32_t k = s.listed[r];
    const u64* from = cluster.map_shared_rank(&s.list[0], r);
    for (uint32_t i = threadIdx.x; i < k; i += NT) s.list[at + i] = from[i];
    at += k;
  }
  __syncthreads();
}

// Block 0: s.list in s.sorted, largest first.  All keys differ, so the order does not depend on how the list was filled.
template <int NT>
__device__ void sort_list(ChooseShared& s, uint32_t n) {
  // a token's rank is the number of larger ones, counted by four lanes
  for (uint32_t i0 = 0; i0 < n; i0 += NT / 4) {
    const uint32_t i = i0 + threadIdx.x / 4;
    const u64 mine = i < n ? s.list[i] : 0;
    uint32_t rank = 0;
#pragma unroll 8
    for (uint32_t j = threadIdx.x & 3; j < n; j += 4) rank += s.list[j] > mine;
    rank += __shfl_xor_sync(0xffffffffu, rank, 1);
    rank += __shfl_xor_sync(0xffffffffu, rank, 2);
    if (i < n && (threadIdx.x & 3) == 0) s.sorted[rank] = mine;
  }
  __syncthreads();
}

// Block 0, many tokens of one bin in s.list (n <= kList): keeps those of the one of kSplit equal parts of the bin in which
// the cut lies, and adds what lies above it.  Ranking is quadratic (33 rows of 50,021: 34.9 us without this, 32.3
// with).
template <int NT>
__device__ void keep_part(ChooseShared& s, const Masses& M, float scale, int B, bool by_count, bool masses, u64 target,
                          uint32_t& n, uint32_t& above, u64& above_mass) {
  constexpr int U = kList / NT;
  u64 mine[U];
  int part[U];
  clear_bins<NT, kSplit>(s);
  __syncthreads();
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t i = u * NT + threadIdx.x;
    part[u] = -1;
    if (i < n) {
      mine[u] = s.list[i];
      const float v = key_value((uint32_t)(mine[u] >> 32));
      const float gap = v == M.m ? 0.f : (M.m - v) * scale - (float)B;  // from 0 to 1, more in the last bin
      part[u] = (int)fminf(gap * kSplit, (float)(kSplit - 1));
      atomicAdd(&s.count[part[u]], 1u);
      if (masses) add_mass(s, part[u], M(v));
    }
  }
  if (threadIdx.x == 0) s.list_n = 0;
  __syncthreads();
  const int b = threadIdx.x;
  u64 m = 0;
  if (b < kSplit && masses) m = (u64)s.limb[0][b] + ((u64)s.limb[1][b] << 14) + ((u64)s.limb[2][b] << 28);
  scan_bins<kSplit>(s, b < kSplit ? s.count[b] : 0u, m, s.split_mass, s.split_count);
  const int P = find_bin<kSplit>(s, s.split_mass, s.split_count, by_count, target - (by_count ? above : above_mass));
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (part[u] == P) s.list[atomicAdd(&s.list_n, 1u)] = mine[u];
  n = s.split_count[P + 1] - s.split_count[P];
  above += s.split_count[P];
  above_mass += s.split_mass[P];
  __syncthreads();
}

// Masses of the block's two tokens sorted[2 tid], sorted[2 tid + 1] (0 from `n` on): their sum over all tokens before
// is returned, `all` is the sum over all.
template <int NT>
__device__ u64 scan_sorted(ChooseShared& s, const Masses& M, uint32_t n, u64& w0, u64& w1, u64& all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t i = 2 * threadIdx.x;
  w0 = i < n ? M(key_value((uint32_t)(s.sorted[i] >> 32))) : 0;
  w1 = i + 1 < n ? M(key_value((uint32_t)(s.sorted[i + 1] >> 32))) : 0;
  const u64 run = warp_scan64(w0 + w1, lane);
  if (lane == 31) s.warp64[warp] = run;
  __syncthreads();
  u64 before = run - w0 - w1;
  all = 0;
#pragma unroll 8
  for (int w = 0; w < (NT / 32); ++w) {
    if (w < warp) before += s.warp64[w];
    all += s.warp64[w];
  }
  __syncthreads();
  return before;
}

// Where a row's running count or mass, largest logit first, reaches `target` (1 <= target <= the row's whole), from
// the joined histogram: the bin's tokens are listed and ranked by one block.  A bin of more than kList tokens (ties, or
// a row that is almost level) has its key range split in kSplit until one key is left.
template <int NT, typename Cluster>
__device__ Cut search(Cluster& cluster, ChooseShared& s, const float* y, int lo, int hi, int v0, const Masses& M,
                      float scale, bool by_count, bool masses, u64 target, int which) {
  const int B = find_bin<kBins>(s, s.mass_before, s.count_before, by_count, target);
  u64 above_mass = s.mass_before[B];
  uint32_t above = s.count_before[B];
  begin_list(s);
#pragma unroll 2
  for (int i = threadIdx.x * 4; i < hi; i += NT * 4)
    list_four(s, y, i, lo, hi, v0, [&](float v) { return gap_bin(v, M.m, scale) == B && v > -CUDART_INF_F; });
  uint32_t n = end_list(cluster, s);
  // -infinity is not listed: where the count runs into it, all that is listed is kept
  const bool short_ = by_count && target - above > n;
  if (short_) {
    cluster.sync();  // s.listed is read before it is written again
    return {order_key(-CUDART_INF_F), 0, 0, masses ? s.mass_before[kBins] : 0};
  }
  if (n <= kList) {
    if (cluster.block_rank() == 0) {
      join_lists<NT>(cluster, s);
      if (n > kRank) keep_part<NT>(s, M, scale, B, by_count, masses, target, n, above, above_mass);
      sort_list<NT>(s, n);
      u64 w0, w1, all;
      u64 before = above_mass + scan_sorted<NT>(s, M, masses ? n : 0, w0, w1, all);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint32_t i = 2 * threadIdx.x + e;
        const u64 w = e ? w1 : w0;
        const bool here = i < n && (by_count ? above + i + 1 == target : before < target && target - before <= w);
        if (here) {
          const uint32_t key = (uint32_t)(s.sorted[i] >> 32);
          uint32_t first = i, end = i + 1;
          while (first > 0 && (uint32_t)(s.sorted[first - 1] >> 32) == key) --first;
          while (end < n && (uint32_t)(s.sorted[end] >> 32) == key) ++end;
          s.cut = {key, i + 1 - first, end - first, before + w};
        }
        before += w;
      }
      __syncthreads();
      if (threadIdx.x > 0 && threadIdx.x < cluster.num_blocks()) *cluster.map_shared_rank(&s.cut, threadIdx.x) = s.cut;
    }
    cluster.sync();
    return s.cut;
  }
  // the bin's range of keys
  if (threadIdx.x == 0) {
    s.klo = 0xffffffffu;
    s.khi = 0;
  }
  __syncthreads();
  uint32_t kl = 0xffffffffu, kh = 0;
  for (int i = lo + threadIdx.x; i < hi; i += NT) {
    const float v = y[i];
    if (gap_bin(v, M.m, scale) == B) {
      const uint32_t k = order_key(v);
      kl = min(kl, k);
      kh = max(kh, k);
    }
  }
  kl = __reduce_min_sync(0xffffffffu, kl);
  kh = __reduce_max_sync(0xffffffffu, kh);
  if ((threadIdx.x & 31) == 0) {
    atomicMin(&s.klo, kl);
    atomicMax(&s.khi, kh);
  }
  __syncthreads();
  if (threadIdx.x < cluster.num_blocks()) {
    *cluster.map_shared_rank(&s.lo[which][cluster.block_rank()], threadIdx.x) = s.klo;
    *cluster.map_shared_rank(&s.hi[which][cluster.block_rank()], threadIdx.x) = s.khi;
  }
  cluster.sync();
  kl = 0xffffffffu;
  kh = 0;
  for (unsigned r = 0; r < cluster.num_blocks(); ++r) {
    kl = min(kl, s.lo[which][r]);
    kh = max(kh, s.hi[which][r]);
  }
  uint32_t in = n;
  for (int step = 0; step < 5 && kl != kh; ++step) {  // 32-bit keys are down to one after four
    const int shift = max(0, 24 - __clz(kh - kl));
    cluster.sync();  // the histogram's last readers are done
    clear_bins<NT, kSplit>(s);
    __syncthreads();
    for (int i = lo + threadIdx.x; i < hi; i += NT) {
      const float v = y[i];
      const uint32_t k = order_key(v);
      if (k >= kl && k <= kh) {
        const int b = (kh - k) >> shift;
        atomicAdd(&s.count[b], 1u);
        if (masses) add_mass(s, b, M(v));
      }
    }
    join_bins<NT, kSplit>(cluster, s, masses, s.split_mass, s.split_count);
    const int b = find_bin<kSplit>(s, s.split_mass, s.split_count, by_count, by_count ? target - above : target - above_mass);
    in = s.split_count[b + 1] - s.split_count[b];
    above += s.split_count[b];
    above_mass += s.split_mass[b];
    kh -= (uint32_t)b << shift;
    kl = max(kl, kh - min(kh, (1u << shift) - 1));
    __syncthreads();
  }
  const u64 w = M(key_value(kl));
  const uint32_t ties = by_count ? (uint32_t)(target - above) : (uint32_t)((target - above_mass + w - 1) / max(w, (u64)1));
  return {kl, ties, in, above_mass + ties * w};
}

__device__ __forceinline__ u64 draw_target(float u, u64 K) {
  const double t = floor((double)u * (double)K);
  return min(t > 0.0 ? (u64)t : (u64)0, K - 1);  // NaN and negative: 0
}
__device__ __forceinline__ u64 share_of(float top_p, u64 W) {
  return top_p > 0.f ? max((u64)ceil((double)top_p * (double)W), (u64)1) : (u64)1;
}
__device__ __forceinline__ float log_mass(u64 K) { return logf((float)K * 9.094947017729282e-13f); }  // K / 2^40

// A cluster of blocks per row, each with a slice of the row's processed logits in shared memory.
template <typename T, int NT>
__global__ void __launch_bounds__(NT, 1024 / NT) choose_kernel(sdm_logit_rules r, sdm_choice_params c,
                                                          const T* __restrict__ logits, int64_t ld, int V, int slice,
                                                          int32_t* __restrict__ ids, float* __restrict__ logprob) {
  pdl_enter();
  constexpr int E = Chunk<T>::E, U = 4;
  extern __shared__ __align__(16) uint32_t word[];  // slice words: the marks, then in their place the logits
  __shared__ ChooseShared s;
  float* y = reinterpret_cast<float*>(word);
  float* bias = y + slice;
  auto cluster = cg::this_cluster();
  const unsigned C = cluster.num_blocks(), rank = cluster.block_rank();
  auto started = cluster.barrier_arrive();  // another block's shared memory is touched once all have started
  const int64_t row = blockIdx.x / C;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const T* x = logits + row * ld;
  const int off = row_offset(x);
  const int p0 = (int)rank * slice, v0 = p0 - off;  // v0: the token of y[0]
  const int lo = max(0, -v0), hi = max(lo, min(slice, V - v0));  // this block's tokens: v0 + [lo, hi)

  // the first loads are on their way while the marks are made
  uint4 raw[U];
  auto load = [&](int i) {
    uint4 q = make_uint4(0, 0, 0, 0);
    if (i >= lo && i + E <= hi) q = *reinterpret_cast<const uint4*>(x + v0 + i);
    return q;
  };
#pragma unroll
  for (int k = 0; k < U; ++k) raw[k] = load((k * NT + tid) * E);

  const RowRules q = row_rules(r, row, V);
  const float T0 = c.temperature ? c.temperature[row] : c.temperature_all;
  const bool greedy = !(T0 > 0.f);
  const float Tr = greedy ? 1.f : fminf(T0, FLT_MAX);  // infinite: level; a gap of infinity over it would be NaN
  const int top_k = c.top_k ? c.top_k[row] : c.top_k_all;
  const float top_p = c.top_p ? c.top_p[row] : c.top_p_all;
  const float u = c.u ? c.u[row] : 0.f;
  if (q.marks) mark_tokens<NT>(r, q, row, v0, slice, V, word, bias);
  float top = -CUDART_INF_F;  // of this thread's tokens
  for (int i0 = 0; i0 < hi; i0 += U * NT * E) {
    if (i0 > 0) {
#pragma unroll
      for (int k = 0; k < U; ++k) raw[k] = load(i0 + (k * NT + tid) * E);
    }
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int i = i0 + (k * NT + tid) * E, v = v0 + i;
      if (i >= hi) break;
      float f[E];
      const bool whole = i >= lo && i + E <= hi;
      if (whole) {
        Chunk<T>::unpack(raw[k], f);
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) f[e] = i + e >= lo && i + e < hi ? to_f32(x[v + e]) : -CUDART_INF_F;
      }
      uint32_t bits = 0xffffffffu;
      if (q.mask) {
        if (whole) {
          bits = mask_bits<E>(q.mask, v, V);
        } else {
#pragma unroll
          for (int e = 0; e < E; ++e)
            if (i + e >= lo && i + e < hi && !((q.mask[(v + e) >> 5] >> ((v + e) & 31)) & 1)) bits &= ~(1u << e);
        }
      }
      if (q.marks) rule_chunk<E>(f, word + i, q, bias);
      if (bits != 0xffffffffu) {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (!((bits >> e) & 1)) f[e] = -CUDART_INF_F;
      }
#pragma unroll
      for (int e = 0; e < E; ++e) {
        f[e] = fmaxf(f[e], -CUDART_INF_F);  // NaN is -infinity
        top = fmaxf(top, f[e]);
      }
#pragma unroll
      for (int e = 0; e < E; e += 4)
        *reinterpret_cast<float4*>(y + i + e) = make_float4(f[e], f[e + 1], f[e + 2], f[e + 3]);
    }
  }
  const bool by_k = !greedy && top_k > 0 && top_k < V, by_p = !greedy && top_p < 1.f;
  float mine = warp_max(top), low = top > -CUDART_INF_F ? -top : -CUDART_INF_F;
  low = warp_max(low);  // of the threads' largest, the smallest (negated)
  if (lane == 0) {
    s.warp64[warp] = (u64)__float_as_uint(mine) << 32 | __float_as_uint(low);
  }
  __syncthreads();
  float m = -CUDART_INF_F;
  low = -CUDART_INF_F;
#pragma unroll
  for (int w = 0; w < (NT / 32); ++w) {
    m = fmaxf(m, __uint_as_float((uint32_t)(s.warp64[w] >> 32)));
    low = fmaxf(low, __uint_as_float((uint32_t)s.warp64[w]));
  }

  // A small top_k.  A block's threads' largest logits are as many tokens of its slice, so the top_k-th largest of them
  // is at or below the slice's own: the tokens from there up (a few more than top_k) are listed, and block 0 does the
  // rest on the blocks' lists.
  if (by_k && top_k * (int)C <= kListK) {
    const float scale = (float)(kBins - 1) / (m + low);
    for (int b = tid; b < kBins; b += NT) s.count[b] = 0;
    __syncthreads();
    if (top > -CUDART_INF_F) atomicAdd(&s.count[gap_bin(top, m, scale)], 1u);
    __syncthreads();
    scan_bins<kBins>(s, tid < kBins ? s.count[tid] : 0u, 0, s.mass_before, s.count_before);
    const int last = find_bin<kBins>(s, s.mass_before, s.count_before, true, (u64)top_k);
    // below every logit of the bins 0 .. last (the last bin has all that are smaller still)
    const float least = scale > 0.f && last < kBins - 1 ? m - ((float)last + 1.01f) / scale : -CUDART_INF_F;
    cluster.barrier_wait(std::move(started));
    begin_list(s);
    if (top >= least && top > -CUDART_INF_F) {  // few threads hold one
      for (int i0 = tid * E; i0 < hi; i0 += NT * E) {
#pragma unroll
        for (int e = 0; e < E; e += 4)
          list_four(s, y, i0 + e, lo, hi, v0, [&](float v) { return v >= least && v > -CUDART_INF_F; });
      }
    }
    const uint32_t n = end_list(cluster, s);
    if (n <= kList) {
      if (rank == 0 && n == 0 && tid == 0) {  // nothing is allowed
        ids[row] = -1;
        if (logprob) logprob[row] = -CUDART_INF_F;
      }
      if (rank == 0 && n > 0) {
        join_lists<NT>(cluster, s);
        sort_list<NT>(s, n);
        const float most = key_value((uint32_t)(s.sorted[0] >> 32));
        const Masses M(most, Tr);
        const uint32_t kept = min(n, (uint32_t)top_k);
        u64* mass = s.list;  // the kept tokens' masses, by rank
        if (warp == 0) {
          u64 W = 0;
          for (uint32_t i0 = 0; i0 < kept; i0 += 32) {
            const uint32_t i = i0 + lane;
            const u64 w = i < kept ? M(key_value((uint32_t)(s.sorted[i] >> 32))) : 0;
            if (i < kept) mass[i] = w;
            W += warp_sum64(w);
          }
          const u64 share = by_p ? share_of(top_p, W) : W;
          u64 K = 0;
          uint32_t stay = 0;
          for (uint32_t i0 = 0; i0 < kept; i0 += 32) {
            const uint32_t i = i0 + lane;
            const u64 w = i < kept ? mass[i] : 0, through = K + warp_scan64(w, lane);
            const uint32_t in = __ballot_sync(0xffffffffu, i < kept && through - w < share);
            stay += __popc(in);
            const u64 end = __shfl_sync(0xffffffffu, through, in ? 31 - __clz(in) : 0);
            if (in) K = end;
            if (in != 0xffffffffu) break;
          }
          if (lane == 0) {
            s.list_n = stay;
            s.cut.mass = K;
          }
        }
        __syncthreads();
        const uint32_t stay = s.list_n;
        const u64 K = s.cut.mass, target = draw_target(u, K);
        for (uint32_t i = tid; i < stay; i += NT) {  // the mass of the kept tokens of lower index
          const uint32_t token = 0xffffffffu - (uint32_t)s.sorted[i];
          u64 run = 0;
          for (uint32_t j = 0; j < stay; ++j)
            if (0xffffffffu - (uint32_t)s.sorted[j] < token) run += mass[j];
          if (run <= target && target - run < mass[i]) {
            ids[row] = (int32_t)token;
            if (logprob) logprob[row] = scaled_gap(key_value((uint32_t)(s.sorted[i] >> 32)), most, Tr) - log_mass(K);
          }
        }
      }
      cluster.sync();  // the lists were read by block 0
      return;
    }
    cluster.sync();  // s.listed is read before it is written again
  } else {
    cluster.barrier_wait(std::move(started));
  }

  // the row's largest logit, and its first token
  if (tid < (int)C) *cluster.map_shared_rank(&s.top[rank], tid) = m;
  cluster.sync();
  for (unsigned k = 0; k < C; ++k) m = fmaxf(m, s.top[k]);
  if (m == -CUDART_INF_F) {  // nothing is allowed: the same in every block of the cluster
    if (rank == 0 && tid == 0) {
      ids[row] = -1;
      if (logprob) logprob[row] = -CUDART_INF_F;
    }
    return;
  }
  const Masses M(m, Tr);

  // what is kept
  Cut cut = {0, 0, 0, 0};  // all: every key is above 0
  if (by_k || by_p) {
    const float scale = (float)kBins / (28.5f * Tr);  // beyond exp(-28.5) a mass is 0
    clear_bins<NT, kBins>(s);
    __syncthreads();
    for (int i = lo + tid; i < hi; i += NT) {
      const float v = y[i];
      const int b = gap_bin(v, m, scale);
      if (by_k) atomicAdd(&s.count[b], 1u);
      if (by_p) add_mass(s, b, M(v));
    }
    join_bins<NT, kBins>(cluster, s, by_p, s.mass_before, s.count_before);
    u64 kept = s.mass_before[kBins];
    if (by_k) {
      cut = search<NT>(cluster, s, y, lo, hi, v0, M, scale, true, by_p, (u64)top_k, 0);
      kept = cut.mass;
    }
    if (by_p) cut = search<NT>(cluster, s, y, lo, hi, v0, M, scale, false, true, share_of(top_p, kept), 1);
  }

  // each warp's kept mass over its own stretch of the slice
  const int seg = slice / (NT / 32), s0 = max(lo, warp * seg), s1 = min(hi, (warp + 1) * seg);
  const bool partial = cut.ties < cut.tie_count;
  const u64 tie_mass = cut.tie_count ? M(key_value(cut.key)) : 0;
  uint32_t sum_hi = 0, tied = 0;
  int sum_lo = 0;
  for (int i = s0 + lane; i < s1; i += 32) {
    const float v = y[i];
    const uint32_t k = order_key(v);
    if (k > cut.key) {
      uint32_t h;
      int l;
      M.get(v, h, l);
      sum_hi += h;
      sum_lo += l;
    } else if (k == cut.key) {
      ++tied;
    }
  }
  u64 sum = warp_sum64(((u64)sum_hi << 20) + (u64)(long long)sum_lo);
  tied = __reduce_add_sync(0xffffffffu, tied);
  uint32_t tie_before = 0;
  if (partial) {  // ties are kept from the lowest index on: count the ones before this warp
    if (lane == 0) s.warp32[warp] = tied;
    __syncthreads();
    if (tid < (int)C) {
      uint32_t n = 0;
      for (int w = 0; w < (NT / 32); ++w) n += s.warp32[w];
      *cluster.map_shared_rank(&s.ties[rank], tid) = n;
    }
    cluster.sync();
    for (unsigned k = 0; k < rank; ++k) tie_before += s.ties[k];
    for (int w = 0; w < warp; ++w) tie_before += s.warp32[w];
    tied = cut.ties > tie_before ? min(tied, cut.ties - tie_before) : 0;
  }
  if (cut.tie_count) sum += (u64)tied * tie_mass;
  if (greedy) {  // the first token that has the largest logit
    int at = 0x7fffffff;
    for (int i = s1 - 1 - lane; i >= s0; i -= 32)
      if (y[i] == m) at = v0 + i;
    at = __reduce_min_sync(0xffffffffu, at);
    if (lane == 0) s.warp32[warp] = (uint32_t)at;
  }
  if (lane == 0) s.warp64[warp] = sum;
  __syncthreads();
  if (tid < (int)C) {
    u64 t = 0;
    int at = 0x7fffffff;
    for (int w = 0; w < (NT / 32); ++w) {
      t += s.warp64[w];
      at = min(at, (int)s.warp32[w]);
    }
    *cluster.map_shared_rank(&s.total[rank], tid) = t;
    *cluster.map_shared_rank(&s.first[rank], tid) = at;
  }
  cluster.sync();  // the last access to another block's shared memory is before this
  u64 K = 0, before = 0;
  for (unsigned k = 0; k < C; ++k) {
    if (k < rank) before += s.total[k];
    K += s.total[k];
  }
  const float log_k = log_mass(K);
  if (greedy) {
    if (rank == 0 && tid == 0) {
      int at = s.first[0];
      for (unsigned k = 1; k < C; ++k) at = min(at, s.first[k]);
      ids[row] = at;
      if (logprob) logprob[row] = 0.f - log_k;
    }
    return;
  }
  const u64 target = draw_target(u, K);
  for (int w = 0; w < warp; ++w) before += s.warp64[w];
  if (target < before || target - before >= sum) return;  // another warp's
  u64 left = target - before;  // the first token whose running mass in this stretch exceeds `left`
  for (int i0 = s0; i0 < s1; i0 += 32) {
    const int i = i0 + lane;
    float v = 0.f;
    uint32_t k = 0;
    if (i < s1) {
      v = y[i];
      k = order_key(v);
    }
    const bool tie = i < s1 && cut.tie_count && k == cut.key;
    const uint32_t tie_lanes = __ballot_sync(0xffffffffu, tie);
    u64 w = 0;
    if (i < s1 && k > cut.key) w = M(v);
    if (tie && (!partial || tie_before + __popc(tie_lanes & ((1u << lane) - 1)) < cut.ties)) w = tie_mass;
    tie_before += __popc(tie_lanes);
    const u64 run = warp_scan64(w, lane);
    const uint32_t over = __ballot_sync(0xffffffffu, run > left);
    if (over) {
      if (lane == __ffs(over) - 1) {
        ids[row] = v0 + i;
        if (logprob) logprob[row] = scaled_gap(v, m, Tr) - log_k;
      }
      return;
    }
    left -= __shfl_sync(0xffffffffu, run, 31);
  }
}

template <typename T, int U>
cudaError_t process_u(const sdm_logit_rules& r, const T* x, int64_t ld, int64_t S, int V, T* out, int64_t ld_out,
                      cudaStream_t st) {
  constexpr int E = Chunk<T>::E, tile = kProcessThreads * E * U;
  const int64_t slices = ceil_div((int64_t)V + E - 1, tile);
  if (slices * S > 0x7fffffff) return cudaErrorInvalidValue;
  const bool marks = (r.history && r.history_n > 0) || (r.bias_ids && r.bias_n > 0);
  LaunchScope scope_("logits_process", st);
  return launch_k(process_kernel<T, U>, dim3((unsigned)(slices * S)), dim3(kProcessThreads),
                  marks ? marks_bytes(r, tile) : 0, st, r, x, ld, V, (int)slices, out, ld_out);
}

template <typename T>
cudaError_t process_t(const sdm_logit_rules& r, const T* x, int64_t ld, int64_t S, int V, T* out, int64_t ld_out,
                      cudaStream_t st) {
  // four chunks per thread (few blocks read a row's history, many bytes are in flight) where that fills the SMs twice
  constexpr int E = Chunk<T>::E;
  if (S * ceil_div((int64_t)V + E - 1, kProcessThreads * E * 4) >= 2 * kSMs)
    return process_u<T, 4>(r, x, ld, S, V, out, ld_out, st);
  return process_u<T, 1>(r, x, ld, S, V, out, ld_out, st);
}

template <typename T, int NT>
cudaError_t choose_n(const sdm_logit_rules& r, const sdm_choice_params& c, const T* x, int64_t ld, int64_t S, int V, int C,
                     int slice, int32_t* ids, float* logprob, cudaStream_t st) {
  LaunchScope scope_("logits_choose", st);
  return launch_clusters(choose_kernel<T, NT>, (unsigned)(S * C), C, NT, marks_bytes(r, slice), st, r, c, x, ld, V, slice,
                         ids, logprob);
}

template <typename T>
cudaError_t choose_t(const sdm_logit_rules& r, const sdm_choice_params& c, const T* x, int64_t ld, int64_t S, int V,
                     int32_t* ids, float* logprob, cudaStream_t st) {
  constexpr int E = Chunk<T>::E;
  int C = 1;
  auto slice_of = [&](int n) { return (int)(ceil_div(ceil_div((int64_t)V + E - 1, n), 1024) * 1024); };
  // More blocks per row while all of them can be on the GPU together (two per SM, and a cluster within a GPC), or while
  // a slice does not fit a block's shared memory.  A block's time is mostly that of its phases, whatever
  // its slice: 256 rows of 32,768 take 34 us as whole rows, 57 in halves, 64 in quarters.
  while (C < kMaxCluster && (S * C * 2 <= 256 || slice_of(C) * 4 > 144 * 1024)) C *= 2;
  if (S * C > 0x7fffffff) return cudaErrorInvalidValue;
  const int slice = slice_of(C);
  // 1,024 threads where each still has eight tokens (33 rows of 50,021 in quarters: 34 us, 39 with 512), else 512 (one
  // row of 32,768 in eighths: 8.3 us, 9.9 with 1,024)
  if (slice > 8192) return choose_n<T, 1024>(r, c, x, ld, S, V, C, slice, ids, logprob, st);
  return choose_n<T, 512>(r, c, x, ld, S, V, C, slice, ids, logprob, st);
}

}  // namespace

cudaError_t launch_logits_process(const sdm_logit_rules& r, const void* logits, int64_t ld, int64_t S, int V,
                                  int dtype, void* out, int64_t ld_out, cudaStream_t st) {
  if (S == 0) return cudaSuccess;
  if (dtype == SDM_BF16)
    return process_t<bf16_t>(r, static_cast<const bf16_t*>(logits), ld, S, V, static_cast<bf16_t*>(out), ld_out, st);
  return process_t<float>(r, static_cast<const float*>(logits), ld, S, V, static_cast<float*>(out), ld_out, st);
}

cudaError_t launch_logits_choose(const sdm_logit_rules& r, const sdm_choice_params& c, const void* logits, int64_t ld,
                                 int64_t S, int V, int dtype, int32_t* ids, float* logprob, cudaStream_t st) {
  if (S == 0) return cudaSuccess;
  if (dtype == SDM_BF16)
    return choose_t<bf16_t>(r, c, static_cast<const bf16_t*>(logits), ld, S, V, ids, logprob, st);
  return choose_t<float>(r, c, static_cast<const float*>(logits), ld, S, V, ids, logprob, st);
}

}  // namespace sdm
