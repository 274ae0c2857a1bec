// Rules on logits (penalties for repeated tokens, biases, grammar masks) and the choice of a token from them.
//
// Both kernels split a row over blocks, each block owning a slice of the vocabulary.  A block marks, in one shared
// word per token of its slice, what the row's history and biases say about the token; then it reads its logits once,
// 16 bytes per thread, and applies the rules where a word is set.
#include <math_constants.h>
#include "vocab.cuh"

namespace sdm {
namespace {

namespace cg = cooperative_groups;
typedef unsigned long long u64;

// A token's word: it occurs in the history; it has bias entries; how often it was generated.
constexpr uint32_t kSeen = 0x80000000u, kBias = 0x40000000u, kTimes = 0x3fffffffu;

struct RowRules {
  float repetition, frequency, presence;
  const uint32_t* mask;  // this row's mask words, or null
  const int32_t* bias_ids;
  const float* bias_values;
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
  q.bias_ids = r.bias_ids + (q.bias_n ? row * r.bias_n : 0);
  q.bias_values = r.bias_values + (q.bias_n ? row * r.bias_n : 0);
  q.marks = q.bias_n > 0 || (r.history && r.history_n > 0);
  return q;
}

// Fills word[0 .. n) for tokens v0 .. v0 + n - 1 (v0 may be negative: a slice that starts before the row) from the
// row's history and biases.  Whole-number atomics: the words do not depend on their order.  Ends with a barrier.
__device__ __forceinline__ void mark_tokens(const sdm_logit_rules& r, const RowRules& q, int64_t row, int v0, int n,
                                            int V, uint32_t* word) {
  for (int i = threadIdx.x; i < n; i += blockDim.x) word[i] = 0;
  __syncthreads();
  if (!q.marks) return;
  if (r.history && r.history_n > 0) {
    int len = r.history_len ? r.history_len[row] : r.history_n;
    len = max(0, min(len, r.history_n));
    int made = r.prompt_len ? r.prompt_len[row] : 0;
    made = max(0, min(made, len));
    const int32_t* h = r.history + row * r.history_ld;
    for (int j = threadIdx.x; j < len; j += blockDim.x) {
      const int v = h[j];
      if (v < 0 || v >= V || v < v0 || v - v0 >= n) continue;
      atomicOr(&word[v - v0], kSeen);
      if (j >= made) atomicAdd(&word[v - v0], 1u);
    }
  }
  for (int j = threadIdx.x; j < q.bias_n; j += blockDim.x) {
    const int v = q.bias_ids[j];
    if (v >= 0 && v < V && v >= v0 && v - v0 < n) atomicOr(&word[v - v0], kBias);
  }
  __syncthreads();
}

// The rules of one marked token, in the plain form's order of operations (each rounded to float32, none fused), so
// that tokens the plain form ties are tied here too.
__device__ __noinline__ float ruled(float x, uint32_t w, const RowRules& q, int v) {
  if (w & kSeen) x = x > 0.f ? __fdiv_rn(x, q.repetition) : __fmul_rn(x, q.repetition);
  const uint32_t g = w & kTimes;
  if (g) {
    x = __fsub_rn(x, __fmul_rn(q.frequency, (float)g));
    x = __fsub_rn(x, q.presence);
  }
  if (w & kBias) {
    float b = 0.f;
    for (int j = 0; j < q.bias_n; ++j)
      if (q.bias_ids[j] == v) b = __fadd_rn(b, q.bias_values[j]);
    x = __fadd_rn(x, b);
  }
  return x;
}

// Mask bits of the E tokens from v on (v >= 0, v < V).
template <int E>
__device__ __forceinline__ uint32_t mask_bits(const uint32_t* mask, int v, int V) {
  const int w = v >> 5, s = v & 31;
  const uint32_t lo = __ldg(mask + w);
  const uint32_t hi = (s > 32 - E && ((int64_t)w + 1) * 32 < V) ? __ldg(mask + w + 1) : 0u;
  return __funnelshift_r(lo, hi, s);
}

// ------------------------------------------------------------------------------------------------------- process
// Block (slice, row): positions [slice * tile, +tile) of the row.
template <typename T>
__global__ void __launch_bounds__(256) process_kernel(sdm_logit_rules r, const T* logits, int64_t ld,
                                                      int V, int tile, int slices, T* out, int64_t ld_out) {
  pdl_enter();
  constexpr int E = Chunk<T>::E;
  extern __shared__ uint32_t word[];
  const int64_t row = blockIdx.x / slices;
  const int slice = blockIdx.x % slices;
  const T* x = logits + row * ld;
  T* y = out + row * ld_out;
  const int off = row_offset(x);
  const bool aligned_out = row_offset(y) == off;
  const int p0 = slice * tile;
  const RowRules q = row_rules(r, row, V);
  if (q.marks) mark_tokens(r, q, row, p0 - off, tile, V, word);
  const int p1 = min(p0 + tile, V + off);
  for (int p = p0 + (int)threadIdx.x * E; p < p1; p += blockDim.x * E) {
    const int v = p - off;
    if (v >= 0 && v + E <= V && aligned_out) {
      float f[E];
      Chunk<T>::unpack(*reinterpret_cast<const uint4*>(x + v), f);
      if (q.marks) {
#pragma unroll
        for (int e = 0; e < E; e += 4) {
          const uint4 w = *reinterpret_cast<const uint4*>(word + (p - p0) + e);
          if (w.x) f[e] = ruled(f[e], w.x, q, v + e);
          if (w.y) f[e + 1] = ruled(f[e + 1], w.y, q, v + e + 1);
          if (w.z) f[e + 2] = ruled(f[e + 2], w.z, q, v + e + 2);
          if (w.w) f[e + 3] = ruled(f[e + 3], w.w, q, v + e + 3);
        }
      }
      if (q.mask) {
        const uint32_t b = mask_bits<E>(q.mask, v, V);
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (!((b >> e) & 1)) f[e] = -CUDART_INF_F;
      }
      *reinterpret_cast<uint4*>(y + v) = Chunk<T>::pack(f);
    } else {
      for (int e = 0; e < E; ++e) {
        const int u = v + e;
        if (u < 0 || u >= V) continue;
        float f = to_f32(x[u]);
        if (q.marks && word[p - p0 + e]) f = ruled(f, word[p - p0 + e], q, u);
        if (q.mask && !((q.mask[u >> 5] >> (u & 31)) & 1)) f = -CUDART_INF_F;
        y[u] = from_f32<T>(f);
      }
    }
  }
}

// -------------------------------------------------------------------------------------------------------- choose
constexpr int kThreads = 512, kWarps = kThreads / 32, kBins = 256;

// float -> unsigned in the same order (-0 has been made +0, NaN -infinity).
__device__ __forceinline__ uint32_t order_key(float y) {
  const uint32_t b = __float_as_uint(y);
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
__device__ __forceinline__ u64 mass_of(float y, float m, float T) {
  return __float2ull_rn(__fmul_rn(expf(scaled_gap(y, m, T)), 1099511627776.f));
}

__device__ __forceinline__ u64 warp_sum64(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

struct ChooseShared {
  u64 best[kMaxCluster], total[kMaxCluster];
  uint32_t ties[kMaxCluster];
  uint32_t lo[2][kMaxCluster], hi[2][kMaxCluster];
  u64 mass[2][kBins];        // this block's histogram, two buffers in turn
  uint32_t count[2][kBins];
  u64 mass_before[kBins + 1];       // over the cluster: of the bins above each bin
  uint32_t count_before[kBins + 1];
  u64 first_mass[kBins + 1];        // the first histogram's, kept for the second search
  uint32_t first_count[kBins + 1];
  u64 warp64[kWarps];
  uint32_t warp32[kWarps];
  int bin;
  uint32_t klo, khi;
};

// kept: key > cut, and of the tokens with key == cut the first `ties` in index order
struct Cut {
  uint32_t key;
  uint32_t ties, tie_count;  // kept and all tokens of that key (tie_count 0: key is below every kept token)
  u64 mass;                  // all kept tokens'
};

// Sums this block's histogram `buf` over the cluster, and writes its sums over the bins before each bin.
template <typename Cluster>
__device__ void join_bins(Cluster& cluster, ChooseShared& s, int buf, u64* mass_before, uint32_t* count_before) {
  cluster.sync();
  const int b = threadIdx.x, lane = b & 31, warp = b >> 5;
  u64 m = 0;
  uint32_t c = 0;
  if (b < kBins) {
    for (unsigned r = 0; r < cluster.num_blocks(); ++r) {
      m += *cluster.map_shared_rank(&s.mass[buf][b], r);
      c += *cluster.map_shared_rank(&s.count[buf][b], r);
    }
    u64 im = m;
    uint32_t ic = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 um = __shfl_up_sync(0xffffffffu, im, o);
      const uint32_t uc = __shfl_up_sync(0xffffffffu, ic, o);
      if (lane >= o) {
        im += um;
        ic += uc;
      }
    }
    if (lane == 31) {
      s.warp64[warp] = im;
      s.warp32[warp] = ic;
    }
    m = im - m;
    c = ic - c;
  }
  __syncthreads();
  if (b < kBins) {
    for (int w = 0; w < warp; ++w) {
      m += s.warp64[w];
      c += s.warp32[w];
    }
    mass_before[b] = m;
    count_before[b] = c;
    if (b == kBins - 1) {
      u64 tm = 0;
      uint32_t tc = 0;
      for (int w = 0; w < kBins / 32; ++w) {
        tm += s.warp64[w];
        tc += s.warp32[w];
      }
      mass_before[kBins] = tm;
      count_before[kBins] = tc;
    }
  }
  __syncthreads();
}

// The bin in which the running count (by_count) or mass reaches `target`.
__device__ __forceinline__ int find_bin(ChooseShared& s, const u64* mass_before, const uint32_t* count_before,
                                        bool by_count, u64 target) {
  const int b = threadIdx.x;
  if (b < kBins) {
    const u64 before = by_count ? (u64)count_before[b] : mass_before[b];
    const u64 through = by_count ? (u64)count_before[b + 1] : mass_before[b + 1];
    if (before < target && target <= through) s.bin = b;
  }
  __syncthreads();
  const int bin = s.bin;
  __syncthreads();
  return bin;
}

// Where a row's running count or mass, largest logit first, reaches `target` (1 <= target <= the row's whole).  The
// first histogram is linear in m - y; below it the bin's key range is split in 256 until one key, or one token, is
// left: masses are exact whole numbers, so every step is.
template <typename Cluster>
__device__ Cut search(Cluster& cluster, ChooseShared& s, const float* y, int lo, int hi, float m, float T, float inv,
                      bool by_count, u64 target, int which, int& buf) {
  const int B = find_bin(s, s.first_mass, s.first_count, by_count, target);
  u64 above_mass = s.first_mass[B], in_mass = s.first_mass[B + 1] - above_mass;
  uint32_t above = s.first_count[B], in = s.first_count[B + 1] - above;
  // the bin's range of keys
  if (threadIdx.x == 0) {
    s.klo = 0xffffffffu;
    s.khi = 0;
  }
  __syncthreads();
  uint32_t kl = 0xffffffffu, kh = 0;
  for (int i = lo + threadIdx.x; i < hi; i += kThreads) {
    const float v = y[i];
    const int b = v == m ? 0 : min(kBins - 1, (int)((m - v) * inv));
    if (b == B) {
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
  // keys kl .. kh hold `in` tokens of in_mass; `above` tokens of above_mass are larger
  for (int step = 0; step < 6; ++step) {  // 32-bit keys are down to one after four
    if (by_count ? target - above == in : in == 1) return {kl - 1, 0, 0, above_mass + in_mass};
    if (kl == kh) {
      const u64 w = mass_of(key_value(kl), m, T);
      const uint32_t ties = by_count ? (uint32_t)(target - above) : (uint32_t)((target - above_mass + w - 1) / w);
      return {kl, ties, in, above_mass + ties * w};
    }
    const int shift = max(0, 24 - __clz(kh - kl));
    for (int b = threadIdx.x; b < kBins; b += kThreads) {
      s.mass[buf][b] = 0;
      s.count[buf][b] = 0;
    }
    __syncthreads();
    for (int i = lo + threadIdx.x; i < hi; i += kThreads) {
      const float v = y[i];
      const uint32_t k = order_key(v);
      if (k >= kl && k <= kh) {
        const int b = (kh - k) >> shift;
        atomicAdd(&s.count[buf][b], 1u);
        atomicAdd(&s.mass[buf][b], mass_of(v, m, T));
      }
    }
    join_bins(cluster, s, buf, s.mass_before, s.count_before);
    buf ^= 1;
    const int b = find_bin(s, s.mass_before, s.count_before, by_count, by_count ? target - above : target - above_mass);
    in = s.count_before[b + 1] - s.count_before[b];
    in_mass = s.mass_before[b + 1] - s.mass_before[b];
    above += s.count_before[b];
    above_mass += s.mass_before[b];
    kh -= (uint32_t)b << shift;
    kl = max(kl, kh - min(kh, (1u << shift) - 1));
    __syncthreads();
  }
  return {kl - 1, 0, 0, above_mass + in_mass};
}

// A cluster of blocks per row, each with a slice of the row's processed logits in shared memory.
template <typename T>
__global__ void __launch_bounds__(kThreads) choose_kernel(sdm_logit_rules r, sdm_choice_params c,
                                                          const T* __restrict__ logits, int64_t ld, int V, int slice,
                                                          int32_t* __restrict__ ids, float* __restrict__ logprob) {
  pdl_enter();
  constexpr int E = Chunk<T>::E;
  extern __shared__ __align__(16) uint32_t word[];  // slice words: the marks, then in their place the logits
  __shared__ ChooseShared s;
  float* y = reinterpret_cast<float*>(word);
  auto cluster = cg::this_cluster();
  const unsigned C = cluster.num_blocks(), rank = cluster.block_rank();
  auto started = cluster.barrier_arrive();  // another block's shared memory is touched once all have started
  const int64_t row = blockIdx.x / C;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const T* x = logits + row * ld;
  const int off = row_offset(x);
  const int p0 = (int)rank * slice;
  const RowRules q = row_rules(r, row, V);
  const float T0 = c.temperature ? c.temperature[row] : c.temperature_all;
  const bool greedy = !(T0 > 0.f);
  const float Tr = greedy ? 1.f : T0;
  const int top_k = c.top_k ? c.top_k[row] : c.top_k_all;
  const float top_p = c.top_p ? c.top_p[row] : c.top_p_all;
  const int lo = max(0, off - p0), hi = max(lo, min(slice, V + off - p0));  // this block's tokens: p0 - off + [lo, hi)

  if (q.marks) mark_tokens(r, q, row, p0 - off, slice, V, word);
  u64 best = 0;
  for (int i = tid * E; i < hi; i += kThreads * E) {
    const int v = p0 + i - off;
    float f[E];
    const bool whole = v >= 0 && v + E <= V;
    if (whole) {
      Chunk<T>::unpack(*reinterpret_cast<const uint4*>(x + v), f);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) f[e] = v + e >= 0 && v + e < V ? to_f32(x[v + e]) : -CUDART_INF_F;
    }
    uint32_t bits = 0xffffffffu;
    if (q.mask) {
      if (whole) {
        bits = mask_bits<E>(q.mask, v, V);
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (v + e >= 0 && v + e < V && !((q.mask[(v + e) >> 5] >> ((v + e) & 31)) & 1)) bits &= ~(1u << e);
      }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (q.marks && word[i + e]) f[e] = ruled(f[e], word[i + e], q, v + e);
      if (!((bits >> e) & 1) || isnan(f[e])) f[e] = -CUDART_INF_F;
      f[e] = __fadd_rn(f[e], 0.f);  // -0 and +0 are one value in the order
      if (v + e >= 0 && v + e < V) best = max(best, (u64)order_key(f[e]) << 32 | (0xffffffffu - (uint32_t)(v + e)));
    }
#pragma unroll
    for (int e = 0; e < E; e += 4) *reinterpret_cast<float4*>(y + i + e) = make_float4(f[e], f[e + 1], f[e + 2], f[e + 3]);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
  if (lane == 0) s.warp64[warp] = best;
  __syncthreads();
  cluster.barrier_wait(std::move(started));
  if (tid < (int)C) {
    u64 b = 0;
    for (int w = 0; w < kWarps; ++w) b = max(b, s.warp64[w]);
    *cluster.map_shared_rank(&s.best[rank], tid) = b;
  }
  cluster.sync();
  best = 0;
  for (unsigned k = 0; k < C; ++k) best = max(best, s.best[k]);
  const float m = key_value((uint32_t)(best >> 32));
  if (m == -CUDART_INF_F) {  // nothing is allowed: the same in every block of the cluster
    if (rank == 0 && tid == 0) {
      ids[row] = -1;
      if (logprob) logprob[row] = -CUDART_INF_F;
    }
    return;
  }

  // what is kept
  Cut cut = {0, 0, 0, 0};  // all: every key is above 0
  const bool by_k = !greedy && top_k > 0 && top_k < V, by_p = !greedy && top_p < 1.f;
  if (by_k || by_p) {
    const float inv = (float)kBins / (28.1f * Tr);  // beyond exp(-28.1) a mass is 0
    for (int b = tid; b < kBins; b += kThreads) {
      s.mass[0][b] = 0;
      s.count[0][b] = 0;
    }
    __syncthreads();
    for (int i = lo + tid; i < hi; i += kThreads) {
      const float v = y[i];
      const int b = v == m ? 0 : min(kBins - 1, (int)((m - v) * inv));
      atomicAdd(&s.count[0][b], 1u);
      const u64 w = mass_of(v, m, Tr);
      if (w) atomicAdd(&s.mass[0][b], w);
    }
    join_bins(cluster, s, 0, s.first_mass, s.first_count);
    int buf = 1;
    u64 kept = s.first_mass[kBins];
    if (by_k) {
      cut = search(cluster, s, y, lo, hi, m, Tr, inv, true, (u64)top_k, 0, buf);
      kept = cut.mass;
    }
    if (by_p) {
      const u64 share = (u64)ceil((double)top_p * (double)kept);  // a negative or NaN top_p keeps one token
      cut = search(cluster, s, y, lo, hi, m, Tr, inv, false, top_p > 0.f ? max(share, (u64)1) : (u64)1, 1, buf);
    }
  }

  // each warp's kept mass over its own stretch of the slice
  const int seg = slice / kWarps, s0 = max(lo, warp * seg), s1 = min(hi, (warp + 1) * seg);
  const bool partial = cut.ties < cut.tie_count;
  const u64 tie_mass = cut.tie_count ? mass_of(key_value(cut.key), m, Tr) : 0;
  u64 sum = 0;
  uint32_t tied = 0;
  for (int i = s0 + lane; i < s1; i += 32) {
    const float v = y[i];
    const uint32_t k = order_key(v);
    if (k > cut.key) sum += mass_of(v, m, Tr);
    else if (k == cut.key) ++tied;
  }
  sum = warp_sum64(sum);
  tied = __reduce_add_sync(0xffffffffu, tied);
  uint32_t tie_before = 0;
  if (partial) {  // ties are kept from the lowest index on: count the ones before this warp
    if (lane == 0) s.warp32[warp] = tied;
    __syncthreads();
    if (tid < (int)C) {
      uint32_t n = 0;
      for (int w = 0; w < kWarps; ++w) n += s.warp32[w];
      *cluster.map_shared_rank(&s.ties[rank], tid) = n;
    }
    cluster.sync();
    for (unsigned k = 0; k < rank; ++k) tie_before += s.ties[k];
    for (int w = 0; w < warp; ++w) tie_before += s.warp32[w];
    tied = cut.ties > tie_before ? min(tied, cut.ties - tie_before) : 0;
  }
  if (cut.tie_count) sum += (u64)tied * tie_mass;
  if (lane == 0) s.warp64[warp] = sum;
  __syncthreads();
  if (tid < (int)C) {
    u64 t = 0;
    for (int w = 0; w < kWarps; ++w) t += s.warp64[w];
    *cluster.map_shared_rank(&s.total[rank], tid) = t;
  }
  cluster.sync();  // the last access to another block's shared memory is before this
  u64 K = 0, before = 0;
  for (unsigned k = 0; k < C; ++k) {
    if (k < rank) before += s.total[k];
    K += s.total[k];
  }
  const float log_k = logf((float)K * 9.094947017729282e-13f);  // K / 2^40
  if (greedy) {
    if (rank == 0 && tid == 0) {
      ids[row] = (int32_t)(0xffffffffu - (uint32_t)best);
      if (logprob) logprob[row] = 0.f - log_k;
    }
    return;
  }
  const float u = c.u ? c.u[row] : 0.f;
  const double ur = floor((double)u * (double)K);
  u64 target = ur > 0.0 ? (u64)ur : 0;  // NaN and negative: 0
  target = min(target, K - 1);
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
    if (i < s1 && k > cut.key) w = mass_of(v, m, Tr);
    if (tie && (!partial || tie_before + __popc(tie_lanes & ((1u << lane) - 1)) < cut.ties)) w = tie_mass;
    tie_before += __popc(tie_lanes);
    u64 run = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 up = __shfl_up_sync(0xffffffffu, run, o);
      if (lane >= o) run += up;
    }
    const uint32_t over = __ballot_sync(0xffffffffu, run > left);
    if (over) {
      if (lane == __ffs(over) - 1) {
        ids[row] = p0 + i - off;
        if (logprob) logprob[row] = scaled_gap(v, m, Tr) - log_k;
      }
      return;
    }
    left -= __shfl_sync(0xffffffffu, run, 31);
  }
}

template <typename T>
cudaError_t process_t(const sdm_logit_rules& r, const T* x, int64_t ld, int64_t S, int V, T* out, int64_t ld_out,
                      cudaStream_t st) {
  // the largest slice (so that a row's history is read by few blocks) that still gives every SM two blocks
  int tile = 16384;
  while (tile > 1024 && ceil_div((int64_t)V + 7, tile) * S < 2 * kSMs) tile /= 2;
  const int64_t slices = ceil_div((int64_t)V + 7, tile);
  if (slices * S > 0x7fffffff) return cudaErrorInvalidValue;
  const size_t smem = (size_t)tile * 4;
  cudaError_t e = cudaFuncSetAttribute(process_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, 16384 * 4);
  if (e != cudaSuccess) return e;
  LaunchScope scope_("logits_process", st);
  return launch_k(process_kernel<T>, dim3((unsigned)(slices * S)), dim3(256), smem, st, r, x, ld, V, tile, (int)slices,
                  out, ld_out);
}

template <typename T>
cudaError_t choose_t(const sdm_logit_rules& r, const sdm_choice_params& c, const T* x, int64_t ld, int64_t S, int V,
                     int32_t* ids, float* logprob, cudaStream_t st) {
  constexpr int E = Chunk<T>::E;
  int C = 1;
  auto slice_of = [&](int n) { return (int)(ceil_div(ceil_div((int64_t)V + E - 1, n), kThreads) * kThreads); };
  while (C < kMaxCluster && (S * C < kSMs || slice_of(C) * 4 > 100 * 1024)) C *= 2;
  if (S * C > 0x7fffffff) return cudaErrorInvalidValue;
  const int slice = slice_of(C);
  LaunchScope scope_("logits_choose", st);
  return launch_clusters(choose_kernel<T>, (unsigned)(S * C), C, kThreads, (size_t)slice * 4, st, r, c, x, ld, V, slice,
                         ids, logprob);
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
