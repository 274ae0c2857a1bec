// The scaled token lookup and its gradient, the sum of dout's rows over the positions of each token.
//
// Gradient.  group_kernel sorts the positions by token (a counting sort; each block owns the tokens of one remainder
// and scans all ids, so blocks exchange nothing).  sum_kernel adds up each token's rows in order; a token with more
// than kPiece positions is summed in pieces cut at multiples of kPiece of the sorted order, spread over the GPU, which
// join_kernel adds in order.  No float atomics: the result is a function of the inputs alone.
#include "vocab.cuh"

namespace sdm {
namespace {

constexpr int kPiece = 32;       // positions summed by one warp
constexpr int kGroupThreads = 1024, kGroupWarps = kGroupThreads / 32;
constexpr int kSumThreads = 256, kSumWarps = kSumThreads / 32;
constexpr int kCols = 256;       // columns of one warp's sum

struct GroupWs {
  int32_t *order;    // (N) positions, grouped by token
  int32_t *start;    // (V) where a token's group begins
  int32_t *count;    // (V)
  int32_t *hot;      // (owners, tokens of an owner): tokens with more than kPiece positions, by owner
  int32_t *hot_n;    // (owners)
  int32_t *total;    // grouped positions
  float *partial;    // (2 * pieces, d)
};

__host__ int owner_bits(int V) {  // 128 blocks, more where an owner's tokens would exceed a block's 1,024 counters
  int b = 7;
  while (((int64_t)1 << b) * 1024 < V) ++b;
  return b;
}

size_t carve(GroupWs& w, void* base, int64_t N, int d, int V) {
  size_t off = 0;
  auto take = [&](size_t bytes) {
    char* p = base ? static_cast<char*>(base) + off : nullptr;
    off += (bytes + 255) & ~(size_t)255;
    return p;
  };
  const int64_t owners = (int64_t)1 << owner_bits(V), per = ceil_div(V, owners);
  w.order = reinterpret_cast<int32_t*>(take(N * 4));
  w.start = reinterpret_cast<int32_t*>(take((size_t)V * 4));
  w.count = reinterpret_cast<int32_t*>(take((size_t)V * 4));
  w.hot = reinterpret_cast<int32_t*>(take(owners * per * 4));
  w.hot_n = reinterpret_cast<int32_t*>(take(owners * 4));
  w.total = reinterpret_cast<int32_t*>(take(4));
  w.partial = reinterpret_cast<float*>(take((size_t)2 * ceil_div(N, kPiece) * d * 4));
  return off;
}

// Block b owns the tokens v with v mod owners == b (v = local * owners + b).  Each warp counts and later places one
// stretch of the ids, so the sort is stable.
__global__ void __launch_bounds__(kGroupThreads) group_kernel(const int32_t* __restrict__ ids, int N, int V, int bits,
                                                              int per, int padding_id, GroupWs w) {
  pdl_enter();
  extern __shared__ uint32_t count[];  // (warps, per)
  __shared__ uint32_t warp_sum_[kGroupWarps];
  __shared__ uint32_t hot_n;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t me = blockIdx.x, low = (1u << bits) - 1;
  for (int i = tid; i < kGroupWarps * per; i += kGroupThreads) count[i] = 0;
  if (tid == 0) hot_n = 0;
  __syncthreads();
  const int seg = (int)(ceil_div(ceil_div(N, kGroupWarps), 32) * 32);
  const int n0 = (int)min((int64_t)N, (int64_t)warp * seg), n1 = (int)min((int64_t)N, (int64_t)n0 + seg);
  uint32_t* mine = count + warp * per;
  uint32_t below = 0;
  for (int n = n0 + lane; n < n1; n += 32) {
    const int id = ids[n];
    if (id < 0 || id >= V || id == padding_id) continue;
    const uint32_t owner = (uint32_t)id & low;
    below += owner < me;
    if (owner == me) atomicAdd(&mine[id >> bits], 1u);
  }
  below = __reduce_add_sync(0xffffffffu, below);
  if (lane == 0) warp_sum_[warp] = below;
  __syncthreads();
  uint32_t base = 0;
  for (int i = 0; i < kGroupWarps; ++i) base += warp_sum_[i];
  __syncthreads();
  // the group of local token tid: its size, then its start
  uint32_t size = 0;
  if (tid < per)
    for (int i = 0; i < kGroupWarps; ++i) {
      const uint32_t c = count[i * per + tid];
      count[i * per + tid] = size;
      size += c;
    }
  uint32_t run = size;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t up = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= o) run += up;
  }
  if (lane == 31) warp_sum_[warp] = run;
  __syncthreads();
  uint32_t first = base + run - size;
  for (int i = 0; i < warp; ++i) first += warp_sum_[i];
  if (tid < per) {
    const int64_t v = ((int64_t)tid << bits) + me;
    if (v < V) {
      w.start[v] = (int32_t)first;
      w.count[v] = (int32_t)size;
      if (size > kPiece) w.hot[(int64_t)me * per + atomicAdd(&hot_n, 1u)] = (int32_t)v;
    }
    for (int i = 0; i < kGroupWarps; ++i) count[i * per + tid] += first;
  }
  if (me == low && tid == kGroupThreads - 1) *w.total = (int32_t)(first + size);
  __syncthreads();
  if (tid == 0) w.hot_n[me] = (int32_t)hot_n;
  for (int nb = n0; nb < n1; nb += 32) {
    const int n = nb + lane;
    const int id = n < n1 ? ids[n] : -1;
    const bool owned = id >= 0 && id < V && id != padding_id && ((uint32_t)id & low) == me;
    if (!__any_sync(0xffffffffu, owned)) continue;
    const int local = owned ? id >> bits : -1;
    const uint32_t same = __match_any_sync(0xffffffffu, local);
    const int rank = __popc(same & ((1u << lane) - 1));
    uint32_t at = 0;
    if (owned) at = mine[local] + rank;
    __syncwarp();
    if (owned) {
      w.order[at] = n;
      if (rank == 0) mine[local] += __popc(same);
    }
    __syncwarp();
  }
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

// One warp's sum over positions order[j0 .. j1) of the 256 columns from c0 on; lane's columns are c0 + VEC * (lane +
// 32 q) + e.
template <typename T, int VEC>
struct Sum {
  static constexpr int NQ = kCols / (32 * VEC);
  float acc[NQ][VEC];

  __device__ void run(const T* __restrict__ dout, int64_t ld, const int32_t* __restrict__ order, int j0, int j1,
                      int c0, int d) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int q = 0; q < NQ; ++q)
#pragma unroll
      for (int e = 0; e < VEC; ++e) acc[q][e] = 0.f;
    for (int jb = j0; jb < j1; jb += 32) {
      const int n = min(32, j1 - jb);
      const int pos = lane < n ? order[jb + lane] : 0;
#pragma unroll 4
      for (int j = 0; j < n; ++j) {
        const T* r = dout + (int64_t)__shfl_sync(0xffffffffu, pos, j) * ld;
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
          const int c = c0 + VEC * (lane + 32 * q);
          if (c < d) {
            const Pack<T, VEC> p = {__ldg(reinterpret_cast<const typename Word<VEC * sizeof(T)>::type*>(r + c))};
#pragma unroll
            for (int e = 0; e < VEC; ++e) acc[q][e] += p.get(e);
          }
        }
      }
    }
  }
};

template <typename G, int VEC>
__device__ __forceinline__ void store_grad(G* at, const float* v, float scale, int accumulate) {
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    const float s = v[e] * scale;
    at[e] = from_f32<G>(accumulate ? to_f32(at[e]) + s : s);
  }
}

// Items: (token, 256 columns) for every token, then (piece, 256 columns).
template <typename T, typename G, int VEC>
__global__ void __launch_bounds__(kSumThreads) sum_kernel(const int32_t* __restrict__ ids, const T* __restrict__ dout,
                                                          int64_t ld, int d, int V, int col_blocks, int64_t items,
                                                          float scale, int accumulate, GroupWs w,
                                                          G* __restrict__ grad) {
  pdl_enter();
  const int64_t item = (int64_t)blockIdx.x * kSumWarps + (threadIdx.x >> 5);
  if (item >= items) return;
  const int lane = threadIdx.x & 31;
  const int64_t what = item / col_blocks;
  const int c0 = (int)(item % col_blocks) * kCols;
  Sum<T, VEC> s;
  if (what < V) {
    const int n = w.count[what];
    if (n > kPiece || (n == 0 && accumulate)) return;
    const int j0 = w.start[what];
    s.run(dout, ld, w.order, j0, j0 + n, c0, d);
#pragma unroll
    for (int q = 0; q < Sum<T, VEC>::NQ; ++q) {
      const int c = c0 + VEC * (lane + 32 * q);
      if (c < d) store_grad<G, VEC>(grad + what * d + c, s.acc[q], scale, accumulate);
    }
    return;
  }
  const int64_t piece = what - V;
  const int total = *w.total;
  const int j0 = (int)(piece * kPiece), j1 = min(total, j0 + kPiece);
  if (j0 >= j1) return;
  const int a = ids[w.order[j0]], b = ids[w.order[j1 - 1]];
#pragma unroll
  for (int side = 0; side < 2; ++side) {  // the group that the piece begins in, and the one that begins in it
    const int v = side ? b : a;
    if (side && b == a) break;
    const int n = w.count[v];
    if (n <= kPiece) continue;
    const int g0 = w.start[v], g1 = g0 + n;
    s.run(dout, ld, w.order, max(g0, j0), min(g1, j1), c0, d);
    float* out = w.partial + (2 * piece + side) * d;
#pragma unroll
    for (int q = 0; q < Sum<T, VEC>::NQ; ++q) {
      const int c = c0 + VEC * (lane + 32 * q);
      if (c < d) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) out[c + e] = s.acc[q][e];
      }
    }
  }
}

// Block (owner, 32 columns): adds up the pieces of the owner's large groups.  Warp w takes every eighth piece, and the
// warps' sums are added in order.
template <typename G>
__global__ void __launch_bounds__(256) join_kernel(int d, int per, float scale, int accumulate, GroupWs w,
                                                   G* __restrict__ grad) {
  pdl_enter();
  __shared__ float part[8][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int n = w.hot_n[blockIdx.x];
  const int c = blockIdx.y * 32 + lane;
  for (int i = 0; i < n; ++i) {
    const int64_t v = w.hot[(int64_t)blockIdx.x * per + i];
    const int g0 = w.start[v], g1 = g0 + w.count[v];
    const int m0 = g0 / kPiece, m1 = (g1 - 1) / kPiece;
    float sum = 0.f;
    if (c < d) {
#pragma unroll 4
      for (int m = m0 + warp; m <= m1; m += 8)
        sum += w.partial[(2 * (int64_t)m + (g0 > m * kPiece ? 1 : 0)) * d + c];
    }
    part[warp][lane] = sum;
    __syncthreads();
    if (warp == 0 && c < d) {
#pragma unroll
      for (int k = 1; k < 8; ++k) sum += part[k][lane];
      store_grad<G, 1>(grad + v * d + c, &sum, scale, accumulate);
    }
    __syncthreads();
  }
}

template <typename T, int VEC>
__global__ void __launch_bounds__(256) lookup_kernel(const int32_t* __restrict__ ids, const T* __restrict__ emb,
                                                     int64_t N, int d, int V, float scale, T* __restrict__ out,
                                                     int* bad) {
  pdl_enter();
  const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= N) return;
  const int id = ids[row];
  const bool ok = id >= 0 && id < V;
  if (!ok && lane == 0 && bad) atomicExch(bad, 1);
  typedef typename Word<VEC * sizeof(T)>::type W;
  for (int c = VEC * lane; c < d; c += VEC * 32) {
    union {
      W u;
      T t[VEC];
    } y;
    if (ok) {
      y.u = __ldg(reinterpret_cast<const W*>(emb + (int64_t)id * d + c));
#pragma unroll
      for (int e = 0; e < VEC; ++e) y.t[e] = from_f32<T>(to_f32(y.t[e]) * scale);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) y.t[e] = from_f32<T>(0.f);
    }
    *reinterpret_cast<W*>(out + row * d + c) = y.u;
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

template <typename T, typename G, int VEC>
cudaError_t launch_sum(const int32_t* ids, const T* dout, int64_t ld, int64_t N, int d, int V, float scale,
                       int accumulate, const GroupWs& w, G* grad, cudaStream_t st) {
  const int col_blocks = (int)ceil_div(d, kCols);
  const int64_t items = (V + ceil_div(N, kPiece)) * col_blocks, blocks = ceil_div(items, kSumWarps);
  if (blocks > 0x7fffffff) return cudaErrorInvalidValue;
  LaunchScope scope_("embed_grad_sum", st);
  return launch_k(sum_kernel<T, G, VEC>, dim3((unsigned)blocks), dim3(kSumThreads), 0, st, ids, dout, ld, d, V,
                  col_blocks, items, scale, accumulate, w, grad);
}

template <typename T, typename G>
cudaError_t grad_t(const int32_t* ids, const T* dout, int64_t ld, int64_t N, int d, int V, float scale,
                   int padding_id, int accumulate, G* grad, void* ws, cudaStream_t st) {
  GroupWs w;
  carve(w, ws, N, d, V);
  const int bits = owner_bits(V), owners = 1 << bits, per = (int)ceil_div(V, owners);
  const size_t smem = (size_t)kGroupWarps * per * 4;
  cudaError_t e = cudaFuncSetAttribute(group_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kGroupWarps * 1024 * 4);
  if (e != cudaSuccess) return e;
  {
    LaunchScope scope_("embed_grad_group", st);
    e = launch_k(group_kernel, dim3((unsigned)owners), dim3(kGroupThreads), smem, st, ids, (int)N, V, bits, per,
                 padding_id, w);
    if (e != cudaSuccess) return e;
  }
  switch (vec_of(16 / sizeof(T), d, ld, dout, sizeof(T), grad, sizeof(G))) {
    case 8:
      if constexpr (sizeof(T) == 2) e = launch_sum<T, G, 8>(ids, dout, ld, N, d, V, scale, accumulate, w, grad, st);
      else e = cudaErrorInvalidValue;
      break;
    case 4: e = launch_sum<T, G, 4>(ids, dout, ld, N, d, V, scale, accumulate, w, grad, st); break;
    case 2: e = launch_sum<T, G, 2>(ids, dout, ld, N, d, V, scale, accumulate, w, grad, st); break;
    default: e = launch_sum<T, G, 1>(ids, dout, ld, N, d, V, scale, accumulate, w, grad, st); break;
  }
  if (e != cudaSuccess || N <= kPiece) return e;
  LaunchScope scope_("embed_grad_join", st);
  return launch_k(join_kernel<G>, dim3((unsigned)owners, (unsigned)ceil_div(d, 32)), dim3(256), 0, st, d, per, scale,
                  accumulate, w, grad);
}

}  // namespace

size_t embed_grad_workspace_bytes(int64_t N, int d, int V) {
  GroupWs w;
  return carve(w, nullptr, N, d, V);
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
