// Distillation loss against a teacher's top logits, and its gradient, in one pass over the student's logits.
//
// With z = logits / T, q = softmax(z) and the teacher's p on its listed tokens (sum P), the soft loss of a row is
// T^2 sum p_i (log p_i - log q_i) and its gradient T (P q - p); with the teacher's remaining mass p_r as one more
// event, q_r = sum of q over the tokens that are not listed, the loss gains T^2 p_r (log p_r - log q_r) and a token
// that is not listed T p_r (q - q / q_r).  The hard loss's gradient is softmax(logits) - [target].
//
// A row (64 KB at 32,768 bfloat16 logits) is read from memory once, into the shared memory of a block, or of a
// cluster of blocks that exchange their maxima and sums; the gradient is formed from that copy.
#include <math_constants.h>
#include "vocab.cuh"

namespace sdm {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 512, kWarps = kThreads / 32;

struct DistillShared {
  float warp[3][kWarps];
  float part[4][kMaxCluster];  // max, soft sum, hard sum by block
  int id[kMaxTeacher];
  float logp[kMaxTeacher], val[kMaxTeacher];
  float target_val;
  float p_sum, lse;
};

__device__ __forceinline__ float block_max(float v, float* warp) {
  v = warp_max(v);
  if ((threadIdx.x & 31) == 0) warp[threadIdx.x >> 5] = v;
  __syncthreads();
  float r = warp[0];
#pragma unroll
  for (int w = 1; w < kWarps; ++w) r = fmaxf(r, warp[w]);
  return r;
}
__device__ __forceinline__ float block_sum(float v, float* warp) {
  v = warp_sum(v);
  if ((threadIdx.x & 31) == 0) warp[threadIdx.x >> 5] = v;
  __syncthreads();
  float r = 0.f;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) r += warp[w];
  return r;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) distill_kernel(DistillArgs a, int slice) {
  pdl_enter();
  constexpr int E = Chunk<T>::E;
  extern __shared__ uint4 buf4[];  // this block's slice of the row, by 16-byte chunk
  T* buf = reinterpret_cast<T*>(buf4);
  __shared__ DistillShared s;
  auto cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  if (C > 1) cluster.sync();
  const int64_t row = blockIdx.x / C;
  const int tid = threadIdx.x;
  const int V = a.V, k = a.k;
  const T* x = static_cast<const T*>(a.logits) + row * a.ld;
  T* g = a.dlogits ? static_cast<T*>(a.dlogits) + row * a.ld_grad : nullptr;
  const float w = a.row_weight ? a.row_weight[row] : 1.f;
  const int tgt = a.targets ? a.targets[row] : -1;
  const bool hard = tgt >= 0 && tgt < V;
  const int off = row_offset(x);
  const int p0 = rank * slice;
  const int v0 = p0 - off;  // the token of buf[0]
  const int lo = max(0, -v0), hi = max(lo, min(slice, V - v0));
  const bool vec_out = g && row_offset(g) == off;

  if (w == 0.f) {
    if (rank == 0 && tid == 0) a.loss[row] = 0.f;
    if (g) {
      const uint4 zero = make_uint4(0, 0, 0, 0);
      for (int i = tid * E; i < hi; i += kThreads * E) {
        if (vec_out && i >= lo && i + E <= hi) {
          *reinterpret_cast<uint4*>(g + v0 + i) = zero;
        } else {
          for (int e = max(i, lo); e < min(i + E, hi); ++e) g[v0 + e] = from_f32<T>(0.f);
        }
      }
    }
    return;
  }

  // the row into shared memory; the tail of the last chunk and the head of the first are filled with -infinity
  float mx = -CUDART_INF_F;
  for (int i = tid * E; i < hi; i += kThreads * E) {
    uint4 u;
    float f[E];
    if (i >= lo && i + E <= hi) {
      u = *reinterpret_cast<const uint4*>(x + v0 + i);
      Chunk<T>::unpack(u, f);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) f[e] = i + e >= lo && i + e < hi ? to_f32(x[v0 + i + e]) : -CUDART_INF_F;
      u = Chunk<T>::pack(f);
    }
    buf4[i / E] = u;
#pragma unroll
    for (int e = 0; e < E; ++e) mx = fmaxf(mx, f[e]);
  }

  // the teacher's distribution (every block of the cluster computes it)
  const float inv_t = 1.f / a.temperature;
  for (int j = tid; j < k; j += kThreads) {
    int id = a.t_ids[row * k + j];
    const float t = a.t_logits[row * k + j];
    if (id < 0 || id >= V || t == -CUDART_INF_F) id = -1;
    s.id[j] = id;
    s.logp[j] = id >= 0 ? __fdiv_rn(t, a.temperature) : -CUDART_INF_F;
    s.val[j] = id >= 0 ? to_f32(x[id]) : 0.f;
  }
  if (hard && tid == 0) s.target_val = to_f32(x[tgt]);
  mx = block_max(mx, s.warp[0]);
  if (tid < 32) {
    float tm = -CUDART_INF_F;
    for (int j = tid; j < k; j += 32) tm = fmaxf(tm, s.logp[j]);
    tm = warp_max(tm);
    const bool some = tm > -CUDART_INF_F || tm != tm;
    float lse = 0.f;
    if (a.t_lse) {
      lse = a.t_lse[row];
    } else if (some) {
      float sum = 0.f;
      for (int j = tid; j < k; j += 32) sum += s.id[j] >= 0 ? expf(s.logp[j] - tm) : 0.f;
      lse = tm + logf(warp_sum(sum));
    }
    float ps = 0.f;
    for (int j = tid; j < k; j += 32) {
      s.logp[j] -= lse;
      if (s.id[j] >= 0) ps += expf(s.logp[j]);
    }
    ps = warp_sum(ps);
    bool any = false;
    for (int j = tid; j < k; j += 32) any |= s.id[j] >= 0;
    any = __any_sync(0xffffffffu, any);
    if (tid == 0) {
      s.p_sum = any ? ps : -1.f;
    }
  }
  __syncthreads();
  if (C > 1) {
    if (tid < C) *cluster.map_shared_rank(&s.part[0][rank], tid) = mx;
    cluster.sync();
    for (int r = 0; r < C; ++r) mx = fmaxf(mx, s.part[0][r]);
  }
  const bool soft = s.p_sum >= 0.f || s.p_sum != s.p_sum;
  const float P = soft ? s.p_sum : 0.f;
  const bool tail = a.t_lse != nullptr && soft;
  // listed tokens leave the sums below; their terms are added once each, so that the mass of the others is a sum of
  // its own and no difference
  for (int j = tid; j < k; j += kThreads) {
    const int i = s.id[j] - v0;
    if (s.id[j] >= 0 && i >= lo && i < hi) buf[i] = from_f32<T>(-CUDART_INF_F);
  }
  __syncthreads();

  // sums of exp over the row, at T and (for the hard loss) at 1
  const float ct = inv_t * 1.4426950408889634f, c1 = 1.4426950408889634f;
  float st = 0.f, s1 = 0.f;
  for (int i = tid * E; i < hi; i += kThreads * E) {
    float f[E];
    Chunk<T>::unpack(buf4[i / E], f);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float d = f[e] - mx;
      if (soft) st += exp2f(d * ct);
      if (hard) s1 += exp2f(d * c1);
    }
  }
  st = block_sum(st, s.warp[1]);
  s1 = block_sum(s1, s.warp[2]);
  if (C > 1) {
    if (tid < C) {
      *cluster.map_shared_rank(&s.part[1][rank], tid) = st;
      *cluster.map_shared_rank(&s.part[2][rank], tid) = s1;
    }
    cluster.sync();
    st = s1 = 0.f;
    for (int r = 0; r < C; ++r) {
      st += s.part[1][r];
      s1 += s.part[2][r];
    }
  }
  // the listed tokens' terms, each distinct one once: warp 0 of every block
  __shared__ float listed[2];
  if (tid < 32) {
    float lt = 0.f, l1 = 0.f;
    for (int j = tid; j < k; j += 32) {
      const int id = s.id[j];
      bool first = id >= 0;
      for (int i = 0; i < j && first; ++i) first = s.id[i] != id;
      if (first) {
        const float d = s.val[j] - mx;
        lt += exp2f(d * ct);
        l1 += exp2f(d * c1);
      }
    }
    lt = warp_sum(lt);
    l1 = warp_sum(l1);
    if (tid == 0) {
      listed[0] = lt;
      listed[1] = l1;
    }
  }
  __syncthreads();
  const float rest = st;
  st += listed[0];
  s1 += listed[1];
  const float pr = tail ? fmaxf(0.f, 1.f - P) : 0.f;
  const float lst = logf(st);

  if (rank == 0 && tid < 32) {
    float sum = 0.f;
    if (soft) {
      for (int j = tid; j < k; j += 32) {
        if (s.id[j] < 0) continue;
        const float lp = s.logp[j], p = expf(lp);
        if (p > 0.f || p != p) sum += p * (lp - ((s.val[j] - mx) * inv_t - lst));
      }
      sum = warp_sum(sum);
      if (pr > 0.f) sum += pr * (logf(pr) - (logf(rest) - lst));
    }
    if (tid == 0) {
      float loss = a.alpha * sum * (a.temperature * a.temperature);
      if (hard) loss += (1.f - a.alpha) * (logf(s1) - (s.target_val - mx));
      a.loss[row] = w * loss;
    }
  }
  if (!g) return;

  // the gradient: a token that is not listed has ct_rest exp(z) + c1_all exp(logit), both over their sums
  const float scale = w * a.grad_scale;
  const float ks = soft ? scale * a.alpha * a.temperature : 0.f, kh = hard ? scale * (1.f - a.alpha) : 0.f;
  const float qt = ks * (P + pr) / st;                         // listed
  const float qr = pr > 0.f ? qt - ks * pr / rest : qt;        // not listed
  const float q1 = hard ? kh / s1 : 0.f;
  for (int i = tid * E; i < hi; i += kThreads * E) {
    float f[E];
    Chunk<T>::unpack(buf4[i / E], f);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float d = f[e] - mx;
      float r = 0.f;
      if (soft) r = qr * exp2f(d * ct);
      if (hard) r = fmaf(q1, exp2f(d * c1), r);
      f[e] = r;
    }
    if (vec_out && i >= lo && i + E <= hi) {
      *reinterpret_cast<uint4*>(g + v0 + i) = Chunk<T>::pack(f);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (i + e >= lo && i + e < hi) g[v0 + i + e] = from_f32<T>(f[e]);
    }
  }
  __syncthreads();  // the tokens with a term of their own are written over the pass above
  for (int j = tid; j < k; j += kThreads) {
    const int id = s.id[j];
    if (id < 0 || id - v0 < lo || id - v0 >= hi) continue;
    bool first = true;
    for (int i = 0; i < j && first; ++i) first = s.id[i] != id;
    if (!first) continue;
    float p = 0.f;
    for (int i = j; i < k; ++i)
      if (s.id[i] == id) p += expf(s.logp[i]);
    const float d = s.val[j] - mx;
    float r = qt * exp2f(d * ct) - ks * p;
    if (hard) {
      r += q1 * exp2f(d * c1);
      if (id == tgt) r -= kh;
    }
    g[id] = from_f32<T>(r);
  }
  if (hard && tid == 0 && tgt - v0 >= lo && tgt - v0 < hi) {
    bool own = true;
    for (int j = 0; j < k && own; ++j) own = s.id[j] != tgt;
    if (own) {
      const float d = s.target_val - mx;
      g[tgt] = from_f32<T>((soft ? qr * exp2f(d * ct) : 0.f) + q1 * exp2f(d * c1) - kh);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(256) scale_rows_kernel(T* __restrict__ x, int64_t ld, int V,
                                                         const float* __restrict__ g, int g_stride) {
  pdl_enter();
  constexpr int E = Chunk<T>::E;
  const int64_t row = blockIdx.x;
  const float f = g[row * g_stride];
  if (f == 1.f) return;
  T* r = x + row * ld;
  const int off = row_offset(r);
  for (int64_t p = threadIdx.x * E; p < (int64_t)V + off; p += 256 * E) {
    const int64_t v = p - off;
    if (v >= 0 && v + E <= V) {
      uint4* at = reinterpret_cast<uint4*>(r + v);
      float y[E];
      Chunk<T>::unpack(*at, y);
#pragma unroll
      for (int e = 0; e < E; ++e) y[e] *= f;
      *at = Chunk<T>::pack(y);
    } else {
      for (int e = 0; e < E; ++e)
        if (v + e >= 0 && v + e < V) r[v + e] = from_f32<T>(to_f32(r[v + e]) * f);
    }
  }
}

template <typename T>
cudaError_t distill_t(const DistillArgs& a, cudaStream_t st) {
  constexpr int E = Chunk<T>::E;
  auto slice_of = [&](int n) { return (int)(ceil_div(ceil_div((int64_t)a.V + E - 1, n), E) * E); };
  int C = 1;
  while (C < kMaxCluster && (a.N * C < kSMs || slice_of(C) * (int64_t)sizeof(T) > 104 * 1024)) C *= 2;
  if (a.N * C > 0x7fffffff) return cudaErrorInvalidValue;
  const int slice = slice_of(C);
  LaunchScope scope_("distill", st);
  return launch_clusters(distill_kernel<T>, (unsigned)(a.N * C), C, kThreads, (size_t)slice * sizeof(T), st, a, slice);
}

}  // namespace

cudaError_t launch_distill(const DistillArgs& a, int dtype, cudaStream_t st) {
  if (a.N == 0) return cudaSuccess;
  return dtype == SDM_BF16 ? distill_t<bf16_t>(a, st) : distill_t<float>(a, st);
}

cudaError_t launch_scale_rows(void* x, int64_t ld, int64_t N, int V, int dtype, const float* g, int g_stride,
                              cudaStream_t st) {
  if (N == 0) return cudaSuccess;
  if (N > 0x7fffffff) return cudaErrorInvalidValue;
  LaunchScope scope_("scale_rows", st);
  if (dtype == SDM_BF16)
    return launch_k(scale_rows_kernel<bf16_t>, dim3((unsigned)N), dim3(256), 0, st, static_cast<bf16_t*>(x), ld, V, g,
                    g_stride);
  return launch_k(scale_rows_kernel<float>, dim3((unsigned)N), dim3(256), 0, st, static_cast<float*>(x), ld, V, g,
                  g_stride);
}

}  // namespace sdm
