// Distillation loss against a teacher's top logits, and its gradient, in one pass over the student's logits.
//
// With z = logits / T, q = softmax(z) and the teacher's p on its listed tokens (sum P), the soft loss of a row is
// T^2 sum p_i (log p_i - log q_i) and its gradient T (P q - p); with the teacher's remaining mass p_r as one more
// event, q_r = sum of q over the tokens that are not listed, the loss gains T^2 p_r (log p_r - log q_r) and a token
// that is not listed T p_r (q - q / q_r).  The hard loss's gradient is softmax(logits) - [target].
//
// With the gradient, a row (64 KB at 32,768 bfloat16 logits) is read from memory once, into the shared memory of a
// block, or of a cluster of blocks that exchange their maxima and sums; the gradient is formed from that copy.
#include <float.h>
#include <math_constants.h>
#include <type_traits>
#include "tma.cuh"
#include "vocab.cuh"

namespace sdm {
namespace {

namespace cg = cooperative_groups;

constexpr int kMaxWarps = 8;  // a block has NT = 32, 64, 128 or 256 threads
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct DistillShared {
  float warp[4][kMaxWarps];
  float part[4][kMaxCluster];     // by block: max, sums
  int id[kMaxTeacher];            // the row's entries, -1 where unused
  float logp[kMaxTeacher], val[kMaxTeacher];
  float target_val, p_sum;
  int repeated;                   // some id of this block's slice is listed twice
};

// Exponentials are 2^(v c - B), c = log2(e) / T and B = c max rounded to float32: the one rounding of B cancels in
// every quotient and logarithm, which take the same B.  It has to be small beside float32's exponents, though: below
// |c max| = kFar it is at most 2^-5.
constexpr float kFar = 1048576.f;
__device__ __forceinline__ float ex2(float t) {
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
  return e;
}

// How many exponentials a logit takes.  kOne: the one at T serves, as T = 1 or no hard target is given.  kTwo: one at T and
// one at 1.  kSquare, kFourth: T = 2 or 4, so that the one at 1 is the other's square or fourth power (c and B are then
// exactly half or a quarter of those at 1, and it leaves float32's range at the same logit).  16,384 rows of 32,768
// bfloat16 logits with their gradient: 378 us, 532, 392, 429.
enum Exps { kOne, kTwo, kSquare, kFourth };
template <Exps X>
__device__ __forceinline__ float power(float e) {
  const float sq = e * e;
  return X == kFourth ? sq * sq : sq;
}

// Two floats in one 64-bit register, for the paired instructions.
typedef unsigned long long pair_t;
__device__ __forceinline__ pair_t pair(float a, float b) {
  pair_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 both(pair_t p) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(p));
  return r;
}
__device__ __forceinline__ pair_t fma_pair(pair_t a, pair_t b, pair_t c) {
  pair_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ pair_t add_pair(pair_t a, pair_t b) {
  pair_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// 2^t on the FMA pipe, for a kernel that would wait on the exponential unit (16 a clock and SM against 128 FMAs):
// t = n + f with n = rint(t) (Cody and Waite's reduction), a polynomial in f in [-1/2, 1/2] fitted by Remez's exchange
// to the least relative error (1.6e-7 with its coefficients in float32, 2.2e-7 evaluated there), and n added to the
// exponent.  Below -126 it stays at 2^-126.
__device__ __forceinline__ pair_t exp2_pair(pair_t t) {
  float2 v = both(t);
  t = pair(fmaxf(v.x, -126.f), fmaxf(v.y, -126.f));
  const pair_t z = add_pair(t, pair(12582912.f, 12582912.f));  // 2^23 + 2^22 + n
  const pair_t n = add_pair(z, pair(-12582912.f, -12582912.f));
  const pair_t f = fma_pair(n, pair(-1.f, -1.f), t);
  constexpr float kExp2[6] = {1.0000001192092896f, 0.6931469440460205f, 0.24022120237350464f,
                              0.05550713092088699f, 0.009675540961325169f, 0.0013276472454890609f};
  pair_t p = pair(kExp2[5], kExp2[5]);
#pragma unroll
  for (int i = 4; i >= 0; --i) p = fma_pair(p, f, pair(kExp2[i], kExp2[i]));
  const float2 pv = both(p), zv = both(z);
  return pair(__int_as_float(__float_as_int(pv.x) + (__float_as_int(zv.x) << 23)),
              __int_as_float(__float_as_int(pv.y) + (__float_as_int(zv.y) << 23)));
}

// Largest of a chunk's elements (NaN is passed over).
template <typename T>
__device__ __forceinline__ float chunk_max(uint4 u);
template <>
__device__ __forceinline__ float chunk_max<float>(uint4 u) {
  return fmaxf(fmaxf(__uint_as_float(u.x), __uint_as_float(u.y)), fmaxf(__uint_as_float(u.z), __uint_as_float(u.w)));
}
template <>
__device__ __forceinline__ float chunk_max<bf16_t>(uint4 u) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&u);
  const __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
  return fmaxf(__low2float(m), __high2float(m));
}

// Sum of up to three values over the block, each in the same order in every thread.
template <int NT>
__device__ __forceinline__ void block_sum3(DistillShared& s, float& a, float& b, float& c) {
  a = warp_sum(a);
  b = warp_sum(b);
  c = warp_sum(c);
  if ((threadIdx.x & 31) == 0) {
    s.warp[1][threadIdx.x >> 5] = a;
    s.warp[2][threadIdx.x >> 5] = b;
    s.warp[3][threadIdx.x >> 5] = c;
  }
  __syncthreads();
  a = b = c = 0.f;
#pragma unroll
  for (int w = 0; w < (NT / 32); ++w) {
    a += s.warp[1][w];
    b += s.warp[2][w];
    c += s.warp[3][w];
  }
}

// What a block needs to know of its row.
struct Row {
  int64_t row;
  int V, k, tgt;
  float w, inv_t;
  bool hard;
  int C, rank, v0, lo, hi;  // the block's tokens are v0 + [lo, hi), at positions [lo, hi) of its slice
};

template <typename T>
__device__ __forceinline__ Row row_of(const DistillArgs& a, int slice, int C, int rank, int64_t row, const T*& x) {
  Row q;
  q.C = C;
  q.rank = rank;
  q.row = row;
  x = static_cast<const T*>(a.logits) + q.row * a.ld;
  q.V = a.V;
  q.k = a.k;
  q.inv_t = 1.f / a.temperature;
  q.v0 = rank * slice - row_offset(x);
  q.lo = max(0, -q.v0);
  q.hi = max(q.lo, min(slice, q.V - q.v0));
  return q;
}
__device__ __forceinline__ void load_terms(const DistillArgs& a, Row& q) {
  q.w = a.row_weight ? a.row_weight[q.row] : 1.f;
  q.tgt = a.targets ? a.targets[q.row] : -1;
  q.hard = q.tgt >= 0 && q.tgt < q.V;
}

// The row's entries and the logits they point at (every block of a cluster takes all of them).
template <int NT, typename T>
__device__ __forceinline__ void load_teacher(const DistillArgs& a, const Row& q, const T* x, DistillShared& s) {
  for (int j = threadIdx.x; j < q.k; j += NT) {
    int id = a.t_ids[q.row * q.k + j];
    const float t = a.t_logits[q.row * q.k + j];
    if (id < 0 || id >= q.V || t == -CUDART_INF_F) id = -1;
    s.id[j] = id;
    s.logp[j] = id >= 0 ? __fdiv_rn(t, a.temperature) : -CUDART_INF_F;
    s.val[j] = id >= 0 ? to_f32(x[id]) : 0.f;
  }
  if (threadIdx.x == NT - 1) s.target_val = q.hard ? to_f32(x[q.tgt]) : 0.f;
}

// One warp: log p of each entry, and their sum (-1: the row has no entry).
template <typename S>
__device__ __forceinline__ void teacher_softmax(const DistillArgs& a, const Row& q, S& s) {
  const int lane = threadIdx.x & 31;
  float lse, tm = -CUDART_INF_F;
  bool any = false;
  for (int j = lane; j < q.k; j += 32) {
    tm = fmaxf(tm, s.logp[j]);
    any |= s.id[j] >= 0;
  }
  any = __any_sync(0xffffffffu, any);
  if (a.t_lse) {
    lse = a.t_lse[q.row];
  } else {
    tm = warp_max(tm);
    float sum = 0.f;
    for (int j = lane; j < q.k; j += 32) sum += s.id[j] >= 0 ? expf(s.logp[j] - tm) : 0.f;
    lse = tm + logf(warp_sum(sum));
  }
  float ps = 0.f;
  for (int j = lane; j < q.k; j += 32) {
    s.logp[j] -= lse;
    if (a.t_lse && s.id[j] >= 0) ps += expf(s.logp[j]);
  }
  if (a.t_lse) ps = warp_sum(ps);
  if (lane == 0) s.p_sum = !any ? -1.f : a.t_lse ? ps : lse != lse ? lse : 1.f;  // a softmax's sum is 1
}

// Whether entry j is the first with its id; ids are looked through only where one is repeated.
template <typename S>
__device__ __forceinline__ bool is_first(const S& s, int j) {
  if (s.repeated)
    for (int i = 0; i < j; ++i)
      if (s.id[i] == s.id[j]) return false;
  return true;
}

// The student's mass on the unlisted tokens is a sum of its own, relative to the row's largest logit like the others
// until it falls below kApart: terms under 2^-126 are 0, and 2^18 of those may have counted.  From there on (listed
// tokens that lead by 55 T and more) it is taken again, relative to the largest unlisted logit.
constexpr float kApart = 8.271806125530277e-25f;  // 2^-80

// The row's loss from its sums (one warp): st, s1 over all tokens at T and at 1, lrest the logarithm of the sum over the
// unlisted ones at T.
template <typename S>
__device__ __forceinline__ float row_loss(const DistillArgs& a, const Row& q, const S& s, float ct,
                                          float Bt, float B1, float st, float s1, float lrest) {
  const int lane = threadIdx.x & 31;
  float loss = 0.f;
  if (s.p_sum != -1.f) {
    const float lst = log2f(st);
    float sum = 0.f;
    for (int j = lane; j < q.k; j += 32) {
      if (s.id[j] < 0) continue;
      const float lp = s.logp[j], p = expf(lp);
      if (p > 0.f || p != p) sum += p * (lp - kLn2 * (fmaf(s.val[j], ct, -Bt) - lst));
    }
    sum = warp_sum(sum);
    const float pr = a.t_lse ? fmaxf(0.f, 1.f - s.p_sum) : 0.f;
    if (pr > 0.f) sum += pr * (logf(pr) - kLn2 * (lrest - lst));
    loss = a.alpha * sum * (a.temperature * a.temperature);
  }
  if (q.hard) loss += (1.f - a.alpha) * kLn2 * (log2f(s1) - fmaf(s.target_val, kLog2e, -B1));
  return q.w * loss;
}

// A block's slice in 16-byte chunks: whole ones [c0, c1), and up to 2 E tokens of its first and last chunk that other
// blocks or rows share (edge(t), t < 2 E; a position or -1).
struct Chunks {
  int c0, c1, lo, hi, E;
  __device__ Chunks(const Row& q, int e) {
    E = e;
    lo = q.lo;
    hi = q.hi;
    c0 = (lo + E - 1) / E;
    c1 = max(c0, hi / E);
  }
  __device__ int edge(int t) const {
    if (t < E) return lo + t < min(c0 * E, hi) ? lo + t : -1;
    const int i = c1 * E + t - E;
    return t < 2 * E && i >= lo && i < hi ? i : -1;
  }
};

// Whether a row's largest logit, times the larger c that is used, is at or beyond kFar (a row that is all at a mask's
// lowest value).  Its logits are then taken relative to the largest first: such differences are exact where a logit is
// within a factor of two of the largest, and any other is 2^19 / c or more below.  (At that c: the rounding of such a
// difference to bfloat16, 2^-9 of it, counts only where T is above 5,000 and a hard target asks for T = 1 besides.)
template <Exps X>
__device__ __forceinline__ bool is_far(float mx, float ct, float c1) {
  return fabsf(mx) < CUDART_INF_F && !(fabsf(mx) * (X == kOne ? ct : fmaxf(ct, c1)) < kFar);
}
template <typename T, int NT>
__device__ __forceinline__ void lower_row(T* buf, int c0, int c1, int edge, int tid, float mx) {
  constexpr int E = Chunk<T>::E;
#pragma unroll 1
  for (int c = c0 + tid; c < c1; c += NT) {
#pragma unroll 1
    for (int i = c * E; i < c * E + E; ++i) buf[i] = from_f32<T>(to_f32(buf[i]) - mx);
  }
  if (edge >= 0) buf[edge] = from_f32<T>(to_f32(buf[edge]) - mx);
}

// Largest value and sum over a row's threads: a block's, and its cluster's; or a team's of the kernel of persistent blocks.
template <int NT>
struct BlockReduce {
  DistillShared& s;
  int C, rank;
  __device__ float max(float m) const {
    m = warp_max(m);
    if ((threadIdx.x & 31) == 0) s.warp[0][threadIdx.x >> 5] = m;
    __syncthreads();
    for (int w = 0; w < (NT / 32); ++w) m = fmaxf(m, s.warp[0][w]);
    return across(0, m, true);
  }
  __device__ float sum(float v) const {
    float none = 0.f, none_ = 0.f;
    block_sum3<NT>(s, v, none, none_);
    return across(1, v, false);
  }
  __device__ float across(int part, float v, bool largest) const {
    if (C == 1) return v;
    auto cluster = cg::this_cluster();
    if ((int)threadIdx.x < C) *cluster.map_shared_rank(&s.part[part][rank], threadIdx.x) = v;
    cluster.sync();
    v = s.part[part][0];
    for (int r = 1; r < C; ++r) v = largest ? fmaxf(v, s.part[part][r]) : v + s.part[part][r];
    return v;
  }
};

// The gradient of a row's unlisted tokens where the listed ones lead by so much (kApart), from its copy in `buf`, where
// the listed ones are at -infinity: T (q - p_r q / q_r) without the first term, which is below 2^-56 of the second, and the hard
// target's.  nBt, nB1: the row's base; kr: the factor of q / q_r.  Returns the logarithm of their sum, for row_loss.
// Out of line, so that ordinary rows keep their registers (16,384 x 32,768: 391 us, 401 with this inlined).
template <typename T, int NT, typename Reduce>
__device__ __noinline__ float apart_gradient(DistillArgs a, int slice, int64_t row, int C, int rank, int tid, const T* buf,
                                             Reduce over, float nBt, float nB1, float kr, float q1, float kh) {
  constexpr int E = Chunk<T>::E;
  const T* x;
  Row q = row_of<T>(a, slice, C, rank, row, x);
  load_terms(a, q);
  T* g = static_cast<T*>(a.dlogits) + row * a.ld_grad;
  const Chunks ch(q, E);
  const int edge = ch.edge(tid);
  const float ct = q.inv_t * kLog2e, c1 = kLog2e;
  auto each = [&](auto f) {
#pragma unroll 1
    for (int i = ch.c0 * E + tid; i < ch.c1 * E; i += NT) f(i, to_f32(buf[i]));
    if (edge >= 0) f(edge, to_f32(buf[edge]));
  };
  float mr = -CUDART_INF_F, sum = 0.f;
  each([&](int, float v) { mr = fmaxf(mr, v); });
  mr = over.max(mr);
  const bool none = mr == -CUDART_INF_F;  // no unlisted token is possible, and none has a gradient
  if (none) mr = 0.f;
  each([&](int, float v) { sum += ex2((v - mr) * ct); });
  sum = over.sum(sum);
  kr = none ? 0.f : kr / sum;
  each([&](int i, float v) {
    const float y = q1 * ex2(fmaf(v, c1, nB1)) - kr * ex2((v - mr) * ct);
    g[q.v0 + i] = from_f32<T>(q.hard && q.v0 + i == q.tgt ? y - kh : y);
  });
  return log2f(sum) + fmaf(mr, ct, nBt);
}

// Threads of an SM, by the registers (64, 72 and 80) that the loops over an ordinary row take, where the call in the kernel
// would have them take more.
template <typename T, Exps X>
constexpr int kGradThreads = sizeof(T) == 4 ? 768 : X == kTwo ? 896 : 1024;

// Loss and gradient.  kTail: the teacher's remaining mass counts (teacher_lse is given).
template <typename T, Exps X, int NT, bool kTail>
__global__ void __launch_bounds__(NT, (kTail ? kGradThreads<T, X> : 768) / NT) distill_grad_kernel(DistillArgs a, int slice) {
  pdl_enter();
  constexpr int E = Chunk<T>::E;
  typedef typename std::conditional<sizeof(T) == 2, uint16_t, uint32_t>::type Tag;
  extern __shared__ uint4 buf4[];  // this block's slice of the row, by 16-byte chunk
  T* buf = reinterpret_cast<T*>(buf4);
  __shared__ DistillShared s;
  auto cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), tid = threadIdx.x;
  if (C > 1) cluster.sync();
  const T* x;
  Row q = row_of<T>(a, slice, C, (int)cluster.block_rank(), blockIdx.x / C, x);
  load_terms(a, q);
  T* g = static_cast<T*>(a.dlogits) + q.row * a.ld_grad;
  const int lo = q.lo, hi = q.hi, v0 = q.v0, k = q.k;
  const bool vec_out = row_offset(g) == row_offset(x);
  const Chunks ch(q, E);
  const int edge = ch.edge(tid);  // at most one token of the ragged chunks per thread

  if (q.w == 0.f) {
    if (q.rank == 0 && tid == 0) a.loss[q.row] = 0.f;
    const uint4 zero = make_uint4(0, 0, 0, 0);
    for (int c = ch.c0 + tid; c < ch.c1; c += NT) {
      if (vec_out) {
        *reinterpret_cast<uint4*>(g + v0 + c * E) = zero;
      } else {
        for (int e = 0; e < E; ++e) g[v0 + c * E + e] = from_f32<T>(0.f);
      }
    }
    if (edge >= 0) g[v0 + edge] = from_f32<T>(0.f);
    return;
  }

  // the row into shared memory, all of it on its way at once
  for (int c = ch.c0 + tid; c < ch.c1; c += NT)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(buf4 + c)),
                 "l"(x + v0 + c * E)
                 : "memory");
  load_teacher<NT>(a, q, x, s);
  float mx = -CUDART_INF_F;
  if (edge >= 0) {
    const T v = x[v0 + edge];
    buf[edge] = v;
    mx = to_f32(v);
    if (mx != mx) mx = -CUDART_INF_F;
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  for (int c = ch.c0 + tid; c < ch.c1; c += NT) mx = fmaxf(mx, chunk_max<T>(buf4[c]));  // its own copies
  mx = warp_max(mx);
  if ((tid & 31) == 0) s.warp[0][tid >> 5] = mx;
  if (tid == 0) s.repeated = 0;
  __syncthreads();
  // The listed tokens of this block leave the sums below; their terms are added once each, so that the mass of the
  // others is a sum of its own and no difference.  Each entry first writes its number in its token's place: one that
  // does not find it again is not alone.
  Tag* tag = reinterpret_cast<Tag*>(buf);
  for (int j = tid; j < k; j += NT) {
    const int i = s.id[j] - v0;
    if (s.id[j] >= 0 && i >= lo && i < hi) tag[i] = (Tag)j;
  }
#pragma unroll
  for (int w = 0; w < (NT / 32); ++w) mx = fmaxf(mx, s.warp[0][w]);
  if (tid >= NT - 32) teacher_softmax(a, q, s);
  __syncthreads();
  for (int j = tid; j < k; j += NT) {
    const int i = s.id[j] - v0;
    if (s.id[j] < 0 || i < lo || i >= hi) continue;
    if (tag[i] != (Tag)j) s.repeated = 1;
    buf[i] = from_f32<T>(-CUDART_INF_F);
  }
  if (C > 1) {
    if (tid < C) *cluster.map_shared_rank(&s.part[0][q.rank], tid) = mx;
    cluster.sync();
    for (int r = 0; r < C; ++r) mx = fmaxf(mx, s.part[0][r]);
  } else {
    __syncthreads();
  }

  // sums of exp over the row, at T and at 1
  const float ct = q.inv_t * kLog2e, c1 = kLog2e;
  if (is_far<X>(mx, ct, c1)) {
    lower_row<T, NT>(buf, ch.c0, ch.c1, edge, tid, mx);
    for (int j = tid; j < k; j += NT) s.val[j] -= mx;
    if (tid == 0) s.target_val -= mx;
    mx = 0.f;
  }
  const float nBt = -(mx * ct), nB1 = -(mx * c1);
  float st = 0.f, s1 = 0.f, listed = 0.f;
  // Four exponentials per bfloat16 logit would take the exponential unit longer than memory takes for the logit and
  // its gradient: half of those at T = 1 go to the FMA pipe here, and a quarter below (16,384 rows of 32,768: 558 us when this
  // was measured; all of these here and none below 590).
  constexpr bool kMix = X == kTwo && sizeof(T) == 2;
  pair_t s1p = pair(0.f, 0.f);
#pragma unroll 2
  for (int c = ch.c0 + tid; c < ch.c1; c += NT) {
    float f[E];
    Chunk<T>::unpack(buf4[c], f);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float t = ex2(fmaf(f[e], ct, nBt));
      st += t;
      if (X == kTwo && !kMix) s1 += ex2(fmaf(f[e], c1, nB1));
      if (X > kTwo) s1 += power<X>(t);
    }
    if (kMix) {
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        if (e % 4) {
          s1p = add_pair(s1p, exp2_pair(fma_pair(pair(f[e], f[e + 1]), pair(c1, c1), pair(nB1, nB1))));
        } else {
          s1 += ex2(fmaf(f[e], c1, nB1));
          s1 += ex2(fmaf(f[e + 1], c1, nB1));
        }
      }
    }
  }
  if (kMix) s1 += both(s1p).x + both(s1p).y;
  if (edge >= 0) {
    const float f = to_f32(buf[edge]);
    st += ex2(fmaf(f, ct, nBt));
    if (X != kOne) s1 += ex2(fmaf(f, c1, nB1));
  }
  for (int j = tid; j < k; j += NT) {
    const int i = s.id[j] - v0;
    if (s.id[j] < 0 || i < lo || i >= hi || !is_first(s, j)) continue;
    listed += ex2(fmaf(s.val[j], ct, nBt));
    if (X != kOne) s1 += ex2(fmaf(s.val[j], c1, nB1));
  }
  block_sum3<NT>(s, st, s1, listed);
  if (C > 1) {
    if (tid < C) {
      *cluster.map_shared_rank(&s.part[1][q.rank], tid) = st;
      *cluster.map_shared_rank(&s.part[2][q.rank], tid) = s1;
      *cluster.map_shared_rank(&s.part[3][q.rank], tid) = listed;
    }
    cluster.sync();
    st = s1 = listed = 0.f;
    for (int r = 0; r < C; ++r) {
      st += s.part[1][r];
      s1 += s.part[2][r];
      listed += s.part[3][r];
    }
  }
  const float rest = st;
  st += listed;
  if (X == kOne || st != st) s1 = st;  // a NaN or an infinity shows in st
  const float P = s.p_sum;
  const bool soft = P != -1.f;
  const float pr = kTail && soft ? fmaxf(0.f, 1.f - P) : 0.f;

  // the gradient: a token that is not listed has qr exp(logit / T) + q1 exp(logit), each over its sum
  const float scale = q.w * a.grad_scale;
  const float ks = soft ? scale * a.alpha * a.temperature : 0.f, kh = q.hard ? scale * (1.f - a.alpha) : 0.f;
  const float qt = soft ? ks * (P + pr) / st : 0.f;          // listed
  const float qr = pr > 0.f ? qt - ks * pr / rest : qt;      // not listed
  const float q1 = q.hard ? kh / s1 : 0.f;
  const float qm = X == kOne ? qr + q1 : qr;
  auto value = [&](float f) {
    const float t = ex2(fmaf(f, ct, nBt));
    if (X == kTwo) return fmaf(q1, ex2(fmaf(f, c1, nB1)), qm * t);
    if (X == kSquare) return t * fmaf(q1, t, qm);
    if (X == kFourth) return fmaf(q1, power<X>(t), qm * t);
    return qm * t;
  };
  const bool apart = kTail && pr > 0.f && rest < kApart;  // the same in all blocks of the row
  float lrest = 0.f;
  if (kTail && apart) {
    lrest = apart_gradient<T, NT>(a, slice, q.row, C, q.rank, tid, buf, BlockReduce<NT>{s, C, q.rank}, nBt, nB1, ks * pr,
                                  q1, kh);
  } else if (vec_out) {
#pragma unroll 2
    for (int c = ch.c0 + tid; c < ch.c1; c += NT) {
      float f[E];
      Chunk<T>::unpack(buf4[c], f);
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        if (kMix && e == 2) {
          const float2 t = both(fma_pair(pair(f[e], f[e + 1]), pair(c1, c1), pair(nB1, nB1)));
          float2 e1 = both(exp2_pair(pair(t.x, t.y)));
          if (t.x < -126.f) e1.x = 0.f;  // a logit of -infinity has no gradient
          if (t.y < -126.f) e1.y = 0.f;
          f[e] = fmaf(q1, e1.x, qm * ex2(fmaf(f[e], ct, nBt)));
          f[e + 1] = fmaf(q1, e1.y, qm * ex2(fmaf(f[e + 1], ct, nBt)));
        } else {
          f[e] = value(f[e]);
          f[e + 1] = value(f[e + 1]);
        }
      }
      *reinterpret_cast<uint4*>(g + v0 + c * E) = Chunk<T>::pack(f);
    }
  } else {
    for (int i = ch.c0 * E + tid; i < ch.c1 * E; i += NT) g[v0 + i] = from_f32<T>(value(to_f32(buf[i])));
  }
  if (edge >= 0 && !apart) g[v0 + edge] = from_f32<T>(value(to_f32(buf[edge])));
  if (q.rank == 0 && tid >= NT - 32) {
    const float loss = row_loss(a, q, s, ct, -nBt, -nB1, st, s1, apart ? lrest : log2f(rest));
    if (tid == NT - 1) a.loss[q.row] = loss;
  }
  __syncthreads();  // the tokens with a term of their own are written over the pass above
  for (int j = tid; j < k; j += NT) {
    const int id = s.id[j];
    if (id < 0 || id - v0 < lo || id - v0 >= hi || !is_first(s, j)) continue;
    float p = expf(s.logp[j]);
    if (s.repeated)
      for (int i = j + 1; i < k; ++i)
        if (s.id[i] == id) p += expf(s.logp[i]);
    float r = qt * ex2(fmaf(s.val[j], ct, nBt)) - ks * p;
    if (q.hard) {
      r += q1 * ex2(fmaf(s.val[j], c1, nB1));
      if (id == q.tgt) r -= kh;
    }
    g[id] = from_f32<T>(r);
  }
  if (q.hard && tid < 32 && q.tgt - v0 >= lo && q.tgt - v0 < hi) {
    bool listed_too = false;
    for (int j = tid; j < k; j += 32) listed_too |= s.id[j] == q.tgt;
    if (!__any_sync(0xffffffffu, listed_too) && tid == 0 && !apart)
      g[q.tgt] = from_f32<T>(qr * ex2(fmaf(s.target_val, ct, nBt)) + q1 * ex2(fmaf(s.target_val, c1, nB1)) - kh);
  }
}

// Loss and gradient of many rows that fit a block's shared memory three times: a persistent block per SM, so that a
// row's time is that of its arithmetic alone.  Two teams of eight warps take the rows in turn, so that one's reductions
// fall into the other's sums; a warp for each team runs ahead, copies rows into three buffers and prepares their teachers.

constexpr int kTeams = 2, kTeam = 256, kTeamWarps = kTeam / 32, kBuffers = 3, kTeamTeacher = 128;
constexpr int kRowsThreads = kTeams * (kTeam + 32);
// Barriers go by rows mod 6, the teams' and the buffers' common period: each has one team that waits on it and one that
// arrives, row by row, so that no wait can mistake a phase for the one two before it.
constexpr int kRing = kTeams * kBuffers;

struct TeamTeacher {
  int id[kTeamTeacher];
  float logp[kTeamTeacher], val[kTeamTeacher];
  float target_val, p_sum;
  int repeated, tgt;
};

struct TeamReduce {
  float (*red)[kTeamWarps];
  int barrier;
  __device__ void sync() const { asm volatile("bar.sync %0, %1;" ::"r"(barrier), "n"(kTeam) : "memory"); }
  __device__ float max(float m) const {
    m = warp_max(m);
    if ((threadIdx.x & 31) == 0) red[0][threadIdx.x % kTeam / 32] = m;
    sync();
    for (int w = 0; w < kTeamWarps; ++w) m = fmaxf(m, red[0][w]);
    return m;
  }
  __device__ float sum(float v) const {
    v = warp_sum(v);
    if ((threadIdx.x & 31) == 0) red[1][threadIdx.x % kTeam / 32] = v;
    sync();
    v = 0.f;
    for (int w = 0; w < kTeamWarps; ++w) v += red[1][w];
    return v;
  }
};

template <typename T, Exps X, bool kTail>
__global__ void __launch_bounds__(kRowsThreads, 1) distill_rows_kernel(DistillArgs a, int slice) {
  pdl_enter();
  constexpr int E = Chunk<T>::E;
  typedef typename std::conditional<sizeof(T) == 2, uint16_t, uint32_t>::type Tag;
  extern __shared__ __align__(128) uint4 buffers[];
  __shared__ TeamTeacher teachers[kBuffers];
  __shared__ float red[kTeams][4][kTeamWarps];
  __shared__ uint64_t full[kRing], empty[kRing];
  const int lane = threadIdx.x & 31, k = a.k;
  const int words = slice / E;
  if (threadIdx.x == 0) {
    for (int r = 0; r < kRing; ++r) {
      tma::mbar_init(&full[r], 2);  // the copy is under way (and its bytes), the teacher is there
      tma::mbar_init(&empty[r], kTeam);
    }
    tma::mbar_init_fence();
  }
  __syncthreads();
  // Row i of the block goes to team i mod 2 and buffer i mod 3.  Where a wait gives up, those who meet at a barrier leave
  // together: a team finds out at its first barrier of a row whether all of its threads saw the row arrive, and a warp that
  // runs ahead waits by one lane.  The block's shared memory is kept until the copies into it have landed, by the warps
  // that issued them.
  if (threadIdx.x >= kTeams * kTeam) {  // the warps that run ahead
    int i = ((int)threadIdx.x - kTeams * kTeam) / 32;
    for (int64_t row = blockIdx.x + (int64_t)i * gridDim.x; row < a.N; row += (int64_t)kTeams * gridDim.x, i += kTeams) {
      const int b = i % kBuffers;
      const T* x;
      Row q = row_of<T>(a, slice, 1, 0, row, x);
      load_terms(a, q);
      int id[kTeamTeacher / 32];
      float t[kTeamTeacher / 32], val[kTeamTeacher / 32];
#pragma unroll
      for (int u = 0; u < kTeamTeacher / 32; ++u) {
        const int j = lane + 32 * u;
        id[u] = j < k && q.w != 0.f ? a.t_ids[row * k + j] : -1;
        t[u] = j < k ? a.t_logits[row * k + j] : 0.f;
      }
#pragma unroll
      for (int u = 0; u < kTeamTeacher / 32; ++u) {
        if (id[u] < 0 || id[u] >= q.V || t[u] == -CUDART_INF_F) id[u] = -1;
        val[u] = id[u] >= 0 ? to_f32(x[id[u]]) : 0.f;
      }
      const float target_val = q.hard && q.w != 0.f ? to_f32(x[q.tgt]) : 0.f;
      const int last = i - kBuffers;  // the row that had the buffer
      if (last >= 0) {
        const int free_ = lane == 0 ? tma::mbar_wait(&empty[last % kRing], (last / kRing) & 1) : 0;
        __syncwarp();
        if (!__shfl_sync(0xffffffffu, free_, 0)) break;
      }
      const Chunks ch(q, E);
      TeamTeacher& s = teachers[b];
      if (lane == 0) {
        const uint32_t bytes = q.w != 0.f ? (uint32_t)(ch.c1 - ch.c0) * 16 : 0;
        tma::mbar_arrive_expect_tx(&full[i % kRing], bytes);
        if (bytes) tma::load_1d(buffers + b * words + ch.c0, x + q.v0 + ch.c0 * E, bytes, &full[i % kRing]);
        s.target_val = target_val;
        s.repeated = 0;
        s.tgt = q.tgt;
      }
#pragma unroll
      for (int u = 0; u < kTeamTeacher / 32; ++u) {
        const int j = lane + 32 * u;
        if (j < k) {
          s.id[j] = id[u];
          s.logp[j] = id[u] >= 0 ? __fdiv_rn(t[u], a.temperature) : -CUDART_INF_F;
          s.val[j] = val[u];
        }
      }
      __syncwarp();
      teacher_softmax(a, q, s);
      __syncwarp();
      if (lane == 0) tma::mbar_arrive(&full[i % kRing]);
    }
    if (lane == 0) {  // its last rows, one for each barrier it uses: no older copy can be in flight
      for (int u = 1; u <= kRing / kTeams; ++u)
        if (i - u * kTeams >= 0) tma::mbar_land(&full[(i - u * kTeams) % kRing], ((i - u * kTeams) / kRing) & 1);
    }
    return;
  }

  const int team = (int)threadIdx.x / kTeam;
  const int tid = (int)threadIdx.x % kTeam, warp = tid >> 5;
  auto team_sync = [&]() { asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "n"(kTeam) : "memory"); };
  // a barrier of the team: whether `ok` holds for all of it
  auto team_all = [&](bool ok) {
    uint32_t all;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 p, %1, 0;\n\t"
        "bar.red.and.pred q, %2, %3, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(all)
        : "r"((uint32_t)ok), "r"(team + 1), "n"(kTeam)
        : "memory");
    return all != 0;
  };
  // weights come from memory, a row ahead: whether a row counts is the same for all of the team, whatever its waits saw
  auto weight = [&](int64_t row) { return row < a.N && a.row_weight ? a.row_weight[row] : 1.f; };
  const float ct = (1.f / a.temperature) * kLog2e, c1 = kLog2e;
  bool here = true;  // no wait of this thread has given up
  int i = team;
  float w_next = weight(blockIdx.x + (int64_t)team * gridDim.x);
  for (int64_t row = blockIdx.x + (int64_t)team * gridDim.x; row < a.N; row += (int64_t)kTeams * gridDim.x, i += kTeams) {
    const int b = i % kBuffers;
    const T* x;
    Row q = row_of<T>(a, slice, 1, 0, row, x);
    T* g = static_cast<T*>(a.dlogits) + row * a.ld_grad;
    const bool vec_out = row_offset(g) == row_offset(x);
    const Chunks ch(q, E);
    const int edge = ch.edge(tid), lo = q.lo, hi = q.hi, v0 = q.v0;
    uint4* buf4 = buffers + b * words;
    T* buf = reinterpret_cast<T*>(buf4);
    TeamTeacher& s = teachers[b];
    float mx = -CUDART_INF_F, edge_val = 0.f;
    q.w = w_next;
    if (edge >= 0 && q.w != 0.f) {
      edge_val = to_f32(x[v0 + edge]);
      mx = edge_val == edge_val ? edge_val : -CUDART_INF_F;
    }
    w_next = weight(row + (int64_t)kTeams * gridDim.x);
    here = here && tma::mbar_wait(&full[i % kRing], (i / kRing) & 1);
    if (q.w == 0.f) {
      if (tid == 0) a.loss[row] = 0.f;
      for (int c = ch.c0 + tid; c < ch.c1; c += kTeam) {
        if (vec_out) {
          *reinterpret_cast<uint4*>(g + v0 + c * E) = make_uint4(0, 0, 0, 0);
        } else {
          for (int e = 0; e < E; ++e) g[v0 + c * E + e] = from_f32<T>(0.f);
        }
      }
      if (edge >= 0) g[v0 + edge] = from_f32<T>(0.f);
      if (here) {
        tma::fence_proxy_async();
        tma::mbar_arrive(&empty[i % kRing]);
      }
      continue;
    }
    if (here && edge >= 0) buf[edge] = from_f32<T>(edge_val);
    for (int c = ch.c0 + tid; c < ch.c1; c += kTeam) mx = fmaxf(mx, chunk_max<T>(buf4[c]));
    mx = warp_max(mx);
    if (lane == 0) red[team][0][warp] = mx;
    if (!team_all(here)) {  // the rows that are left: no loss that could be taken for one
      for (; tid == 0 && row < a.N; row += (int64_t)kTeams * gridDim.x) a.loss[row] = CUDART_NAN_F;
      return;
    }
    q.tgt = s.tgt;
    q.hard = q.tgt >= 0 && q.tgt < q.V;
    // the listed tokens leave the sums, as in the kernel of a block per row
    Tag* tag = reinterpret_cast<Tag*>(buf);
    const int mine = tid < k && s.id[tid] >= 0 ? s.id[tid] - v0 : -1;  // k <= kTeamTeacher < kTeam
    if (mine >= 0) tag[mine] = (Tag)tid;
#pragma unroll
    for (int w = 0; w < kTeamWarps; ++w) mx = fmaxf(mx, red[team][0][w]);
    team_sync();
    if (mine >= 0) {
      if (tag[mine] != (Tag)tid) s.repeated = 1;
      buf[mine] = from_f32<T>(-CUDART_INF_F);
    }
    team_sync();
    if (is_far<X>(mx, ct, c1)) {
      lower_row<T, kTeam>(buf, ch.c0, ch.c1, edge, tid, mx);
      if (tid < k) s.val[tid] -= mx;
      if (tid == 0) s.target_val -= mx;
      mx = 0.f;
    }
    const float nBt = -(mx * ct), nB1 = -(mx * c1);
    float st = 0.f, s1 = 0.f, listed = 0.f;
#pragma unroll 4
    for (int c = ch.c0 + tid; c < ch.c1; c += kTeam) {
      float f[E];
      Chunk<T>::unpack(buf4[c], f);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float t = ex2(fmaf(f[e], ct, nBt));
        st += t;
        if (X != kOne) s1 += power<X>(t);
      }
    }
    if (edge >= 0) {
      const float f = to_f32(buf[edge]);
      st += ex2(fmaf(f, ct, nBt));
      if (X != kOne) s1 += ex2(fmaf(f, c1, nB1));
    }
    const bool own = mine >= 0 && is_first(s, tid);
    if (own) {
      listed = ex2(fmaf(s.val[tid], ct, nBt));
      if (X != kOne) s1 += ex2(fmaf(s.val[tid], c1, nB1));
    }
    st = warp_sum(st);
    s1 = warp_sum(s1);
    listed = warp_sum(listed);
    if (lane == 0) {
      red[team][1][warp] = st;
      red[team][2][warp] = s1;
      red[team][3][warp] = listed;
    }
    team_sync();
    st = s1 = listed = 0.f;
#pragma unroll
    for (int w = 0; w < kTeamWarps; ++w) {
      st += red[team][1][w];
      s1 += red[team][2][w];
      listed += red[team][3][w];
    }
    const float rest = st;
    st += listed;
    if (X == kOne || st != st) s1 = st;
    const float P = s.p_sum;
    const bool soft = P != -1.f;
    const float pr = kTail && soft ? fmaxf(0.f, 1.f - P) : 0.f;
    const float scale = q.w * a.grad_scale;
    const float ks = soft ? scale * a.alpha * a.temperature : 0.f, kh = q.hard ? scale * (1.f - a.alpha) : 0.f;
    const float qt = soft ? ks * (P + pr) / st : 0.f;
    const float qr = pr > 0.f ? qt - ks * pr / rest : qt;
    const float q1 = q.hard ? kh / s1 : 0.f;
    const float qm = X == kOne ? qr + q1 : qr;
    auto value = [&](float f) {
      const float t = ex2(fmaf(f, ct, nBt));
      if (X == kSquare) return t * fmaf(q1, t, qm);
      if (X == kFourth) return fmaf(q1, power<X>(t), qm * t);
      return qm * t;
    };
    const bool apart = kTail && pr > 0.f && rest < kApart;
    float lrest = 0.f;
    if (kTail && apart) {
      lrest = apart_gradient<T, kTeam>(a, slice, row, 1, 0, tid, buf, TeamReduce{red[team], team + 1}, nBt, nB1, ks * pr,
                                       q1, kh);
    } else if (vec_out) {
#pragma unroll 4
      for (int c = ch.c0 + tid; c < ch.c1; c += kTeam) {
        float f[E];
        Chunk<T>::unpack(buf4[c], f);
#pragma unroll
        for (int e = 0; e < E; ++e) f[e] = value(f[e]);
        *reinterpret_cast<uint4*>(g + v0 + c * E) = Chunk<T>::pack(f);
      }
    } else {
      for (int p = ch.c0 * E + tid; p < ch.c1 * E; p += kTeam) g[v0 + p] = from_f32<T>(value(to_f32(buf[p])));
    }
    if (edge >= 0 && !apart) g[v0 + edge] = from_f32<T>(value(to_f32(buf[edge])));
    team_sync();
    if (own) {
      const int id = s.id[tid];
      float p = expf(s.logp[tid]);
      if (s.repeated)
        for (int j = tid + 1; j < k; ++j)
          if (s.id[j] == id) p += expf(s.logp[j]);
      float r = qt * ex2(fmaf(s.val[tid], ct, nBt)) - ks * p;
      if (q.hard) {
        r += q1 * ex2(fmaf(s.val[tid], c1, nB1));
        if (id == q.tgt) r -= kh;
      }
      g[id] = from_f32<T>(r);
    }
    if (warp == kTeamWarps - 1) {
      const float loss = row_loss(a, q, s, ct, -nBt, -nB1, st, s1, apart ? lrest : log2f(rest));
      if (lane == 0) a.loss[row] = loss;
      if (q.hard) {
        bool listed_too = false;
        for (int j = lane; j < k; j += 32) listed_too |= s.id[j] == q.tgt;
        if (!__any_sync(0xffffffffu, listed_too) && lane == 0 && !apart)
          g[q.tgt] = from_f32<T>(qr * ex2(fmaf(s.target_val, ct, nBt)) + q1 * ex2(fmaf(s.target_val, c1, nB1)) - kh);
      }
    }
    tma::fence_proxy_async();  // this row's marks before the next row's copy
    tma::mbar_arrive(&empty[i % kRing]);
  }
}

// The largest value of a row, and the sums of three, over its blocks.
template <int NT, typename Cluster>
__device__ __forceinline__ float row_max(Cluster& cluster, DistillShared& s, const Row& q, float m) {
  const int tid = threadIdx.x;
  m = warp_max(m);
  if ((tid & 31) == 0) s.warp[0][tid >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < (NT / 32); ++w) m = fmaxf(m, s.warp[0][w]);
  if (q.C > 1) {
    if (tid < q.C) *cluster.map_shared_rank(&s.part[0][q.rank], tid) = m;
    cluster.sync();
    for (int r = 0; r < q.C; ++r) m = fmaxf(m, s.part[0][r]);
  }
  return m;
}
template <int NT, typename Cluster>
__device__ __forceinline__ void row_sum3(Cluster& cluster, DistillShared& s, const Row& q, float& a, float& b, float& c) {
  const int tid = threadIdx.x;
  block_sum3<NT>(s, a, b, c);
  if (q.C > 1) {
    if (tid < q.C) {
      *cluster.map_shared_rank(&s.part[1][q.rank], tid) = a;
      *cluster.map_shared_rank(&s.part[2][q.rank], tid) = b;
      *cluster.map_shared_rank(&s.part[3][q.rank], tid) = c;
    }
    cluster.sync();
    a = b = c = 0.f;
    for (int r = 0; r < q.C; ++r) {
      a += s.part[1][r];
      b += s.part[2][r];
      c += s.part[3][r];
    }
  }
}

// The loss alone of a far row, or of one whose listed tokens lead by so much (kApart), from the row once more: its largest
// logit (all of them may lie below where the threads began), the sums over differences to it, and the unlisted
// tokens' over differences to the largest of those.  Out of line: inlined, it took registers from the loop over
// ordinary rows.
template <typename T, int NT, bool kTail>
__device__ __noinline__ void careful_loss(const DistillArgs& a, int slice, DistillShared& s, const uint32_t* is_listed,
                                          bool two) {
  auto cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks();
  const T* x;
  Row q = row_of<T>(a, slice, C, (int)cluster.block_rank(), blockIdx.x / C, x);
  load_terms(a, q);
  const int tid = threadIdx.x;
  const float ct = q.inv_t * kLog2e, c1 = kLog2e;
  constexpr bool tail = kTail;
  auto apart = [&](int i) { return tail && ((is_listed[i >> 5] >> (i & 31)) & 1); };
  float mx = -CUDART_INF_F;
#pragma unroll 1
  for (int i = q.lo + tid; i < q.hi; i += NT) mx = fmaxf(mx, to_f32(x[q.v0 + i]));
  mx = row_max<NT>(cluster, s, q, mx);
  float st = 0.f, s1 = 0.f, listed = 0.f;
#pragma unroll 1
  for (int i = q.lo + tid; i < q.hi; i += NT) {
    const float f = to_f32(x[q.v0 + i]) - mx;
    if (apart(i)) continue;
    st += ex2(f * ct);
    if (two) s1 += ex2(f * c1);
  }
  for (int j = tid; j < q.k; j += NT) {
    const int i = s.id[j] - q.v0;
    s.val[j] -= mx;
    if (!tail || s.id[j] < 0 || i < q.lo || i >= q.hi || !is_first(s, j)) continue;
    listed += ex2(s.val[j] * ct);
    if (two) s1 += ex2(s.val[j] * c1);
  }
  if (tid == 0) s.target_val -= mx;
  row_sum3<NT>(cluster, s, q, st, s1, listed);
  float lrest = log2f(st);
  st += listed;
  if (!two) s1 = st;
  if (tail) {
    float mr = -CUDART_INF_F, sum = 0.f, none = 0.f, none_ = 0.f;
#pragma unroll 1
    for (int i = q.lo + tid; i < q.hi; i += NT)
      if (!apart(i)) mr = fmaxf(mr, to_f32(x[q.v0 + i]));
    mr = row_max<NT>(cluster, s, q, mr);
    if (mr == -CUDART_INF_F) {
      lrest = mr;
    } else {
#pragma unroll 1
      for (int i = q.lo + tid; i < q.hi; i += NT)
        if (!apart(i)) sum += ex2((to_f32(x[q.v0 + i]) - mr) * ct);
      row_sum3<NT>(cluster, s, q, sum, none, none_);
      lrest = log2f(sum) + (mr - mx) * ct;
    }
  }
  if (q.rank == 0 && tid < 32) {
    const float loss = row_loss(a, q, s, ct, 0.f, 0.f, st, s1, lrest);
    if (tid == 0) a.loss[q.row] = loss;
  }
}

// The loss alone: the row streams through registers, each thread keeping the largest logit it has seen and its sums
// relative to that, or to a value below all rows that are not far (kFar) while it has seen none above: tokens at a mask's
// lowest value count for nothing beside a row's others, and their product with c may be beyond float32.  Where the
// teacher's remaining mass counts, a bit per token tells which are listed.
template <typename T, Exps X, int NT, bool kTail>
__global__ void __launch_bounds__(NT, 1536 / NT) distill_loss_kernel(const __grid_constant__ DistillArgs a, int slice) {
  pdl_enter();
  constexpr int E = Chunk<T>::E, U = 4;
  extern __shared__ uint32_t is_listed[];
  __shared__ DistillShared s;
  auto cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), tid = threadIdx.x;
  if (C > 1) cluster.sync();
  const T* x;
  Row q = row_of<T>(a, slice, C, (int)cluster.block_rank(), blockIdx.x / C, x);
  load_terms(a, q);
  const int lo = q.lo, hi = q.hi, v0 = q.v0, k = q.k;
  if (q.w == 0.f) {
    if (q.rank == 0 && tid == 0) a.loss[q.row] = 0.f;
    return;
  }
  constexpr bool tail = kTail;
  const Chunks ch(q, E);
  // the row is on its way to L2 while its teacher is fetched (8,192 rows of 50,021: 150 us without,
  // 148 with; 65,536 of 8,192: 204 and 192)
  if (tid == 0 && ch.c1 > ch.c0)
    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(x + v0 + ch.c0 * E), "r"((ch.c1 - ch.c0) * 16)
                 : "memory");
  if (tail) {
    for (int i = tid; i < (slice + 31) / 32; i += NT) is_listed[i] = 0;
    if (tid == 0) s.repeated = 0;
  }
  load_teacher<NT>(a, q, x, s);
  if (tail) {
    __syncthreads();
    for (int j = tid; j < k; j += NT) {
      const int i = s.id[j] - v0;
      if (s.id[j] < 0 || i < lo || i >= hi) continue;
      const uint32_t bit = 1u << (i & 31);
      if (atomicOr(&is_listed[i >> 5], bit) & bit) s.repeated = 1;
    }
    __syncthreads();
  }
  const float ct = q.inv_t * kLog2e, c1 = kLog2e;
  float mt = fmaxf(-2.f * kFar * kLn2 * (X == kOne ? a.temperature : fminf(a.temperature, 1.f)), -FLT_MAX);
  float nBt = -__fmul_rn(mt, ct), nB1 = -__fmul_rn(mt, c1), st = 0.f, s1 = 0.f;
  auto raise = [&](float cm) {  // the largest logit so far
    if (cm > mt) {
      const float nt = -__fmul_rn(cm, ct), n1 = -__fmul_rn(cm, c1);
      if ((X == kOne ? st : st + s1) != 0.f) {
        st *= ex2(nt - nBt);
        if (X != kOne) s1 *= ex2(n1 - nB1);
      }
      mt = cm;
      nBt = nt;
      nB1 = n1;
    }
  };
  auto add = [&](uint4 u, int c) {
    float f[E];
    Chunk<T>::unpack(u, f);
    if (tail) {  // a listed token's term is added once, below
      const uint32_t bits = (is_listed[c * E >> 5] >> (c * E & 31)) & ((1u << E) - 1);
      if (bits) {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if ((bits >> e) & 1) f[e] = -CUDART_INF_F;
      }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float t = ex2(fmaf(f[e], ct, nBt));
      st += t;
      if (X == kTwo) s1 += ex2(fmaf(f[e], c1, nB1));
      if (X > kTwo) s1 += power<X>(t);
    }
  };
  const uint4* x4 = reinterpret_cast<const uint4*>(x + v0);  // chunk c, for c in [c0, c1)
  int c = ch.c0 + tid;
  for (; c + (U - 1) * NT < ch.c1; c += U * NT) {
    uint4 u[U];
#pragma unroll
    for (int j = 0; j < U; ++j) u[j] = __ldg(x4 + c + j * NT);
    float cm = chunk_max<T>(u[0]);
#pragma unroll
    for (int j = 1; j < U; ++j) cm = fmaxf(cm, chunk_max<T>(u[j]));
    raise(cm);
#pragma unroll
    for (int j = 0; j < U; ++j) add(u[j], c + j * NT);
  }
  for (; c < ch.c1; c += NT) {
    const uint4 u = __ldg(x4 + c);
    raise(chunk_max<T>(u));
    add(u, c);
  }
  const int edge = ch.edge(tid);
  if (edge >= 0) {
    const float f = to_f32(x[v0 + edge]);
    raise(f);
    if (!(tail && ((is_listed[edge >> 5] >> (edge & 31)) & 1))) {
      st += ex2(fmaf(f, ct, nBt));
      if (X != kOne) s1 += ex2(fmaf(f, c1, nB1));
    }
  }
  const float mx = row_max<NT>(cluster, s, q, mt);
  if (tid >= NT - 32) teacher_softmax(a, q, s);
  // all sums relative to the row's largest logit
  const float Mt = __fmul_rn(mx, ct), M1 = __fmul_rn(mx, c1);
  float listed = 0.f;
  st *= ex2(-nBt - Mt);
  s1 *= ex2(-nB1 - M1);
  if (tail)
    for (int j = tid; j < k; j += NT) {
      const int i = s.id[j] - v0;
      if (s.id[j] < 0 || i < lo || i >= hi || !is_first(s, j)) continue;
      listed += ex2(fmaf(s.val[j], ct, -Mt));
      if (X != kOne) s1 += ex2(fmaf(s.val[j], c1, -M1));
    }
  row_sum3<NT>(cluster, s, q, st, s1, listed);
  const float rest = st;
  st += listed;
  if (X == kOne) s1 = st;
  if (q.rank == 0 && tid < 32) {
    const float loss = row_loss(a, q, s, ct, Mt, M1, st, s1, log2f(rest));
    if (tid == 0) a.loss[q.row] = loss;
  }
  if (is_far<X>(mx, ct, c1) || (tail && rest < kApart)) {  // the same in all blocks of the row
    __syncthreads();
    careful_loss<T, NT, kTail>(a, slice, s, is_listed, X != kOne);
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

template <typename T, Exps X, int NT>
cudaError_t distill_n(const DistillArgs& a, int C, int slice, cudaStream_t st) {
  const unsigned grid = (unsigned)(a.N * C);
  LaunchScope scope_(a.dlogits ? "distill_grad" : "distill_loss", st);
  if (a.dlogits)
    return launch_clusters(a.t_lse ? distill_grad_kernel<T, X, NT, true> : distill_grad_kernel<T, X, NT, false>, grid, C, NT,
                           (size_t)slice * sizeof(T), st, a, slice);
  const size_t smem = a.t_lse ? (size_t)(slice / 32) * 4 : 0;
  return launch_clusters(a.t_lse ? distill_loss_kernel<T, X, NT, true> : distill_loss_kernel<T, X, NT, false>, grid, C, NT,
                         smem, st, a, slice);
}

template <typename T, Exps X>
cudaError_t distill_x(const DistillArgs& a, cudaStream_t st) {
  constexpr int E = Chunk<T>::E;
  auto slice_of = [&](int n) { return (int)(ceil_div(ceil_div((int64_t)a.V + E - 1, n), 32) * 32); };
  // one block per row, more where rows are too few to fill the SMs, or a block's copy of the row is too large for two
  // blocks to share an SM
  const int64_t most = a.dlogits ? 104 * 1024 : (int64_t)1 << 40;
  int C = 1;
  while (C < kMaxCluster && (a.N * C < kSMs || slice_of(C) * (int64_t)sizeof(T) > most)) C *= 2;
  if (a.N * C > 0x7fffffff) return cudaErrorInvalidValue;
  const int slice = slice_of(C);
  // Rows of which three fit a block's shared memory, but of which the SM does not hold four for the other kernel, enough
  // of them that every SM gets several.  16,384 rows of 32,768 bfloat16 take 392 us on persistent blocks and 417 on a block
  // per row, of 26,000 347 and 376, but of 24,000 363 and 309.  (With two exponentials a logit persistent blocks took 552 us
  // at 32,768 when a block per row took 529.)
  const size_t row_bytes = (size_t)slice * sizeof(T);
  if constexpr (X != kTwo) {
    constexpr int kMost = 200 * 1024;
    if (a.dlogits && C == 1 && a.k <= kTeamTeacher && a.N >= 4 * kSMs && row_bytes > 50 * 1024 &&
        kBuffers * row_bytes <= kMost) {
      auto kern = a.t_lse ? distill_rows_kernel<T, X, true> : distill_rows_kernel<T, X, false>;
      cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost);
      if (e != cudaSuccess) return e;
      LaunchScope scope_("distill_rows", st);
      return launch_k(kern, dim3(kSMs), dim3(kRowsThreads), kBuffers * row_bytes, st, a, slice);
    }
  }
  // few threads where rows are short, so that many blocks hide one another's reductions.  131,072 rows of 2,048 bfloat16
  // logits with their gradient take 423 us with 32 threads and 449 with 64 (of 1,000 325 and 413), 65,536 of 4,096 337 and
  // 309; the loss alone (T = 2, hard targets) of 65,536 rows of 8,192 193 with 64 and 240 with 128, of 32,768 rows of
  // 16,384 218 and 178, of 16,384 rows of 32,768 199 with 128 and 177 with 256.  A cluster's blocks keep 64: 48 rows of
  // 1,000 float32 logits take 6.8 us, and 7.7 with 32.
  if (C == 1 && row_bytes <= 6 * 1024) return distill_n<T, X, 32>(a, C, slice, st);
  if (row_bytes <= 16896) return distill_n<T, X, 64>(a, C, slice, st);
  if (row_bytes <= 33024) return distill_n<T, X, 128>(a, C, slice, st);
  return distill_n<T, X, 256>(a, C, slice, st);
}

template <typename T>
cudaError_t distill_t(const DistillArgs& a, cudaStream_t st) {
  if (!a.targets || a.temperature == 1.f) return distill_x<T, kOne>(a, st);
  if (a.temperature == 2.f) return distill_x<T, kSquare>(a, st);
  if (a.temperature == 4.f) return distill_x<T, kFourth>(a, st);
  return distill_x<T, kTwo>(a, st);
}

}  // namespace

cudaError_t read_and_clear_distill_timeout(int* flag, cudaStream_t st) { return tma::read_and_clear_wait_timeout(flag, st); }
cudaError_t set_distill_wait_limit(unsigned long long ns) { return tma::set_wait_limit(ns); }

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
