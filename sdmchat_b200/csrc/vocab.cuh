// The vocabulary-end operators (rules on logits, token choice, distillation, scaled lookup and its gradient): launch
// functions behind the C ABI, and the helpers their kernels share.
#pragma once
#include <cooperative_groups.h>
#include "common.cuh"

namespace sdm {

constexpr int kSMs = 148;
constexpr int kMaxCluster = 8;          // portable cluster size
constexpr int kMaxChoiceV = 1 << 18;    // a row's float32 logits fit a cluster's shared memory: 8 x 128 KB
constexpr int kMaxBias = 1024;
constexpr int kMaxHistory = (1 << 20) - 1;
constexpr int kMaxTeacher = 512;

cudaError_t launch_logits_process(const sdm_logit_rules& r, const void* logits, int64_t ld, int64_t S, int V,
                                  int dtype, void* out, int64_t ld_out, cudaStream_t st);
cudaError_t launch_logits_choose(const sdm_logit_rules& r, const sdm_choice_params& c, const void* logits, int64_t ld,
                                 int64_t S, int V, int dtype, int32_t* ids, float* logprob, cudaStream_t st);

struct DistillArgs {
  const void* logits;
  int64_t ld, N;
  int V, k;
  const int32_t* t_ids;
  const float* t_logits;
  const float* t_lse;
  const int32_t* targets;
  const float* row_weight;
  float temperature, alpha, grad_scale;
  float* loss;
  void* dlogits;
  int64_t ld_grad;
};
cudaError_t launch_distill(const DistillArgs& a, int dtype, cudaStream_t st);
cudaError_t launch_scale_rows(void* x, int64_t ld, int64_t N, int V, int dtype, const float* g, int g_stride,
                              cudaStream_t st);

cudaError_t launch_embed_scaled(const int32_t* ids, const void* emb, int64_t N, int d, int V, float scale, int dtype,
                                void* out, int* bad, cudaStream_t st);
size_t embed_grad_workspace_bytes(int64_t N, int d, int V);
cudaError_t launch_embed_grad(const int32_t* ids, const void* dout, int64_t ld, int64_t N, int d, int V, float scale,
                              int padding_id, int dtype, int grad_dtype, int accumulate, void* grad, void* ws,
                              cudaStream_t st);

// A launch that may start while its predecessor in the stream ends, whatever its size (launch_k allows that to small
// ones only): for kernels that always follow one of their own operator's and whose blocks wait in pdl_enter.
template <typename... KArgs, typename... Args>
inline cudaError_t launch_next(void (*kern)(KArgs...), unsigned grid, int block, cudaStream_t st, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3((unsigned)block);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, static_cast<Args&&>(args)...);
}

// A kernel's limit of dynamic shared memory belongs to the function, not to a launch: it is set to the same number by every
// call, so that host threads which launch one kernel at several sizes do not lower it under one another.
constexpr size_t kMaxDynamicSmem = 160 * 1024;

// A cluster launch of kern (blocks of one row share a cluster).  Programmatic dependent launch as in launch_k.  A cluster
// of one block is launched as a plain block: with the attribute, blocks start late (distillation of 131,072 rows
// of 2,048: 826 us with it, 423 without).
template <typename... KArgs, typename... Args>
inline cudaError_t launch_clusters(void (*kern)(KArgs...), unsigned grid, int cluster, int block, size_t smem,
                                   cudaStream_t st, Args&&... args) {
  if (smem > kMaxDynamicSmem) return cudaErrorInvalidValue;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMaxDynamicSmem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3((unsigned)block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  cfg.attrs = attr;
  if (cluster > 1) {
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)cluster;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.numAttrs = 1;
  }
  if ((int64_t)grid * block <= PDL_MAX_THREADS && smem <= PDL_MAX_SMEM) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  return cudaLaunchKernelEx(&cfg, kern, static_cast<Args&&>(args)...);
}

// A row of T seen from the 16-byte boundary at or below its first element: position p of the row's 16-byte chunks is
// element p - off, so chunks are aligned whatever the row's own alignment (an odd vocabulary in bfloat16).
template <typename T>
__device__ __forceinline__ int row_offset(const T* row) {
  return (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
}

// The E = 16 / sizeof(T) elements of a 16-byte chunk as float32.
template <typename T>
struct Chunk;
template <>
struct Chunk<float> {
  static constexpr int E = 4;
  __device__ static void unpack(uint4 u, float* x) {
    x[0] = __uint_as_float(u.x);
    x[1] = __uint_as_float(u.y);
    x[2] = __uint_as_float(u.z);
    x[3] = __uint_as_float(u.w);
  }
  __device__ static uint4 pack(const float* x) {
    return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
  }
};
template <>
struct Chunk<bf16_t> {
  static constexpr int E = 8;
  __device__ static void two(uint32_t u, float* x) {
    x[0] = __uint_as_float(u << 16);
    x[1] = __uint_as_float(u & 0xffff0000u);
  }
  __device__ static void unpack(uint4 u, float* x) {
    two(u.x, x);
    two(u.y, x + 2);
    two(u.z, x + 4);
    two(u.w, x + 6);
  }
  __device__ static uint32_t both(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  __device__ static uint4 pack(const float* x) {
    return make_uint4(both(x[0], x[1]), both(x[2], x[3]), both(x[4], x[5]), both(x[6], x[7]));
  }
};

}  // namespace sdm
