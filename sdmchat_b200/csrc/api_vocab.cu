// C entry points of the vocabulary-end operators (declared in include/sdm_b200.h): argument checks, then the launch.
#include <math.h>
#include "vocab.cuh"

using namespace sdm;

namespace {

inline cudaStream_t S(void* st) { return static_cast<cudaStream_t>(st); }
inline sdm_status to_status(cudaError_t e) { return e == cudaSuccess ? SDM_OK : SDM_ERR_CUDA; }
inline bool dtype_ok(int dt) { return dt == SDM_F32 || dt == SDM_BF16; }
inline bool aligned(const void* p, int dtype) { return (reinterpret_cast<uintptr_t>(p) & (dtype == SDM_BF16 ? 1 : 3)) == 0; }

const sdm_logit_rules kNoRules = {nullptr, 0,       0,       nullptr, nullptr, nullptr, nullptr, nullptr,
                                  1.f,     0.f,     0.f,     nullptr, nullptr, 0,       nullptr, 0,       nullptr};

// Rules for S rows over V tokens.
sdm_status check_rules(const sdm_logit_rules& r, int64_t rows) {
  if (r.history) {
    if (r.history_n < 0 || r.history_n > kMaxHistory || r.history_ld < r.history_n) return SDM_ERR_SHAPE;
  } else if (r.history_len || r.prompt_len) {
    return SDM_ERR_ARG;
  }
  if ((r.bias_ids != nullptr) != (r.bias_values != nullptr)) return SDM_ERR_ARG;
  if (r.bias_ids && (r.bias_n < 0 || r.bias_n > kMaxBias)) return SDM_ERR_SHAPE;
  if (r.mask) {
    if (r.mask_rows < 1) return SDM_ERR_SHAPE;
    if (!r.mask_row && r.mask_rows != 1 && r.mask_rows != rows) return SDM_ERR_SHAPE;
  } else if (r.mask_row) {
    return SDM_ERR_ARG;
  }
  return SDM_OK;
}

}  // namespace

extern "C" {

sdm_status sdm_logits_process(const sdm_logit_rules* rules, const void* logits, int64_t ld, int64_t rows, int V,
                              int dtype, void* out, int64_t ld_out, void* stream) {
  if ((rows != 0 && (!logits || !out)) || !dtype_ok(dtype) || !aligned(logits, dtype) || !aligned(out, dtype))
    return SDM_ERR_ARG;
  if (rows < 0 || V < 1 || V > (1 << 30) || ld < V || ld_out < V) return SDM_ERR_SHAPE;
  if (rows == 0) return SDM_OK;
  if (logits == out && ld != ld_out) return SDM_ERR_ARG;
  const sdm_logit_rules& r = rules ? *rules : kNoRules;
  const sdm_status s = check_rules(r, rows);
  if (s != SDM_OK) return s;
  if (ceil_div((int64_t)V + 7, 1024) > 0x7fffffff / (rows > 0 ? rows : 1)) return SDM_ERR_SHAPE;
  return to_status(launch_logits_process(r, logits, ld, rows, V, dtype, out, ld_out, S(stream)));
}

sdm_status sdm_logits_choose(const sdm_logit_rules* rules, const sdm_choice_params* choice, const void* logits,
                             int64_t ld, int64_t rows, int V, int dtype, int32_t* ids, float* logprob, void* stream) {
  if (!choice || (rows != 0 && (!logits || !ids)) || !dtype_ok(dtype) || !aligned(logits, dtype)) return SDM_ERR_ARG;
  if (rows < 0 || rows > 0x7fffffff / kMaxCluster || V < 1 || V > kMaxChoiceV || ld < V) return SDM_ERR_SHAPE;
  if (rows == 0) return SDM_OK;
  if (!choice->temperature && !(choice->temperature_all >= 0.f)) return SDM_ERR_ARG;
  if (!choice->u && (choice->temperature || choice->temperature_all > 0.f)) return SDM_ERR_ARG;
  const sdm_logit_rules& r = rules ? *rules : kNoRules;
  const sdm_status s = check_rules(r, rows);
  if (s != SDM_OK) return s;
  return to_status(launch_logits_choose(r, *choice, logits, ld, rows, V, dtype, ids, logprob, S(stream)));
}

sdm_status sdm_distill(const void* logits, int64_t ld, int64_t N, int V, int dtype, const int32_t* teacher_ids,
                       const float* teacher_logits, int k, const float* teacher_lse, const int32_t* targets,
                       const float* row_weight, float temperature, float alpha, float grad_scale, float* loss,
                       void* dlogits, int64_t ld_grad, void* stream) {
  if ((N != 0 && (!logits || !teacher_ids || !teacher_logits || !loss)) || !dtype_ok(dtype) ||
      !aligned(logits, dtype) || !aligned(dlogits, dtype))
    return SDM_ERR_ARG;
  // 1 / T scales every logit, T^2 the loss
  if (!(temperature > 0.f) || !isfinite(1.f / temperature) || !isfinite(temperature * temperature) || !isfinite(alpha) ||
      !isfinite(grad_scale))
    return SDM_ERR_ARG;
  if (N < 0 || N > 0x7fffffff / kMaxCluster || V < 1 || V > kMaxChoiceV || ld < V || (dlogits && ld_grad < V) ||
      k < 1 || k > kMaxTeacher)
    return SDM_ERR_SHAPE;
  if (N == 0) return SDM_OK;
  if (logits == dlogits && ld != ld_grad) return SDM_ERR_ARG;
  DistillArgs a = {logits, ld,    N,     V,          k,    teacher_ids, teacher_logits, teacher_lse, targets, row_weight,
                   temperature, alpha, grad_scale, loss, dlogits,     ld_grad};
  return to_status(launch_distill(a, dtype, S(stream)));
}

sdm_status sdm_scale_rows(void* x, int64_t ld, int64_t N, int V, int dtype, const float* g, int g_stride,
                          void* stream) {
  if ((N != 0 && !x) || !g || !dtype_ok(dtype) || !aligned(x, dtype) || (g_stride != 0 && g_stride != 1)) return SDM_ERR_ARG;
  if (N < 0 || N > 0x7fffffff || V < 1 || ld < V) return SDM_ERR_SHAPE;
  return to_status(launch_scale_rows(x, ld, N, V, dtype, g, g_stride, S(stream)));
}

sdm_status sdm_embed_scaled(const int32_t* ids, const void* emb, int64_t N, int d, int V, float scale, int dtype,
                            void* out, int* bad, void* stream) {
  if (!emb || (N != 0 && (!ids || !out)) || !dtype_ok(dtype) || !aligned(emb, dtype) || !aligned(out, dtype)) return SDM_ERR_ARG;
  if (N < 0 || N > (1 << 30) || d < 1 || d > (1 << 30) || V < 1) return SDM_ERR_SHAPE;  // columns are counted in an int
  return to_status(launch_embed_scaled(ids, emb, N, d, V, scale, dtype, out, bad, S(stream)));
}

size_t sdm_embed_grad_workspace_size(int64_t N, int d, int V) {
  if (N < 0 || N > (1 << 30) || d < 1 || d > (1 << 20) || V < 1 || V > (1 << 24)) return 0;
  return embed_grad_workspace_bytes(N, d, V);
}

sdm_status sdm_embed_grad(const int32_t* ids, const void* dout, int64_t ld, int64_t N, int d, int V, float scale,
                          int padding_id, int dtype, int grad_dtype, int accumulate, void* grad, void* workspace,
                          size_t workspace_bytes, void* stream) {
  if (!grad || !dtype_ok(dtype) || !dtype_ok(grad_dtype) || !aligned(grad, grad_dtype)) return SDM_ERR_ARG;
  if (N > 0 && (!ids || !dout || !aligned(dout, dtype))) return SDM_ERR_ARG;
  if (N < 0 || N > (1 << 30) || d < 1 || d > (1 << 20) || V < 1 || V > (1 << 24) || ld < d) return SDM_ERR_SHAPE;
  if (workspace_bytes < embed_grad_workspace_bytes(N, d, V) || !workspace) return SDM_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(workspace) & 15) return SDM_ERR_ARG;
  return to_status(launch_embed_grad(ids, dout, ld, N, d, V, scale, padding_id, dtype, grad_dtype, accumulate, grad,
                                     workspace, S(stream)));
}

}  // extern "C"
