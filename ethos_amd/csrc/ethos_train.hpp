// Operators of a training step around the blocks: the loss over the vocabulary (loss.hip), the
// embedding (embed.hip), the experts' balance (balance.hip) and gradient clipping (clip.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace ethos {

enum Reduction : int { kLossMean = 0, kLossSum = 1, kLossNone = 2 };

// Softmax cross entropy of rows h against a head matrix w [vocab, d].
size_t linear_ce_state_bytes(int64_t n, int d, int dtype);
size_t linear_ce_workspace_bytes(int64_t n, int d, int64_t vocab, int dtype, int num_cus);
size_t linear_ce_exps_bytes(int64_t n, int64_t vocab, int dtype, int num_cus);
size_t linear_ce_grad_workspace_bytes(int64_t n, int d, int64_t vocab, int dtype, int num_cus, bool kept);
int launch_linear_ce(const void* h, int64_t ldh, const void* w, const int64_t* labels, int64_t n, int d, int64_t vocab,
                     int64_t ignore, int reduction, int dtype, void* state, void* exps, void* ws, float* loss, int num_cus,
                     hipStream_t stream);
int launch_linear_ce_grad(const void* state, void* exps, const void* w, const float* dloss, int64_t n, int d, int64_t vocab, int reduction,
                          int dtype, void* ws, void* dh, void* dw, int num_cus, hipStream_t stream);

int launch_embedding(const void* ids, int ids_64, const void* w, int64_t n, int d, int64_t vocab, float scale, int64_t padding,
                     int dtype, void* out, int32_t* keys, int num_cus, hipStream_t stream);
size_t embedding_grad_workspace_bytes(int64_t n, int d, int64_t vocab);
int launch_embedding_grad(const int32_t* keys, const void* dy, int64_t n, int d, int64_t vocab, float scale, int dtype, void* ws,
                          void* dw, int num_cus, hipStream_t stream);

size_t balance_workspace_bytes(int64_t pairs, int64_t n_experts);
int launch_balance(const void* gates, const void* ids, int ids_64, int64_t pairs, int64_t n_experts, double scale, int dtype,
                   void* ws, int32_t* counts, float* loss, int num_cus, hipStream_t stream);
int launch_balance_grad(const void* ids, int ids_64, const int32_t* counts, const float* dloss, int64_t pairs, int64_t n_experts,
                        double scale, int dtype, void* dgates, int num_cus, hipStream_t stream);

size_t clip_workspace_bytes(const int64_t* sizes, int n_tensors);
int launch_clip(const void* const* in, void* const* out, const int64_t* sizes, const int32_t* dtypes, int n_tensors, int inf_norm,
                double max_norm, void* ws, float* total, hipStream_t stream);

}  // namespace ethos
