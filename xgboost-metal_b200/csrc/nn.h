// Device operators that put a learned model on top of leaf indices: embedding
// lookup with scaling (one token or a summed bag a row), its gradient by
// sorted tokens, and layer norm's forward and backward pass. Every pointer is
// a device pointer of the caller's, work is enqueued on the caller's stream
// and nothing is allocated or waited for.
#pragma once
#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

namespace xgbb::nn {

// The dtype codes of XGBufferDescriptor (include/xgboost/c_api.h).
enum Type : int { kF32 = 1, kF16 = 3, kBF16 = 4, kI32 = 7, kI64 = 8 };
size_t type_size(int type);

// A matrix whose rows are contiguous; stride in elements.
struct Mat {
  const void* data;
  int type;
  int64_t stride;
};

// tokens[rows][per_row], strides in elements; below 0: missing.
struct Tokens {
  const void* data;
  int type;
  uint64_t rows, per_row;
  int64_t stride_row, stride_col;
};

// f32 [rows][per_row] or null (all ones); strides may be 0 (broadcast).
struct Scales {
  const float* data;
  int64_t stride_row, stride_col;
};

// out[r] = scale * sum_t scales[r][t] * table[tokens[r][t]].
void embedding(const Tokens& k, const Mat& table, uint64_t vocab, uint64_t dim, float scale, const Scales& s,
               const Mat& out, cudaStream_t stream);
// out[v] (+)= scale * sum over tokens[r][t] == v of scales[r][t] * grad[r].
size_t embedding_backward_workspace(const Tokens& k, uint64_t vocab, uint64_t dim);
void embedding_backward(const Mat& grad, const Tokens& k, uint64_t vocab, uint64_t dim, float scale,
                        const Scales& s, const Mat& out, bool accumulate, void* workspace,
                        cudaStream_t stream);
// out[r][t] = scale * <grad[r], table[tokens[r][t]]>, contiguous.
void embedding_scale_backward(const Mat& grad, const Tokens& k, const Mat& table, uint64_t vocab, uint64_t dim,
                              float scale, float* out, cudaStream_t stream);

// y = (x - mean) * rstd * weight + bias over rows of `dim`; weight and bias
// share a type and may be null; mean and rstd may be null.
void layer_norm(const Mat& x, uint64_t rows, uint64_t dim, const void* weight, const void* bias, int param_type,
                float eps, const Mat& y, float* mean, float* rstd, cudaStream_t stream);
// dx and, where not null, the gradients of weight and bias.
size_t layer_norm_backward_workspace(uint64_t rows, uint64_t dim);
void layer_norm_backward(const Mat& grad, const Mat& x, const float* mean, const float* rstd, uint64_t rows,
                         uint64_t dim, const void* weight, int param_type, const Mat& dx, void* dweight,
                         void* dbias, void* workspace, cudaStream_t stream);

}  // namespace xgbb::nn
