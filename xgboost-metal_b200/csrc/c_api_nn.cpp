// C ABI of the device operators of nn.h: argument checks, device selection
// and dispatch. All checks come before anything is enqueued.
#include <cmath>

#include "c_api_common.h"
#include "nn.h"
#include "xgb_b200.h"

using namespace xgbb::capi;
using xgbb::require;
namespace nn = xgbb::nn;

namespace {

// Makes `device` current for the call (-1: the calling thread's current one).
class OnDevice {
 public:
  explicit OnDevice(int device) {
    int now = 0;
    cudaError_t e = cudaGetDevice(&now);
    if (e == cudaErrorNoDevice || e == cudaErrorInsufficientDriver) ensure_device();
    xgbb::cuda_check(e, "cudaGetDevice");
    if (device < 0 || device == now) return;
    XGBB_CUDA(cudaSetDevice(device));
    back_ = now;
  }
  ~OnDevice() {
    if (back_ >= 0) cudaSetDevice(back_);
  }
  OnDevice(const OnDevice&) = delete;

 private:
  int back_ = -1;
};

bool is_float(int t) { return t == nn::kF32 || t == nn::kF16 || t == nn::kBF16; }

void require_pointer(const void* p, size_t align, const char* what) {
  if (!p) throw xgbb::Error(std::string(what) + " is a null pointer");
  if (reinterpret_cast<uintptr_t>(p) % align) throw xgbb::Error(std::string(what) + " is not aligned to its type");
}

void require_mat(const nn::Mat& m, uint64_t rows, uint64_t dim, bool written, const char* what) {
  if (!is_float(m.type)) throw xgbb::Error(std::string(what) + " must be float32 (1), float16 (3) or bfloat16 (4)");
  if (!rows) return;
  require_pointer(m.data, nn::type_size(m.type), what);
  if (m.stride < 0 || (written && rows > 1 && uint64_t(m.stride) < dim))
    throw xgbb::Error(std::string(what) + (written ? " has rows that overlap" : " has a negative row stride"));
}

void require_types(int a, int b, const char* message) { require(a == b || a == nn::kF32 || b == nn::kF32, message); }

constexpr uint64_t kMaxDim = 1u << 20, kMaxTokens = 0x7fffffffu;

void require_dim(uint64_t dim) { require(dim >= 1 && dim <= kMaxDim, "dim must be between 1 and 1048576"); }

void require_tokens(const nn::Tokens& k, uint64_t vocab, uint64_t dim) {
  require_dim(dim);
  require(k.type == nn::kI32 || k.type == nn::kI64, "tokens must be int32 (7) or int64 (8)");
  require(vocab >= 1 && vocab <= kMaxTokens, "vocab must be between 1 and 2147483647");
  require(k.rows <= kMaxTokens && k.per_row <= kMaxTokens && k.rows * k.per_row <= kMaxTokens,
          "there may be at most 2147483647 tokens");
  if (k.rows * k.per_row) require_pointer(k.data, nn::type_size(k.type), "tokens");
}

void require_scales(const nn::Scales& s) {
  if (s.data) require_pointer(s.data, 4, "token_scale");
}

void require_finite(float v, const char* message) { require(std::isfinite(v), message); }

}  // namespace

XGB_DLL int XGBBEmbedding(int device, const void* tokens, int token_type, bst_ulong rows, bst_ulong per_row,
                          int64_t token_stride_row, int64_t token_stride_col, const void* table, int table_type,
                          bst_ulong vocab, bst_ulong dim, int64_t table_stride, float scale,
                          const float* token_scale, int64_t scale_stride_row, int64_t scale_stride_col, void* out,
                          int out_type, int64_t out_stride, void* stream) {
  return guarded([&] {
    const nn::Tokens k{tokens, token_type, rows, per_row, token_stride_row, token_stride_col};
    const nn::Mat w{table, table_type, table_stride}, y{out, out_type, out_stride};
    const nn::Scales s{token_scale, scale_stride_row, scale_stride_col};
    require_tokens(k, vocab, dim);
    require_mat(w, vocab, dim, false, "table");
    require_mat(y, rows, dim, true, "out");
    require_types(table_type, out_type, "out must have the table's type, or one of them must be float32");
    require_scales(s);
    require_finite(scale, "scale must be finite");
    require(!rows || out != table, "out must not be the table");
    const OnDevice on(device);
    nn::embedding(k, w, vocab, dim, scale, s, y, static_cast<cudaStream_t>(stream));
  });
}

XGB_DLL int XGBBEmbeddingBackwardWorkspace(bst_ulong rows, bst_ulong per_row, bst_ulong vocab, bst_ulong dim,
                                           size_t* bytes) {
  return guarded([&] {
    require(bytes != nullptr, "bytes is a null pointer");
    const nn::Tokens k{bytes, nn::kI32, rows, per_row, 0, 0};
    require_tokens(k, vocab, dim);
    *bytes = nn::embedding_backward_workspace(k, vocab, dim);
  });
}

XGB_DLL int XGBBEmbeddingBackward(int device, const void* grad, int grad_type, int64_t grad_stride,
                                  const void* tokens, int token_type, bst_ulong rows, bst_ulong per_row,
                                  int64_t token_stride_row, int64_t token_stride_col, bst_ulong vocab,
                                  bst_ulong dim, float scale, const float* token_scale, int64_t scale_stride_row,
                                  int64_t scale_stride_col, void* out, int out_type, int64_t out_stride,
                                  int accumulate, void* workspace, size_t workspace_bytes, void* stream) {
  return guarded([&] {
    const nn::Tokens k{tokens, token_type, rows, per_row, token_stride_row, token_stride_col};
    const nn::Mat g{grad, grad_type, grad_stride}, y{out, out_type, out_stride};
    const nn::Scales s{token_scale, scale_stride_row, scale_stride_col};
    require_tokens(k, vocab, dim);
    require_mat(g, rows, dim, false, "grad");
    require_mat(y, vocab, dim, true, "out");
    require_types(grad_type, out_type, "out must have grad's type, or one of them must be float32");
    require_scales(s);
    require_finite(scale, "scale must be finite");
    require(!rows || out != grad, "out must not be grad");
    if (nn::embedding_backward_workspace(k, vocab, dim)) require_pointer(workspace, 256, "workspace");
    const OnDevice on(device);
    nn::embedding_backward(g, k, vocab, dim, scale, s, y, accumulate != 0, workspace, workspace_bytes,
                           static_cast<cudaStream_t>(stream));
  });
}

XGB_DLL int XGBBEmbeddingScaleBackward(int device, const void* grad, int grad_type, int64_t grad_stride,
                                       const void* tokens, int token_type, bst_ulong rows, bst_ulong per_row,
                                       int64_t token_stride_row, int64_t token_stride_col, const void* table,
                                       int table_type, bst_ulong vocab, bst_ulong dim, int64_t table_stride,
                                       float scale, float* out, void* stream) {
  return guarded([&] {
    const nn::Tokens k{tokens, token_type, rows, per_row, token_stride_row, token_stride_col};
    const nn::Mat g{grad, grad_type, grad_stride}, w{table, table_type, table_stride};
    require_tokens(k, vocab, dim);
    require_mat(g, rows, dim, false, "grad");
    require_mat(w, vocab, dim, false, "table");
    require_types(table_type, grad_type, "grad must have the table's type, or one of them must be float32");
    require_finite(scale, "scale must be finite");
    if (rows * per_row) require_pointer(out, 4, "out");
    const OnDevice on(device);
    nn::embedding_scale_backward(g, k, w, vocab, dim, scale, out, static_cast<cudaStream_t>(stream));
  });
}

XGB_DLL int XGBBLayerNorm(int device, const void* x, int type, bst_ulong rows, bst_ulong dim, int64_t x_stride,
                          const void* weight, const void* bias, int param_type, float eps, void* y,
                          int64_t y_stride, float* mean, float* rstd, void* stream) {
  return guarded([&] {
    const nn::Mat in{x, type, x_stride}, out{y, type, y_stride};
    require_dim(dim);
    require(rows <= kMaxTokens, "there may be at most 2147483647 rows");
    require_mat(in, rows, dim, false, "x");
    require_mat(out, rows, dim, true, "y");
    require(is_float(param_type), "weight and bias must be float32 (1), float16 (3) or bfloat16 (4)");
    require(param_type == type || param_type == nn::kF32, "weight and bias must have x's type or be float32");
    if (weight) require_pointer(weight, nn::type_size(param_type), "weight");
    if (bias) require_pointer(bias, nn::type_size(param_type), "bias");
    if (mean) require_pointer(mean, 4, "mean");
    if (rstd) require_pointer(rstd, 4, "rstd");
    require(std::isfinite(eps) && eps >= 0.0f, "eps must be finite and not negative");
    require(!rows || x != y, "y must not be x");
    const OnDevice on(device);
    nn::layer_norm(in, rows, dim, weight, bias, param_type, eps, out, mean, rstd,
                   static_cast<cudaStream_t>(stream));
  });
}

XGB_DLL int XGBBLayerNormBackwardWorkspace(bst_ulong rows, bst_ulong dim, size_t* bytes) {
  return guarded([&] {
    require(bytes != nullptr, "bytes is a null pointer");
    require_dim(dim);
    require(rows <= kMaxTokens, "there may be at most 2147483647 rows");
    *bytes = nn::layer_norm_backward_workspace(rows, dim);
  });
}

XGB_DLL int XGBBLayerNormBackward(int device, const void* grad, int64_t grad_stride, const void* x, int type,
                                  bst_ulong rows, bst_ulong dim, int64_t x_stride, const float* mean,
                                  const float* rstd, const void* weight, int param_type, void* dx,
                                  int64_t dx_stride, void* dweight, void* dbias, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  return guarded([&] {
    const nn::Mat g{grad, type, grad_stride}, in{x, type, x_stride}, out{dx, type, dx_stride};
    require_dim(dim);
    require(rows <= kMaxTokens, "there may be at most 2147483647 rows");
    require_mat(g, rows, dim, false, "grad");
    require_mat(in, rows, dim, false, "x");
    require_mat(out, rows, dim, true, "dx");
    require(is_float(param_type), "weight must be float32 (1), float16 (3) or bfloat16 (4)");
    require(param_type == type || param_type == nn::kF32, "weight must have x's type or be float32");
    if (rows) {
      require_pointer(mean, 4, "mean");
      require_pointer(rstd, 4, "rstd");
    }
    if (weight) require_pointer(weight, nn::type_size(param_type), "weight");
    if (dweight) require_pointer(dweight, nn::type_size(param_type), "dweight");
    if (dbias) require_pointer(dbias, nn::type_size(param_type), "dbias");
    require(!rows || (dx != grad && dx != x), "dx must be neither grad nor x");
    if ((dweight || dbias) && nn::layer_norm_backward_workspace(rows, dim))
      require_pointer(workspace, 256, "workspace");
    const OnDevice on(device);
    nn::layer_norm_backward(g, in, mean, rstd, rows, dim, weight, param_type, out, dweight, dbias, workspace,
                            workspace_bytes, static_cast<cudaStream_t>(stream));
  });
}
