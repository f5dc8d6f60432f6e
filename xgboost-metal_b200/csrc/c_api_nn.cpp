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

// The default stream has two handles.
bool is_default(cudaStream_t s) { return s == nullptr || s == cudaStreamLegacy; }

// The capture that a stream is in, 0 for none. The default stream is in none,
// and may not be asked during one.
unsigned long long capture_of(cudaStream_t s) {
  if (is_default(s)) return 0;
  cudaStreamCaptureStatus status;
  unsigned long long id = 0;
  XGBB_CUDA(cudaStreamGetCaptureInfo(s, &status, &id));
  return status == cudaStreamCaptureStatusNone ? 0 : id;
}

void stream_wait(cudaStream_t stream, cudaStream_t after) {
  if (stream == after || (is_default(stream) && is_default(after))) return;
  const unsigned long long capture = capture_of(stream);
  if (capture && capture_of(after) != capture) return;
  cudaEvent_t event;
  XGBB_CUDA(cudaEventCreateWithFlags(&event, cudaEventDisableTiming));
  cudaError_t e = cudaEventRecord(event, after);
  if (e == cudaSuccess) e = cudaStreamWaitEvent(stream, event, 0);
  cudaEventDestroy(event);  // freed once it is done
  xgbb::cuda_check(e, "cudaStreamWaitEvent");
}

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

nn::Tokens tokens_of(const XGBBTokens& t, uint64_t vocab, uint64_t dim) {
  const nn::Tokens k{t.tokens, t.type, t.rows, t.per_row, t.stride_row, t.stride_col};
  require_tokens(k, vocab, dim);
  require(std::isfinite(t.scale), "scale must be finite");
  return k;
}

nn::Scales scales_of(const XGBBTokens& t) {
  if (t.token_scale) require_pointer(t.token_scale, 4, "token_scale");
  return {t.token_scale, t.scale_stride_row, t.scale_stride_col};
}

void require_rows(uint64_t rows, uint64_t dim) {
  require_dim(dim);
  require(rows <= kMaxTokens, "there may be at most 2147483647 rows");
}

void require_params(int type, int param_type) {
  require(is_float(param_type), "weight and bias must be float32 (1), float16 (3) or bfloat16 (4)");
  require(param_type == type || param_type == nn::kF32, "weight and bias must have x's type or be float32");
}

}  // namespace

XGB_DLL int XGBBEmbedding(const XGBBEmbeddingArgs* args) {
  return guarded([&] {
    require(args != nullptr, "args is a null pointer");
    const XGBBEmbeddingArgs& a = *args;
    const nn::Tokens k = tokens_of(a.tokens, a.vocab, a.dim);
    const nn::Scales s = scales_of(a.tokens);
    const nn::Mat w{a.table, a.table_type, a.table_stride}, y{a.out, a.out_type, a.out_stride};
    require_mat(w, a.vocab, a.dim, false, "table");
    require_mat(y, k.rows, a.dim, true, "out");
    require_types(a.table_type, a.out_type, "out must have the table's type, or one of them must be float32");
    require(!k.rows || a.out != a.table, "out must not be the table");
    const OnDevice on(a.device);
    nn::embedding(k, w, a.vocab, a.dim, a.tokens.scale, s, y, static_cast<cudaStream_t>(a.stream));
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

XGB_DLL int XGBBEmbeddingBackward(const XGBBEmbeddingBackwardArgs* args) {
  return guarded([&] {
    require(args != nullptr, "args is a null pointer");
    const XGBBEmbeddingBackwardArgs& a = *args;
    const nn::Tokens k = tokens_of(a.tokens, a.vocab, a.dim);
    const nn::Scales s = scales_of(a.tokens);
    const nn::Mat g{a.grad, a.grad_type, a.grad_stride}, y{a.out, a.out_type, a.out_stride};
    require_mat(g, k.rows, a.dim, false, "grad");
    require_mat(y, a.vocab, a.dim, true, "out");
    require_types(a.grad_type, a.out_type, "out must have grad's type, or one of them must be float32");
    require(!k.rows || a.out != a.grad, "out must not be grad");
    if (const size_t need = nn::embedding_backward_workspace(k, a.vocab, a.dim)) {
      require_pointer(a.workspace, 256, "workspace");
      require(a.workspace_bytes >= need, "the workspace is smaller than its query says");
    }
    const OnDevice on(a.device);
    nn::embedding_backward(g, k, a.vocab, a.dim, a.tokens.scale, s, y, a.accumulate != 0, a.workspace,
                           static_cast<cudaStream_t>(a.stream));
  });
}

XGB_DLL int XGBBEmbeddingScaleBackward(const XGBBEmbeddingScaleBackwardArgs* args) {
  return guarded([&] {
    require(args != nullptr, "args is a null pointer");
    const XGBBEmbeddingScaleBackwardArgs& a = *args;
    const nn::Tokens k = tokens_of(a.tokens, a.vocab, a.dim);
    const nn::Mat g{a.grad, a.grad_type, a.grad_stride}, w{a.table, a.table_type, a.table_stride};
    require_mat(g, k.rows, a.dim, false, "grad");
    require_mat(w, a.vocab, a.dim, false, "table");
    require_types(a.table_type, a.grad_type, "grad must have the table's type, or one of them must be float32");
    if (k.rows * k.per_row) require_pointer(a.out, 4, "out");
    const OnDevice on(a.device);
    nn::embedding_scale_backward(g, k, w, a.vocab, a.dim, a.tokens.scale, a.out,
                                 static_cast<cudaStream_t>(a.stream));
  });
}

XGB_DLL int XGBBLayerNorm(const XGBBLayerNormArgs* args) {
  return guarded([&] {
    require(args != nullptr, "args is a null pointer");
    const XGBBLayerNormArgs& a = *args;
    const nn::Mat in{a.x, a.type, a.x_stride}, out{a.y, a.type, a.y_stride};
    require_rows(a.rows, a.dim);
    require_mat(in, a.rows, a.dim, false, "x");
    require_mat(out, a.rows, a.dim, true, "y");
    require_params(a.type, a.param_type);
    if (a.weight) require_pointer(a.weight, nn::type_size(a.param_type), "weight");
    if (a.bias) require_pointer(a.bias, nn::type_size(a.param_type), "bias");
    if (a.mean) require_pointer(a.mean, 4, "mean");
    if (a.rstd) require_pointer(a.rstd, 4, "rstd");
    require(std::isfinite(a.eps) && a.eps >= 0.0f, "eps must be finite and not negative");
    require(!a.rows || a.x != a.y, "y must not be x");
    const OnDevice on(a.device);
    nn::layer_norm(in, a.rows, a.dim, a.weight, a.bias, a.param_type, a.eps, out, a.mean, a.rstd,
                   static_cast<cudaStream_t>(a.stream));
  });
}

XGB_DLL int XGBBLayerNormBackwardWorkspace(bst_ulong rows, bst_ulong dim, size_t* bytes) {
  return guarded([&] {
    require(bytes != nullptr, "bytes is a null pointer");
    require_rows(rows, dim);
    *bytes = nn::layer_norm_backward_workspace(rows, dim);
  });
}

XGB_DLL int XGBBLayerNormBackward(const XGBBLayerNormBackwardArgs* args) {
  return guarded([&] {
    require(args != nullptr, "args is a null pointer");
    const XGBBLayerNormBackwardArgs& a = *args;
    const nn::Mat g{a.grad, a.type, a.grad_stride}, in{a.x, a.type, a.x_stride}, out{a.dx, a.type, a.dx_stride};
    require_rows(a.rows, a.dim);
    require_mat(g, a.rows, a.dim, false, "grad");
    require_mat(in, a.rows, a.dim, false, "x");
    require_mat(out, a.rows, a.dim, true, "dx");
    require_params(a.type, a.param_type);
    if (a.rows) {
      require_pointer(a.mean, 4, "mean");
      require_pointer(a.rstd, 4, "rstd");
    }
    if (a.weight) require_pointer(a.weight, nn::type_size(a.param_type), "weight");
    if (a.dweight) require_pointer(a.dweight, nn::type_size(a.param_type), "dweight");
    if (a.dbias) require_pointer(a.dbias, nn::type_size(a.param_type), "dbias");
    require(!a.rows || (a.dx != a.grad && a.dx != a.x), "dx must be neither grad nor x");
    const size_t need = a.dweight || a.dbias ? nn::layer_norm_backward_workspace(a.rows, a.dim) : 0;
    if (need) {
      require_pointer(a.workspace, 256, "workspace");
      require(a.workspace_bytes >= need, "the workspace is smaller than its query says");
    }
    const OnDevice on(a.device);
    nn::layer_norm_backward(g, in, a.mean, a.rstd, a.rows, a.dim, a.weight, a.param_type, out, a.dweight, a.dbias,
                            a.workspace, static_cast<cudaStream_t>(a.stream));
  });
}

XGB_DLL int XGBBStreamWait(int32_t device, void* stream, void* after) {
  return guarded([&] {
    const OnDevice on(device);
    stream_wait(static_cast<cudaStream_t>(stream), static_cast<cudaStream_t>(after));
  });
}
