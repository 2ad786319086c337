// extern "C" boundary of the layer operators (declared in
// include/muspace_msda.h): linear_act, layer norm and 8-bit checkpoints.
#include <cuda_runtime.h>

#include <limits>
#include <string>

#include "../../include/muspace_msda.h"
#include "capi_common.h"
#include "layer_norm.h"
#include "linear_act.h"

namespace {

using capi::check_launch;
using capi::fail;
using capi::guarded;
using capi::require;

constexpr int64_t kMax = std::numeric_limits<int32_t>::max();

void check_dtype(int dtype, const char* name = "dtype") {
  require(dtype == MSDA_DTYPE_FLOAT32 || dtype == MSDA_DTYPE_BFLOAT16,
          std::string(name) + " must be float32 or bfloat16");
}

void check_size(int64_t n, const char* name) {
  require(n >= 0, "sizes must be non-negative");
  require(n <= kMax, std::string(name) + " exceeds the supported range (< 2^31)");
}

void check_pointer(bool needed, const void* p, const char* name) {
  require(!needed || p != nullptr, std::string(name) + " is null");
}

void check_workspace(const void* p, size_t has, size_t needs) {
  if (needs == 0) return;
  require(p != nullptr && has >= needs,
          "workspace has " + std::to_string(p ? has : 0) + " bytes, " + std::to_string(needs) + " are needed");
  require((reinterpret_cast<uintptr_t>(p) & 255) == 0, "workspace must be 256-byte aligned");
}

lin::Args linear_args(const msda_linear_t* in, bool backward) {
  require(in != nullptr, "args is null");
  check_dtype(in->dtype);
  require(in->activation >= MSDA_ACTIVATION_NONE && in->activation <= MSDA_ACTIVATION_SILU,
          "activation must be none, relu, gelu or silu");
  check_size(in->rows, "rows");
  check_size(in->in_features, "in_features");
  check_size(in->out_features, "out_features");
  require(in->input_stride >= 0 && in->weight_stride >= 0 && in->residual_stride >= 0 && in->output_stride >= 0 &&
              in->grad_output_stride >= 0,
          "strides must be non-negative");
  const bool some_x = in->rows > 0 && in->in_features > 0, some_w = in->out_features > 0 && in->in_features > 0;
  const bool some_y = in->rows > 0 && in->out_features > 0;
  if (backward) {
    const bool recompute = in->activation != MSDA_ACTIVATION_NONE && in->slope == nullptr;
    require((in->codes == nullptr) == (in->exponents == nullptr), "codes and exponents go together");
    check_pointer(some_w && (recompute || in->grad_input), in->weight, "weight");
    check_pointer(some_x && !in->codes && (recompute || in->grad_weight), in->input, "input");
    check_pointer(some_y, in->grad_output, "grad_output");
  } else {
    check_pointer(some_w, in->weight, "weight");
    check_pointer(some_x, in->input, "input");
    check_pointer(some_y, in->output, "output");
    require(in->rows <= 1 || in->output_stride >= in->out_features, "output rows must not overlap");
  }
  lin::Args a{};
  a.dtype = static_cast<lin::DType>(in->dtype);
  a.act = static_cast<lin::Act>(in->activation);
  a.rows = in->rows, a.in = in->in_features, a.out = in->out_features;
  a.x_stride = in->input_stride, a.w_stride = in->weight_stride, a.r_stride = in->residual_stride;
  a.y_stride = in->output_stride, a.g_stride = in->grad_output_stride;
  a.x = in->input, a.w = in->weight, a.bias = in->bias;
  a.slope = in->slope;
  if (backward) {
    a.g = in->grad_output;
    a.dx = in->grad_input, a.dw = in->grad_weight, a.db = in->grad_bias;
    a.codes = in->codes, a.exps = in->exponents;
  } else {
    a.r = in->residual;
    a.y = in->output;
  }
  a.workspace = in->workspace;
  a.workspace_bytes = in->workspace_bytes;
  return a;
}

lnorm::Args norm_args(const msda_layer_norm_t* in, bool backward) {
  require(in != nullptr, "args is null");
  check_dtype(in->dtype);
  check_dtype(in->weight_dtype, "weight_dtype");
  require(in->weight_dtype == in->dtype || in->weight_dtype == MSDA_DTYPE_FLOAT32,
          "weight_dtype must be dtype or float32");
  check_size(in->rows, "rows");
  check_size(in->cols, "cols");
  require(in->input_stride >= 0 && in->grad_output_stride >= 0, "strides must be non-negative");
  require((in->codes == nullptr) == (in->exponents == nullptr), "codes and exponents go together");
  require((in->mean == nullptr) == (in->rstd == nullptr), "mean and rstd go together");
  const bool some = in->rows > 0 && in->cols > 0;
  lnorm::Args a{};
  a.dtype = static_cast<lnorm::DType>(in->dtype);
  a.weight_dtype = static_cast<lnorm::DType>(in->weight_dtype);
  a.rows = in->rows, a.cols = in->cols;
  a.x_stride = in->input_stride, a.g_stride = in->grad_output_stride;
  a.eps = in->eps;
  a.x = in->input, a.w = in->weight;
  a.mean = in->mean, a.rstd = in->rstd;
  if (backward) {
    check_pointer(some, in->grad_output, "grad_output");
    check_pointer(some && !in->codes, in->input, "input");
    check_pointer(some && !in->codes, in->mean, "mean");
    a.g = in->grad_output;
    a.codes_in = in->codes, a.exps_in = in->exponents;
    a.dx = in->grad_input, a.dw = in->grad_weight, a.db = in->grad_bias;
    a.parts = static_cast<float*>(in->workspace);
  } else {
    check_pointer(some, in->input, "input");
    check_pointer(some, in->output, "output");
    a.b = in->bias;
    a.y = in->output;
    a.codes = in->codes, a.exps = in->exponents;
  }
  return a;
}

size_t norm_workspace(const msda_layer_norm_t& in) {
  if (!in.grad_weight && !in.grad_bias) return 0;
  return static_cast<size_t>(lnorm::backward_parts(in.rows, in.cols)) * 2 * in.cols * sizeof(float);
}

}  // namespace

extern "C" {

int msda_checkpoint_pack(msda_dtype_t dtype, const void* input, int64_t rows, int64_t cols, int64_t input_stride,
                         int8_t* codes, uint8_t* exponents, void* stream) {
  return guarded([&] {
    check_dtype(dtype);
    check_size(rows, "rows");
    check_size(cols, "cols");
    require(input_stride >= 0, "strides must be non-negative");
    const bool some = rows > 0 && cols > 0;
    check_pointer(some, input, "input");
    check_pointer(some, codes, "codes");
    check_pointer(some, exponents, "exponents");
    check_launch(ckpt::pack(dtype == MSDA_DTYPE_BFLOAT16, input, input_stride, rows, cols, codes, exponents,
                            static_cast<cudaStream_t>(stream)),
                 "msda_checkpoint_pack");
  });
}

int msda_checkpoint_unpack(msda_dtype_t dtype, const int8_t* codes, const uint8_t* exponents, int64_t rows,
                           int64_t cols, void* output, void* stream) {
  return guarded([&] {
    check_dtype(dtype);
    check_size(rows, "rows");
    check_size(cols, "cols");
    const bool some = rows > 0 && cols > 0;
    check_pointer(some, output, "output");
    check_pointer(some, codes, "codes");
    check_pointer(some, exponents, "exponents");
    check_launch(ckpt::unpack(dtype == MSDA_DTYPE_BFLOAT16, codes, exponents, rows, cols, output,
                              static_cast<cudaStream_t>(stream)),
                 "msda_checkpoint_unpack");
  });
}

int msda_linear_act_forward_workspace(const msda_linear_t* args, size_t* bytes) {
  return guarded([&] {
    require(bytes != nullptr, "bytes is null");
    *bytes = lin::forward_workspace(linear_args(args, false));
  });
}

int msda_linear_act_forward(const msda_linear_t* args, void* stream) {
  return guarded([&] {
    const lin::Args a = linear_args(args, false);
    check_workspace(a.workspace, a.workspace_bytes, lin::forward_workspace(a));
    check_launch(lin::forward(a, static_cast<cudaStream_t>(stream)), "msda_linear_act_forward");
  });
}

int msda_linear_act_backward_workspace(const msda_linear_t* args, size_t* bytes) {
  return guarded([&] {
    require(bytes != nullptr, "bytes is null");
    *bytes = lin::backward_workspace(linear_args(args, true));
  });
}

int msda_linear_act_backward(const msda_linear_t* args, void* stream) {
  return guarded([&] {
    const lin::Args a = linear_args(args, true);
    check_workspace(a.workspace, a.workspace_bytes, lin::backward_workspace(a));
    check_launch(lin::backward(a, static_cast<cudaStream_t>(stream)), "msda_linear_act_backward");
  });
}

int msda_layer_wait_timeouts(unsigned int* count) {
  return guarded([&] {
    require(count != nullptr, "count is null");
    unsigned int linear = 0, norm = 0;
    check_launch(lin::wait_timeouts(&linear), "msda_layer_wait_timeouts");
    check_launch(lnorm::wait_timeouts(&norm), "msda_layer_wait_timeouts");
    *count = linear + norm;
  });
}

int msda_layer_wait_probe(int64_t clocks, void* stream) {
  return guarded([&] {
    require(clocks >= 0 && clocks <= 2000000000, "clocks must be between 0 and 2000000000");
    check_launch(lnorm::wait_probe(clocks, static_cast<cudaStream_t>(stream)), "msda_layer_wait_probe");
  });
}

int msda_layer_norm_forward(const msda_layer_norm_t* args, void* stream) {
  return guarded([&] {
    check_launch(lnorm::forward(norm_args(args, false), static_cast<cudaStream_t>(stream)),
                 "msda_layer_norm_forward");
  });
}

int msda_layer_norm_backward_workspace(const msda_layer_norm_t* args, size_t* bytes) {
  return guarded([&] {
    require(bytes != nullptr, "bytes is null");
    (void)norm_args(args, true);
    *bytes = norm_workspace(*args);
  });
}

int msda_layer_norm_backward(const msda_layer_norm_t* args, void* stream) {
  return guarded([&] {
    const lnorm::Args a = norm_args(args, true);
    check_workspace(args->workspace, args->workspace_bytes, norm_workspace(*args));
    check_launch(lnorm::backward(a, static_cast<cudaStream_t>(stream)), "msda_layer_norm_backward");
  });
}

}  // extern "C"
