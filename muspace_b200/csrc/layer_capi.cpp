// extern "C" boundary of the layer operators (declared in
// include/muspace_msda.h): linear_act, layer norm, 8-bit checkpoints, dropout, the
// norms with their residual and the gated product.
#include <cuda_runtime.h>

#include <limits>
#include <string>

#include "../../include/muspace_msda.h"
#include "capi_common.h"
#include "dropout.h"
#include "layer_norm.h"
#include "linear_act.h"
#include "residual_norm.h"

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

void check_wide_dtype(int dtype) {
  require(dtype == MSDA_DTYPE_FLOAT32 || dtype == MSDA_DTYPE_BFLOAT16 || dtype == MSDA_DTYPE_FLOAT16,
          "dtype must be float32, bfloat16 or float16");
}

drop::Rule rule_of(int64_t threshold, int64_t seed, int64_t sequence, const int64_t* seed_at) {
  require(threshold >= 0 && threshold <= 65536, "threshold must be between 0 and 65536");
  drop::Rule rule;
  rule.threshold = static_cast<uint32_t>(threshold);
  rule.scale = drop::scale_of(rule.threshold);
  rule.seed = static_cast<uint64_t>(seed);
  rule.sequence = static_cast<uint64_t>(sequence);
  rule.seed_at = threshold ? seed_at : nullptr;
  return rule;
}

resnorm::Args residual_norm_args(const msda_residual_norm_t* in, bool branch, bool backward) {
  require(in != nullptr, "args is null");
  check_wide_dtype(in->dtype);
  require(in->weight_dtype == in->dtype || in->weight_dtype == MSDA_DTYPE_FLOAT32, "weight_dtype must be dtype or float32");
  require(in->gate_dtype == in->dtype || in->gate_dtype == MSDA_DTYPE_FLOAT32, "gate_dtype must be dtype or float32");
  const int kind = in->kind & ~MSDA_NORM_KEEP;
  const bool keep = kind != in->kind;
  require(kind == MSDA_NORM_LAYER || kind == MSDA_NORM_RMS, "kind must be layer or rms");
  check_size(in->rows, "rows");
  check_size(in->cols, "cols");
  for (int64_t stride : {in->input_stride, in->residual_stride, in->gate_stride, in->sum_stride,
                         in->grad_output_stride, in->grad_sum_stride})
    require(stride >= 0, "strides must be non-negative");
  const bool some = in->rows > 0 && in->cols > 0, gated = in->gate || in->grad_gate;
  require(!keep || (!branch && !backward && (!some || (in->sum && in->rstd))),
          "MSDA_NORM_KEEP goes with add_norm's forward, sum and rstd");
  require(in->gate_groups >= 0, "sizes must be non-negative");
  require(!some || !gated || (in->gate_groups > 0 && in->rows % in->gate_groups == 0),
          "gate_groups must divide rows");
  resnorm::Args a{};
  a.dtype = static_cast<drop::DType>(in->dtype);
  a.weight_f32 = in->weight_dtype == MSDA_DTYPE_FLOAT32, a.gate_f32 = in->gate_dtype == MSDA_DTYPE_FLOAT32;
  a.branch = branch, a.rms = kind == MSDA_NORM_RMS, a.keep = keep;
  a.rows = in->rows, a.cols = in->cols;
  a.gate_groups = gated ? in->gate_groups : 1;
  a.gate_rows = a.gate_groups ? a.rows / a.gate_groups : 0;
  a.h_stride = in->input_stride, a.r_stride = in->residual_stride, a.gate_stride = in->gate_stride;
  a.gy_stride = in->grad_output_stride, a.gs_stride = in->grad_sum_stride, a.sum_stride = in->sum_stride;
  a.alpha = in->residual_scale, a.eps = in->eps;
  a.share = a.cols ? 1.f / static_cast<float>(a.cols) : 0.f;
  a.rule = rule_of(in->threshold, in->seed, in->sequence, in->seed_at);
  a.gate = in->gate, a.w = in->weight, a.b = in->bias;
  a.rstd = in->rstd;
  if (backward) {
    const bool normed = branch || in->grad_output;
    require(branch || !some || in->grad_output || in->grad_sum, "grad_output and grad_sum are null");
    require(normed || !some || (!in->grad_weight && !in->grad_bias), "grad_weight and grad_bias need grad_output");
    check_pointer(some && branch, in->grad_sum, "grad_sum");
    check_pointer(some && (branch || in->grad_gate), in->input, "input");
    check_pointer(some && !branch && normed, in->sum, "sum");
    check_pointer(some && normed, in->rstd, "rstd");
    check_pointer(some && normed && !a.rms, in->mean, "mean");
    a.mean = a.rms ? nullptr : in->mean;
    a.h = in->input;
    a.gs = in->grad_sum;
    if (!branch) a.gy = in->grad_output, a.sum = in->sum;
    a.dh = in->grad_input, a.dr = in->grad_residual;
    a.dw = in->grad_weight, a.db = in->grad_bias, a.dgate = in->grad_gate;
    a.parts = static_cast<float*>(in->workspace);
  } else {
    check_pointer(some, in->input, "input");
    check_pointer(some, in->residual, "residual");
    check_pointer(some, branch ? in->sum : in->output, branch ? "sum" : "output");
    a.mean = in->mean;
    a.h = in->input, a.r = in->residual;
    if (!branch) a.y = in->output;
    a.s = in->sum;
  }
  return a;
}

lin::GatedArgs gated_args(const msda_gated_linear_t* in, bool backward) {
  require(in != nullptr, "args is null");
  check_dtype(in->dtype);
  require(in->activation >= MSDA_ACTIVATION_NONE && in->activation <= MSDA_ACTIVATION_SILU,
          "activation must be none, relu, gelu or silu");
  check_size(in->rows, "rows");
  check_size(in->in_features, "in_features");
  check_size(in->out_features, "out_features");
  require(2 * in->out_features <= kMax, "out_features exceeds the supported range (< 2^30)");
  require(in->input_stride >= 0 && in->weight_stride >= 0 && in->output_stride >= 0 && in->grad_output_stride >= 0,
          "strides must be non-negative");
  const bool some_x = in->rows > 0 && in->in_features > 0, some_w = in->out_features > 0 && in->in_features > 0;
  const bool some_y = in->rows > 0 && in->out_features > 0;
  lin::GatedArgs a{};
  a.dtype = static_cast<lin::DType>(in->dtype);
  a.act = static_cast<lin::Act>(in->activation);
  a.rows = in->rows, a.in = in->in_features, a.out = in->out_features;
  a.x_stride = in->input_stride, a.w_stride = in->weight_stride;
  a.y_stride = in->output_stride, a.g_stride = in->grad_output_stride;
  a.factors = in->factors;
  a.exponents = in->dtype == MSDA_DTYPE_BFLOAT16 ? in->exponents : nullptr;
  check_pointer(some_y && in->factors && in->dtype == MSDA_DTYPE_BFLOAT16, in->exponents, "exponents");
  require((reinterpret_cast<uintptr_t>(a.exponents) & 3) == 0, "exponents must be 4-byte aligned");
  if (backward) {
    check_pointer(some_w && in->grad_input, in->weight, "weight");
    check_pointer(some_x && in->grad_weight, in->input, "input");
    check_pointer(some_y, in->grad_output, "grad_output");
    check_pointer(some_y, in->factors, "factors");
    a.g = in->grad_output;
    a.dx = in->grad_input, a.dw = in->grad_weight, a.db = in->grad_bias;
  } else {
    check_pointer(some_w, in->weight, "weight");
    check_pointer(some_x, in->input, "input");
    check_pointer(some_y, in->output, "output");
    require(in->rows <= 1 || in->output_stride >= in->out_features, "output rows must not overlap");
    a.rule = rule_of(in->threshold, in->seed, in->sequence, in->seed_at);
    a.bias = in->bias;
    a.y = in->output;
  }
  a.x = in->input, a.w = in->weight;
  a.workspace = in->workspace;
  a.workspace_bytes = in->workspace_bytes;
  return a;
}

int residual_norm_forward(const msda_residual_norm_t* args, bool branch, const char* name, void* stream) {
  return guarded([&] {
    check_launch(resnorm::forward(residual_norm_args(args, branch, false), static_cast<cudaStream_t>(stream)), name);
  });
}

size_t residual_norm_workspace(const resnorm::Args& a) {
  return static_cast<size_t>(resnorm::backward_parts(a)) * sizeof(float);
}

int residual_norm_workspace(const msda_residual_norm_t* args, bool branch, size_t* bytes) {
  return guarded([&] {
    require(bytes != nullptr, "bytes is null");
    *bytes = residual_norm_workspace(residual_norm_args(args, branch, true));
  });
}

int residual_norm_backward(const msda_residual_norm_t* args, bool branch, const char* name, void* stream) {
  return guarded([&] {
    const resnorm::Args a = residual_norm_args(args, branch, true);
    check_workspace(args->workspace, args->workspace_bytes, residual_norm_workspace(a));
    check_launch(resnorm::backward(a, static_cast<cudaStream_t>(stream)), name);
  });
}

}  // namespace

extern "C" {

int msda_dropout(msda_dtype_t dtype, const void* input, int64_t rows, int64_t cols, int64_t input_stride,
                 int64_t threshold, int64_t seed, int64_t sequence, const int64_t* seed_at, void* output,
                 void* stream) {
  return guarded([&] {
    check_wide_dtype(dtype);
    check_size(rows, "rows");
    check_size(cols, "cols");
    require(input_stride >= 0, "strides must be non-negative");
    const drop::Rule rule = rule_of(threshold, seed, sequence, seed_at);
    const bool some = rows > 0 && cols > 0;
    check_pointer(some, input, "input");
    check_pointer(some, output, "output");
    check_launch(drop::dropout(static_cast<drop::DType>(dtype), input, input_stride, rows, cols, rule, output,
                               static_cast<cudaStream_t>(stream)),
                 "msda_dropout");
  });
}

int msda_gated_linear_forward_workspace(const msda_gated_linear_t* args, size_t* bytes) {
  return guarded([&] {
    require(bytes != nullptr, "bytes is null");
    *bytes = lin::gated_forward_workspace(gated_args(args, false));
  });
}

int msda_gated_linear_forward(const msda_gated_linear_t* args, void* stream) {
  return guarded([&] {
    const lin::GatedArgs a = gated_args(args, false);
    check_workspace(a.workspace, a.workspace_bytes, lin::gated_forward_workspace(a));
    check_launch(lin::gated_forward(a, static_cast<cudaStream_t>(stream)), "msda_gated_linear_forward");
  });
}

int msda_gated_linear_backward_workspace(const msda_gated_linear_t* args, size_t* bytes) {
  return guarded([&] {
    require(bytes != nullptr, "bytes is null");
    *bytes = lin::gated_backward_workspace(gated_args(args, true));
  });
}

int msda_gated_linear_backward(const msda_gated_linear_t* args, void* stream) {
  return guarded([&] {
    const lin::GatedArgs a = gated_args(args, true);
    check_workspace(a.workspace, a.workspace_bytes, lin::gated_backward_workspace(a));
    check_launch(lin::gated_backward(a, static_cast<cudaStream_t>(stream)), "msda_gated_linear_backward");
  });
}

int msda_add_norm_forward(const msda_residual_norm_t* args, void* stream) {
  return residual_norm_forward(args, false, "msda_add_norm_forward", stream);
}

int msda_add_norm_backward_workspace(const msda_residual_norm_t* args, size_t* bytes) {
  return residual_norm_workspace(args, false, bytes);
}

int msda_add_norm_backward(const msda_residual_norm_t* args, void* stream) {
  return residual_norm_backward(args, false, "msda_add_norm_backward", stream);
}

int msda_norm_add_forward(const msda_residual_norm_t* args, void* stream) {
  return residual_norm_forward(args, true, "msda_norm_add_forward", stream);
}

int msda_norm_add_backward_workspace(const msda_residual_norm_t* args, size_t* bytes) {
  return residual_norm_workspace(args, true, bytes);
}

int msda_norm_add_backward(const msda_residual_norm_t* args, void* stream) {
  return residual_norm_backward(args, true, "msda_norm_add_backward", stream);
}

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
    unsigned int linear = 0, gated = 0, norm = 0;
    check_launch(lin::wait_timeouts(&linear), "msda_layer_wait_timeouts");
    check_launch(lin::gated_wait_timeouts(&gated), "msda_layer_wait_timeouts");
    check_launch(lnorm::wait_timeouts(&norm), "msda_layer_wait_timeouts");
    *count = linear + gated + norm;
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
