// The fused linear operators: lay their operands out where that is needed and
// string the products of linear_gemm.cu and linear_gated.cu together.
//
// float32 runs on the same bfloat16 tensor-core product: every operand is
// split into three bfloat16 planes (24 bits), and the six products of planes
// that matter at 2^-24 are added up.
//
// Backward: dz = g * act'(z) is one operand of two products (dx = dz W,
// dW = dz^T x). In bfloat16 it is rounded to bfloat16 for them, as the tensor core
// takes it in one product (two planes would double both): with the output's own
// rounding the gradients are off by 0.0024 of their size, by 0.0017 without (40000
// x 256 x 512). db is added up before that rounding. Where the forward kept the
// slope act'(z), dz is one elementwise pass; where it kept nothing (a checkpoint of
// x in 8 bits), z is computed again and dz leaves that product's epilogue.
//
// The gated operator's backward is the same with dz = [g P, g Q], whose factors the
// forward kept: one elementwise pass, then products over all 2 n rows of the weight.
// In bfloat16 the factors are kept in float16, eight under one exponent: 11 bits down to
// 2^-28 of the largest, where bfloat16's 8 added as much to the gradients' error as dz's rounding does
// (40000 x 256 x 512: 0.0029 of their size instead of 0.0024).
#include <algorithm>

#include "checkpoint8.cuh"
#include "linear_act.h"

namespace lin {
namespace {

// Hands out the workspace piece by piece; without a base it only measures, and
// the calls that would launch are skipped.
struct Arena {
  char* base = nullptr;
  size_t used = 0, size = 0;
  bool measuring = true;
  void* take(size_t bytes) {
    const size_t at = used;
    used += (bytes + 255) & ~static_cast<size_t>(255);
    return measuring ? nullptr : base + at;
  }
};

#define LIN_TRY(call)                              \
  do {                                             \
    const cudaError_t lin_err = (call);            \
    if (lin_err != cudaSuccess) return lin_err;    \
  } while (0)

inline int64_t padded(int64_t n) { return (n + 7) / 8 * 8; }

// Room for the planes of a [rows, cols] operand.
Operand fresh(DType dtype, int64_t rows, int64_t cols, int planes, Arena& arena) {
  Operand o;
  o.rows = rows, o.cols = cols, o.ld = padded(cols), o.planes = planes;
  o.plane = rows * o.ld;
  o.p = static_cast<const __nv_bfloat16*>(arena.take(static_cast<size_t>(planes) * o.plane * 2));
  return o;
}

bool direct(DType dtype, const void* p, int64_t cols, int64_t ld) {
  return dtype == DType::kBF16 && (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld % 8 == 0 && ld >= cols;
}

// A caller's matrix as an operand: as it stands, or laid out in the workspace.
cudaError_t operand_of(DType dtype, const void* p, int64_t rows, int64_t cols, int64_t ld, Arena& arena,
                       Operand* out, cudaStream_t stream) {
  if (direct(dtype, p, cols, ld)) {
    out->p = static_cast<const __nv_bfloat16*>(p);
    out->rows = rows, out->cols = cols, out->ld = ld;
    return cudaSuccess;
  }
  *out = fresh(dtype, rows, cols, dtype == DType::kF32 ? 3 : 1, arena);
  return arena.measuring ? cudaSuccess : copy_operand(dtype, p, ld, *out, stream);
}

int multiprocessors() {
  static const int count = [] {
    int device = 0, n = 148;
    if (cudaGetDevice(&device) == cudaSuccess) cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device);
    return n;
  }();
  return count;
}

int plane_pairs(const Operand& a, const Operand& b) {
  return a.planes == 3 ? (b.planes == 3 ? 6 : 3) : (b.planes == 3 ? 3 : 1);
}

cudaError_t run_product(Product& pr, Arena& arena, cudaStream_t stream) {
  const Plan plan = plan_product(pr.dtype, pr.m, pr.n, pr.k, plane_pairs(pr.a, pr.b), multiprocessors());
  if (finished_apart(pr, plan)) pr.partial = static_cast<float*>(arena.take(partial_bytes(plan, pr.m, pr.n)));
  return arena.measuring ? cudaSuccess : launch_product(pr, plan, stream);
}

cudaError_t forward_in(const Args& a, Arena& arena, cudaStream_t stream) {
  if (a.rows == 0 || a.out == 0) return cudaSuccess;
  if (few_rows(a)) return arena.measuring ? cudaSuccess : forward_few_rows(a, stream);
  Product pr;
  LIN_TRY(operand_of(a.dtype, a.x, a.rows, a.in, a.x_stride, arena, &pr.a, stream));
  LIN_TRY(operand_of(a.dtype, a.w, a.out, a.in, a.w_stride, arena, &pr.b, stream));
  pr.m = a.rows, pr.n = a.out, pr.k = a.in, pr.dtype = a.dtype;
  pr.epi.mode = Epilogue::kFwd;
  pr.epi.act = a.act;
  pr.epi.bias = a.bias;
  pr.epi.extra = a.r;
  pr.epi.extra_ld = a.r_stride;
  pr.epi.out = a.y;
  pr.epi.out_ld = a.y_stride;
  pr.epi.slope = a.slope;
  return run_product(pr, arena, stream);
}

// dx = dz W and dW = dz^T x, each where it is asked for.
cudaError_t products_of(DType dtype, int64_t rows, int64_t in, int64_t out, const Operand& dz, const Operand& w,
                        const Operand& x, void* dx, void* dw, Arena& arena, cudaStream_t stream) {
  if (dx && rows && in) {
    Product pr;
    pr.a = dz, pr.b = w, pr.b_mn = true;
    pr.m = rows, pr.n = in, pr.k = out, pr.dtype = dtype;
    pr.epi.out = dx;
    pr.epi.out_ld = in;
    LIN_TRY(run_product(pr, arena, stream));
  }
  if (dw && out && in) {
    Product pr;
    pr.a = dz, pr.a_mn = true;
    pr.b = x, pr.b_mn = true;
    pr.m = out, pr.n = in, pr.k = rows, pr.dtype = dtype;
    pr.epi.out = dw;
    pr.epi.out_ld = in;
    LIN_TRY(run_product(pr, arena, stream));
  }
  return cudaSuccess;
}

cudaError_t backward_in(const Args& a, Arena& arena, cudaStream_t stream) {
  const bool f32 = a.dtype == DType::kF32;
  const bool recompute = a.act != Act::kNone && a.slope == nullptr;
  const bool need_w = a.dx != nullptr || recompute, need_x = a.dw != nullptr || recompute;
  Operand x, w, dz;
  if (need_w) LIN_TRY(operand_of(a.dtype, a.w, a.out, a.in, a.w_stride, arena, &w, stream));
  if (need_x) {
    if (a.codes) {
      x = fresh(a.dtype, a.rows, a.in, 1, arena);  // 7 bits and a power of two: one plane holds a code exactly
      if (!arena.measuring) LIN_TRY(unpack_operand(a.codes, a.exps, x, stream));
    } else {
      LIN_TRY(operand_of(a.dtype, a.x, a.rows, a.in, a.x_stride, arena, &x, stream));
    }
  }
  // db: the columns' sums come from whatever makes dz, over ranges of rows
  const bool need_b = a.db != nullptr && a.out > 0;
  const bool as_it_is = a.act == Act::kNone && direct(a.dtype, a.g, a.out, a.g_stride);
  const int64_t parts_count = a.rows == 0 ? 0 : recompute ? (a.rows + 31) / 32 : column_parts(a.rows, a.out);
  float* parts = nullptr;
  if (need_b) parts = static_cast<float*>(arena.take(static_cast<size_t>(parts_count) * a.out * sizeof(float)));
  if (as_it_is) {
    LIN_TRY(operand_of(a.dtype, a.g, a.rows, a.out, a.g_stride, arena, &dz, stream));
    if (need_b && !arena.measuring) LIN_TRY(column_sums(dz, parts, stream));
  } else {
    dz = fresh(a.dtype, a.rows, a.out, f32 ? 3 : 1, arena);
    if (recompute) {
      Product pr;
      pr.a = x, pr.b = w;
      pr.m = a.rows, pr.n = a.out, pr.k = a.in, pr.dtype = a.dtype;
      pr.epi.mode = Epilogue::kDz;
      pr.epi.act = a.act;
      pr.epi.bias = a.bias;
      pr.epi.extra = a.g;
      pr.epi.extra_ld = a.g_stride;
      pr.epi.out = const_cast<__nv_bfloat16*>(dz.p);
      pr.epi.out_ld = dz.ld;
      pr.epi.out_plane = f32 ? dz.plane : 0;
      pr.epi.sums = parts;
      if (a.rows && a.out) LIN_TRY(run_product(pr, arena, stream));
    } else if (!arena.measuring) {
      const void* slope = a.act == Act::kNone ? nullptr : a.slope;
      if (need_b)
        LIN_TRY(operand_and_sums(a.dtype, a.g, a.g_stride, slope, dz, parts, stream));
      else if (slope)
        LIN_TRY(scale_operand(a.dtype, a.g, a.g_stride, slope, dz, stream));
      else
        LIN_TRY(copy_operand(a.dtype, a.g, a.g_stride, dz, stream));
    }
  }
  if (need_b && !arena.measuring) LIN_TRY(add_parts(a.dtype, parts, parts_count, a.out, a.db, stream));
  return products_of(a.dtype, a.rows, a.in, a.out, dz, w, x, a.dx, a.dw, arena, stream);
}

cudaError_t gated_forward_in(const GatedArgs& a, Arena& arena, cudaStream_t stream) {
  if (a.rows == 0 || a.out == 0) return cudaSuccess;
  if (gated_few_rows(a)) return arena.measuring ? cudaSuccess : gated_forward_few_rows(a, stream);
  Product pr;
  LIN_TRY(operand_of(a.dtype, a.x, a.rows, a.in, a.x_stride, arena, &pr.a, stream));
  LIN_TRY(operand_of(a.dtype, a.w, 2 * a.out, a.in, a.w_stride, arena, &pr.b, stream));
  pr.m = a.rows, pr.n = a.out, pr.k = a.in, pr.dtype = a.dtype;
  pr.epi.act = a.act;
  pr.epi.bias = a.bias;
  pr.epi.out = a.y;
  pr.epi.out_ld = a.y_stride;
  pr.epi.slope = a.factors;
  pr.epi.exponents = a.exponents;
  pr.epi.rule = a.rule;
  const Plan plan = plan_product(pr.dtype, pr.m, 2 * pr.n, pr.k, plane_pairs(pr.a, pr.b), multiprocessors());
  if (gated_apart(pr, plan)) pr.partial = static_cast<float*>(arena.take(partial_bytes(plan, pr.m, 2 * pr.n)));
  return arena.measuring ? cudaSuccess : launch_gated(pr, plan, stream);
}

cudaError_t gated_backward_in(const GatedArgs& a, Arena& arena, cudaStream_t stream) {
  const int64_t both = 2 * a.out;
  Operand x, w, dz;
  if (a.dx) LIN_TRY(operand_of(a.dtype, a.w, both, a.in, a.w_stride, arena, &w, stream));
  if (a.dw) LIN_TRY(operand_of(a.dtype, a.x, a.rows, a.in, a.x_stride, arena, &x, stream));
  const bool need_b = a.db != nullptr && a.out > 0;
  const int64_t parts_count = a.rows == 0 ? 0 : column_parts(a.rows, a.out);
  float* parts = nullptr;
  if (need_b) parts = static_cast<float*>(arena.take(static_cast<size_t>(parts_count) * both * sizeof(float)));
  dz = fresh(a.dtype, a.rows, both, a.dtype == DType::kF32 ? 3 : 1, arena);
  if (!arena.measuring) {
    LIN_TRY(gate_operand(a.dtype, a.g, a.g_stride, a.factors, a.exponents, dz, parts, stream));
    if (need_b) LIN_TRY(add_parts(a.dtype, parts, parts_count, both, a.db, stream));
  }
  return products_of(a.dtype, a.rows, a.in, both, dz, w, x, a.dx, a.dw, arena, stream);
}

Arena arena_of(void* workspace, size_t bytes) {
  Arena arena;
  arena.base = static_cast<char*>(workspace);
  arena.size = bytes;
  arena.measuring = false;
  return arena;
}

}  // namespace

size_t forward_workspace(const Args& a) {
  Arena arena;
  (void)forward_in(a, arena, nullptr);
  return arena.used;
}

size_t backward_workspace(const Args& a) {
  Arena arena;
  (void)backward_in(a, arena, nullptr);
  return arena.used;
}

cudaError_t forward(const Args& a, cudaStream_t stream) {
  Arena arena = arena_of(a.workspace, a.workspace_bytes);
  return forward_in(a, arena, stream);
}

cudaError_t backward(const Args& a, cudaStream_t stream) {
  Arena arena = arena_of(a.workspace, a.workspace_bytes);
  return backward_in(a, arena, stream);
}

size_t gated_forward_workspace(const GatedArgs& a) {
  Arena arena;
  (void)gated_forward_in(a, arena, nullptr);
  return arena.used;
}

size_t gated_backward_workspace(const GatedArgs& a) {
  Arena arena;
  (void)gated_backward_in(a, arena, nullptr);
  return arena.used;
}

cudaError_t gated_forward(const GatedArgs& a, cudaStream_t stream) {
  Arena arena = arena_of(a.workspace, a.workspace_bytes);
  return gated_forward_in(a, arena, stream);
}

cudaError_t gated_backward(const GatedArgs& a, cudaStream_t stream) {
  Arena arena = arena_of(a.workspace, a.workspace_bytes);
  return gated_backward_in(a, arena, stream);
}

}  // namespace lin
