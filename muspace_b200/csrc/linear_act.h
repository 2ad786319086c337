// Host-side interface of the fused linear kernels: linear_gemm.cu (tensor-core
// product), linear_prep.cu (operand layouts) and linear_act.cu (the operator).
//
//   forward   z = x W^T + b,  y = act(z) + r
//   backward  dz = g * act'(z),  dx = dz W,  dW = dz^T x,  db = sum over rows of dz
//
// x [rows, in], W [out, in], y / r / g [rows, out]; rows may be apart
// (a row stride in elements), elements of a row are adjacent.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace lin {

enum class DType : int { kF32 = 0, kBF16 = 1 };
enum class Act : int { kNone = 0, kRelu = 1, kGelu = 2, kSilu = 3 };

// ---- the operator (linear_act.cu) -------------------------------------------------

struct Args {
  DType dtype;
  Act act;
  int64_t rows, in, out;
  int64_t x_stride, w_stride, r_stride, y_stride, g_stride;
  const void* x;        // forward; backward without codes
  const void* w;
  const void* bias;     // may be null
  const void* r;        // forward, may be null
  void* y;              // forward
  void* slope;          // act'(z), [rows, out] contiguous: float16 beside bfloat16, float32 beside float32; may be null
  const void* g;        // backward
  void* dx;             // [rows, in] contiguous, may be null
  void* dw;             // [out, in] contiguous, may be null
  void* db;             // [out], may be null
  const int8_t* codes;  // backward from an 8-bit checkpoint of x: [rows, in] contiguous
  const uint8_t* exps;  // [rows, ceil(in / 32)]
  void* workspace;
  size_t workspace_bytes;
};

// Bytes of workspace that forward / backward need for these arguments (the
// pointers' alignment counts, their contents do not); 0 for many calls.
size_t forward_workspace(const Args& a);
size_t backward_workspace(const Args& a);
cudaError_t forward(const Args& a, cudaStream_t stream);
cudaError_t backward(const Args& a, cudaStream_t stream);

// ---- operands of the product -------------------------------------------------------

// A matrix [rows, cols] of bfloat16 as the tensor map sees it: base and row
// stride on 16-byte boundaries. A float32 matrix is held as three planes whose
// sum it is (hi + mid + lo, each the bfloat16 nearest to what is left), one
// plane after another.
struct Operand {
  const __nv_bfloat16* p = nullptr;
  int64_t rows = 0, cols = 0, ld = 0, plane = 0;  // ld, plane: elements
  int planes = 1;
};

// What happens to the product's elements on their way out.
struct Epilogue {
  enum Mode : int {
    kStore = 0,  // out = v
    kFwd = 1,    // z = v + bias; out = act(z) + extra; slope = act'(z)
    kDz = 2,     // z = v + bias; out = extra * act'(z)
  };
  Mode mode = kStore;
  Act act = Act::kNone;
  const void* bias = nullptr;   // [n]
  const void* extra = nullptr;  // residual (kFwd) or gradient of the output (kDz)
  int64_t extra_ld = 0;
  void* out = nullptr;
  int64_t out_ld = 0;
  void* slope = nullptr;  // kFwd, [m, n] contiguous
  int64_t out_plane = 0;  // kDz, float32: out is three bfloat16 planes, out_plane elements apart
  float* sums = nullptr;  // kDz, may be null: [ceil(m / 32), n], the columns' sums over 32 rows
  float* unrounded = nullptr;  // finished apart with sums: where out is left in float32 for them, rows of partial_ld(n)
};

// ---- the product (linear_gemm.cu) --------------------------------------------------

// D[m, n] = sum_k A(m, k) B(n, k). An operand is stored [m or n, k], or, if
// `*_mn`, [k, m or n].
struct Product {
  Operand a, b;
  bool a_mn = false, b_mn = false;
  int64_t m = 0, n = 0, k = 0;
  DType dtype = DType::kBF16;  // of bias, extra, out
  Epilogue epi;
  float* partial = nullptr;  // where finished apart: [splits, m, partial_ld(n)]
};

struct Plan {
  int bn;        // columns of a tile
  int pair;      // 1: a tile of 128 rows on one SM; 2: 256 rows on two SMs
  int splits;    // ranges of k whose partial sums are added in a second kernel
  int kblocks;   // k blocks of 64 in one range
};

Plan plan_product(DType dtype, int64_t m, int64_t n, int64_t k, int pairs_of_planes, int sms);
// Whether the product leaves float32 sums that a second kernel adds up and
// finishes: ranges of k, outputs that TMA cannot address (rows off 16-byte
// boundaries), and empty sums.
bool finished_apart(const Product& pr, const Plan& p);
// Floats from one row of the sums to the next: they are read in whole eights, the last of a row too.
__host__ __device__ inline int64_t partial_ld(int64_t n) { return (n + 7) / 8 * 8; }
inline size_t partial_bytes(const Plan& p, int64_t m, int64_t n) {
  return static_cast<size_t>(p.splits) * m * partial_ld(n) * sizeof(float);
}
cudaError_t launch_product(const Product& pr, const Plan& plan, cudaStream_t stream);
cudaError_t wait_timeouts(unsigned int* count);

// ---- operand layouts and column sums (linear_prep.cu) ------------------------------

// dst planes (1 or 3) of src [rows, cols]; elements of dst beyond cols are not written.
cudaError_t copy_operand(DType dtype, const void* src, int64_t src_ld, const Operand& dst, cudaStream_t stream);
// dst = g * slope
cudaError_t scale_operand(DType dtype, const void* g, int64_t g_ld, const void* slope, const Operand& dst,
                          cudaStream_t stream);
// Either of them (slope null: the copy), with the sums of dst's columns over
// ranges of rows on the way: parts [column_parts(rows, cols), cols].
cudaError_t operand_and_sums(DType dtype, const void* g, int64_t g_ld, const void* slope, const Operand& dst,
                             float* parts, cudaStream_t stream);
cudaError_t unpack_operand(const int8_t* codes, const uint8_t* exps, const Operand& dst, cudaStream_t stream);
// The sums of src's columns over ranges of rows; and of parts [count, cols], in order.
int column_parts(int64_t rows, int64_t cols);
cudaError_t column_sums(const Operand& src, float* parts, cudaStream_t stream);
cudaError_t add_parts(DType out_dtype, const float* parts, int64_t count, int64_t cols, void* sums,
                      cudaStream_t stream);

// ---- few rows (linear_gemv.cu) -----------------------------------------------------

bool few_rows(const Args& a);
cudaError_t forward_few_rows(const Args& a, cudaStream_t stream);

}  // namespace lin
