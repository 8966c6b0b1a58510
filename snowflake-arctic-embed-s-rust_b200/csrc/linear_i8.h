// Host interface of the general int8 product with token and channel scales (linear_i8.cu) and of the
// query / key norm with rotation (qk_rope.cu).
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <cstdint>

namespace ae {

// Element types of float operands and results (AE_F32, AE_F16, AE_BF16 of the C ABI).
enum FloatType : int { FT_F32 = 0, FT_F16 = 1, FT_BF16 = 2 };
inline size_t float_type_bytes(int t) { return t == FT_F32 ? 4 : 2; }

// out[m, n] = fma(float(sum_k a[m, k] w[n, k]), a_scale[m] * w_scale[n], bias[n])
struct ProductArgs {
  int M, N, K;
  const int8_t* a;        // [M, K], row pitch lda bytes
  size_t lda;
  const float* a_scale;   // [M]
  const int8_t* w;        // [N, K], row pitch ldw bytes
  size_t ldw;
  const float* w_scale;   // [N]
  const float* bias;      // [N] or nullptr
  void* out;              // [M, N] of out_type, row pitch ldo elements
  size_t ldo;
  int out_type;
  int* err;               // device error word
};

// q[m, k] = round_half_even(y * (127 / top)), scale[m] = top / 127 with y = x * inv_smooth, top = max_k |y|
struct QuantArgs {
  int M, K;
  const void* x;            // [M, K] of x_type, row pitch ldx elements
  size_t ldx;
  int x_type;
  const float* inv_smooth;  // [K] or nullptr
  int8_t* q;                // [M, K], row pitch ldq bytes (a multiple of 16, q 16-byte aligned)
  size_t ldq;
  float* scale;             // [M]
};

int launch_quant_rows(const QuantArgs& a, cudaStream_t st);
// Scratch (256-byte aligned) for the operands whose rows TMA cannot read where they are.
size_t product_scratch(const ProductArgs& a);
// tokens_ahead: the kernel launched right before on st is this call's launch_quant_rows, so all work ahead of
// that one (whatever wrote the weights) is done once the product starts. *kernels += the launches made.
int launch_product_i8(const ProductArgs& a, uint8_t* scratch, int tokens_ahead, cudaStream_t st, int* kernels);

// The product from float activations in one kernel; 1 where it is not for these sizes (nothing is launched then).
int launch_product_fused(const ProductArgs& a, const QuantArgs& q, cudaStream_t st);

struct QkArgs {
  int tokens, heads[2], dim, rotary;  // heads[0] queries, heads[1] keys
  int type;
  int neighbours;                     // pairs (2i, 2i + 1) instead of (i, i + rotary / 2)
  int norm;                           // 0: rotation only
  const void* x[2];                   // element (t, h, i) at t * x_ts + h * x_hs + i
  size_t x_ts[2], x_hs[2];
  void* y[2];
  size_t y_ts[2], y_hs[2];
  const float* weight[2];             // [dim] or nullptr (ones)
  float eps;
  const float* table;                 // [table_rows, rotary]: rotary / 2 cosines, then as many sines
  int table_rows;
  const int32_t* positions;           // [tokens], or nullptr: counted from cu
  const uint32_t* cu;                 // [n_seqs + 1]
  int n_seqs;
  int* err;
};
int launch_qk_norm_rope(const QkArgs& a, cudaStream_t st);

}  // namespace ae
