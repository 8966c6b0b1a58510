// Per-token quantization of float activations, the int8 operand of the general product (product_i8.cu):
//
//   y = x * inv_smooth;  top = max_k |y|;  a = round_half_even(y * (127 / top));  a_scale = top / 127
#include "linear_i8.h"

#include "floatio.cuh"
#include "kernels.h"
#include "ptx.cuh"
#include "rowquant.cuh"

namespace ae {

// ------------------------------------------------------------------------------- row quantization
// TPR threads to a row. The row is read once into registers (NV 16-byte pieces a thread), or, when it is
// longer than that (NV = 0), twice, the second time from L2.
template <class T, int TPR, int NV>
__global__ void __launch_bounds__(TPR < 128 ? 128 : TPR) k_quant_rows(QuantArgs a) {
  constexpr int VE = kPiece<T>;
  constexpr int RPB = TPR < 128 ? 128 / TPR : 1;
  // in this order, so that what starts early behind this kernel finds all work ahead of it done
  pdl_wait();
  pdl_trigger();
  const int row = blockIdx.x * RPB + threadIdx.x / TPR;
  const int t = threadIdx.x % TPR;
  const bool live = row < a.M;
  const T* x = static_cast<const T*>(a.x) + (live ? size_t(row) * a.ldx : 0);
  const bool wide = ((reinterpret_cast<uintptr_t>(a.x) | (a.ldx * sizeof(T))) & 15) == 0;
  const int pieces = (a.K + VE - 1) / VE;

  auto load = [&](int p, float (&v)[VE]) {
    const int k = p * VE;
    if (wide && k + VE <= a.K) {
      widen<T>(*reinterpret_cast<const uint4*>(x + k), v);
    } else {
#pragma unroll
      for (int e = 0; e < VE; ++e) v[e] = k + e < a.K ? to_f32(x[k + e]) : 0.0f;
    }
    if (a.inv_smooth) {
#pragma unroll
      for (int e = 0; e < VE; ++e)
        if (k + e < a.K) v[e] *= a.inv_smooth[k + e];
    }
  };
  // |y| compared by its bits: the order is the same, and a NaN is above every number
  uint32_t top = 0;
  auto take = [&](const float (&v)[VE]) {
#pragma unroll
    for (int e = 0; e < VE; ++e) top = max(top, __float_as_uint(v[e]) & 0x7fffffffu);
  };
  float keep[NV > 0 ? NV : 1][VE];
  if (live) {
    if constexpr (NV > 0) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (t + i * TPR < pieces) {
          load(t + i * TPR, keep[i]);
          take(keep[i]);
        }
    } else {
      for (int p = t; p < pieces; p += TPR) {
        load(p, keep[0]);
        take(keep[0]);
      }
    }
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if constexpr (TPR > 32) {
    __shared__ uint32_t s_top[TPR / 32];
    if ((threadIdx.x & 31) == 0) s_top[threadIdx.x >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < TPR / 32; ++w) top = max(top, s_top[w]);
  }
  if (!live) return;
  const RowScale rs(top);
  if (t == 0) a.scale[row] = rs.scale;
  int8_t* q = a.q + size_t(row) * a.ldq;
  auto store = [&](int p, const float (&v)[VE]) {
    uint32_t w[VE / 4];
#pragma unroll
    for (int j = 0; j < VE / 4; ++j) w[j] = rs.four(v + 4 * j);
    if constexpr (VE == 8)
      *reinterpret_cast<uint2*>(q + p * VE) = make_uint2(w[0], w[1]);
    else
      *reinterpret_cast<uint32_t*>(q + p * VE) = w[0];
  };
  if constexpr (NV > 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (t + i * TPR < pieces) store(t + i * TPR, keep[i]);
  } else {
    for (int p = t; p < pieces; p += TPR) {
      load(p, keep[0]);
      store(p, keep[0]);
    }
  }
}

template <class T, int TPR, int NV>
static cudaError_t quant(const QuantArgs& a, cudaStream_t st) {
  constexpr int RPB = TPR < 128 ? 128 / TPR : 1;
  return launch_pdl(k_quant_rows<T, TPR, NV>, dim3((a.M + RPB - 1) / RPB), dim3(TPR < 128 ? 128 : TPR), 0, st, a);
}

// A warp holds 4 pieces a thread (1,024 16-bit values), 128 threads 4,096, 512 threads 16,384.
template <class T>
static cudaError_t quant_type(const QuantArgs& a, cudaStream_t st) {
  const int pieces = (a.K + kPiece<T> - 1) / kPiece<T>;
  if (pieces <= 32 * 4) return quant<T, 32, 4>(a, st);
  if (pieces <= 128 * 4) return quant<T, 128, 4>(a, st);
  if (pieces <= 512 * 4) return quant<T, 512, 4>(a, st);
  return quant<T, 512, 0>(a, st);
}

int launch_quant_rows(const QuantArgs& a, cudaStream_t st) {
  const cudaError_t e = a.x_type == FT_F32   ? quant_type<float>(a, st)
                        : a.x_type == FT_F16 ? quant_type<__half>(a, st)
                                             : quant_type<__nv_bfloat16>(a, st);
  return e == cudaSuccess ? 0 : -100 - int(e);
}

}  // namespace ae
