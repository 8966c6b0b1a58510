// Per-token quantization of float activations, the int8 operand of the general product (product_i8.cu):
//
//   y = x * inv_smooth;  top = max_k |y|;  a = round_half_even(y * (127 / top));  a_scale = top / 127
#include "linear_i8.h"

#include <algorithm>

#include "floatio.cuh"
#include "gemm_i8.h"
#include "kernels.h"
#include "ptx.cuh"
#include "rowquant.cuh"

namespace ae {

// Threads an SM that the grid is sized for. Where the registers leave room for fewer (k_quant_rows<bfloat16, 128, 4>: 512),
// the other half of the blocks follows as a second wave; a grid of what fits takes as long within 1 % where rows are
// long (16,384 x 4,096 bfloat16 and 128 channels: 47.0 us, 46.8 this way) and 3 to 10 % less where they are short (8,192 x
// 2,048: 17.1 and 16.0 us in two runs, 19.0 and 17.1 this way).
constexpr int kQuantThreads = 1024;

// ------------------------------------------------------------------------------- row quantization
// max(|a|, |b|) with some sign; a NaN stays one.
__device__ __forceinline__ float max_abs(float a, float b) {
  float r;
  asm("max.NaN.xorsign.abs.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// A 16-byte piece of a row from element k on, zeros past the row's end.
template <class T>
__device__ __forceinline__ uint4 load_piece(const T* x, int k, int K, bool wide) {
  constexpr int VE = kPiece<T>;
  if (wide && k + VE <= K) return __ldcs(reinterpret_cast<const uint4*>(x + k));
  uint4 p = make_uint4(0, 0, 0, 0);
  uint32_t* w = &p.x;
#pragma unroll
  for (int e = 0; e < VE; ++e) {
    if (k + e < K) {
      if constexpr (sizeof(T) == 4) w[e] = reinterpret_cast<const uint32_t*>(x)[k + e];
      else w[e / 2] |= uint32_t(reinterpret_cast<const uint16_t*>(x)[k + e]) << (16 * (e & 1));
    }
  }
  return p;
}

template <class T>
__device__ __forceinline__ void load_smooth(const float* s, int k, int K, float (&v)[kPiece<T>]) {
  constexpr int VE = kPiece<T>;
  if (s && (reinterpret_cast<uintptr_t>(s) & 15) == 0 && k + VE <= K) {
#pragma unroll
    for (int e = 0; e < VE; e += 4) {
      const float4 f = *reinterpret_cast<const float4*>(s + k + e);
      v[e] = f.x, v[e + 1] = f.y, v[e + 2] = f.z, v[e + 3] = f.w;
    }
  } else {
#pragma unroll
    for (int e = 0; e < VE; ++e) v[e] = s && k + e < K ? s[k + e] : 1.0f;
  }
}

template <class T>
__device__ __forceinline__ void smoothed(uint4 piece, const float (&s)[kPiece<T>], float (&y)[kPiece<T>]) {
  widen<T>(piece, y);
#pragma unroll
  for (int e = 0; e < kPiece<T>; ++e) y[e] *= s[e];
}

template <class T>
__device__ __forceinline__ void store_quantized(int8_t* q, const RowScale& rs, const float (&y)[kPiece<T>]) {
  if constexpr (kPiece<T> == 8) *reinterpret_cast<uint2*>(q) = make_uint2(rs.four(y), rs.four(y + 4));
  else *reinterpret_cast<uint32_t*>(q) = rs.four(y);
}

// The largest |y| of a row's TPR threads, as bits; `turn` alternates, so that one barrier a row is enough.
template <int TPR>
__device__ __forceinline__ uint32_t row_top(float top, int turn) {
  uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(top) & 0x7fffffffu);
  if constexpr (TPR > 32) {
    __shared__ uint32_t s_top[2][TPR / 32];
    if ((threadIdx.x & 31) == 0) s_top[turn][threadIdx.x >> 5] = bits;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < TPR / 32; ++w) bits = max(bits, s_top[turn][w]);
  }
  return bits;
}

// TPR threads to a row, which is read once into registers, NV pieces a thread. A fixed number of blocks walks the rows, the
// smoothing factors in registers, the next row's pieces on their way while a row is reduced and quantized (16,384
// rows of 4,096 bfloat16, smoothed: 76 us with a block to a row and the factors loaded for each).
// The registers are held to four blocks of 128 an SM (16,384 rows of 4,096 bfloat16 and their product with 128 channels:
// 46.6 us, 51.5 with the compiler's own choice) and, where that spills nothing, two of 512 (17,316 rows of 5,056
// float: 101 us, 119 with one block).
template <class T, int TPR, int NV>
__global__ void __launch_bounds__(TPR < 128 ? 128 : TPR, TPR <= 128 ? 4 : (sizeof(T) == 4 || NV <= 2) ? 2 : 1)
    k_quant_rows(QuantArgs a) {
  constexpr int VE = kPiece<T>;
  constexpr int RPB = TPR < 128 ? 128 / TPR : 1;
  // in this order, so that what starts early behind this kernel finds all work ahead of it done
  pdl_wait();
  pdl_trigger();
  const int t = threadIdx.x % TPR;
  const bool wide = ((reinterpret_cast<uintptr_t>(a.x) | (a.ldx * sizeof(T))) & 15) == 0;
  float s[NV][VE];
#pragma unroll
  for (int i = 0; i < NV; ++i) load_smooth<T>(a.inv_smooth, (t + i * TPR) * VE, a.K, s[i]);
  int row = blockIdx.x * RPB + threadIdx.x / TPR;
  uint4 next[NV];
  auto fetch = [&](int r) {
    const T* x = static_cast<const T*>(a.x) + size_t(r) * a.ldx;
#pragma unroll
    for (int i = 0; i < NV; ++i) next[i] = load_piece(x, (t + i * TPR) * VE, r < a.M ? a.K : 0, wide);
  };
  fetch(row);
  // the same count of rounds in every warp of a block: the reductions meet
  for (int base = blockIdx.x * RPB, turn = 0; base < a.M; base += int(gridDim.x) * RPB, turn ^= 1) {
    uint4 piece[NV];
    float top = 0.0f, y[VE];
#pragma unroll
    for (int i = 0; i < NV; ++i) piece[i] = next[i];
    const int now = row;
    row += int(gridDim.x) * RPB;
    if (base + int(gridDim.x) * RPB < a.M) fetch(row);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      smoothed<T>(piece[i], s[i], y);
#pragma unroll
      for (int e = 0; e < VE; ++e) top = max_abs(top, y[e]);
    }
    const RowScale rs(row_top<TPR>(top, turn));
    if (now < a.M) {
      if (t == 0) a.scale[now] = rs.scale;
      int8_t* q = a.q + size_t(now) * a.ldq;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int k = (t + i * TPR) * VE;
        if (k < a.K) {
          smoothed<T>(piece[i], s[i], y);
          store_quantized<T>(q + k, rs, y);
        }
      }
    }
  }
}

// Rows longer than that: a block to a row, which is read twice, the second time from L2.
template <class T>
__global__ void __launch_bounds__(512) k_quant_long(QuantArgs a) {
  constexpr int VE = kPiece<T>;
  pdl_wait();
  pdl_trigger();
  const T* x = static_cast<const T*>(a.x) + size_t(blockIdx.x) * a.ldx;
  const bool wide = ((reinterpret_cast<uintptr_t>(a.x) | (a.ldx * sizeof(T))) & 15) == 0;
  float top = 0.0f, s[VE], y[VE];
  for (int k = threadIdx.x * VE; k < a.K; k += 512 * VE) {
    load_smooth<T>(a.inv_smooth, k, a.K, s);
    smoothed<T>(load_piece(x, k, a.K, wide), s, y);
#pragma unroll
    for (int e = 0; e < VE; ++e) top = max_abs(top, y[e]);
  }
  const RowScale rs(row_top<512>(top, 0));
  if (threadIdx.x == 0) a.scale[blockIdx.x] = rs.scale;
  int8_t* q = a.q + size_t(blockIdx.x) * a.ldq;
  for (int k = threadIdx.x * VE; k < a.K; k += 512 * VE) {
    load_smooth<T>(a.inv_smooth, k, a.K, s);
    smoothed<T>(load_piece(x, k, a.K, wide), s, y);
    store_quantized<T>(q + k, rs, y);
  }
}

template <class T, int TPR, int NV>
static cudaError_t quant(const QuantArgs& a, cudaStream_t st) {
  constexpr int RPB = TPR < 128 ? 128 / TPR : 1, threads = TPR < 128 ? 128 : TPR;
  const int blocks = std::min((a.M + RPB - 1) / RPB, num_sms() * (kQuantThreads / threads));
  return launch_pdl(k_quant_rows<T, TPR, NV>, dim3(blocks), dim3(threads), 0, st, a);
}

// A warp holds 4 pieces a thread (1,024 16-bit values), 128 threads 4,096, 512 threads 16,384.
template <class T>
static cudaError_t quant_type(const QuantArgs& a, cudaStream_t st) {
  const int pieces = (a.K + kPiece<T> - 1) / kPiece<T>;
  if (pieces <= 32) return quant<T, 32, 1>(a, st);
  if (pieces <= 32 * 2) return quant<T, 32, 2>(a, st);
  if (pieces <= 32 * 4) return quant<T, 32, 4>(a, st);
  if (pieces <= 128 * 2) return quant<T, 128, 2>(a, st);
  if (pieces <= 128 * 4) return quant<T, 128, 4>(a, st);
  if (pieces <= 512 * 2) return quant<T, 512, 2>(a, st);
  if (pieces <= 512 * 4) return quant<T, 512, 4>(a, st);
  return launch_pdl(k_quant_long<T>, dim3(a.M), dim3(512), 0, st, a);
}

int launch_quant_rows(const QuantArgs& a, cudaStream_t st) {
  const cudaError_t e = a.x_type == FT_F32   ? quant_type<float>(a, st)
                        : a.x_type == FT_F16 ? quant_type<__half>(a, st)
                                             : quant_type<__nv_bfloat16>(a, st);
  return e == cudaSuccess ? 0 : -100 - int(e);
}

}  // namespace ae
