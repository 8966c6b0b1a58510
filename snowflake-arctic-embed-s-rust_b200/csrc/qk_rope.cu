// RMS norm of every query and key head and the rotation of its first `rotary` dims by the token's
// position, in one pass over the heads:
//
//   y = x / sqrt(mean(x^2) + eps) * weight;  (y_i, y_j) -> (y_i c - y_j s, y_j c + y_i s)
//
// for the pairs (i, i + rotary / 2) or (2i, 2i + 1), with c and s from a float table row of the position.
// All of it in float; one rounding to the heads' type.
#include "floatio.cuh"
#include "linear_i8.h"
#include "ptx.cuh"

namespace ae {

constexpr int kQkMaxDim = 512;

// Position of token t: given, or counted from the start of its sequence (cu[s] <= t < cu[s + 1]); -1 if
// there is none inside the table.
__device__ __forceinline__ int qk_position(const QkArgs& a, int t) {
  int p;
  if (a.positions) {
    p = a.positions[t];
  } else {
    int lo = 0, hi = a.n_seqs;  // the last s with cu[s] <= t, among 0 .. n_seqs
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (a.cu[mid] <= uint32_t(t)) lo = mid;
      else hi = mid - 1;
    }
    p = lo < a.n_seqs && a.cu[lo] <= uint32_t(t) ? t - int(a.cu[lo]) : -1;
  }
  return p >= 0 && p < a.table_rows ? p : -1;
}

// A warp to a (token, head): lane l takes the pairs l, l + 32, ... and the unrotated dims after them.
template <class T>
__global__ void __launch_bounds__(256) k_qk_norm_rope(QkArgs a) {
  const int lane = threadIdx.x & 31;
  const int H = a.heads[0] + a.heads[1];
  const long long unit = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (unit >= (long long)a.tokens * H) return;
  const int t = int(unit / H);
  int h = int(unit % H);
  const int w = h >= a.heads[0];
  if (w) h -= a.heads[0];
  const T* x = static_cast<const T*>(a.x[w]) + size_t(t) * a.x_ts[w] + size_t(h) * a.x_hs[w];
  T* y = static_cast<T*>(a.y[w]) + size_t(t) * a.y_ts[w] + size_t(h) * a.y_hs[w];
  const int p = a.rotary ? qk_position(a, t) : 0;
  if (p < 0) {
    if (lane == 0) record_err(a.err, DEV_ERR_BAD_POSITION);
    return;
  }
  const int half = a.rotary / 2;
  const float* cs = a.table + size_t(p) * a.rotary;
  float v[kQkMaxDim / 32];
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < kQkMaxDim / 32; ++i) {
    const int d = lane + 32 * i;
    v[i] = d < a.dim ? to_f32(x[d]) : 0.0f;
    sum = fmaf(v[i], v[i], sum);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  const float r = a.norm ? 1.0f / sqrtf(sum / float(a.dim) + a.eps) : 1.0f;
  const float* wt = a.weight[w];
  auto normed = [&](int d) { return to_f32(x[d]) * r * (wt ? wt[d] : 1.0f); };
#pragma unroll
  for (int i = 0; i < kQkMaxDim / 32; ++i) {
    const int d = lane + 32 * i;
    if (d < a.dim) v[i] = normed(d);
    if (d < a.rotary) {
      const bool second = a.neighbours ? (d & 1) : d >= half;
      const int e = a.neighbours ? d ^ 1 : (second ? d - half : d + half);
      const int pair = a.neighbours ? d >> 1 : (second ? d - half : d);
      const float c = cs[pair], s = cs[half + pair], o = normed(e);
      v[i] = second ? v[i] * c + o * s : v[i] * c - o * s;
    }
  }
  __syncwarp();  // y may be x: every read of the head is done before the first write
#pragma unroll
  for (int i = 0; i < kQkMaxDim / 32; ++i) {
    const int d = lane + 32 * i;
    if (d < a.dim) y[d] = from_f32<T>(v[i]);
  }
}

int launch_qk_norm_rope(const QkArgs& a, cudaStream_t st) {
  const long long units = (long long)a.tokens * (a.heads[0] + a.heads[1]);
  const long long blocks = (units + 7) / 8;
  if (blocks > 0x7fffffffll) return -1;
  if (a.type == FT_F32) k_qk_norm_rope<float><<<unsigned(blocks), 256, 0, st>>>(a);
  else if (a.type == FT_F16) k_qk_norm_rope<__half><<<unsigned(blocks), 256, 0, st>>>(a);
  else k_qk_norm_rope<__nv_bfloat16><<<unsigned(blocks), 256, 0, st>>>(a);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : -100 - int(e);
}

}  // namespace ae
