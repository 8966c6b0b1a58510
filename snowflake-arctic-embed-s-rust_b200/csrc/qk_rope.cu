// RMS norm of every query and key head and the rotation of its first `rotary` dims by the token's
// position, in one pass over the heads:
//
//   y = x / sqrt(mean(x^2) + eps) * weight;  (y_i, y_j) -> (y_i c - y_j s, y_j c + y_i s)
//
// for the pairs (i, i + rotary / 2) or (2i, 2i + 1), with c and s from a float table row of the position.
// All of it in float; one rounding to the heads' type.
#include <algorithm>

#include "floatio.cuh"
#include "kernels.h"
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

// Heads of any dim at any address, a warp to a (token, head): lane l takes the pairs l, l + 32, ... and the unrotated dims after them.
template <class T>
__global__ void __launch_bounds__(256) k_qk_norm_rope(QkArgs a) {
  pdl_trigger();
  pdl_wait();
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

// VE elements as one load or store.
template <class T, int VE>
struct Piece {
  static constexpr int WORDS = VE * int(sizeof(T)) / 4;
  uint32_t w[WORDS];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (WORDS == 4) {
      const uint4 v = *reinterpret_cast<const uint4*>(p);
      w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    } else if constexpr (WORDS == 2) {
      const uint2 v = *reinterpret_cast<const uint2*>(p);
      w[0] = v.x, w[1] = v.y;
    } else {
      w[0] = *reinterpret_cast<const uint32_t*>(p);
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (WORDS == 4) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    else if constexpr (WORDS == 2) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint32_t*>(p) = w[0];
  }
  __device__ __forceinline__ void get(float (&v)[VE]) const {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < VE; ++i) v[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
      for (int i = 0; i < WORDS; ++i) {
        const float2 f = unpack2<T>(w[i]);
        v[2 * i] = f.x, v[2 * i + 1] = f.y;
      }
    }
  }
  __device__ __forceinline__ void set(const float (&v)[VE]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < VE; ++i) w[i] = __float_as_uint(v[i]);
    } else {
#pragma unroll
      for (int i = 0; i < WORDS; ++i) w[i] = pack2<T>(v[2 * i], v[2 * i + 1]);
    }
  }
};

constexpr int kQkThreads = 256;
constexpr int kQkHeads = 4;  // heads to a thread

struct QkGrid {
  int lanes_log2;   // lanes to a head: the power of two from dim / (2 VE)
  int slots[2];     // groups of kQkHeads heads of a token
  int tokens[2];    // tokens to a block
  int blocks_q;     // blocks of queries; those of the keys follow
};

// Heads whose halves are whole pieces. A thread holds the two pieces of a head that rotate against one another
// (or, unrotated, two neighbouring ones), for kQkHeads heads of one token, so a token's table row and the norm
// weights are loaded once for four heads, all of a thread's loads of heads are in flight together, and every
// element is read and written by one thread (outputs may be the inputs).
template <class T, int VE>
__global__ void __launch_bounds__(kQkThreads) k_qk_pieces(QkArgs a, QkGrid g) {
  __shared__ int s_pos[kQkThreads];
  pdl_trigger();
  pdl_wait();
  const int w = int(blockIdx.x) >= g.blocks_q;
  const int t0 = (int(blockIdx.x) - (w ? g.blocks_q : 0)) * g.tokens[w];
  const int nt = min(g.tokens[w], a.tokens - t0);
  const int tid = threadIdx.x;
  if (tid < nt) {
    const int p = a.rotary ? qk_position(a, t0 + tid) : 0;
    s_pos[tid] = p;
    if (p < 0) record_err(a.err, DEV_ERR_BAD_POSITION);
  }
  __syncthreads();
  const int lanes = 1 << g.lanes_log2;
  const int j = tid & (lanes - 1);
  const int turning = a.rotary / (2 * VE);       // lanes whose pieces are rotated
  const bool in = j * 2 * VE < a.dim;
  const bool turns = j < turning;
  int d0, d1;                                     // where the two pieces start
  if (turns && !a.neighbours) d0 = j * VE, d1 = a.rotary / 2 + j * VE;
  else d0 = j * 2 * VE, d1 = d0 + VE;
  float w0[VE], w1[VE];
  if (in && a.weight[w]) {
    Piece<float, VE < 4 ? VE : 4> v;
    constexpr int S = VE < 4 ? VE : 4;
#pragma unroll
    for (int i = 0; i < VE; i += S) {
      float f[S];
      v.load(a.weight[w] + d0 + i);
      v.get(f);
#pragma unroll
      for (int e = 0; e < S; ++e) w0[i + e] = f[e];
      v.load(a.weight[w] + d1 + i);
      v.get(f);
#pragma unroll
      for (int e = 0; e < S; ++e) w1[i + e] = f[e];
    }
  } else {
#pragma unroll
    for (int i = 0; i < VE; ++i) w0[i] = w1[i] = 1.0f;
  }
  const int H = a.heads[w], slots = g.slots[w], groups = kQkThreads >> g.lanes_log2;
  const T* x = static_cast<const T*>(a.x[w]);
  T* y = static_cast<T*>(a.y[w]);
  const int items = nt * slots;
  for (int base = 0; base < items; base += groups) {  // uniform: the shuffles below take whole warps
    const int item = base + (tid >> g.lanes_log2);
    const int tt = item < items ? item / slots : 0;
    const int t = t0 + tt, p = s_pos[tt];
    const bool live = item < items && in && p >= 0;
    const int h0 = (item - tt * slots) * kQkHeads;
    Piece<T, VE> p0[kQkHeads], p1[kQkHeads];
#pragma unroll
    for (int h = 0; h < kQkHeads; ++h) {
      if (live && h0 + h < H) {
        const T* at = x + size_t(t) * a.x_ts[w] + size_t(h0 + h) * a.x_hs[w];
        p0[h].load(at + d0);
        p1[h].load(at + d1);
      } else {
#pragma unroll
        for (int i = 0; i < Piece<T, VE>::WORDS; ++i) p0[h].w[i] = p1[h].w[i] = 0;
      }
    }
    float c[VE], s[VE];
    if (live && turns) {
      const float* row = a.table + size_t(p) * a.rotary + j * VE;
      constexpr int S = VE < 4 ? VE : 4;
      Piece<float, S> v;
#pragma unroll
      for (int i = 0; i < VE; i += S) {
        float f[S];
        v.load(row + i);
        v.get(f);
#pragma unroll
        for (int e = 0; e < S; ++e) c[i + e] = f[e];
        v.load(row + a.rotary / 2 + i);
        v.get(f);
#pragma unroll
        for (int e = 0; e < S; ++e) s[i + e] = f[e];
      }
    } else {
#pragma unroll
      for (int i = 0; i < VE; ++i) c[i] = 1.0f, s[i] = 0.0f;
    }
#pragma unroll
    for (int h = 0; h < kQkHeads; ++h) {
      float u[VE], v[VE];
      p0[h].get(u);
      p1[h].get(v);
      if (a.norm) {
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < VE; ++i) sum = fmaf(u[i], u[i], fmaf(v[i], v[i], sum));
        for (int o = lanes >> 1; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        const float r = 1.0f / sqrtf(sum / float(a.dim) + a.eps);
#pragma unroll
        for (int i = 0; i < VE; ++i) u[i] = u[i] * r * w0[i], v[i] = v[i] * r * w1[i];
      }
      if (turns) {
        if (!a.neighbours) {
#pragma unroll
          for (int i = 0; i < VE; ++i) {
            const float e = u[i], f = v[i];
            u[i] = e * c[i] - f * s[i];
            v[i] = f * c[i] + e * s[i];
          }
        } else if constexpr (VE >= 2) {
#pragma unroll
          for (int i = 0; i < VE; i += 2) {
            const float e = u[i], f = u[i + 1], k = v[i], l = v[i + 1];
            u[i] = e * c[i / 2] - f * s[i / 2];
            u[i + 1] = f * c[i / 2] + e * s[i / 2];
            v[i] = k * c[VE / 2 + i / 2] - l * s[VE / 2 + i / 2];
            v[i + 1] = l * c[VE / 2 + i / 2] + k * s[VE / 2 + i / 2];
          }
        } else {
          const float e = u[0], f = v[0];  // one pair to a thread
          u[0] = e * c[0] - f * s[0];
          v[0] = f * c[0] + e * s[0];
        }
      }
      if (live && h0 + h < H) {
        T* at = y + size_t(t) * a.y_ts[w] + size_t(h0 + h) * a.y_hs[w];
        p0[h].set(u);
        p1[h].set(v);
        p0[h].store(at + d0);
        p1[h].store(at + d1);
      }
    }
  }
}

template <class T, int VE>
static cudaError_t launch_pieces(const QkArgs& a, cudaStream_t st) {
  QkGrid g{};
  while ((1 << g.lanes_log2) * 2 * VE < a.dim) ++g.lanes_log2;
  const int groups = kQkThreads >> g.lanes_log2;
  long long blocks[2];
  for (int w = 0; w < 2; ++w) {
    g.slots[w] = (a.heads[w] + kQkHeads - 1) / kQkHeads;
    g.tokens[w] = g.slots[w] ? std::max(1, std::min(kQkThreads, groups / g.slots[w])) : 1;
    blocks[w] = g.slots[w] ? (a.tokens + g.tokens[w] - 1) / g.tokens[w] : 0;
  }
  if (blocks[0] + blocks[1] > 0x7fffffffll) return cudaErrorInvalidValue;
  g.blocks_q = int(blocks[0]);
  return launch_pdl(k_qk_pieces<T, VE>, dim3(unsigned(blocks[0] + blocks[1])), dim3(kQkThreads), 0, st, a, g);
}

// Whether every piece of VE elements (and of a head's weights and table rows) is whole and on its own size.
static bool whole_pieces(const QkArgs& a, int VE, size_t size) {
  if (a.dim % (2 * VE) || a.rotary % (2 * VE) || a.dim > 64 * VE) return false;
  uintptr_t bits = 0, fbits = reinterpret_cast<uintptr_t>(a.table);
  for (int w = 0; w < 2; ++w) {
    if (!a.heads[w]) continue;
    bits |= reinterpret_cast<uintptr_t>(a.x[w]) | reinterpret_cast<uintptr_t>(a.y[w]);
    if (a.tokens > 1) bits |= (a.x_ts[w] | a.y_ts[w]) * size;
    if (a.heads[w] > 1) bits |= (a.x_hs[w] | a.y_hs[w]) * size;
    fbits |= reinterpret_cast<uintptr_t>(a.weight[w]);
  }
  return bits % (VE * size) == 0 && fbits % (std::min(VE, 4) * 4) == 0;
}

template <class T>
static cudaError_t launch_type(const QkArgs& a, cudaStream_t st) {
  constexpr int VE = kPiece<T>;
  if (whole_pieces(a, VE, sizeof(T))) return launch_pieces<T, VE>(a, st);
  if (whole_pieces(a, VE / 2, sizeof(T))) return launch_pieces<T, VE / 2>(a, st);
  if (whole_pieces(a, VE / 4, sizeof(T))) return launch_pieces<T, VE / 4>(a, st);
  const long long units = (long long)a.tokens * (a.heads[0] + a.heads[1]);
  const long long blocks = (units + 7) / 8;
  if (blocks > 0x7fffffffll) return cudaErrorInvalidValue;
  return launch_pdl(k_qk_norm_rope<T>, dim3(unsigned(blocks)), dim3(256), 0, st, a);
}

int launch_qk_norm_rope(const QkArgs& a, cudaStream_t st) {
  const cudaError_t e = a.type == FT_F32   ? launch_type<float>(a, st)
                        : a.type == FT_F16 ? launch_type<__half>(a, st)
                                           : launch_type<__nv_bfloat16>(a, st);
  return e == cudaSuccess ? 0 : -100 - int(e);
}

}  // namespace ae
