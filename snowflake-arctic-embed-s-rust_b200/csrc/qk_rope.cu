// RMS norm of every query and key head and the rotation of its first `rotary` dims by the token's
// position, in one pass over the heads:
//
//   y = x / sqrt(mean(x^2) + eps) * weight;  (y_i, y_j) -> (y_i c - y_j s, y_j c + y_i s)
//
// for the pairs (i, i + rotary / 2) or (2i, 2i + 1), with c and s from a float table row of the position.
// All of it in float; one rounding to the heads' type.
#include <algorithm>

#include "floatio.cuh"
#include "gemm_i8.h"
#include "kernels.h"
#include "linear_i8.h"
#include "ptx.cuh"

namespace ae {

constexpr int kQkMaxDim = 512;

// Position of token t: given, or counted from the start of its sequence (cu[s] <= t < cu[s + 1], s among lo .. hi);
// -1 if there is none inside the table.
__device__ __forceinline__ int qk_position(const QkArgs& a, int t, int lo, int hi) {
  int p;
  if (a.positions) {
    p = a.positions[t];
  } else {
    while (lo < hi) {  // the last s with cu[s] <= t
      const int mid = (lo + hi + 1) >> 1;
      if (a.cu[mid] <= uint32_t(t)) lo = mid;
      else hi = mid - 1;
    }
    p = lo < a.n_seqs && a.cu[lo] <= uint32_t(t) ? t - int(a.cu[lo]) : -1;
  }
  return p >= 0 && p < a.table_rows ? p : -1;
}

// The last s among 0 .. n with cu[s] <= t (0 if there is none), by a converged warp: 32 entries a round, so two
// rounds for a thousand sequences where halving takes ten loads one after the other.
__device__ __forceinline__ int warp_search(const uint32_t* cu, int n, int t) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = n;
  while (lo < hi) {
    const int step = (hi - lo + 31) >> 5;
    const long long at = lo + (long long)(lane + 1) * step;
    const unsigned below = __ballot_sync(0xffffffffu, at <= hi && cu[at <= hi ? at : hi] <= uint32_t(t));
    lo += __popc(below) * step;
    hi = min(hi, lo + step - 1);
  }
  return lo;
}

// Heads of any dim at any address, a warp to a (token, head), lane l the dims l, l + 32, ...: single elements, those that
// rotate read three times (for the sum, as themselves, as their partner's), from L1 after the first. 16,384 tokens of
// 32 + 8 heads of 128 bfloat16 that start on odd elements take 554 us, bound by the issue of instructions (70 % of the
// slots, DRAM 6 %), and 64 in pieces; heads of 33 take 440.
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
  const int p = a.rotary ? qk_position(a, t, 0, a.n_seqs) : 0;
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
  __device__ __forceinline__ void get(float2 (&v)[(VE + 1) / 2]) const {
#pragma unroll
    for (int i = 0; i < (VE + 1) / 2; ++i) {
      if constexpr (sizeof(T) == 2) v[i] = unpack2<T>(w[i]);
      else if constexpr (VE == 1) v[i] = make_float2(__uint_as_float(w[0]), 0.0f);
      else v[i] = make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
    }
  }
  __device__ __forceinline__ void set(const float2 (&v)[(VE + 1) / 2]) {
#pragma unroll
    for (int i = 0; i < (VE + 1) / 2; ++i) {
      if constexpr (sizeof(T) == 2) {
        w[i] = pack2<T>(v[i].x, v[i].y);
      } else {
        w[i * (VE == 1 ? 1 : 2)] = __float_as_uint(v[i].x);
        if constexpr (VE > 1) w[2 * i + 1] = __float_as_uint(v[i].y);
      }
    }
  }
};

constexpr int kQkThreads = 64;

struct QkGrid {
  int lanes_log2;   // lanes to a head: the power of two from dim / (2 VE)
  int slots[2];     // groups of HPT heads of a token; a group of lanes takes one
  int blocks_q;     // blocks of queries; those of the keys follow
};

__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }

// VE floats from an address that is a multiple of min(VE, 4) of them, as pairs (VE = 1: the first of one pair).
template <int VE>
__device__ __forceinline__ void load_floats(const float* p, float2 (&v)[(VE + 1) / 2]) {
  if constexpr (VE == 1) {
    v[0] = make_float2(*p, 0.0f);
  } else if constexpr (VE == 2) {
    v[0] = *reinterpret_cast<const float2*>(p);
  } else {
#pragma unroll
    for (int i = 0; i < VE; i += 4) {
      const float4 f = *reinterpret_cast<const float4*>(p + i);
      v[i / 2] = make_float2(f.x, f.y);
      v[i / 2 + 1] = make_float2(f.z, f.w);
    }
  }
}

// Factors of a first piece's own values (a0) and of their partners (b0), and of a second piece's (a1, b1): on entry
// a0 and a1 hold the weights, c and s the angles'.
template <int VE, bool NEIGHBOURS>
__device__ __forceinline__ void turn_factors(const float2* c, const float2* s, float2* a0, float2* b0,
                                             float2* a1, float2* b1) {
  constexpr int P = (VE + 1) / 2;
  if constexpr (!NEIGHBOURS || VE == 1) {
#pragma unroll
    for (int i = 0; i < P; ++i) {
      b0[i] = mul2(a1[i], make_float2(-s[i].x, -s[i].y));
      b1[i] = mul2(a0[i], s[i]);
      a0[i] = mul2(a0[i], c[i]);
      a1[i] = mul2(a1[i], c[i]);
    }
  } else {
    // pair i of the first piece turns by angle i, of the second by angle VE / 2 + i
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const float c0 = i & 1 ? c[i / 2].y : c[i / 2].x, s0 = i & 1 ? s[i / 2].y : s[i / 2].x;
      const int k = VE / 2 + i;
      const float c1 = k & 1 ? c[k / 2].y : c[k / 2].x, s1 = k & 1 ? s[k / 2].y : s[k / 2].x;
      b0[i] = make_float2(-a0[i].y * s0, a0[i].x * s0);
      b1[i] = make_float2(-a1[i].y * s1, a1[i].x * s1);
      a0[i] = mul2(a0[i], make_float2(c0, c0));
      a1[i] = mul2(a1[i], make_float2(c1, c1));
    }
  }
}

// One head's two pieces, normed and turned in place; every lane of its group takes part in the sum.
template <int VE, bool NEIGHBOURS>
__device__ __forceinline__ void norm_and_turn(const QkArgs& a, float scale, int lanes, bool turns, const float2* a0,
                                              const float2* b0, const float2* a1, const float2* b1, float2* u,
                                              float2* v) {
  constexpr int P = (VE + 1) / 2;
  if (a.norm) {
    float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < P; ++i) sum = fma2(u[i], u[i], fma2(v[i], v[i], sum));
    float all = sum.x + sum.y;
    for (int o = lanes >> 1; o; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
    const float r = rsqrtf(all * scale + a.eps);
#pragma unroll
    for (int i = 0; i < P; ++i) u[i] = mul2(u[i], make_float2(r, r)), v[i] = mul2(v[i], make_float2(r, r));
  }
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const float2 e = u[i], f = v[i];
    u[i] = mul2(e, a0[i]);
    v[i] = mul2(f, a1[i]);
    if (turns) {  // not by factors of zero: an infinity stays in its own pair
      if constexpr (!NEIGHBOURS || VE == 1) {
        u[i] = fma2(f, b0[i], u[i]);
        v[i] = fma2(e, b1[i], v[i]);
      } else {
        u[i] = fma2(make_float2(e.y, e.x), b0[i], u[i]);
        v[i] = fma2(make_float2(f.y, f.x), b1[i], v[i]);
      }
    }
  }
}

// Heads whose halves are whole pieces. A thread holds the two pieces of a head that rotate against one another
// (or, with neighbouring pairs or no rotation, two pieces in a row) for HPT heads of one token, so that a token's
// table row and the norm weights, multiplied together once, serve all of them, all of a thread's loads of heads
// are in flight together, and every element is read and written by one thread (outputs may be the inputs):
//   y_0 = (r x_0) (w_0 c) + (r x_1) (-w_1 s),   y_1 = (r x_1) (w_1 c) + (r x_0) (w_0 s),   r = 1 / rms
// in packed float pairs, 5 instructions an element with its conversions. HPT is 4 where that leaves threads for
// every SM, else 1: one token takes 2.2 us with one head to a thread and 4.3 with four.
template <class T, int VE, int HPT, bool NEIGHBOURS>
__global__ void __launch_bounds__(kQkThreads) k_qk_pieces(QkArgs a, QkGrid g) {
  constexpr int P = (VE + 1) / 2;                 // float pairs to a piece
  __shared__ int s_pos[kQkThreads], s_seq[2];
  pdl_trigger();
  pdl_wait();
  const int w = int(blockIdx.x) >= g.blocks_q;
  const int tid = threadIdx.x, slots = g.slots[w];
  const int groups = kQkThreads >> g.lanes_log2, group = tid >> g.lanes_log2;
  // the block's first group's token and slot, then this group's
  const unsigned block = blockIdx.x - (w ? unsigned(g.blocks_q) : 0u);
  const unsigned long long first = (unsigned long long)block * groups;
  const int t0 = first >> 32 ? int(first / unsigned(slots)) : int(unsigned(first) / unsigned(slots));
  const int s0 = int(first - (unsigned long long)t0 * slots);
  const int tt = (s0 + group) / slots, t = t0 + tt;
  const int h0 = (s0 + group - tt * slots) * HPT;
  const bool counted = a.rotary && !a.positions;  // places in sequences are searched for once a token
  if (counted) {
    const int nt = min((s0 + groups - 1) / slots + 1, a.tokens - t0);
    if (tid < 64) {  // the sequences of the block's first and last token, and between them those of the others
      const int found = warp_search(a.cu, a.n_seqs, t0 + (tid < 32 ? 0 : nt - 1));
      if ((tid & 31) == 0) s_seq[tid >> 5] = found;
    }
    __syncthreads();
    if (tid < nt) s_pos[tid] = qk_position(a, t0 + tid, s_seq[0], s_seq[1]);
    __syncthreads();
  }
  const int lanes = 1 << g.lanes_log2;
  const int j = tid & (lanes - 1);
  const bool in = j * 2 * VE < a.dim;
  const bool turns = j * 2 * VE < a.rotary;
  int d0, d1;                                     // where the two pieces start
  if (turns && !NEIGHBOURS) d0 = j * VE, d1 = a.rotary / 2 + j * VE;
  else d0 = j * 2 * VE, d1 = d0 + VE;
  const int H = a.heads[w];
  const float scale = 1.0f / float(a.dim);
  const bool work = t < a.tokens && in;
  const T* x = static_cast<const T*>(a.x[w]) + size_t(t) * a.x_ts[w] + size_t(h0) * a.x_hs[w];
  Piece<T, VE> p0[HPT], p1[HPT];
#pragma unroll
  for (int h = 0; h < HPT; ++h) {
    if (work && h0 + h < H) {
      p0[h].load(x + d0);
      p1[h].load(x + d1);
    } else {
#pragma unroll
      for (int i = 0; i < Piece<T, VE>::WORDS; ++i) p0[h].w[i] = p1[h].w[i] = 0;
    }
    x += a.x_hs[w];
  }
  int p = 0;
  if (counted) {
    p = t < a.tokens ? s_pos[tt] : 0;
  } else if (a.rotary && t < a.tokens) {
    p = a.positions[t];
    if (p < 0 || p >= a.table_rows) p = -1;
  }
  const bool live = work && p >= 0;
  if (p < 0 && j == 0 && h0 == 0) record_err(a.err, DEV_ERR_BAD_POSITION);
  float2 a0[P], b0[P], a1[P], b1[P];
  if (live && a.weight[w]) {
    load_floats<VE>(a.weight[w] + d0, a0);
    load_floats<VE>(a.weight[w] + d1, a1);
  } else {
#pragma unroll
    for (int i = 0; i < P; ++i) a0[i] = a1[i] = make_float2(1.0f, 1.0f);
  }
  if (live && turns) {
    const float* row = a.table + size_t(p) * a.rotary + j * VE;
    float2 c[P], s[P];
    load_floats<VE>(row, c);
    load_floats<VE>(row + a.rotary / 2, s);
    turn_factors<VE, NEIGHBOURS>(c, s, a0, b0, a1, b1);
  }
  T* y = static_cast<T*>(a.y[w]) + size_t(t) * a.y_ts[w] + size_t(h0) * a.y_hs[w];
#pragma unroll
  for (int h = 0; h < HPT; ++h) {
    float2 u[P], v[P];
    p0[h].get(u);
    p1[h].get(v);
    norm_and_turn<VE, NEIGHBOURS>(a, scale, lanes, turns, a0, b0, a1, b1, u, v);
    if (live && h0 + h < H) {
      p0[h].set(u);
      p1[h].set(v);
      p0[h].store(y + d0);
      p1[h].store(y + d1);
    }
    y += a.y_hs[w];
  }
}


template <class T, int VE, int HPT>
static cudaError_t launch_heads(const QkArgs& a, cudaStream_t st) {
  QkGrid g{};
  while ((1 << g.lanes_log2) * 2 * VE < a.dim) ++g.lanes_log2;
  const int groups = kQkThreads >> g.lanes_log2;
  long long blocks[2];
  for (int w = 0; w < 2; ++w) {
    g.slots[w] = (a.heads[w] + HPT - 1) / HPT;
    blocks[w] = ((long long)a.tokens * g.slots[w] + groups - 1) / groups;
  }
  if (blocks[0] + blocks[1] > 0x7fffffffll) return cudaErrorInvalidValue;
  g.blocks_q = int(blocks[0]);
  return launch_pdl(a.neighbours ? k_qk_pieces<T, VE, HPT, true> : k_qk_pieces<T, VE, HPT, false>,
                    dim3(unsigned(blocks[0] + blocks[1])), dim3(kQkThreads), 0, st, a, g);
}

template <class T, int VE>
static cudaError_t launch_pieces(const QkArgs& a, cudaStream_t st) {
  // four heads to a thread from 256 threads an SM on (777 tokens of 10 + 5 heads of 80, 210 threads an SM: 5.5 us with
  // four, 3.7 with one; 690 of 32 + 2 heads of 96 in float, 500 threads: 5.2 and 6.3)
  const long long threads = (long long)a.tokens * ((a.heads[0] + 3) / 4 + (a.heads[1] + 3) / 4) * (a.dim / (2 * VE));
  return threads >= 256ll * num_sms() ? launch_heads<T, VE, 4>(a, st) : launch_heads<T, VE, 1>(a, st);
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
