// General int8 product on the tensor cores (tcgen05.mma kind::i8):
//
//   out[m, n] = fma(float(sum_k a[m, k] w[n, k]), a_scale[m] * w_scale[n], bias[n])
//
// The integer sum is exact in any order, so the only roundings are float(sum), the product of the scales, the
// fused multiply-add, and one to the output's type; every variant below gives the same bits.
//
// Weights are the MMA's A operand (128 channels to a CTA), tokens its B operand (16 to 256): a TMEM lane is
// then a channel, so w_scale and bias are one register each, a warp's 32 lanes store 32 neighbouring channels
// of one token, whatever the output's pitch, alignment or width, and a single token costs an MMA of N = 16
// instead of one of 128 rows.
//   warp 0      TMA producer: 128-byte depth blocks of both operands into a ring (128-byte swizzle; bytes past
//               the depth, rows past the operands' ends are filled with zeros by the copy)
//   warp 1      one thread issues the MMAs into one of two TMEM accumulators taken in turn
//   warps 2-17  epilogue, four warps to a lane quadrant, a quarter of the tokens each; overlaps the next tile's
//               MMAs (with 8 warps the TMEM and shared-memory latencies showed)
// Variants:
//   PAIR   two CTAs hold a 256-channel tile (cta_group::2): each stages 128 channels and half of the tokens, a
//          third less L2 traffic a product at 256 tokens, where that traffic is what one CTA alone waits for.
//   SPLIT  a cluster of 2..8 CTAs splits the depth of one tile and adds the partial sums through distributed
//          shared memory, where there are too few tiles for the SMs.
// Device times and what bounds them: 16,384 x 8,192 x 4,096 to bfloat16 351 us (PAIR: 512 cycles a depth block, the
// tensor pipe's rate, at the 1.3 GHz that the power cap leaves); 65,536 x 1,536 x 384 46-49 us (the epilogue, 3,200 cycles a
// 256 x 256 tile against 1,536 of MMAs); 1 x 4,096 x 4,096 5 us, 1 x 18,944 x 4,096 16 us (the weights' bytes: 6.5 TB/s
// beyond the first 4 us).
#include <algorithm>
#include <cmath>

#include "floatio.cuh"
#include "gemm_i8.h"
#include "kernels.h"
#include "linear_i8.h"
#include "ptx.cuh"
#include "rowmath.cuh"
#include "rowquant.cuh"

namespace ae {

namespace {

constexpr int kChannels = 128;                 // weight rows to a CTA
constexpr int kBlock = 128;                    // depth bytes to a ring stage
constexpr int kEpi = 16;                       // epilogue warps
constexpr int kThreads = 32 * (2 + kEpi);
constexpr int kSmemMost = 232448;
constexpr int kMaxSplit = 8;
constexpr int kBoxBytes = 2048;                // a warp's box of results: 32 channels x kBoxTokens

// Tokens to a box: 32 of 16-bit results (16 where a warp has no more), 16 of float.
template <class T, int BT>
constexpr int kBoxTokens = sizeof(T) == 4 || BT == 64 ? 16 : 32;

enum Mode { ONE = 0, PAIR = 1, SPLIT = 2 };

// FUSE: the most depth blocks of quantized tokens a CTA holds (16 tokens, 2 KB a block).
constexpr int kFuseBlocks = 32;
constexpr size_t kFuseMost = 16 << 10;         // bytes of activations

template <int BT, int MODE, bool FUSE = false>
struct Shape {
  static constexpr int CG = MODE == PAIR ? 2 : 1;
  static constexpr int W_BYTES = kChannels * kBlock;
  static constexpr int T_BYTES = FUSE ? 0 : BT / CG * kBlock;           // tokens of a ring stage
  static constexpr int TOK = FUSE ? kFuseBlocks * BT * kBlock : 0;          // all of a fused CTA's
  static constexpr int STAGE = W_BYTES + T_BYTES;
  static constexpr int RED = MODE == SPLIT ? (BT + kMaxSplit) * kChannels * 4 : 0;  // partial sums sent here
  static constexpr bool BOXES = MODE != SPLIT && BT >= 64;    // results leave as boxes where the output allows
  static constexpr int OUT = BOXES ? kEpi * kBoxBytes : 0;
  static constexpr int FIXED = OUT + RED + TOK + kEpi * 32 * 4 + (FUSE ? 128 : 0) + 256;
  static constexpr int FIT = (kSmemMost - FIXED) / STAGE;
  static constexpr int STAGES = FIT < 12 ? FIT : 12;
  static constexpr int TOTAL = FIXED + STAGES * STAGE;
  static constexpr uint32_t TCOLS = 2 * BT < 32 ? 32 : 2 * BT;
  static_assert(STAGES >= 3 && TCOLS <= 512, "tile does not fit");
};

struct Grid {
  QuantArgs q;   // FUSE: the float activations (q.q and q.scale unused)
  int tiles_n, tiles_m;
  int split;     // CTAs that share a tile's depth
  int early_w;   // the weights may be read before the kernel ahead has ended
  int group;     // log2 of the token tiles walked together
  int boxes;     // the channels below leave as TMA boxes: a TMA store writes a row's last 16 bytes whole, so where rows
                 // end inside them the last box's channels leave from the lanes
};

// The tiles a CTA (or pair, or cluster) takes, `units` apart in an order that walks the channels of 1 << group token
// tiles at a time. Divides only where a step leaves such a group.
struct Walk {
  int r, first, per, gm, full;
  __device__ __forceinline__ Walk(const Grid& g, int tile)
      : r(tile), first(0), per(g.tiles_n << g.group), full(1 << g.group) {
    settle(g);
  }
  __device__ __forceinline__ void step(const Grid& g, int units) {
    r += units;
    settle(g);
  }
  __device__ __forceinline__ void settle(const Grid& g) {
    if (r >= per) {
      const int q = r / per;
      r -= q * per;
      first += q << g.group;
    }
    gm = min(full, g.tiles_m - first);
  }
  __device__ __forceinline__ bool more(const Grid& g) const { return gm > 0 && r < gm * g.tiles_n; }
  __device__ __forceinline__ int nt(const Grid& g) const { return gm == full ? r >> g.group : r / gm; }
  __device__ __forceinline__ int mt(const Grid& g) const { return first + (gm == full ? r & (full - 1) : r % gm); }
};

template <int W>
__device__ __forceinline__ void tmem_ld_cols(uint32_t at, uint32_t (&r)[W]) {
  if constexpr (W == 32) tmem_ld32(at, r);
  else if constexpr (W == 16) tmem_ld16(at, r);
  else if constexpr (W == 8) tmem_ld8(at, r);
  else tmem_ld4(at, r);
}

template <class T>
__device__ __forceinline__ void put(T* p, float v) { *p = from_f32<T>(v); }

// Eight activations of a row from k on, smoothed; zeros past the row's end.
__device__ __forceinline__ void load8(const QuantArgs& q, const void* row, int k, bool wide, float (&v)[8]) {
  if (wide && k + 8 <= q.K) {
    if (q.x_type == FT_F32) {
      const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(row) + k);
      const float4 a = p[0], b = p[1];
      v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
      const uint4 p = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(row) + k);
      if (q.x_type == FT_F16) widen<__half>(p, v);
      else widen<__nv_bfloat16>(p, v);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float x = 0.0f;
      if (k + e < q.K) {
        if (q.x_type == FT_F32) x = static_cast<const float*>(row)[k + e];
        else if (q.x_type == FT_F16) x = to_f32(static_cast<const __half*>(row)[k + e]);
        else x = to_f32(static_cast<const __nv_bfloat16*>(row)[k + e]);
      }
      v[e] = x;
    }
  }
  if (q.inv_smooth) {
    if ((reinterpret_cast<uintptr_t>(q.inv_smooth) & 15) == 0 && k + 8 <= q.K) {
      const float4* p = reinterpret_cast<const float4*>(q.inv_smooth + k);
      const float4 a = p[0], b = p[1];
      v[0] *= a.x, v[1] *= a.y, v[2] *= a.z, v[3] *= a.w, v[4] *= b.x, v[5] *= b.y, v[6] *= b.z, v[7] *= b.w;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (k + e < q.K) v[e] *= q.inv_smooth[k + e];
    }
  }
}

template <int BT, int MODE, class T, bool FUSE = false>
__global__ void __launch_bounds__(kThreads, 1)
    k_product_i8(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_t,
                 const __grid_constant__ CUtensorMap map_o, ProductArgs a, Grid g) {
  using S = Shape<BT, MODE, FUSE>;
  constexpr int STAGES = S::STAGES;
  constexpr int CG = S::CG;
  static_assert(!FUSE || (BT == 16 && MODE != PAIR), "fused quantization is for up to 16 tokens");
  extern __shared__ __align__(1024) uint8_t smem_product[];  // the swizzles' 8-row atoms
  uint8_t* ring = smem_product;
  uint8_t* s_tok = ring + STAGES * S::STAGE;
  uint8_t* s_out = s_tok + S::TOK;
  int* red = reinterpret_cast<int*>(s_out + S::OUT);
  float* s_scale = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(red) + S::RED);  // 32 tokens' to a warp
  float* s_tscale = s_scale + kEpi * 32;            // FUSE: the tokens' scales, and the warps' maxima
  uint32_t* s_top = reinterpret_cast<uint32_t*>(s_tscale + 16);
  uint64_t* full = reinterpret_cast<uint64_t*>(s_tscale + (FUSE ? 32 : 0));
  uint64_t* empty = full + STAGES;
  uint64_t* acc_full = empty + STAGES;
  uint64_t* acc_empty = acc_full + 2;
  uint64_t* red_full = acc_empty + 2;
  uint64_t* tok_full = red_full + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tok_full + 1);

  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);  // uniform, for the compiler too
  const uint32_t rank = MODE == ONE ? 0u : cluster_ctarank();
  const int unit = int(blockIdx.x) / (MODE == PAIR ? 2 : g.split);          // tile walker
  const int units = int(gridDim.x) / (MODE == PAIR ? 2 : g.split);
  const int KB = (a.K + kBlock - 1) / kBlock;
  const int kb0 = MODE == SPLIT ? int((long long)(KB) * rank / g.split) : 0;
  const int kb1 = MODE == SPLIT ? int((long long)(KB) * (rank + 1) / g.split) : KB;

  if (tid == 0) {
    tma_prefetch_desc(&map_w);
    tma_prefetch_desc(&map_t);
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], kEpi * CG);
    }
    mbar_init(red_full, 1);
    mbar_init(tok_full, kEpi * 32);
    fence_mbar_init();
  }
  // SPLIT: the tile's tokens are finished in runs of `run`, CTA r taking `mine` of them from token r * run on
  int run = 0, mine = 0;
  if constexpr (MODE == SPLIT) {
    const Walk w(g, unit);
    const int mv = min(BT, a.M - w.mt(g) * BT);
    run = (mv + g.split - 1) / g.split;
    mine = max(0, min(run, mv - int(rank) * run));
    if (tid == 0 && mine) mbar_arrive_expect_tx(red_full, uint32_t(g.split - 1) * mine * kChannels * 4);
  }
  __syncthreads();
  // the peers' barriers and shared memory are there before anything reaches for them: at once in a pair, when its partial
  // sums leave in a split
  if constexpr (MODE != ONE) cluster_arrive_release();
  if constexpr (MODE == PAIR) cluster_wait_acquire();
  if (!g.early_w) pdl_wait();
  pdl_trigger();
  // the first blocks of weights are asked for before the kernel ahead (which quantizes the tokens) has ended
  int early = 0;
  if (g.early_w) {
    const Walk w(g, unit);
    if (warp == 0 && w.more(g)) {
      const int nt = w.nt(g);
      uint32_t lead = 0;
      if constexpr (MODE == PAIR) lead = map_peer(full, 0);
      early = min(STAGES, kb1 - kb0);
      for (int s = 0; s < early; ++s) {
        uint8_t* st = ring + s * S::STAGE;
        if (elect_one()) {
          if constexpr (MODE == PAIR) {
            if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * S::STAGE);
            tma_load_2d_pair(st, &map_w, lead + 8 * s, (kb0 + s) * kBlock, (nt * 2 + int(rank)) * kChannels);
          } else {
            mbar_arrive_expect_tx(&full[s], S::STAGE);
            tma_load_2d(st, &map_w, &full[s], (kb0 + s) * kBlock, nt * kChannels);
          }
        }
        __syncwarp();
      }
    }
    pdl_wait();
  }
  // TMEM only now: a CTA that still waits for the kernel ahead holds none, so that kernel can always get its own
  uint32_t tmem = 0;
  auto meet_tmem = [&] {  // warps 1..17: the allocation's address
    if (warp == 1) {
      if constexpr (MODE == PAIR) {
        tmem_alloc_pair(tmem_slot, S::TCOLS);
        tmem_relinquish_pair();
      } else {
        tmem_alloc(tmem_slot, S::TCOLS);
        tmem_relinquish();
      }
    }
    tc_fence_before();
    named_bar(1, kThreads - 32);
    tc_fence_after();
    tmem = *tmem_slot;
  };
  if (warp >= 1 && (!FUSE || warp == 1)) meet_tmem();

  if (warp == 0) {
    // ------------------------------------------------ TMA producer
    uint32_t lead = 0;
    if constexpr (MODE == PAIR) lead = map_peer(full, 0);
    bool ok = true;
    int kc = 0, s = 0;
    uint32_t phase = 1;  // of the ring's last round; its first finds every stage empty
    for (Walk w(g, unit); w.more(g) && ok; w.step(g, units)) {
      const int wy = (w.nt(g) * CG + (MODE == PAIR ? int(rank) : 0)) * kChannels;
      const int ty = w.mt(g) * BT + (MODE == PAIR ? int(rank) * (BT / 2) : 0);
      for (int kb = kb0; kb < kb1; ++kb, ++kc) {
        if (kc >= STAGES && !(ok = mbar_wait_warp(&empty[s], phase, a.err, DEV_ERR_TIMEOUT_PRODUCER))) break;
        uint8_t* st = ring + s * S::STAGE;
        if (elect_one()) {
          if constexpr (MODE == PAIR) {
            if (kc >= early) {
              if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * S::STAGE);
              tma_load_2d_pair(st, &map_w, lead + 8 * s, kb * kBlock, wy);
            }
            tma_load_2d_pair(st + S::W_BYTES, &map_t, lead + 8 * s, kb * kBlock, ty);
          } else {
            if (kc >= early) {
              mbar_arrive_expect_tx(&full[s], S::STAGE);
              tma_load_2d(st, &map_w, &full[s], kb * kBlock, wy);
            }
            if constexpr (!FUSE) tma_load_2d(st + S::W_BYTES, &map_t, &full[s], kb * kBlock, ty);
          }
        }
        __syncwarp();
        if (++s == STAGES) s = 0, phase ^= 1;
      }
    }
    // no load is in flight when the CTA ends, even where the MMAs gave up waiting for one
    if (MODE != PAIR || rank == 0)
      for (int i = max(0, kc - STAGES); i < kc; ++i)
        mbar_wait(&full[i % STAGES], (i / STAGES) & 1, a.err, DEV_ERR_TIMEOUT_PRODUCER);
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------ MMA issuer (CTA 0 of a pair issues for both)
    if (MODE != PAIR || rank == 0) {
      constexpr uint32_t idesc = idesc_i8(kChannels * CG, BT);
      bool ok = true;
      int it = 0, s = 0;
      uint32_t phase = 0;
      if constexpr (FUSE) ok = mbar_wait_warp(tok_full, 0, a.err, DEV_ERR_TIMEOUT_MMA);
      for (Walk w(g, unit); w.more(g) && ok; w.step(g, units), ++it) {
        const int b = it & 1, u = it >> 1;
        if (u >= 1 && !(ok = mbar_wait_warp(&acc_empty[b], (u - 1) & 1, a.err, DEV_ERR_TIMEOUT_MMA))) break;
        tc_fence_after();
        const uint32_t d = tmem + uint32_t(b * BT);
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!(ok = mbar_wait_warp(&full[s], phase, a.err, DEV_ERR_TIMEOUT_MMA))) break;
          tc_fence_after();
          const uint64_t wd = sdesc_sw128(smem_u32(ring) + uint32_t(s) * S::STAGE);
          const uint64_t td =
              FUSE ? sdesc_sw128(smem_u32(s_tok) + uint32_t(kb - kb0) * (BT * kBlock)) : wd + (S::W_BYTES >> 4);
          if (elect_one()) {
#pragma unroll
            for (int ks = 0; ks < kBlock / 32; ++ks) {  // 32 bytes on: + 2 in the descriptors' address field
              const uint32_t more = kb > kb0 || ks > 0;
              if constexpr (MODE == PAIR) mma_i8_pair(d, wd + 2 * ks, td + 2 * ks, idesc, more);
              else mma_i8(d, wd + 2 * ks, td + 2 * ks, idesc, more);
            }
            if constexpr (MODE == PAIR) {
              mma_commit_pair(&empty[s]);
              if (kb == kb1 - 1) mma_commit_pair(&acc_full[b]);
            } else {
              mma_commit(&empty[s]);
              if (kb == kb1 - 1) mma_commit(&acc_full[b]);
            }
          }
          __syncwarp();
          if (++s == STAGES) s = 0, phase ^= 1;
        }
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------ epilogue
    const int et = tid - 64;                 // 0..511
    const int part4 = (warp - 2) >> 2;       // which quarter of the tokens
    constexpr int QW = BT / 4;               // tokens to a quarter
    const int ch = (warp & 3) * 32 + lane;   // channel within the CTA's 128 = TMEM lane
    const int c0 = part4 * QW;
    float* as = s_scale + (warp - 2) * 32;   // scales of the 32 tokens at hand
    // Each warp keeps its own scales and biases: a lane's channel's, and those of tokens lane and lane + 32 of
    // its quarter, asked for a tile ahead. Warps meet only at the accumulators' barriers, so that one's TMEM
    // and shared-memory latencies pass under another's arithmetic.
    constexpr int TW = (QW + 31) / 32;
    float ws_next, bias_next, as_next[TW];
    int n_next = 0, m_next = 0;
    Walk w(g, unit);
    auto fetch = [&] {
      n_next = (w.nt(g) * CG + (MODE == PAIR ? int(rank) : 0)) * kChannels + ch;
      m_next = w.mt(g) * BT;
      ws_next = n_next < a.N ? a.w_scale[n_next] : 0.0f;
      bias_next = n_next < a.N && a.bias ? a.bias[n_next] : 0.0f;
#pragma unroll
      for (int i = 0; i < TW; ++i) {
        const int t = lane + 32 * i, m = m_next + c0 + t;
        if constexpr (!FUSE) as_next[i] = t < QW && m < a.M ? a.a_scale[m] : 0.0f;
      }
    };
    bool more = w.more(g);
    if (more) fetch();
    if constexpr (FUSE) {
      // The tokens of this CTA's depth, quantized here: every CTA takes the maxima over whole rows (the tokens
      // are few, and L2 holds them) while its weights are on their way. `per` threads to a row.
      const int per = (32 * kEpi) >> (a.M <= 1 ? 0 : 32 - __clz(a.M - 1));
      const int row = et / per, t = et % per;
      const bool mine_too = row < a.M;
      const size_t size = g.q.x_type == FT_F32 ? 4 : 2;
      const uint8_t* x = static_cast<const uint8_t*>(g.q.x) + (mine_too ? size_t(row) * g.q.ldx * size : 0);
      const bool wide = (reinterpret_cast<uintptr_t>(x) & 15) == 0;
      uint32_t top = 0;
      if (mine_too)
        for (int p = t; p * 8 < a.K; p += per) {
          float v[8];
          load8(g.q, x, p * 8, wide, v);
#pragma unroll
          for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(v[e]) & 0x7fffffffu);
        }
      top = __reduce_max_sync(0xffffffffu, top);
      if (lane == 0) s_top[warp - 2] = top;
      named_bar(6, 32 * kEpi);
      for (int i = 0; i < per / 32; ++i) top = max(top, s_top[et / per * (per / 32) + i]);
      const RowScale rs(top);
      if (mine_too && t == 0) s_tscale[row] = rs.scale;
      if (mine_too)
        for (int p = t; p < (kb1 - kb0) * (kBlock / 8); p += per) {
          float v[8];
          load8(g.q, x, kb0 * kBlock + p * 8, wide, v);
          // 128-byte swizzle: 16-byte piece c of token r lies at c ^ (r % 8)
          uint8_t* at = s_tok + (p >> 4) * (BT * kBlock) + row * kBlock + ((((p >> 1) & 7) ^ (row & 7)) << 4) + (p & 1) * 8;
          *reinterpret_cast<uint2*>(at) = make_uint2(rs.four(v), rs.four(v + 4));
        }
      fence_proxy_async();
      mbar_arrive(tok_full);
      meet_tmem();  // the tokens' scales are there for every warp too
    }
    const uint32_t lane_base = tmem + (uint32_t((warp & 3) * 32) << 16);
    bool ok = true;
    int it = 0;
    for (; more; ++it) {
      const int b = it & 1, u = it >> 1;
      const int n = n_next, m0 = m_next;
      const int mv = min(BT, a.M - m0);      // tokens of this tile
      const bool live = n < a.N;
      const float ws = ws_next, bias = bias_next;
      float as_own[TW];
#pragma unroll
      for (int i = 0; i < TW; ++i) as_own[i] = FUSE ? s_tscale[(c0 + lane) & 15] : as_next[i];
      w.step(g, units);
      more = w.more(g);
      if (more) fetch();
      if (ok) ok = mbar_wait(&acc_full[b], u & 1, a.err, DEV_ERR_TIMEOUT_EPILOGUE);
      ok = __all_sync(0xffffffffu, ok);
      tc_fence_after();
      // the four warps of a quarter write their channels of a token together: whole stretches of the output's rows
      // reach L2 and memory close in time (13,944 x 10,515 float, K = 128: 192 us apart, 131 together)
      named_bar(2 + part4, 128);
      // before the columns from c on: the scales of their 32 tokens
      auto scales = [&](int c) {
        if (((c - c0) & 31) == 0) {
          __syncwarp();
          as[lane] = TW == 1 || c == c0 ? as_own[0] : as_own[TW - 1];
          __syncwarp();
        }
      };
      T* out = static_cast<T*>(a.out) + size_t(m0) * a.ldo + n;
      if constexpr (MODE != SPLIT) {
        const int c_end = min(mv, c0 + QW);
        auto drained = [&] {  // this warp has read its part of the accumulator
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if constexpr (MODE == PAIR) mbar_arrive_cluster(map_peer(&acc_empty[b], 0));
            else mbar_arrive(&acc_empty[b]);
          }
        };
        if (S::BOXES && __any_sync(0xffffffffu, n < g.boxes)) {  // a vote: the same branch for the whole warp
          if constexpr (S::BOXES) {
            uint8_t* box = s_out + (warp - 2) * kBoxBytes;
            const int x = n - lane;
            constexpr int CT = kBoxTokens<T, BT>;
            [[maybe_unused]] float ws4[4], bias4[4];
            if constexpr (sizeof(T) == 2) {  // the fragments' lanes: channels lane / 4 + 8 i
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                ws4[i] = __shfl_sync(0xffffffffu, ws, (lane >> 2) + 8 * i);
                bias4[i] = __shfl_sync(0xffffffffu, bias, (lane >> 2) + 8 * i);
              }
            }
#pragma unroll 1
            for (int c = c0; c < c_end; c += CT) {
              const uint32_t at = lane_base + uint32_t(b * BT + c);
              scales(c);
              const float* cs = as + ((c - c0) & 31);
              if constexpr (sizeof(T) == 2) {
                uint32_t lo[CT / 2], hi[CT / 2];
                if (ok) {
                  if constexpr (CT == 32) {
                    tmem_ld_16x32(at, lo);
                    tmem_ld_16x32(at + (16u << 16), hi);
                  } else {
                    tmem_ld_16x16(at, lo);
                    tmem_ld_16x16(at + (16u << 16), hi);
                  }
                  tmem_ld_wait();
                }
                if (c + CT >= c_end) drained();
                if (lane == 0) bulk_wait_read<0>();  // the box's last store has left
                __syncwarp();
                const uint32_t row = smem_u32(box) + (lane & 7) * 64;
#pragma unroll
                for (int j = 0; j < CT / 8; ++j) {
                  const float2 ts = *reinterpret_cast<const float2*>(cs + 8 * j + 2 * (lane & 3));
                  uint32_t p[4];
#pragma unroll
                  for (int i = 0; i < 4; ++i) {
                    const uint32_t* r = (i < 2 ? lo : hi) + 4 * j + 2 * (i & 1);
                    const float2 v = __ffma2_rn(make_float2(float(int(r[0])), float(int(r[1]))),
                                                __fmul2_rn(ts, make_float2(ws4[i], ws4[i])),
                                                make_float2(bias4[i], bias4[i]));
                    p[i] = pack2<T>(v.x, v.y);
                  }
                  // block i = lane / 8 (channels 8 i ..), token 8 j + lane % 8; 64-byte swizzle: 16-byte piece
                  // i of token t lies at i ^ (t / 2 % 4)
                  stmatrix_x4_trans(row + j * 512 + ((((lane >> 3) ^ (lane >> 1)) & 3) << 4), p[0], p[1], p[2], p[3]);
                }
              } else {
                uint32_t r[16];
                if (ok) {
                  tmem_ld16(at, r);
                  tmem_ld_wait();
                }
                if (c + CT >= c_end) drained();
                if (lane == 0) bulk_wait_read<0>();
                __syncwarp();
                const float2 w2 = make_float2(ws, ws), b2 = make_float2(bias, bias);
#pragma unroll
                for (int j = 0; j < 16; j += 4) {
                  const float4 ts = *reinterpret_cast<const float4*>(cs + j);
                  const float2 v0 = __ffma2_rn(make_float2(float(int(r[j])), float(int(r[j + 1]))),
                                               __fmul2_rn(make_float2(ts.x, ts.y), w2), b2);
                  const float2 v1 = __ffma2_rn(make_float2(float(int(r[j + 2])), float(int(r[j + 3]))),
                                               __fmul2_rn(make_float2(ts.z, ts.w), w2), b2);
                  const float v[4] = {v0.x, v0.y, v1.x, v1.y};
#pragma unroll
                  for (int e = 0; e < 4; ++e)  // 128-byte swizzle: piece lane / 4 of token t lies at (lane / 4) ^ (t % 8)
                    *reinterpret_cast<float*>(box + (j + e) * 128 + (((lane >> 2) ^ ((j + e) & 7)) << 4) +
                                              (lane & 3) * 4) = v[e];
                }
              }
              fence_proxy_async();
              __syncwarp();
              if (lane == 0) {
                if (ok) tma_store_2d(&map_o, box, x, m0 + c);
                bulk_commit();
              }
            }
            if (c0 >= c_end) drained();
          }
        } else {
          constexpr int CW = QW < 32 ? QW : 32;  // columns to a TMEM load
#pragma unroll 1
          for (int c = c0; ok && c < c_end; c += CW) {
            uint32_t r[CW];
            scales(c);
            tmem_ld_cols<CW>(lane_base + uint32_t(b * BT + c), r);
            tmem_ld_wait();
            T* p = out + size_t(c) * a.ldo;
            // Whole chunks in packed pairs (512 x 1,002, K = 384 to bfloat16: 3.0 -> 2.8 us), but not the wide tiles of
            // long batches: there the four warps' stores of a token, value by value, still reach a row's shared
            // sectors together (13,944 x 10,515, K = 128 to float: 121 us value by value, 154 in pairs)
            if (CW <= 16 && live && c + CW <= c_end) {
#pragma unroll
              for (int j = 0; j < CW; j += 2) {
                const float2 v = __ffma2_rn(make_float2(float(int(r[j])), float(int(r[j + 1]))),
                                            __fmul2_rn(*reinterpret_cast<const float2*>(as + j), make_float2(ws, ws)),
                                            make_float2(bias, bias));
                put(p, v.x);
                put(p + a.ldo, v.y);
                p += 2 * a.ldo;
              }
            } else if (live) {
#pragma unroll
              for (int j = 0; j < CW; ++j) {
                if (c + j < c_end) put(p, fmaf(float(int(r[j])), as[j] * ws, bias));
                p += a.ldo;
              }
            }
          }
          drained();
        }
      } else {
        // this CTA's partial sums, token by token, where the ring was (every load into it has been multiplied),
        // and from there in one copy to each of the CTAs that finish them
        int* part = reinterpret_cast<int*>(ring);
        if (ok && c0 < mv) {
          uint32_t r[QW];
          tmem_ld_cols<QW>(lane_base + uint32_t(c0), r);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < QW; ++j) part[(c0 + j) * kChannels + ch] = int(r[j]);
        }
        fence_proxy_async();
        cluster_wait_acquire();
        named_bar(6, 32 * kEpi);
        if (ok && et < g.split && et != int(rank)) {
          const int count = max(0, min(run, mv - et * run));
          if (count)
            bulk_send(map_peer(red + int(rank) * run * kChannels, et), part + et * run * kChannels,
                      uint32_t(count) * kChannels * 4, map_peer(red_full, et));
        }
        if (mine) {
          if (!mbar_wait(red_full, 0, a.err, DEV_ERR_TIMEOUT_EPILOGUE)) ok = false;
          if (ok && live) {
            for (int t = part4; t < mine; t += 4) {
              const int c = int(rank) * run + t;
              int sum = part[c * kChannels + ch];
              for (int r = 0; r < g.split; ++r)
                if (r != int(rank)) sum += red[(r * run + t) * kChannels + ch];
              put(out + size_t(c) * a.ldo, fmaf(float(sum), (FUSE ? s_tscale[c] : a.a_scale[m0 + c]) * ws, bias));
            }
          }
        }
      }
    }
    if (S::BOXES && lane == 0) bulk_wait_all();
  }

  __syncwarp();
  if (MODE == SPLIT && warp < 2) cluster_wait_acquire();
  tc_fence_before();
  __syncthreads();
  if constexpr (MODE != ONE) {  // no CTA leaves while another may still reach into it
    cluster_arrive_release();
    cluster_wait_acquire();
  }
  if (warp == 1) {
    if constexpr (MODE == PAIR) tmem_dealloc_pair(tmem, S::TCOLS);
    else tmem_dealloc(tmem, S::TCOLS);
  }
}

// --------------------------------------------------------------------------- operands as TMA reads them
// Rows that do not start on 16 bytes are laid out at a pitch that does: 4 bytes a thread, read one by one at any address.
// Each call does so again: 4,096 x 4,095 weights take 12 us, bound by the issue of instructions (68 % of the slots, DRAM
// 12 %); 1 x 4,096 x 4,095 to bfloat16 takes 18.4 us with them and 6.5 from rows of 4,096 bytes, 33 x 30,522 x 383 to
// float 15.6 and 6.0.
__global__ void __launch_bounds__(256) k_lay_rows(const int8_t* src, size_t ld, int rows, int K, uint32_t* dst,
                                                  int words) {
  pdl_wait();
  pdl_trigger();
  const size_t total = size_t(rows) * words;
  for (size_t i = size_t(blockIdx.x) * blockDim.x + threadIdx.x; i < total; i += size_t(gridDim.x) * blockDim.x) {
    const size_t r = i / words;
    const int k = int(i % words) * 4;
    const uint8_t* p = reinterpret_cast<const uint8_t*>(src) + r * ld + k;
    uint32_t v = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (k + e < K) v |= uint32_t(p[e]) << (8 * e);
    dst[i] = v;
  }
}

// The channels that TMA can store to the output (4,096 x 30,522, K = 384 to bfloat16 in rows of 30,528: 59 us, 93
// with every channel from the lanes).
int box_channels(const ProductArgs& a) {
  const size_t size = float_type_bytes(a.out_type), pitch = a.ldo * size;
  if ((reinterpret_cast<uintptr_t>(a.out) & 15) || pitch % 16 || pitch >> 40) return 0;
  return a.N * size % 16 ? a.N & ~31 : a.N;
}

// Token tiles walked together. One after the other the CTAs at work write neighbouring stretches of the same
// rows, which is what counts while the weights stay in L2; eight tiles share each read of weights that do not.
int walk_group(const ProductArgs& a) { return size_t(a.N) * a.K <= (size_t(64) << 20) ? 0 : 3; }

template <int BT, int MODE, class T, bool FUSE = false>
cudaError_t launch(const ProductArgs& a, const CUtensorMap& map_w, const CUtensorMap& map_t, int split, int early_w,
                   cudaStream_t st, const QuantArgs* q = nullptr) {
  using S = Shape<BT, MODE, FUSE>;
  auto kernel = k_product_i8<BT, MODE, T, FUSE>;
  static bool ready[kMaxDevices] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (!ready[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::TOTAL);
    if (e != cudaSuccess) return e;
    ready[dev] = true;
  }
  Grid g{};
  if (FUSE) g.q = *q;
  const int wide = kChannels * S::CG;
  g.tiles_n = (a.N + wide - 1) / wide;
  g.tiles_m = (a.M + BT - 1) / BT;
  g.split = split;
  g.early_w = early_w;
  g.group = walk_group(a);
  CUtensorMap map_o = map_t;  // unused unless boxes
  g.boxes = S::BOXES ? box_channels(a) : 0;
  if (g.boxes && make_tmap_store(&map_o, a.out, size_t(a.M), size_t(g.boxes), a.ldo * sizeof(T), int(sizeof(T)), kBoxTokens<T, BT>))
    return cudaErrorInvalidValue;
  const long long tiles = (long long)g.tiles_n * g.tiles_m;
  if (tiles > 0x7fffffffll / 16) return cudaErrorInvalidValue;
  const int cluster = MODE == PAIR ? 2 : split;
  const int room = num_sms() / cluster;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned((MODE == SPLIT || tiles < room ? int(tiles) : room) * cluster));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = S::TOTAL;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = unsigned(cluster);
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = MODE == ONE ? 1 : 2;
  return cudaLaunchKernelEx(&cfg, kernel, map_w, map_t, map_o, a, g);
}

struct Pick {
  int bt, mode, split;
};

// How many clusters of `split` CTAs run at once (a cluster lies within a GPC, so not always SMs / split).
int room_for(int split) {
  static int known[kMaxDevices][kMaxSplit + 1] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  int& n = known[dev][split];
  if (!n) {
    auto kernel = k_product_i8<16, SPLIT, float>;
    cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<16, SPLIT>::TOTAL);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(split * 64));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = Shape<16, SPLIT>::TOTAL;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = unsigned(split);
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    int found = 0;
    if (cudaOccupancyMaxActiveClusters(&found, kernel, &cfg) != cudaSuccess || found < 1) found = 1;
    n = found;
  }
  return n;
}

// The tile by an estimate of the device time in cycles, whose parts are fits of measurements. Over 1,002 products of
// random shapes its choice takes 2 % longer than the fastest tile on average, over 12 % longer in 59 of them (the most:
// 1,255 x 72, K = 144, 4.0 us and 2.8, where 79 CTAs ask L2 for the same few rows of weights at once):
//   block   128 bytes of depth of one tile: its MMAs (8,192 products a cycle); 145 cycles and its bytes at 125 a
//           cycle for a CTA alone; its share of the 62 bytes a cycle and SM that L2 gives when all SMs read
//   tile    `blocks` of them, or its epilogue where that takes longer: 400 cycles and 15 a token of 16-bit results, 22
//           of float, 25 where TMA cannot store to the output, a tenth less in a pair
//   turns   tiles that an SM takes one after the other; the last one's epilogue (or depth) is not hidden
// A split's exchange adds 1,600 cycles and 60 a token, a pair 400.
Pick pick(int M, int N, int K, bool boxes, bool wide) {
  const int sms = num_sms();
  const int KB = (K + kBlock - 1) / kBlock;
  Pick best{0, 0, 0};
  const float box_cost = wide ? 22.0f : 15.0f;
  float least = 1e30f;
  auto consider = [&](int bt, int mode, int split) {
    const int cg = mode == PAIR ? 2 : 1;
    const float tiles = float((N + 128 * cg - 1) / (128 * cg)) * float((M + bt - 1) / bt);
    if (mode == SPLIT && tiles > float(room_for(split))) return;
    const float turns = std::ceil(tiles / float(sms / cg));
    const float busy = std::min(1.0f, tiles * float(cg * split) / float(sms));
    const float bytes = 16384.0f + 128.0f * bt / cg;
    const float block = std::max({2.0f * bt, 145.0f + bytes / 125.0f, busy * bytes / 62.0f});
    const float main = float((KB + split - 1) / split) * block;
    const int tokens = std::min(bt, M);
    const float epi = (mode == PAIR ? 0.9f : 1.0f) *
                      (400.0f + (boxes && mode != SPLIT && bt >= 64 ? box_cost : 25.0f) * tokens / split);
    const float more = mode == SPLIT ? 1600.0f + 60.0f * tokens : mode == PAIR ? 400.0f : 0.0f;
    const float t = turns * std::max(main, epi) + std::min(main, epi) + more;
    if (t < least) {
      least = t;
      best = {bt, mode, split};
    }
  };
  for (int bt = 16; bt <= 256 && (bt == 16 || bt / 2 < M); bt *= 2) {  // none wider than the tokens need
    consider(bt, ONE, 1);
    if (bt >= 128) consider(bt, PAIR, 1);
    if (bt <= 64)
      for (int s : {2, 3, 4, 8})
        if (s <= KB) consider(bt, SPLIT, s);
  }
  return best;
}

template <class T>
cudaError_t launch_pick(const Pick& p, const ProductArgs& a, const CUtensorMap& w, const CUtensorMap& t, int early_w,
                        cudaStream_t st) {
  switch (p.bt * 4 + p.mode) {
    case 16 * 4 + ONE: return launch<16, ONE, T>(a, w, t, 1, early_w, st);
    case 32 * 4 + ONE: return launch<32, ONE, T>(a, w, t, 1, early_w, st);
    case 64 * 4 + ONE: return launch<64, ONE, T>(a, w, t, 1, early_w, st);
    case 128 * 4 + ONE: return launch<128, ONE, T>(a, w, t, 1, early_w, st);
    case 256 * 4 + ONE: return launch<256, ONE, T>(a, w, t, 1, early_w, st);
    case 128 * 4 + PAIR: return launch<128, PAIR, T>(a, w, t, 1, early_w, st);
    case 256 * 4 + PAIR: return launch<256, PAIR, T>(a, w, t, 1, early_w, st);
    case 16 * 4 + SPLIT: return launch<16, SPLIT, T>(a, w, t, p.split, early_w, st);
    case 32 * 4 + SPLIT: return launch<32, SPLIT, T>(a, w, t, p.split, early_w, st);
    case 64 * 4 + SPLIT: return launch<64, SPLIT, T>(a, w, t, p.split, early_w, st);
  }
  return cudaErrorInvalidValue;
}

template <class T>
cudaError_t launch_fused(const Pick& p, const ProductArgs& a, const CUtensorMap& w, const QuantArgs& q, cudaStream_t st) {
  return p.mode == SPLIT ? launch<16, SPLIT, T, true>(a, w, w, p.split, 0, st, &q)
                         : launch<16, ONE, T, true>(a, w, w, 1, 0, st, &q);
}

size_t row_pitch(int K) { return (size_t(K) + 15) / 16 * 16; }

bool in_place(const int8_t* p, size_t ld, int rows) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (rows == 1 || ld % 16 == 0);
}

}  // namespace

size_t product_scratch(const ProductArgs& a) {
  size_t n = 0;
  if (!in_place(a.a, a.lda, a.M)) n += (size_t(a.M) * row_pitch(a.K) + 255) / 256 * 256;
  if (!in_place(a.w, a.ldw, a.N)) n += size_t(a.N) * row_pitch(a.K);
  return n;
}

// Up to 16 tokens whose depth (its share of a split) fits a CTA's token blocks, and little enough to read in each of
// some 130 CTAs at once. On the device one 4,096-deep bfloat16 token takes 6.3 us this way and 6.7 us in two kernels,
// two smoothed ones 7.3 and 6.8, sixteen 11.6 and 7.1. A launch less spares the host about 2 us, so up to the bound a
// call that the host makes gains; one replayed from a graph loses up to 0.5 us near it.
int launch_product_fused(const ProductArgs& args, const QuantArgs& q, cudaStream_t st) {
  ProductArgs a = args;
  if (a.M > 16 || size_t(a.M) * a.K * float_type_bytes(q.x_type) > kFuseMost || !in_place(a.w, a.ldw, a.N)) return 1;
  const Pick p = pick(a.M, a.N, a.K, box_channels(a) > 0, a.out_type == FT_F32);
  if (p.bt != 16 || ((a.K + kBlock - 1) / kBlock + p.split - 1) / p.split > kFuseBlocks) return 1;
  if (a.N == 1) a.ldw = row_pitch(a.K);
  CUtensorMap map_w;
  if (make_tmap_i8_rows(&map_w, a.w, size_t(a.N), size_t(a.K), a.ldw, kChannels)) return -3;
  const cudaError_t e = a.out_type == FT_F32   ? launch_fused<float>(p, a, map_w, q, st)
                        : a.out_type == FT_F16 ? launch_fused<__half>(p, a, map_w, q, st)
                                               : launch_fused<__nv_bfloat16>(p, a, map_w, q, st);
  return e == cudaSuccess ? 0 : -100 - int(e);
}

int launch_product_i8(const ProductArgs& args, uint8_t* scratch, int tokens_ahead, cudaStream_t st, int* kernels) {
  ProductArgs a = args;
  auto lay = [&](const int8_t*& p, size_t& ld, int rows) {
    const size_t pitch = row_pitch(a.K);
    if (!in_place(p, ld, rows)) {
      const size_t words = size_t(rows) * (pitch / 4);
      const unsigned blocks = unsigned(std::min<size_t>((words + 255) / 256, size_t(num_sms()) * 32));
      if (launch_pdl(k_lay_rows, dim3(blocks), dim3(256), 0, st, p, ld, rows, a.K, reinterpret_cast<uint32_t*>(scratch),
                     int(pitch / 4)) != cudaSuccess)
        return false;
      p = reinterpret_cast<const int8_t*>(scratch);
      ld = pitch;
      scratch += (size_t(rows) * pitch + 255) / 256 * 256;
      ++*kernels;
      tokens_ahead = 0;
    } else if (rows == 1) {
      ld = pitch;
    }
    return true;
  };
  if (!lay(a.a, a.lda, a.M) || !lay(a.w, a.ldw, a.N)) return -2;
  const Pick p = pick(a.M, a.N, a.K, box_channels(a) > 0, a.out_type == FT_F32);
  CUtensorMap map_w, map_t;
  if (make_tmap_i8_rows(&map_w, a.w, size_t(a.N), size_t(a.K), a.ldw, kChannels) ||
      make_tmap_i8_rows(&map_t, a.a, size_t(a.M), size_t(a.K), a.lda, p.mode == PAIR ? p.bt / 2 : p.bt))
    return -3;
  ++*kernels;
  const cudaError_t e = a.out_type == FT_F32   ? launch_pick<float>(p, a, map_w, map_t, tokens_ahead, st)
                        : a.out_type == FT_F16 ? launch_pick<__half>(p, a, map_w, map_t, tokens_ahead, st)
                                               : launch_pick<__nv_bfloat16>(p, a, map_w, map_t, tokens_ahead, st);
  return e == cudaSuccess ? 0 : -100 - int(e);
}

}  // namespace ae
