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
//   warps 2-9   epilogue, two warps to a lane quadrant, half of the tokens each; overlaps the next tile's MMAs
// Variants:
//   PAIR   two CTAs hold a 256-channel tile (cta_group::2): each stages 128 channels and half of the tokens, a
//          third less L2 traffic a product at 256 tokens, where that traffic is what one CTA alone waits for.
//   SPLIT  a cluster of 2..8 CTAs splits the depth of one tile and adds the partial sums through distributed
//          shared memory, where there are too few tiles for the SMs.
#include <algorithm>

#include "floatio.cuh"
#include "gemm_i8.h"
#include "kernels.h"
#include "linear_i8.h"
#include "ptx.cuh"
#include "rowmath.cuh"

namespace ae {

namespace {

constexpr int kChannels = 128;                 // weight rows to a CTA
constexpr int kBlock = 128;                    // depth bytes to a ring stage
constexpr int kEpi = 8;                        // epilogue warps
constexpr int kThreads = 32 * (2 + kEpi);
constexpr int kSmemMost = 232448;
constexpr int kMaxSplit = 8;
constexpr int kGroupM = 8;                     // token tiles walked together, for L2 reuse of the weights

enum Mode { ONE = 0, PAIR = 1, SPLIT = 2 };

template <int BT, int MODE>
struct Shape {
  static constexpr int CG = MODE == PAIR ? 2 : 1;
  static constexpr int W_BYTES = kChannels * kBlock;
  static constexpr int T_BYTES = BT / CG * kBlock;
  static constexpr int STAGE = W_BYTES + T_BYTES;
  static constexpr int RED = MODE == SPLIT ? (BT + kMaxSplit) * kChannels * 4 : 0;  // partial sums sent here
  static constexpr int FIXED = 1024 + RED + 2 * BT * 4 + 512;
  static constexpr int FIT = (kSmemMost - FIXED) / STAGE;
  static constexpr int STAGES = FIT < 12 ? FIT : 12;
  static constexpr int TOTAL = FIXED + STAGES * STAGE;
  static constexpr uint32_t TCOLS = 2 * BT < 32 ? 32 : 2 * BT;
  static_assert(STAGES >= 3 && TCOLS <= 512, "tile does not fit");
};

struct Grid {
  int tiles_n, tiles_m;
  int split;     // CTAs that share a tile's depth
  int early_w;   // the weights may be read before the kernel ahead has ended
};

__device__ __forceinline__ void tile_at(const Grid& g, int tile, int& nt, int& mt) {
  const int per = kGroupM * g.tiles_n;
  const int first = tile / per * kGroupM;
  const int gm = min(kGroupM, g.tiles_m - first);
  const int r = tile % per;
  mt = first + r % gm;
  nt = r / gm;
}

template <class T>
__device__ __forceinline__ void put(T* p, float v) { *p = from_f32<T>(v); }

template <int BT, int MODE, class T>
__global__ void __launch_bounds__(kThreads, 1)
    k_product_i8(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_t, ProductArgs a,
                 Grid g) {
  using S = Shape<BT, MODE>;
  constexpr int STAGES = S::STAGES;
  constexpr int CG = S::CG;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t* ring = smem;
  int* red = reinterpret_cast<int*>(ring + STAGES * S::STAGE);
  float* s_as = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(red) + S::RED);  // [2][BT] token scales
  uint64_t* full = reinterpret_cast<uint64_t*>(s_as + 2 * BT);
  uint64_t* empty = full + STAGES;
  uint64_t* acc_full = empty + STAGES;
  uint64_t* acc_empty = acc_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = MODE == ONE ? 0u : cluster_ctarank();
  const int unit = int(blockIdx.x) / (MODE == PAIR ? 2 : g.split);          // tile walker
  const int units = int(gridDim.x) / (MODE == PAIR ? 2 : g.split);
  const int tiles = g.tiles_n * g.tiles_m;
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
    fence_mbar_init();
  }
  __syncthreads();
  if constexpr (MODE != ONE) {  // the peers' barriers and shared memory are there before anything reaches for them
    cluster_arrive_release();
    cluster_wait_acquire();
  }
  if (!g.early_w) pdl_wait();
  pdl_trigger();
  // the first blocks of weights are asked for before the kernel ahead (which quantizes the tokens) has ended
  int early = 0;
  if (g.early_w) {
    if (warp == 0 && lane == 0 && unit < tiles) {
      int nt, mt;
      tile_at(g, unit, nt, mt);
      uint32_t lead = 0;
      if constexpr (MODE == PAIR) lead = map_peer(full, 0);
      for (; early < STAGES && kb0 + early < kb1; ++early) {
        uint8_t* st = ring + early * S::STAGE;
        if constexpr (MODE == PAIR) {
          if (rank == 0) mbar_arrive_expect_tx(&full[early], 2 * S::STAGE);
          tma_load_2d_pair(st, &map_w, lead + 8 * early, (kb0 + early) * kBlock, (nt * 2 + int(rank)) * kChannels);
        } else {
          mbar_arrive_expect_tx(&full[early], S::STAGE);
          tma_load_2d(st, &map_w, &full[early], (kb0 + early) * kBlock, nt * kChannels);
        }
      }
    }
    pdl_wait();
  }
  // TMEM only now: a CTA that still waits for the kernel ahead holds none, so that kernel can always get its own
  uint32_t tmem = 0;
  if (warp >= 1) {
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
  }

  if (warp == 0) {
    // ------------------------------------------------ TMA producer
    if (lane == 0) {
      uint32_t lead = 0;
      if constexpr (MODE == PAIR) lead = map_peer(full, 0);
      bool ok = true;
      int kc = 0;
      for (int tile = unit; tile < tiles && ok; tile += units) {
        int nt, mt;
        tile_at(g, tile, nt, mt);
        for (int kb = kb0; kb < kb1; ++kb, ++kc) {
          const int s = kc % STAGES;
          if (kc >= STAGES && !(ok = mbar_wait(&empty[s], ((kc / STAGES) - 1) & 1, a.err, DEV_ERR_TIMEOUT_PRODUCER)))
            break;
          uint8_t* st = ring + s * S::STAGE;
          if constexpr (MODE == PAIR) {
            if (kc >= early) {
              if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * S::STAGE);
              tma_load_2d_pair(st, &map_w, lead + 8 * s, kb * kBlock, (nt * 2 + int(rank)) * kChannels);
            }
            tma_load_2d_pair(st + S::W_BYTES, &map_t, lead + 8 * s, kb * kBlock, mt * BT + int(rank) * (BT / 2));
          } else {
            if (kc >= early) {
              mbar_arrive_expect_tx(&full[s], S::STAGE);
              tma_load_2d(st, &map_w, &full[s], kb * kBlock, nt * kChannels);
            }
            tma_load_2d(st + S::W_BYTES, &map_t, &full[s], kb * kBlock, mt * BT);
          }
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------ MMA issuer (CTA 0 of a pair issues for both)
    if (lane == 0 && (MODE != PAIR || rank == 0)) {
      constexpr uint32_t idesc = idesc_i8(kChannels * CG, BT);
      bool ok = true;
      int kc = 0, it = 0;
      for (int tile = unit; tile < tiles && ok; tile += units, ++it) {
        const int b = it & 1, u = it >> 1;
        if (u >= 1 && !(ok = mbar_wait(&acc_empty[b], (u - 1) & 1, a.err, DEV_ERR_TIMEOUT_MMA))) break;
        tc_fence_after();
        const uint32_t d = tmem + uint32_t(b * BT);
        for (int kb = kb0; kb < kb1; ++kb, ++kc) {
          const int s = kc % STAGES;
          if (!(ok = mbar_wait(&full[s], (kc / STAGES) & 1, a.err, DEV_ERR_TIMEOUT_MMA))) break;
          tc_fence_after();
          const uint32_t w_addr = smem_u32(ring + s * S::STAGE), t_addr = w_addr + S::W_BYTES;
#pragma unroll
          for (int ks = 0; ks < kBlock / 32; ++ks) {
            const uint32_t more = kb > kb0 || ks > 0;
            if constexpr (MODE == PAIR)
              mma_i8_pair(d, sdesc_sw128(w_addr + ks * 32), sdesc_sw128(t_addr + ks * 32), idesc, more);
            else
              mma_i8(d, sdesc_sw128(w_addr + ks * 32), sdesc_sw128(t_addr + ks * 32), idesc, more);
          }
          if constexpr (MODE == PAIR) mma_commit_pair(&empty[s]);
          else mma_commit(&empty[s]);
        }
        if (ok) {
          if constexpr (MODE == PAIR) mma_commit_pair(&acc_full[b]);
          else mma_commit(&acc_full[b]);
        }
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------ epilogue
    const int et = tid - 64;                 // 0..255
    const int half = (warp - 2) >> 2;        // which half of the tokens
    const int ch = (warp & 3) * 32 + lane;   // channel within the CTA's 128 = TMEM lane
    const uint32_t lane_base = tmem + (uint32_t((warp & 3) * 32) << 16);
    bool ok = true;
    int it = 0;
    for (int tile = unit; tile < tiles; tile += units, ++it) {
      const int b = it & 1, u = it >> 1;
      int nt, mt;
      tile_at(g, tile, nt, mt);
      const int n = (nt * CG + (MODE == PAIR ? int(rank) : 0)) * kChannels + ch;
      const int m0 = mt * BT;
      const int mv = min(BT, a.M - m0);      // tokens of this tile
      const bool live = n < a.N;
      float* as = s_as + b * BT;
      if (et < mv) as[et] = a.a_scale[m0 + et];
      const float ws = live ? a.w_scale[n] : 0.0f;
      const float bias = live && a.bias ? a.bias[n] : 0.0f;
      T* out = static_cast<T*>(a.out) + size_t(m0) * a.ldo + n;
      named_bar(2, 32 * kEpi);               // the scales are there; the other buffer's readers are done
      if (ok) ok = mbar_wait(&acc_full[b], u & 1, a.err, DEV_ERR_TIMEOUT_EPILOGUE);
      ok = __all_sync(0xffffffffu, ok);
      tc_fence_after();
      if constexpr (MODE != SPLIT) {
        constexpr int CW = BT / 2 < 32 ? BT / 2 : 32;  // columns to a TMEM load
        if (ok) {
#pragma unroll 1
          for (int c = half * (BT / 2); c < (half + 1) * (BT / 2) && c < mv; c += CW) {
            uint32_t r[CW];
            if constexpr (CW == 32) tmem_ld32(lane_base + uint32_t(b * BT + c), r);
            else if constexpr (CW == 16) tmem_ld16(lane_base + uint32_t(b * BT + c), r);
            else tmem_ld8(lane_base + uint32_t(b * BT + c), r);
            tmem_ld_wait();
            T* p = out + size_t(c) * a.ldo;
            if (live) {
#pragma unroll
              for (int j = 0; j < CW; ++j) {
                if (c + j < mv) put(p, fmaf(float(int(r[j])), as[c + j] * ws, bias));
                p += a.ldo;
              }
            }
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if constexpr (MODE == PAIR) mbar_arrive_cluster(map_peer(&acc_empty[b], 0));
          else mbar_arrive(&acc_empty[b]);
        }
      } else {
        // partial sums to the CTA that finishes their token: token c to CTA c % split, slot c / split
        const int slots = (BT + g.split - 1) / g.split;
        if (ok) {
          constexpr int CW = BT / 2 < 16 ? BT / 2 : 16;
#pragma unroll 1
          for (int c = half * (BT / 2); c < (half + 1) * (BT / 2) && c < mv; c += CW) {
            uint32_t r[CW];
            if constexpr (CW == 16) tmem_ld16(lane_base + uint32_t(c), r);
            else tmem_ld8(lane_base + uint32_t(c), r);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < CW; ++j) {
              if (c + j < mv) {
                const int owner = (c + j) % g.split, slot = (c + j) / g.split;
                st_cluster_u32(map_peer(red + (int(rank) * slots + slot) * kChannels + ch, owner), r[j]);
              }
            }
          }
        }
      }
    }
  }

  __syncwarp();
  if constexpr (MODE == SPLIT) {
    tc_fence_before();
    cluster_arrive_release();
    cluster_wait_acquire();
    tc_fence_after();
    if (unit < tiles) {
      int nt, mt;
      tile_at(g, unit, nt, mt);
      const int m0 = mt * BT, mv = min(BT, a.M - m0);
      const int slots = (BT + g.split - 1) / g.split;
      const int ch = tid & (kChannels - 1), n = nt * kChannels + ch;
      if (tid < 2 * kChannels && n < a.N) {
        const float ws = a.w_scale[n], bias = a.bias ? a.bias[n] : 0.0f;
        for (int slot = tid / kChannels; slot * g.split + int(rank) < mv; slot += 2) {
          const int c = slot * g.split + int(rank);
          int sum = 0;
          for (int r = 0; r < g.split; ++r) sum += red[(r * slots + slot) * kChannels + ch];
          put(static_cast<T*>(a.out) + size_t(m0 + c) * a.ldo + n,
              fmaf(float(sum), s_as[c] * ws, bias));
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (MODE == PAIR) {  // neither CTA leaves while the other may still reach into it
    cluster_arrive_release();
    cluster_wait_acquire();
  }
  if (warp == 1) {
    if constexpr (MODE == PAIR) tmem_dealloc_pair(tmem, S::TCOLS);
    else tmem_dealloc(tmem, S::TCOLS);
  }
}

// --------------------------------------------------------------------------- operands as TMA reads them
// Rows that do not start on 16 bytes are laid out at a pitch that does: 4 bytes a thread.
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

template <int BT, int MODE, class T>
cudaError_t launch(const ProductArgs& a, const CUtensorMap& map_w, const CUtensorMap& map_t, int split, int early_w,
                   cudaStream_t st) {
  using S = Shape<BT, MODE>;
  auto kernel = k_product_i8<BT, MODE, T>;
  static bool ready[kMaxDevices] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (!ready[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::TOTAL);
    if (e != cudaSuccess) return e;
    ready[dev] = true;
  }
  Grid g{};
  const int wide = kChannels * S::CG;
  g.tiles_n = (a.N + wide - 1) / wide;
  g.tiles_m = (a.M + BT - 1) / BT;
  g.split = split;
  g.early_w = early_w;
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
  return cudaLaunchKernelEx(&cfg, kernel, map_w, map_t, a, g);
}

struct Pick {
  int bt, mode, split;
};

// The tile by an estimate of the slowest SM's cycles: the blocks of one tile, each the slower of its MMAs
// (8,192 products a cycle) and its bytes (about 56 a cycle from L2), times the tiles an SM takes in turn, and
// the last tile's epilogue. A split adds about 1,000 cycles of exchange.
Pick pick(int M, int N, int K) {
  const int sms = num_sms();
  const int KB = (K + kBlock - 1) / kBlock;
  Pick best{0, 0, 0};
  double least = 1e300;
  auto consider = [&](int bt, int mode, int split) {
    const int cg = mode == PAIR ? 2 : 1;
    const long long tiles = (long long)((N + 128 * cg - 1) / (128 * cg)) * ((M + bt - 1) / bt);
    if (mode == SPLIT && tiles * split > sms) return;
    const int room = sms / cg;
    const double turns = mode == SPLIT ? 1.0 : double((tiles + room - 1) / room);
    const double block = std::max(2.0 * bt, std::max(64.0, (16384.0 + 128.0 * bt / cg) / 56.0));
    const double main = ((KB + split - 1) / split) * block;
    const double epi = 300.0 + 8.0 * std::min(bt, M);
    const double t = turns * std::max(main, epi) + std::min(main, epi) + (mode == SPLIT ? 1000.0 : 0.0);
    if (t < least) {
      least = t;
      best = {bt, mode, split};
    }
  };
  for (int bt = 16; bt <= 256 && (bt == 16 || bt / 2 < M); bt *= 2) {  // none wider than the tokens need
    consider(bt, ONE, 1);
    if (bt >= 128) consider(bt, PAIR, 1);
    if (bt <= 64)
      for (int s : {2, 3, 4, 6, 8})
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
  const Pick p = pick(a.M, a.N, a.K);
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
