// Low-rank adapters of many requests at once beside a shared projection:
//   s_j[t]   = scale_a A_{a(t), j} x[t]                (first product, rank r)
//   y[t, n]  = base[t, n] + sum_r B_{a(t)}[r, n] s_{j(n)}[t, r]
// for every token t of the batch, where a(t) is the token's adapter, j(n) the
// fused slice of column n (q | k | v, gate | up) and base the projection's
// float32 output.  Optionally y goes through the SwiGLU of the interleaved
// gate/up columns and out in the model's type.
//
// The plan lists tiles of up to 64 tokens that share an adapter (adapter -1:
// none).  Two launches: lora_shrink computes s (k shared out over the CTAs of
// a cluster when there are few tiles, the parts summed in a fixed order, so
// results do not depend on timing), lora_expand adds B s to the base.  Calls of
// little work take one (lora_one_kernel; the any-shape kernels for small K);
// tiles of many tokens go to the tcgen05 kernels of lora_tc.cu.
//
// s is a float32 sum.  The second product takes it in bf16 terms (s rounded,
// then what is left rounded, ...) whose sum is s: one term would put 2^-9 of
// the adapter's part into the result.  Two (2^-17 and better) for a bf16
// result, three (2^-25) for a float32 one.
#include <cmath>

#include <cooperative_groups.h>

#include "lora_device.cuh"

namespace ms {

int launch_cluster(void (*kernel)(ShrinkArgs), dim3 grid, int threads, int smem, int split,
                   cudaStream_t s, const ShrinkArgs& p) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = threads;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2]{};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim = {1, 1, (unsigned)split};
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  (void)cudaLaunchKernelEx(&cfg, kernel, p);
  return check_launch("lora_shrink");
}

namespace {

// ---- first product, bf16 ------------------------------------------------------
// mma m16n8k16 with the rank rows of A as M and the tokens as N (8 of them:
// small groups waste less than with 16).  Both operands come straight from
// global memory: the sum over k may take its terms in any order, so lane
// (g, t) of a fragment takes the 16 bytes k0 + 8t .. 8t+7 of its row for two
// MMAs at once, instead of the four separate pairs of the nominal layout.
// A CTA takes 16 * MT rank rows, 8 * NT tokens at a time; its 8 warps and the CTAs of its
// cluster share out k, and the parts meet in (distributed) shared memory.
// An MMA truncates its sum to the accumulator's 24 bits, always towards zero: four or
// eight of them make a partial sum, which is added in float32 with rounding (a running
// sum of n MMAs comes out about n 2^-26 too small: 1.6e-6 for K = 14336 over 8 warps).
// The steps of a partial sum have their loads in flight together.
// Each slice's rank rows are padded to a multiple of 16 (`rank_p`), with
// zeros in s.  Bound by HBM where every few tokens bring an adapter of their own:
// 1536 tokens of 256 adapters of rank 16, K = 14336 (161 MB), 28.7 us (5.6 TB/s).
constexpr int kShrinkWarps = 8;

template <int MT, int NT>
__global__ void __launch_bounds__(kShrinkWarps * 32, 2) lora_shrink_kernel(ShrinkArgs p) {
  pdl_enter();
  constexpr int kShrinkTokens = 8 * NT;
  extern __shared__ __align__(16) float s_red[];  // [warps][kShrinkTokens][16 MT]
  constexpr int kOuts = kShrinkTokens * 16 * MT;
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int splits = (int)cluster.num_blocks(), split = (int)cluster.block_rank();
  Tile tile;
  if (!load_tile(p.plan, p.ad, blockIdx.x, tile, p.err)) return;
  const int rank_p = pad16(tile.rank);
  const int rows = p.ns * rank_p, m0 = blockIdx.y * 16 * MT;
  if (m0 >= rows) return;  // the whole cluster alike
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;

  const __nv_bfloat16* ar[MT][2];
  bool row_in[MT][2];  // the rows that pad the rank are zero
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int mp = min(m0 + 16 * m, rows - 16) + 8 * h + g;
      const int j = mp / rank_p, r = min(mp - j * rank_p, tile.rank - 1);
      row_in[m][h] = mp - j * rank_p < tile.rank;
      ar[m][h] = p.a + ((int64_t)p.ns * tile.offset + j * tile.rank + r) * p.K + 8 * t;
    }
  const int k_end = min(p.K, (split + 1) * p.k_per);
  const uint4 zero = make_uint4(0, 0, 0, 0);
  for (int first = 0; first < tile.count; first += kShrinkTokens) {
    const int count = min(tile.count - first, kShrinkTokens);
    const __nv_bfloat16* xr[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int tok = token_at(p.plan, tile.start + first + min(8 * n + g, count - 1), p.err);
      xr[n] = p.x + (int64_t)max(tok, 0) * p.x_stride + 8 * t;
    }
    float acc[MT][NT][4] = {};
    constexpr int kParts = MT + NT <= 3 ? 4 : 2;  // steps of a partial sum
    for (int k1 = split * p.k_per + 32 * warp; k1 < k_end; k1 += 32 * kShrinkWarps * kParts) {
      float sum[MT][NT][4] = {};
#pragma unroll
      for (int i = 0; i < kParts; ++i) {
        const int k0 = k1 + 32 * kShrinkWarps * i;
        const bool in = k0 + 8 * t < k_end;
        uint4 xv[NT], av[MT][2];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            av[m][h] = in && row_in[m][h] ? __ldg(reinterpret_cast<const uint4*>(ar[m][h] + k0)) : zero;
#pragma unroll
        for (int n = 0; n < NT; ++n)
          xv[n] = in && 8 * n < count ? __ldg(reinterpret_cast<const uint4*>(xr[n] + k0)) : zero;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          if (8 * n >= count) break;
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            mma_bf16(sum[m][n], av[m][0].x, av[m][1].x, av[m][0].y, av[m][1].y, xv[n].x, xv[n].y);
            mma_bf16(sum[m][n], av[m][0].z, av[m][1].z, av[m][0].w, av[m][1].w, xv[n].z, xv[n].w);
          }
        }
      }
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[m][n][e] += sum[m][n][e];
    }
    // the warps' parts, summed in warp order
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int row = 16 * m + g + 8 * (e >> 1), col = 8 * n + 2 * t + (e & 1);
          s_red[warp * kOuts + col * 16 * MT + row] = acc[m][n][e];
        }
    __syncthreads();
    const int todo = count * 16 * MT;
    for (int i = threadIdx.x; i < todo; i += kShrinkWarps * 32) {
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < kShrinkWarps; ++w) v += s_red[w * kOuts + i];
      s_red[i] = v;  // only this thread reads or writes column i of the parts
    }
    if (splits > 1) cluster.sync(); else __syncthreads();
    finish_s(p, cluster, s_red, 16 * MT, tile.start + first, count, m0, min(16 * MT, rows - m0), tile.rank,
             p.ad.scales[tile.adapter]);
    // no CTA leaves, or starts on s_red again, while another reads its part
    if (splits > 1) cluster.sync(); else __syncthreads();
  }
}

// The same for larger tiles: 64 tokens x RB rank rows per CTA, both operands
// through shared memory (each is read RB / 16 and 4 times), k in steps of 64
// behind a ring of cp.async.  Warp (m, n) of the 4 x 2 has 16 tokens and RB / 2
// rank rows; each step's four MMAs make a partial sum, added with rounding.  1280
// tokens of 32 adapters, K = 2048, two slices, rank 16-32 (11 MB): 9.7 us, the
// latency of the ring's first steps and of the cluster's sum.
constexpr int kBigK = 64;
constexpr int kBigLd = kBigK + 8;  // padded row (elements): conflict-free ldmatrix
constexpr int kBigStages = 4;

template <int RB>
__global__ void __launch_bounds__(256, 2) lora_shrink_tile_kernel(ShrinkArgs p) {
  pdl_enter();
  extern __shared__ __align__(16) unsigned char smem[];
  constexpr int kStage = (kTile + RB) * kBigLd;  // elements
  constexpr int kOutLd = RB + 4;                 // floats per token of the parts
  static_assert(kTile * kOutLd * 4 <= kBigStages * kStage * 2, "the parts fit the ring");
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int splits = (int)cluster.num_blocks(), split = (int)cluster.block_rank();
  Tile tile;
  if (!load_tile(p.plan, p.ad, blockIdx.x, tile, p.err)) return;
  const int rank_p = pad16(tile.rank), rows = p.ns * rank_p, m0 = blockIdx.y * RB;
  if (tile.count == 0 || m0 >= rows) return;  // the whole cluster alike
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int wm = warp & 3, wn = warp >> 2;
  __nv_bfloat16* ring = reinterpret_cast<__nv_bfloat16*>(smem);

  // This thread's loads of a step: 16 bytes at k offset kq of rows r0, r0 + 32, ...
  constexpr int kLoads = (kTile + RB) / 32;
  const int kq = 8 * (threadIdx.x & 7), r0 = threadIdx.x >> 3;
  const __nv_bfloat16* src[kLoads];
  bool have[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int r = r0 + 32 * i;
    src[i] = p.a;
    if (r < kTile) {
      const int tok = r < tile.count ? token_at(p.plan, tile.start + r, p.err) : -1;
      have[i] = tok >= 0;
      if (have[i]) src[i] = p.x + (int64_t)tok * p.x_stride + kq;
    } else {
      const int mp = m0 + r - kTile, j = mp / rank_p, q = mp - j * rank_p;
      have[i] = mp < rows && q < tile.rank;
      if (have[i]) src[i] = p.a + ((int64_t)p.ns * tile.offset + j * tile.rank + q) * p.K + kq;
    }
  }
  const int k_begin = split * p.k_per, k_end = min(p.K, k_begin + p.k_per);
  const int steps = k_end > k_begin ? (k_end - k_begin + kBigK - 1) / kBigK : 0;
  auto load = [&](int step) {
    if (step < steps) {
      const int k = k_begin + step * kBigK;
      const uint32_t dst = s_addr(ring + (step % kBigStages) * kStage + r0 * kBigLd + kq);
      const bool in = k + kq < k_end;
#pragma unroll
      for (int i = 0; i < kLoads; ++i)
        cp_async16(dst + 32 * i * kBigLd * 2, have[i] && in ? src[i] + k : p.a, have[i] && in);
    }
    cp_commit();
  };
  for (int i = 0; i < kBigStages - 1; ++i) load(i);
  constexpr int NT = RB / 16;  // 8-row tiles per warp
  float acc[NT][4] = {};
  const bool active = 16 * wm < tile.count && m0 + wn * (RB / 2) < rows;
  for (int step = 0; step < steps; ++step) {
    cp_wait<kBigStages - 2>();
    __syncthreads();  // this step's data is there, the last step's slot is free
    load(step + kBigStages - 1);
    if (!active) continue;
    const __nv_bfloat16* xs = ring + (step % kBigStages) * kStage;
    const uint32_t xa = s_addr(xs + (16 * wm + (lane & 15)) * kBigLd + 8 * (lane >> 4));
    const uint32_t aa = s_addr(xs + (kTile + wn * (RB / 2) + (lane & 7) + 8 * (lane >> 4)) * kBigLd +
                               8 * ((lane >> 3) & 1));
    float sum[NT][4];
#pragma unroll
    for (int k = 0; k < kBigK; k += 16) {
      uint32_t xf[4];
      ldsm4(xf, xa + 2 * k);
#pragma unroll
      for (int n = 0; n < NT; n += 2) {
        uint32_t af[4];  // rank rows 8n .. 8n+15: b0, b1 of n, then of n + 1
        ldsm4(af, aa + n * 8 * kBigLd * 2 + 2 * k);
        if (k == 0) {
          mma_bf16_first(sum[n], xf[0], xf[1], xf[2], xf[3], af[0], af[1]);
          mma_bf16_first(sum[n + 1], xf[0], xf[1], xf[2], xf[3], af[2], af[3]);
        } else {
          mma_bf16(sum[n], xf[0], xf[1], xf[2], xf[3], af[0], af[1]);
          mma_bf16(sum[n + 1], xf[0], xf[1], xf[2], xf[3], af[2], af[3]);
        }
      }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[n][e] += sum[n][e];
  }
  cp_wait<0>();
  __syncthreads();
  float* part = reinterpret_cast<float*>(smem);  // [token][kOutLd]
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      part[(16 * wm + g + 8 * (e >> 1)) * kOutLd + wn * (RB / 2) + 8 * n + 2 * t + (e & 1)] = acc[n][e];
  if (splits > 1) cluster.sync(); else __syncthreads();
  finish_s(p, cluster, part, kOutLd, tile.start, tile.count, m0, min(RB, rows - m0), tile.rank,
           tile.rank > 0 ? p.ad.scales[tile.adapter] : 0.f);
  if (splits > 1) cluster.sync();  // no CTA leaves while another reads its part
}

// ---- both products in one launch, for a few tokens ----------------------------------
// A call of a few tokens and a rank of at most 16 is bound by the host's launches
// and by latency.  A cluster of 8 CTAs takes a tile: its CTAs share out k for the
// first product (as lora_shrink_kernel, 16 rows of A, 8 tokens at a time), meet,
// and share out the columns for the second, on the CUDA cores: a thread has 2
// columns of 8 tokens, s stays float32.  B and the base, which the first product
// does not wait for, are loaded before it.
// One token at 2048 x 2048, rank 16: 20 us a call from the host and 5.4 us in a
// replayed graph, to 28 and 6.3 us as two launches; 32 tokens of 32 adapters at
// 4096 x 4096, 9.7 to 10.3 us in a graph.  K = 14336 costs a graph 0.7 us more than
// two launches, and the host 8 us less.  The rule (one_launch) stops where a graph
// would lose much: at rank 64, 9.9 to 6.8 us; at 28672 columns, 14.5 to 9.1 us.
constexpr int kOneTokens = 8;
constexpr int kOneRank = 16;
constexpr int kOneSplit = 8;
constexpr int kOneN = kOneSplit * kShrinkWarps * 64;  // 4096 columns

template <typename TO>
__global__ void __launch_bounds__(kShrinkWarps * 32) lora_one_kernel(ShrinkArgs p, ExpandArgs e) {
  pdl_enter();
  __shared__ float s_red[kShrinkWarps][kOneTokens][kOneRank];
  __shared__ float s_part[kOneTokens][kOneRank];  // this CTA's share of k
  __shared__ __align__(16) float s_sum[kOneTokens][kOneRank];
  __shared__ int s_tok[kOneTokens];
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int split = (int)cluster.block_rank();
  Tile tile;
  if (!load_tile(p.plan, p.ad, blockIdx.x, tile, p.err)) return;  // the whole cluster alike
  if (tile.count == 0 || (e.in_place && tile.rank == 0)) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int k_end = min(p.K, (split + 1) * p.k_per);
  const uint4 zero = make_uint4(0, 0, 0, 0);
  const float scale = tile.rank > 0 ? p.ad.scales[tile.adapter] : 0.f;

  const int per = (e.N + 2 * kOneSplit - 1) / (2 * kOneSplit) * 2;  // columns of a CTA, at most 512
  const int c = split * per + 2 * threadIdx.x;
  const bool in = 2 * threadIdx.x < per && c < e.N;
  __nv_bfloat162 w[kOneRank];
  const __nv_bfloat16* b = e.b + (int64_t)tile.offset * e.N + c;
#pragma unroll
  for (int r = 0; r < kOneRank; ++r)
    w[r] = in && r < tile.rank ? __ldg(reinterpret_cast<const __nv_bfloat162*>(b + r * e.N))
                               : __nv_bfloat162{};

  for (int first = 0; first < tile.count; first += kOneTokens) {
    const int count = min(tile.count - first, kOneTokens);
    if (threadIdx.x < kOneTokens)
      s_tok[threadIdx.x] =
          threadIdx.x < count ? token_at(p.plan, tile.start + first + threadIdx.x, p.err) : -1;
    __syncthreads();
    float2 base[kOneTokens];
#pragma unroll
    for (int k = 0; k < kOneTokens; ++k) {
      const int tok = s_tok[k];
      base[k] = in && tok >= 0 ? *reinterpret_cast<const float2*>(e.base + tok * e.base_stride + c)
                               : make_float2(0.f, 0.f);
    }
    if (tile.rank > 0) {
      const __nv_bfloat16* xr = p.x + (int64_t)max(s_tok[min(g, count - 1)], 0) * p.x_stride + 8 * t;
      const __nv_bfloat16* ar[2];
#pragma unroll
      for (int h = 0; h < 2; ++h)
        ar[h] = p.a + (int64_t)(tile.offset + min(8 * h + g, tile.rank - 1)) * p.K + 8 * t;
      float acc[4] = {};
#pragma unroll 2
      for (int k0 = split * p.k_per + 32 * warp; k0 < k_end; k0 += 32 * kShrinkWarps) {
        const bool kin = k0 + 8 * t < k_end;
        const uint4 xv = kin ? __ldg(reinterpret_cast<const uint4*>(xr + k0)) : zero;
        const uint4 a0 = kin && g < tile.rank ? __ldg(reinterpret_cast<const uint4*>(ar[0] + k0)) : zero;
        const uint4 a1 = kin && 8 + g < tile.rank ? __ldg(reinterpret_cast<const uint4*>(ar[1] + k0)) : zero;
        float sum[4];
        mma_bf16_first(sum, a0.x, a1.x, a0.y, a1.y, xv.x, xv.y);
        mma_bf16(sum, a0.z, a1.z, a0.w, a1.w, xv.z, xv.w);
#pragma unroll
        for (int q = 0; q < 4; ++q) acc[q] += sum[q];
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) s_red[warp][2 * t + (q & 1)][g + 8 * (q >> 1)] = acc[q];
      __syncthreads();
      const int token = (threadIdx.x >> 4) & 7, row = threadIdx.x & 15;
      if (threadIdx.x < kOneTokens * kOneRank) {
        float v = 0.f;
#pragma unroll
        for (int k = 0; k < kShrinkWarps; ++k) v += s_red[k][token][row];
        s_part[token][row] = v;
      }
      cluster.sync();
      if (threadIdx.x < kOneTokens * kOneRank) {
        float v = 0.f;
#pragma unroll
        for (int k = 0; k < kOneSplit; ++k) v += *cluster.map_shared_rank(&s_part[token][row], k);
        s_sum[token][row] = row < tile.rank ? v * scale : 0.f;
      }
      cluster.sync();  // the parts have been read; s is complete
    }
#pragma unroll
    for (int k = 0; k < kOneTokens; ++k) {
      const int tok = s_tok[k];
      if (!in || tok < 0) continue;
      float x0 = 0.f, x1 = 0.f;
      if (tile.rank > 0) {
#pragma unroll
        for (int r = 0; r < kOneRank; r += 4) {
          const float4 s = *reinterpret_cast<const float4*>(&s_sum[k][r]);
          const float2 w0 = __bfloat1622float2(w[r]), w1 = __bfloat1622float2(w[r + 1]),
                       w2 = __bfloat1622float2(w[r + 2]), w3 = __bfloat1622float2(w[r + 3]);
          x0 = fmaf(s.x, w0.x, fmaf(s.y, w1.x, fmaf(s.z, w2.x, fmaf(s.w, w3.x, x0))));
          x1 = fmaf(s.x, w0.y, fmaf(s.y, w1.y, fmaf(s.z, w2.y, fmaf(s.w, w3.y, x1))));
        }
      }
      x0 += base[k].x;
      x1 += base[k].y;
      if constexpr (std::is_same_v<TO, float>)
        *reinterpret_cast<float2*>(static_cast<float*>(e.out) + tok * e.out_stride + c) = make_float2(x0, x1);
      else
        *reinterpret_cast<__nv_bfloat162*>(static_cast<__nv_bfloat16*>(e.out) + tok * e.out_stride + c) =
            __floats2bfloat162_rn(x0, x1);
    }
    __syncthreads();  // s and the tokens have been read
  }
}

// ---- second product, bf16 -----------------------------------------------------
// A CTA keeps the s rows of up to 16 WM tokens of a tile in shared memory and
// goes through its share of the columns, 32 WN at a step: their base values
// and adapter rows come in by cp.async, up to three steps ahead.  mma m16n8k16
// with tokens as M, columns as N, the rank as K; warp (m, n) of the WM x WN
// has 16 tokens and 32 columns.  The result leaves through the base's buffer, in
// whole 32-byte sectors.
// 1536 tokens of 256 adapters, rank 16, N = 4096 (84 MB): 21.8 us (3.9 TB/s, near the
// rate at which half of it can be written).  1280 tokens of 32 adapters, rank 16-32,
// N = 11264 with the SwiGLU (89 MB): 26 us after the first product (3.4 TB/s); 14
// warps a SM keep the issue slots half busy, and what they wait for most is the
// result of the last instruction.  Small CTAs do best: 512 threads took 42 us for the
// call's two products, 256 38 and 128 36 (37 with the base added last); more of them
// per SM by fewer registers (96 of 122) take 8B's two products from 57 to 76 us.
constexpr int kPad = 8;  // elements after each shared-memory row: conflict-free fragment reads

// Which slice a warp's 32 columns take their s from.  kMixed: several slices', one after
// another for all columns, of which the other slices' keep what they had (B as zeros
// there would do, but for an infinite s).
enum SliceMode { kOneSlice, kInterleaved, kMixed };

// acc += s B for one warp: sa, sb the shared addresses of this lane's ldmatrix
// rows (first rank step), term and slice offsets in bytes.
template <int TERMS, int MODE>
__device__ __forceinline__ void expand_mma(float (&acc)[4][4], uint32_t sa, uint32_t sb, int rank_p,
                                           uint32_t b_step, const ExpandArgs& p, int c, int j0,
                                           int j1) {
  const uint32_t term = 2u * rank_p, slice = TERMS * term;
  const int t = threadIdx.x & 3;
#pragma unroll (MODE == kMixed ? 1 : 2)
  for (int k = 0; k < rank_p; k += 16, sa += 32, sb += b_step) {
    uint32_t b[8];  // n-tile n: b[2n], b[2n + 1]
    {
      uint32_t b01[4], b23[4];
      ldsm4_t(b01, sb);
      ldsm4_t(b23, sb + 32);
#pragma unroll
      for (int e = 0; e < 4; ++e) b[e] = b01[e], b[4 + e] = b23[e];
    }
    if constexpr (MODE == kMixed) {
      for (int j = j0; j <= j1; ++j) {
        uint32_t a[TERMS][4];
#pragma unroll
        for (int e = 0; e < TERMS; ++e) ldsm4(a[e], sa + j * slice + e * term);
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          float had[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) had[e] = acc[n][e];
#pragma unroll
          for (int e = TERMS - 1; e >= 0; --e)
            mma_bf16(acc[n], a[e][0], a[e][1], a[e][2], a[e][3], b[2 * n], b[2 * n + 1]);
#pragma unroll
          for (int e = 0; e < 4; ++e)  // this lane's columns 2t and 2t + 1 of the 8
            if (slice_of(p, c + 8 * n + 2 * t + (e & 1)) != j) acc[n][e] = had[e];
        }
      }
    } else {
#pragma unroll
      for (int h = 0; h < (MODE == kInterleaved ? 2 : 1); ++h) {
        uint32_t a[TERMS][4];
        const uint32_t at = sa + (MODE == kInterleaved ? h : j0) * slice;
#pragma unroll
        for (int e = 0; e < TERMS; ++e) ldsm4(a[e], at + e * term);
#pragma unroll
        for (int e = TERMS - 1; e >= 0; --e)  // the small terms first
#pragma unroll
          for (int n = h; n < 4; n += MODE == kInterleaved ? 2 : 1)
            mma_bf16(acc[n], a[e][0], a[e][1], a[e][2], a[e][3], b[2 * n], b[2 * n + 1]);
      }
    }
  }
}

template <int EPI, int WM, int WN>
__global__ void __launch_bounds__(32 * WM * WN, 1) lora_expand_kernel(ExpandArgs p) {
  constexpr int TERMS = EPI == kLoraF32 ? 3 : 2;
  constexpr int kTm = 16 * WM, kCols = 32 * WN, kThreads = 32 * WM * WN;
  constexpr int kBaseLd = kCols + kPad, kBLd = kCols + kPad;
  constexpr int kBRows = kThreads / (kCols / 8), kBaseRows = kThreads / (kCols / 4);  // rows a pass of loads
  static_assert(kBaseRows >= 1, "a row of loads fits the block");
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ int s_tok[kTile];
  // The plan and the adapters are read before the launch wait when
  // lora_shrink runs directly before: it does not write them, and everything
  // before it has completed once its blocks allow this kernel to start.
  if (!p.after_shrink) pdl_enter();
  Tile tile;
  const bool ok = load_tile(p.plan, p.ad, blockIdx.y, tile, p.err);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int wm = warp % WM, wn = warp / WM;
  const int rank_p = pad16(tile.rank);
  const int s_row = p.ns * TERMS * rank_p, s_ld = s_row + kPad;
  // s rows, then the ring of (base rows, adapter rows)
  const int s_bytes = kTm * (p.ns * TERMS * p.rank_pm + kPad) * 2;
  constexpr int kBaseBytes = kTm * kBaseLd * 4;
  const int stage_bytes = kBaseBytes + p.rank_pm * kBLd * 2;
  __nv_bfloat16* s_s = reinterpret_cast<__nv_bfloat16*>(smem);
  unsigned char* ring = smem + s_bytes;
  const int at = kTm * blockIdx.z;  // a long tile's tokens among the CTAs of z
  const bool work = ok && tile.count > at && !(p.in_place && tile.rank == 0);
  const int step = kCols * gridDim.x, c_first = kCols * blockIdx.x;

  if (work)
    for (int i = threadIdx.x; i < tile.count; i += kThreads)
      s_tok[i] = token_at(p.plan, tile.start + i, p.err);
  __syncthreads();
  // adapter rows / base rows of columns c .. c + kCols - 1 into ring slot `slot`
  auto load_b = [&](int c, int slot) {
    __nv_bfloat16* s_b = reinterpret_cast<__nv_bfloat16*>(ring + slot * stage_bytes + kBaseBytes);
    const int q = 8 * (threadIdx.x % (kCols / 8)), r0 = threadIdx.x / (kCols / 8);
    const bool in = c + q < p.N;
    const __nv_bfloat16* src = p.b + ((int64_t)tile.offset + r0) * p.N + (in ? c + q : 0);
    uint32_t dst = s_addr(s_b + r0 * kBLd + q);
    for (int r = r0; r < rank_p; r += kBRows) {
      const bool row = r < tile.rank;
      cp_async16(dst, row ? src : p.b, row && in);
      src += (int64_t)kBRows * p.N;
      dst += kBRows * kBLd * 2;
    }
  };
  // Element offsets (lora_add checks that they fit 32 bits) of the rows that
  // this thread loads, r0 + kBaseRows i, and of those it stores.
  constexpr int kBaseLoads = kTm / kBaseRows;
  constexpr int kChunks = EPI == kLoraF32 ? 8 : EPI == kLoraBf16 ? 4 : 2;  // of 16 bytes per row
  constexpr int kPer = EPI == kLoraF32 ? 4 : 8;                            // outputs per chunk
  constexpr int kStores = kChunks / 2;                                     // 16 rows
  uint32_t base_at[kBaseLoads], out_at[kStores], has = 0;
  const int base_q = 4 * (threadIdx.x % (kCols / 4)), base_r = threadIdx.x / (kCols / 4);
  auto find_rows = [&](int first, int here) {
    has = 0;
#pragma unroll
    for (int i = 0; i < kBaseLoads; ++i) {
      const int r = base_r + kBaseRows * i, tok = r < here ? s_tok[first + r] : -1;
      has |= (uint32_t)(tok >= 0) << i;
      base_at[i] = (uint32_t)(max(tok, 0) * p.base_stride + base_q);
    }
#pragma unroll
    for (int i = 0; i < kStores; ++i) {
      const int at = lane + 32 * i, r = 16 * wm + at / kChunks;
      const int tok = r < here ? s_tok[first + r] : -1;
      has |= (uint32_t)(tok >= 0) << (16 + i);
      out_at[i] = (uint32_t)(max(tok, 0) * p.out_stride + at % kChunks * kPer);
    }
  };
  auto load_base = [&](int c, int slot) {
    const bool in = c + base_q < p.N;
    const uint32_t dst = s_addr(reinterpret_cast<float*>(ring + slot * stage_bytes) + base_r * kBaseLd + base_q);
#pragma unroll
    for (int i = 0; i < kBaseLoads; ++i)
      if (has >> i & 1u)
        cp_async16(dst + i * kBaseRows * kBaseLd * 4, in ? p.base + (base_at[i] + c) : p.base, in);
  };
  if (work && p.after_shrink) load_b(c_first, 0);
  if (p.after_shrink) pdl_enter();
  if (!work) return;

  for (int first = at; first < tile.count; first += kTm * gridDim.z) {
    const int here = min(tile.count - first, kTm);
    if (first > at) __syncthreads();  // the last pass is done with s and the ring
    find_rows(first, here);
    for (int i = threadIdx.x; i < here * (s_row / 8); i += kThreads) {
      const int row = i / (s_row / 8), q = 8 * (i - row * (s_row / 8));
      cp_async16(s_addr(s_s + row * s_ld + q), p.s + (tile.start + first + row) * p.s_stride + q, true);
    }
    for (int k = 0; k + 1 < p.stages; ++k) {
      if (c_first + k * step < p.N) {
        if (first > at || k > 0 || !p.after_shrink) load_b(c_first + k * step, k);
        load_base(c_first + k * step, k);
      }
      cp_commit();
    }
    int slot = 0;
    for (int c0 = c_first; c0 < p.N; c0 += step) {
      if (p.stages > 3) cp_wait<2>(); else if (p.stages > 2) cp_wait<1>(); else cp_wait<0>();
      __syncthreads();  // this step's data is there, the last step's slot is free
      const int ahead = p.stages - 1, cn = c0 + ahead * step;
      if (cn < p.N) {
        const int free = slot == 0 ? p.stages - 1 : slot - 1;
        load_b(cn, free);
        load_base(cn, free);
      }
      cp_commit();
      const int c = c0 + 32 * wn, m = 16 * wm;
      float* s_base = reinterpret_cast<float*>(ring + slot * stage_bytes) + m * kBaseLd + 32 * wn;
      const __nv_bfloat16* s_b =
          reinterpret_cast<const __nv_bfloat16*>(ring + slot * stage_bytes + kBaseBytes) + 32 * wn;
      slot = slot + 1 == p.stages ? 0 : slot + 1;
      if (m >= here || c >= p.N) continue;
      const bool upper = here - m > 8;  // tokens in the upper 8 rows
      float acc[4][4] = {};
      const uint32_t sa = s_addr(s_s + (m + (lane & 15)) * s_ld + 8 * (lane >> 4));
      const uint32_t sb = s_addr(s_b + (lane & 15) * kBLd + 8 * (lane >> 4));
      if (p.interleaved) {
        expand_mma<TERMS, kInterleaved>(acc, sa, sb, rank_p, 32 * kBLd, p, c, 0, 1);
      } else {
        const int j0 = slice_of(p, c), j1 = slice_of(p, min(c + 31, p.N - 1));
        if (j0 == j1)
          expand_mma<TERMS, kOneSlice>(acc, sa, sb, rank_p, 32 * kBLd, p, c, j0, j0);
        else
          expand_mma<TERMS, kMixed>(acc, sa, sb, rank_p, 32 * kBLd, p, c, j0, j1);
      }
      // the base is added last: an MMA truncates its sum to the accumulator's 24 bits
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (h == 1 && !upper) break;
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const float2 v = *reinterpret_cast<const float2*>(s_base + (g + 8 * h) * kBaseLd + 8 * n + 2 * t);
          acc[n][2 * h] += v.x;
          acc[n][2 * h + 1] += v.y;
        }
      }
      // out through this warp's part of the base rows, which all its lanes have read
      __syncwarp();
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (h == 1 && !upper) break;
        float* row = s_base + (g + 8 * h) * kBaseLd;
        if constexpr (EPI == kLoraSwiGLU) {
#pragma unroll
          for (int n = 0; n < 4; n += 2)
            reinterpret_cast<__nv_bfloat162*>(row)[2 * n + t] =
                __floats2bfloat162_rn(silu(acc[n][2 * h]) * acc[n + 1][2 * h],
                                      silu(acc[n][2 * h + 1]) * acc[n + 1][2 * h + 1]);
        } else {
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            const float2 v = make_float2(acc[n][2 * h], acc[n][2 * h + 1]);
            if constexpr (EPI == kLoraF32)
              reinterpret_cast<float2*>(row)[4 * n + t] = v;
            else
              reinterpret_cast<__nv_bfloat162*>(row)[4 * n + t] = __floats2bfloat162_rn(v.x, v.y);
          }
        }
      }
      __syncwarp();
      const int c_out = EPI == kLoraSwiGLU ? c / 2 : c, n_out = EPI == kLoraSwiGLU ? p.N / 2 : p.N;
#pragma unroll
      for (int i = 0; i < kStores; ++i) {
        const int at = lane + 32 * i, row = at / kChunks, q = at % kChunks;
        if (!(has >> (16 + i) & 1u) || c_out + q * kPer >= n_out) continue;
        const float4 v = reinterpret_cast<const float4*>(s_base + row * kBaseLd)[q];
        if constexpr (EPI == kLoraF32)
          *reinterpret_cast<float4*>(static_cast<float*>(p.out) + (out_at[i] + c_out)) = v;
        else
          *reinterpret_cast<float4*>(static_cast<__nv_bfloat16*>(p.out) + (out_at[i] + c_out)) = v;
      }
    }
  }
}

// ---- any type, size and alignment ----------------------------------------------
// The float32 models and shapes the tensor-core kernels do not take.  Second
// product: a CTA has 8 tokens of a tile, a thread one output of each, so that an
// element of B is read once for 8 tokens.  With K up to 256 the same CTA computes
// its tokens' s (a warp per 4 rows of A, again for 8 tokens), which costs less than
// another launch; above, a CTA of lora_shrink_any_kernel has 4 rows and 8 tokens,
// its warps share out k.  Latency bounds both: in a replayed graph of float32
// calls, one token to 256, K = 128 takes 5.6 to 7.9 us at rank 8 (6.9 to 9.9 as two
// launches), K = 256 7.0 to 9.9 (7.2 to 11.3), K = 512 9.0 to 15.9 fused and 7.4 to
// 9.1 as two launches; K = N = 2048 at rank 64 16 to 22 us.
constexpr int kAnyTokens = 8;
constexpr int kAnyThreads = 256;
constexpr int kFusedK = 256;
constexpr int kFusedRows = 256;

// 4 rows of A times 8 tokens over this warp's k: lane l gets the sum for row
// l / 8 and token l % 8 (a reduction that halves the values at every exchange: 31
// shuffles for the 32 sums).
template <typename T, typename X>
__device__ __forceinline__ float dots_4x8(const T* a, int K, int row, int rows, X x, int k, int step) {
  const int lane = threadIdx.x & 31;
  const T* ar[4];
#pragma unroll
  for (int m = 0; m < 4; ++m) ar[m] = a + (int64_t)min(row + m, rows - 1) * K;
  float v[32] = {};
#pragma unroll 2
  for (int i = k + lane; i < K; i += step) {
    float w[4], y[kAnyTokens];
#pragma unroll
    for (int m = 0; m < 4; ++m) w[m] = to_f(ar[m][i]);
#pragma unroll
    for (int t = 0; t < kAnyTokens; ++t) y[t] = x(t, i);
#pragma unroll
    for (int m = 0; m < 4; ++m)
#pragma unroll
      for (int t = 0; t < kAnyTokens; ++t) v[8 * m + t] = fmaf(y[t], w[m], v[8 * m + t]);
  }
#pragma unroll
  for (int h = 16; h > 0; h >>= 1)
#pragma unroll
    for (int i = 0; i < h; ++i) {
      const bool up = lane & h;
      v[i] = (up ? v[i + h] : v[i]) + __shfl_xor_sync(0xffffffffu, up ? v[i] : v[i + h], h);
    }
  return v[0];
}

template <typename T>
__global__ void __launch_bounds__(kAnyThreads)
    lora_shrink_any_kernel(const T* __restrict__ x, int64_t x_stride, const T* __restrict__ a, int K,
                           int ns, int width, ms_lora_adapters ad, ms_lora_plan plan,
                           float* __restrict__ s, int* err) {
  pdl_enter();
  __shared__ float s_part[kAnyThreads / 32][32];
  Tile tile;
  if (!load_tile(plan, ad, blockIdx.x, tile, err)) return;
  const int q0 = blockIdx.y * kAnyTokens, row = 4 * blockIdx.z, rows = ns * tile.rank;
  if (q0 >= tile.count || row >= rows) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const T* xr[kAnyTokens];
#pragma unroll
  for (int t = 0; t < kAnyTokens; ++t)
    xr[t] = x + (int64_t)max(token_at(plan, tile.start + min(q0 + t, tile.count - 1), err), 0) * x_stride;
  s_part[warp][lane] = dots_4x8(a + (int64_t)ns * tile.offset * K, K, row, rows,
                                [&](int t, int i) { return to_f(xr[t][i]); }, 32 * warp, kAnyThreads);
  __syncthreads();
  const int m = row + lane / kAnyTokens, q = q0 + lane % kAnyTokens;
  if (warp > 0 || m >= rows || q >= tile.count) return;
  float v = 0.f;
#pragma unroll
  for (int k = 0; k < kAnyThreads / 32; ++k) v += s_part[k][lane];
  s[((int64_t)tile.start + q) * width + m] = v * ad.scales[tile.adapter];
}

template <typename T, typename TO, bool FUSED>
__global__ void __launch_bounds__(kAnyThreads)
    lora_expand_any_kernel(const T* __restrict__ x, int64_t x_stride, const T* __restrict__ a, int K,
                           const T* __restrict__ b, TO* out, int swiglu, ExpandArgs p) {
  pdl_enter();
  extern __shared__ __align__(16) float s_any_mem[];
  float4* s_row = reinterpret_cast<float4*>(s_any_mem);           // per rank row: the 8 tokens' s
  float* s_x = s_any_mem + p.ns * p.ad.max_rank * kAnyTokens;     // FUSED: x, a row per token
  __shared__ int s_tok[kAnyTokens];
  Tile tile;
  if (!load_tile(p.plan, p.ad, blockIdx.x, tile, p.err)) return;
  const int q0 = blockIdx.y * kAnyTokens, count = min(tile.count - q0, kAnyTokens);
  if (count <= 0 || (p.in_place && tile.rank == 0)) return;
  if (threadIdx.x < kAnyTokens)
    s_tok[threadIdx.x] = threadIdx.x < count ? token_at(p.plan, tile.start + q0 + threadIdx.x, p.err) : -1;
  __syncthreads();
  const int o = blockIdx.z * kAnyThreads + threadIdx.x;
  const bool in = o < (swiglu ? p.N / 2 : p.N);
  const int n = swiglu ? (o >> 3) * 16 + (o & 7) : o;
  float base[kAnyTokens], up[kAnyTokens];
#pragma unroll
  for (int k = 0; k < kAnyTokens; ++k) {
    const float* row = p.base + max(s_tok[k], 0) * p.base_stride + n;
    const bool has = in && s_tok[k] >= 0;
    base[k] = has ? row[0] : 0.f;
    up[k] = has && swiglu ? row[8] : 0.f;
  }
  const int rows = p.ns * tile.rank;
  if constexpr (FUSED) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (rows > 0) {
      for (int k = warp; k < kAnyTokens; k += kAnyThreads / 32)
        for (int i = lane; i < K; i += 32)
          s_x[k * K + i] = s_tok[k] >= 0 ? to_f(x[s_tok[k] * x_stride + i]) : 0.f;
      __syncthreads();
    }
    for (int row = 4 * warp; row < rows; row += kAnyThreads / 8) {
      const float v = dots_4x8(a + (int64_t)p.ns * tile.offset * K, K, row, rows,
                               [&](int t, int i) { return s_x[t * K + i]; }, 0, 32);
      const int m = row + lane / kAnyTokens;
      if (m < rows) s_any_mem[m * kAnyTokens + lane % kAnyTokens] = v * p.ad.scales[tile.adapter];
    }
  } else {
    for (int i = threadIdx.x; i < kAnyTokens * rows; i += kAnyThreads) {
      const int k = i / rows, m = i - k * rows;
      s_any_mem[m * kAnyTokens + k] =
          k < count ? p.s_any[((int64_t)tile.start + q0 + k) * p.width_any + m] : 0.f;
    }
  }
  __syncthreads();
  if (!in) return;
  auto column = [&](int c, float (&y)[kAnyTokens]) {
    const float4* sj = s_row + 2 * slice_of(p, c) * tile.rank;
    const T* bn = b + (int64_t)tile.offset * p.N + c;
    float v[kAnyTokens] = {};
    for (int r0 = 0; r0 < tile.rank; r0 += 16) {  // 16 loads in flight
      float w[16];
#pragma unroll
      for (int r = 0; r < 16; ++r)
        w[r] = r0 + r < tile.rank ? to_f(bn[(int64_t)(r0 + r) * p.N]) : 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        if (r0 + r >= tile.rank) break;
        const float4 lo = sj[2 * (r0 + r)], hi = sj[2 * (r0 + r) + 1];
        v[0] = fmaf(lo.x, w[r], v[0]), v[1] = fmaf(lo.y, w[r], v[1]);
        v[2] = fmaf(lo.z, w[r], v[2]), v[3] = fmaf(lo.w, w[r], v[3]);
        v[4] = fmaf(hi.x, w[r], v[4]), v[5] = fmaf(hi.y, w[r], v[5]);
        v[6] = fmaf(hi.z, w[r], v[6]), v[7] = fmaf(hi.w, w[r], v[7]);
      }
    }
#pragma unroll
    for (int k = 0; k < kAnyTokens; ++k) y[k] += v[k];
  };
  column(n, base);
  if (swiglu) column(n + 8, up);
#pragma unroll
  for (int k = 0; k < kAnyTokens; ++k) {
    const int tok = s_tok[k];
    if (tok < 0) continue;
    const float y = swiglu ? base[k] / (1.f + expf(-base[k])) * up[k] : base[k];
    out[tok * p.out_stride + o] = from_f<TO>(y);
  }
}

constexpr int kMostSmem = 226 * 1024;

// CTAs of a cluster that share out k: as many as one round over the GPU takes (two
// a SM), at least 256 k values for each.  Sharing on into a second round costs:
// 256 tiles of 6 tokens, K = 14336, rank 16, 33.7 us by two CTAs and 28.9 by one;
// 64 tiles of 4, 22.5 us by eight and 15.9 by four.
int shrink_split(int n_tiles, int K, int rows, int mt) {
  const int64_t ctas = (int64_t)n_tiles * ceil_div(rows, 16 * mt);
  int split = 1;
  while (split < 8 && ctas * split <= 148 && K / (2 * split) >= 256) split *= 2;
  return split;
}

template <int EPI, int WM, int WN>
int launch_expand(ExpandArgs p, cudaStream_t s) {
  constexpr int terms = EPI == kLoraF32 ? 3 : 2, cols = 32 * WN;
  auto smem = [&]() {
    return 16 * WM * (p.ns * terms * p.rank_pm + kPad) * 2 +
           p.stages * (cols + kPad) * (16 * WM * 4 + p.rank_pm * 2);
  };
  // As deep a ring as two CTAs per SM allow, or one where two do not fit
  p.stages = 2;
  const int room = smem() > 112 * 1024 ? kMostSmem : 112 * 1024;
  while (p.stages < 4 && (++p.stages, smem() > room)) {
    --p.stages;
    break;
  }
  if constexpr (WM * WN > 2)
    if (smem() > kMostSmem) return launch_expand<EPI, 1, 2>(p, s);  // ranks of 128 and more
  static std::atomic<uint64_t> granted{0};
  MS_TRY(grant_dynamic_smem(lora_expand_kernel<EPI, WM, WN>, kMostSmem, granted));
  // Where tiles are short on average, a long one (the tokens of no adapter) would
  // take the longest: two CTAs share its tokens (256 tokens, 64 adapters, N = 2560:
  // 20.8 -> 15.4 us; four 16.8).
  // CTAs per tile: the number whose rounds over the GPU take the fewest steps,
  // a CTA's start counted as three
  const int resident = max(1, min(64 / (WM * WN), 227 * 1024 / (smem() + 1536)));
  const int slots = 148 * resident, steps = ceil_div(p.N, cols);
  int gx = 1;
  int64_t best = INT64_MAX;
  for (int n = 1; n <= min(steps, 64); ++n) {
    const int64_t cost = (int64_t)ceil_div(p.plan.n_tiles * n, slots) * (ceil_div(steps, n) + 3);
    if (cost < best) {
      best = cost;
      gx = n;
    }
  }
  launch_pdl(lora_expand_kernel<EPI, WM, WN>, dim3(gx, p.plan.n_tiles, WM == 1 ? 2 : 1), 32 * WM * WN, smem(), s, p);
  return check_launch("lora_expand_kernel");
}

// By the tiles' mean size, the padded rank and N.  1024 tokens at N = 28672 with
// the SwiGLU, first product of K = 512 included, in us, for 1 x 4 warps, 2 x 2 and
// tcgen05:      rank 16           rank 32           rank 64           rank 128
//   6 tokens    98  153  301      96  121  317      176  189  360     280  366  525
//  12           62   89  167      64   76  182      109  108  200     170  203  289
//  22           55   60   92      63   54   98      107   80  111     162  140  157
//  40           47   63   59      57   57   64       94   80   74     140  140  102
//  52           55   61   52      59   53   55       99   74   66     150  130   93
// N = 2560 to 11264 agree, but that tcgen05 at 40 tokens pays from rank x N on
// (rank 64: 24.3 to 23.0 us at 2560, 42.0 to 42.5 at 11264).
constexpr int kTcTokens = 48;
template <int EPI>
int dispatch_expand(const ExpandArgs& p, cudaStream_t s) {
  const int mean = p.plan.n_tokens / p.plan.n_tiles;
  const bool wide = (int64_t)p.rank_pm * p.N >= 64 * 8192;
  if (mean > (wide ? 32 : kTcTokens)) {
    const int rc = lora_expand_tc(p, EPI, s);
    if (rc != MS_ERR_UNSUPPORTED) return rc;
  }
  if (mean > 16 && p.rank_pm > 16) return launch_expand<EPI, 2, 2>(p, s);
  return launch_expand<EPI, 1, 4>(p, s);
}

template <int MT, int NT>
int launch_shrink(ShrinkArgs p, int rows, cudaStream_t s) {
  const int smem = kShrinkWarps * 16 * MT * 8 * NT * 4;
  const int split = shrink_split(p.plan.n_tiles, p.K, rows, MT);
  p.k_per = ceil_div(ceil_div(p.K, split), 32) * 32;
  return launch_cluster(lora_shrink_kernel<MT, NT>,
                        dim3(p.plan.n_tiles, ceil_div(rows, 16 * MT), split), kShrinkWarps * 32,
                        smem, split, s, p);
}

template <int RB>
int launch_shrink_tile(ShrinkArgs p, int rows, cudaStream_t s) {
  const int smem = kBigStages * (kTile + RB) * kBigLd * 2;
  static std::atomic<uint64_t> granted{0};
  MS_TRY(grant_dynamic_smem(lora_shrink_tile_kernel<RB>, smem, granted));
  const int blocks = ceil_div(rows, RB);
  int split = 1;
  while (split < 8 && (int64_t)p.plan.n_tiles * blocks * split <= 148 && p.K / (2 * split) >= 256)
    split *= 2;
  p.k_per = ceil_div(ceil_div(p.K, split), kBigK) * kBigK;
  return launch_cluster(lora_shrink_tile_kernel<RB>, dim3(p.plan.n_tiles, blocks, split), 256, smem,
                        split, s, p);
}

template <int NT>
int dispatch_shrink(const ShrinkArgs& p, int rows, cudaStream_t s) {
  return rows <= 16 ? launch_shrink<1, NT>(p, rows, s) : launch_shrink<2, NT>(p, rows, s);
}

// Little work (the comment at lora_one_kernel): one launch, and no workspace.
bool one_launch(const LoraCall& c, const ms_lora_plan& plan, int max_rank) {
  return c.n_slices == 1 && max_rank <= kOneRank && c.N <= kOneN && plan.n_tokens <= 32 &&
         plan.n_tokens <= kOneTokens * plan.n_tiles;
}

template <typename TO>
int launch_one(ShrinkArgs p, const ExpandArgs& e, cudaStream_t s) {
  p.k_per = ceil_div(ceil_div(p.K, kOneSplit), 32) * 32;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(p.plan.n_tiles, 1, kOneSplit);
  cfg.blockDim = kShrinkWarps * 32;
  cfg.stream = s;
  cudaLaunchAttribute attr[2]{};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim = {1, 1, kOneSplit};
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  (void)cudaLaunchKernelEx(&cfg, lora_one_kernel<TO>, p, e);
  return check_launch("lora_one_kernel");
}

// K and rank rows small enough for the second product's CTAs to make s: no workspace.
bool any_fused(const LoraCall& c, int max_rank) {
  return c.K <= kFusedK && c.n_slices * max_rank <= kFusedRows;
}

template <typename T, typename TO>
int launch_any(const LoraCall& c, const ExpandArgs& e, cudaStream_t s) {
  const int outs = c.swiglu ? c.N / 2 : c.N, rows = c.n_slices * e.ad.max_rank;
  const dim3 grid(e.plan.n_tiles, kTile / kAnyTokens, ceil_div(outs, kAnyThreads));
  const T *x = static_cast<const T*>(c.x), *a = static_cast<const T*>(c.a), *b = static_cast<const T*>(c.b);
  if (any_fused(c, e.ad.max_rank)) {
    launch_pdl(lora_expand_any_kernel<T, TO, true>, grid, kAnyThreads, (rows + c.K) * kAnyTokens * 4, s,
               x, c.x_stride, a, c.K, b, static_cast<TO*>(c.out), c.swiglu ? 1 : 0, e);
    return check_launch("lora_expand_any_kernel");
  }
  if (rows > 0) {
    launch_pdl(lora_shrink_any_kernel<T>,
               dim3(e.plan.n_tiles, kTile / kAnyTokens, ceil_div(rows, 4)), kAnyThreads, 0, s, x, c.x_stride, a, c.K,
               c.n_slices, e.width_any, e.ad, e.plan, const_cast<float*>(e.s_any), e.err);
    MS_TRY(check_launch("lora_shrink_any_kernel"));
  }
  launch_pdl(lora_expand_any_kernel<T, TO, false>, grid, kAnyThreads, rows * kAnyTokens * 4, s, x,
             c.x_stride, a, c.K, b, static_cast<TO*>(c.out), c.swiglu ? 1 : 0, e);
  return check_launch("lora_expand_any_kernel");
}

}  // namespace

// s: three bf16 terms of the padded rank per token and slice, or float32.
size_t lora_workspace_size(int n_tokens, int n_slices, int max_rank) {
  if (n_tokens <= 0 || n_slices <= 0 || max_rank <= 0) return 0;
  return (size_t)n_tokens * n_slices * ((max_rank + 15) & ~15) * 6;
}

int validate_lora(const ms_lora_adapters* ad, const ms_lora_plan* plan) {
  MS_REQUIRE(ad != nullptr && plan != nullptr, "lora: null adapters or plan");
  MS_REQUIRE(ad->n_adapters >= 0 && ad->total_rank >= 0 && ad->max_rank >= 0, "lora: bad adapter sizes");
  MS_REQUIRE(ad->max_rank <= kMaxRank, "lora: rank %d above %d", ad->max_rank, kMaxRank);
  MS_REQUIRE(ad->n_adapters == 0 || (ad->offsets && ad->ranks && ad->scales),
             "lora: null adapter arrays");
  MS_REQUIRE(plan->n_tokens >= 0 && plan->n_tiles >= 0, "lora: bad plan sizes");
  MS_REQUIRE(plan->n_tiles <= kMaxTiles, "lora: more than %d tiles", kMaxTiles);
  MS_REQUIRE(plan->n_tiles == 0 || (plan->order && plan->tiles), "lora: null plan arrays");
  MS_REQUIRE((reinterpret_cast<uintptr_t>(plan->tiles) & 15) == 0, "lora: tiles not 16-byte aligned");
  return MS_OK;
}

int lora_add(const LoraCall& c, const ms_lora_adapters& ad, const ms_lora_plan& plan,
             void* workspace, size_t workspace_bytes, cudaStream_t s) {
  if (plan.n_tiles == 0 || plan.n_tokens == 0) return MS_OK;
  auto aligned = [](const void* p, int n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; };
  const bool out_f32 = c.out_dtype == MS_DTYPE_F32;
  ExpandArgs e{};
  e.base = c.base;
  e.base_stride = c.base_stride;
  e.out = c.out;
  e.out_stride = c.out_stride;
  e.b = static_cast<const __nv_bfloat16*>(c.b);
  e.N = c.N;
  e.ns = c.n_slices;
  e.terms = out_f32 ? 3 : 2;
  for (int k = 0; k < 3; ++k) e.slice_end[k] = c.slice_end[k];
  e.interleaved = c.interleaved;
  e.in_place = static_cast<const void*>(c.base) == c.out;
  e.rank_pm = (ad.max_rank + 15) & ~15;
  e.s_stride = (int64_t)c.n_slices * e.terms * e.rank_pm;
  e.ad = ad;
  e.plan = plan;
  e.s = static_cast<const __nv_bfloat16*>(workspace);
  e.s_any = static_cast<const float*>(workspace);
  e.width_any = c.n_slices * ad.max_rank;
  e.err = device_error_word();
  // 16-byte loads and stores of x, A, B, the base and the result
  const bool tensor = c.dtype == MS_DTYPE_BF16 && c.K % 8 == 0 && c.x_stride % 8 == 0 &&
                      c.N % (c.swiglu ? 16 : 8) == 0 && aligned(c.x, 16) && aligned(c.a, 16) &&
                      aligned(c.b, 16) && aligned(c.base, 16) && c.base_stride % 4 == 0 &&
                      aligned(c.out, 16) && c.out_stride % (out_f32 ? 4 : 8) == 0 &&
                      !(c.swiglu && out_f32) &&
                      // 32-bit element offsets in the second product
                      plan.n_tokens * (c.base_stride > c.out_stride ? c.base_stride : c.out_stride) <=
                          (int64_t)UINT32_MAX;
  ShrinkArgs p{};
  p.x = static_cast<const __nv_bfloat16*>(c.x);
  p.x_stride = c.x_stride;
  p.a = static_cast<const __nv_bfloat16*>(c.a);
  p.K = c.K;
  p.ns = c.n_slices;
  p.terms = e.terms;
  p.s_stride = e.s_stride;
  p.ad = ad;
  p.plan = plan;
  p.s = static_cast<__nv_bfloat16*>(workspace);
  p.err = e.err;
  if (tensor && one_launch(c, plan, ad.max_rank))
    return out_f32 ? launch_one<float>(p, e, s) : launch_one<__nv_bfloat16>(p, e, s);
  const size_t need = !tensor && any_fused(c, ad.max_rank)
                          ? 0
                          : lora_workspace_size(plan.n_tokens, c.n_slices, ad.max_rank);
  if (workspace_bytes < need || (need > 0 && workspace == nullptr))
    return fail(MS_ERR_WORKSPACE, "lora: workspace too small (%zu < %zu)", workspace_bytes, need);
  MS_REQUIRE(need == 0 || aligned(workspace, 16), "lora: workspace not 16-byte aligned");
  if (!tensor) {
    if (c.dtype == MS_DTYPE_F32 && out_f32) return launch_any<float, float>(c, e, s);
    if (c.dtype == MS_DTYPE_F32) return launch_any<float, __nv_bfloat16>(c, e, s);
    if (out_f32) return launch_any<__nv_bfloat16, float>(c, e, s);
    return launch_any<__nv_bfloat16, __nv_bfloat16>(c, e, s);
  }
  if (ad.max_rank > 0) {
    e.after_shrink = 1;
    // Tokens at a time by the tiles' mean size.  1024 tokens, K = 4096, two slices, in us
    // (N = 128), for 8 and 16 tokens at a time and through shared memory, with one running
    // sum over k (partial sums take 0.9 to 1.0 of it for 8 and 16, 1.0 to 1.06 in shared
    // memory, 1.01 to 1.04 on tcgen05):
    //              rank 16           rank 64
    //   6 tokens   23   26   32      50   58   60
    //  12          26   20   22      50   40   38
    //  22          30   25   18      47   41   28
    //  40          27   21   14      55   43   22
    // Shared memory with 64 rank rows a CTA or 128: 26 or 32 (4096 tokens, rank 16),
    // 70 or 62 (8192, rank 64).  tcgen05 pays where tiles of one adapter follow one
    // another in pairs, as only prompts' do, and there are enough of them: runs of 512
    // tokens, rank 128, 50 us to 48 at 2048 tokens, 44 to 67 at 4096, 66 to 107 at
    // 8192; 8192 tokens of 128 adapters, rank 64, 74 to 63.
    const int rows = c.n_slices * e.rank_pm, mean = plan.n_tokens / plan.n_tiles;
    const bool long_runs = plan.n_tiles >= 64 && plan.n_tiles >= 2 * (ad.n_adapters + 1);
    if (mean <= 8)
      MS_TRY(dispatch_shrink<1>(p, rows, s));
    else if (mean <= 16)
      MS_TRY(dispatch_shrink<2>(p, rows, s));
    else if (mean > kTcTokens && long_runs)
      MS_TRY(lora_shrink_tc(p, rows, s));
    else if (rows <= 64)
      MS_TRY(launch_shrink_tile<64>(p, rows, s));
    else
      MS_TRY(launch_shrink_tile<128>(p, rows, s));
  }
  if (c.swiglu) return dispatch_expand<kLoraSwiGLU>(e, s);
  return out_f32 ? dispatch_expand<kLoraF32>(e, s) : dispatch_expand<kLoraBf16>(e, s);
}

}  // namespace ms

using namespace ms;

extern "C" size_t ms_lora_workspace_size(const ms_lora_adapters* adapters,
                                         const ms_lora_plan* plan, int n_slices) {
  if (adapters == nullptr || plan == nullptr) return 0;
  return lora_workspace_size(plan->n_tokens, n_slices, adapters->max_rank);
}

extern "C" int ms_lora_add(const void* x, int64_t x_stride, const float* base, int64_t base_stride,
                           void* out, int64_t out_stride, const void* a, const void* b, int K,
                           int N, int n_slices, const int32_t* slice_cols, int interleaved,
                           int swiglu, const ms_lora_adapters* adapters, const ms_lora_plan* plan,
                           int dtype, int out_dtype, void* workspace, size_t workspace_bytes,
                           void* stream) {
  MS_TRY(validate_lora(adapters, plan));
  MS_REQUIRE(K > 0 && N > 0 && n_slices >= 1 && n_slices <= 4, "ms_lora_add: bad sizes K=%d N=%d (%d slices)",
             K, N, n_slices);
  MS_REQUIRE((dtype == MS_DTYPE_F32 || dtype == MS_DTYPE_BF16) &&
                 (out_dtype == MS_DTYPE_F32 || out_dtype == MS_DTYPE_BF16),
             "ms_lora_add: dtypes %d -> %d", dtype, out_dtype);
  MS_REQUIRE(!interleaved || (n_slices == 2 && N % 16 == 0),
             "ms_lora_add: interleaved columns are two slices of N %% 16 == 0 columns");
  MS_REQUIRE(!swiglu || interleaved, "ms_lora_add: SwiGLU needs interleaved gate/up columns");
  LoraCall c{};
  if (!interleaved && n_slices > 1) {
    MS_REQUIRE(slice_cols != nullptr, "ms_lora_add: null slice_cols");
    int end = 0;
    for (int k = 0; k < n_slices; ++k) {
      MS_REQUIRE(slice_cols[k] > 0, "ms_lora_add: slice %d has %d columns", k, slice_cols[k]);
      end += slice_cols[k];
      if (k < 3) c.slice_end[k] = end;
    }
    MS_REQUIRE(end == N, "ms_lora_add: slices of %d columns in all, N = %d", end, N);
  }
  if (plan->n_tokens == 0 || plan->n_tiles == 0) return MS_OK;
  MS_REQUIRE(x && base && out, "ms_lora_add: null pointer");
  MS_REQUIRE(adapters->total_rank == 0 || (a && b), "ms_lora_add: null adapter weights");
  const int outs = swiglu ? N / 2 : N;
  MS_REQUIRE(x_stride >= K && base_stride >= N && out_stride >= outs, "ms_lora_add: row stride too small");
  const bool in_place = static_cast<const void*>(base) == out;
  MS_REQUIRE(!in_place || (out_dtype == MS_DTYPE_F32 && !swiglu && base_stride == out_stride),
             "ms_lora_add: only a float32 sum can go back into the base");
  if (!in_place) {
    const char* b0 = reinterpret_cast<const char*>(base);
    const char* b1 = b0 + 4 * ((int64_t)(plan->n_tokens - 1) * base_stride + N);
    const char* o0 = static_cast<const char*>(out);
    const char* o1 = o0 + (out_dtype == MS_DTYPE_F32 ? 4 : 2) *
                              ((int64_t)(plan->n_tokens - 1) * out_stride + outs);
    MS_REQUIRE(o1 <= b0 || b1 <= o0, "ms_lora_add: base and out overlap");
  }
  {
    const char* x0 = static_cast<const char*>(x);
    const char* x1 = x0 + (dtype == MS_DTYPE_F32 ? 4 : 2) *
                              ((int64_t)(plan->n_tokens - 1) * x_stride + K);
    const char* o0 = static_cast<const char*>(out);
    const char* o1 = o0 + (out_dtype == MS_DTYPE_F32 ? 4 : 2) *
                              ((int64_t)(plan->n_tokens - 1) * out_stride + outs);
    MS_REQUIRE(o1 <= x0 || x1 <= o0, "ms_lora_add: x and out overlap");
  }
  c.x = x;
  c.x_stride = x_stride;
  c.base = base;
  c.base_stride = base_stride;
  c.out = out;
  c.out_stride = out_stride;
  c.a = a;
  c.b = b;
  c.K = K;
  c.N = N;
  c.n_slices = n_slices;
  c.interleaved = interleaved != 0;
  c.swiglu = swiglu != 0;
  c.dtype = dtype;
  c.out_dtype = out_dtype;
  return lora_add(c, *adapters, *plan, workspace, workspace_bytes, as_stream(stream));
}
