// Low-rank adapters of many requests at once beside a shared projection:
//   s_j[t]   = A_{a(t), j} x[t]                        (first product, rank r)
//   y[t, n]  = base[t, n] + scale_a * sum_r B_{a(t)}[r, n] s_{j(n)}[t, r]
// for every token t of the batch, where a(t) is the token's adapter, j(n) the
// fused slice of column n (q | k | v, gate | up) and base the projection's
// float32 output.  Optionally y goes through the SwiGLU of the interleaved
// gate/up columns and out in the model's type.
//
// The plan lists tiles of up to 64 tokens that share an adapter (adapter -1:
// none).  Two launches: lora_shrink computes s (float32, K split over CTAs as
// needed, the parts summed by the reader in a fixed order, so results do not
// depend on timing), lora_expand adds B s to the base.
//
// s stays float32 between the launches; the bf16 second product takes it as
// hi + lo, both bf16 (hi = s rounded, lo = the rest rounded: s to about
// 2^-17), because a single bf16 s would put 2^-9 of the adapter's part into
// a float32 output.
#include <cmath>

#include "lora.cuh"

namespace ms {
namespace {

constexpr int kTile = MS_LORA_TILE;  // most tokens of a tile
constexpr int kMaxRank = MS_LORA_MAX_RANK;

struct Tile {
  int start, count, adapter, rank, offset;
};

// Tile `i` of the plan with its adapter's rank and offset, every index checked:
// false (and the device error word) when one is out of range.
__device__ __forceinline__ bool load_tile(const ms_lora_plan& p, const ms_lora_adapters& ad, int i,
                                          Tile& t, int* err) {
  const int4 q = reinterpret_cast<const int4*>(p.tiles)[i];
  t.start = q.x;
  t.count = q.y;
  t.adapter = q.z;
  t.rank = 0;
  t.offset = 0;
  bool ok = t.start >= 0 && t.count >= 0 && t.count <= kTile && t.start <= p.n_tokens - t.count &&
            t.adapter < ad.n_adapters;
  if (ok && t.adapter >= 0) {
    t.rank = ad.ranks[t.adapter];
    t.offset = ad.offsets[t.adapter];
    ok = t.rank >= 0 && t.rank <= ad.max_rank && t.offset >= 0 &&
         t.offset <= ad.total_rank - t.rank;
  }
  if (!ok) {
    if (threadIdx.x == 0) raise_device_error(err, kErrAdapter);
    t.count = 0;
  }
  return ok;
}

// The token (row of x and out) at sorted position `pos`, or -1 (and the error word).
__device__ __forceinline__ int token_at(const ms_lora_plan& p, int pos, int* err) {
  const int t = p.order[pos];
  if (t >= 0 && t < p.n_tokens) return t;
  raise_device_error(err, kErrAdapter);
  return -1;
}

__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t s_addr(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
  const int n = valid ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n)
               : "memory");
}
__device__ __forceinline__ void cp_wait_all() {
  asm volatile("cp.async.wait_all;" ::: "memory");
}

// ---- first product, bf16 ------------------------------------------------------
// mma m16n8k16 with the rank rows of A as M and the tokens as N (8 of them:
// small groups waste less than with 16).  Both operands come straight from
// global memory: the sum over k may take its terms in any order, so lane
// (g, t) of a fragment takes the 16 bytes k0 + 8t .. 8t+7 of its row for two
// MMAs at once, instead of the four separate pairs of the nominal layout.
// A CTA takes 16 * MT rank rows x 32 tokens; its 8 warps share out k.
constexpr int kShrinkWarps = 8;
constexpr int kShrinkNT = 4;
constexpr int kShrinkTokens = 8 * kShrinkNT;

struct ShrinkArgs {
  const __nv_bfloat16* x;
  int64_t x_stride;
  const __nv_bfloat16* a;
  int K, ns, width, k_split, k_per;  // k_per: k values per split, a multiple of 32
  ms_lora_adapters ad;
  ms_lora_plan plan;
  float* s;  // (k_split, n_tokens, width)
  int* err;
};

template <int MT>
__global__ void __launch_bounds__(kShrinkWarps * 32) lora_shrink_kernel(ShrinkArgs p) {
  pdl_enter();
  extern __shared__ __align__(16) float s_red[];  // [warps][16 MT][kShrinkTokens]
  constexpr int kHalves = kTile / kShrinkTokens;
  Tile tile;
  if (!load_tile(p.plan, p.ad, blockIdx.x / kHalves, tile, p.err)) return;
  const int first = (blockIdx.x % kHalves) * kShrinkTokens;  // of this CTA's tokens in the tile
  const int rows = p.ns * tile.rank, m0 = blockIdx.y * 16 * MT;
  const int count = min(tile.count - first, kShrinkTokens);
  if (count <= 0 || m0 >= rows) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;

  const __nv_bfloat16* xr[kShrinkNT];
#pragma unroll
  for (int n = 0; n < kShrinkNT; ++n) {
    const int tok = token_at(p.plan, tile.start + first + min(8 * n + g, count - 1), p.err);
    xr[n] = p.x + (int64_t)max(tok, 0) * p.x_stride + 8 * t;
  }
  const __nv_bfloat16* ar[MT][2];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = min(m0 + 16 * m + 8 * h + g, rows - 1);
      ar[m][h] = p.a + ((int64_t)p.ns * tile.offset + row) * p.K + 8 * t;
    }
  float acc[MT][kShrinkNT][4] = {};
  const int k_end = min(p.K, (int)(blockIdx.z + 1) * p.k_per);
  const uint4 zero = make_uint4(0, 0, 0, 0);
#pragma unroll 2
  for (int k0 = blockIdx.z * p.k_per + 32 * warp; k0 < k_end; k0 += 32 * kShrinkWarps) {
    const bool in = k0 + 8 * t < k_end;
    uint4 xv[kShrinkNT], av[MT][2];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        av[m][h] = in ? __ldg(reinterpret_cast<const uint4*>(ar[m][h] + k0)) : zero;
#pragma unroll
    for (int n = 0; n < kShrinkNT; ++n)
      xv[n] = in && 8 * n < count ? __ldg(reinterpret_cast<const uint4*>(xr[n] + k0)) : zero;
#pragma unroll
    for (int n = 0; n < kShrinkNT; ++n) {
      if (8 * n >= count) break;
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        mma_bf16(acc[m][n], av[m][0].x, av[m][1].x, av[m][0].y, av[m][1].y, xv[n].x, xv[n].y);
        mma_bf16(acc[m][n], av[m][0].z, av[m][1].z, av[m][0].w, av[m][1].w, xv[n].z, xv[n].w);
      }
    }
  }
  // the warps' parts, summed in warp order
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int n = 0; n < kShrinkNT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int row = 16 * m + g + 8 * (e >> 1), col = 8 * n + 2 * t + (e & 1);
        s_red[(warp * kShrinkTokens + col) * (16 * MT) + row] = acc[m][n][e];
      }
  __syncthreads();
  float* out = p.s + ((int64_t)blockIdx.z * p.plan.n_tokens + tile.start + first) * p.width;
  const int here = min(16 * MT, rows - m0);
  for (int i = threadIdx.x; i < count * 16 * MT; i += kShrinkWarps * 32) {
    const int col = i / (16 * MT), row = i % (16 * MT);
    if (row >= here) continue;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < kShrinkWarps; ++w) v += s_red[(w * kShrinkTokens) * (16 * MT) + i];
    out[(int64_t)col * p.width + m0 + row] = v;
  }
}

// ---- second product, bf16 -----------------------------------------------------
// A CTA of 4 warps: up to 64 tokens of a tile x 128 columns (32 per warp).
// mma m16n8k16 with tokens as M, columns as N, the rank as K: s (hi, lo) and
// the adapter's B rows in shared memory, the base read into registers while
// the MMAs run.
constexpr int kExpWarps = 4;
constexpr int kExpCols = 32 * kExpWarps;
constexpr int kBLd = kExpCols + 8;  // padded row (elements): conflict-free ldmatrix

struct ExpandArgs {
  const float* base;
  int64_t base_stride;
  void* out;
  int64_t out_stride;
  const __nv_bfloat16* b;
  int N, ns, width, k_split;
  int slice_end[3];
  int interleaved, in_place, after_shrink;
  int tm;  // tokens per pass (16, 32 or 64)
  ms_lora_adapters ad;
  ms_lora_plan plan;
  const float* s;
  int* err;
};

__device__ __forceinline__ int slice_of(const ExpandArgs& p, int n) {
  if (p.interleaved) return (n >> 3) & 1;
  int j = 0;
#pragma unroll
  for (int k = 0; k < 3; ++k) j += k < p.ns - 1 && n >= p.slice_end[k];
  return j;
}

enum LoraEpilogue { kLoraF32, kLoraBf16, kLoraSwiGLU };

__device__ __forceinline__ float silu(float x) { return __fdividef(x, 1.f + __expf(-x)); }

template <int EPI>
__global__ void __launch_bounds__(kExpWarps * 32) lora_expand_kernel(ExpandArgs p) {
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ int s_tok[kTile];
  Tile tile;
  // The plan and the adapters are read before the launch wait when
  // lora_shrink runs directly before: it does not write them, and everything
  // before it has completed once its blocks allow this kernel to start.
  if (!p.after_shrink) pdl_enter();
  const bool ok = load_tile(p.plan, p.ad, blockIdx.y, tile, p.err);
  const int n0 = blockIdx.x * kExpCols;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int rank_p = (tile.rank + 15) & ~15;
  const int j0 = p.interleaved ? 0 : slice_of(p, n0);
  const int j1 = p.interleaved ? 1 : slice_of(p, min(n0 + kExpCols, p.N) - 1);
  const int s_ld = (j1 - j0 + 1) * rank_p + 8;
  __nv_bfloat16* s_b = reinterpret_cast<__nv_bfloat16*>(smem);  // [rank_p][kBLd]
  __nv_bfloat16* s_hi = s_b + rank_p * kBLd;                    // [tm][s_ld]
  __nv_bfloat16* s_lo = s_hi + p.tm * s_ld;
  const bool work = ok && tile.count > 0 && !(p.in_place && tile.rank == 0);
  if (work) {
    for (int i = threadIdx.x; i < rank_p * (kExpCols / 8); i += kExpWarps * 32) {
      const int r = i / (kExpCols / 8), c = 8 * (i % (kExpCols / 8));
      const bool in = r < tile.rank && n0 + c < p.N;
      cp_async16(s_addr(s_b + r * kBLd + c),
                 p.b + (in ? ((int64_t)tile.offset + r) * p.N + n0 + c : 0), in);
    }
    if (threadIdx.x < kTile)
      s_tok[threadIdx.x] =
          threadIdx.x < tile.count ? token_at(p.plan, tile.start + threadIdx.x, p.err) : -1;
  }
  if (p.after_shrink) pdl_enter();
  if (!work) return;
  const float scale = tile.rank > 0 ? p.ad.scales[tile.adapter] : 0.f;
  const int64_t split_stride = (int64_t)p.plan.n_tokens * p.width;
  for (int p0 = 0; p0 < tile.count; p0 += p.tm) {
    const int here = min(p.tm, tile.count - p0);
    const int rows_p = (here + 15) & ~15;
    __syncthreads();  // the previous pass has read s
    const int cols = (j1 - j0 + 1) * rank_p;
    for (int i = threadIdx.x; i < rows_p * cols; i += kExpWarps * 32) {
      const int row = i / cols, c = i - row * cols;
      const int j = c / rank_p, r = c - j * rank_p;
      float v = 0.f;
      if (row < here && r < tile.rank) {
        const float* src = p.s + ((int64_t)tile.start + p0 + row) * p.width +
                           (j0 + j) * tile.rank + r;
        for (int k = 0; k < p.k_split; ++k) v += src[k * split_stride];
        v *= scale;
      }
      const __nv_bfloat16 hi = __float2bfloat16_rn(v);
      s_hi[row * s_ld + c] = hi;
      s_lo[row * s_ld + c] = __float2bfloat16_rn(v - __bfloat162float(hi));
    }
    cp_wait_all();
    __syncthreads();
    const int wc = n0 + 32 * warp;  // this warp's first column
    if (wc >= p.N) continue;
    for (int m = 0; m < rows_p; m += 16) {
      int64_t row_at[2];
      bool has[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int tok = m + g + 8 * h < here ? s_tok[p0 + m + g + 8 * h] : -1;
        has[h] = tok >= 0;
        row_at[h] = max(tok, 0);
      }
      float acc[4][4];
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int c = wc + 8 * n + 2 * t;
          float2 v = make_float2(0.f, 0.f);
          if (has[h] && c < p.N)
            v = *reinterpret_cast<const float2*>(p.base + row_at[h] * p.base_stride + c);
          acc[n][2 * h] = v.x;
          acc[n][2 * h + 1] = v.y;
        }
      int slice[4];
#pragma unroll
      for (int n = 0; n < 4; ++n) slice[n] = slice_of(p, min(wc + 8 * n, p.N - 1));
      for (int j = slice[0]; j <= max(slice[1], slice[3]); ++j) {
        for (int k = 0; k < rank_p; k += 16) {
          uint32_t hi[4], lo[4], b01[4], b23[4];
          const int srow = (m + (lane & 15)) * s_ld + (j - j0) * rank_p + k + 8 * (lane >> 4);
          ldsm4(hi, s_addr(s_hi + srow));
          ldsm4(lo, s_addr(s_lo + srow));
          const int brow = (k + (lane & 15)) * kBLd + 32 * warp + 8 * (lane >> 4);
          ldsm4_t(b01, s_addr(s_b + brow));
          ldsm4_t(b23, s_addr(s_b + brow + 16));
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            if (slice[n] != j) continue;
            const uint32_t w0 = n < 2 ? b01[2 * n] : b23[2 * n - 4];
            const uint32_t w1 = n < 2 ? b01[2 * n + 1] : b23[2 * n - 3];
            mma_bf16(acc[n], lo[0], lo[1], lo[2], lo[3], w0, w1);
            mma_bf16(acc[n], hi[0], hi[1], hi[2], hi[3], w0, w1);
          }
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (!has[h]) continue;
        if constexpr (EPI == kLoraSwiGLU) {
          __nv_bfloat16* o = static_cast<__nv_bfloat16*>(p.out) + row_at[h] * p.out_stride;
#pragma unroll
          for (int n = 0; n < 4; n += 2) {
            const int c = (wc + 8 * n) / 2 + 2 * t;  // 8 outputs per 16 columns
            if (wc + 8 * n < p.N)
              *reinterpret_cast<__nv_bfloat162*>(o + c) =
                  __floats2bfloat162_rn(silu(acc[n][2 * h]) * acc[n + 1][2 * h],
                                        silu(acc[n][2 * h + 1]) * acc[n + 1][2 * h + 1]);
          }
        } else {
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            const int c = wc + 8 * n + 2 * t;
            if (c >= p.N) continue;
            const float2 v = make_float2(acc[n][2 * h], acc[n][2 * h + 1]);
            if constexpr (EPI == kLoraF32)
              *reinterpret_cast<float2*>(static_cast<float*>(p.out) + row_at[h] * p.out_stride + c) = v;
            else
              *reinterpret_cast<__nv_bfloat162*>(static_cast<__nv_bfloat16*>(p.out) +
                                                 row_at[h] * p.out_stride + c) =
                  __floats2bfloat162_rn(v.x, v.y);
          }
        }
      }
    }
  }
}

// ---- any type, size and alignment ----------------------------------------------
// The float32 models and shapes the tensor-core kernels do not take: one warp
// per (token, rank row) dot product, one thread per output.
template <typename T>
__global__ void lora_shrink_any_kernel(const T* __restrict__ x, int64_t x_stride,
                                       const T* __restrict__ a, int K, int ns, int width,
                                       ms_lora_adapters ad, ms_lora_plan plan,
                                       float* __restrict__ s, int* err) {
  pdl_enter();
  Tile tile;
  if (!load_tile(plan, ad, blockIdx.x, tile, err)) return;
  const int lane = threadIdx.x & 31, nw = blockDim.x >> 5;
  const int rows = ns * tile.rank, work = tile.count * rows;
  for (int i = blockIdx.y * nw + (threadIdx.x >> 5); i < work; i += gridDim.y * nw) {
    const int q = i / rows, m = i - q * rows;
    const int tok = token_at(plan, tile.start + q, err);
    const T* xr = x + (int64_t)max(tok, 0) * x_stride;
    const T* ar = a + ((int64_t)ns * tile.offset + m) * K;
    float v = 0.f;
    for (int k = lane; k < K; k += 32) v = fmaf(to_f(xr[k]), to_f(ar[k]), v);
    v = warp_sum(v);
    if (lane == 0) s[((int64_t)tile.start + q) * width + m] = v;
  }
}

template <typename T, typename TO>
__global__ void lora_expand_any_kernel(const float* base, int64_t base_stride, TO* out,
                                       int64_t out_stride, const T* __restrict__ b, int swiglu,
                                       ExpandArgs p) {
  pdl_enter();
  Tile tile;
  if (!load_tile(p.plan, p.ad, blockIdx.x, tile, p.err)) return;
  if (p.in_place && tile.rank == 0) return;
  const float scale = tile.rank > 0 ? p.ad.scales[tile.adapter] : 0.f;
  const int outs = swiglu ? p.N / 2 : p.N;
  for (int64_t i = (int64_t)blockIdx.y * blockDim.x + threadIdx.x; i < (int64_t)tile.count * outs;
       i += (int64_t)gridDim.y * blockDim.x) {
    const int q = (int)(i / outs), o = (int)(i - (int64_t)q * outs);
    const int tok = token_at(p.plan, tile.start + q, p.err);
    if (tok < 0) continue;
    const float* sr = p.s + ((int64_t)tile.start + q) * p.width;
    auto column = [&](int n) {
      const float* sj = sr + slice_of(p, n) * tile.rank;
      float v = 0.f;
      for (int r = 0; r < tile.rank; ++r)
        v = fmaf(sj[r], to_f(b[((int64_t)tile.offset + r) * p.N + n]), v);
      return fmaf(scale, v, base[(int64_t)tok * base_stride + n]);
    };
    float y;
    if (swiglu) {
      const int n = (o >> 3) * 16 + (o & 7);
      const float gate = column(n);
      y = gate / (1.f + expf(-gate)) * column(n + 8);
    } else {
      y = column(o);
    }
    out[(int64_t)tok * out_stride + o] = from_f<TO>(y);
  }
}

// Number of parts k is cut into: enough CTAs for the GPU, at least 256 k values per CTA.
int shrink_split(int n_tiles, int K, int n_slices, int max_rank) {
  const int rows = n_slices * max_rank;
  const int mt = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
  const int64_t ctas = (int64_t)n_tiles * ceil_div(rows, 16 * mt);
  int split = 1;
  while (split < 16 && ctas * split < 2 * 148 && K / (2 * split) >= 256) split *= 2;
  return split;
}

constexpr int kMostSmem = 226 * 1024;

template <int EPI>
int launch_expand(const ExpandArgs& p, int smem, cudaStream_t s) {
  static std::atomic<uint64_t> granted{0};
  if (smem > 48 * 1024) MS_TRY(grant_dynamic_smem(lora_expand_kernel<EPI>, kMostSmem, granted));
  const dim3 grid(ceil_div(p.N, kExpCols), p.plan.n_tiles);
  launch_pdl(lora_expand_kernel<EPI>, grid, kExpWarps * 32, smem, s, p);
  return check_launch("lora_expand_kernel");
}

template <int MT>
int launch_shrink(const ShrinkArgs& p, int row_blocks, cudaStream_t s) {
  const int smem = kShrinkWarps * 16 * MT * kShrinkTokens * 4;
  static std::atomic<uint64_t> granted{0};
  if (smem > 48 * 1024) MS_TRY(grant_dynamic_smem(lora_shrink_kernel<MT>, smem, granted));
  const dim3 grid(p.plan.n_tiles * (kTile / kShrinkTokens), row_blocks, p.k_split);
  launch_pdl(lora_shrink_kernel<MT>, grid, kShrinkWarps * 32, smem, s, p);
  return check_launch("lora_shrink_kernel");
}

template <typename T, typename TO>
int launch_any(const LoraCall& c, const ExpandArgs& e, cudaStream_t s) {
  const int per = c.n_slices * e.ad.max_rank;
  const dim3 g1(e.plan.n_tiles, min(64, max(1, ceil_div(kTile * per, 64))));
  launch_pdl(lora_shrink_any_kernel<T>, g1, 256, 0, s, static_cast<const T*>(c.x), c.x_stride,
             static_cast<const T*>(c.a), c.K, c.n_slices, e.width, e.ad, e.plan,
             const_cast<float*>(e.s), e.err);
  MS_TRY(check_launch("lora_shrink_any_kernel"));
  const int outs = c.swiglu ? c.N / 2 : c.N;
  const dim3 g2(e.plan.n_tiles, (int)min((int64_t)256, ((int64_t)kTile * outs + 1023) / 1024));
  launch_pdl(lora_expand_any_kernel<T, TO>, g2, 256, 0, s, c.base, c.base_stride,
             static_cast<TO*>(c.out), c.out_stride, static_cast<const T*>(c.b), c.swiglu ? 1 : 0, e);
  return check_launch("lora_expand_any_kernel");
}

}  // namespace

size_t lora_workspace_size(int n_tokens, int n_tiles, int K, int n_slices, int max_rank) {
  if (n_tokens <= 0 || n_tiles <= 0 || K <= 0 || n_slices <= 0 || max_rank <= 0) return 0;
  return (size_t)shrink_split(n_tiles, K, n_slices, max_rank) * n_tokens * n_slices * max_rank * 4;
}

int validate_lora(const ms_lora_adapters* ad, const ms_lora_plan* plan) {
  MS_REQUIRE(ad != nullptr && plan != nullptr, "lora: null adapters or plan");
  MS_REQUIRE(ad->n_adapters >= 0 && ad->total_rank >= 0 && ad->max_rank >= 0, "lora: bad adapter sizes");
  MS_REQUIRE(ad->max_rank <= kMaxRank, "lora: rank %d above %d", ad->max_rank, kMaxRank);
  MS_REQUIRE(ad->n_adapters == 0 || (ad->offsets && ad->ranks && ad->scales),
             "lora: null adapter arrays");
  MS_REQUIRE(plan->n_tokens >= 0 && plan->n_tiles >= 0, "lora: bad plan sizes");
  MS_REQUIRE(plan->n_tiles <= 65535, "lora: more than 65535 tiles");
  MS_REQUIRE(plan->n_tiles == 0 || (plan->order && plan->tiles), "lora: null plan arrays");
  MS_REQUIRE((reinterpret_cast<uintptr_t>(plan->tiles) & 15) == 0, "lora: tiles not 16-byte aligned");
  return MS_OK;
}

int lora_add(const LoraCall& c, const ms_lora_adapters& ad, const ms_lora_plan& plan,
             void* workspace, size_t workspace_bytes, cudaStream_t s) {
  if (plan.n_tiles == 0 || plan.n_tokens == 0) return MS_OK;
  const bool in_place = static_cast<const void*>(c.base) == c.out;
  const size_t need = lora_workspace_size(plan.n_tokens, plan.n_tiles, c.K, c.n_slices, ad.max_rank);
  if (workspace_bytes < need || (need > 0 && workspace == nullptr))
    return fail(MS_ERR_INVALID, "lora: workspace too small (%zu < %zu)", workspace_bytes, need);
  ExpandArgs e{};
  e.base = c.base;
  e.base_stride = c.base_stride;
  e.out = c.out;
  e.out_stride = c.out_stride;
  e.b = static_cast<const __nv_bfloat16*>(c.b);
  e.N = c.N;
  e.ns = c.n_slices;
  e.width = c.n_slices * ad.max_rank;
  e.k_split = 1;
  for (int k = 0; k < 3; ++k) e.slice_end[k] = c.slice_end[k];
  e.interleaved = c.interleaved;
  e.in_place = in_place;
  e.ad = ad;
  e.plan = plan;
  e.s = static_cast<float*>(workspace);
  e.err = device_error_word();
  auto aligned = [](const void* p, int n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; };
  bool slices8 = true;
  for (int k = 0; k + 1 < c.n_slices && !c.interleaved; ++k) slices8 &= c.slice_end[k] % 8 == 0;
  const bool tensor =
      c.dtype == MS_DTYPE_BF16 && c.K % 8 == 0 && c.x_stride % 8 == 0 && c.N % 8 == 0 && slices8 &&
      aligned(c.x, 16) && aligned(c.a, 16) && aligned(c.b, 16) && aligned(c.base, 8) &&
      c.base_stride % 2 == 0 && aligned(c.out, 8) && c.out_stride % 2 == 0 &&
      !(c.swiglu && c.out_dtype != MS_DTYPE_BF16);
  if (!tensor) {
    if (c.dtype == MS_DTYPE_F32 && c.out_dtype == MS_DTYPE_F32) return launch_any<float, float>(c, e, s);
    if (c.dtype == MS_DTYPE_F32) return launch_any<float, __nv_bfloat16>(c, e, s);
    if (c.out_dtype == MS_DTYPE_F32) return launch_any<__nv_bfloat16, float>(c, e, s);
    return launch_any<__nv_bfloat16, __nv_bfloat16>(c, e, s);
  }
  if (ad.max_rank > 0) {
    ShrinkArgs p{};
    p.x = static_cast<const __nv_bfloat16*>(c.x);
    p.x_stride = c.x_stride;
    p.a = static_cast<const __nv_bfloat16*>(c.a);
    p.K = c.K;
    p.ns = c.n_slices;
    p.width = e.width;
    p.k_split = shrink_split(plan.n_tiles, c.K, c.n_slices, ad.max_rank);
    p.k_per = ceil_div(ceil_div(c.K, p.k_split), 32) * 32;
    p.ad = ad;
    p.plan = plan;
    p.s = static_cast<float*>(workspace);
    p.err = e.err;
    e.k_split = p.k_split;
    e.after_shrink = 1;
    const int rows = e.width;
    if (rows <= 16)
      MS_TRY(launch_shrink<1>(p, 1, s));
    else if (rows <= 32)
      MS_TRY(launch_shrink<2>(p, 1, s));
    else
      MS_TRY(launch_shrink<4>(p, ceil_div(rows, 64), s));
  }
  const int rank_p = (ad.max_rank + 15) & ~15;
  const int s_ld = c.n_slices * rank_p + 8;
  e.tm = 64;
  auto smem = [&]() { return rank_p * kBLd * 2 + e.tm * s_ld * 4; };
  while (e.tm > 16 && smem() > 100 * 1024) e.tm /= 2;
  if (c.swiglu) return launch_expand<kLoraSwiGLU>(e, smem(), s);
  if (c.out_dtype == MS_DTYPE_F32) return launch_expand<kLoraF32>(e, smem(), s);
  return launch_expand<kLoraBf16>(e, smem(), s);
}

}  // namespace ms

using namespace ms;

extern "C" size_t ms_lora_workspace_size(const ms_lora_adapters* adapters,
                                         const ms_lora_plan* plan, int K, int n_slices) {
  if (adapters == nullptr || plan == nullptr) return 0;
  return lora_workspace_size(plan->n_tokens, plan->n_tiles, K, n_slices, adapters->max_rank);
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
