// What the adapter kernels share (lora.cu, lora_tc.cu): the plan's tiles, the
// second product's arguments and epilogues, and small PTX helpers.
#pragma once
#include <cmath>

#include "lora.cuh"

namespace ms {

struct ShrinkArgs {
  const __nv_bfloat16* x;
  int64_t x_stride;
  const __nv_bfloat16* a;
  int K, ns, k_per;  // k_per: k values per CTA of a cluster, a multiple of 32
  int terms;
  int64_t s_stride;  // row stride of s (elements)
  ms_lora_adapters ad;
  ms_lora_plan plan;
  __nv_bfloat16* s;  // row per position: [slice][term][rank_p]
  int* err;
};

enum LoraEpilogue { kLoraF32, kLoraBf16, kLoraSwiGLU };

struct ExpandArgs {
  const float* base;
  int64_t base_stride;
  void* out;
  int64_t out_stride;
  const __nv_bfloat16* b;
  int N, ns, terms;
  int slice_end[3];
  int interleaved, in_place, after_shrink;
  int stages;  // steps in the ring (2 to 4)
  int rank_pm;     // padded largest rank: buffer sizes
  int64_t s_stride;
  ms_lora_adapters ad;
  ms_lora_plan plan;
  const __nv_bfloat16* s;
  const float* s_any;  // any-shape kernels: float32 s, one row per position
  int width_any;
  int* err;
};

namespace {

constexpr int kTile = MS_LORA_TILE;  // most tokens of a tile
constexpr int kMaxRank = MS_LORA_MAX_RANK;
constexpr int kMaxTiles = 65535;  // the second product's grid

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
// c = the product alone (an accumulator of zero).
__device__ __forceinline__ void mma_bf16_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                               uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%10,%10,%10,%10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
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
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ int pad16(int r) { return (r + 15) & ~15; }

__device__ __forceinline__ int slice_of(const ExpandArgs& p, int n) {
  if (p.interleaved) return (n >> 3) & 1;
  int j = 0;
#pragma unroll
  for (int k = 0; k < 3; ++k) j += k < p.ns - 1 && n >= p.slice_end[k];
  return j;
}


// x / (1 + e^-x) with the fast exponential and reciprocal instructions (the
// result is rounded to bf16): one multiplication where a division would also
// scale for denominators past 2^126.  Those, of x below -87.3, give -0 here, where
// the quotient is at most 1e-36 in magnitude.
__device__ __forceinline__ float silu(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + __expf(-x)));
  return x * r;
}

// What a bf16 term leaves of a value: nothing of an infinite one (inf - inf is NaN).
__device__ __forceinline__ float rest(float v, float term) {
  return fabsf(term) == INFINITY ? 0.f : v - term;
}

// Four neighbouring values as `terms` bf16 terms each, at dst, dst + step, ...
__device__ __forceinline__ void store_terms(__nv_bfloat16* dst, int step, int terms, float4 v) {
  for (int k = 0; k < terms; ++k) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
    uint2 w;
    w.x = *reinterpret_cast<const uint32_t*>(&a);
    w.y = *reinterpret_cast<const uint32_t*>(&b);
    *reinterpret_cast<uint2*>(dst + k * step) = w;
    const float2 fa = __bfloat1622float2(a), fb = __bfloat1622float2(b);
    v.x = rest(v.x, fa.x);
    v.y = rest(v.y, fa.y);
    v.z = rest(v.z, fb.x);
    v.w = rest(v.w, fb.y);
  }
}

// This CTA's share of a cluster's outputs: the parts ([token][ld] floats in each
// CTA's shared memory) of tokens [0, count) and rank rows [m0, m0 + here), `here`
// a multiple of 16, summed in cluster order, scaled, and stored as terms.  The rows
// that pad a slice's rank are stored as zeros: 0 times an infinite x is NaN.
template <int SPLITS, typename Cluster>
__device__ __forceinline__ void finish_part(const ShrinkArgs& p, const Cluster& cluster, const float* part,
                                            int ld, int start, int count, int m0, int here, int rank,
                                            float scale) {
  const int rank_p = pad16(rank);
  const int split = SPLITS > 1 ? (int)cluster.block_rank() : 0, quads = here / 4;
#pragma unroll (SPLITS > 2 ? 2 : 4)
  for (int o = split * blockDim.x + threadIdx.x; o < count * quads; o += SPLITS * blockDim.x) {
    const int col = o / quads, row = 4 * (o - col * quads);
    const float* at = part + col * ld + row;
    float4 q[SPLITS];
#pragma unroll
    for (int k = 0; k < SPLITS; ++k)
      q[k] = *reinterpret_cast<const float4*>(SPLITS > 1 ? cluster.map_shared_rank(at, k) : at);
    float4 v = q[0];
#pragma unroll
    for (int k = 1; k < SPLITS; ++k) {
      v.x += q[k].x;
      v.y += q[k].y;
      v.z += q[k].z;
      v.w += q[k].w;
    }
    const int j = (m0 + row) / rank_p, r = m0 + row - j * rank_p;
    store_terms(p.s + (start + col) * p.s_stride + j * p.terms * rank_p + r, rank_p, p.terms,
                make_float4(r < rank ? v.x * scale : 0.f, r + 1 < rank ? v.y * scale : 0.f,
                            r + 2 < rank ? v.z * scale : 0.f, r + 3 < rank ? v.w * scale : 0.f));
  }
}

template <typename Cluster>
__device__ __forceinline__ void finish_s(const ShrinkArgs& p, const Cluster& cluster, const float* part,
                                         int ld, int start, int count, int m0, int here, int rank,
                                         float scale) {
  switch ((int)cluster.num_blocks()) {  // 1, 2, 4 or 8
    case 1: return finish_part<1>(p, cluster, part, ld, start, count, m0, here, rank, scale);
    case 2: return finish_part<2>(p, cluster, part, ld, start, count, m0, here, rank, scale);
    case 4: return finish_part<4>(p, cluster, part, ld, start, count, m0, here, rank, scale);
    default: return finish_part<8>(p, cluster, part, ld, start, count, m0, here, rank, scale);
  }
}

}  // namespace

// The second product on tcgen05 (lora_tc.cu), for tiles of many tokens:
// MS_ERR_UNSUPPORTED when the shape does not apply.
int lora_expand_tc(const ExpandArgs& p, int epilogue, cudaStream_t s);
// The first product likewise.
int lora_shrink_tc(ShrinkArgs p, int rows, cudaStream_t s);
// A launch of the first product in clusters of `split` CTAs along z.
int launch_cluster(void (*kernel)(ShrinkArgs), dim3 grid, int threads, int smem, int split,
                   cudaStream_t s, const ShrinkArgs& p);

}  // namespace ms
