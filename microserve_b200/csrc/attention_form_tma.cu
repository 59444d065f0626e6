// Attention with score forms over bf16 caches, for few rows: up to 32 (16 at heads
// of 128) a sequence and kv head, as single tokens and small trees have.
//
// One CTA per (KV range, kv head, sequence).  Row r is (token r / group, head-in-group
// r % group), so that keys and values are read once per kv head.
//   producer warp   TMA loads of each chunk of 64 places (whole pages or parts
//                   of one) into a ring, a lane a page;
//   consumer warps  one for each 16 rows: S = Q K^T and O += P V by mma.sync
//                   m16n8k16, online softmax in base 2 in float32.  P enters the
//                   second product rounded to bf16 (its operand type); the sum
//                   that divides it is of the rounded values, so the rounding of a
//                   dominant p cancels.
// Bound by HBM, less the start and the end of each CTA: 128 sequences of one token, 32 heads over 8 of 128,
// cap and a window of 2048 (990 MB) 187 us, 5.3 TB/s; one of 332 keys 14 us, which is latency.
//
// Masks cost nothing in chunks that every row sees in full; elsewhere each row
// has its 64 places as bits.  In those chunks values may be anything (a stale
// page's tail, a branch that overflowed): what is not finite enters the product
// as 0 and is added afterwards to the rows that see it.  Rows whose sums are not finite
// are looked at again at the end (form_row_again).
#include <cfloat>
#include <mutex>

#include "attention_form_device.cuh"

namespace ms {
namespace {

constexpr int kRows = 32;
constexpr int kCh = 64;  // keys per chunk

template <int DH, int MT, int NS>
struct Cfg {
  static constexpr int kThreads = (MT + 1) * 32;
  static constexpr int kTile = kCh * DH * 2;  // K or V of a chunk
  static constexpr int kLdQ = DH + 8;
  static constexpr int kQBytes = MT * 16 * kLdQ * 2;
  static constexpr int kSmem = 1024 + NS * 2 * kTile + kQBytes + 128;
};

__device__ __forceinline__ void ldm_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldm_x4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// 16-byte chunk c of key row k in a tile (see form_pool_map).
template <int DH>
__device__ __forceinline__ uint32_t tile_addr(uint32_t tile, int k, int c) {
  return tile + (uint32_t)((k >> 3) * (DH * 16) + (c >> 3) * 1024 + (k & 7) * 128 + (((c & 7) ^ (k & 7)) << 4));
}
__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

template <int DH, int MT, int NS, int MINB>
__global__ void __launch_bounds__((MT + 1) * 32, MINB)
    form_tma_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                    const __grid_constant__ FormArgs a, int log2_bs, int vec) {
  pdl_enter();
  using C = Cfg<DH, MT, NS>;
  constexpr int NT = DH / 8;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  const uint32_t raw = s_addr(smem_raw);
  unsigned char* smem = smem_raw + ((1024u - (raw & 1023u)) & 1023u);
  const uint32_t ring = s_addr(smem);
  __nv_bfloat16* Qs = reinterpret_cast<__nv_bfloat16*>(smem + NS * 2 * C::kTile);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + NS * 2 * C::kTile + C::kQBytes);
  const uint32_t full = s_addr(bars), empty = full + 8 * NS;
  volatile int* stop = reinterpret_cast<volatile int*>(bars + 2 * NS);

  const int g = blockIdx.y, b = a.order ? a.order[blockIdx.z] : blockIdx.z;
  const int split = blockIdx.x % a.n_splits, tile = blockIdx.x / a.n_splits;
  const FormSeq s = form_seq(a, b);
  const int r0 = tile * kRows;
  if (r0 >= s.qlen * a.group) return;
  const int nr = min(kRows, s.qlen * a.group - r0);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int minpos = 0, maxpos = 0;
  if (needs_positions(a)) position_range(a, s, r0, nr, minpos, maxpos);
  const FormKeys keys = form_keys(a, s, minpos, maxpos);
  const int xbeg = min(split * a.split_len, keys.total);
  const int xend = split == a.n_splits - 1 ? keys.total : min(keys.total, xbeg + a.split_len);
  const int chunks = (xend - xbeg + kCh - 1) / kCh;

  if (threadIdx.x == 0) {
    for (int i = 0; i < NS; ++i) {
      mbar_init(full + 8 * i, 1);
      mbar_init(empty + 8 * i, MT);
    }
    *stop = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  __syncthreads();

  if (warp == MT) {
    // ---- producer: lane l loads box l / 2 of the chunk, K or V
    static_assert(kCh / 8 * 2 <= 32, "a lane for each box");
    const int box = min(a.bs, kCh), boxes = kCh / box;
    const int i = lane / 2, is_v = lane & 1;
    const int32_t* table = a.tables + (int64_t)b * a.max_blocks;
    auto row_of = [&](int chunk) {  // the pool row of this lane's box (-1: none)
      const int x = xbeg + chunk * kCh + i * box;
      if (i >= boxes || x >= xend) return -1;
      const int j = keys.key(x);
      return (form_block(a, table, j >> log2_bs) * a.hkv + g) * a.bs + (j & (a.bs - 1));
    };
    int next = chunks > 0 ? row_of(0) : -1, issued = 0;
    bool ok = true;
    for (int ch = 0; ch < chunks; ++ch) {
      const int slot = ch % NS, row = next;
      if (ch + 1 < chunks) next = row_of(ch + 1);
      if (ch >= NS) ok = mbar_wait(empty + 8 * slot, ((ch / NS) - 1) & 1, stop, a.err);
      if (!__all_sync(0xffffffffu, ok)) break;
      const int n = (min(kCh, xend - (xbeg + ch * kCh)) + box - 1) / box;
      if (lane == 0) mbar_expect_tx(full + 8 * slot, (uint32_t)(n * box * DH * 2 * 2));
      __syncwarp();
      if (row >= 0) {
        const uint32_t dst = ring + slot * 2 * C::kTile + is_v * C::kTile + i * box * DH * 2;
        tma_load_rows(dst, is_v ? &vmap : &kmap, full + 8 * slot, row);
      }
      ++issued;
    }
    // a block that gave up still waits for its loads in flight
    if (*stop) {
      int none = 0;
      for (int ch = max(0, issued - NS); ch < issued; ++ch)
        mbar_wait(full + 8 * (ch % NS), (ch / NS) & 1, &none, a.err);
    }
    return;
  }

  // ---- consumers
  const int wr = warp * 16;
  const bool live = wr < nr;
  const int ra = wr + (lane >> 2), rb = ra + 8;
  const bool upper = wr + 8 < nr;  // any of the rows rb
  if (live) {
    const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(a.q);
    if (vec) {
      for (int idx = lane; idx < 16 * (DH / 8); idx += 32) {
        const int r = wr + idx / (DH / 8), c = (idx % (DH / 8)) * 8, rr = r0 + r;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (r < nr)
          v = *reinterpret_cast<const uint4*>(q + (int64_t)(s.t0 + rr / a.group) * a.q_stride +
                                              (int64_t)(g * a.group + rr % a.group) * DH + c);
        *reinterpret_cast<uint4*>(Qs + r * C::kLdQ + c) = v;
      }
    } else {
      for (int idx = lane; idx < 16 * DH; idx += 32) {
        const int r = wr + idx / DH, c = idx % DH, rr = r0 + r;
        Qs[r * C::kLdQ + c] = r < nr ? q[(int64_t)(s.t0 + rr / a.group) * a.q_stride +
                                         (int64_t)(g * a.group + rr % a.group) * DH + c]
                                     : __float2bfloat16_rn(0.f);
      }
    }
    __syncwarp();
  }
  const int tok_a = s.t0 + (r0 + min(ra, nr - 1)) / a.group, tok_b = s.t0 + (r0 + min(rb, nr - 1)) / a.group;
  const int pos_a = a.positions[tok_a], pos_b = a.positions[tok_b];
  float slope_a = 0.f, slope_b = 0.f;  // in base 2
  if (a.slopes) {
    slope_a = a.slopes[g * a.group + (r0 + min(ra, nr - 1)) % a.group] * kLog2e;
    slope_b = a.slopes[g * a.group + (r0 + min(rb, nr - 1)) % a.group] * kLog2e;
  }
  const bool cap = a.softcap > 0.f;
  Cap capped{};
  if (cap) capped.set(a);
  // scores as the exponent takes them: x * mul
  const float mul = cap || a.slopes ? 1.f : a.scale * kLog2e;
  const float lin = a.scale * kLog2e;

  float m_a = -INFINITY, m_b = -INFINITY, l_a = 0.f, l_b = 0.f;
  float o[NT][4];
#pragma unroll
  for (int i = 0; i < NT; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  const uint32_t q_lane = s_addr(Qs + (wr + (lane & 15)) * C::kLdQ + (lane >> 4) * 8);

  bool ok = true;
  for (int ch = 0; ch < chunks; ++ch) {
    const int slot = ch % NS, x0 = xbeg + ch * kCh;
    ok = mbar_wait(full + 8 * slot, (ch / NS) & 1, stop, a.err);
    if (!__all_sync(0xffffffffu, ok)) break;
    if (live) {
      const uint32_t Kt = ring + slot * 2 * C::kTile, Vt = Kt + C::kTile;
      float sc[kCh / 8][4];
#pragma unroll
      for (int i = 0; i < kCh / 8; ++i) sc[i][0] = sc[i][1] = sc[i][2] = sc[i][3] = 0.f;
#pragma unroll
      for (int k = 0; k < DH / 16; ++k) {
        uint32_t qf[4], kb[kCh / 16][4];
        ldm_x4(q_lane + k * 32, qf);
#pragma unroll
        for (int p = 0; p < kCh / 16; ++p)
          ldm_x4(tile_addr<DH>(Kt, p * 16 + (lane & 7) + ((lane >> 4) << 3), 2 * k + ((lane >> 3) & 1)), kb[p]);
#pragma unroll
        for (int p = 0; p < kCh / 16; ++p) {
          mma_bf16(sc[2 * p], qf, kb[p][0], kb[p][1]);
          mma_bf16(sc[2 * p + 1], qf, kb[p][2], kb[p][3]);
        }
      }
      const bool free = all_see<kCh>(a, s, keys, x0, xend, minpos, maxpos);
      // ---- scores: cap, distance
      if (cap) {
        float top[4] = {};  // of |score|, NaN if there is one
#pragma unroll
        for (int i = 0; i < kCh / 8; ++i) {
          top[i & 1] = max3_abs(top[i & 1], sc[i][0], sc[i][1]);
          if (upper) top[2 + (i & 1)] = max3_abs(top[2 + (i & 1)], sc[i][2], sc[i][3]);
        }
        // some score is beyond the cap's series
        const bool far = !(max3_abs(top[0], top[1], max3_abs(0.f, top[2], top[3])) <= capped.limit);
        if (__any_sync(0xffffffffu, far)) {
#pragma unroll
          for (int i = 0; i < kCh / 8; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (e < 2 || upper) sc[i][e] = capped.any(sc[i][e]);
        } else {
#pragma unroll
          for (int i = 0; i < kCh / 8; ++i)
#pragma unroll
            for (int e = 0; e < 4; e += 2)
              if (e < 2 || upper)
                unpair(capped.series(pair(__float_as_uint(sc[i][e]), __float_as_uint(sc[i][e + 1]))), sc[i][e],
                       sc[i][e + 1]);
        }
      }
      if (a.slopes) {
        const float in = cap ? 1.f : lin;
        const int jl = keys.key(x0) + 2 * (lane & 3);
#pragma unroll
        for (int i = 0; i < kCh / 8; ++i)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int at = free ? jl + i * 8 + e : key_position(a, s, keys, x0 + i * 8 + 2 * (lane & 3) + e);
            sc[i][e] = fmaf(-slope_a, fabsf((float)(pos_a - at)), sc[i][e] * in);
            sc[i][2 + e] = fmaf(-slope_b, fabsf((float)(pos_b - at)), sc[i][2 + e] * in);
          }
      }
      // ---- maxima, over what each row sees
      float mx_a = -INFINITY, mx_b = -INFINITY;
      if (!free) {
        const uint64_t see_a = seen_places(a, s, keys, tok_a, pos_a, x0, xend) >> (2 * (lane & 3));
        const uint64_t see_b = seen_places(a, s, keys, tok_b, pos_b, x0, xend) >> (2 * (lane & 3));
#pragma unroll
        for (int i = 0; i < kCh / 8; ++i)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            sc[i][e] = (see_a >> (8 * i + e)) & 1 ? sc[i][e] : -INFINITY;
            sc[i][2 + e] = (see_b >> (8 * i + e)) & 1 ? sc[i][2 + e] : -INFINITY;
          }
      }
#pragma unroll
      for (int i = 0; i < kCh / 8; ++i) {
        mx_a = fmaxf(mx_a, fmaxf(sc[i][0], sc[i][1]));
        mx_b = fmaxf(mx_b, fmaxf(sc[i][2], sc[i][3]));
      }
#pragma unroll
      for (int d = 1; d <= 2; d <<= 1) {
        mx_a = fmaxf(mx_a, __shfl_xor_sync(0xffffffffu, mx_a, d));
        mx_b = fmaxf(mx_b, __shfl_xor_sync(0xffffffffu, mx_b, d));
      }
      const float mn_a = fmaxf(m_a, mx_a * mul), mn_b = fmaxf(m_b, mx_b * mul);
      const bool grow = mn_a > m_a || mn_b > m_b;
      const float sub_a = mn_a == -INFINITY ? 0.f : mn_a, sub_b = mn_b == -INFINITY ? 0.f : mn_b;
      float by = mul;
      if (__any_sync(0xffffffffu, fmaxf(fabsf(sub_a), fabsf(sub_b)) > kBig)) {
        by = 1.f;
#pragma unroll
        for (int i = 0; i < kCh / 8; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[i][e] *= mul;
      }
      const float al_a = fast_exp2(m_a - sub_a), al_b = fast_exp2(m_b - sub_b);
      m_a = mn_a;
      m_b = mn_b;
      // ---- p, rounded to bf16, and their sums
      uint32_t pf[kCh / 16][4];
      float ps_a = 0.f, ps_b = 0.f;
#pragma unroll
      for (int i = 0; i < kCh / 8; ++i) {
        const uint32_t pa = pack2(fast_exp2(fmaf(sc[i][0], by, -sub_a)), fast_exp2(fmaf(sc[i][1], by, -sub_a)));
        uint32_t pb = 0;
        if (upper)
          pb = pack2(fast_exp2(fmaf(sc[i][2], by, -sub_b)), fast_exp2(fmaf(sc[i][3], by, -sub_b)));
        ps_a += low_half(pa) + high_half(pa);
        ps_b += low_half(pb) + high_half(pb);
        pf[i / 2][(i & 1) * 2] = pa;
        pf[i / 2][(i & 1) * 2 + 1] = pb;
      }
      l_a = fmaf(l_a, al_a, ps_a);
      l_b = fmaf(l_b, al_b, ps_b);
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          o[i][0] *= al_a;
          o[i][1] *= al_a;
          o[i][2] *= al_b;
          o[i][3] *= al_b;
        }
      }
      // ---- O += P V
      uint32_t odd = 0;  // values that are not finite
#pragma unroll
      for (int kt = 0; kt < kCh / 16; ++kt) {
        uint32_t vb[NT / 2][4];
#pragma unroll
        for (int p = 0; p < NT / 2; ++p)
          ldm_x4_t(tile_addr<DH>(Vt, kt * 16 + (lane & 15), 2 * p + (lane >> 4)), vb[p]);
        if (!free) {
#pragma unroll
          for (int p = 0; p < NT / 2; ++p)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              // register e: keys kt * 16 + 8 (e & 1) + 2 (lane & 3) and the next
              const int left = xend - x0 - (kt * 16 + 8 * (e & 1) + 2 * (lane & 3));
              uint32_t v = left >= 2 ? vb[p][e] : left == 1 ? vb[p][e] & 0xffffu : 0u;
              const uint32_t bad = __vcmpeq2(v & 0x7f807f80u, 0x7f807f80u);
              odd |= bad;
              vb[p][e] = v & ~bad;
            }
        }
#pragma unroll
        for (int p = 0; p < NT / 2; ++p) {
          mma_bf16(o[2 * p], pf[kt], vb[p][0], vb[p][1]);
          mma_bf16(o[2 * p + 1], pf[kt], vb[p][2], vb[p][3]);
        }
      }
      if (!free && __any_sync(0xffffffffu, odd != 0)) {
        const uint64_t see_a = seen_places(a, s, keys, tok_a, pos_a, x0, xend);
        const uint64_t see_b = seen_places(a, s, keys, tok_b, pos_b, x0, xend);
        for (int k = 0; k < kCh && x0 + k < xend; ++k)
#pragma unroll
          for (int i = 0; i < NT; ++i) {
            const uint32_t v = lds32(tile_addr<DH>(Vt, k, i) + 4 * (lane & 3));
            const uint32_t bad = __vcmpeq2(v & 0x7f807f80u, 0x7f807f80u);
            if ((bad & 0xffffu) && ((see_a >> k) & 1)) o[i][0] += low_half(v);
            if ((bad >> 16) && ((see_a >> k) & 1)) o[i][1] += high_half(v);
            if ((bad & 0xffffu) && ((see_b >> k) & 1)) o[i][2] += low_half(v);
            if ((bad >> 16) && ((see_b >> k) & 1)) o[i][3] += high_half(v);
          }
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(empty + 8 * slot);
  }
#pragma unroll
  for (int d = 1; d <= 2; d <<= 1) {
    l_a += __shfl_xor_sync(0xffffffffu, l_a, d);
    l_b += __shfl_xor_sync(0xffffffffu, l_b, d);
  }
  if (!live || !ok) return;
  const int col = 2 * (lane & 3);
  const int64_t part_row0 = ((((int64_t)b * a.hkv + g) * a.row_tiles + tile) * a.n_splits + split) * kRows;
  uint32_t again[2];  // rows that have weights, all finite, and sums that are not
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int r = half ? rb : ra;
    const float l = half ? l_b : l_a;
    float top[2] = {};
#pragma unroll
    for (int i = 0; i < NT; ++i) top[i & 1] = max3_abs(top[i & 1], o[i][2 * half], o[i][2 * half + 1]);
    again[half] = __ballot_sync(0xffffffffu, r < nr && !(max3_abs(top[0], top[1], 0.f) < INFINITY) && l > 0.f &&
                                                 l < INFINITY);
    if (r >= nr) continue;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    if (a.n_splits == 1) {
      __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(a.out) + (int64_t)(half ? tok_b : tok_a) * a.out_stride +
                           (int64_t)(g * a.group + (r0 + r) % a.group) * DH + col;
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const uint32_t v = l == 0.f ? 0u : pack2(o[i][2 * half] * inv, o[i][2 * half + 1] * inv);
        if (vec) {
          *reinterpret_cast<uint32_t*>(dst + i * 8) = v;
        } else {
          dst[i * 8] = __ushort_as_bfloat16((unsigned short)(v & 0xffffu));
          dst[i * 8 + 1] = __ushort_as_bfloat16((unsigned short)(v >> 16));
        }
      }
    } else {
      if ((lane & 3) == 0)
        *reinterpret_cast<float2*>(a.part_ml + (part_row0 + r) * 2) = make_float2(half ? m_b : m_a, l);
      if (l == 0.f) continue;
      float* po = a.part_o + (part_row0 + r) * DH + col;
#pragma unroll
      for (int i = 0; i < NT; ++i)
        *reinterpret_cast<float2*>(po + i * 8) = make_float2(o[i][2 * half] * inv, o[i][2 * half + 1] * inv);
    }
  }
  if ((again[0] | again[1]) == 0) return;
  __syncwarp();
  const int32_t* table = a.tables + (int64_t)b * a.max_blocks;
  float common[DH / 32];
  form_odd_values<__nv_bfloat16, DH>(a, s, keys, table, g, xbeg, xend, minpos, maxpos, 0, DH, 0, 1, common);
  for (int i = 0; i < 16; ++i)  // (four lanes a row)
    if ((again[i >> 3] >> (4 * (i & 7))) & 15)
      form_row_again<__nv_bfloat16, DH, true>(a, s, keys, table, g, r0 + wr + i, xbeg, xend, minpos, maxpos, 0, DH,
                                              part_row0 + wr + i, true, common);
}

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                              const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                              CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                              CUtensorMapFloatOOBfill);

EncodeFn encode_fn() {
  static EncodeFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeFn>(p);
  });
  return fn;
}

template <int DH, int MT, int NS, int MINB>
int launch(const FormArgs& a, const CUtensorMap& km, const CUtensorMap& vm, int vec, cudaStream_t s) {
  using C = Cfg<DH, MT, NS>;
  static_assert(MINB * (C::kSmem + 1024) <= 228 * 1024, "CTAs per SM exceed shared memory");
  static std::atomic<uint64_t> granted{0};
  MS_TRY(grant_dynamic_smem(form_tma_kernel<DH, MT, NS, MINB>, C::kSmem, granted));
  dim3 grid(a.row_tiles * a.n_splits, a.hkv, a.n_seqs);
  launch_pdl(form_tma_kernel<DH, MT, NS, MINB>, grid, C::kThreads, C::kSmem, s, km, vm, a,
             __builtin_ctz((unsigned)a.bs), vec);
  MS_TRY(check_launch("form_tma_kernel"));
  return a.n_splits > 1 ? form_combine<__nv_bfloat16, true>(a, kRows, DH, s) : MS_OK;
}

}  // namespace

int form_pool_map(const void* pool, int64_t rows, int dh, int box, CUtensorMap* out) {
  EncodeFn enc = encode_fn();
  if (!enc) return fail(MS_ERR_CUDA, "form_pool_map: cuTensorMapEncodeTiled unavailable");
  const cuuint64_t dims[4] = {64, 8, (cuuint64_t)dh / 64, (cuuint64_t)rows / 8};
  const cuuint64_t strides[3] = {(cuuint64_t)dh * 2, 128, (cuuint64_t)dh * 16};
  const cuuint32_t sizes[4] = {64, 8, (cuuint32_t)dh / 64, (cuuint32_t)box / 8}, estr[4] = {1, 1, 1, 1};
  const CUresult r = enc(out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(pool), dims, strides,
                         sizes, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(MS_ERR_CUDA, "form_pool_map: tensor map encode failed (%d)", (int)r);
  return MS_OK;
}

// bf16, heads of 64 or 128, pages of 8 to 256 keys (a power of two), pools that TMA can address.
bool form_tma_takes(const ms_kv_cache& c) {
  const int bs = c.block_size;
  return c.dtype == MS_DTYPE_BF16 && (c.d_head == 64 || c.d_head == 128) && bs >= 8 && bs <= 256 &&
         (bs & (bs - 1)) == 0 && (int64_t)c.num_blocks * c.n_kv_heads * bs < (1ll << 31);
}

int form_tma(const FormArgs& a, int dh, cudaStream_t s) {
  CUtensorMap km, vm;
  const int64_t rows = (int64_t)a.num_blocks * a.hkv * a.bs;
  MS_TRY(form_pool_map(a.k, rows, dh, min(a.bs, kCh), &km));
  MS_TRY(form_pool_map(a.v, rows, dh, min(a.bs, kCh), &vm));
  const int vec = ((reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.out)) & 15) == 0 &&
                  a.q_stride % 8 == 0 && a.out_stride % 8 == 0;
  if (dh == 128) return launch<128, 1, 2, 3>(a, km, vm, vec, s);
  return a.max_q * a.group <= 16 ? launch<64, 1, 2, 6>(a, km, vm, vec, s) : launch<64, 2, 3, 4>(a, km, vm, vec, s);
}

}  // namespace ms
