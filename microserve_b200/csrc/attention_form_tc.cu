// Attention with score forms over bf16 caches on tcgen05, for many rows:
// prompts and the rows of larger trees.
//
// A CTA takes ST streams of 128 rows each of one kv head of one sequence (row r is
// (token r / group, head-in-group r % group)) and a range of its keys, KC places
// at a step; the streams share the keys and values.
//   softmax warps (4 a stream)  a thread has a row: scores out of TMEM, cap,
//        distance, mask (bits, only where some row does not see all keys), p =
//        2^(x - m) rounded to bf16 back into TMEM over the scores, and the sum of the
//        rounded values.  m is raised only when a row's maximum has grown by
//        more than 2^8, so O is rescaled a few times a row at most;
//   producer warp  TMA loads of whole pages (or parts of one), a box a lane, into
//        rings of their own for K and V;
//   MMA warp  one thread issues S = Q K^T (both from shared memory) and O += P V (P in
//        TMEM, V MN-major as it lies in the page).  With SB score buffers the
//        scores of the next SB steps are there when p of this one is.
// Two shapes: ST 2, KC 128, SB 1, one CTA an SM (all 512 TMEM columns at d_head 128): the
// streams' softmax and MMAs take turns; and ST 1, KC 64, SB 2, two CTAs an SM, for up to 128
// rows, where HBM is the bound.
//
// Values that no row should meet: where a mask is needed the softmax warps look
// at the step's values first and put 0 for what is not finite.  If one of those belongs
// to a key that some row may see, the CTA computes its rows again on the
// CUDA cores, key by key.
#include <cfloat>

#include "attention_form_device.cuh"

namespace ms {
namespace {

constexpr int kTileRows = 128;

// The shape of a CTA: up to 64 rows (twice, each copy half of the keys), 128, or 256 in two streams.
enum Shape { kHalf, kOne, kTwo };

template <int DH, int SH>
struct TcCfg {
  static constexpr int ST = SH == kTwo ? 2 : 1;                  // streams of 128 rows
  static constexpr bool kTwin = SH == kHalf;
  static constexpr int KC = kTwin && DH == 64 ? 128 : 64;        // keys per step
  static constexpr int SB = kTwin ? 1 : 2;                       // score buffers
  static constexpr int kWidth = kTwin ? KC / 2 : KC;             // scores of a step per thread
  static constexpr int kTile = KC * DH * 2;                      // K or V of a step
  static constexpr int kSlots = SH == kTwo ? 144 : kTwin && DH == 64 ? 96 : DH == 64 ? 96 : 80;  // KB of K and V
  static constexpr int NK = (kSlots * 1024 / kTile + 1) / 2, NV = kSlots * 1024 / kTile / 2;
  static constexpr int kQ = kTileRows * DH * 2;
  static constexpr int kPCol = kTwin ? KC : 0;                   // p stands behind the scores, or over them
  static constexpr int kOCol = kTwin ? KC + KC / 2 : SB * KC;
  static constexpr int kStreamCols = kOCol + DH;
  static constexpr int kCols = ST == 2 ? 512 : 256;
  static constexpr int kWarps = 4 * ST + (ST == 2 ? 4 : 2);
  static constexpr int kThreads = kWarps * 32;
  static constexpr int kBars = 2 * NK + 2 * NV + 3 + ST * (2 * SB + 2);
  static constexpr int kSmem = ST * kQ + (NK + NV) * kTile + kBars * 8 + 16;
  static_assert(ST * kStreamCols <= kCols, "TMEM columns");
  static_assert((3 - ST) * (kSmem + 1024) <= 228 * 1024, "shared memory of the CTAs of an SM");
  static_assert(!kTwin || 64 * DH * 4 + 64 * 8 <= NK * kTile, "the copies meet in the K ring");
};

// Descriptors with the 128-byte swizzle.  K-major (Q, K): rows of 64 values, 8-row
// groups 1024 bytes apart.  MN-major (V): 64 dimensions a row, groups of 8 keys
// 1024 bytes apart, blocks of 64 dimensions `lead` bytes apart.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lead) {
  uint64_t d = (uint64_t)((addr & 0x3FFFFu) >> 4);
  d |= (uint64_t)(lead >> 4) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}
// float32 accumulator, bf16 operands, M 128.
__device__ __forceinline__ constexpr uint32_t instr_desc(int n, bool b_mn_major) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(kTileRows >> 4) << 24);
}
// One thread of the warp issues: `one` is 1 in an elected lane.  The whole warp runs the code
// around, so that descriptors stay in uniform registers (issued inside a branch of one
// lane an MMA cost 75 to 110 cycles, more than it takes to execute).
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t accumulate,
                                       uint32_t one) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(id), "r"(accumulate), "r"(one)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t accumulate,
                                       uint32_t one) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(id), "r"(accumulate), "r"(one)
      : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t bar, uint32_t one) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar),
      "r"(one)
      : "memory");
}
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t one;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.b32 %0, 1, 0, p;\n\t}"
      : "=r"(one));
  return one;
}
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]),
      "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]),
      "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// Nothing that uses r comes before this (the loads' outputs are there only after the wait).
__device__ __forceinline__ void pin32(uint32_t* r) {
  asm volatile(""
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]));
  asm volatile(""
               : "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]),
                 "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]),
                 "+r"(r[29]));
  asm volatile("" : "+r"(r[30]), "+r"(r[31]));
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
__device__ __forceinline__ void sts128(uint32_t addr, const uint4& v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
               : "memory");
}
__device__ __forceinline__ void st32(uint32_t addr, float v) {
  asm volatile("st.shared.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}
__device__ __forceinline__ float ld32(uint32_t addr) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t not_finite(uint32_t v) {
  return __vcmpeq2(v & 0x7f807f80u, 0x7f807f80u);
}

// Two floats in a register pair: the packed operations of sm_100 halve the issue slots.
__device__ __forceinline__ uint64_t pair(uint32_t lo, uint32_t hi) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(lo), "r"(hi));
  return d;
}
__device__ __forceinline__ uint64_t twice(float v) { return pair(__float_as_uint(v), __float_as_uint(v)); }
__device__ __forceinline__ void unpair(uint64_t v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float max3(float a, uint32_t b, uint32_t c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(__uint_as_float(b)), "f"(__uint_as_float(c)));
  return d;
}
__device__ __forceinline__ float min3(float a, uint32_t b, uint32_t c) {
  float d;
  asm("min.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(__uint_as_float(b)), "f"(__uint_as_float(c)));
  return d;
}

// Adds the two bf16 of a word to two float32 sums.
__device__ __forceinline__ void add_bf16(uint32_t v, float& lo, float& hi) {
  asm("{\n\t.reg .b16 l, h;\n\t"
      "mov.b32 {l, h}, %2;\n\t"
      "add.f32.bf16 %0, l, %0;\n\t"
      "add.f32.bf16 %1, h, %1;\n\t}"
      : "+f"(lo), "+f"(hi)
      : "r"(v));
}

// cap tanh(u) in base 2, u = k s.  For |u| <= 0.75 an odd polynomial in s (tanh(u) = u (1 + c1
// u^2 + .. + c4 u^8), fitted to the least maximum of |error|, 2.7e-7; no SFU), whose
// coefficients take k in; else cap (1 - 2 / (1 + e^2u)), off by 2^-22 of the cap.
struct Cap {
  float d0, d1, d2, d3, d4;  // of s, s^3, ...
  float limit;               // of |s|
  float cap2, in;
  __device__ __forceinline__ void set(const FormArgs& a) {
    cap2 = a.softcap * kLog2e;
    const float k = a.scale / a.softcap, kk = k * k;
    in = 2.f * kLog2e * k;
    d0 = a.scale * kLog2e;
    d1 = d0 * (-0.333280453f * kk);
    d2 = d0 * (0.132533633f * kk * kk);
    d3 = d0 * (-0.0498660865f * kk * kk * kk);
    d4 = d0 * (0.0127505842f * kk * kk * kk * kk);
    limit = k <= 1024.f ? 0.75f / k : -1.f;  // (k^8 stays within float32)
  }
  __device__ __forceinline__ float exact(float s) const {
    return fmaf(-2.f * cap2, fast_rcp(1.f + fast_exp2(s * in)), cap2);
  }
  __device__ __forceinline__ float series(float s) const {
    const float w = s * s;
    return s * fmaf(w, fmaf(w, fmaf(w, fmaf(w, d4, d3), d2), d1), d0);
  }
};

// p = 2^(x - sub) of 2 kWords values, rounded to bf16; `sum` gets the rounded values.
// kWay 0: x * mul; 1: the cap's series of x; 2: x as it is.
template <int kWay, int kWords>
__device__ __forceinline__ void exps(const uint32_t* x, uint32_t* p, float mul, float sub, const Cap& cap,
                                     float (&sum)[4]) {
  const uint64_t minus = twice(-sub);
#pragma unroll
  for (int e = 0; e < kWords; ++e) {
    const uint64_t v = pair(x[2 * e], x[2 * e + 1]);
    uint64_t arg;
    if constexpr (kWay == 0) {
      arg = fma2(v, twice(mul), minus);
    } else if constexpr (kWay == 1) {
      const uint64_t w = mul2(v, v);
      uint64_t c = fma2(w, twice(cap.d4), twice(cap.d3));
      c = fma2(w, c, twice(cap.d2));
      c = fma2(w, c, twice(cap.d1));
      c = fma2(w, c, twice(cap.d0));
      arg = fma2(v, c, minus);
    } else {
      arg = add2(v, minus);
    }
    float lo, hi;
    unpair(arg, lo, hi);
    p[e] = pack2(fast_exp2(lo), fast_exp2(hi));
    add_bf16(p[e], sum[2 * (e & 1)], sum[2 * (e & 1) + 1]);
  }
}

// The rows of a CTA once more, a warp a row: every seen key by itself, a lane a key for the
// scores and DH / 32 dimensions a lane for the sums.
template <int DH>
__device__ __noinline__ void rows_by_key(const FormArgs& a, const FormSeq& s, const FormKeys& keys,
                                         const int32_t* table, int g, int r0, int nr, int xbeg, int xend,
                                         int64_t part_row0, int warp, int warps) {
  const int lane = threadIdx.x & 31;
  const __nv_bfloat16 *kp = static_cast<const __nv_bfloat16*>(a.k), *vp = static_cast<const __nv_bfloat16*>(a.v);
  for (int r = warp; r < nr; r += warps) {
    const int rr = r0 + r, tok = s.t0 + rr / a.group, head = g * a.group + rr % a.group;
    const int pos = a.positions[tok];
    const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(a.q) + (int64_t)tok * a.q_stride + (int64_t)head * DH;
    const float slope = a.slopes ? a.slopes[head] : 0.f;
    float m = -INFINITY, l = 0.f, acc[DH / 32] = {};
    for (int x0 = xbeg; x0 < xend; x0 += 32) {
      const int x = min(x0 + lane, xend - 1), j = keys.key(x);
      int distance = 0;
      const bool seen = x0 + lane < xend && form_sees(a, s, tok, pos, j, distance);
      const int64_t at =
          (((int64_t)form_block(a, table, j / a.bs) * a.hkv + g) * a.bs + j % a.bs) * DH;
      float v = 0.f;
      for (int d = 0; d < DH; ++d) v = fmaf(to_f(q[d]), to_f(kp[at + d]), v);
      v = a.softcap > 0.f ? a.softcap * tanhf(v * a.scale / a.softcap) : v * a.scale;
      v = seen ? (v - slope * fabsf((float)distance)) * kLog2e : -INFINITY;
      const uint32_t all = __ballot_sync(0xffffffffu, seen);
      const float mn = fmaxf(m, warp_max(v)), sub = mn == -INFINITY ? 0.f : mn;
      const float alpha = m == -INFINITY ? 0.f : exp2f(m - sub), p = seen ? exp2f(v - sub) : 0.f;
      l = l * alpha + warp_sum(p);
      m = mn;
#pragma unroll
      for (int e = 0; e < DH / 32; ++e) acc[e] *= alpha;
      for (int k = 0; k < 32; ++k) {
        const float pk = __shfl_sync(0xffffffffu, p, k);
        const int64_t ak = __shfl_sync(0xffffffffu, at, k);
        if (!((all >> k) & 1)) continue;
#pragma unroll
        for (int e = 0; e < DH / 32; ++e) acc[e] = fmaf(pk, to_f(vp[ak + lane + 32 * e]), acc[e]);
      }
    }
    if (a.n_splits == 1) {
      const float inv = l == 0.f ? 0.f : 1.f / l;
      __nv_bfloat16* o =
          static_cast<__nv_bfloat16*>(a.out) + (int64_t)tok * a.out_stride + (int64_t)head * DH;
#pragma unroll
      for (int e = 0; e < DH / 32; ++e) o[lane + 32 * e] = __float2bfloat16_rn(acc[e] * inv);
    } else {
#pragma unroll
      for (int e = 0; e < DH / 32; ++e) a.part_o[(part_row0 + r) * DH + lane + 32 * e] = acc[e];
      if (lane == 0) {
        a.part_ml[(part_row0 + r) * 2] = m;
        a.part_ml[(part_row0 + r) * 2 + 1] = l;
      }
    }
  }
}

template <int DH, int SH>
__global__ void __launch_bounds__(TcCfg<DH, SH>::kThreads, SH == kTwo ? 1 : 2)
    form_tc_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                   const __grid_constant__ FormArgs a, int log2_bs, int vec) {
  pdl_enter();
  using C = TcCfg<DH, SH>;
  constexpr int ST = C::ST, KC = C::KC, SB = C::SB, NK = C::NK, NV = C::NV, W = C::kWidth;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  const uint32_t raw = s_addr(smem_raw), q_s = raw;  // (1024-byte aligned, as declared)
  const uint32_t k_s = q_s + ST * C::kQ, v_s = k_s + NK * C::kTile, bars = v_s + NV * C::kTile;
  const uint32_t k_full = bars, k_empty = k_full + 8 * NK, v_full = k_empty + 8 * NK, v_empty = v_full + 8 * NV;
  const uint32_t q_ready = v_empty + 8 * NV, ended = q_ready + 8, s_read = ended + 8, s_full = s_read + 8;
  const uint32_t p_ready = s_full + 8 * ST * SB, pv_done = p_ready + 8 * ST * SB, slot_at = pv_done + 16 * ST;
  unsigned char* words = smem_raw + (slot_at - raw);
  volatile uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(words);
  volatile int* stop = reinterpret_cast<int*>(words) + 1;
  volatile int* odd = reinterpret_cast<int*>(words) + 2;  // a value that is not finite and may be seen

  if (raw & 1023u) {
    if (threadIdx.x == 0) raise_device_error(a.err, kErrTimeout);
    return;
  }
  // the last tiles of the sequences, which see the most keys, come first
  const int g = blockIdx.x / a.n_splits, b = blockIdx.y, split = blockIdx.x % a.n_splits;
  const int tile = (int)gridDim.z - 1 - (int)blockIdx.z;
  const FormSeq s = form_seq(a, b);
  constexpr int kCtaRows = C::kTwin ? 64 : ST * kTileRows;
  const int r0 = tile * kCtaRows;
  if (r0 >= s.qlen * a.group) return;
  const int nr = min(kCtaRows, s.qlen * a.group - r0);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int minpos, maxpos;
  position_range(a, s, r0, nr, minpos, maxpos);
  const FormKeys keys = form_keys(a, s, minpos, maxpos);
  const int xbeg = min(split * a.split_len, keys.total);
  const int xend = split == a.n_splits - 1 ? keys.total : min(keys.total, xbeg + a.split_len);
  const int steps = (xend - xbeg + KC - 1) / KC;
  const int32_t* table = a.tables + (int64_t)b * a.max_blocks;
  constexpr int kProducer = 4 * ST, kMma = kProducer + 1;

  if (threadIdx.x == 0) {
    for (int i = 0; i < NK; ++i) {
      mbar_init(k_full + 8 * i, 1);
      mbar_init(k_empty + 8 * i, 1);
    }
    for (int i = 0; i < NV; ++i) {
      mbar_init(v_full + 8 * i, 1);
      mbar_init(v_empty + 8 * i, 1);
    }
    mbar_init(q_ready, 4 * ST);
    mbar_init(ended, 1);
    mbar_init(s_read, 4);
    for (int i = 0; i < ST * SB; ++i) {
      mbar_init(s_full + 8 * i, 1);
      mbar_init(p_ready + 8 * i, 4);
    }
    for (int i = 0; i < 2 * ST; ++i) mbar_init(pv_done + 8 * i, 1);
    *stop = 0;
    *odd = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == kMma) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot_at),
                 "r"(C::kCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp >= kProducer) {
    if constexpr (ST == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
    if (warp == kProducer) {
      // ---- loads
      constexpr int kHalves = DH / 64;
      static_assert(KC / 8 * kHalves <= 32, "a lane for each box");
      const int box = min(a.bs, KC), boxes = KC / box;
      const int i = lane / kHalves, half = lane % kHalves;
      auto row_of = [&](int step) {  // the pool row of this lane's box (-1: none)
        const int x = xbeg + step * KC + i * box;
        if (i >= boxes || x >= xend) return -1;
        const int j = keys.key(x);
        return (form_block(a, table, j >> log2_bs) * a.hkv + g) * a.bs + (j & (a.bs - 1));
      };
      int next = steps > 0 ? row_of(0) : -1, k_issued = 0, v_issued = 0;
      for (int it = 0; it < steps; ++it) {
        const int row = next;
        if (it + 1 < steps) next = row_of(it + 1);
        const int n = (min(KC, xend - (xbeg + it * KC)) + box - 1) / box;
        const uint32_t bytes = (uint32_t)(n * box * DH * 2), off = half * (KC * 128) + i * box * 128;
        const int ks = it % NK, vs = it % NV;
        bool ok = it < NK || mbar_wait(k_empty + 8 * ks, (it / NK - 1) & 1, stop, a.err);
        if (!__all_sync(0xffffffffu, ok)) break;
        if (lane == 0) mbar_expect_tx(k_full + 8 * ks, bytes);
        __syncwarp();
        if (row >= 0) tma_load_2d(k_s + ks * C::kTile + off, &kmap, k_full + 8 * ks, half * 64, row);
        ++k_issued;
        ok = it < NV || mbar_wait(v_empty + 8 * vs, (it / NV - 1) & 1, stop, a.err);
        if (!__all_sync(0xffffffffu, ok)) break;
        if (lane == 0) mbar_expect_tx(v_full + 8 * vs, bytes);
        __syncwarp();
        if (row >= 0) tma_load_2d(v_s + vs * C::kTile + off, &vmap, v_full + 8 * vs, half * 64, row);
        ++v_issued;
      }
      if (*stop) {  // a block that gave up still waits for its loads in flight
        int none = 0;
        for (int it = max(0, k_issued - NK); it < k_issued; ++it)
          mbar_wait(k_full + 8 * (it % NK), (it / NK) & 1, &none, a.err);
        for (int it = max(0, v_issued - NV); it < v_issued; ++it)
          mbar_wait(v_full + 8 * (it % NV), (it / NV) & 1, &none, a.err);
      }
    } else if (warp == kMma && steps > 0) {
      // ---- MMAs
      constexpr uint32_t id_s = instr_desc(KC, false), id_o = instr_desc(DH, true);
      const uint32_t one = elect_one();
      // (values that the compiler knows to be the same in all lanes)
      const int n = __reduce_max_sync(0xffffffffu, steps);
      const uint32_t cols = ST == 2 ? 0u : __any_sync(0xffffffffu, (tmem & 0xffffu) != 0) ? 256u : 0u;
      auto wait = [&](uint32_t bar, uint32_t parity) {
        return __all_sync(0xffffffffu, mbar_wait(bar, parity, stop, a.err));
      };
      auto scores = [&](int it, int st) {
        const uint32_t d = cols + st * C::kStreamCols + (it % SB) * KC;
        const uint64_t qd = smem_desc(q_s + st * C::kQ, 16), kd = smem_desc(k_s + (it % NK) * C::kTile, 16);
#pragma unroll
        for (int k = 0; k < DH / 16; ++k)
          mma_ss(d, qd + (k >> 2) * (kTileRows * 128 / 16) + (k & 3) * 2,
                 kd + (k >> 2) * (KC * 128 / 16) + (k & 3) * 2, id_s, k > 0, one);
        mma_commit(s_full + 8 * (st * SB + it % SB), one);
      };
      auto add_values = [&](int it, int st) {
        const uint32_t o = cols + st * C::kStreamCols + C::kOCol;
        const uint32_t p = cols + st * C::kStreamCols + C::kPCol + (it % SB) * KC;
        const uint64_t vd = smem_desc(v_s + (it % NV) * C::kTile, KC * 128);
#pragma unroll
        for (int k = 0; k < KC / 16; ++k) mma_ts(o, p + 8 * k, vd + k * (2048 / 16), id_o, it > 0 || k > 0, one);
        mma_commit(pv_done + 8 * (2 * st + (it & 1)), one);
      };
      bool ok = wait(q_ready, 0);
      for (int it = 0; it < SB && it < n && ok; ++it) {
        ok = wait(k_full + 8 * (it % NK), (it / NK) & 1);
        if (!ok) break;
        fence_after();
        for (int st = 0; st < ST; ++st) scores(it, st);
        mma_commit(k_empty + 8 * (it % NK), one);
      }
      for (int it = 0; it < n && ok; ++it) {
        const int ahead = it + SB;
        if constexpr (C::kTwin) {  // the next scores as soon as these are read
          if (ahead < n) {
            ok = wait(k_full + 8 * (ahead % NK), (ahead / NK) & 1) && wait(s_read, it & 1);
            if (!ok) break;
            fence_after();
            scores(ahead, 0);
            mma_commit(k_empty + 8 * (ahead % NK), one);
          }
        }
        ok = wait(v_full + 8 * (it % NV), (it / NV) & 1);
        if (!ok) break;
#pragma unroll
        for (int st = 0; st < ST; ++st) {
          ok = wait(p_ready + 8 * (st * SB + it % SB), (it / SB) & 1);
          if (!ok) break;
          fence_after();
          add_values(it, st);
          if (st == ST - 1) mma_commit(v_empty + 8 * (it % NV), one);
          if constexpr (!C::kTwin) {
            if (ahead < n) {
              if (st == 0) {
                ok = wait(k_full + 8 * (ahead % NK), (ahead / NK) & 1);
                if (!ok) break;
                fence_after();
              }
              scores(ahead, st);
              if (st == ST - 1) mma_commit(k_empty + 8 * (ahead % NK), one);
            }
          }
        }
      }
      if (!ok) {  // a block that gave up still waits for its MMAs
        int none = 0;
        mma_commit(ended, one);
        mbar_wait(ended, 0, &none, a.err);
      }
    }
  } else {
    if constexpr (ST == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    // ---- softmax: stream st, row t of its tile
    const int st = warp >> 2, t = threadIdx.x & 127;
    // which half of a step's keys a copy of a row has (one copy: all of them)
    const int mine = C::kTwin ? (t >> 6) * W : 0;
    const int r = C::kTwin ? t & 63 : st * kTileRows + t;  // row of the CTA
    const bool live = r < nr;
    const bool warp_live = __any_sync(0xffffffffu, live);
    const int rr = r0 + (live ? r : 0), tok = s.t0 + rr / a.group, head = g * a.group + rr % a.group;
    const int pos = a.positions[tok];
    {
      const __nv_bfloat16* q =
          static_cast<const __nv_bfloat16*>(a.q) + (int64_t)tok * a.q_stride + (int64_t)head * DH;
      uint4 v[DH / 8];
      if (vec) {
#pragma unroll
        for (int c = 0; c < DH / 8; ++c)
          v[c] = live ? *reinterpret_cast<const uint4*>(q + c * 8) : make_uint4(0, 0, 0, 0);
      } else {
#pragma unroll
        for (int c = 0; c < DH / 8; ++c) {
          uint32_t w[4];
          for (int e = 0; e < 4; ++e)
            w[e] = !live ? 0u
                         : (uint32_t)__bfloat16_as_ushort(q[c * 8 + 2 * e]) |
                               (uint32_t)__bfloat16_as_ushort(q[c * 8 + 2 * e + 1]) << 16;
          v[c] = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
      const uint32_t to = q_s + st * C::kQ + t * 128;
#pragma unroll
      for (int c = 0; c < DH / 8; ++c)
        sts128(to + (c >> 3) * (kTileRows * 128) + (((c & 7) ^ (t & 7)) << 4), v[c]);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(q_ready);
    }
    const bool capped = a.softcap > 0.f, sloped = a.slopes != nullptr;
    Cap cap{};
    if (capped) cap.set(a);
    const float lin = a.scale * kLog2e, slope = sloped ? a.slopes[head] * kLog2e : 0.f;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_col = tmem + st * C::kStreamCols + lanes, o_col = s_col + C::kOCol;
    if constexpr (C::kTwin) {  // p of the other copy's keys: 0 for good
      uint32_t zero[32] = {};
      const uint32_t to = s_col + C::kPCol + (W - mine) / 2;
      if constexpr (W == 64) tmem_st32(to, zero); else tmem_st16(to, zero);
    }
    // the steps that every row sees in full: those inside the prefix, and [free0, free1)
    const int lead = max(0, min(keys.a > 0 ? min(keys.a, s.pfx) : s.pfx, xend) - xbeg) / KC;
    const int oldest = a.window > 0 ? max(0, max(maxpos, 0) - a.window + 1) : 0;  // a key in every window
    const int free0 = (max(0, max(keys.a, oldest - keys.shift) - xbeg) + KC - 1) / KC;
    const int free1 = max(0, min((a.mask ? s.base : min(minpos, INT_MAX - 1) + 1) - keys.shift, xend) - xbeg) / KC;
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    for (int it = 0; it < steps; ++it) {
      const int x0 = xbeg + it * KC;
      const bool free = it < lead || (it >= free0 && it < free1);
      if (!free) {
        // ---- the step's values: nothing that is not finite may enter the product
        ok = mbar_wait(v_full + 8 * (it % NV), (it / NV) & 1, stop, a.err);
        if (!__all_sync(0xffffffffu, ok)) break;
        const uint32_t vt = v_s + (it % NV) * C::kTile;
#pragma unroll 4
        for (int i = t; i < KC * DH / 8; i += kTileRows) {
          uint4 v = lds128(vt + i * 16);
          const uint4 n = make_uint4(not_finite(v.x), not_finite(v.y), not_finite(v.z), not_finite(v.w));
          if (n.x | n.y | n.z | n.w) {
            if (x0 + (i >> 3) % KC < xend) *odd = 1;
            sts128(vt + i * 16, make_uint4(v.x & ~n.x, v.y & ~n.y, v.z & ~n.z, v.w & ~n.w));
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      }
      ok = mbar_wait(s_full + 8 * (st * SB + it % SB), (it / SB) & 1, stop, a.err);
      // (these scores came after the values of step it - SB or earlier were added: of pv_done's
      // two barriers, each has at most one phase open)
      if (!__all_sync(0xffffffffu, ok)) break;
      fence_after();
      const uint32_t s_at = s_col + (it % SB) * KC, p_at = s_at + C::kPCol + mine / 2;
      if (warp_live) {
        uint32_t x[W];
#pragma unroll
        for (int c = 0; c < W; c += 32) tmem_ld32(s_at + mine + c, x + c);
        tmem_wait_ld();
#pragma unroll
        for (int c = 0; c < W; c += 32) pin32(x + c);
        if constexpr (C::kTwin) {
          fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(s_read);
        }
        // `way` says what the exponent still has to do (see exps)
        int way = capped ? 2 : 0;
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        if (capped) {
          float mn[4] = {INFINITY, INFINITY, INFINITY, INFINITY};
#pragma unroll
          for (int c = 0; c < W; c += 2) {
            mx[(c >> 1) & 3] = max3(mx[(c >> 1) & 3], x[c], x[c + 1]);
            mn[(c >> 1) & 3] = min3(mn[(c >> 1) & 3], x[c], x[c + 1]);
          }
          const float far = fmaxf(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])),
                                  -fminf(fminf(mn[0], mn[1]), fminf(mn[2], mn[3])));
          if (free && !sloped && __all_sync(0xffffffffu, far <= cap.limit)) {
            way = 1;
          } else {
#pragma unroll
            for (int c = 0; c < W; ++c) x[c] = __float_as_uint(cap.exact(__uint_as_float(x[c])));
          }
        }
        if (sloped) {
          way = 2;
          const float in = capped ? 1.f : lin;
          if (free) {
            const float away = (float)(pos - keys.key(x0 + mine));
#pragma unroll
            for (int c = 0; c < W; ++c)
              x[c] = __float_as_uint(fmaf(-slope, fabsf(away - (float)c), __uint_as_float(x[c]) * in));
          } else {
#pragma unroll
            for (int c = 0; c < W; ++c)
              x[c] = __float_as_uint(fmaf(-slope, fabsf((float)(pos - key_position(a, s, keys, x0 + mine + c))),
                                          __uint_as_float(x[c]) * in));
          }
        }
        if (!free) {
          const uint64_t see = live ? seen_places(a, s, keys, tok, pos, x0 + mine, xend) : 0ull;
#pragma unroll
          for (int c = 0; c < W; ++c)
            if (!(((uint32_t)(see >> (c & 32)) >> (c & 31)) & 1)) x[c] = 0xff800000u;  // -inf
        }
        if (way != 1) {
          mx[0] = mx[1] = mx[2] = mx[3] = -INFINITY;
#pragma unroll
          for (int c = 0; c < W; c += 2) mx[(c >> 1) & 3] = max3(mx[(c >> 1) & 3], x[c], x[c + 1]);
        }
        float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
        top = way == 0 ? top * lin : way == 1 ? cap.series(top) : top;
        const bool grow = top > m + 8.f || (m == -INFINITY && top > m);
        if (__any_sync(0xffffffffu, grow)) {
          const float mn = grow ? top : m;
          const float al = grow ? fast_exp2(m - mn) : 1.f;
          m = mn;
          l *= al;
          if (it > 0) {
            ok = mbar_wait(pv_done + 8 * (2 * st + ((it - 1) & 1)), ((it - 1) >> 1) & 1, stop, a.err);
            if (!__all_sync(0xffffffffu, ok)) break;
            fence_after();
#pragma unroll
            for (int c = 0; c < DH; c += 32) {
              uint32_t o[32];
              tmem_ld32(o_col + c, o);
              tmem_wait_ld();
              pin32(o);
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * al);
              tmem_st32(o_col + c, o);
            }
          }
        }
        const float sub = m == -INFINITY ? 0.f : m;
        float sum[4] = {};
        uint32_t p[W / 2];
        if (way == 0)
          exps<0, W / 2>(x, p, lin, sub, cap, sum);
        else if (way == 1)
          exps<1, W / 2>(x, p, lin, sub, cap, sum);
        else
          exps<2, W / 2>(x, p, lin, sub, cap, sum);
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        if constexpr (C::kTwin) {  // the values of the step before have been added: p may be replaced
          if (it > 0) ok = mbar_wait(pv_done + 8 * ((it - 1) & 1), ((it - 1) >> 1) & 1, stop, a.err);
          if (!__all_sync(0xffffffffu, ok)) break;
          fence_after();
        }
        if constexpr (W == 64) tmem_st32(p_at, p); else tmem_st16(p_at, p);
        tmem_wait_st();
      } else if (C::kTwin) {
        if (lane == 0) mbar_arrive(s_read);
        // (p_ready has one phase open at a time: not ahead of the other warps' step before)
        if (it > 0) ok = mbar_wait(pv_done + 8 * ((it - 1) & 1), ((it - 1) >> 1) & 1, stop, a.err);
        if (!__all_sync(0xffffffffu, ok)) break;
      }
      fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_ready + 8 * (st * SB + it % SB));
    }
    if (ok && steps > 0)
      ok = mbar_wait(pv_done + 8 * (2 * st + ((steps - 1) & 1)), ((steps - 1) >> 1) & 1, stop, a.err);
    ok = __all_sync(0xffffffffu, ok);
    fence_after();
    asm volatile("bar.sync 1, %0;" ::"r"(ST * 128) : "memory");
    const int64_t part_row0 = ((((int64_t)b * a.hkv + g) * a.row_tiles + tile) * a.n_splits + split) * kCtaRows;
    // the copies' parts: the second one's (m, l, O) through shared memory (all copies and MMAs have ended)
    float w0 = 1.f, w1 = 0.f;
    const uint32_t meet = k_s + (t & 63) * 4;
    if constexpr (C::kTwin) {
      if (t >= 64 && warp_live) {
        st32(meet, m);
        st32(meet + 256, l);
#pragma unroll
        for (int c = 0; c < DH; c += 32) {
          uint32_t o[32] = {};
          if (steps > 0) {
            tmem_ld32(o_col + c, o);
            tmem_wait_ld();
            pin32(o);
          }
#pragma unroll
          for (int e = 0; e < 32; ++e) st32(meet + 512 + (c + e) * 256, __uint_as_float(o[e]));
        }
      }
      asm volatile("bar.sync 1, 128;" ::: "memory");
      if (t < 64 && warp_live) {
        const float m1 = ld32(meet), l1 = ld32(meet + 256), top = fmaxf(m, m1), sub = top == -INFINITY ? 0.f : top;
        w0 = fast_exp2(m - sub);
        w1 = fast_exp2(m1 - sub);
        l = l * w0 + l1 * w1;
        m = top;
      }
    }
    if (*stop) {
    } else if (*odd) {
      rows_by_key<DH>(a, s, keys, table, g, r0, nr, xbeg, xend, part_row0, warp, 4 * ST);
    } else if (warp_live && (!C::kTwin || t < 64)) {
      // ---- a thread writes its row
      const float inv = l == 0.f ? 0.f : 1.f / l;
      __nv_bfloat16* dst =
          static_cast<__nv_bfloat16*>(a.out) + (int64_t)tok * a.out_stride + (int64_t)head * DH;
      float* po = a.part_o + (part_row0 + r) * DH;
      if (a.n_splits > 1 && live)
        *reinterpret_cast<float2*>(a.part_ml + (part_row0 + r) * 2) = make_float2(m, l);
#pragma unroll
      for (int c = 0; c < DH; c += 32) {
        uint32_t o[32] = {};
        if (steps > 0) {
          tmem_ld32(o_col + c, o);
          tmem_wait_ld();
          pin32(o);
        }
        if constexpr (C::kTwin) {
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            // (a copy without a key has sums of 0, its m - sub may be -inf)
            const float v = __uint_as_float(o[e]) * w0, u = ld32(meet + 512 + (c + e) * 256) * w1;
            o[e] = __float_as_uint(v + u);
          }
        }
        if (!live) continue;
        if (a.n_splits > 1) {
#pragma unroll
          for (int e = 0; e < 32; e += 4)
            *reinterpret_cast<uint4*>(po + c + e) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
          continue;
        }
        uint32_t w[16];
#pragma unroll
        for (int e = 0; e < 16; ++e)
          w[e] = l == 0.f ? 0u : pack2(__uint_as_float(o[2 * e]) * inv, __uint_as_float(o[2 * e + 1]) * inv);
        if (vec) {
#pragma unroll
          for (int e = 0; e < 16; e += 4)
            *reinterpret_cast<uint4*>(dst + c + 2 * e) = make_uint4(w[e], w[e + 1], w[e + 2], w[e + 3]);
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            dst[c + 2 * e] = __ushort_as_bfloat16((unsigned short)(w[e] & 0xffffu));
            dst[c + 2 * e + 1] = __ushort_as_bfloat16((unsigned short)(w[e] >> 16));
          }
        }
      }
    }
    fence_before();
  }
  __syncwarp();
  __syncthreads();
  if (warp == kMma) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::kCols));
  }
}

template <int DH, int SH>
int launch(const FormArgs& a, cudaStream_t s) {
  using C = TcCfg<DH, SH>;
  CUtensorMap km, vm;
  const int64_t rows = (int64_t)a.num_blocks * a.hkv * a.bs;
  MS_TRY(form_pool_map(a.k, rows, DH, min(a.bs, C::KC), &km));
  MS_TRY(form_pool_map(a.v, rows, DH, min(a.bs, C::KC), &vm));
  const int vec = ((reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.out)) & 15) == 0 &&
                  a.q_stride % 8 == 0 && a.out_stride % 8 == 0;
  static std::atomic<uint64_t> granted{0};
  MS_TRY(grant_dynamic_smem(form_tc_kernel<DH, SH>, C::kSmem, granted));
  dim3 grid(a.hkv * a.n_splits, a.n_seqs, a.row_tiles);
  launch_pdl(form_tc_kernel<DH, SH>, grid, C::kThreads, C::kSmem, s, km, vm, a,
             __builtin_ctz((unsigned)a.bs), vec);
  MS_TRY(check_launch("form_tc_kernel"));
  return a.n_splits > 1 ? form_combine<__nv_bfloat16, true>(a, C::kTwin ? 64 : C::ST * kTileRows, DH, s) : MS_OK;
}

}  // namespace

int form_tc(const FormArgs& a, int dh, int rows, cudaStream_t s) {
  if (dh == 64) return rows <= 64 ? launch<64, kHalf>(a, s) : rows <= 128 ? launch<64, kOne>(a, s) : launch<64, kTwo>(a, s);
  return rows <= 64 ? launch<128, kHalf>(a, s) : rows <= 128 ? launch<128, kOne>(a, s) : launch<128, kTwo>(a, s);
}

}  // namespace ms
