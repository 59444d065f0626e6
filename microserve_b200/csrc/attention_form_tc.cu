// Attention with score forms over bf16 caches on tcgen05, for many rows:
// prompts and the rows of larger trees.
//
// With t = scale q k (capped, less slope x distance, -inf where unseen): p = 2^(t log2 e - m), O = sum p v,
// l = sum p, out = O / l, and where m grows O and l are scaled by 2^(old - new).
//
// A CTA takes ST streams of 128 rows each of one kv head of one sequence (row r is
// (token r / group, head-in-group r % group)) and a range of its keys, KC places
// at a step; the streams share the keys and values.
//   softmax warps  two threads (kParts) share a row, 32 scores of a step each: scores out of
//        TMEM, cap, distance, mask (bits, only where some row does not see all keys), p
//        rounded to bf16 back into TMEM over the scores (the operand type of the second product:
//        2^-8 of a p at most), and the sum of the rounded values
//        (the rounding of a dominant p cancels).  m is raised only when a row's maximum has
//        grown by more than 2^8, so O is rescaled a few times a row at most;
//   producer warp  TMA loads of whole pages (or parts of one), a lane a page, into
//        rings of their own for K and V;
//   MMA warp  S = Q K^T (both from shared memory) and O += P V (P in TMEM, V MN-major as it
//        lies in the page).  With SB score buffers the scores of the next SB steps are
//        there when p of this one is.
// Three shapes.  kTwo: 256 rows in two streams, all of TMEM, one CTA an SM.  kOne: 128 rows, two CTAs an
// SM.  kHalf: up to 64 rows of many sequences, twice in the tile; each copy takes half of the step's keys, so that no
// lane of the softmax idles, and the copies meet at the end; two CTAs an SM.
//
// What it measured, in a burst and under steady load (the 1000 W cap takes the clock to 1.7 GHz): 64 trees of 33 to
// 61 nodes, 32 heads over 8 of 128, 1 to 4 k keys (127 GFLOP, 733 MB) 208 and 242 us, 0.61 PFLOP/s and 3.5 TB/s in
// the burst; 4 prompts of up to 4096 with cap and prefix (309 GFLOP) 474 and 488 us, 0.65 PFLOP/s; 256 trees of 8
// nodes, 32 heads over 4 of 64, 1.3 k keys (351 MB) 92 and 97 us, 3.8 TB/s; one tree of 16 nodes over 32 k keys (134 MB)
// 36 and 37 us with the joining of its 37 ranges (kOne).
// Every pipe is half idle (tensor 24 to 42%, issue 31 to 56%, SFU 12 to 33%).  The bound of kTwo is the
// softmax of a step, about 2200 cycles (2700 with a cap) for 64 keys: TMEM load 160, maxima
// and vote 400, exponentials 750 to 1100 for the four warps of a scheduler, the store and its hand-off
// 350; products and copies are done by then.  The bound of kHalf at heads of 64 is the copy unit, 73
// cycles for a page of 2 KB.  Before its first and after its last step a CTA spends 12 to 16 thousand
// cycles on loads that depend on one another, Q and the result.
//
// Values that no row should meet: where a mask is needed the softmax warps look
// at the step's values first and put 0 for what is not finite.  If one of those belongs
// to a key that some row may see, every row of the CTA looks for such values among those that it sees
// (form_row_again).  So does a row whose sums are not finite at the end: large values that overflow
// float32 before the division by l (p reaches 2^8), or an infinite one in a step without a mask, which kHalf
// multiplies by the zeros that stand for the other copy's weights.
#include <cfloat>

#include "attention_form_device.cuh"

namespace ms {
namespace {

constexpr int kTileRows = 128;

// The shape of a CTA: up to 64 rows (twice, each copy half of the keys), 128, or 256 in two streams.  64 keys
// a step with two score buffers took trees of heads of 64 from 215 to 197 us against 128 with one.
enum Shape { kHalf, kOne, kTwo };

template <int DH, int SH>
struct TcCfg {
  static constexpr int ST = SH == kTwo ? 2 : 1;                  // streams of 128 rows
  static constexpr bool kTwin = SH == kHalf;
  static constexpr int KC = kTwin && DH == 64 ? 128 : 64;        // keys per step
  static constexpr int SB = kTwin ? 1 : 2;                       // score buffers
  static constexpr int kParts = kTwin && DH == 128 ? 1 : 2;      // threads that share a row's scores
  static constexpr int kTile = KC * DH * 2;                      // K or V of a step
  static constexpr int kSlots = SH == kTwo ? 144 : DH == 64 || kTwin ? 80 : 64;  // KB of K and V
  static constexpr int NK = (kSlots * 1024 / kTile + 1) / 2, NV = kSlots * 1024 / kTile / 2;
  static constexpr int kQ = kTileRows * DH * 2;
  static constexpr int kPCol = kTwin ? KC : 0;                   // p behind the scores, or over them
  static constexpr int kOCol = kTwin ? KC + KC / 2 : SB * KC;
  static constexpr int kStreamCols = kOCol + DH;
  static constexpr int kCols = ST == 2 ? 512 : 256;
  static constexpr int kSoft = 4 * kParts;                       // softmax warps of a stream
  static constexpr int kWarps = kSoft * ST + (ST == 2 ? 4 : 2);
  static constexpr int kThreads = kWarps * 32;
  static constexpr int kBars = 2 * NK + 2 * NV + 3 + ST * (2 * SB + 2);
  static constexpr int kShare = ST * kParts * kTileRows * 4;     // what the threads of a row tell one another
  static constexpr int kSmem = ST * kQ + (NK + NV) * kTile + kShare + kBars * 8 + 16;
  static_assert(KC / (kTwin ? 2 : 1) / kParts == 32, "32 scores of a step per thread");
  static_assert(ST * kStreamCols <= kCols, "TMEM columns");
  static_assert((3 - ST) * (kSmem + 1024) <= 228 * 1024 && kSmem <= 227 * 1024, "shared memory of an SM's CTAs");
  static_assert(!kTwin || 64 * DH * 4 + 64 * 8 <= NK * kTile, "the copies meet in the K ring");
};

// Descriptors with the 128-byte swizzle: atoms of 8 rows x 128 bytes, groups of 8 rows `stride` bytes
// apart.  K-major (Q, K): rows of 64 values (`lead` not used).  MN-major (V): 64 dimensions a row,
// blocks of 64 dimensions `lead` bytes apart.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lead, uint32_t stride) {
  uint64_t d = (uint64_t)((addr & 0x3FFFFu) >> 4);
  d |= (uint64_t)(lead >> 4) << 16;
  d |= (uint64_t)(stride >> 4) << 32;
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
// 32 lanes x N columns, N a multiple of 16 (loads) or 8 (stores).  Nothing that uses the values of a
// load comes between it and its wait: the outputs of the empty asm are the values.
__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
}
__device__ __forceinline__ void pin16(uint32_t* r) {
  asm volatile(""
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]));
  asm volatile(""
               : "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]));
}
template <int N>
__device__ __forceinline__ void tmem_ld(uint32_t addr, uint32_t (&r)[N]) {
  static_assert(N % 16 == 0, "whole loads");
#pragma unroll
  for (int c = 0; c < N; c += 16) tmem_ld16(addr + c, r + c);
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int c = 0; c < N; c += 16) pin16(r + c);
}
__device__ __forceinline__ void tmem_st8(uint32_t addr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(addr), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
template <int N>
__device__ __forceinline__ void tmem_st(uint32_t addr, const uint32_t (&r)[N]) {
  static_assert(N % 8 == 0, "whole stores");
#pragma unroll
  for (int c = 0; c < N; c += 8) tmem_st8(addr + c, r + c);
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

// (a NaN among the three is the result)
__device__ __forceinline__ float max3(float a, uint32_t b, uint32_t c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(__uint_as_float(b)), "f"(__uint_as_float(c)));
  return d;
}
__device__ __forceinline__ float min3(float a, uint32_t b, uint32_t c) {
  float d;
  asm("min.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(__uint_as_float(b)), "f"(__uint_as_float(c)));
  return d;
}

// The largest of 32 values, NaN if there is one; or the smallest.
template <bool kMax>
__device__ __forceinline__ float reduce(const uint32_t (&x)[32]) {
  float v[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) v[c] = __uint_as_float(x[c]);
#pragma unroll
  for (int c = 4; c < 32; c += 2) {
    float& to = v[(c >> 1) & 3];
    to = kMax ? max3(to, x[c], x[c + 1]) : min3(to, x[c], x[c + 1]);
  }
  if constexpr (kMax)
    return max3(max3(v[0], __float_as_uint(v[1]), __float_as_uint(v[2])), __float_as_uint(v[3]), __float_as_uint(v[3]));
  return fminf(fminf(v[0], v[1]), fminf(v[2], v[3]));
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

// 2^x of two values on the FMA units: x = n + f, |f| <= 1/2 (n by adding and taking off 1.5 2^23), 2^f
// by a cubic (fitted to the least maximum of the relative error, 1.0e-4, a fortieth of bf16's
// rounding), n into the exponent.  From -128 down that leaves a negative word, and 0 (an unseen key's p
// has to be 0: its value may be anything finite).  NaN is taken for -128: the caller sees to such a row.
__device__ __forceinline__ void exp2_fma(uint64_t v, float& lo, float& hi) {
  float a, b;
  unpair(v, a, b);
  v = pair(__float_as_uint(fmaxf(a, -128.f)), __float_as_uint(fmaxf(b, -128.f)));
  const uint64_t t = add2(v, twice(12582912.f)), n = add2(t, twice(-12582912.f));
  const uint64_t f = fma2(n, twice(-1.f), v);
  uint64_t c = fma2(f, twice(0.0551716684f), twice(0.242611122f));
  c = fma2(f, c, twice(0.693260986f));
  c = fma2(f, c, twice(0.999928074f));
  float tl, th, cl, ch;
  unpair(t, tl, th);
  unpair(c, cl, ch);
  lo = __int_as_float(max((int)(__float_as_uint(cl) + (__float_as_uint(tl) << 23)), 0));
  hi = __int_as_float(max((int)(__float_as_uint(ch) + (__float_as_uint(th) << 23)), 0));
}

// p = 2^(x - sub) of 32 values, rounded to bf16; returns the sum of the rounded values.
// kWay 0: x * mul; 1: the cap's series of x; 2: x as it is.  16 values at a time, each operation
// over all of them before the next: a packed operation with three fresh operands takes 3
// cycles, with one repeated from the operation before 2.
// kFma: a quarter of the exponentials on the FMA units, where the SFU (8 cycles a warp and value) is the
// bound (8B trees of 61 nodes 223 -> 207 us; half of them 213).
template <int kWay, bool kFma>
__device__ __forceinline__ float exps(const uint32_t (&x)[32], uint32_t* p16, float mul, float sub, const Cap& cap) {
  const uint64_t minus = twice(-sub);
  float sum[4] = {};
#pragma unroll
  for (int g = 0; g < 32; g += 16) {
    uint64_t v[8], c[8];
    uint32_t* p = p16 + g / 2;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = pair(x[g + 2 * j], x[g + 2 * j + 1]);
    if constexpr (kWay == 0) {
#pragma unroll
      for (int j = 0; j < 8; ++j) c[j] = fma2(v[j], twice(mul), minus);
    } else if constexpr (kWay == 1) {
      uint64_t w[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = mul2(v[j], v[j]);
#pragma unroll
      for (int j = 0; j < 8; ++j) c[j] = fma2(w[j], twice(cap.d4), twice(cap.d3));
#pragma unroll
      for (int j = 0; j < 8; ++j) c[j] = fma2(w[j], c[j], twice(cap.d2));
#pragma unroll
      for (int j = 0; j < 8; ++j) c[j] = fma2(w[j], c[j], twice(cap.d1));
#pragma unroll
      for (int j = 0; j < 8; ++j) c[j] = fma2(w[j], c[j], twice(cap.d0));
#pragma unroll
      for (int j = 0; j < 8; ++j) c[j] = fma2(v[j], c[j], minus);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) c[j] = add2(v[j], minus);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float lo, hi;
      if (kFma && (j == 1 || j == 4)) {
        exp2_fma(c[j], lo, hi);
      } else {
        unpair(c[j], lo, hi);
        lo = fast_exp2(lo);
        hi = fast_exp2(hi);
      }
      p[j] = pack2(lo, hi);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) add_bf16(p[j], sum[2 * (j & 1)], sum[2 * (j & 1) + 1]);
  }
  return (sum[0] + sum[1]) + (sum[2] + sum[3]);
}

template <int DH, int SH>
__global__ void __launch_bounds__(TcCfg<DH, SH>::kThreads, SH == kTwo ? 1 : 2)
    form_tc_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                   const __grid_constant__ FormArgs a, int log2_bs, int vec) {
  pdl_enter();
  using C = TcCfg<DH, SH>;
  constexpr int ST = C::ST, KC = C::KC, SB = C::SB, NK = C::NK, NV = C::NV, W = 32;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  const uint32_t raw = s_addr(smem_raw), q_s = raw;  // (1024-byte aligned, as declared)
  const uint32_t k_s = q_s + ST * C::kQ, v_s = k_s + NK * C::kTile, share = v_s + NV * C::kTile;
  const uint32_t bars = share + C::kShare;
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
  const int g = blockIdx.x / a.n_splits, b = a.order ? a.order[blockIdx.y] : blockIdx.y, split = blockIdx.x % a.n_splits;
  const int tile = (int)gridDim.z - 1 - (int)blockIdx.z;
  const FormSeq s = form_seq(a, b);
  constexpr int kCtaRows = C::kTwin ? 64 : ST * kTileRows;
  const int r0 = tile * kCtaRows;
  if (r0 >= s.qlen * a.group) return;
  const int nr = min(kCtaRows, s.qlen * a.group - r0);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int minpos = 0, maxpos = 0;
  if (needs_positions(a)) position_range(a, s, r0, nr, minpos, maxpos);
  const FormKeys keys = form_keys(a, s, minpos, maxpos);
  const int xbeg = min(split * a.split_len, keys.total);
  const int xend = split == a.n_splits - 1 ? keys.total : min(keys.total, xbeg + a.split_len);
  const int steps = (xend - xbeg + KC - 1) / KC;
  const int32_t* table = a.tables + (int64_t)b * a.max_blocks;
  constexpr int kProducer = C::kSoft * ST, kMma = kProducer + 1;

  if (threadIdx.x == 0) {
    for (int i = 0; i < NK; ++i) {
      mbar_init(k_full + 8 * i, 1);
      mbar_init(k_empty + 8 * i, 1);
    }
    for (int i = 0; i < NV; ++i) {
      mbar_init(v_full + 8 * i, 1);
      mbar_init(v_empty + 8 * i, 1);
    }
    mbar_init(q_ready, C::kSoft * ST);
    mbar_init(ended, 1);
    mbar_init(s_read, C::kSoft);
    for (int i = 0; i < ST * SB; ++i) {
      mbar_init(s_full + 8 * i, 1);
      mbar_init(p_ready + 8 * i, C::kSoft);
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
    if constexpr (ST == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    if (warp == kProducer) {
      // ---- loads
      static_assert(KC / 8 <= 32, "a lane for each box");
      const int box = min(a.bs, KC), boxes = KC / box, i = lane;
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
        const uint32_t bytes = (uint32_t)(n * box * DH * 2), off = i * box * DH * 2;
        const int ks = it % NK, vs = it % NV;
        bool ok = it < NK || mbar_wait(k_empty + 8 * ks, (it / NK - 1) & 1, stop, a.err);
        if (!__all_sync(0xffffffffu, ok)) break;
        if (lane == 0) mbar_expect_tx(k_full + 8 * ks, bytes);
        __syncwarp();
        if (row >= 0) tma_load_rows(k_s + ks * C::kTile + off, &kmap, k_full + 8 * ks, row);
        ++k_issued;
        ok = it < NV || mbar_wait(v_empty + 8 * vs, (it / NV - 1) & 1, stop, a.err);
        if (!__all_sync(0xffffffffu, ok)) break;
        if (lane == 0) mbar_expect_tx(v_full + 8 * vs, bytes);
        __syncwarp();
        if (row >= 0) tma_load_rows(v_s + vs * C::kTile + off, &vmap, v_full + 8 * vs, row);
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
      const uint32_t cols = ST == 2 ? 0u : __reduce_max_sync(0xffffffffu, tmem);
      auto wait = [&](uint32_t bar, uint32_t parity) {
        return __all_sync(0xffffffffu, mbar_wait(bar, parity, stop, a.err));
      };
      auto scores = [&](int it, int st) {
        const uint32_t d = cols + st * C::kStreamCols + (it % SB) * KC;
        const uint64_t qd = smem_desc(q_s + st * C::kQ, 16, 1024);
        const uint64_t kd = smem_desc(k_s + (it % NK) * C::kTile, 16, DH * 16);
#pragma unroll
        for (int k = 0; k < DH / 16; ++k)
          mma_ss(d, qd + (k >> 2) * (kTileRows * 128 / 16) + (k & 3) * 2,
                 kd + (k >> 2) * (1024 / 16) + (k & 3) * 2, id_s, k > 0, one);
        mma_commit(s_full + 8 * (st * SB + it % SB), one);
      };
      auto add_values = [&](int it, int st) {
        const uint32_t o = cols + st * C::kStreamCols + C::kOCol;
        const uint32_t p = cols + st * C::kStreamCols + C::kPCol + (it % SB) * KC;
        const uint64_t vd = smem_desc(v_s + (it % NV) * C::kTile, 1024, DH * 16);
#pragma unroll
        for (int k = 0; k < KC / 16; ++k) {
          // over the scores, each part's p starts where its scores did
          const int at = C::kTwin ? 8 * k : 8 * (k % (W / 16)) + k / (W / 16) * W;
          mma_ts(o, p + at, vd + k * (2 * DH * 16 / 16), id_o, it > 0 || k > 0, one);
        }
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
    if constexpr (ST == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 104;");
    // ---- softmax: lane t of stream st.  A row has kParts threads, in warps of one scheduler, that
    // share its maximum; in a twin two copies (lanes t and t + 64) with a maximum each
    const int st = warp / C::kSoft, part = (warp >> 2) % C::kParts, t = threadIdx.x & 127;
    const int mine = (C::kTwin ? (t >> 6) * (KC / 2) : 0) + part * W;  // the first of its keys in a step
    const int r = C::kTwin ? t & 63 : st * kTileRows + t;              // row of the CTA
    const bool live = r < nr;
    const bool warp_live = __any_sync(0xffffffffu, live);
    const int rr = r0 + (live ? r : 0), tok = s.t0 + rr / a.group, head = g * a.group + rr % a.group;
    const int pos = a.positions[tok];
    constexpr int kMyDims = DH / C::kParts;  // of the row's O and result
    const int dim0 = part * kMyDims;
    {
      // ---- Q into the swizzled tile: DH / 8 lanes a row, so that whole rows are read
      constexpr int kLanes = DH / 8, kRowsAtOnce = 32 / kLanes, kMine = kTileRows / C::kSoft;
      const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(a.q);
      const int c = lane % kLanes, first = (warp % C::kSoft) * kMine + lane / kLanes;
      uint4 v[kMine / kRowsAtOnce];
#pragma unroll
      for (int i = 0; i < kMine / kRowsAtOnce; ++i) {
        const int at = first + i * kRowsAtOnce, row = C::kTwin ? at & 63 : st * kTileRows + at;
        v[i] = make_uint4(0, 0, 0, 0);
        if (row < nr) {
          const int k = r0 + row, tk = k / a.group;
          const __nv_bfloat16* src =
              q + (int64_t)(s.t0 + tk) * a.q_stride + (int64_t)(g * a.group + k - tk * a.group) * DH + c * 8;
          if (vec) {
            v[i] = *reinterpret_cast<const uint4*>(src);
          } else {
            uint32_t w[4];
            for (int e = 0; e < 4; ++e)
              w[e] = (uint32_t)__bfloat16_as_ushort(src[2 * e]) | (uint32_t)__bfloat16_as_ushort(src[2 * e + 1]) << 16;
            v[i] = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < kMine / kRowsAtOnce; ++i) {
        const int at = first + i * kRowsAtOnce;
        sts128(q_s + st * C::kQ + at * 128 + (c >> 3) * (kTileRows * 128) + (((c & 7) ^ (at & 7)) << 4), v[i]);
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(q_ready);
    }
    // whether any thread of the warps that share these rows says so
    auto any_part = [&](bool pred) {
      if constexpr (C::kParts == 1) return __any_sync(0xffffffffu, pred) != 0;
      uint32_t any;
      asm volatile(
          "{\n\t.reg .pred p, q;\n\t"
          "setp.ne.u32 p, %1, 0;\n\t"
          "bar.red.or.pred q, %2, 64, p;\n\t"
          "selp.u32 %0, 1, 0, q;\n\t}"
          : "=r"(any)
          : "r"((uint32_t)pred), "r"(2 + 4 * st + (warp & 3))
          : "memory");
      return any != 0;
    };
    // whether a score (or a maximum of some) is too large for its product with `lin` to be taken as it is
    auto beyond = [](float v) { return fabsf(v) > kBig && v > -INFINITY; };
    // a wait that gives up sets `stop`: the later ones return at once, and nothing is written
    auto wait = [&](uint32_t bar, uint32_t parity) {
      mbar_wait(bar, parity, stop, a.err);
      __syncwarp();
      fence_after();
    };
    const uint32_t mine_at = share + ((st * C::kParts + part) * kTileRows + t) * 4;
    const uint32_t other_at = share + ((st * C::kParts + (part ^ (C::kParts - 1))) * kTileRows + t) * 4;
    const bool capped = a.softcap > 0.f, sloped = a.slopes != nullptr;
    Cap cap{};
    if (capped) cap.set(a);
    const float lin = a.scale * kLog2e, slope = sloped ? a.slopes[head] * kLog2e : 0.f;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_col = tmem + st * C::kStreamCols + lanes, o_col = s_col + C::kOCol + dim0;
    if constexpr (C::kTwin) {  // p of the other copy's keys: 0 for good
      uint32_t zero[W / 2] = {};
      tmem_st(s_col + C::kPCol + (KC / 4) * (1 - (t >> 6)) + part * (W / 2), zero);
    }
    // the steps that every row sees in full: those inside the prefix, and [free0, free1)
    const int lead = max(0, min(keys.a > 0 ? min(keys.a, s.pfx) : s.pfx, xend) - xbeg) / KC;
    const int oldest = a.window > 0 ? max(0, max(maxpos, 0) - a.window + 1) : 0;  // a key in every window
    const int free0 = (max(0, max(keys.a, oldest - keys.shift) - xbeg) + KC - 1) / KC;
    const int free1 = max(0, min((a.mask ? s.base : min(minpos, INT_MAX - 1) + 1) - keys.shift, xend) - xbeg) / KC;
    float m = -INFINITY, l = 0.f;
    // scores (as they come out of the product) above and below which a step is not plain
    float plain_top = -INFINITY;
    const float plain_bottom = capped ? -cap.limit : -INFINITY;
    for (int it = 0; it < steps; ++it) {
      const int x0 = xbeg + it * KC;
      const bool free = it < lead || (it >= free0 && it < free1);
      if (!free) {
        // ---- the step's values: nothing that is not finite may enter the product
        wait(v_full + 8 * (it % NV), (it / NV) & 1);
        const uint32_t vt = v_s + (it % NV) * C::kTile;
#pragma unroll 4
        for (int i = part * kTileRows + t; i < KC * DH / 8; i += C::kParts * kTileRows) {
          uint4 v = lds128(vt + i * 16);
          const uint4 n = make_uint4(not_finite(v.x), not_finite(v.y), not_finite(v.z), not_finite(v.w));
          if (n.x | n.y | n.z | n.w) {
            if (x0 + (i >> 6) / (DH / 64) * 8 + ((i >> 3) & 7) < xend) *odd = 1;
            sts128(vt + i * 16, make_uint4(v.x & ~n.x, v.y & ~n.y, v.z & ~n.z, v.w & ~n.w));
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      }
      // (the scores of this step came after the values of step it - SB or earlier were added: of
      // pv_done's two barriers, each has at most one phase open)
      wait(s_full + 8 * (st * SB + it % SB), (it / SB) & 1);
      const uint32_t s_at = s_col + (it % SB) * KC + mine;
      const uint32_t p_at = C::kTwin ? s_col + C::kPCol + mine / 2 : s_at;
      const uint32_t added = pv_done + 8 * (2 * st + ((it - 1) & 1)), added_parity = ((it - 1) >> 1) & 1;
      if (warp_live) {
        uint32_t x[W], p[W / 2];
        tmem_ld(s_at, x);
        if constexpr (C::kTwin) {  // the next scores may be computed
          fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(s_read);
        }
        float top = reduce<true>(x), bottom = INFINITY;
        if (capped) bottom = reduce<false>(x);
        // `way` says what the exponent still has to do (see exps).  Almost every step of a long context
        // is plain: all keys seen, no maximum grown, the cap's series good for all
        int way = capped ? 1 : 0;
        if (any_part(!free || sloped || !(top <= plain_top) || bottom < plain_bottom)) {
          // some score is beyond the cap's series
          const bool far = capped && any_part(!(top <= cap.limit && bottom >= -cap.limit));
          if (!free || sloped || far) {
            // ---- the scores as the exponent takes them: capped, with the distance, -inf where unseen
            way = capped || sloped ? 2 : 0;
            if (capped && far) {
#pragma unroll
              for (int c = 0; c < W; ++c) x[c] = __float_as_uint(cap.any(__uint_as_float(x[c])));
            } else if (capped) {
#pragma unroll
              for (int c = 0; c < W; c += 2) {
                float lo, hi;
                unpair(cap.series(pair(x[c], x[c + 1])), lo, hi);
                x[c] = __float_as_uint(lo);
                x[c + 1] = __float_as_uint(hi);
              }
            }
            if (sloped) {
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
              const uint32_t see = live ? (uint32_t)seen_places(a, s, keys, tok, pos, x0 + mine, xend) : 0u;
#pragma unroll
              for (int c = 0; c < W; ++c)
                if (!((see >> c) & 1)) x[c] = 0xff800000u;  // -inf
            }
            top = reduce<true>(x);
            if (way == 0) top *= lin;
          } else {
            top = capped ? cap.any(top) : top * lin;
          }
          // a seen score of NaN or +inf: the row is NaN, whatever becomes of the exponentials (see exp2_fma)
          if (!(top < INFINITY)) l = NAN;
          bool big = beyond(top) || beyond(m);
          if constexpr (C::kParts == 2) {
            st32(mine_at, top);
            big = any_part(big);
            top = fmaxf(top, ld32(other_at));
          } else {
            big = any_part(big);
          }
          if (way == 0 && big) {
            way = 2;
#pragma unroll
            for (int c = 0; c < W; ++c) x[c] = __float_as_uint(__uint_as_float(x[c]) * lin);
          }
          const bool grow = top > m + 8.f || (m == -INFINITY && top > m);
          // (the same for all threads of a row, and the barrier keeps `share` until all have read it)
          if (any_part(grow)) {
            const float mn = grow ? top : m;
            const float al = grow ? fast_exp2(m - mn) : 1.f;
            m = mn;
            l *= al;
            if (it > 0) {
              wait(added, added_parity);
#pragma unroll 1
              for (int c = 0; c < kMyDims; c += 16) {
                uint32_t o[16];
                tmem_ld(o_col + c, o);
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * al);
                tmem_st(o_col + c, o);
              }
            }
          }
          // (tanh(u) <= u for u >= 0: a capped score grows past the limit only if s * lin does)
          // An infinite score is never plain.
          plain_top = fminf((m + 8.f) / lin, capped ? cap.limit : FLT_MAX);
          if ((capped && m + 8.f < 0.f) || fabsf(m) > kBig) plain_top = -INFINITY;
        }
        const float sub = m == -INFINITY ? 0.f : m;
        if (way == 0)
          l += exps<0, !C::kTwin>(x, p, lin, sub, cap);
        else if (way == 1)
          l += exps<1, false>(x, p, lin, sub, cap);
        else
          l += exps<2, !C::kTwin>(x, p, lin, sub, cap);
        if constexpr (C::kTwin) {  // the values of the step before have been added: p may be replaced
          if (it > 0) wait(added, added_parity);
        }
        tmem_st(p_at, p);
        tmem_wait_st();
      } else if (C::kTwin) {
        if (lane == 0) mbar_arrive(s_read);
        // (p_ready has one phase open at a time: not ahead of the other warps' step before)
        if (it > 0) wait(added, added_parity);
      }
      fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_ready + 8 * (st * SB + it % SB));
    }
    if (steps > 0) wait(pv_done + 8 * (2 * st + ((steps - 1) & 1)), ((steps - 1) >> 1) & 1);
    if constexpr (C::kParts == 2) {
      st32(mine_at, l);
      asm volatile("bar.sync 1, %0;" ::"r"(ST * C::kSoft * 32) : "memory");
      l += ld32(other_at);
    }
    asm volatile("bar.sync 1, %0;" ::"r"(ST * C::kSoft * 32) : "memory");
    const int64_t part_row0 = ((((int64_t)b * a.hkv + g) * a.row_tiles + tile) * a.n_splits + split) * kCtaRows;
    // the second copies' (m, l, O) through shared memory (all copies and MMAs have ended)
    float w0 = 1.f, w1 = 0.f;
    const uint32_t meet = k_s + (t & 63) * 4, meet_o = meet + 512 + dim0 * 256;  // floats [value][row]
    if constexpr (C::kTwin) {
      if (t >= 64 && warp_live) {
        st32(meet, m);
        st32(meet + 256, l);
#pragma unroll
        for (int c = 0; c < kMyDims; c += 32) {
          uint32_t o[32] = {};
          if (steps > 0) tmem_ld(o_col + c, o);
#pragma unroll
          for (int e = 0; e < 32; ++e) st32(meet_o + (c + e) * 256, __uint_as_float(o[e]));
        }
      }
      asm volatile("bar.sync 1, %0;" ::"r"(ST * C::kSoft * 32) : "memory");
      if (t < 64 && warp_live) {
        const float m1 = ld32(meet), l1 = ld32(meet + 256), top = fmaxf(m, m1), sub = top == -INFINITY ? 0.f : top;
        w0 = fast_exp2(m - sub);
        w1 = fast_exp2(m1 - sub);
        l = l * w0 + l1 * w1;
        m = top;
      }
    }
    uint32_t again = 0;
    if (!*stop && warp_live && (!C::kTwin || t < 64)) {
      // ---- the warp's rows through its share of the Q tile, so that whole lines are written
      const float inv = l == 0.f ? 0.f : 1.f / l;
      __nv_bfloat16* dst =
          static_cast<__nv_bfloat16*>(a.out) + (int64_t)tok * a.out_stride + (int64_t)head * DH + dim0;
      if (a.n_splits > 1 && live && part == 0)
        *reinterpret_cast<float2*>(a.part_ml + (part_row0 + r) * 2) = make_float2(m, l);
      constexpr int kPitch = kMyDims * 2, kPieces = kPitch / 16;  // bytes and 16-byte pieces of a row
      const uint32_t stage = q_s + warp * 32 * kPitch;
      auto piece = [&](int row, int c) {
        return stage + row * kPitch + ((kPieces >= 8 ? c ^ (row & 7) : c ^ ((row >> 1) & 3)) << 4);
      };
      float far[2] = {};  // the largest sums, NaN if there is one
      // the sums of 16 dimensions
      auto sums = [&](int c, uint32_t (&o)[16]) {
        if (steps > 0)
          tmem_ld(o_col + c, o);
        else
          for (int e = 0; e < 16; ++e) o[e] = 0u;
        if constexpr (C::kTwin) {
#pragma unroll
          for (int e = 0; e < 16; ++e)
            o[e] = __float_as_uint(__uint_as_float(o[e]) * w0 + ld32(meet_o + (c + e) * 256) * w1);
        }
#pragma unroll
        for (int e = 0; e < 16; e += 2)
          far[(e >> 1) & 1] = max3_abs(far[(e >> 1) & 1], __uint_as_float(o[e]), __uint_as_float(o[e + 1]));
      };
      // rows that are read back: 32 / kPieces at once
      const int back = lane / kPieces, c_back = lane % kPieces;
      if (a.n_splits == 1) {
#pragma unroll
        for (int c = 0; c < kMyDims; c += 16) {
          uint32_t o[16], w[8];
          sums(c, o);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            w[e] = l == 0.f ? 0u : pack2(__uint_as_float(o[2 * e]) * inv, __uint_as_float(o[2 * e + 1]) * inv);
          sts128(piece(lane, c / 8), make_uint4(w[0], w[1], w[2], w[3]));
          sts128(piece(lane, c / 8 + 1), make_uint4(w[4], w[5], w[6], w[7]));
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
          const int row = i * (32 / kPieces) + back;
          __nv_bfloat16* to = reinterpret_cast<__nv_bfloat16*>(
              __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(dst), row));
          if (!__shfl_sync(0xffffffffu, (int)live, row)) continue;
          const uint4 v = lds128(piece(row, c_back));
          if (vec) {
            *reinterpret_cast<uint4*>(to + c_back * 8) = v;
          } else {
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
            for (int e = 0; e < 4; ++e) {
              to[c_back * 8 + 2 * e] = __ushort_as_bfloat16((unsigned short)(w[e] & 0xffffu));
              to[c_back * 8 + 2 * e + 1] = __ushort_as_bfloat16((unsigned short)(w[e] >> 16));
            }
          }
        }
      } else {
        float* po = a.part_o + (part_row0 + r - lane) * DH + dim0;  // of the warp's first row
#pragma unroll
        for (int half = 0; half < kMyDims; half += kMyDims / 2) {
#pragma unroll
          for (int c = 0; c < kMyDims / 2; c += 16) {
            uint32_t o[16];
            sums(half + c, o);
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * inv);
#pragma unroll
            for (int e = 0; e < 16; e += 4)
              sts128(piece(lane, (c + e) / 4), make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]));
          }
          __syncwarp();
#pragma unroll
          for (int i = 0; i < kPieces; ++i) {
            const int row = i * (32 / kPieces) + back;
            if (__shfl_sync(0xffffffffu, (int)live, row))
              *reinterpret_cast<uint4*>(po + (int64_t)row * DH + half + c_back * 4) = lds128(piece(row, c_back));
          }
          __syncwarp();
        }
      }
      // rows whose sums are not finite, or lack values that are not (with weights: else they are 0 or NaN anyway)
      again = __ballot_sync(0xffffffffu, live && (*odd || !(max3_abs(far[0], far[1], 0.f) < INFINITY)) && l > 0.f &&
                                             l < INFINITY);
    }
    constexpr int kThreads = ST * C::kSoft * 32;
    uint32_t any;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 p, %1, 0;\n\t"
        "bar.red.or.pred q, 1, %2, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(any)
        : "r"(again), "n"(kThreads)
        : "memory");
    if (any) {
      float* sums = reinterpret_cast<float*>(smem_raw + (k_s - raw));  // (the K ring: all products have ended)
      float common[(DH + 31) / 32];
      if (threadIdx.x < DH) sums[threadIdx.x] = 0.f;
      asm volatile("bar.sync 1, %0;" ::"n"(kThreads) : "memory");
      form_odd_values<__nv_bfloat16, DH>(a, s, keys, table, g, xbeg, xend, minpos, maxpos, 0, DH, warp, C::kSoft * ST,
                                         common);
#pragma unroll
      for (int e = 0; e < DH / 32; ++e)
        if (common[e] != 0.f) atomicAdd(sums + lane + 32 * e, common[e]);  // (infinities and NaN: in any order)
      asm volatile("bar.sync 1, %0;" ::"n"(kThreads) : "memory");
#pragma unroll
      for (int e = 0; e < DH / 32; ++e) common[e] = lane + 32 * e < kMyDims ? sums[dim0 + lane + 32 * e] : 0.f;
      for (; again; again &= again - 1) {
        const int row = r - lane + __ffs(again) - 1;
        form_row_again<__nv_bfloat16, DH, true>(a, s, keys, table, g, r0 + row, xbeg, xend, minpos, maxpos, dim0,
                                                dim0 + kMyDims, part_row0 + row, *odd != 0, common);
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
