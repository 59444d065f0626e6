// Device helpers of the matrix kernels of attention with score forms
// (attention_form_tma.cu, attention_form_tc.cu), and their tensor maps.
#pragma once

#include <cuda.h>

#include <cfloat>

#include "attention_form.cuh"

namespace ms {

constexpr int kErrTimeout = 5;
constexpr long long kFormWaitCycles = 1ll << 32;
constexpr float kLog2e = 1.4426950408889634f;
// Scores (in base 2) up to this size enter the exponent as one fma(product, scale, -maximum): the maximum's own
// rounding is 2^-4 at most, and cancels.  Larger ones are rounded like their maximum first, so that the
// largest gives exactly 2^0: at 2^33 a maximum is off by 2^9, and its weight would be 0 or infinite.
constexpr float kBig = 1048576.f;

__device__ __forceinline__ uint32_t s_addr(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool mbar_try_wait(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.b32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
// Waits for a phase, up to a limit; after that (or when another thread of the block gave
// up) false.
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile int* stop, int* err) {
  if (mbar_try_wait(bar, parity)) return true;
  const long long t0 = clock64();
  while (!mbar_try_wait(bar, parity)) {
    if (*stop) return false;
    if (clock64() - t0 > kFormWaitCycles) {
      *stop = 1;
      atomicCAS(err, 0, kErrTimeout);
      return false;
    }
  }
  return true;
}
// `row`: the first of the box's rows (a multiple of 8) of a pool's map (form_pool_map).
__device__ __forceinline__ void tma_load_rows(uint32_t dst, const CUtensorMap* map, uint32_t bar, int row) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %3, %3, %4}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(0), "r"(row >> 3)
      : "memory");
}
// 2^x by the SFU (ftz; 2^-inf = 0): 2 ulp of a result that is rounded to bf16 next.
__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float fast_rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float low_half(uint32_t x) { return __uint_as_float(x << 16); }
__device__ __forceinline__ float high_half(uint32_t x) { return __uint_as_float(x & 0xffff0000u); }

// The largest of |a|, |b| and |c|, NaN if one of them is.
__device__ __forceinline__ float max3_abs(float a, float b, float c) {
  float d;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
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
// cap tanh(u) in base 2, u = k s, k = scale / cap.  For |u| <= 0.75 an odd polynomial (tanh(u) = u (1 + c1 u^2 +
// .. + c4 u^8), fitted to the least maximum of |error|, 2.7e-7; no SFU), beyond that cap (1 - 2 / (1 + e^2u)),
// whose error is 2^-22 of the cap and so only good where the score is near it.
struct Cap {
  static constexpr float c1 = -0.333280453f, c2 = 0.132533633f, c3 = -0.0498660865f, c4 = 0.0127505842f;
  float d0, d1, d2, d3, d4;  // of s, s^3, ...
  float limit;               // of |s| for `series`
  float cap2, k;
  __device__ __forceinline__ void set(const FormArgs& a) {
    cap2 = fminf(a.softcap * kLog2e, FLT_MAX);
    k = fmaxf(a.scale / a.softcap, 1e-44f);  // (not 0: an infinite score is capped too)
    const float kk = k * k;
    d0 = a.scale * kLog2e;
    d1 = d0 * (c1 * kk);
    d2 = d0 * (c2 * kk * kk);
    d3 = d0 * (c3 * kk * kk * kk);
    d4 = d0 * (c4 * kk * kk * kk * kk);
    // k^8 has to stay within float32.  Below 1e-4 it does not, but up to |u| = 0.03 the terms that are lost do not
    // matter (s^2 stays within float32 too).  Scores that pass kBig are all computed alike: equal ones stay equal.
    limit = k > 1024.f || cap2 > kBig ? -1.f : k >= 1e-4f ? 0.75f / k : fminf(0.03f / k, 1e19f);
  }
  // |s| <= limit: the coefficients take k in.
  __device__ __forceinline__ uint64_t series(uint64_t v) const {
    const uint64_t w = mul2(v, v);
    uint64_t c = fma2(w, twice(d4), twice(d3));
    c = fma2(w, c, twice(d2));
    c = fma2(w, c, twice(d1));
    return mul2(v, fma2(w, c, twice(d0)));
  }
  // Any s (NaN stays NaN).
  __device__ __forceinline__ float any(float s) const {
    const float u = s * k, w = u * u;
    const float near = s * d0 * fmaf(w, fmaf(w, fmaf(w, fmaf(w, c4, c3), c2), c1), 1.f);
    const float far = cap2 * fmaf(-2.f, fast_rcp(1.f + fast_exp2(u * (2.f * kLog2e))), 1.f);
    return fabsf(u) <= 0.75f ? near : far;
  }
};

// Whether the keys of a tile depend on its tokens' positions.  A tree without a window takes every key up to its
// context's end, and a round trip less before its first load (1.1B trees 93.7 -> 91.4 us, 8B 218 -> 214).
__device__ __forceinline__ bool needs_positions(const FormArgs& a) { return !a.mask || a.window > 0; }
// Smallest and largest position of the tokens of rows [r0, r0 + nr) (the whole warp calls it).
__device__ __forceinline__ void position_range(const FormArgs& a, const FormSeq& s, int r0, int nr,
                                               int& lo, int& hi) {
  lo = INT_MAX;
  hi = INT_MIN;
  const int last = (r0 + nr - 1) / a.group;
  for (int t = r0 / a.group + (threadIdx.x & 31); t <= last; t += 32) {
    const int p = a.positions[s.t0 + t];
    lo = min(lo, p);
    hi = max(hi, p);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    lo = min(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = max(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
}

// Whether every row of the tile sees all N keys from place x0 on.
template <int N>
__device__ __forceinline__ bool all_see(const FormArgs& a, const FormSeq& s, const FormKeys& k, int x0,
                                        int xend, int minpos, int maxpos) {
  if (x0 + N > xend || (x0 < k.a && x0 + N > k.a)) return false;
  const int j0 = k.key(x0);
  if (j0 + N <= s.pfx) return true;
  return (a.mask ? j0 + N <= s.base : j0 + N - 1 <= minpos) &&
         (a.window <= 0 || maxpos - j0 < a.window);
}

__device__ __forceinline__ uint64_t low_bits(int n) {
  return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1;
}

// How many keys from j0 on (up to 64) lie before the window of a token at `pos`.
__device__ __forceinline__ int before_window(const FormArgs& a, int pos, int j0) {
  return (int)min(max((int64_t)pos - a.window - j0 + 1, (int64_t)0), (int64_t)64);
}

// Bit i: whether the token at row t of the batch (position pos) sees key j0 + i.
__device__ __forceinline__ uint64_t seen_from(const FormArgs& a, const FormSeq& s, int t, int pos, int j0) {
  uint64_t seen;
  if (a.mask) {
    const int node0 = j0 - s.base, w0 = node0 >> 5, sh = node0 & 31;
    const uint32_t* row = a.mask + (int64_t)t * a.mask_words;
    auto word = [&](int w) { return w >= 0 && w < a.mask_words ? (uint64_t)row[w] : 0ull; };
    seen = (word(w0) | word(w0 + 1) << 32) >> sh;
    if (sh) seen |= word(w0 + 2) << (64 - sh);
    seen = (seen & low_bits(s.qlen - node0)) | low_bits(-node0);
    if (a.window > 0) {
      // keys before the pass's own tokens by their place, those by their positions
      seen &= ~(low_bits(before_window(a, pos, j0)) & low_bits(-node0));
      for (int i = max(0, -node0); i < 64 && node0 + i < s.qlen; ++i)
        if (pos - a.positions[s.t0 + node0 + i] >= a.window) seen &= ~(1ull << i);
    }
  } else {
    seen = pos < j0 ? 0ull : low_bits(min(pos - j0, 63) + 1);
    if (a.window > 0) seen &= ~low_bits(before_window(a, pos, j0));
  }
  return seen | low_bits(s.pfx - j0);
}

// The same for the 64 places from x0 on, cut to those below xend.
__device__ __forceinline__ uint64_t seen_places(const FormArgs& a, const FormSeq& s, const FormKeys& k,
                                                int t, int pos, int x0, int xend) {
  uint64_t seen;
  if (x0 >= k.a) {
    seen = seen_from(a, s, t, pos, x0 + k.shift);
  } else {
    seen = seen_from(a, s, t, pos, x0);
    if (x0 + 64 > k.a) {
      const uint64_t first = low_bits(k.a - x0);
      seen = (seen & first) | (seen_from(a, s, t, pos, x0 + k.shift) & ~first);
    }
  }
  return seen & low_bits(xend - x0);
}

// The position of the key at place x.
__device__ __forceinline__ int key_position(const FormArgs& a, const FormSeq& s, const FormKeys& k, int x) {
  const int j = k.key(x), node = j - s.base;
  return a.mask && node >= 0 ? a.positions[s.t0 + min(node, s.qlen - 1)] : j;
}

// attention_form_tma.cu: the pool's rows of dh bf16 as (64 columns, 8 rows, dh / 64 column blocks, groups of
// 8 rows), boxes of `box` rows with the 128-byte swizzle: a whole page in one copy, of which a
// group of 8 rows fills dh / 64 swizzle atoms of 1024 bytes, one behind the other.  (A copy of 2
// KB costs 73 cycles of an SM's copy unit, one of 4 KB 96: with a copy for each column block
// the unit's 28 bytes a cycle were the bound.)
int form_pool_map(const void* pool, int64_t rows, int dh, int box, CUtensorMap* out);

}  // namespace ms
