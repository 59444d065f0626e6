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

// 16 bytes of values as float32; `wide`: they are aligned to it.
template <typename T, int N>
__device__ __forceinline__ void load_vec(const T* p, bool wide, float (&f)[N]) {
  static_assert(N * sizeof(T) == 16, "16 bytes");
  if (wide) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    const T* x = reinterpret_cast<const T*>(&v);
#pragma unroll
    for (int e = 0; e < N; ++e) f[e] = to_f(x[e]);
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) f[e] = to_f(p[e]);
  }
}
// The row of key j in a pool, in elements.
template <int DH>
__device__ __forceinline__ int64_t form_key_row(const FormArgs& a, const int32_t* table, int g, int j) {
  return (((int64_t)form_block(a, table, j / a.bs) * a.hkv + g) * a.bs + j % a.bs) * DH;
}
// Adds to odd what is not finite of the values of 32 keys (a lane has one's row, `sees` a bit for each), in
// dimensions d0 + lane, d0 + lane + 32, .. below d1.
template <typename T, int DH>
__device__ __forceinline__ void add_odd(const T* v, int64_t at, uint32_t sees, int d0, int d1,
                                        float (&odd)[(DH + 31) / 32]) {
  const int lane = threadIdx.x & 31;
  if (sees == 0) return;
#pragma unroll 8
  for (int k = 0; k < 32; ++k) {
    const T* row = v + __shfl_sync(0xffffffffu, at, k) + d0 + lane;
#pragma unroll
    for (int e = 0; e < (DH + 31) / 32; ++e) {
      const float x = ((sees >> k) & 1) && d0 + lane + 32 * e < d1 ? to_f(row[32 * e]) : 0.f;
      if (!(fabsf(x) < INFINITY)) odd[e] += x;
    }
  }
}

// The sums of the values that are not finite of the keys that all rows of a tile see, as far as whole groups of 32 places
// show it: every `warps`th group, by the calling warp.
template <typename T, int DH>
__device__ __noinline__ void form_odd_values(const FormArgs& a, FormSeq s, FormKeys keys, const int32_t* table, int g,
                                             int xbeg, int xend, int minpos, int maxpos, int d0, int d1, int warp,
                                             int warps, float (&out)[(DH + 31) / 32]) {
  float odd[(DH + 31) / 32] = {};  // (not `out` itself: a load would wait for each possible store)
  for (int x0 = xbeg + 32 * warp; x0 < xend; x0 += 32 * warps)
    if (all_see<32>(a, s, keys, x0, xend, minpos, maxpos))
      add_odd<T, DH>(static_cast<const T*>(a.v), form_key_row<DH>(a, table, g, keys.key(x0 + (threadIdx.x & 31))),
                     0xffffffffu, d0, d1, odd);
#pragma unroll
  for (int e = 0; e < (DH + 31) / 32; ++e) out[e] = odd[e];
}

// Dimensions d0 to d1 of one row of a sequence once more, by a warp, after the kernel has written them: for rows whose
// weights are finite and whose sums of p v are not, or that may see values which the kernel left out because they are
// not finite.  Where a value that the row sees is infinite or NaN, so is the result, however small its weight.  Elsewhere
// what is not finite has overflowed: terms p reach 1 (2^8 on tcgen05) before the division.  Then the row is computed
// key by key, with the weights divided by their sum first, so that a mean of finite values is finite.  A lane a key for
// visibility and scores, dimensions over the lanes for the values; maxima in base 2 or e, as the kernel has them.
// part_row: the row's place in the workspace; common: form_odd_values of the same dimensions; masked: among the keys
// that not all rows see there may be such values too.  (4 prompts of up to 4096 tokens of which all see a NaN 0.55 -> 1.0
// ms, 256 trees of 8 nodes 0.22 -> 0.30; all values too large 0.46 s and 0.08.)
template <typename T, int DH, bool kBase2>
__device__ __noinline__ void form_row_again(const FormArgs& a, FormSeq s, FormKeys keys, const int32_t* table, int g,
                                            int rr, int xbeg, int xend, int minpos, int maxpos, int d0, int d1,
                                            int64_t part_row, bool masked,
                                            const float (&common)[(DH + 31) / 32]) {
  constexpr int kMine = (DH + 31) / 32;
  const int lane = threadIdx.x & 31;
  const T *kp = static_cast<const T*>(a.k), *vp = static_cast<const T*>(a.v);
  const int tok = s.t0 + rr / a.group, head = g * a.group + rr % a.group, pos = a.positions[tok];
  const T* q = static_cast<const T*>(a.q) + (int64_t)tok * a.q_stride + (int64_t)head * DH;
  T* o = static_cast<T*>(a.out) + (int64_t)tok * a.out_stride + (int64_t)head * DH;
  float* part = a.part_o + part_row * DH;
  const float slope = a.slopes ? a.slopes[head] : 0.f;
  // the key at place x0 + lane: its row in the pools, the distance, and whether the row sees it
  auto look = [&](int x0, int64_t& at, int& distance) {
    const int j = keys.key(min(x0 + lane, xend - 1));
    at = form_key_row<DH>(a, table, g, j);
    return x0 + lane < xend && form_sees(a, s, tok, pos, j, distance);
  };
  int64_t at;
  int distance = 0;
  float odd[kMine];  // the sum of the values that are not finite
#pragma unroll
  for (int e = 0; e < kMine; ++e) odd[e] = common[e];
  for (int x0 = xbeg; masked && x0 < xend; x0 += 32) {
    if (all_see<32>(a, s, keys, x0, xend, minpos, maxpos)) continue;
    const uint32_t sees = __ballot_sync(0xffffffffu, look(x0, at, distance));
    add_odd<T, DH>(vp, at, sees, d0, d1, odd);
  }
  bool over[kMine], any = false;
#pragma unroll
  for (int e = 0; e < kMine; ++e) {
    const int d = d0 + lane + 32 * e;
    over[e] = false;
    if (d >= d1) continue;
    if (odd[e] == 0.f) {
      over[e] = !(fabsf(a.n_splits == 1 ? to_f(o[d]) : part[d]) < INFINITY);
      any |= over[e];
    } else if (a.n_splits == 1) {
      o[d] = from_f<T>(odd[e]);
    } else {
      part[d] = odd[e];
    }
  }
  if (!__any_sync(0xffffffffu, any)) return;
  constexpr int kVec = 16 / (int)sizeof(T);
  const bool q_wide = reinterpret_cast<uintptr_t>(q) % 16 == 0, k_wide = reinterpret_cast<uintptr_t>(kp) % 16 == 0;
  auto score = [&](int x0) {
    const bool seen = look(x0, at, distance);
    float v = 0.f;
    for (int d = 0; d < DH; d += kVec) {
      float qd[kVec], kd[kVec];
      load_vec(q + d, q_wide, qd);
      load_vec(kp + at + d, k_wide, kd);
#pragma unroll
      for (int e = 0; e < kVec; ++e) v = fmaf(qd[e], kd[e], v);
    }
    v *= a.scale;
    if (a.softcap > 0.f && !(fabsf(v) <= 1e-4f * a.softcap)) v = a.softcap * tanhf(v / a.softcap);
    if (a.slopes) v -= slope * fabsf((float)distance);
    return !seen ? -INFINITY : kBase2 ? v * 1.4426950408889634f : v;
  };
  auto power = [](float v) { return v == -INFINITY ? 0.f : kBase2 ? exp2f(v) : expf(v); };
  float m = -INFINITY, l = 0.f, mean[kMine] = {};
  for (int x0 = xbeg; x0 < xend; x0 += 32) {
    const float v = score(x0), mn = fmaxf(m, warp_max(v));
    if (mn == -INFINITY) continue;
    l = l * power(m - mn) + warp_sum(power(v - mn));
    m = mn;
  }
  const float inv = 1.f / l;  // (the weights are not all 0: the sums were not)
  for (int x0 = xbeg; x0 < xend; x0 += 32) {
    const float w = power(score(x0) - m) * inv;
    for (int k = 0; k < 32; ++k) {
      const float wk = __shfl_sync(0xffffffffu, w, k);
      const int64_t ak = __shfl_sync(0xffffffffu, at, k) + d0 + lane;
      if (wk == 0.f) continue;
#pragma unroll
      for (int e = 0; e < kMine; ++e)
        if (d0 + lane + 32 * e < d1) mean[e] = fmaf(wk, to_f(vp[ak + 32 * e]), mean[e]);
    }
  }
#pragma unroll
  for (int e = 0; e < kMine; ++e) {
    if (!over[e]) continue;
    const int d = d0 + lane + 32 * e;
    if (a.n_splits == 1)
      o[d] = from_f<T>(mean[e]);
    else
      part[d] = mean[e];
  }
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
