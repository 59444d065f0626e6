// Paged attention with score forms: what its kernels share (attention_form*.cu).
//
//   o[t, h] = sum_j softmax_j(x[t, h, j]) v[j],
//   x = cap tanh(s / cap) - slope_h |p_t - p_j|,   s = scale q[t, h] . k[j],
// over the keys j that token t sees:
//   j < prefix_b,  or  seen(t, j) and p_t - p_j < window,
//   seen = p_j <= p_t, or with a tree mask: j < base (the cached context) or
//   bit j - base of the token's mask.
// base = context - q_len.  p_j is j, and with a tree mask the position of the
// token itself for the pass's own tokens (siblings share one).  A token that
// sees no key gives 0.
#pragma once

#include <climits>

#include "common.cuh"

namespace ms {

struct FormArgs {
  const void *q, *k, *v;
  void* out;
  int64_t q_stride, out_stride;  // elements between tokens
  const int32_t *q_start, *context_lens, *positions, *tables;
  const int32_t* prefix;  // null: none
  const float* slopes;    // null: none
  const int32_t* order;   // the sequences, longest first (null: as they come)
  const uint32_t* mask;   // null: causal
  int mask_words, window;
  float scale, softcap;   // softcap 0: none
  int n_tokens, n_seqs, max_blocks, max_q, bs, num_blocks, hq, hkv, group;
  int row_tiles, n_splits, split_len;
  // n_splits > 1: (unit, row, dh) results of the range alone, and (unit, row, 2) its maximum and sum of weights
  float *part_o, *part_ml;
  int* err;
};

struct FormSeq {
  int t0, qlen, ctx, base, pfx;
};

// Sequence b, with lengths that do not fit the call's arrays cut to them (and
// reported): no later access can leave the arrays.
__device__ __forceinline__ FormSeq form_seq(const FormArgs& a, int b) {
  FormSeq s;
  s.t0 = a.q_start[b];
  int end = a.q_start[b + 1];
  s.ctx = a.context_lens[b];
  s.pfx = a.prefix ? a.prefix[b] : 0;
  const int64_t held = (int64_t)a.max_blocks * a.bs;
  if (s.t0 < 0 || end > a.n_tokens || end < s.t0 || end - s.t0 > a.max_q || s.ctx < 0 || s.ctx > held) {
    if (threadIdx.x == 0) raise_device_error(a.err, kErrLength);
    s.t0 = min(max(s.t0, 0), a.n_tokens);
    end = min(max(end, s.t0), a.n_tokens);
    end = min(end, s.t0 + a.max_q);
    s.ctx = s.ctx < 0 ? 0 : s.ctx > held ? (int)held : s.ctx;
  }
  s.qlen = end - s.t0;
  s.base = s.ctx - s.qlen;
  s.pfx = min(max(s.pfx, 0), s.ctx);
  return s;
}

// The keys that some row of a tile may see, in whole pages from the first of
// them: [0, a) and then [a + shift, end), as places x in [0, total).  A window
// behind a prefix leaves a hole between the two; without one a is 0.
struct FormKeys {
  int a, shift, total, end;
  __device__ __forceinline__ int key(int x) const { return x < a ? x : x + shift; }
};

__device__ __forceinline__ FormKeys form_keys(const FormArgs& f, const FormSeq& s, int minpos, int maxpos) {
  FormKeys k;
  const int past = maxpos < 0 ? 0 : maxpos < s.ctx ? maxpos + 1 : s.ctx;  // maxpos + 1, without overflow
  k.end = max(f.mask ? s.ctx : past, s.pfx);
  int lo = f.window > 0 ? max(0, max(minpos, 0) - f.window + 1) : 0;
  if (f.mask) lo = min(lo, max(s.base, 0));
  lo = min(lo, k.end) / f.bs * f.bs;
  k.a = (s.pfx + f.bs - 1) / f.bs * f.bs;
  if (k.a >= lo) {
    if (s.pfx > 0) lo = 0;
    k.a = 0;
  }
  k.shift = lo - k.a;
  k.total = k.a + k.end - lo;
  return k;
}

// The block that holds key j (a block outside the pool is reported, and read as block 0).
__device__ __forceinline__ int form_block(const FormArgs& a, const int32_t* table, int page) {
  int blk = table[page];
  if (blk < 0 || blk >= a.num_blocks) {
    raise_device_error(a.err, kErrBlock);
    blk = 0;
  }
  return blk;
}

// Whether the token at row `t` of the batch (position pos) sees key j < end, and the distance.
__device__ __forceinline__ bool form_sees(const FormArgs& a, const FormSeq& s, int t, int pos, int j,
                                          int& distance) {
  const int node = j - s.base;
  bool seen;
  if (a.mask && node >= 0) {
    distance = pos - a.positions[s.t0 + min(node, s.qlen - 1)];
    seen = node < s.qlen && (node >> 5) < a.mask_words &&
           (a.mask[(int64_t)t * a.mask_words + (node >> 5)] >> (node & 31)) & 1;
  } else {
    distance = pos - j;
    seen = a.mask || j <= pos;
  }
  return j < s.pfx || (seen && (a.window <= 0 || distance < a.window));
}

// One row of a sequence by a warp, key by key: what the kernels give when their sums of p v are not finite, whose
// terms p reach 1 (2^8 on tcgen05) before the division.  The weights are divided by their sum
// first, so that a mean of finite values is finite.  A lane a key for the scores, dimensions d0 to d1 over the lanes for
// the means; maxima in base 2 or e, as the kernel has them.  part_row: the row's place in the workspace.
template <typename T, int DH, bool kBase2>
__device__ __noinline__ void form_row_by_key(const FormArgs& a, FormSeq s, FormKeys keys, const int32_t* table, int g,
                                             int rr, int xbeg, int xend, int d0, int d1, int64_t part_row) {
  constexpr int kMine = (DH + 31) / 32;
  const int lane = threadIdx.x & 31;
  const T *kp = static_cast<const T*>(a.k), *vp = static_cast<const T*>(a.v);
  const int tok = s.t0 + rr / a.group, head = g * a.group + rr % a.group, pos = a.positions[tok];
  const T* q = static_cast<const T*>(a.q) + (int64_t)tok * a.q_stride + (int64_t)head * DH;
  const float slope = a.slopes ? a.slopes[head] : 0.f;
  auto score = [&](int x0, int64_t& at, bool& seen) {
    const int j = keys.key(min(x0 + lane, xend - 1));
    int distance = 0;
    seen = x0 + lane < xend && form_sees(a, s, tok, pos, j, distance);
    at = (((int64_t)form_block(a, table, j / a.bs) * a.hkv + g) * a.bs + j % a.bs) * DH;
    float v = 0.f;
    for (int d = 0; d < DH; ++d) v = fmaf(to_f(q[d]), to_f(kp[at + d]), v);
    v *= a.scale;
    if (a.softcap > 0.f && !(fabsf(v) <= 1e-4f * a.softcap)) v = a.softcap * tanhf(v / a.softcap);
    if (a.slopes) v -= slope * fabsf((float)distance);
    return !seen ? -INFINITY : kBase2 ? v * 1.4426950408889634f : v;
  };
  auto power = [](float v) { return kBase2 ? exp2f(v) : expf(v); };
  float m = -INFINITY, l = 0.f, mean[kMine] = {};
  int64_t at;
  bool seen;
  for (int x0 = xbeg; x0 < xend; x0 += 32) {
    const float v = score(x0, at, seen), mn = fmaxf(m, warp_max(v)), sub = mn == -INFINITY ? 0.f : mn;
    l = l * (m == -INFINITY ? 0.f : power(m - sub)) + warp_sum(seen ? power(v - sub) : 0.f);
    m = mn;
  }
  const float sub = m == -INFINITY ? 0.f : m, inv = l == 0.f ? 0.f : 1.f / l;
  for (int x0 = xbeg; x0 < xend; x0 += 32) {
    const float v = score(x0, at, seen), w = seen ? power(v - sub) * inv : 0.f;
    const uint32_t all = __ballot_sync(0xffffffffu, seen), some = __ballot_sync(0xffffffffu, seen && v > -INFINITY);
    for (int k = 0; k < 32; ++k) {
      const float wk = __shfl_sync(0xffffffffu, w, k);
      const int64_t ak = __shfl_sync(0xffffffffu, at, k);
      if (!((all >> k) & 1)) continue;
#pragma unroll
      for (int e = 0; e < kMine; ++e) {
        if (d0 + lane + 32 * e >= d1) continue;
        const float vk = to_f(vp[ak + d0 + lane + 32 * e]);
        // (an infinite value counts however small its weight is)
        mean[e] = fmaf(wk == 0.f && ((some >> k) & 1) && !(fabsf(vk) < INFINITY) ? 1.f : wk, vk, mean[e]);
      }
    }
  }
  T* o = static_cast<T*>(a.out) + (int64_t)tok * a.out_stride + (int64_t)head * DH;
#pragma unroll
  for (int e = 0; e < kMine; ++e) {
    const int d = d0 + lane + 32 * e;
    if (d >= d1) continue;
    if (a.n_splits == 1)
      o[d] = from_f<T>(mean[e]);
    else
      a.part_o[part_row * DH + d] = mean[e];
  }
  if (a.n_splits > 1 && lane == 0) {
    a.part_ml[part_row * 2] = m;
    a.part_ml[part_row * 2 + 1] = l;
  }
}

// attention_form.cu: joins the KV ranges' partial results; `rows` per tile, maxima in base 2 or e.
template <typename T, bool kBase2>
int form_combine(const FormArgs& a, int rows, int dh, cudaStream_t s);

// attention_form_tma.cu: one tile of up to 32 rows a sequence (16 at heads of 128).
bool form_tma_takes(const ms_kv_cache& c);
int form_tma(const FormArgs& a, int dh, cudaStream_t s);
// attention_form_tc.cu: tiles of 64, 128 or 256 rows, for the caches that form_tma_takes.
int form_tc(const FormArgs& a, int dh, int rows, cudaStream_t s);

}  // namespace ms
