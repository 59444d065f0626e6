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

// attention_form.cu: joins the KV ranges' partial results; `rows` per tile, maxima in base 2 or e.
template <typename T, bool kBase2>
int form_combine(const FormArgs& a, int rows, int dh, cudaStream_t s);

// attention_form_tma.cu: one tile of up to 32 rows a sequence (16 at heads of 128).
bool form_tma_takes(const ms_kv_cache& c);
int form_tma(const FormArgs& a, int dh, cudaStream_t s);
// attention_form_tc.cu: tiles of 64, 128 or 256 rows, for the caches that form_tma_takes.
int form_tc(const FormArgs& a, int dh, int rows, cudaStream_t s);

}  // namespace ms
