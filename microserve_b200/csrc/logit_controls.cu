// Per-request controls on logits before a draw: penalties for repeated
// tokens, sparse biases and grammar masks, and the token counts they read.
//
// For row i of request b (it sees the request's first f + i proposals as
// already said) and token v, with x the raw logit, all in float32:
//   c = counts[slot][v] + #{j < f + i : proposal j == v}   generated so far
//   s = seen bit of v, or v among those proposals          prompt or generated
//   y = s ? (x > 0 ? x / repetition : x * repetition) : x
//   y = (y - frequency * c) - (c > 0 ? presence : 0)
//   y = y + bias(v);   out = mask bit of v unset ? -inf : y
// The operations are rounded one by one (no contraction), as elementary
// float32 operations would be.
#include <cmath>

#include "common.cuh"

namespace ms {
namespace {

constexpr int kThreads = 256;
constexpr int kUnroll = 4;
constexpr int kSlice = kThreads * 4 * kUnroll;  // tokens per CTA
constexpr int kMaxProposals = 64;               // the draft lanes of one round

struct ControlArgs {
  const float* in;
  int64_t in_stride;
  float* out;
  int64_t out_stride;
  int n_requests, rows, rows_per_cta, vocab, words;
  ms_logit_controls c;
  int* err;
};

struct Penalty {
  float rep, pres, freq;
};

__device__ __forceinline__ float penalise(float x, const Penalty& p, int count) {
  float y = x > 0.f ? __fdiv_rn(x, p.rep) : __fmul_rn(x, p.rep);
  y = __fsub_rn(y, __fmul_rn(p.freq, (float)count));
  return count > 0 ? __fsub_rn(y, p.pres) : y;
}

// One CTA: kSlice tokens of rows_per_cta rows of one request.
template <bool VEC, bool INPLACE>
__global__ void __launch_bounds__(kThreads) logit_controls_kernel(ControlArgs a) {
  pdl_enter();
  __shared__ int s_prop[kMaxProposals];  // proposals inside this slice: id - first token
  __shared__ int s_when[kMaxProposals];  // and their positions
  __shared__ int s_nprop;
  __shared__ int s_bias_lo, s_bias_hi;
  __shared__ float s_bias[kSlice];
  const ms_logit_controls& c = a.c;
  const int tid = threadIdx.x;
  const int t0 = blockIdx.x * kSlice;
  const int b = blockIdx.y;
  const int r0 = blockIdx.z * a.rows_per_cta;
  const int r1 = min(a.rows, r0 + a.rows_per_cta);
  const int n_here = min(kSlice, a.vocab - t0);

  int slot = c.slots ? c.slots[b] : -1;
  if (slot >= c.n_slots) {
    if (tid == 0) raise_device_error(a.err, kErrSlot);
    slot = -1;
  }
  if (slot < 0) slot = -1;
  Penalty p{1.f, 0.f, 0.f};
  if (slot >= 0) p = Penalty{c.penalties[3 * b], c.penalties[3 * b + 1], c.penalties[3 * b + 2]};

  // What of the proposals and the bias list falls into this slice.
  if (tid == 0) s_nprop = 0;
  if (tid < 2 && c.bias_start) {
    int lo = c.bias_start[b], hi = c.bias_start[b + 1];
    if (lo < 0 || hi < lo || hi > c.n_bias) {
      raise_device_error(a.err, kErrOrder);
      lo = hi = 0;
    }
    // first entry at or past the slice's first / one-past-last token
    const int want = tid == 0 ? t0 : t0 + n_here;
    const bool edge = tid == 0 ? blockIdx.x == 0 : blockIdx.x + 1 == gridDim.x;
    if (!edge) {
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (c.bias_ids[mid] < want) lo = mid + 1; else hi = mid;
      }
    } else if (tid == 1) {
      lo = hi;  // the last slice also takes (and reports) ids past the vocabulary
    }
    (tid == 0 ? s_bias_lo : s_bias_hi) = lo;
  }
  __syncthreads();
  if (slot >= 0 && c.proposals && tid < c.n_proposals) {
    const int v = c.proposals[(int64_t)tid * a.n_requests + b];
    if (v < 0 || v >= a.vocab) {
      raise_device_error(a.err, kErrToken);
    } else if (v >= t0 && v < t0 + n_here) {
      const int k = atomicAdd(&s_nprop, 1);
      s_prop[k] = v - t0;
      s_when[k] = tid;
    }
  }
  const int blo = c.bias_start ? s_bias_lo : 0, bhi = c.bias_start ? s_bias_hi : 0;
  const bool biased = bhi > blo;
  if (biased) {
    for (int i = tid; i < n_here; i += kThreads) s_bias[i] = 0.f;
    __syncthreads();
    const int first = c.bias_start[b];
    for (int e = blo + tid; e < bhi; e += kThreads) {
      const int v = c.bias_ids[e];
      if (v < 0 || v >= a.vocab)
        raise_device_error(a.err, kErrToken);
      else if (e > first && c.bias_ids[e - 1] >= v)
        raise_device_error(a.err, kErrOrder);  // not ascending: the entry is skipped
      else if (v >= t0 && v < t0 + n_here)
        s_bias[v - t0] = c.bias_values[e];
    }
  }
  __syncthreads();
  const int nprop = s_nprop;

  // Token group u of this thread: VEC: 4 tokens at 4 * (u * kThreads + tid);
  // else single tokens at (4 u + k) * kThreads + tid, so a warp's 32 tokens
  // are one bit word.
  auto token = [&](int u, int k) {
    return VEC ? 4 * (u * kThreads + tid) + k : (4 * u + k) * kThreads + tid;
  };
  auto bits_of = [&](const uint32_t* words, int u) -> uint32_t {
    if constexpr (VEC) {
      const int o = token(u, 0);
      return o < n_here ? (__ldg(words + ((t0 + o) >> 5)) >> (o & 31)) & 15u : 0u;
    } else {
      uint32_t r = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int o = token(u, k);
        if (o < n_here) r |= ((__ldg(words + ((t0 + o) >> 5)) >> (o & 31)) & 1u) << k;
      }
      return r;
    }
  };
  uint32_t seen[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u)
    seen[u] = slot >= 0 ? bits_of(c.seen + (int64_t)slot * a.words, u) : 0u;
  const int32_t* count_row = slot >= 0 ? c.counts + (int64_t)slot * a.vocab + t0 : nullptr;

  for (int r = r0; r < r1; ++r) {
    const int64_t row = (int64_t)b * a.rows + r;
    const float* xin = a.in + row * a.in_stride + t0;
    float* yout = a.out + row * a.out_stride + t0;
    int mrow = c.mask_rows ? c.mask_rows[row] : -1;
    if (mrow >= c.n_masks) {
      if (tid == 0) raise_device_error(a.err, kErrMask);
      mrow = -1;
    }
    const uint32_t* mask = mrow >= 0 ? c.masks + (int64_t)mrow * a.words : nullptr;
    const int visible = c.first_proposal + r;  // proposals this row sees
    float v[kUnroll][4];
    if constexpr (!INPLACE) {
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        if constexpr (VEC) {
          const int o = token(u, 0);
          float4 q = make_float4(0.f, 0.f, 0.f, 0.f);
          if (o < n_here) q = __ldcs(reinterpret_cast<const float4*>(xin + o));
          v[u][0] = q.x, v[u][1] = q.y, v[u][2] = q.z, v[u][3] = q.w;
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int o = token(u, k);
            v[u][k] = o < n_here ? __ldcs(xin + o) : 0.f;
          }
        }
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (token(u, 0) >= n_here) break;
      uint32_t said = seen[u];
      for (int j = 0; j < nprop; ++j) {
        if (s_when[j] >= visible) continue;
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (s_prop[j] == token(u, k)) said |= 1u << k;
      }
      const uint32_t ok = mask ? bits_of(mask, u) : 15u;
      uint32_t touched = said;
      if (biased) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int o = token(u, k);
          if (o < n_here && s_bias[o] != 0.f) touched |= 1u << k;
        }
      }
      if (touched & ok) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (!((touched & ok) >> k & 1u)) continue;
          const int o = token(u, k);
          float y = INPLACE ? xin[o] : v[u][k];
          if (said >> k & 1u) {
            int n = count_row[o];
            for (int j = 0; j < nprop; ++j) n += s_prop[j] == o && s_when[j] < visible;
            y = penalise(y, p, n);
          }
          if (biased && s_bias[o] != 0.f) y = __fadd_rn(y, s_bias[o]);
          v[u][k] = y;
          if (INPLACE) yout[o] = y;
        }
      }
      if (ok != 15u) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (ok >> k & 1u) continue;
          v[u][k] = -INFINITY;
          if (INPLACE && (!VEC || ok != 0u) && token(u, k) < n_here) yout[token(u, k)] = -INFINITY;
        }
        if (INPLACE && VEC && ok == 0u)
          *reinterpret_cast<float4*>(yout + token(u, 0)) =
              make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
      }
    }
    if constexpr (!INPLACE) {
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        if constexpr (VEC) {
          const int o = token(u, 0);
          if (o < n_here)
            __stcs(reinterpret_cast<float4*>(yout + o),
                   make_float4(v[u][0], v[u][1], v[u][2], v[u][3]));
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int o = token(u, k);
            if (o < n_here) __stcs(yout + o, v[u][k]);
          }
        }
      }
    }
  }
}

// Sequence i's tokens [0, len) into the counts and seen bits of its slot;
// the first n_prompt[i] set only the bit.  Integer atomics: the result does
// not depend on their order, and a slot may appear more than once.
__global__ void token_counts_append_kernel(int32_t* counts, uint32_t* seen, int n_slots, int vocab,
                                           int words, const int32_t* __restrict__ slots,
                                           const int32_t* __restrict__ tokens,
                                           const int64_t* __restrict__ row_start,
                                           int64_t row_stride, const int32_t* __restrict__ lens,
                                           int len_add, int max_len,
                                           const int32_t* __restrict__ n_prompt, int* err) {
  pdl_enter();
  const int i = blockIdx.x;
  const int slot = slots[i];
  if (slot < 0) return;  // a request without counts
  if (slot >= n_slots) {
    if (threadIdx.x == 0) raise_device_error(err, kErrSlot);
    return;
  }
  const int len = min((lens ? lens[i] : 0) + len_add, max_len);
  const int prompt = n_prompt ? n_prompt[i] : 0;
  const int32_t* row = tokens + (row_start ? row_start[i] : (int64_t)i * row_stride);
  for (int t = blockIdx.y * blockDim.x + threadIdx.x; t < len; t += gridDim.y * blockDim.x) {
    const int v = row[t];
    if (v < 0 || v >= vocab) {
      raise_device_error(err, kErrToken);
      continue;
    }
    if (t >= prompt) atomicAdd(counts + (int64_t)slot * vocab + v, 1);
    atomicOr(seen + (int64_t)slot * words + (v >> 5), 1u << (v & 31));
  }
}

__global__ void token_counts_reset_kernel(int32_t* counts, uint32_t* seen, int n_slots, int vocab,
                                          int words, const int32_t* __restrict__ slots, int* err) {
  pdl_enter();
  const int slot = slots[blockIdx.y];
  if (slot < 0) return;
  if (slot >= n_slots) {
    if (threadIdx.x == 0) raise_device_error(err, kErrSlot);
    return;
  }
  const int stride = gridDim.x * blockDim.x;
  for (int v = blockIdx.x * blockDim.x + threadIdx.x; v < vocab; v += stride)
    counts[(int64_t)slot * vocab + v] = 0;
  for (int w = blockIdx.x * blockDim.x + threadIdx.x; w < words; w += stride)
    seen[(int64_t)slot * words + w] = 0u;
}

int validate_controls(const ms_logit_controls* c, int n_requests, int rows_per_request) {
  MS_REQUIRE(c != nullptr, "ms_logit_controls: null");
  if (c->slots) {
    MS_REQUIRE(c->penalties && c->counts && c->seen && c->n_slots > 0,
               "ms_logit_controls: slots need penalties, counts and seen");
  }
  if (c->proposals) {
    MS_REQUIRE(c->n_proposals > 0 && c->n_proposals <= kMaxProposals,
               "ms_logit_controls: %d proposals (1..%d)", c->n_proposals, kMaxProposals);
  }
  MS_REQUIRE(c->first_proposal >= 0, "ms_logit_controls: first_proposal %d", c->first_proposal);
  MS_REQUIRE(!c->proposals || c->first_proposal + rows_per_request - 1 <= c->n_proposals,
             "ms_logit_controls: the last row sees %d proposals of %d",
             c->first_proposal + rows_per_request - 1, c->n_proposals);
  if (c->bias_start)
    MS_REQUIRE(c->n_bias == 0 || (c->n_bias > 0 && c->bias_ids && c->bias_values),
               "ms_logit_controls: bias_start needs bias_ids and bias_values");
  if (c->mask_rows)
    MS_REQUIRE(c->masks && c->n_masks > 0, "ms_logit_controls: mask_rows need masks");
  (void)n_requests;
  return MS_OK;
}

}  // namespace
}  // namespace ms

using namespace ms;

extern "C" int ms_apply_logit_controls(const float* logits, int64_t row_stride, float* out,
                                       int64_t out_stride, int n_requests, int rows_per_request,
                                       int vocab, const ms_logit_controls* controls,
                                       void* stream) {
  MS_REQUIRE(n_requests >= 0 && rows_per_request > 0 && vocab > 0,
             "ms_apply_logit_controls: bad sizes (%d requests x %d rows, vocab %d)", n_requests,
             rows_per_request, vocab);
  MS_TRY(validate_controls(controls, n_requests, rows_per_request));
  if (n_requests == 0) return MS_OK;
  MS_REQUIRE(logits && out, "ms_apply_logit_controls: null pointer");
  MS_REQUIRE(row_stride >= vocab && out_stride >= vocab,
             "ms_apply_logit_controls: row stride below the vocabulary");
  MS_REQUIRE(n_requests <= 65535 && rows_per_request <= 65535,
             "ms_apply_logit_controls: more than 65535 requests or rows per request");
  const bool in_place = logits == out;
  MS_REQUIRE(!in_place || row_stride == out_stride,
             "ms_apply_logit_controls: in place with two row strides");
  const int64_t n_rows = (int64_t)n_requests * rows_per_request;
  if (!in_place) {
    const float* in_end = logits + (n_rows - 1) * row_stride + vocab;
    const float* out_end = out + (n_rows - 1) * out_stride + vocab;
    MS_REQUIRE(out_end <= logits || in_end <= out,
               "ms_apply_logit_controls: input and output overlap");
  }
  ControlArgs a{};
  a.in = logits;
  a.in_stride = row_stride;
  a.out = out;
  a.out_stride = out_stride;
  a.n_requests = n_requests;
  a.rows = rows_per_request;
  a.vocab = vocab;
  a.words = (vocab + 31) / 32;
  a.c = *controls;
  a.err = device_error_word();
  const int slices = ceil_div(vocab, kSlice);
  a.rows_per_cta = rows_per_request;
  const dim3 grid(slices, n_requests, ceil_div(rows_per_request, a.rows_per_cta));
  const bool vec = vocab % 4 == 0 && row_stride % 4 == 0 && out_stride % 4 == 0 &&
                   ((reinterpret_cast<uintptr_t>(logits) | reinterpret_cast<uintptr_t>(out)) & 15) == 0;
  cudaStream_t s = as_stream(stream);
  ProfScope prof(kClsSample, s);
  if (vec && in_place)
    launch_pdl(logit_controls_kernel<true, true>, grid, kThreads, 0, s, a);
  else if (vec)
    launch_pdl(logit_controls_kernel<true, false>, grid, kThreads, 0, s, a);
  else if (in_place)
    launch_pdl(logit_controls_kernel<false, true>, grid, kThreads, 0, s, a);
  else
    launch_pdl(logit_controls_kernel<false, false>, grid, kThreads, 0, s, a);
  return check_launch("logit_controls_kernel");
}

extern "C" int ms_token_counts_append(int32_t* counts, uint32_t* seen, int n_slots, int vocab,
                                      const int32_t* slots, int n_seqs, const int32_t* tokens,
                                      const int64_t* row_start, int64_t row_stride,
                                      const int32_t* lens, int len_add, int max_len,
                                      const int32_t* n_prompt, void* stream) {
  MS_REQUIRE(n_slots > 0 && vocab > 0 && n_seqs >= 0 && max_len >= 0 && len_add >= 0,
             "ms_token_counts_append: bad sizes");
  if (n_seqs == 0 || max_len == 0) return MS_OK;
  MS_REQUIRE(counts && seen && slots && tokens, "ms_token_counts_append: null pointer");
  const int threads = max_len >= 256 ? 256 : 32;
  const dim3 grid(n_seqs, max_len >= 256 ? (max_len < 4096 ? ceil_div(max_len, 256) : 16) : 1);
  launch_pdl(token_counts_append_kernel, grid, threads, 0, as_stream(stream), counts, seen,
             n_slots, vocab, (vocab + 31) / 32, slots, tokens, row_start, row_stride, lens, len_add,
             max_len, n_prompt, device_error_word());
  return check_launch("token_counts_append_kernel");
}

extern "C" int ms_token_counts_reset(int32_t* counts, uint32_t* seen, int n_slots, int vocab,
                                     const int32_t* slots, int n_seqs, void* stream) {
  MS_REQUIRE(n_slots > 0 && vocab > 0 && n_seqs >= 0, "ms_token_counts_reset: bad sizes");
  if (n_seqs == 0) return MS_OK;
  MS_REQUIRE(n_seqs <= 65535, "ms_token_counts_reset: more than 65535 sequences");
  MS_REQUIRE(counts && seen && slots, "ms_token_counts_reset: null pointer");
  const dim3 grid(ceil_div(vocab, 2048), n_seqs);
  launch_pdl(token_counts_reset_kernel, grid, 256, 0, as_stream(stream), counts, seen, n_slots,
             vocab, (vocab + 31) / 32, slots, device_error_word());
  return check_launch("token_counts_reset_kernel");
}
