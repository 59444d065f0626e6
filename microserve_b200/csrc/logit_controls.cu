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
constexpr int kSlice = 4096;       // tokens per CTA
constexpr int kMaxProposals = 64;  // the draft lanes of one round

struct ControlArgs {
  const float* in;
  int64_t in_stride;
  float* out;
  int64_t out_stride;
  int n_requests, rows, vocab, words;
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

// The edits of one request in one slice of the vocabulary, gathered once per
// CTA and applied to each of its rows: few tokens are touched (the seen ones,
// the round's proposals, the biased ones), so they are listed and shared out
// over the threads instead of being looked for at every logit of every row.
// A thread keeps its first entry and that token's count in registers.
struct Slice {
  // proposals inside the slice: offset and position in the round
  int prop[kMaxProposals];
  int when[kMaxProposals];
  int n_prop;
  int bias_lo, bias_hi;  // the bias entries to look at
  int n_list;
  // mask words of the row at hand and of the next one
  uint32_t mask[2][kSlice / 32];
  // touched tokens: offset | seen << 12
  uint16_t list[kSlice];
};
static_assert(kSlice == 4096, "12 bits of offset");

__device__ __forceinline__ int valid_slot(const ControlArgs& a, int b) {
  const int slot = a.c.slots ? a.c.slots[b] : -1;
  if (slot < a.c.n_slots) return max(slot, -1);
  if (threadIdx.x == 0) raise_device_error(a.err, kErrSlot);
  return -1;
}

// Word `threadIdx.x` of the row's mask in the slice (all ones: no mask).
__device__ __forceinline__ uint32_t mask_word(const ControlArgs& a, int64_t row, int t0, bool& masked) {
  int m = a.c.mask_rows ? a.c.mask_rows[row] : -1;
  if (m >= a.c.n_masks) {
    if (threadIdx.x == 0) raise_device_error(a.err, kErrMask);
    m = -1;
  }
  masked = m >= 0;
  const int w = (t0 >> 5) + threadIdx.x;
  return masked && threadIdx.x < kSlice / 32 && w < a.words
             ? __ldg(a.c.masks + (int64_t)m * a.words + w)
             : 0xffffffffu;
}

struct Entry {
  int o;      // offset in the slice (-1: none)
  bool seen;  // else listed for a proposal only
  int count;
};

__device__ __forceinline__ Entry list_entry(const ControlArgs& a, const Slice& sl, int slot, int t0,
                                            int e) {
  if (e >= sl.n_list) return Entry{-1, false, 0};
  const int v = sl.list[e];
  const int o = v & (kSlice - 1);
  return Entry{o, (v >> 12) != 0, a.c.counts[(int64_t)slot * a.vocab + t0 + o]};
}

// Gathers the slice's edits and the first row's mask; block-wide, ends with a barrier.
__device__ void load_slice(const ControlArgs& a, int b, int slot, int64_t row0, int t0, int n_here,
                           Slice& sl, bool& masked) {
  const ms_logit_controls& c = a.c;
  const int tid = threadIdx.x;
  if (tid == 0) sl.n_prop = sl.n_list = 0;
  uint32_t seen = 0;
  const int w = (t0 >> 5) + tid;
  if (slot >= 0 && tid < kSlice / 32 && w < a.words) {
    seen = __ldg(c.seen + (int64_t)slot * a.words + w);
    const int left = n_here - 32 * tid;  // bits past the vocabulary mean nothing
    if (left < 32) seen &= left > 0 ? (1u << left) - 1u : 0u;
  }
  const uint32_t first_mask = mask_word(a, row0, t0, masked);
  if (tid < kSlice / 32) sl.mask[0][tid] = first_mask;
  // threads 64 and 65 cut the request's bias list to the slice; the outer
  // slices also take (and report) ids outside the vocabulary
  if (tid == 64 || tid == 65) {
    int lo = 0, hi = 0;
    if (c.bias_start) {
      lo = c.bias_start[b];
      hi = c.bias_start[b + 1];
      if (lo < 0 || hi < lo || hi > c.n_bias) {
        raise_device_error(a.err, kErrOrder);
        lo = hi = 0;
      }
      const int want = tid == 64 ? t0 : t0 + n_here;
      if (tid == 64 ? blockIdx.x > 0 : blockIdx.x + 1 < gridDim.x) {
        while (lo < hi) {
          const int mid = (lo + hi) >> 1;
          if (c.bias_ids[mid] < want) lo = mid + 1; else hi = mid;
        }
      } else if (tid == 65) {
        lo = hi;
      }
    }
    (tid == 64 ? sl.bias_lo : sl.bias_hi) = lo;
  }
  __syncthreads();
  int at = seen ? atomicAdd(&sl.n_list, __popc(seen)) : 0;
  for (uint32_t m = seen; m; m &= m - 1)
    sl.list[at++] = (uint16_t)((32 * tid + __ffs(m) - 1) | 1 << 12);
  // those that the last row sees; the others may not have been drawn yet
  if (slot >= 0 && c.proposals && tid < c.first_proposal + a.rows - 1) {
    const int v = c.proposals[(int64_t)tid * a.n_requests + b];
    if (v < 0 || v >= a.vocab) {
      raise_device_error(a.err, kErrToken);
    } else if (v >= t0 && v < t0 + n_here) {
      const int k = atomicAdd(&sl.n_prop, 1);
      sl.prop[k] = v - t0;
      sl.when[k] = tid;
    }
  }
  __syncthreads();
  if (tid < sl.n_prop) {  // list the proposals that no other entry stands for
    const int o = sl.prop[tid];
    bool fresh = !(__ldg(c.seen + (int64_t)slot * a.words + ((t0 + o) >> 5)) >> (o & 31) & 1u);
    for (int j = 0; j < sl.n_prop; ++j)
      fresh &= !(sl.prop[j] == o && sl.when[j] < sl.when[tid]);
    if (fresh) sl.list[atomicAdd(&sl.n_list, 1)] = (uint16_t)o;
  }
  if (c.proposals) __syncthreads();
}

// Applies the edits to one row's slice x (shared or global memory; token o of
// the slice at x[o], `mis` floats past a 16-byte boundary): penalties, biases,
// then the mask.  Block-wide; the caller's barrier follows.
template <bool SHARED>
__device__ __forceinline__ void edit_row(const ControlArgs& a, const Slice& sl, int b, int slot,
                                         const Penalty& p, const Entry& own, int visible, int t0, int n_here,
                                         const uint32_t* mask, bool masked, float* x, int mis) {
  const ms_logit_controls& c = a.c;
  const int tid = threadIdx.x;
  for (int e = tid; e < sl.n_list; e += blockDim.x) {
    Entry t = e == tid ? own : list_entry(a, sl, slot, t0, e);
    for (int j = 0; j < sl.n_prop; ++j) {
      const bool hit = sl.prop[j] == t.o && sl.when[j] < visible;
      t.seen |= hit;
      t.count += hit;
    }
    if (t.seen) x[t.o] = penalise(x[t.o], p, t.count);
  }
  if (sl.bias_hi > sl.bias_lo) {
    __syncthreads();
    const int first = c.bias_start[b];
    for (int e = sl.bias_lo + tid; e < sl.bias_hi; e += blockDim.x) {
      const int v = c.bias_ids[e];
      if (v < 0 || v >= a.vocab)
        raise_device_error(a.err, kErrToken);
      else if (e > first && c.bias_ids[e - 1] >= v)
        raise_device_error(a.err, kErrOrder);  // not ascending: the entry is skipped
      else if (v >= t0 && v < t0 + n_here)
        x[v - t0] = __fadd_rn(x[v - t0], c.bias_values[e]);
    }
  }
  if (!masked) return;
  if (sl.n_list > 0 || sl.bias_hi > sl.bias_lo) __syncthreads();
  // groups of 4 tokens on 16-byte boundaries
  for (int o = 4 * tid - mis; o < n_here; o += 4 * blockDim.x) {
    uint32_t ok;
    if (o >= 0) {
      const int sh = o & 31;
      ok = mask[o >> 5] >> sh;
      if (sh > 28 && o + 32 - sh < n_here) ok |= mask[(o >> 5) + 1] << (32 - sh);
    } else {
      ok = mask[0] << -o;
    }
    const int lo = max(0, -o), hi = min(4, n_here - o);  // its tokens inside the slice
    const uint32_t in = (1u << hi) - (1u << lo);
    const uint32_t no = ~ok & in;
    if (no == 15u) {
      *reinterpret_cast<float4*>(x + o) = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
    } else if (SHARED && no && in == 15u) {
      float4 q = *reinterpret_cast<float4*>(x + o);
      if (no & 1u) q.x = -INFINITY;
      if (no & 2u) q.y = -INFINITY;
      if (no & 4u) q.z = -INFINITY;
      if (no & 8u) q.w = -INFINITY;
      *reinterpret_cast<float4*>(x + o) = q;
    } else if (no) {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (no >> k & 1u) x[o + k] = -INFINITY;
    }
  }
}

// ---- out of place, through shared memory ------------------------------------
// A CTA takes kSlice tokens of all rows of one request.  Each row's slice comes in
// by one bulk copy, is edited in shared memory and goes out by one bulk copy,
// in a ring of rows.  The kernel moves 8 bytes per logit and is bound by HBM:
// 256 requests x 6 rows x 128256 take 290 us (5.5 TB/s), x 5 x 32000 61 us.  A
// deeper ring (347 us with 3 rows), half a slice (355) and 128 or 384 threads
// (314, 327) take more: what hides the latency is the CTAs beside this one.
// A row that does not start on 16 bytes keeps its misalignment in shared
// memory; its up to 3 first and last logits are copied one by one.
constexpr int kRing = 2;
constexpr int kRowFloats = kSlice + 4;
constexpr long long kWaitCycles = 1ll << 32;  // ~2.2 s
constexpr int kErrTimeout = 5;

__device__ __forceinline__ uint32_t s_addr(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          dst),
      "l"(src), "r"(bytes), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void bulk_store(void* dst, uint32_t src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(src),
               "r"(bytes)
               : "memory");
}
__device__ __forceinline__ bool wait_full(uint32_t bar, uint32_t parity, int* err) {
  const long long t0 = clock64();
  while (true) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.b32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    if (ok) return true;
    if (clock64() - t0 > kWaitCycles) {
      atomicCAS(err, 0, kErrTimeout);
      return false;
    }
  }
}

__global__ void __launch_bounds__(kThreads) logit_controls_kernel(ControlArgs a, int ring) {
  extern __shared__ __align__(16) float smem[];  // [ring][kRowFloats]
  __shared__ Slice sl;
  __shared__ __align__(8) uint64_t bars[kRing];
  const ms_logit_controls& c = a.c;
  const int tid = threadIdx.x;
  const int t0 = blockIdx.x * kSlice;
  const int b = blockIdx.y;
  const int n_here = min(kSlice, a.vocab - t0);
  const int64_t row0 = (int64_t)b * a.rows;

  // Row it: misalignment (in floats), loose first logits, bulk-copied logits.
  struct Cut {
    int mis, head, body;
  };
  auto cut = [&](int it) {
    const uintptr_t p = reinterpret_cast<uintptr_t>(a.in + (row0 + it) * a.in_stride + t0);
    Cut q;
    q.mis = (int)(p >> 2) & 3;
    q.head = min((4 - q.mis) & 3, n_here);
    q.body = (n_here - q.head) & ~3;
    return q;
  };
  auto issue = [&](int it) {  // thread 0
    const Cut q = cut(it);
    const uint32_t bar = s_addr(&bars[it % ring]);
    const uint32_t bytes = 4u * q.body;
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes)
                 : "memory");
    if (bytes)
      bulk_load(s_addr(smem + (it % ring) * kRowFloats + q.mis + q.head),
                a.in + (row0 + it) * a.in_stride + t0 + q.head, bytes, bar);
  };
  const int ahead = ring > 1 ? ring - 1 : 1;  // rows in flight
  if (tid == 0) {
    for (int k = 0; k < ring; ++k)
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(s_addr(&bars[k])) : "memory");
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  pdl_enter();
  if (tid == 0)
    for (int it = 0; it < min(ahead, a.rows); ++it) issue(it);
  const int slot = valid_slot(a, b);
  Penalty p{1.f, 0.f, 0.f};
  if (slot >= 0) p = Penalty{c.penalties[3 * b], c.penalties[3 * b + 1], c.penalties[3 * b + 2]};
  bool masked;
  load_slice(a, b, slot, row0, t0, n_here, sl, masked);
  const Entry own = list_entry(a, sl, slot, t0, tid);

  for (int it = 0; it < a.rows; ++it) {
    float* buf = smem + (it % ring) * kRowFloats;
    const Cut q = cut(it);
    const float* xin = a.in + (row0 + it) * a.in_stride + t0;
    float* yout = a.out + (row0 + it) * a.out_stride + t0;
    const int tail0 = q.head + q.body;
    const bool loose = q.head > 0 || tail0 < n_here;
    if (tid < q.head) buf[q.mis + tid] = xin[tid];
    if (tid >= 32 && tail0 + tid - 32 < n_here) buf[q.mis + tail0 + tid - 32] = xin[tail0 + tid - 32];
    bool next_masked = false;
    uint32_t next_mask = 0;
    if (it + 1 < a.rows) next_mask = mask_word(a, row0 + it + 1, t0, next_masked);
    const bool ok = wait_full(s_addr(&bars[it % ring]), (it / ring) & 1, a.err);
    if (loose) __syncthreads();
    float* x = buf + q.mis;
    edit_row<true>(a, sl, b, slot, p, own, c.first_proposal + it, t0, n_here, sl.mask[it & 1],
                   masked, x, q.mis);
    if (tid < kSlice / 32) sl.mask[(it + 1) & 1][tid] = next_mask;
    masked = next_masked;
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    // all threads agree to stop when a copy did not arrive in time
    if (__syncthreads_or(!ok)) {
      if (tid == 0)  // no copy may arrive after the block has gone
        for (int k = it; k < min(it + ahead, a.rows); ++k)
          wait_full(s_addr(&bars[k % ring]), (k / ring) & 1, a.err);
      break;
    }
    if (tid < q.head) yout[tid] = x[tid];
    if (tid >= 32 && tail0 + tid - 32 < n_here) yout[tail0 + tid - 32] = x[tail0 + tid - 32];
    if (tid == 0) {
      if (q.body) bulk_store(yout + q.head, s_addr(x + q.head), 4u * q.body);
      asm volatile("cp.async.bulk.commit_group;" ::: "memory");
      if (it + ahead < a.rows) {
        // the row `ahead` from here takes the buffer of the row before this one
        asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
        issue(it + ahead);
      }
    }
    // Its loose logits are out before the buffer is filled again, and thread 0 has
    // seen the store from the next row's buffer end before loose logits go there
    // (rows of one alignment are all loose or none is).
    if (loose || (a.in_stride & 3)) __syncthreads();
  }
  if (tid == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
}

// ---- in place, or with input and output rows aligned differently ---------------
// In place only what a control touches is read and written; else the slice is
// copied first and then edited where it is.  128 threads a CTA: its work is
// a chain of short dependent reads, so more CTAs per SM beat more threads
// (grammar masks over 256 x 128256: 28.6 us, 33.9 with 256).  That case writes
// 104 MB (a plain fill: 3.9 TB/s) as 190 MB of sectors at L2; reading what a partly
// masked group of 4 holds, to write it whole, takes 36.7 us.  Penalties in place, 256 x 5
// rows x 32000 with 1114 tokens touched in each: 44 us, for 110 MB of sectors read and 35
// written around 11 MB of logits.
constexpr int kDirectThreads = 128;
__global__ void __launch_bounds__(kDirectThreads) logit_controls_direct_kernel(ControlArgs a) {
  pdl_enter();
  __shared__ Slice sl;
  const ms_logit_controls& c = a.c;
  const int tid = threadIdx.x;
  const int t0 = blockIdx.x * kSlice;
  const int b = blockIdx.y;
  const int n_here = min(kSlice, a.vocab - t0);
  const int64_t row0 = (int64_t)b * a.rows;
  const int slot = valid_slot(a, b);
  Penalty p{1.f, 0.f, 0.f};
  if (slot >= 0) p = Penalty{c.penalties[3 * b], c.penalties[3 * b + 1], c.penalties[3 * b + 2]};
  bool masked;
  load_slice(a, b, slot, row0, t0, n_here, sl, masked);
  const Entry own = list_entry(a, sl, slot, t0, tid);
  for (int it = 0; it < a.rows; ++it) {
    float* x = a.out + (row0 + it) * a.out_stride + t0;
    if (a.in != a.out) {
      const float* xin = a.in + (row0 + it) * a.in_stride + t0;
#pragma unroll 8
      for (int o = tid; o < n_here; o += kDirectThreads) x[o] = xin[o];
      __syncthreads();
    }
    bool next_masked = false;
    uint32_t next_mask = 0;
    if (it + 1 < a.rows) next_mask = mask_word(a, row0 + it + 1, t0, next_masked);
    edit_row<false>(a, sl, b, slot, p, own, c.first_proposal + it, t0, n_here, sl.mask[it & 1],
                    masked, x, (int)(reinterpret_cast<uintptr_t>(x) >> 2) & 3);
    if (it + 1 < a.rows) {
      if (tid < kSlice / 32) sl.mask[(it + 1) & 1][tid] = next_mask;
      masked = next_masked;
      __syncthreads();
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
  MS_REQUIRE(!c->proposals || (int64_t)c->first_proposal + rows_per_request - 1 <= c->n_proposals,
             "ms_logit_controls: rows after the first %d proposals, %d of them, see more than %d",
             c->first_proposal, rows_per_request, c->n_proposals);
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
  MS_REQUIRE(n_requests <= 65535, "ms_apply_logit_controls: more than 65535 requests");
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
  const dim3 grid(slices, n_requests);
  const uintptr_t pi = reinterpret_cast<uintptr_t>(logits), po = reinterpret_cast<uintptr_t>(out);
  cudaStream_t s = as_stream(stream);
  ProfScope prof(kClsSample, s);
  // every row of the input and of the output equally far from 16 bytes
  if (!in_place && ((pi ^ po) & 15) == 0 && (row_stride - out_stride) % 4 == 0) {
    const int ring = rows_per_request < kRing ? rows_per_request : kRing;
    static_assert(sizeof(Slice) + kRing * (kRowFloats * 4 + 8) <= 48 * 1024, "the default shared memory");
    launch_pdl(logit_controls_kernel, grid, kThreads, ring * kRowFloats * 4, s, a, ring);
    return check_launch("logit_controls_kernel");
  }
  launch_pdl(logit_controls_direct_kernel, grid, kDirectThreads, 0, s, a);
  return check_launch("logit_controls_direct_kernel");
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
