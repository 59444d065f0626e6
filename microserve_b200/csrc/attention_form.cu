// Paged attention with score forms: entry points, the plan, the kernel on the
// CUDA cores (float32 caches, and bf16 ones whose head or block size the
// matrix kernels do not take) and the joining of KV ranges.
#include <cfloat>

#include "attention_form_device.cuh"
#include "model_kernels.cuh"

namespace ms {
namespace {

constexpr int kWarps = 8;
template <int DH> constexpr int rows_per_warp() { return DH <= 64 ? 4 : 2; }
// Keys per step: as many as 48 KB hold beside the queries (a step costs a round trip to memory).
template <int DH> constexpr int step_keys() { return DH <= 32 ? 128 : DH == 64 ? 64 : 32; }

template <typename T>
__device__ __forceinline__ float4 load4(const T* p) {
  if constexpr (sizeof(T) == 4) {
    return *reinterpret_cast<const float4*>(p);
  } else {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    return make_float4(__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u),
                       __uint_as_float(v.y << 16), __uint_as_float(v.y & 0xffff0000u));
  }
}

// One CTA per (row tile, KV range, kv head, sequence); row r of a tile is
// (token r / group, head-in-group r % group).  A step's keys in shared memory (rows
// padded by 4 floats: the lanes of a quarter warp read 16 bytes each from different
// banks), a lane a key for the scores and a dimension for the sums; online softmax in base
// e, everything in float32.  The small models that take this kernel are bound by latency:
// 8 trees of 7 tokens, 4 heads of 32, contexts up to 97: 8.5 us, 14.2 with 32 keys a step.
template <typename T, int DH>
__global__ void __launch_bounds__(kWarps * 32) form_simt_kernel(const __grid_constant__ FormArgs a) {
  pdl_enter();
  constexpr int PER_LANE = DH >= 32 ? DH / 32 : 1;
  constexpr int RPW = rows_per_warp<DH>();
  constexpr int ROWS = kWarps * RPW;
  constexpr int CK = step_keys<DH>(), SUB = CK / 32, LD = DH + 4;
  __shared__ __align__(16) float Qs[ROWS * DH];
  __shared__ __align__(16) float Ks[CK * LD];
  __shared__ __align__(16) float Vs[CK * DH];

  const int b = blockIdx.z, g = blockIdx.y;
  const int split = blockIdx.x % a.n_splits, tile = blockIdx.x / a.n_splits;
  const FormSeq s = form_seq(a, b);
  const int nrows = s.qlen * a.group, r0 = tile * ROWS;
  if (r0 >= nrows) return;
  const int nr = min(ROWS, nrows - r0);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int minpos = 0, maxpos = 0;
  if (needs_positions(a)) position_range(a, s, r0, nr, minpos, maxpos);
  const T* q = static_cast<const T*>(a.q);
  for (int idx = threadIdx.x; idx < nr * DH; idx += blockDim.x) {
    const int r = idx / DH, d = idx - r * DH, rr = r0 + r;
    Qs[idx] = to_f(q[(int64_t)(s.t0 + rr / a.group) * a.q_stride +
                     (int64_t)(g * a.group + rr % a.group) * DH + d]);
  }
  const FormKeys keys = form_keys(a, s, minpos, maxpos);
  const int xbeg = min(split * a.split_len, keys.total);
  const int xend = split == a.n_splits - 1 ? keys.total : min(keys.total, xbeg + a.split_len);

  float m[RPW], l[RPW], acc[RPW][PER_LANE];
  int tok[RPW], pos[RPW];
  float slope[RPW];
#pragma unroll
  for (int i = 0; i < RPW; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int e = 0; e < PER_LANE; ++e) acc[i][e] = 0.f;
    const int r = warp + i * kWarps, rr = r0 + r;
    tok[i] = s.t0 + (r < nr ? rr / a.group : 0);
    pos[i] = a.positions[tok[i]];
    slope[i] = a.slopes && r < nr ? a.slopes[g * a.group + rr % a.group] : 0.f;
  }
  const T *kp = static_cast<const T*>(a.k), *vp = static_cast<const T*>(a.v);
  const int32_t* table = a.tables + (int64_t)b * a.max_blocks;
  const float inv_cap = a.softcap > 0.f ? a.scale / a.softcap : 0.f;
  // (rows of 4 values are aligned to them where the pools are)
  const bool vec = ((reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v)) & 15) == 0;
  for (int x0 = xbeg; x0 < xend; x0 += CK) {
    const int n = min(CK, xend - x0);
    __syncthreads();
#pragma unroll 4
    for (int idx = threadIdx.x; idx < n * (DH / 4); idx += kWarps * 32) {
      const int kk = idx / (DH / 4), d = (idx - kk * (DH / 4)) * 4, j = keys.key(x0 + kk);
      const int64_t o = (((int64_t)form_block(a, table, j / a.bs) * a.hkv + g) * a.bs + (j % a.bs)) * DH + d;
      float4 kv, vv;
      if (vec) {
        kv = load4(kp + o);
        vv = load4(vp + o);
      } else {
        kv = make_float4(to_f(kp[o]), to_f(kp[o + 1]), to_f(kp[o + 2]), to_f(kp[o + 3]));
        vv = make_float4(to_f(vp[o]), to_f(vp[o + 1]), to_f(vp[o + 2]), to_f(vp[o + 3]));
      }
      *reinterpret_cast<float4*>(Ks + kk * LD + d) = kv;
      *reinterpret_cast<float4*>(Vs + kk * DH + d) = vv;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < RPW; ++i) {
      const int r = warp + i * kWarps;
      if (r >= nr) continue;
      float x[SUB];
      uint32_t seen[SUB];
      float top = -INFINITY;
#pragma unroll
      for (int u = 0; u < SUB; ++u) {
        seen[u] = 0;
        if (u * 32 >= n) continue;
        const int kk = u * 32 + lane;
        // (keys behind the last one are rows of an earlier step, or never written: not seen)
        float v = 0.f;
        const float4* kr = reinterpret_cast<const float4*>(Ks + kk * LD);
        const float4* qr = reinterpret_cast<const float4*>(Qs + r * DH);
#pragma unroll 8
        for (int d = 0; d < DH / 4; ++d) {
          const float4 k4 = kr[d], q4 = qr[d];
          v = fmaf(q4.x, k4.x, v);
          v = fmaf(q4.y, k4.y, v);
          v = fmaf(q4.z, k4.z, v);
          v = fmaf(q4.w, k4.w, v);
        }
        int distance = 0;
        const bool sees = kk < n && form_sees(a, s, tok[i], pos[i], keys.key(x0 + min(kk, n - 1)), distance);
        // (tanh(u) = u to 3e-9 up to 1e-4, where u itself may be too small for float32)
        const float raw = v * a.scale;
        v = a.softcap > 0.f && !(fabsf(raw) <= 1e-4f * a.softcap) ? a.softcap * tanhf(v * inv_cap) : raw;
        if (a.slopes) v -= slope[i] * fabsf((float)distance);
        x[u] = sees ? v : -INFINITY;
        seen[u] = __ballot_sync(0xffffffffu, sees);
        top = fmaxf(top, x[u]);
      }
      const float mn = fmaxf(m[i], warp_max(top));
      const float sub = mn == -INFINITY ? 0.f : mn;
      const float alpha = m[i] == -INFINITY ? 0.f : expf(m[i] - sub);
      m[i] = mn;
      float sum = 0.f;
#pragma unroll
      for (int e = 0; e < PER_LANE; ++e) acc[i][e] *= alpha;
#pragma unroll
      for (int u = 0; u < SUB; ++u) {
        if (seen[u] == 0) continue;
        const float p = (seen[u] >> lane) & 1 ? expf(x[u] - sub) : 0.f;
        sum += p;
        const float* vr = Vs + u * 32 * DH + (DH >= 32 ? lane : lane % DH);
#pragma unroll 8
        for (int kk = 0; kk < 32; ++kk) {
          const float pk = __shfl_sync(0xffffffffu, p, kk);
          if (!((seen[u] >> kk) & 1)) continue;  // an unseen value may be anything
#pragma unroll
          for (int e = 0; e < PER_LANE; ++e) acc[i][e] = fmaf(pk, vr[kk * DH + 32 * e], acc[i][e]);
        }
      }
      l[i] = l[i] * alpha + warp_sum(sum);
    }
  }
#pragma unroll
  for (int i = 0; i < RPW; ++i) {
    const int r = warp + i * kWarps;
    if (r >= nr) continue;
    const int rr = r0 + r;
    const int64_t part_row = ((((int64_t)b * a.hkv + g) * a.row_tiles + tile) * a.n_splits + split) * ROWS + r;
    const float inv = l[i] == 0.f ? 0.f : 1.f / l[i];
    float zero = 0.f;  // NaN if a sum is not finite
#pragma unroll
    for (int e = 0; e < PER_LANE; ++e) zero = fmaf(acc[i][e], 0.f, zero);
    if (a.n_splits == 1) {
      T* o = static_cast<T*>(a.out) + (int64_t)(s.t0 + rr / a.group) * a.out_stride +
             (int64_t)(g * a.group + rr % a.group) * DH;
#pragma unroll
      for (int e = 0; e < PER_LANE; ++e)
        if (DH >= 32 || lane < DH) o[lane + 32 * e] = from_f<T>(l[i] == 0.f ? 0.f : acc[i][e] * inv);
    } else {
#pragma unroll
      for (int e = 0; e < PER_LANE; ++e)
        if (DH >= 32 || lane < DH) a.part_o[part_row * DH + lane + 32 * e] = acc[i][e] * inv;
      if (lane == 0) {
        a.part_ml[part_row * 2] = m[i];
        a.part_ml[part_row * 2 + 1] = l[i];
      }
    }
    if (__any_sync(0xffffffffu, zero != 0.f) && l[i] > 0.f && l[i] < INFINITY) {
      float common[(DH + 31) / 32];
      form_odd_values<T, DH>(a, s, keys, table, g, xbeg, xend, minpos, maxpos, 0, DH, 0, 1, common);
      form_row_again<T, DH, false>(a, s, keys, table, g, rr, xbeg, xend, minpos, maxpos, 0, DH, part_row, true, common);
    }
  }
}

// A row a block: the ranges' weights l 2^(m - max) over their sum first, then the ranges' results, a range
// a warp at a time with 16 bytes a lane, the warps' sums added in order: the result
// does not depend on timing.  (A warp a row, range after range, took 24 us for 37
// ranges of 64 rows x 8 kv heads; this about 4.  Three ranges a warp are loaded before their weights are known:
// attention and joining 37.6 -> 35.8 us.)
template <typename T, bool kBase2>
__global__ void __launch_bounds__(256) form_combine_kernel(FormArgs a, int rows, int dh) {
  pdl_enter();
  extern __shared__ __align__(16) float s_comb[];  // weights, then (warps, dh) sums
  __shared__ float s_red[32];
  const int b = blockIdx.z, g = blockIdx.y, rr = blockIdx.x;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int tile = rr / rows, r = rr - tile * rows;
  const int64_t unit0 = (((int64_t)b * a.hkv + g) * a.row_tiles + tile) * a.n_splits;
  const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + unit0 * rows + r;
  const float* po = a.part_o + (unit0 * rows + r) * dh;
  // (rows that the sequence does not have are part of the workspace too: nothing waits for its length)
  constexpr int kAhead = 3;
  float4 ahead[kAhead];
#pragma unroll
  for (int u = 0; u < kAhead; ++u) {
    const int i = warp + u * warps;
    if (i < a.n_splits && lane * 4 < dh)
      ahead[u] = *reinterpret_cast<const float4*>(po + (int64_t)i * rows * dh + lane * 4);
  }
  float mx = -INFINITY;
  for (int i = threadIdx.x; i < a.n_splits; i += blockDim.x) mx = fmaxf(mx, ml[(int64_t)i * rows].x);
  const FormSeq s = form_seq(a, b);
  if (rr >= s.qlen * a.group) return;
  mx = warp_max(mx);
  if (lane == 0) s_red[warp] = mx;
  __syncthreads();
  mx = warp_max(lane < warps ? s_red[lane] : -INFINITY);
  const float sub = mx == -INFINITY ? 0.f : mx;
  float l = 0.f;
  for (int i = threadIdx.x; i < a.n_splits; i += blockDim.x) {
    const float2 v = ml[(int64_t)i * rows];
    // (a range without a key for this row has a sum of 0, and its values may be unset)
    const float w = v.y == 0.f ? 0.f : kBase2 ? exp2f(v.x - sub) : expf(v.x - sub);
    s_comb[i] = v.y == 0.f ? -1.f : w * v.y;
    l = fmaf(w, v.y, l);
  }
  l = block_sum(l, s_red);  // (its barriers cover the weights)
  const float inv = l == 0.f ? 0.f : 1.f / l;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](float w, const float4& v) {
    if (w == -1.f) return;
    w *= inv;
    if (w == 0.f) {  // (an infinite value counts however small its weight is)
      auto odd = [](float x) { return fabsf(x) < INFINITY ? 0.f : x; };
      acc.x += odd(v.x);
      acc.y += odd(v.y);
      acc.z += odd(v.z);
      acc.w += odd(v.w);
      return;
    }
    acc.x = fmaf(w, v.x, acc.x);
    acc.y = fmaf(w, v.y, acc.y);
    acc.z = fmaf(w, v.z, acc.z);
    acc.w = fmaf(w, v.w, acc.w);
  };
  if (lane * 4 < dh) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (warp + u * warps < a.n_splits) add(s_comb[warp + u * warps], ahead[u]);
#pragma unroll 4
    for (int i = warp + kAhead * warps; i < a.n_splits; i += warps)
      add(s_comb[i], *reinterpret_cast<const float4*>(po + (int64_t)i * rows * dh + lane * 4));
  }
  float* sums = s_comb + ((a.n_splits + 3) & ~3);
  if (lane * 4 < dh) *reinterpret_cast<float4*>(sums + warp * dh + lane * 4) = acc;
  __syncthreads();
  T* o = static_cast<T*>(a.out) + (int64_t)(s.t0 + rr / a.group) * a.out_stride +
         (int64_t)(g * a.group + rr % a.group) * dh;
  for (int d = threadIdx.x; d < dh; d += blockDim.x) {
    float v = 0.f;
    for (int w = 0; w < warps; ++w) v += sums[w * dh + d];
    o[d] = from_f<T>(v);
  }
}

// Tiles of `rows` rows; KV ranges where the tiles alone leave SMs without work,
// of at least `least` keys and in whole chunks of `chunk`, up to `wave` CTAs in all.  (Not where a little more
// than a wave is left: the ranges' sums cost more than the second wave, 123 against 87 us for 40
// trees of 16 nodes over up to 4 k keys.)
void plan(FormArgs& a, int max_context, int rows, int chunk, int least, int wave) {
  int64_t span = max_context;
  if (a.window > 0 && !a.prefix) span = min(span, (int64_t)a.window + a.max_q + 2 * a.bs);
  a.row_tiles = ceil_div(a.max_q * a.group, rows);
  const int64_t units = (int64_t)a.n_seqs * a.hkv * a.row_tiles;
  int64_t splits = units < wave ? wave / units : 1;
  splits = max((int64_t)1, min(splits, (span + least - 1) / least));
  int64_t len = (span + splits - 1) / splits;
  len = max((int64_t)chunk, (len + chunk - 1) / chunk * chunk);
  a.split_len = (int)len;
  a.n_splits = (int)max((int64_t)1, (span + len - 1) / len);
}

size_t part_bytes(const FormArgs& a, int rows, int dh) {
  if (a.n_splits == 1) return 0;
  const size_t units = (size_t)a.n_seqs * a.hkv * a.row_tiles * a.n_splits;
  return units * rows * (dh + 2) * sizeof(float);
}

int simt_rows(int dh) { return kWarps * (dh <= 64 ? 4 : 2); }

// How a call is cut up: which kernel, its rows per tile, the KV ranges, and whether the sequences are
// put in order first.
enum Kernel { kSimt, kTma, kTc };
struct Way {
  Kernel kernel;
  int rows;
  bool order;
};
Way choose(FormArgs& a, const ms_kv_cache& c, int max_context) {
  const int64_t rows = (int64_t)a.max_q * a.group;
  if (!form_tma_takes(c) || ((reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v)) & 15)) {
    const Way w{kSimt, simt_rows(c.d_head), false};
    plan(a, max_context, w.rows, 128, 256, 148 * 4);
    return w;
  }
  // mma.sync for few rows, tcgen05 for many, where 128 rows of a tile cost what 16 do (us, mma.sync and
  // tcgen05; 128 sequences of 2 k keys, cap and window): heads of 128, 4, 16 and 32 rows 185 and
  // 201, 210 and 204, 258 and 208 (without either 335 and 354, 345 and 358, 382 and 365); heads of
  // 64, 4, 16 and 32 rows 104 and 126, 119 and 129, 149 and 128; trees of 256 sequences, heads of
  // 64, 32, 40 and 64 rows 78 and 94, 90 and 94, 120 and 95.
  Way w{rows <= (c.d_head == 128 ? 16 : 32) ? kTma : kTc, 0, false};
  // The least tile that holds a sequence (us; trees of 64 sequences, heads of 128): 64 rows in a tile of
  // 64 and of 128 127 and 137; 128 rows in 128 and 256 145 and 185; 192 rows in two of 128 and one of
  // 256 257 and 221.
  // Sequences of up to 64 rows that fit in one wave take tiles of 128 too, whose second score buffer makes a
  // step shorter: one tree of 16 nodes, 8 kv heads, 400, 8 k and 32 k keys 13.1, 19.7 and 37.3 us instead
  // of 14.9, 21.4 and 38.5, 32 of them over 2 k keys 53.3 instead of 55.0.
  const bool few = (int64_t)a.n_seqs * c.n_kv_heads <= 148 * 2;
  w.rows = w.kernel == kTma ? 32 : rows <= 64 && !few ? 64 : rows <= 128 ? 128 : 256;
  const int resident = 148 * (w.kernel == kTma ? 3 : w.rows == 256 ? 1 : 2);
  if (w.kernel == kTma)
    plan(a, max_context, w.rows, 64, 512, 148 * 4);
  else
    plan(a, max_context, w.rows, 128, 512, resident);
  // Longest first where the CTAs take more than one wave: the last wave is then of short ones.
  // (ordering: a launch of about 2 us, n_seqs^2 comparisons)
  w.order = a.n_seqs > 1 && a.n_seqs <= 4096 &&
            (int64_t)a.n_seqs * a.hkv * a.row_tiles * a.n_splits > resident;
  return w;
}

template <typename T, int DH>
int launch_simt(FormArgs& a, cudaStream_t s) {
  dim3 grid(a.row_tiles * a.n_splits, a.hkv, a.n_seqs);
  launch_pdl(form_simt_kernel<T, DH>, grid, kWarps * 32, 0, s, a);
  MS_TRY(check_launch("form_simt_kernel"));
  return a.n_splits > 1 ? form_combine<T, false>(a, simt_rows(DH), DH, s) : MS_OK;
}

template <typename T>
int simt_by_dh(FormArgs& a, int dh, cudaStream_t s) {
  switch (dh) {
    case 8: return launch_simt<T, 8>(a, s);
    case 16: return launch_simt<T, 16>(a, s);
    case 32: return launch_simt<T, 32>(a, s);
    case 64: return launch_simt<T, 64>(a, s);
    default: return launch_simt<T, 128>(a, s);
  }
}

// Everything of a call that does not depend on the device's data, checked.
int form_args(FormArgs& a, const ms_kv_cache& c, int layer, const ms_batch& bt, int hq,
              const ms_attention_form* form, int* max_context) {
  MS_REQUIRE(bt.n_seqs >= 0 && bt.n_tokens >= 0, "ms_paged_attention_form: bad batch sizes");
  MS_REQUIRE(hq > 0 && hq % c.n_kv_heads == 0,
             "ms_paged_attention_form: n_heads %d not a multiple of n_kv_heads %d", hq, c.n_kv_heads);
  if (c.dtype != MS_DTYPE_F32 && c.dtype != MS_DTYPE_BF16)
    return fail(MS_ERR_UNSUPPORTED, "ms_paged_attention_form: dtype %d", c.dtype);
  if (c.d_head != 8 && c.d_head != 16 && c.d_head != 32 && c.d_head != 64 && c.d_head != 128)
    return fail(MS_ERR_UNSUPPORTED, "ms_paged_attention_form: d_head %d (8/16/32/64/128)", c.d_head);
  const bool empty = bt.n_seqs == 0 || bt.n_tokens == 0;
  MS_REQUIRE(empty || (bt.max_q_len > 0 && bt.max_blocks > 0),
             "ms_paged_attention_form: max_q_len and max_blocks must be > 0");
  MS_REQUIRE((int64_t)bt.max_blocks * c.block_size <= INT_MAX && (int64_t)bt.max_q_len * hq <= INT_MAX / 2,
             "ms_paged_attention_form: contexts or queries beyond 2^31");
  if ((int64_t)bt.max_q_len * (hq / c.n_kv_heads) > 65535 * 128)
    return fail(MS_ERR_TOO_LARGE, "ms_paged_attention_form: %d tokens of a sequence", bt.max_q_len);
  if (bt.n_seqs > 65535 || c.n_kv_heads > 65535)
    return fail(MS_ERR_TOO_LARGE, "ms_paged_attention_form: more than 65535 sequences or kv heads");
  a.q_start = bt.q_start;
  a.context_lens = bt.context_lens;
  a.positions = bt.positions;
  a.tables = bt.block_tables;
  a.n_tokens = bt.n_tokens;
  a.n_seqs = bt.n_seqs;
  a.max_blocks = bt.max_blocks;
  a.max_q = bt.max_q_len;
  a.bs = c.block_size;
  a.num_blocks = c.num_blocks;
  a.hq = hq;
  a.hkv = c.n_kv_heads;
  a.group = hq / c.n_kv_heads;
  a.k = c.k_pool[layer];
  a.v = c.v_pool[layer];
  a.scale = 1.f / sqrtf((float)c.d_head);
  if (form) {
    MS_REQUIRE(form->scale >= 0.f && form->scale <= FLT_MAX && form->softcap >= 0.f &&
                   form->softcap <= FLT_MAX && form->window >= 0 && form->mask_words >= 0,
               "ms_paged_attention_form: scale, softcap, window and mask_words must be >= 0 and finite");
    MS_REQUIRE(!form->tree_mask || form->mask_words > 0, "ms_paged_attention_form: a mask of no words");
    if (form->scale > 0.f) a.scale = form->scale;
    // (scale / softcap is a factor of its own in the kernels)
    MS_REQUIRE(form->softcap == 0.f || a.scale / form->softcap <= 1e30f,
               "ms_paged_attention_form: a softcap of %g is too small for a scale of %g", form->softcap, a.scale);
    a.softcap = form->softcap;
    a.window = form->window;
    a.slopes = form->slopes;
    a.prefix = form->prefix_lens;
    a.mask = form->tree_mask;
    a.mask_words = form->mask_words;
  }
  const int bound = bt.max_blocks * c.block_size;
  *max_context = bt.max_context > 0 ? min(bt.max_context, bound) : bound;
  return MS_OK;
}

}  // namespace

template <typename T, bool kBase2>
int form_combine(const FormArgs& a, int rows, int dh, cudaStream_t s) {
  const int warps = min(8, max(2, a.n_splits / 2));
  dim3 grid(a.max_q * a.group, a.hkv, a.n_seqs);
  launch_pdl(form_combine_kernel<T, kBase2>, grid, warps * 32,
             (((a.n_splits + 3) & ~3) + warps * dh) * sizeof(float), s, a, rows, dh);
  return check_launch("form_combine_kernel");
}
template int form_combine<__nv_bfloat16, true>(const FormArgs& a, int rows, int dh, cudaStream_t s);

int attention_form(const void* q, int64_t q_stride, const ms_kv_cache& c, int layer,
                   const ms_batch& bt, int hq, const ms_attention_form* form, void* out,
                   int64_t out_stride, void* workspace, size_t workspace_bytes, cudaStream_t s,
                   const int32_t* seq_order) {
  FormArgs a{};
  int max_context = 0;
  MS_TRY(form_args(a, c, layer, bt, hq, form, &max_context));
  if (bt.n_seqs == 0 || bt.n_tokens == 0) return MS_OK;
  a.q = q;
  a.q_stride = q_stride;
  a.out = out;
  a.out_stride = out_stride;
  a.err = device_error_word();
  ProfScope prof(kClsAttention, s);
  const Way way = choose(a, c, max_context);
  const int rows = way.rows;
  size_t parts = part_bytes(a, rows, c.d_head);
  if (parts > workspace_bytes) {  // one range a tile
    a.n_splits = 1;
    a.split_len = INT_MAX;
    parts = 0;
  }
  if (a.n_splits > 1) {
    a.part_o = static_cast<float*>(workspace);
    a.part_ml = a.part_o + (size_t)a.n_seqs * a.hkv * a.row_tiles * a.n_splits * rows * c.d_head;
  }
  if (way.order) {
    a.order = seq_order;
    if (!seq_order && workspace_bytes - parts >= (size_t)a.n_seqs * sizeof(int32_t)) {
      int32_t* order = reinterpret_cast<int32_t*>(static_cast<unsigned char*>(workspace) + parts);
      MS_TRY(attn_seq_order(bt.context_lens, a.n_seqs, order, s));
      a.order = order;
    }
  }
  if (way.kernel == kTma) return form_tma(a, c.d_head, s);
  if (way.kernel == kTc) return form_tc(a, c.d_head, rows, s);
  return c.dtype == MS_DTYPE_F32 ? simt_by_dh<float>(a, c.d_head, s)
                                 : simt_by_dh<__nv_bfloat16>(a, c.d_head, s);
}

size_t attention_form_workspace(const ms_kv_cache& c, const ms_batch& bt, int hq,
                                const ms_attention_form* form) {
  FormArgs a{};
  int max_context = 0;
  if (form_args(a, c, 0, bt, hq, form, &max_context) != MS_OK || bt.n_seqs == 0 || bt.n_tokens == 0)
    return 0;
  const Way way = choose(a, c, max_context);
  return part_bytes(a, way.rows, c.d_head) + (way.order ? a.n_seqs * sizeof(int32_t) : 0);
}

}  // namespace ms

using namespace ms;

extern "C" size_t ms_attention_form_workspace_size(const ms_kv_cache* cache, int n_heads,
                                                   const ms_batch* batch,
                                                   const ms_attention_form* form) {
  if (validate_cache(cache, 0) != MS_OK || batch == nullptr) return 0;
  return attention_form_workspace(*cache, *batch, n_heads, form);
}

extern "C" int ms_paged_attention_form(const void* q, int64_t q_stride, const ms_kv_cache* cache,
                                       int layer, const ms_batch* batch, int n_heads,
                                       const ms_attention_form* form, void* out, int64_t out_stride,
                                       void* workspace, size_t workspace_bytes, void* stream) {
  MS_TRY(validate_cache(cache, layer));
  MS_REQUIRE(batch != nullptr, "ms_paged_attention_form: null batch");
  if (batch->n_seqs > 0 && batch->n_tokens > 0) {
    MS_REQUIRE(q && out, "ms_paged_attention_form: null pointer");
    MS_REQUIRE(batch->q_start && batch->context_lens && batch->positions && batch->block_tables,
               "ms_paged_attention_form: batch has null arrays");
    const int64_t width = (int64_t)n_heads * cache->d_head;
    MS_REQUIRE(q_stride >= width && out_stride >= width,
               "ms_paged_attention_form: strides below n_heads * d_head");
    MS_REQUIRE(workspace != nullptr || workspace_bytes == 0,
               "ms_paged_attention_form: workspace missing");
    MS_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 16 == 0,
               "ms_paged_attention_form: workspace must be 16-byte aligned");
  }
  return attention_form(q, q_stride, *cache, layer, *batch, n_heads, form, out, out_stride,
                        workspace, workspace_bytes, as_stream(stream));
}
