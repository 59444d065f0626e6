// Trees of drafted tokens: their visibility masks, and the walk down each
// tree along the target's tokens.
#include <climits>

#include <cooperative_groups.h>

#include "common.cuh"

namespace ms {
namespace {

constexpr int kWide = 256;  // threads of a CTA that walks a tree over long rows of logits

// The nodes [t0, t0 + n) of sequence b, cut to the call's arrays (and reported).
__device__ __forceinline__ int tree_nodes(const int32_t* q_start, int b, int n_tokens, int max_nodes,
                                          int& t0, int* err) {
  t0 = q_start[b];
  int end = q_start[b + 1];
  if (t0 < 0 || end < t0 || end > n_tokens || end - t0 > max_nodes) {
    if (threadIdx.x == 0) raise_device_error(err, kErrLength);
    t0 = min(max(t0, 0), n_tokens);
    end = min(max(end, t0), min(n_tokens, t0 + max_nodes));
  }
  return end - t0;
}

// The parents of a tree in shared memory, bad ones as roots.
__device__ __forceinline__ void load_parents(const int32_t* parents, int t0, int n, int* s_parent, int* err) {
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    int p = parents[t0 + i];
    if (p < -1 || p >= i) {
      raise_device_error(err, kErrTree);
      p = -1;
    }
    s_parent[i] = p;
  }
}

// One CTA a tree, a thread a word column: row i = the parent's row and bit i.
// Parents come before their children, so a thread goes through the nodes once; the
// chain of shared-memory reads (about 30 cycles a node) is what it takes.  Rows
// of large trees stay in the output itself.
__global__ void __launch_bounds__(128)
    tree_masks_kernel(const int32_t* __restrict__ parents, const int32_t* __restrict__ q_start,
                      int n_tokens, int max_nodes, uint32_t* masks, int words, int32_t* depths, int shared_words,
                      int* err) {
  pdl_enter();
  __shared__ int s_parent[MS_TREE_MAX];
  __shared__ int s_depth[MS_TREE_MAX];
  extern __shared__ uint32_t s_rows[];  // (max_nodes, words) when shared_words
  int t0;
  const int n = tree_nodes(q_start, blockIdx.x, n_tokens, max_nodes, t0, err);
  load_parents(parents, t0, n, s_parent, err);
  __syncthreads();
  uint32_t* out = masks + (int64_t)t0 * words;
  uint32_t* rows = shared_words ? s_rows : out;
  if (threadIdx.x == blockDim.x - 1) {
    for (int i = 0; i < n; ++i) s_depth[i] = s_parent[i] < 0 ? 0 : s_depth[s_parent[i]] + 1;
  }
  for (int w = threadIdx.x; w < words; w += blockDim.x)
    for (int i = 0; i < n; ++i) {
      const int p = s_parent[i];
      const uint32_t up = p < 0 ? 0u : rows[p * words + w];
      rows[i * words + w] = up | ((i >> 5) == w ? 1u << (i & 31) : 0u);
    }
  __syncthreads();
  if (shared_words)
    for (int i = threadIdx.x; i < n * words; i += blockDim.x) out[i] = s_rows[i];
  if (depths)
    for (int i = threadIdx.x; i < n; i += blockDim.x) depths[t0 + i] = s_depth[i];
}

struct AcceptArgs {
  const float* logits;
  int64_t stride;
  int vocab;
  const int32_t* target;
  const int32_t *ids, *q_start, *context_lens, *tables, *parents;
  int n_tokens, max_nodes, max_blocks, max_accept, bs, num_blocks;
  int32_t *out_tokens, *out_num, *out_nodes, *src, *dst;
  int* err;
};

struct Best {
  float v;
  int i;
};
// The larger value, the lower index of equals; NaN compares false and never wins.
__device__ __forceinline__ Best better(Best a, Best b) {
  return b.v > a.v || (b.v == a.v && b.i < a.i) ? b : a;
}

// The best of x[lo, hi): 16 bytes at a time from the first aligned element on.  A thread's
// indices ascend, so only a larger value replaces its best; of four values their maximum
// is compared first (a row of -inf or NaN leaves the index at INT_MAX).
template <int kThreads>
__device__ __forceinline__ Best best_of(const float* x, int lo, int hi) {
  constexpr int kUnroll = 4;
  Best m{-INFINITY, INT_MAX};
  const int tid = threadIdx.x;
  const int head = min(hi, lo + (int)((4 - ((reinterpret_cast<uintptr_t>(x + lo) >> 2) & 3)) & 3));
  const int quads = (hi - head) >> 2;
  auto take = [&](float v, int i) {
    if (v > m.v) m = Best{v, i};
  };
  if (tid < head - lo) take(x[lo + tid], lo + tid);
  const float4* x4 = reinterpret_cast<const float4*>(x + head);
  for (int q0 = tid; q0 < quads; q0 += kUnroll * kThreads) {
    float4 v[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      v[u] = q0 + u * kThreads < quads ? __ldcs(x4 + q0 + u * kThreads)
                                           : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (fmaxf(fmaxf(v[u].x, v[u].y), fmaxf(v[u].z, v[u].w)) > m.v) {
        const int i = head + 4 * (q0 + u * kThreads);
        take(v[u].x, i);
        take(v[u].y, i + 1);
        take(v[u].z, i + 2);
        take(v[u].w, i + 3);
      }
    }
  }
  const int tail = head + 4 * quads + tid;
  if (tail < hi) take(x[tail], tail);
  return m;
}

__device__ __forceinline__ Best warp_best(Best m) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    m = better(m, Best{__shfl_xor_sync(0xffffffffu, m.v, o), __shfl_xor_sync(0xffffffffu, m.i, o)});
  return m;
}

// A cluster of CTAs a sequence.  Each step: the largest logit of the current
// node's row, a slice a CTA, the slices' bests exchanged through distributed
// shared memory (two buffers in turn, so one cluster barrier a step), then the
// lowest child with that token.  All CTAs of a cluster take the same steps.
// Short rows, and tokens that are given, take one warp: 256 trees take 8.7 us with it and 9.7 with 8
// warps at 65 logits, 9.7 and 8.9 at 1024.  Long ones wait for HBM, at a rate that
// falls as paths end: 192 trees of 128256 logits, 511 rows of which are read (262 MB), 53 us, 5.0 TB/s
// (8 values of 16 bytes a thread in flight instead of 4 57 us, 2 of them 83; 512 threads 58).
template <int kThreads>
__global__ void __launch_bounds__(kThreads) tree_accept_kernel(AcceptArgs a) {
  pdl_enter();
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int parts = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  __shared__ int s_parent[MS_TREE_MAX];
  __shared__ int s_token[MS_TREE_MAX];
  __shared__ Best s_warp[kThreads / 32];
  __shared__ Best s_part[2][8];
  __shared__ int s_child;
  const int b = blockIdx.x / parts, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int t0;
  const int n = tree_nodes(a.q_start, b, a.n_tokens, a.max_nodes, t0, a.err);
  load_parents(a.parents, t0, n, s_parent, a.err);
  for (int i = tid; i < n; i += kThreads) s_token[i] = a.ids[t0 + i];
  const int64_t held = (int64_t)a.max_blocks * a.bs;
  int ctx = a.src ? a.context_lens[b] : n;
  if (a.src && (ctx < n || ctx > held)) {
    if (tid == 0) raise_device_error(a.err, kErrLength);
    ctx = ctx < n ? n : (int)held;
  }
  const int base = ctx - n;
  const int32_t* table = a.tables + (int64_t)b * a.max_blocks;
  auto slot = [&](int j) {
    if (j >= held) return -1;
    const int blk = table[j / a.bs];
    if (blk < 0 || blk >= a.num_blocks) {
      raise_device_error(a.err, kErrBlock);
      return -1;
    }
    return blk * a.bs + j % a.bs;
  };
  // (shared memory of another CTA may be written once that CTA has started)
  if (parts > 1) cluster.sync(); else __syncthreads();

  const int per = ((a.vocab + parts - 1) / parts + 3) & ~3;
  const int lo = min(rank * per, a.vocab), hi = min(lo + per, a.vocab);
  const bool writes = rank == 0 && tid == 0;
  int32_t* tokens = a.out_tokens + (int64_t)b * (a.max_accept + 1);
  const int64_t at = (int64_t)b * a.max_accept;
  int node = 0, accepted = 0, said = 0;
  for (int step = 0; step <= a.max_accept && n > 0; ++step) {
    int token;
    if (a.logits) {
      Best m = warp_best(best_of<kThreads>(a.logits + (int64_t)(t0 + node) * a.stride, lo, hi));
      if (lane == 0) s_warp[warp] = m;
      if (tid == 0) s_child = INT_MAX;
      __syncthreads();
      if (warp == 0) {
        m = lane < kThreads / 32 ? s_warp[lane] : Best{-INFINITY, INT_MAX};
        m = warp_best(m);
        if (lane < parts) *cluster.map_shared_rank(&s_part[step & 1][rank], lane) = m;
      }
      if (parts > 1) cluster.sync(); else __syncthreads();
      m = s_part[step & 1][0];
      for (int k = 1; k < parts; ++k) m = better(m, s_part[step & 1][k]);
      token = m.i == INT_MAX ? 0 : m.i;
    } else {
      if (tid == 0) s_child = INT_MAX;
      token = a.target[t0 + node];
      __syncthreads();
    }
    if (writes) tokens[step] = token;
    ++said;
    if (step == a.max_accept) break;
    for (int i = node + 1 + tid; i < n; i += kThreads)
      if (s_parent[i] == node && s_token[i] == token) {
        atomicMin(&s_child, i);
        break;
      }
    __syncthreads();
    const int child = s_child;
    __syncthreads();
    if (child == INT_MAX) break;
    node = child;
    if (writes) {
      a.out_nodes[at + accepted] = node;
      if (a.src) {
        const int from = slot(base + node), to = slot(base + accepted + 1);
        a.src[at + accepted] = from < 0 || to < 0 ? -1 : from;
        a.dst[at + accepted] = from < 0 || to < 0 ? -1 : to;
      }
    }
    ++accepted;
  }
  if (rank != 0) return;
  if (tid == 0) a.out_num[b] = accepted;
  for (int k = said + tid; k <= a.max_accept; k += kThreads) tokens[k] = -1;
  for (int k = accepted + tid; k < a.max_accept; k += kThreads) {
    a.out_nodes[at + k] = -1;
    if (a.src) a.src[at + k] = a.dst[at + k] = -1;
  }
}

}  // namespace
}  // namespace ms

using namespace ms;

extern "C" int ms_tree_masks(const int32_t* parents, const int32_t* q_start, int n_seqs, int n_tokens,
                             int max_nodes, uint32_t* masks, int mask_words, int32_t* depths,
                             void* stream) {
  MS_REQUIRE(n_seqs >= 0 && n_tokens >= 0 && max_nodes >= 0, "ms_tree_masks: bad sizes");
  if (max_nodes > MS_TREE_MAX)
    return fail(MS_ERR_TOO_LARGE, "ms_tree_masks: trees of %d nodes (at most %d)", max_nodes, MS_TREE_MAX);
  if (n_seqs == 0 || n_tokens == 0) return MS_OK;
  MS_REQUIRE(parents && q_start && masks, "ms_tree_masks: null pointer");
  MS_REQUIRE(mask_words >= ceil_div(max_nodes, 32), "ms_tree_masks: %d words for %d nodes", mask_words,
             max_nodes);
  // (the kernel's row indices are 32 bits wide)
  MS_REQUIRE((int64_t)max_nodes * mask_words <= INT_MAX, "ms_tree_masks: %d words for each of %d nodes",
             mask_words, max_nodes);
  const int64_t bytes = (int64_t)max_nodes * mask_words * 4;
  const bool shared = bytes <= 32 * 1024;  // with the parents and depths within 48 KB
  launch_pdl(tree_masks_kernel, n_seqs, 128, shared ? (size_t)bytes : 0, as_stream(stream), parents,
             q_start, n_tokens, max_nodes, masks, mask_words, depths, (int)shared, device_error_word());
  return check_launch("tree_masks_kernel");
}

extern "C" int ms_tree_accept(const float* logits, int64_t logits_stride, int vocab,
                              const int32_t* target_tokens, const ms_batch* batch,
                              const int32_t* parents, int max_accept, int block_size, int num_blocks,
                              int32_t* out_tokens, int32_t* out_num_accepted, int32_t* out_nodes,
                              int32_t* src_slots, int32_t* dst_slots, void* stream) {
  MS_REQUIRE(batch != nullptr, "ms_tree_accept: null batch");
  MS_REQUIRE((logits != nullptr) != (target_tokens != nullptr) || batch->n_tokens == 0,
             "ms_tree_accept: either logits or target_tokens");
  MS_REQUIRE(batch->n_seqs >= 0 && batch->n_tokens >= 0 && batch->max_q_len >= 0 && max_accept >= 0,
             "ms_tree_accept: bad sizes");
  MS_REQUIRE(!logits || (vocab > 0 && (logits_stride >= vocab || batch->n_tokens == 1)),
             "ms_tree_accept: vocab %d, stride %lld", vocab, (long long)logits_stride);
  MS_REQUIRE((src_slots != nullptr) == (dst_slots != nullptr) || max_accept == 0,
             "ms_tree_accept: src_slots and dst_slots, both or neither");
  MS_REQUIRE(!src_slots || (block_size > 0 && num_blocks > 0 && batch->max_blocks > 0),
             "ms_tree_accept: bad cache sizes");
  if (batch->max_q_len > MS_TREE_MAX)
    return fail(MS_ERR_TOO_LARGE, "ms_tree_accept: trees of %d nodes (at most %d)", batch->max_q_len,
                MS_TREE_MAX);
  if (batch->n_seqs == 0) return MS_OK;
  MS_REQUIRE(batch->q_start && (!src_slots || (batch->context_lens && batch->block_tables)) && out_tokens &&
                 out_num_accepted && (out_nodes || max_accept == 0) &&
                 (batch->n_tokens == 0 || (batch->input_ids && parents)),
             "ms_tree_accept: null pointer");
  MS_REQUIRE((int64_t)batch->max_blocks * max(block_size, 1) <= INT_MAX, "ms_tree_accept: contexts beyond 2^31");
  AcceptArgs a{};
  a.logits = logits;
  a.stride = logits_stride;
  a.vocab = vocab;
  a.target = target_tokens;
  a.ids = batch->input_ids;
  a.q_start = batch->q_start;
  a.context_lens = batch->context_lens;
  a.tables = batch->block_tables;
  a.parents = parents;
  a.n_tokens = batch->n_tokens;
  a.max_nodes = batch->max_q_len;
  a.max_blocks = batch->max_blocks;
  a.max_accept = max_accept;
  a.bs = block_size > 0 ? block_size : 1;
  a.num_blocks = num_blocks;
  a.out_tokens = out_tokens;
  a.out_num = out_num_accepted;
  a.out_nodes = out_nodes;
  a.src = src_slots;
  a.dst = dst_slots;
  a.err = device_error_word();
  // A cluster as wide as leaves all sequences resident (8 CTAs an SM), slices of at least 2560
  // logits: 8 trees, 4096 logits, 1 CTA 8.7 us and 2 CTAs 10.7; 32000 logits, 1, 4 and 8 CTAs 19.3,
  // 12.6 and 11.2 us; 192 trees, 128256 logits, 1 and 4 CTAs 103.6 and 52.9 us.
  int parts = 1;
  while (logits && parts < 8 && (int64_t)batch->n_seqs * parts * 2 <= 148 * 8 && vocab / (parts * 2) >= 2560)
    parts *= 2;
  if ((int64_t)batch->n_seqs * parts > INT_MAX)
    return fail(MS_ERR_TOO_LARGE, "ms_tree_accept: too many sequences");
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(batch->n_seqs * parts));
  const bool narrow = !logits || vocab <= 512;
  cfg.blockDim = dim3(narrow ? 32 : kWide);
  cfg.stream = as_stream(stream);
  cudaLaunchAttribute attr[2] = {};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)parts;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  (void)cudaLaunchKernelEx(&cfg, narrow ? tree_accept_kernel<32> : tree_accept_kernel<kWide>, a);
  return check_launch("tree_accept_kernel");
}
