// Pages copied and tokens moved inside the paged K/V pools, every layer in one
// launch (up to kLayers of them).
//
// Both only move bytes: 2 x the copied bytes is the floor.
#include "common.cuh"
#include "model_kernels.cuh"

namespace ms {
namespace {

constexpr int kLayers = 128;  // layers per launch: their pool pointers are kernel arguments
constexpr int kThreads = 256;

struct Pools {
  void* p[2 * kLayers];  // K and V of layer l at 2 l and 2 l + 1
};

// The (layer, K or V) pools are copied side by side: element e of a page is
// copied by one thread of the CTA that has its tile of kUnroll * kThreads
// elements; all loads of a thread are in flight before its stores.  Bound by HBM: 4001 pages of 22 layers, 4
// heads of 64 (2.9 GB moved) take 430 us, 6.7 TB/s.
template <typename V>
__global__ void __launch_bounds__(kThreads)
    kv_copy_blocks_kernel(const __grid_constant__ Pools pools, const int32_t* __restrict__ src,
                          const int32_t* __restrict__ dst, int n, int page, int num_blocks, int* err) {
  pdl_enter();
  constexpr int kUnroll = 4;
  V* pool = static_cast<V*>(pools.p[blockIdx.y]);
  const int64_t total = (int64_t)n * page;
  const int64_t e0 = (int64_t)blockIdx.x * (kUnroll * kThreads) + threadIdx.x;
  V v[kUnroll];
  int64_t to[kUnroll];
#pragma unroll
  for (int i = 0; i < kUnroll; ++i) {
    const int64_t e = e0 + i * kThreads;
    to[i] = -1;
    if (e < total) {
      const int pair = (int)(e / page), at = (int)(e - (int64_t)pair * page);
      const int from = src[pair], into = dst[pair];
      if ((unsigned)from >= (unsigned)num_blocks || (unsigned)into >= (unsigned)num_blocks) {
        raise_device_error(err, kErrBlock);
      } else if (from != into) {
        v[i] = pool[(int64_t)from * page + at];
        to[i] = (int64_t)into * page + at;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kUnroll; ++i)
    if (to[i] >= 0) pool[to[i]] = v[i];
}

// The source and destination rows of a pair in (row units of) one head's pool;
// false for a pair that moves nothing.
__device__ __forceinline__ bool move_pair(const int32_t* src, const int32_t* dst, int64_t i, int bs,
                                          int hkv, int num_slots, int64_t& from, int64_t& to, int* err) {
  const int f = src[i], t = dst[i];
  if (f < 0 || t < 0 || f == t) return false;
  if (f >= num_slots || t >= num_slots) {
    raise_device_error(err, kErrSlot);
    return false;
  }
  from = (int64_t)(f / bs) * hkv * bs + f % bs;
  to = (int64_t)(t / bs) * hkv * bs + t % bs;
  return true;
}

// `team` threads (a power of two, 32 to kThreads) a (group, kv head): they hold the group's rows, up to
// kRegs elements of `row` a thread, in registers before the first is stored, kPools pools
// at a time, and go through the pools of their slice (blockIdx.y of gridDim.y).  The
// places are worked out once a slice: their divisions take longer than the copies of a pool.
// Bound by latency: with two slices a warp goes through 32 pools in eight rounds of loads, a barrier and stores, none
// of which begins before the one before has ended (DRAM 31%, warps active 28%).  192 groups, 32
// layers, 8 heads of 128 take 19, 27 and 42 us for up to 5, 8 and 24 moves (82, 95 and 113 MB:
// 4.3, 3.5 and 2.7 TB/s); with 4 elements a thread 23, 26 and 58 us, with 8 pools at a time
// instead of 4 20, 27 and 43.
template <typename V, int kRegs, int kPools>
__global__ void __launch_bounds__(kThreads)
    kv_move_kernel(const __grid_constant__ Pools pools, int n_pools, const int32_t* __restrict__ src,
                   const int32_t* __restrict__ dst, int n_groups, int per_group, int row, int bs,
                   int hkv, int num_slots, int team, int* err) {
  pdl_enter();
  const int member = threadIdx.x & (team - 1), elements = per_group * row;
  const int64_t unit = ((int64_t)blockIdx.x * kThreads + threadIdx.x) / team;
  const int group = (int)(unit / hkv), h = (int)(unit - (int64_t)group * hkv);
  int64_t from[kRegs], to[kRegs];
#pragma unroll
  for (int i = 0; i < kRegs; ++i) {
    to[i] = -1;
    const int e = member + team * i;
    if (e >= elements || group >= n_groups) continue;
    const int m = e / row, at = e - m * row;
    if (move_pair(src, dst, (int64_t)group * per_group + m, bs, hkv, num_slots, from[i], to[i], err)) {
      from[i] = (from[i] + (int64_t)h * bs) * row + at;
      to[i] = (to[i] + (int64_t)h * bs) * row + at;
    }
  }
  const int p0 = (int)((int64_t)n_pools * blockIdx.y / gridDim.y);
  const int p1 = (int)((int64_t)n_pools * (blockIdx.y + 1) / gridDim.y);
  for (int p = p0; p < p1; p += kPools) {
    V v[kPools][kRegs];
#pragma unroll
    for (int u = 0; u < kPools; ++u) {
      if (p + u >= p1) break;
      const V* base = static_cast<const V*>(pools.p[p + u]);
#pragma unroll
      for (int i = 0; i < kRegs; ++i)
        if (to[i] >= 0) v[u][i] = base[from[i]];
    }
    if (team > 32) __syncthreads(); else __syncwarp();
#pragma unroll
    for (int u = 0; u < kPools; ++u) {
      if (p + u >= p1) break;
      V* base = static_cast<V*>(pools.p[p + u]);
#pragma unroll
      for (int i = 0; i < kRegs; ++i)
        if (to[i] >= 0) base[to[i]] = v[u][i];
    }
  }
}

// Groups of more than kRegs * kThreads elements: a CTA a (group, kv head, pool), the rows in shared
// memory (the three groups above would take 118, 128 and 206 us).
template <typename V>
__global__ void __launch_bounds__(kThreads)
    kv_move_shared_kernel(const __grid_constant__ Pools pools, const int32_t* __restrict__ src,
                          const int32_t* __restrict__ dst, int per_group, int row, int bs, int hkv,
                          int num_slots, int* err) {
  pdl_enter();
  extern __shared__ __align__(16) unsigned char smem[];
  V* rows = reinterpret_cast<V*>(smem);
  const int group = blockIdx.x / hkv, h = blockIdx.x % hkv;
  V* pool = static_cast<V*>(pools.p[blockIdx.y]) + (int64_t)h * bs * row;
  for (int e = threadIdx.x; e < per_group * row; e += kThreads) {
    int64_t from, to;
    if (move_pair(src, dst, (int64_t)group * per_group + e / row, bs, hkv, num_slots, from, to, err))
      rows[e] = pool[from * row + e % row];
  }
  __syncthreads();
  for (int e = threadIdx.x; e < per_group * row; e += kThreads) {
    int64_t from, to;
    if (move_pair(src, dst, (int64_t)group * per_group + e / row, bs, hkv, num_slots, from, to, err))
      pool[to * row + e % row] = rows[e];
  }
}

// Calls f(pools, count) for every kLayers layers; 16-byte elements when rows and pools allow.
template <typename F>
int over_layers(const ms_kv_cache& c, F f) {
  for (int l0 = 0; l0 < c.n_layers; l0 += kLayers) {
    Pools p{};
    const int n = min(kLayers, c.n_layers - l0);
    for (int l = 0; l < n; ++l) {
      p.p[2 * l] = c.k_pool[l0 + l];
      p.p[2 * l + 1] = c.v_pool[l0 + l];
    }
    MS_TRY(f(p, 2 * n));
  }
  return MS_OK;
}

int check_pools(const ms_kv_cache* c, int* row_bytes, bool* wide, const char* what) {
  MS_TRY(validate_cache(c, 0));
  MS_REQUIRE(c->dtype == MS_DTYPE_F32 || c->dtype == MS_DTYPE_BF16, "%s: dtype %d", what, c->dtype);
  *row_bytes = c->d_head * (c->dtype == MS_DTYPE_BF16 ? 2 : 4);
  uintptr_t any = (uintptr_t)*row_bytes;
  for (int l = 0; l < c->n_layers; ++l) {
    MS_REQUIRE(c->k_pool[l] && c->v_pool[l], "%s: null pool for layer %d", what, l);
    any |= reinterpret_cast<uintptr_t>(c->k_pool[l]) | reinterpret_cast<uintptr_t>(c->v_pool[l]);
  }
  MS_REQUIRE(any % 4 == 0, "%s: pools and rows must be 4-byte aligned", what);
  MS_REQUIRE((int64_t)c->num_blocks * c->block_size <= INT32_MAX &&
                 (int64_t)c->n_kv_heads * c->block_size * *row_bytes <= INT32_MAX,
             "%s: a pool of 2^31 slots or a page of 2^31 bytes", what);
  *wide = any % 16 == 0;
  return MS_OK;
}

template <typename V>
int copy_blocks(const ms_kv_cache& c, const int32_t* src, const int32_t* dst, int n, int row_bytes,
                cudaStream_t s) {
  const int page = c.n_kv_heads * c.block_size * (row_bytes / (int)sizeof(V));
  const int64_t tiles = ((int64_t)n * page + 4 * kThreads - 1) / (4 * kThreads);
  MS_REQUIRE(tiles <= INT32_MAX, "ms_kv_copy_blocks: too many blocks");
  return over_layers(c, [&](const Pools& p, int count) {
    launch_pdl(kv_copy_blocks_kernel<V>, dim3((unsigned)tiles, count), kThreads, 0, s, p, src,
               dst, n, page, c.num_blocks, device_error_word());
    return check_launch("kv_copy_blocks_kernel");
  });
}

template <typename V>
int move_tokens(const ms_kv_cache& c, const int32_t* src, const int32_t* dst, int n_groups,
                int per_group, int row_bytes, cudaStream_t s) {
  const int row = row_bytes / (int)sizeof(V), num_slots = c.num_blocks * c.block_size;
  const int64_t units = (int64_t)n_groups * c.n_kv_heads;
  MS_REQUIRE(units <= INT32_MAX, "ms_kv_move_tokens: too many groups");
  constexpr int kRegs = 3, kPools = 4;
  int team = 32;
  while (team < kThreads && team * kRegs < per_group * row) team *= 2;
  const bool in_registers = team * kRegs >= per_group * row;
  const int64_t ctas = (units * team + kThreads - 1) / kThreads;
  const int bytes = per_group * row_bytes;
  static std::atomic<uint64_t> granted{0};
  if (!in_registers && bytes > 48 * 1024) {
    if (bytes > 227 * 1024)
      return fail(MS_ERR_TOO_LARGE, "ms_kv_move_tokens: %d rows of %d bytes a group", per_group, row_bytes);
    MS_TRY(grant_dynamic_smem(kv_move_shared_kernel<V>, 227 * 1024, granted));
  }
  return over_layers(c, [&](const Pools& p, int count) {
    int* err = device_error_word();
    // (two CTAs an SM: 64 groups in 22 layers 4.9 us, 6.0 with four)
    const int slices = (int)min((int64_t)ceil_div(count, kPools), (148 * 2 + ctas - 1) / ctas);
    if (in_registers)
      launch_pdl(kv_move_kernel<V, kRegs, kPools>, dim3((unsigned)ctas, slices), kThreads, 0, s, p, count, src, dst,
                 n_groups, per_group, row, c.block_size, c.n_kv_heads, num_slots, team, err);
    else
      launch_pdl(kv_move_shared_kernel<V>, dim3((unsigned)units, count), kThreads, bytes, s, p,
                 src, dst, per_group, row, c.block_size, c.n_kv_heads, num_slots, err);
    return check_launch("kv_move_kernel");
  });
}

}  // namespace
}  // namespace ms

using namespace ms;

extern "C" int ms_kv_copy_blocks(const ms_kv_cache* cache, const int32_t* src_blocks,
                                 const int32_t* dst_blocks, int n_blocks, void* stream) {
  int row_bytes = 0;
  bool wide = false;
  MS_TRY(check_pools(cache, &row_bytes, &wide, "ms_kv_copy_blocks"));
  MS_REQUIRE(n_blocks >= 0, "ms_kv_copy_blocks: n_blocks < 0");
  if (n_blocks == 0) return MS_OK;
  MS_REQUIRE(src_blocks && dst_blocks, "ms_kv_copy_blocks: null pointer");
  return wide ? copy_blocks<uint4>(*cache, src_blocks, dst_blocks, n_blocks, row_bytes, as_stream(stream))
              : copy_blocks<uint32_t>(*cache, src_blocks, dst_blocks, n_blocks, row_bytes, as_stream(stream));
}

extern "C" int ms_kv_move_tokens(const ms_kv_cache* cache, const int32_t* src_slots,
                                 const int32_t* dst_slots, int n_groups, int per_group, void* stream) {
  int row_bytes = 0;
  bool wide = false;
  MS_TRY(check_pools(cache, &row_bytes, &wide, "ms_kv_move_tokens"));
  MS_REQUIRE(n_groups >= 0 && per_group >= 0, "ms_kv_move_tokens: bad sizes");
  if (per_group > MS_KV_MOVE_MAX)
    return fail(MS_ERR_TOO_LARGE, "ms_kv_move_tokens: %d moves a group (at most %d)", per_group, MS_KV_MOVE_MAX);
  if (n_groups == 0 || per_group == 0) return MS_OK;
  MS_REQUIRE(src_slots && dst_slots, "ms_kv_move_tokens: null pointer");
  return wide ? move_tokens<uint4>(*cache, src_slots, dst_slots, n_groups, per_group, row_bytes,
                                   as_stream(stream))
              : move_tokens<uint32_t>(*cache, src_slots, dst_slots, n_groups, per_group, row_bytes,
                                      as_stream(stream));
}
