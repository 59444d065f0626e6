// The adapters' products on tcgen05, for tiles of many tokens (prompts).
//
// The second one,
//   y[t, n] = base[t, n] + sum_r B[r, n] s_{j(n)}[t, r],
// with the epilogues of lora.cu.  A CTA takes up to 128 tokens of one adapter
// (two neighbouring tiles of the plan) and goes through its share of the
// columns, 128 at a step:
//   warps 0, 1  load each step's adapter rows by cp.async, a ring slot per warp, into
//               the 128-byte swizzle that the MMA reads (warp 2 only fills the group);
//   warp 3      allocates TMEM; lane 0 issues tcgen05.mma with s (bf16 terms side
//               by side along k) as A in TMEM, copied there once, so that the
//               MMAs read only B from shared memory.  The adapter rows are (rank,
//               column) in memory, so B is MN-major.  Gate | up columns
//               (alternating every 8) are parted by the load into two blocks of
//               64, one accumulator each; columns where one slice ends and
//               another begins take a step for each, which stores its own slice's;
//   warps 4-19  epilogue: TMEM lane quarter warp % 4, 32 of the columns each; a
//               thread has one row.  Each warp brings its own base in by cp.async,
//               two steps ahead (16 warps keep more copies in flight than a few
//               loading ones: 3 warps moved 30 KB per us), and sends the result
//               out in 32- to 64-byte row segments through a 2 KB exchange.
// TMEM: two accumulators of 128 columns, then s (up to 256).  One CTA per SM.
// The kernel moves 4 bytes in per column and token and 1 to 4 out: HBM is its
// floor, and shared memory sees the base twice and little else.  8192 tokens, rank
// 64-128, N = 28672 with the SwiGLU (1.2 GB): 301 us (4.0 TB/s) on 130 of the 148
// SMs, one wave of a CTA per pair of tiles and half of the columns, about 3700
// cycles for each step of 128 x 128; issue slots 44%, tensor pipe 23%, L2 54% busy.
// The same with s as A in shared memory and both slices against all columns 447 us,
// by mma.sync 671.
#include <cooperative_groups.h>

#include "lora_device.cuh"

namespace ms {
namespace {

constexpr int kRows = 128;          // tokens per CTA
constexpr int kChunk = 128;         // columns per step
constexpr int kSAt = 2 * kChunk;    // TMEM column of s
constexpr int kLoadThreads = 96;  // two loading warps and an idle one: the fourth of their group issues the MMAs
constexpr int kEpiWarps = 16;
constexpr int kThreads = kLoadThreads + 32 + 32 * kEpiWarps;
constexpr int kSegment = 32 * 128;                    // base of 32 rows x 32 columns
constexpr int kEpiBytes = 2 * kSegment + 32 * 64;     // two of them, and the exchange, per warp
constexpr int kStages = 2;          // steps in the ring, a loading warp each
constexpr int kBarBytes = 256;
constexpr int kMostBytes = 226 * 1024;
constexpr long long kWaitCycles = 1ll << 32;  // ~2.2 s
constexpr int kErrTimeout = 5;

__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, volatile int* stop, int* err) {
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
    if (*stop) return false;
    if (clock64() - t0 > kWaitCycles) {
      *stop = 1;
      atomicCAS(err, 0, kErrTimeout);
      return false;
    }
  }
}
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* stop, int* err) {
  return __all_sync(0xffffffffu, bar_wait(bar, parity, stop, err));
}
// After a wait that ran out: the MMAs committed to `bar` end before the block goes.
__device__ __forceinline__ void drain(uint32_t bar, int* err) {
  int go_on = 0;
  bar_wait(bar, 0, &go_on, err);
}
// Descriptors with the 128-byte swizzle.  K-major: rows of 64 k values, groups of
// 8 rows 1024 bytes apart (lead 16: not used).  Adapter rows, MN-major: 64 columns per
// 128-byte row, groups of 8 k rows 1024 bytes apart (stride offset), blocks of
// 64 columns `lead` bytes apart.
__device__ __forceinline__ uint64_t desc(uint32_t addr, uint32_t lead) {
  uint64_t d = (uint64_t)((addr & 0x3FFFFu) >> 4);
  d |= (uint64_t)(lead >> 4) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}
// f32 accumulator, bf16 operands, A (in TMEM) K-major, B MN-major, M 128.
__device__ __forceinline__ uint32_t instr(int n) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(kRows >> 4) << 24);
}
__device__ __forceinline__ void umma(uint32_t d, uint32_t a, uint64_t b, uint32_t id,
                                     uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(id), "r"(accumulate)
      : "memory");
}
// The same with A in shared memory.
__device__ __forceinline__ void umma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(id), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void umma_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar)
               : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_st8(uint32_t addr, const uint4& a, const uint4& b) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(addr),
               "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b.x), "r"(b.y), "r"(b.z), "r"(b.w)
               : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
// The load and its wait in one, so that nothing that uses the values comes between.
__device__ __forceinline__ void tmem_ld8_wait(uint32_t addr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7])
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void st4(uint32_t addr, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(x), "r"(y), "r"(z), "r"(w)
               : "memory");
}
__device__ __forceinline__ uint4 ld4(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// How many tiles directly before tile i continue to it: the same adapter, full,
// the positions before (the whole warp calls it).
__device__ int tiles_before(const ms_lora_plan& p, int i, int start, int adapter) {
  const int lane = threadIdx.x & 31;
  const int4* tiles = reinterpret_cast<const int4*>(p.tiles);
  int n = 0;
  while (true) {
    const int k = n + 1 + lane;  // the k-th tile before
    bool same = false;
    if (i - k >= 0) {
      const int4 q = tiles[i - k];
      same = q.z == adapter && q.y == kTile && q.x == start - kTile * k && q.x >= 0;
    }
    const uint32_t m = __ballot_sync(0xffffffffu, same);
    if (m != 0xffffffffu) return n + __ffs(~m) - 1;
    n += 32;
  }
}

// The tokens of tile `index` and, when it continues it, of the next one: false
// for a bad or empty tile and for one that the tile before has taken.  The same
// for every warp.
__device__ bool load_pair(const ms_lora_plan& p, const ms_lora_adapters& ad, int index, Tile& tile,
                          int& count, int* err) {
  if (!load_tile(p, ad, index, tile, err) || tile.count == 0) return false;
  if (tiles_before(p, index, tile.start, tile.adapter) & 1) return false;
  count = tile.count;
  if (count == kTile && index + 1 < p.n_tiles) {
    const int4 q = reinterpret_cast<const int4*>(p.tiles)[index + 1];
    if (q.z == tile.adapter && q.x == tile.start + kTile) {
      if (q.y >= 0 && q.y <= kTile && q.x <= p.n_tokens - q.y)
        count += q.y;
      else if (threadIdx.x == 0)
        raise_device_error(err, kErrAdapter);
    }
  }
  return true;
}

// ---- first product ---------------------------------------------------------------
// s of up to 128 tokens x 256 rank rows per CTA: both operands K-major, k in steps
// of 64 through a ring of four slots, two loading warps each; k is shared out
// over a cluster, whose parts meet in distributed shared memory, summed in
// cluster order.  The MMAs of eight steps make a partial sum in one of two
// accumulators; the loading warps add it up in float32 registers while their next
// copies are in flight.  (An MMA truncates its sum to 24 bits, always towards zero: a
// running sum over K = 14336 comes out 1.4e-5 too small, over 512 k values 5e-7.  The
// whole call below took 302 us with one running sum, 304 with eight steps, 308 with four.)
// x is read once, A by every pair of tiles out of L2.  8192 tokens,
// K = 4096, two slices of rank 64-128 (73 MB): 48 us, by mma.sync 95; about 15 us of
// it start, the hand-over of 128 KB of sums per CTA through shared memory, and the
// stores of s.
constexpr int kSteps = 4;                       // ring slots
constexpr int kSumSteps = 8;                    // steps of a partial sum, a multiple of kSteps
constexpr int kStepK = 64;
constexpr int kRankRows = 256;                  // most rank rows per CTA
constexpr int kStepBytes = (kRows + kRankRows) * 128;
constexpr int kPartLd = kRankRows + 4;          // floats per token of the parts
constexpr int kShrinkBytes = 1024 + kBarBytes + kSteps * kStepBytes;
constexpr int kShrinkThreads = 288;             // 8 loading warps, 1 for the MMAs
constexpr int kShrinkTmem = 2 * kRankRows;      // two accumulators
static_assert(kRows * kPartLd * 4 <= kSteps * kStepBytes, "the parts fit the ring");

__global__ void __launch_bounds__(kShrinkThreads, 1) lora_shrink_tc_kernel(ShrinkArgs p) {
  pdl_enter();
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  __shared__ int s_tok[kRows];
  __shared__ int s_row[kRankRows];  // row of A, -1: padding
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int splits = (int)cluster.num_blocks(), split = (int)cluster.block_rank();
  const uint32_t raw = s_addr(smem_raw);
  const uint32_t ring = raw + ((1024u - (raw & 1023u)) & 1023u), bars = ring + kSteps * kStepBytes;
  const uint32_t full = bars, empty = full + 8 * kSteps, summed = empty + 8 * kSteps, taken = summed + 16,
                 ended = taken + 16, slot_addr = ended + 8;
  unsigned char* gbars = smem_raw + (bars - raw);
  volatile uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(gbars + (slot_addr - bars));
  volatile int* stop = reinterpret_cast<int*>(gbars + (slot_addr - bars) + 4);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  Tile tile;
  int count = 0;
  if (!load_pair(p.plan, p.ad, blockIdx.x, tile, count, p.err)) return;  // the whole cluster alike
  const int rank_p = pad16(tile.rank), rows = p.ns * rank_p, m0 = blockIdx.y * kRankRows;
  if (m0 >= rows) return;
  const int here = min(kRankRows, rows - m0);  // a multiple of 16
  for (int i = tid; i < kRows; i += kShrinkThreads)
    s_tok[i] = i < count ? token_at(p.plan, tile.start + i, p.err) : -1;
  for (int i = tid; i < here; i += kShrinkThreads) {
    const int j = (m0 + i) / rank_p, r = m0 + i - j * rank_p;
    s_row[i] = r < tile.rank ? p.ns * tile.offset + j * tile.rank + r : -1;
  }
  if (tid == 0) {
    for (int k = 0; k < kSteps; ++k) {
      bar_init(full + 8 * k, 64);
      bar_init(empty + 8 * k, 1);
    }
    for (int k = 0; k < 2; ++k) {
      bar_init(summed + 8 * k, 1);
      bar_init(taken + 8 * k, 8);
    }
    bar_init(ended, 1);
    *stop = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot_addr),
                 "r"(kShrinkTmem));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = *tmem_slot;
  const int k_begin = split * p.k_per, k_end = min(p.K, k_begin + p.k_per);
  const int steps = k_end > k_begin ? (k_end - k_begin + kStepK - 1) / kStepK : 0;

  const int sums = (steps + kSumSteps - 1) / kSumSteps;
  if (warp < 8) {
    // ---- loads: 16 bytes at k offset 8 i of rows r0, r0 + 8, ...
    const int group = warp >> 1, t = tid & 63, i = t & 7, r0 = t >> 3;
    // ---- the partial sums: lane quarter warp & 3, half the columns
    const int row0 = 32 * (warp & 3), c0 = (warp >> 2) * 128;
    float acc[128] = {};
    bool alive = true;
    auto take = [&](int sum) {
      alive = alive && warp_wait(summed + 8 * (sum & 1), (sum >> 1) & 1, stop, p.err);
      if (!alive) return;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t from = tmem + (sum & 1) * kRankRows + c0 + ((uint32_t)row0 << 16);
#pragma unroll
      for (int c = 0; c < 128; c += 8) {
        if (c0 + c >= here) break;
        uint32_t r[8];
        tmem_ld8_wait(from + c, r);
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[c + e] += __uint_as_float(r[e]);
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) bar_arrive(taken + 8 * (sum & 1));
    };
    int taken_sums = 0;
    for (int step = group; step < steps; step += kSteps) {
      if (step >= kSteps) {
        alive = alive && warp_wait(empty + 8 * group, (step / kSteps - 1) & 1, stop, p.err);
        if (!alive) break;
      }
      const int k = k_begin + step * kStepK + 8 * i;
      const bool in = k < k_end;
      // (row & 7 is r0 for all of a thread's rows)
      const uint32_t to = ring + group * kStepBytes + r0 * 128 + ((i ^ r0) << 4);
      const __nv_bfloat16* x = p.x + (in ? k : 0);
#pragma unroll 8
      for (int r = 0; r < kRows; r += 8) {
        const int tok = s_tok[r + r0];
        cp_async16(to + r * 128, x + max(tok, 0) * p.x_stride, in && tok >= 0);
      }
      const __nv_bfloat16* a = p.a + (in ? k : 0);
#pragma unroll 8
      for (int r = 0; r < here; r += 8) {
        const int row = s_row[r + r0];
        cp_async16(to + kRows * 128 + r * 128, a + (int64_t)max(row, 0) * p.K, in && row >= 0);
      }
      cp_commit();
      if (taken_sums < step / kSumSteps) take(taken_sums++);  // while the copies are in flight
      cp_wait<0>();
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      bar_arrive(full + 8 * group);
    }
    while (taken_sums < sums) take(taken_sums++);  // (all MMAs have ended: the ring is free)
    float* part = reinterpret_cast<float*>(smem_raw + (ring - raw));  // [token][kPartLd]
#pragma unroll
    for (int c = 0; c < 128; c += 4) {
      if (c0 + c >= here) break;
      *reinterpret_cast<float4*>(part + (row0 + lane) * kPartLd + c0 + c) =
          make_float4(acc[c], acc[c + 1], acc[c + 2], acc[c + 3]);
    }
  } else if (lane == 0) {
    // ---- MMA
    const uint32_t id = instr(here) & ~(1u << 16);  // B K-major as well
    bool fine = true;
    int step = 0;
    for (; step < steps; ++step) {
      const int slot = step % kSteps, sum = step / kSumSteps;
      const bool first = step % kSumSteps == 0;
      if (first && sum > 1 && !(fine = bar_wait(taken + 8 * (sum & 1), ((sum >> 1) - 1) & 1, stop, p.err))) break;
      if (!(fine = bar_wait(full + 8 * slot, (step / kSteps) & 1, stop, p.err))) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint64_t x = desc(ring + slot * kStepBytes, 16), a = desc(ring + slot * kStepBytes + kRows * 128, 16);
      const uint32_t d = tmem + (sum & 1) * kRankRows;
#pragma unroll
      for (int k = 0; k < kStepK / 16; ++k) umma_ss(d, x + 2 * k, a + 2 * k, id, !first || k > 0);
      umma_commit(empty + 8 * slot);
      if (step % kSumSteps == kSumSteps - 1 || step == steps - 1) umma_commit(summed + 8 * (sum & 1));
    }
    if (!fine && step > 0) {
      umma_commit(ended);
      drain(ended, p.err);
    }
  }
  __syncwarp();
  if (splits > 1) cluster.sync(); else __syncthreads();
  finish_s(p, cluster, reinterpret_cast<const float*>(smem_raw + (ring - raw)), kPartLd, tile.start,
           count, m0, here, tile.rank, p.ad.scales[tile.adapter]);
  if (splits > 1) cluster.sync(); else __syncthreads();  // no CTA leaves while another reads its part
  if (warp == 8)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kShrinkTmem));
}

// Shared memory for a rank; 0 when it or TMEM do not do.
int ring_bytes(int terms, int ns, int rank_pm) {
  const int bytes = 1024 + kBarBytes + kEpiWarps * kEpiBytes + kStages * rank_pm * kChunk * 2;
  return bytes <= kMostBytes && ns * terms * rank_pm / 2 <= 512 - kSAt ? bytes : 0;
}

template <int EPI>
__global__ void __launch_bounds__(kThreads, 1) lora_expand_tc_kernel(ExpandArgs p) {
  constexpr int TERMS = EPI == kLoraF32 ? 3 : 2;
  const bool parted = EPI == kLoraSwiGLU || p.interleaved;  // gate | up columns
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  __shared__ int s_tok[kRows];
  const uint32_t raw = s_addr(smem_raw);
  const uint32_t base = raw + ((1024u - (raw & 1023u)) & 1023u);
  // adapter rows of a step in two blocks of 64 columns; each epilogue warp's base
  // rows and exchange
  const uint32_t ring = base, stage_bytes = p.rank_pm * kChunk * 2;
  const uint32_t s_x = ring + kStages * stage_bytes, bars = s_x + kEpiWarps * kEpiBytes;
  const uint32_t full = bars, empty = full + 8 * kStages, s_ready = empty + 8 * kStages;
  const uint32_t tfull = s_ready + 8, tempty = tfull + 16, drained = tempty + 16, slot_addr = drained + 8;
  unsigned char* gbars = smem_raw + (bars - raw);
  volatile uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(gbars + (slot_addr - bars));
  volatile int* stop = reinterpret_cast<int*>(gbars + (slot_addr - bars) + 4);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // The plan and the adapters are read before the launch wait (see lora.cu).
  if (!p.after_shrink) pdl_enter();
  Tile tile;
  int count = 0;
  const bool work = load_pair(p.plan, p.ad, blockIdx.y, tile, count, p.err) &&
                    !(p.in_place && tile.rank == 0);
  if (!work) {
    if (p.after_shrink) pdl_enter();
    return;
  }
  const int rank_p = pad16(tile.rank);
  const int n_chunks = (p.N + kChunk - 1) / kChunk;
  const int chunks = (n_chunks - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x;
  auto column = [&](int chunk) { return ((int)blockIdx.x + chunk * (int)gridDim.x) * kChunk; };
  // The steps of this CTA, the same for every warp: a chunk of columns each, or one for
  // each slice (pass) where a slice ends inside the chunk.
  struct Walk {
    int chunk, pass, c, passes;
  };
  auto enter = [&](int chunk) {
    const int c = column(chunk);
    return Walk{chunk, 0, c, parted ? 1 : slice_of(p, min(c + kChunk, p.N) - 1) - slice_of(p, c) + 1};
  };
  auto next = [&](Walk w) {
    if (++w.pass < w.passes) return w;
    return w.chunk + 1 < chunks ? enter(w.chunk + 1) : Walk{chunks, 0, 0, 1};
  };
  auto slice_at = [&](const Walk& w) { return parted ? 0 : slice_of(p, w.c) + w.pass; };

  if (threadIdx.x < kRows)
    s_tok[threadIdx.x] =
        threadIdx.x < count ? token_at(p.plan, tile.start + threadIdx.x, p.err) : -1;
  if (threadIdx.x == 0) {
    for (int k = 0; k < kStages; ++k) {
      bar_init(full + 8 * k, 32);
      bar_init(empty + 8 * k, 1);
    }
    bar_init(s_ready, kEpiWarps);
    bar_init(drained, 1);
    for (int k = 0; k < 2; ++k) {
      bar_init(tfull + 8 * k, 1);
      bar_init(tempty + 8 * k, kEpiWarps);
    }
    *stop = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 3) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot_addr),
                 "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = *tmem_slot;

  if (warp < 3) {
    // ---- loads of the adapter rows.  Each warp fills its own slot of the ring, so
    // that a slot waiting to be free does not hold up the others.
    const int q = lane & 15, r0 = lane >> 4;
    auto load_b = [&](uint32_t dst, int c0) {
      const int c = c0 + 8 * q;
      // block and place of these 8 columns: gate | up parted, else in order
      const int block = parted ? q & 1 : q >> 3, at = parted ? q >> 1 : q & 7;
      const uint32_t to = dst + block * (rank_p * 128);
      const bool in = c < p.N;
      const __nv_bfloat16* src = p.b + ((int64_t)tile.offset + r0) * p.N + (in ? c : 0);
      constexpr int kStep = 2;
      const int64_t jump = (int64_t)kStep * p.N;
      const int last = in ? tile.rank : 0;  // rows past it: zeros
#pragma unroll 8
      for (int r = r0; r < rank_p; r += kStep, src += jump)
        cp_async16(to + r * 128 + ((at ^ (r & 7)) << 4), r < last ? src : p.b, r < last);
    };
    int step = 0;
    for (Walk w = enter(0); warp < kStages && w.chunk < chunks; w = next(w), ++step) {
      if (step % kStages != warp) continue;
      if (step >= kStages && !warp_wait(empty + 8 * warp, (step / kStages - 1) & 1, stop, p.err)) break;
      load_b(ring + warp * stage_bytes, w.c);
      cp_commit();
      cp_wait<0>();
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      bar_arrive(full + 8 * warp);
    }
    if (p.after_shrink) pdl_enter();  // lora_shrink does not write the adapter rows
  } else if (warp == 3) {
    // ---- MMA
    if (p.after_shrink) pdl_enter();
    if (lane == 0 && bar_wait(s_ready, 0, stop, p.err)) {
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      int step = 0;
      bool fine = true;
      for (Walk w = enter(0); w.chunk < chunks; w = next(w), ++step) {
        const int buf = step & 1, use = step >> 1, slot = step % kStages;
        if (use >= 1 && !(fine = bar_wait(tempty + 8 * buf, (use - 1) & 1, stop, p.err))) break;
        if (!(fine = bar_wait(full + 8 * slot, (step / kStages) & 1, stop, p.err))) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t d = tmem + buf * kChunk, lead = rank_p * 128;
        const uint64_t b0 = desc(ring + slot * stage_bytes, lead);
        const uint32_t term = rank_p / 2, slice = TERMS * term;  // TMEM columns
        // all terms and rank steps of one slice into `to`
        auto products = [&](uint32_t to, uint32_t a, uint64_t bj, uint32_t id) {
          for (int e = TERMS - 1; e >= 0; --e) {  // the small terms first
            const uint32_t ae = a + e * term;
            umma(to, ae, bj, id, e < TERMS - 1);
#pragma unroll 4
            for (int k = 16; k < rank_p; k += 16) umma(to, ae + k / 2, bj + k * 8, id, 1u);
          }
        };
        if (rank_p > 0 && parted) {
          for (int j = 0; j < 2; ++j)
            products(d + 64 * j, tmem + kSAt + j * slice, b0 + j * (lead >> 4), instr(64));
        } else if (rank_p > 0) {
          products(d, tmem + kSAt + slice_at(w) * slice, b0, instr(kChunk));
        }
        umma_commit(empty + 8 * slot);
        umma_commit(tfull + 8 * buf);
      }
      if (!fine) {
        umma_commit(drained);
        drain(drained, p.err);
      }
    }
    __syncwarp();
  } else {
    // ---- epilogue: one 32-column segment of the chunk per warp
    if (p.after_shrink) pdl_enter();
    const int quarter = warp & 3, part = (warp - 4) >> 2;
    const uint32_t base_buf = s_x + (warp - 4) * kEpiBytes, x = base_buf + 2 * kSegment;
    const int row0 = 32 * quarter;
    const int rows = max(0, min(32, count - row0));
    const uint32_t lanes = (uint32_t)row0 << 16;
    {  // s into TMEM: a row's bytes are the TMEM words of its lane; shared out over `part`
      const __nv_bfloat16* src = p.s + (tile.start + min(row0 + lane, count - 1)) * p.s_stride;
      const int words = p.ns * TERMS * rank_p / 2;
      for (int w = 8 * part; w < words; w += 32) {
        uint4 a = make_uint4(0, 0, 0, 0), b = a;
        if (row0 + lane < count) {
          a = *reinterpret_cast<const uint4*>(src + 2 * w);
          b = *reinterpret_cast<const uint4*>(src + 2 * w + 8);
        }
        tmem_st8(tmem + kSAt + w + lanes, a, b);
      }
      asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) bar_arrive(s_ready);
    }
    // 16-byte chunk k of row r in the exchange
    auto place = [&](int r, int k) { return x + r * 64 + ((k ^ ((r >> 1) & 3)) << 4); };
    const int n_out = EPI == kLoraSwiGLU ? p.N / 2 : p.N;
    constexpr int kHalves = EPI == kLoraF32 ? 2 : 1;
    constexpr int kChunks = EPI == kLoraSwiGLU ? 2 : 4;  // of 16 bytes per row
    constexpr int kPer = EPI == kLoraF32 ? 4 : 8;        // outputs per chunk
    // element offsets of this lane's output rows (lora_add checks that they fit 32 bits)
    uint32_t out_at[kChunks], has = 0;
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const int at = 32 * i + lane, r = at / kChunks;
      const int tok = r < rows ? s_tok[row0 + r] : -1;
      has |= (uint32_t)(tok >= 0) << i;
      out_at[i] = (uint32_t)(max(tok, 0) * p.out_stride + at % kChunks * kPer);
    }
    // The base comes by cp.async, two steps ahead, into this warp's own rows
    // (16-byte chunk k of row r at k ^ (r & 7)); lane l loads chunk l & 7 of rows
    // (l >> 3) + 4 i.
    uint32_t base_at[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = 4 * i + (lane >> 3);
      base_at[i] = (uint32_t)(max(r < rows ? s_tok[row0 + r] : 0, 0) * p.base_stride + 4 * (lane & 7));
    }
    auto load_base = [&](const Walk& w, int buf) {
      if (w.chunk < chunks && rows > 0) {
        const int c = w.c + 32 * part;
        const bool in = c + 4 * (lane & 7) < p.N;
        const uint32_t to = base_buf + buf * kSegment + (lane >> 3) * 128;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          cp_async16(to + 512 * i + (((lane & 7) ^ ((4 * i + (lane >> 3)) & 7)) << 4),
                     in ? p.base + (base_at[i] + c) : p.base, in);
      }
      cp_commit();
    };
    Walk w = enter(0), ahead = next(w);
    load_base(w, 0);
    load_base(ahead, 1);
    for (int step = 0; w.chunk < chunks; w = next(w), ++step) {
      const int buf = step & 1, c = w.c + 32 * part;
      float y[32];
      // the base of this thread's row
      cp_wait<1>();
      __syncwarp();
      if (rows > 0) {
        const uint32_t from = base_buf + buf * kSegment + lane * 128;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const uint4 v = ld4(from + ((k ^ (lane & 7)) << 4));
          y[4 * k] = __uint_as_float(v.x);
          y[4 * k + 1] = __uint_as_float(v.y);
          y[4 * k + 2] = __uint_as_float(v.z);
          y[4 * k + 3] = __uint_as_float(v.w);
        }
      }
      __syncwarp();
      ahead = next(ahead);
      load_base(ahead, buf);
      if (!warp_wait(tfull + 8 * buf, (step >> 1) & 1, stop, p.err)) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      if (rows > 0 && rank_p > 0) {
        uint32_t acc[32];
        const uint32_t d = tmem + buf * kChunk + lanes;
        // two gate groups and two up groups, or 32 columns in order
        tmem_ld16(d + (parted ? 16 * part : 32 * part), acc);
        tmem_ld16(d + (parted ? 64 + 16 * part : 32 * part + 16), acc + 16);
        tmem_wait_ld();
#pragma unroll
        for (int k = 0; k < 32; ++k)
          y[k] += __uint_as_float(parted ? acc[(k & 7) + ((k >> 4) << 3) + ((k >> 3 & 1) << 4)] : acc[k]);
      }
      // the accumulators are in registers: the next MMAs may have them
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) bar_arrive(tempty + 8 * buf);
      if (rows > 0) {
        // the results, rows of up to 64 bytes at a time
        const int c_out = EPI == kLoraSwiGLU ? c / 2 : c;
#pragma unroll
        for (int h = 0; h < kHalves; ++h) {
#pragma unroll
          for (int k = 0; k < kChunks; ++k) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if constexpr (EPI == kLoraF32) {
                w[e] = __float_as_uint(y[16 * h + 4 * k + e]);
              } else if constexpr (EPI == kLoraBf16) {
                w[e] = pack2(y[8 * k + 2 * e], y[8 * k + 2 * e + 1]);
              } else {  // 16 k: gate, 16 k + 8: up
                w[e] = pack2(silu(y[16 * k + 2 * e]) * y[16 * k + 8 + 2 * e],
                             silu(y[16 * k + 2 * e + 1]) * y[16 * k + 9 + 2 * e]);
              }
            }
            st4(place(lane, k), w[0], w[1], w[2], w[3]);
          }
          __syncwarp();
#pragma unroll
          for (int i = 0; i < kChunks; ++i) {
            const int at = 32 * i + lane, r = at / kChunks, k = at % kChunks;
            const int col = c_out + 16 * h;
            if (!(has >> i & 1u) || col + k * kPer >= n_out) continue;
            const uint4 q = ld4(place(r, k));
            if (EPI != kLoraSwiGLU && w.passes > 1) {  // this slice's columns alone
              const int n = col + k * kPer, j = slice_at(w);
              if (slice_of(p, n) != j || slice_of(p, n + kPer - 1) != j) {
                const uint32_t word[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                for (int e = 0; e < kPer; ++e) {
                  if (slice_of(p, n + e) != j) continue;
                  if constexpr (EPI == kLoraF32)
                    static_cast<uint32_t*>(p.out)[out_at[i] + col + e] = word[e];
                  else
                    static_cast<uint16_t*>(p.out)[out_at[i] + col + e] = (uint16_t)(word[e >> 1] >> 16 * (e & 1));
                }
                continue;
              }
            }
            if constexpr (EPI == kLoraF32)
              *reinterpret_cast<uint4*>(static_cast<float*>(p.out) + (out_at[i] + col)) = q;
            else
              *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p.out) + (out_at[i] + col)) = q;
          }
          __syncwarp();
        }
      }
    }
    cp_wait<0>();
  }
  __syncwarp();
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 3)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
}

template <int EPI>
int launch(const ExpandArgs& p, cudaStream_t s) {
  const int bytes = ring_bytes(EPI == kLoraF32 ? 3 : 2, p.ns, p.rank_pm);
  if (bytes == 0) return MS_ERR_UNSUPPORTED;
  static std::atomic<uint64_t> granted{0};
  MS_TRY(grant_dynamic_smem(lora_expand_tc_kernel<EPI>, kMostBytes, granted));
  // CTAs per pair of tiles: the number whose rounds over the GPU take the
  // fewest steps, a CTA's start counted as four
  const int pairs = (p.plan.n_tiles + 1) / 2, chunks = ceil_div(p.N, kChunk);
  int gx = 1;
  int64_t best = INT64_MAX;
  for (int n = 1; n <= min(chunks, 64); ++n) {
    const int64_t cost = (int64_t)ceil_div(pairs * n, 148) * (ceil_div(chunks, n) + 4);
    if (cost < best) {
      best = cost;
      gx = n;
    }
  }
  launch_pdl(lora_expand_tc_kernel<EPI>, dim3(gx, p.plan.n_tiles), kThreads, bytes, s, p);
  return check_launch("lora_expand_tc_kernel");
}

}  // namespace

int lora_shrink_tc(ShrinkArgs p, int rows, cudaStream_t s) {
  static std::atomic<uint64_t> granted{0};
  MS_TRY(grant_dynamic_smem(lora_shrink_tc_kernel, kShrinkBytes, granted));
  // as many CTAs along k as one round over the GPU takes, at least 256 k values each
  const int blocks = ceil_div(rows, kRankRows), ctas = (p.plan.n_tiles + 1) / 2 * blocks;
  int split = 1;
  while (split < 8 && 2 * split * ctas <= 148 && p.K / (2 * split) >= 256) split *= 2;
  p.k_per = ceil_div(ceil_div(p.K, split), kStepK) * kStepK;
  return launch_cluster(lora_shrink_tc_kernel, dim3(p.plan.n_tiles, blocks, split), kShrinkThreads,
                        kShrinkBytes, split, s, p);
}

int lora_expand_tc(const ExpandArgs& p, int epilogue, cudaStream_t s) {
  if (p.rank_pm == 0) return MS_ERR_UNSUPPORTED;
  if (epilogue == kLoraSwiGLU) return launch<kLoraSwiGLU>(p, s);
  return epilogue == kLoraF32 ? launch<kLoraF32>(p, s) : launch<kLoraBf16>(p, s);
}

}  // namespace ms
