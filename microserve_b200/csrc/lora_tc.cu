// The adapters' second product on tcgen05, for tiles of many tokens (prompts):
//   y[t, n] = base[t, n] + sum_r B[r, n] s_{j(n)}[t, r],
// with the epilogues of lora.cu.  A CTA takes up to 128 tokens of one adapter
// (two neighbouring tiles of the plan) and goes through its share of the
// columns, 128 at a step:
//   warps 0-2   load: s once (K-major, the bf16 terms side by side along k),
//               then each step's adapter rows, by cp.async into the 128-byte
//               swizzle that the MMA reads;
//   warp 3      allocates TMEM; lane 0 issues tcgen05.mma M128 N128 K16.  The
//               adapter rows are (rank, column) in memory, so B is MN-major.
//               With two slices in the 128 columns (gate | up alternate every
//               8) both s are multiplied with all of them, into two
//               accumulators, of which the epilogue takes the columns it needs;
//   warps 4-11  epilogue: TMEM lane quarter warp % 4, columns by half.  The base
//               comes in and the result goes out in whole 128-byte row segments
//               through a 4 KB exchange per warp, as in gemm_tc.cu.
// The 4 accumulators (two steps x two slices) fill the 512 TMEM columns, so one
// CTA runs per SM.  The kernel moves 4 bytes in per column and token and 1 to 4
// out, and is bound by HBM.
#include "lora_device.cuh"

namespace ms {
namespace {

constexpr int kRows = 128;          // tokens per CTA
constexpr int kChunk = 128;         // columns per step
constexpr int kPanel = kRows * 128; // bytes of a 64-wide k panel of s
constexpr int kLoadThreads = 96;
constexpr int kEpiWarps = 8;
constexpr int kThreads = kLoadThreads + 32 + 32 * kEpiWarps;
constexpr int kExchange = 32 * 128;
constexpr int kMaxStages = 4;
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
// 128-byte swizzle descriptors.  K-major (s): 8-row groups 1024 bytes apart.
// MN-major (adapter rows): 64 columns per 128-byte row, groups of 8 k rows 1024
// bytes apart (stride offset), blocks of 64 columns `lead` bytes apart.
__device__ __forceinline__ uint64_t desc(uint32_t addr, uint32_t lead) {
  uint64_t d = (uint64_t)((addr & 0x3FFFFu) >> 4);
  d |= (uint64_t)(lead >> 4) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}
// f32 accumulator, bf16 operands, A K-major, B MN-major, M 128, N 128.
constexpr uint32_t kInstr = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) |
                            ((uint32_t)(kChunk >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);
__device__ __forceinline__ void umma(uint32_t d, uint64_t a, uint64_t b, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(kInstr), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void umma_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar)
               : "memory");
}
__device__ __forceinline__ void tmem_ld8(uint32_t addr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_wait_ld() {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
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
      same = q.z == adapter && q.y == kTile && q.x == start - kTile * k;
    }
    const uint32_t m = __ballot_sync(0xffffffffu, same);
    if (m != 0xffffffffu) return n + __ffs(~m) - 1;
    n += 32;
  }
}

// Stage counts and bytes for a rank: 0 stages when the shared memory does not do.
struct Layout {
  int panels;  // k panels of s per slice
  int stages, bytes;
};
template <int TERMS>
__host__ __device__ __forceinline__ Layout layout(int ns, int rank_pm) {
  Layout l;
  l.panels = (TERMS * rank_pm + 63) / 64;
  const int fixed = 1024 + kBarBytes + kEpiWarps * kExchange + ns * l.panels * kPanel;
  const int stage = rank_pm * kChunk * 2;
  l.stages = stage > 0 ? (kMostBytes - fixed) / stage : 0;
  if (l.stages > kMaxStages) l.stages = kMaxStages;
  if (l.stages < 2) l.stages = 0;
  l.bytes = fixed + l.stages * stage;
  return l;
}

template <int EPI>
__global__ void __launch_bounds__(kThreads, 1) lora_expand_tc_kernel(ExpandArgs p) {
  constexpr int TERMS = EPI == kLoraF32 ? 3 : 2;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  __shared__ int s_tok[kRows];
  const uint32_t raw = s_addr(smem_raw);
  const uint32_t base = raw + ((1024u - (raw & 1023u)) & 1023u);
  const Layout lay = layout<TERMS>(p.ns, p.rank_pm);
  const uint32_t s_s = base, s_b = s_s + p.ns * lay.panels * kPanel;
  const uint32_t stage_bytes = p.rank_pm * kChunk * 2;
  const uint32_t s_x = s_b + lay.stages * stage_bytes, bars = s_x + kEpiWarps * kExchange;
  const uint32_t full = bars, empty = full + 8 * kMaxStages, s_ready = empty + 8 * kMaxStages;
  const uint32_t tfull = s_ready + 8, tempty = tfull + 16, slot_addr = tempty + 16;
  unsigned char* gbars = smem_raw + (bars - raw);
  volatile uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(gbars + (slot_addr - bars));
  volatile int* stop = reinterpret_cast<int*>(gbars + (slot_addr - bars) + 4);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // The plan and the adapters are read before the launch wait (see lora.cu).
  if (!p.after_shrink) pdl_enter();
  Tile tile;
  const int index = blockIdx.y;
  bool work = load_tile(p.plan, p.ad, index, tile, p.err) && tile.count > 0 &&
              !(p.in_place && tile.rank == 0);
  int count = tile.count;
  if (work) {
    if (tiles_before(p.plan, index, tile.start, tile.adapter) & 1) {
      work = false;  // the CTA of the tile before has this one
    } else if (count == kTile && index + 1 < p.plan.n_tiles) {
      const int4 q = reinterpret_cast<const int4*>(p.plan.tiles)[index + 1];
      if (q.z == tile.adapter && q.x == tile.start + kTile) {
        if (q.y >= 0 && q.y <= kTile && q.x <= p.plan.n_tokens - q.y)
          count += q.y;
        else if (threadIdx.x == 0)
          raise_device_error(p.err, kErrAdapter);
      }
    }
  }
  if (!work) {
    if (p.after_shrink) pdl_enter();
    return;
  }
  const int rank_p = pad16(tile.rank);
  const int n_chunks = (p.N + kChunk - 1) / kChunk;
  const int steps = (n_chunks - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x;
  auto column = [&](int step) { return ((int)blockIdx.x + step * (int)gridDim.x) * kChunk; };
  // the slices of a step's columns: first, and whether there are two
  auto first_slice = [&](int c) { return p.interleaved ? 0 : slice_of(p, c); };
  auto last_slice = [&](int c) { return p.interleaved ? 1 : slice_of(p, min(c + kChunk, p.N) - 1); };

  if (threadIdx.x < kRows)
    s_tok[threadIdx.x] =
        threadIdx.x < count ? token_at(p.plan, tile.start + threadIdx.x, p.err) : -1;
  if (threadIdx.x == 0) {
    for (int k = 0; k < lay.stages; ++k) {
      bar_init(full + 8 * k, kLoadThreads);
      bar_init(empty + 8 * k, 1);
    }
    bar_init(s_ready, kLoadThreads);
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
    // ---- loads.  A thread's copies of a step: 16 bytes, 8 columns, of rank rows
    // r0, r0 + 6, ...; then a fence, so that the MMA's reads see them, and an arrive.
    const int tid = threadIdx.x;
    const int q = tid & 15, r0 = tid >> 4;
    auto load_b = [&](int step) {
      const int stage = step % lay.stages, c = column(step) + 8 * q;
      const uint32_t block = s_b + stage * stage_bytes + (q >> 3) * (rank_p * 128);
      const bool in = c < p.N;
      const __nv_bfloat16* src = p.b + ((int64_t)tile.offset + r0) * p.N + (in ? c : 0);
      for (int r = r0; r < rank_p; r += kLoadThreads / 16, src += (int64_t)(kLoadThreads / 16) * p.N) {
        const bool ok = in && r < tile.rank;
        cp_async16(block + r * 128 + (((q & 7) ^ (r & 7)) << 4), ok ? src : p.b, ok);
      }
    };
    if (p.after_shrink) {
      load_b(0);  // not written by lora_shrink
      pdl_enter();
    }
    const int row_chunks = TERMS * rank_p / 8;  // 16-byte chunks of one slice of a row
    for (int j = 0; j < p.ns; ++j)
      for (int i = tid; i < kRows * row_chunks; i += kLoadThreads) {
        const int m = i / row_chunks, k = i - m * row_chunks;
        const uint32_t dst = s_s + (j * lay.panels + (k >> 3)) * kPanel + m * 128 + (((k & 7) ^ (m & 7)) << 4);
        const bool ok = m < count;
        cp_async16(dst, ok ? p.s + (tile.start + m) * p.s_stride + j * TERMS * rank_p + 8 * k : p.s, ok);
      }
    if (!p.after_shrink) load_b(0);
    cp_commit();
    const int ahead = lay.stages > 2 ? lay.stages - 2 : 1;  // steps loaded before the one handed over
    for (int step = 1; step < ahead; ++step) {
      if (step < steps) load_b(step);
      cp_commit();
    }
    for (int step = 0; step < steps; ++step) {
      const int next = step + ahead;
      if (next < steps) {
        if (next >= lay.stages &&
            !bar_wait(empty + 8 * (next % lay.stages), (next / lay.stages - 1) & 1, stop, p.err))
          break;
        load_b(next);
      }
      cp_commit();
      if (ahead > 1) cp_wait<2>(); else cp_wait<1>();  // this step's copies have arrived
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      if (step == 0) bar_arrive(s_ready);
      bar_arrive(full + 8 * (step % lay.stages));
    }
    cp_wait<0>();
  } else if (warp == 3) {
    // ---- MMA
    if (p.after_shrink) pdl_enter();
    if (lane == 0 && bar_wait(s_ready, 0, stop, p.err)) {
      for (int step = 0; step < steps; ++step) {
        const int stage = step % lay.stages, buf = step & 1, use = step >> 1;
        if (use >= 1 && !bar_wait(tempty + 8 * buf, (use - 1) & 1, stop, p.err)) break;
        if (!bar_wait(full + 8 * stage, (step / lay.stages) & 1, stop, p.err)) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const int c = column(step), j0 = first_slice(c), j1 = last_slice(c);
        const uint32_t b = s_b + stage * stage_bytes;
        for (int j = j0; j <= j1; ++j) {
          const uint32_t d = tmem + buf * 256 + (j - j0) * kChunk;
          const uint32_t a = s_s + j * lay.panels * kPanel;
          uint32_t acc = 0;
          for (int e = TERMS - 1; e >= 0; --e)  // the small terms first
            for (int k = 0; k < rank_p; k += 16, acc = 1) {
              const int at = e * rank_p + k;
              umma(d, desc(a + (at >> 6) * kPanel + (at & 63) * 2, 16), desc(b + k * 128, rank_p * 128), acc);
            }
        }
        umma_commit(empty + 8 * stage);
        umma_commit(tfull + 8 * buf);
      }
    }
    __syncwarp();
  } else {
    // ---- epilogue
    if (p.after_shrink) pdl_enter();
    const int quarter = warp & 3, half = (warp - 4) >> 2;
    const uint32_t x = s_x + (warp - 4) * kExchange;
    const int row0 = 32 * quarter;
    const int rows = max(0, min(32, count - row0));
    constexpr int kOutCols = EPI == kLoraSwiGLU ? 16 : 32;  // outputs of a segment
    constexpr int kOutBytes = kOutCols * (EPI == kLoraF32 ? 4 : 2);
    const int n_out = EPI == kLoraSwiGLU ? p.N / 2 : p.N;
    // segment u: 32 columns of the step, two per warp
    auto load_base = [&](int c, float4 (&v)[8]) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = 4 * i + (lane >> 3), tok = r < rows ? s_tok[row0 + r] : -1;
        v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (tok >= 0 && c + 4 * (lane & 7) < p.N)
          v[i] = __ldcs(reinterpret_cast<const float4*>(p.base + tok * p.base_stride + c + 4 * (lane & 7)));
      }
    };
    float4 v0[8], v1[8];
    if (rows > 0) {
      load_base(column(0) + 64 * half, v0);
      load_base(column(0) + 64 * half + 32, v1);
    }
    for (int step = 0; step < steps; ++step) {
      const int buf = step & 1, c_step = column(step), j0 = first_slice(c_step), j1 = last_slice(c_step);
      if (!warp_wait(tfull + 8 * buf, (step >> 1) & 1, stop, p.err)) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      if (rows > 0) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int c = c_step + 64 * half + 32 * u;
          // the base, to the thread that has its row
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int r = 4 * i + (lane >> 3);
            const float4 v = u == 0 ? v0[i] : v1[i];
            st4(x + r * 128 + (((lane & 7) ^ (r & 7)) << 4), __float_as_uint(v.x), __float_as_uint(v.y),
                __float_as_uint(v.z), __float_as_uint(v.w));
          }
          uint32_t acc[32];
          const uint32_t d = tmem + buf * 256 + 64 * half + 32 * u + ((uint32_t)row0 << 16);
          if (rank_p > 0) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              tmem_ld8(d + 8 * k + (p.interleaved ? (k & 1) * kChunk : 0), acc + 8 * k);
            tmem_wait_ld();
            if (!p.interleaved && j1 > j0 && c < p.N && slice_of(p, min(c + 31, p.N - 1)) != j0) {
              uint32_t other[32];  // a slice ends in or before these columns
#pragma unroll
              for (int k = 0; k < 4; ++k) tmem_ld8(d + kChunk + 8 * k, other + 8 * k);
              tmem_wait_ld();
#pragma unroll
              for (int k = 0; k < 32; ++k)
                if (slice_of(p, c + k) != j0) acc[k] = other[k];
            }
          } else {
#pragma unroll
            for (int k = 0; k < 32; ++k) acc[k] = 0u;
          }
          __syncwarp();
          float y[32];
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const uint4 v = ld4(x + lane * 128 + ((k ^ (lane & 7)) << 4));
            y[4 * k] = __uint_as_float(v.x) + __uint_as_float(acc[4 * k]);
            y[4 * k + 1] = __uint_as_float(v.y) + __uint_as_float(acc[4 * k + 1]);
            y[4 * k + 2] = __uint_as_float(v.z) + __uint_as_float(acc[4 * k + 2]);
            y[4 * k + 3] = __uint_as_float(v.w) + __uint_as_float(acc[4 * k + 3]);
          }
          __syncwarp();
          // the results of the row, 16 bytes at a time
          constexpr int kChunks = kOutBytes / 16;
#pragma unroll
          for (int k = 0; k < kChunks; ++k) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if constexpr (EPI == kLoraF32) {
                w[e] = __float_as_uint(y[4 * k + e]);
              } else if constexpr (EPI == kLoraBf16) {
                w[e] = pack2(y[8 * k + 2 * e], y[8 * k + 2 * e + 1]);
              } else {  // 16 k: gate, 16 k + 8: up
                w[e] = pack2(silu(y[16 * k + 2 * e]) * y[16 * k + 8 + 2 * e],
                             silu(y[16 * k + 2 * e + 1]) * y[16 * k + 9 + 2 * e]);
              }
            }
            st4(x + lane * 128 + ((k ^ (lane & 7)) << 4), w[0], w[1], w[2], w[3]);
          }
          __syncwarp();
          const int c_out = EPI == kLoraSwiGLU ? c / 2 : c;
          constexpr int kPer = 16 / (EPI == kLoraF32 ? 4 : 2);
#pragma unroll
          for (int i = 0; i < kChunks; ++i) {
            const int at = 32 * i + lane, r = at / kChunks, k = at % kChunks;
            const int tok = r < rows ? s_tok[row0 + r] : -1;
            if (tok >= 0 && c_out + k * kPer < n_out) {
              const uint4 v = ld4(x + r * 128 + ((k ^ (r & 7)) << 4));
              const int64_t o = tok * p.out_stride + c_out + k * kPer;
              if constexpr (EPI == kLoraF32)
                *reinterpret_cast<uint4*>(static_cast<float*>(p.out) + o) = v;
              else
                *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p.out) + o) = v;
            }
          }
          __syncwarp();
          // this segment's base of the next step
          if (step + 1 < steps) {
            const int next = column(step + 1) + 64 * half + 32 * u;
            if (u == 0) load_base(next, v0); else load_base(next, v1);
          }
        }
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) bar_arrive(tempty + 8 * buf);
    }
  }
  __syncwarp();
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 3)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
}

template <int EPI>
int launch(const ExpandArgs& p, cudaStream_t s) {
  const Layout l = layout<EPI == kLoraF32 ? 3 : 2>(p.ns, p.rank_pm);
  if (l.stages == 0) return MS_ERR_UNSUPPORTED;
  static std::atomic<uint64_t> granted{0};
  MS_TRY(grant_dynamic_smem(lora_expand_tc_kernel<EPI>, kMostBytes, granted));
  // at least half the shared memory, so that no second CTA waits for TMEM on the SM
  const int bytes = l.bytes > 116 * 1024 ? l.bytes : 116 * 1024;
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

int lora_expand_tc(const ExpandArgs& p, int epilogue, cudaStream_t s) {
  if (p.rank_pm == 0) return MS_ERR_UNSUPPORTED;
  // no 128 columns with three slices
  for (int k = 0; !p.interleaved && k + 2 < p.ns; ++k)
    if (p.slice_end[k] / kChunk == (p.slice_end[k + 1] - 1) / kChunk &&
        p.slice_end[k + 1] % kChunk != 0 && p.slice_end[k] % kChunk != 0)
      return MS_ERR_UNSUPPORTED;
  if (epilogue == kLoraSwiGLU) return launch<kLoraSwiGLU>(p, s);
  return epilogue == kLoraF32 ? launch<kLoraF32>(p, s) : launch<kLoraBf16>(p, s);
}

}  // namespace ms
