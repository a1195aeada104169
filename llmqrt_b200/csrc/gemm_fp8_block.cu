// FP8 GEMM with a scale for each block of 128: activations a[M, K] with a scale for each token and 128 inputs, weights w[N, K] with
// one for each 128 outputs x 128 inputs,
//   out[m, n] = T( sum_g ( sum_{k in g} a[m, k] w[n, k] ) * (a_scale[m, g] * w_scale[n / 128, g]) + bias[n] ).
//
// A block of 128 inputs is one K block of the tensor cores (128 bytes, four MMAs), and its products have to be scaled before they are
// added up: the accumulator in tensor memory holds ONE K block's sums, and the epilogue warps take it over block by
// block, tcgen05.ld, one multiply-add an element into running sums in registers.  Accumulators rotate, so that the tensor cores
// work on the next block meanwhile.
//
//   TMA (SWIZZLE_128B) -> shared-memory ring -> tcgen05.mma -> tensor memory -> tcgen05.ld -> registers -> epilogue
//
// Two kernels:
//   block_pair_kernel   tokens are the 128-lane operand, the two CTAs of a cluster share a tile of 256 tokens x 256 (128) weight
//                       rows (cta_group::2).  A thread of the epilogue holds half of a token's row of it: its scale is one number
//                       a K block, a_scale of its token times w_scale of its columns.
//   block_split_kernel  few tokens: weights are the 128-lane operand (128 rows: one row of scales), the tokens the 16 .. 128
//                       columns, and the reduction is shared out to a cluster, whose CTAs add their sums up through
//                       distributed shared memory in rank order.
// Measured on the GPU: 64 x 37888 x 3584 28 us (its bytes alone 21.5), 1 x 4864 x 896 5.0 us; 4096 x 3584 x 18944 256 us in a
// burst and 293 under the board's 1000 W (1.9 PFLOP/s), where gemm_tc.cu's fp8 GEMM takes 239 and 266: every K block's sums pass
// through registers.
// All waits are bounded as in gemm_tc.cu.
#include "gemm_w8a8.cuh"
#include "tc_tiles.cuh"

#include <algorithm>

namespace llmqrt {
namespace {

constexpr int kBM = 128;
constexpr int kMaxCluster = 8;
constexpr int kMaxDevices = 64;
constexpr int kMaxPairs = 256;     // clusters of two CTAs that share tiles

struct BlockParams {
  const float* a_scale;            // [M, k_blocks]
  const float* w_scale;            // [ceil(N / 128), k_blocks]
  const void* bias;                // [N] or null
  void* out;                       // [M, ldo] 16-bit
  int64_t ldo;
  int bias_dtype, bf16;
  int M, N, k_blocks;
  int tiles_p, tiles_q, splits, early_w, tma_out;
  int whole_tiles, sharers;        // pair kernel: the tiles behind these are shared out by K blocks among so many clusters
  float* partials;                 // ... and what that needs of the workspace
  int* counters;
  uint32_t idesc;
  unsigned* status;
};

__device__ __forceinline__ uint32_t pack16(float a, float b, int bf16) {
  return bf16 ? pack_pair<__nv_bfloat16>(a, b) : pack_pair<__half>(a, b);
}
__device__ __forceinline__ F2 f2_of(uint32_t a, uint32_t b) { return f2(__uint_as_float(a), __uint_as_float(b)); }

// One arrival on an mbarrier of the cluster that says only that this warp's tcgen05.ld are back (tcgen05.wait::ld has seen to
// that).  Not a release: at cluster scope that waits for the warp's outstanding loads, here the next block's scales, 1400
// cycles a K block.
__device__ __forceinline__ void mbar_arrive_cluster_relaxed(uint32_t bar_cluster) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar_cluster) : "memory");
}

// A load that stays where it stands in the program, one K block ahead of its use.  (Left to the compiler it is waited for early: 322
// against 283 us for 4096 x 3584 x 18944.)
__device__ __forceinline__ void load_now(const float* p, float& v) { asm volatile("ld.global.nc.f32 %0, [%1];" : "=f"(v) : "l"(p)); }

// ---- few tokens --------------------------------------------------------------------------------------
// TMA warp, MMA warp, and four epilogue warps for each 32 tokens: with four for all of them they bound 128 tokens, 1370 cycles a
// K block whose weights come in 700 (37888 x 3584: 44.2 us, now 35 to 37).  Up to 64 tokens two CTAs share an SM, each with half the
// ring and tensor memory: one's start and end lie beside the other's tiles (64 tokens 28.8, then 27.5 us; 4608 x 3584, one token: 9.3 and
// 8.3).  What is left grows with the activations, which each tile of weight rows fetches from L2 again (one token: 24.1 us).
template <int BN> constexpr int split_groups() { return BN <= 32 ? 1 : BN / 32; }
template <int BN> constexpr int split_threads() { return 64 + 128 * split_groups<BN>(); }
template <int BN> constexpr int split_per_sm() { return BN <= 64 ? 2 : 1; }
constexpr int kSplitBufs = 4;                          // accumulators of BN columns
template <int BN> constexpr int split_stage_bytes() { return (kBM + BN) * kRowBytes; }
template <int BN> constexpr int split_stages() {
  const int s = 200 * 1024 / split_per_sm<BN>() / split_stage_bytes<BN>();      // (some shared memory is left for the small kernels ahead in a chain)
  return s > 10 ? 10 : s;
}
template <int BN> constexpr int split_smem() { return split_stages<BN>() * split_stage_bytes<BN>() + 1024; }
template <int BN> constexpr uint32_t split_tmem_cols() { return kSplitBufs * BN; }

__device__ __forceinline__ void ld_chunk(uint32_t taddr, uint32_t (&r)[32]) { tc::tmem_ld_32x32(taddr, r); }
__device__ __forceinline__ void ld_chunk(uint32_t taddr, uint32_t (&r)[16]) { tc::tmem_ld_32x16(taddr, r); }

template <int BN>
__global__ void __launch_bounds__(split_threads<BN>(), split_per_sm<BN>())
block_split_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_a, const BlockParams prm) {
  constexpr int kStages = split_stages<BN>(), kStageBytes = split_stage_bytes<BN>();
  constexpr int kCols = BN < 32 ? BN : 32;             // columns (tokens) of an epilogue warp
  constexpr int kGroups = split_groups<BN>(), kEpilogues = 4 * kGroups;
  static_assert(kStages * kStageBytes >= BN * kBM * 4, "the ring holds the partial sums");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* tiles = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ __align__(8) uint64_t bar_full[kStages];
  __shared__ __align__(8) uint64_t bar_empty[kStages];
  __shared__ __align__(8) uint64_t bar_acc_full[kSplitBufs];
  __shared__ __align__(8) uint64_t bar_acc_empty[kSplitBufs];
  __shared__ __align__(16) float scales[kEpilogues][2][kCols];           // each epilogue warp's own: the tokens' scales of a K block
  __shared__ uint32_t tmem_base_slot;
  __shared__ int abort_flag;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* abort = &abort_flag;
  const uint32_t abort_u32 = tc::smem_u32(&abort_flag);
  const int S = prm.splits, rank = S > 1 ? (int)cluster_ctarank() : 0;
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int s = 0; s < kStages; ++s) {
      tc::mbar_init(tc::smem_u32(&bar_full[s]), 1);
      tc::mbar_init(tc::smem_u32(&bar_empty[s]), 1);
    }
    for (int b = 0; b < kSplitBufs; ++b) {
      tc::mbar_init(tc::smem_u32(&bar_acc_full[b]), 1);
      tc::mbar_init(tc::smem_u32(&bar_acc_empty[b]), kEpilogues);
    }
    tc::mbar_fence_init();
    tc::tma_prefetch_descriptor(&tm_w);
    tc::tma_prefetch_descriptor(&tm_a);
  }
  if (warp == 1) {
    tc::tmem_alloc(tc::smem_u32(&tmem_base_slot), split_tmem_cols<BN>());
    tc::tmem_relinquish();
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem_base = tmem_base_slot;
  if (threadIdx.x != 0) {                              // (the producer's thread may first request weights)
    pdl_wait();
    pdl_trigger();
  }
  // S > 1: a cluster for each tile; otherwise a persistent walk.
  const int num_tiles = prm.tiles_p * prm.tiles_q;
  const int first_tile = (int)blockIdx.x / S, tile_step = S > 1 ? num_tiles : (int)gridDim.x;
  const int kb_begin = (int)((int64_t)rank * prm.k_blocks / S);
  const int kb_count = (int)((int64_t)(rank + 1) * prm.k_blocks / S) - kb_begin;

  F2 acc[kCols / 2];                                   // epilogue: row quad * 32 + lane of the tile, tokens from c_begin on
  const int quad = warp & 3, wrow = quad * 32 + lane, c_begin = (warp - 2) / 4 * kCols;
  const float* a_scale = prm.a_scale;

  if (warp == 0) {
    if (lane == 0) {
      int stage_i = 0;
      uint32_t phase = 0;
      bool ok = true;
      // weights of the first ring ahead of the wait for the preceding kernel, if they are a stored layer's
      const int pre = first_tile < num_tiles ? min(kStages, kb_count) : 0;
      const int tp0 = first_tile / prm.tiles_q, tq0 = first_tile % prm.tiles_q;
      if (!prm.early_w) {
        pdl_wait();
        pdl_trigger();
      }
      for (int i = 0; i < pre; ++i) {
        const uint32_t full = tc::smem_u32(&bar_full[i]);
        tc::mbar_arrive_expect_tx(full, kStageBytes);
        tc::tma_load_2d(tc::smem_u32(tiles + i * kStageBytes), &tm_w, full, (kb_begin + i) * kRowBytes, tp0 * kBM);
      }
      if (prm.early_w) {
        pdl_wait();
        pdl_trigger();
      }
      for (int i = 0; i < pre; ++i)
        tc::tma_load_2d(tc::smem_u32(tiles + i * kStageBytes + kBM * kRowBytes), &tm_a, tc::smem_u32(&bar_full[i]),
                        (kb_begin + i) * kRowBytes, tq0 * BN);
      stage_i = pre == kStages ? 0 : pre;
      if (pre == kStages) phase = 1;
      int done = pre;
      for (int tile = first_tile; tile < num_tiles && ok; tile += tile_step) {
        const int tp = tile / prm.tiles_q, tq = tile % prm.tiles_q;
        for (int it = done; it < kb_count; ++it) {
          tc::mbar_wait_or_flag(tc::smem_u32(&bar_empty[stage_i]), phase ^ 1u, abort_u32);
          const uint32_t full = tc::smem_u32(&bar_full[stage_i]);
          const uint32_t sp = tc::smem_u32(tiles + stage_i * kStageBytes);
          tc::mbar_arrive_expect_tx(full, kStageBytes);
          tc::tma_load_2d(sp, &tm_w, full, (kb_begin + it) * kRowBytes, tp * kBM);
          tc::tma_load_2d(sp + kBM * kRowBytes, &tm_a, full, (kb_begin + it) * kRowBytes, tq * BN);
          if (++stage_i == kStages) { stage_i = 0; phase ^= 1u; }
          if ((it & 3) == 3 && *abort) { ok = false; break; }
        }
        done = 0;
        if (*abort) ok = false;
      }
    }
  } else if (warp == 1) {
    int stage_i = 0, buf = 0;
    uint32_t phase = 0, acc_phase = 0;
    bool ok = true;
    for (int tile = first_tile; tile < num_tiles && ok; tile += tile_step) {
      for (int it = 0; it < kb_count; ++it) {
        if (!tc::mbar_wait_warp(tc::smem_u32(&bar_acc_empty[buf]), acc_phase ^ 1u, abort)) { ok = false; break; }
        tc::mbar_wait_or_flag(tc::smem_u32(&bar_full[stage_i]), phase, abort_u32);
        __syncwarp();
        tc::fence_after_sync();
        const uint32_t sp = tc::smem_u32(tiles + stage_i * kStageBytes), d = tmem_base + (uint32_t)(buf * BN);
        const uint64_t dw = tc::smem_desc_k_major_sw128(sp), da = tc::smem_desc_k_major_sw128(sp + kBM * kRowBytes);
        if (tc::elect_one()) {
#pragma unroll
          for (int j = 0; j < kRowBytes / 32; ++j)
            tc::mma_ss<tc::MMA_F8>(d, dw + (uint64_t)(2 * j), da + (uint64_t)(2 * j), prm.idesc, j > 0 ? 1u : 0u);
          tc::mma_commit(tc::smem_u32(&bar_empty[stage_i]));
          tc::mma_commit(tc::smem_u32(&bar_acc_full[buf]));
        }
        __syncwarp();
        if (++stage_i == kStages) { stage_i = 0; phase ^= 1u; }
        if (++buf == kSplitBufs) { buf = 0; acc_phase ^= 1u; }
      }
      if (tc::warp_aborted(abort)) ok = false;
    }
  } else {
    int buf = 0;
    uint32_t acc_phase = 0;
    bool ready = false;
    for (int tile = first_tile; tile < num_tiles; tile += tile_step) {
      const int tp = tile / prm.tiles_q, tq = tile % prm.tiles_q;
#pragma unroll
      for (int i = 0; i < kCols / 2; ++i) acc[i] = f2(0.f, 0.f);
      // (tokens behind the last one: any valid scale, their columns are not written)
      const float* ws = prm.w_scale + (int64_t)tp * prm.k_blocks + kb_begin;
      const float* as = a_scale + (int64_t)min(tq * BN + c_begin + lane, prm.M - 1) * prm.k_blocks + kb_begin;
      float next, w_next;
      load_now(ws, w_next);
      load_now(as, next);
#pragma unroll 1
      for (int it = 0; it < kb_count; ++it) {
        float* mine = scales[warp - 2][it & 1];
        if (kCols == 32 || lane < kCols) mine[lane] = __fmul_rn(next, w_next);
        const int ahead = min(it + 1, kb_count - 1);
        load_now(ws + ahead, w_next);
        load_now(as + ahead, next);
        if (!ready) tc::mbar_wait_or_flag(tc::smem_u32(&bar_acc_full[buf]), acc_phase, abort_u32);
        __syncwarp();
        tc::fence_after_sync();
        const uint32_t taddr = tmem_base + ((uint32_t)(quad * 32) << 16) + (uint32_t)(buf * BN + c_begin), empty = tc::smem_u32(&bar_acc_empty[buf]);
        if (++buf == kSplitBufs) { buf = 0; acc_phase ^= 1u; }
        uint32_t v[kCols];
        ld_chunk(taddr, v);
        // (whether the next block's accumulator is complete is asked for ahead: the answer takes 100 cycles, be it yes)
        ready = tc::mbar_test_wait(tc::smem_u32(&bar_acc_full[buf]), acc_phase);
        tc::tmem_ld_wait();
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(empty);
#pragma unroll
        for (int c = 0; c < kCols; c += 4) {
          const float4 s = *reinterpret_cast<const float4*>(mine + c);
          acc[c / 2] = f2_fma(f2_of(v[c], v[c + 1]), f2(s.x, s.y), acc[c / 2]);
          acc[c / 2 + 1] = f2_fma(f2_of(v[c + 2], v[c + 3]), f2(s.z, s.w), acc[c / 2 + 1]);
        }
      }
      if (tc::warp_aborted(abort)) break;
      if (S == 1) {                                    // straight from registers: a warp writes 32 neighbours of a token's row
        const int n = tp * kBM + wrow, m0 = tq * BN + c_begin, tokens = min(kCols, prm.M - m0);
        if (n < prm.N) {
          const float b = prm.bias ? load_as_f32(prm.bias, n, prm.bias_dtype) : 0.f;
#pragma unroll
          for (int i = 0; i < kCols; ++i) {
            float lo, hi;
            f2_split(acc[i / 2], lo, hi);
            if (i < tokens) store_from_f32(prm.out, (int64_t)(m0 + i) * prm.ldo + n, prm.bf16 ? LLMQRT_BF16 : LLMQRT_F16, (i & 1 ? hi : lo) + b);
          }
        }
      }
    }
  }

  if (S > 1) {
    // The ring is idle once every MMA of this CTA has been seen to finish: each CTA leaves its sums there, [token][row], and
    // takes its share of the tokens from all of them, in rank order.
    const int tp = first_tile / prm.tiles_q, tq = first_tile % prm.tiles_q, tokens = min(BN, prm.M - tq * BN);
    float* part = reinterpret_cast<float*>(tiles);
    __syncthreads();
    if (warp >= 2) {
#pragma unroll
      for (int i = 0; i < kCols; ++i) {
        float lo, hi;
        f2_split(acc[i / 2], lo, hi);
        if (c_begin + i < tokens) part[(c_begin + i) * kBM + wrow] = i & 1 ? hi : lo;
      }
    }
    cluster_sync_all();
    const int m1 = (rank + 1) * tokens / S, n = tp * kBM + lane * 4;   // a warp takes a token's 128 columns, four a lane
    if (warp >= 2 && n < prm.N) {
      float b[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) b[j] = prm.bias && n + j < prm.N ? load_as_f32(prm.bias, n + j, prm.bias_dtype) : 0.f;
      const bool wide = n + 4 <= prm.N && prm.ldo % 4 == 0 && (reinterpret_cast<uintptr_t>(prm.out) & 7) == 0;
      for (int m = rank * tokens / S + warp - 2; m < m1; m += kEpilogues) {
        const uint32_t local = tc::smem_u32(part + m * kBM + lane * 4);
        float4 v[kMaxCluster];
#pragma unroll
        for (int r = 0; r < kMaxCluster; ++r) {
          v[r] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (r < S)
            asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v[r].x), "=f"(v[r].y), "=f"(v[r].z), "=f"(v[r].w)
                         : "r"(tc::cluster_addr(local, (uint32_t)r)) : "memory");
        }
        float4 sum = v[0];
#pragma unroll
        for (int r = 1; r < kMaxCluster; ++r) {
          sum.x += v[r].x; sum.y += v[r].y; sum.z += v[r].z; sum.w += v[r].w;
        }
        const float o[4] = {sum.x + b[0], sum.y + b[1], sum.z + b[2], sum.w + b[3]};
        const int64_t at = (int64_t)(tq * BN + m) * prm.ldo + n;
        if (wide) {
          *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(prm.out) + at) = make_uint2(pack16(o[0], o[1], prm.bf16), pack16(o[2], o[3], prm.bf16));
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (n + j < prm.N) store_from_f32(prm.out, at + j, prm.bf16 ? LLMQRT_BF16 : LLMQRT_F16, o[j]);
        }
      }
    }
  }

  tc::fence_before_sync();
  __syncthreads();
  if (abort_flag) {                                    // a wait ran out: copies still in flight are given time to land
    const uint64_t t0 = tc::global_timer_ns();
    while (tc::global_timer_ns() - t0 < 100000ull) __nanosleep(1000);
  }
  if (S > 1) cluster_sync_all();                       // nobody leaves while a peer may read its sums
  if (warp == 1) {
    tc::fence_after_sync();
    tc::tmem_dealloc(tmem_base, split_tmem_cols<BN>());
  }
  if (threadIdx.x == 0 && abort_flag && prm.status) *prm.status = 1u;
}

// ---- many tokens -------------------------------------------------------------------------------------
// Accumulators are 128 columns wide, four of them, and take turns: a K block of 256 columns has two, each with an issuing warp and
// epilogue warps of its own, a K block of 128 one, every second block by the other issuer.  An issuer needs about 500 cycles for
// four MMAs and what goes with them -- to find a barrier complete takes 100, the MMAs and two commits 200 -- where the tensor
// cores need 512 for a K block of 256 columns; and an accumulator's round (MMAs, commit, the epilogue's loads, the remote
// arrival that frees it) is longer than either, so that the finer ones keep more going at a time.
//
// Work: tiles dealt out whole, in waves, and the tiles of a last wave that would be mostly empty as one long run of K blocks, of which
// clusters get equal shares, tiles' borders falling where they may.  A tile that several clusters
// have worked on is added up by the last of them to finish (counted off in the workspace, warp by warp, nobody waits), always
// in the clusters' order: the same bits every time.
constexpr int kPairThreads = 128 + 256;                // TMA warp, two MMA warps, one without work; eight epilogue warps
constexpr int kPairOutBytes = 32 * 128;                // staging tile of an epilogue warp
template <int BN> constexpr int pair_stage_bytes() { return (kBM + BN / 2) * kRowBytes; }
template <int BN> constexpr int pair_stages() { return BN == 256 ? 6 : 8; }
// An epilogue thread holds 128 running sums beside 64 columns on their way.  Three warps a scheduler are launched with 168 registers
// each, and the epilogue's two take some of what the other does not need.
// With 256 columns the epilogue wants every register it can have (40 + 2 * 232 = 3 * 168), with 128 it does not.
template <int BN> constexpr int epilogue_regs() { return BN == 256 ? 232 : 224; }
template <int BN> constexpr int other_regs() { return BN == 256 ? 40 : 56; }
constexpr int kIssuers = 2;
constexpr int kAccs = 4, kAccCols = 128;               // accumulators: all of tensor memory
template <int BN>
struct PairShared {
  uint8_t tiles[pair_stages<BN>() * pair_stage_bytes<BN>()];
  uint8_t out[8 * kPairOutBytes];
  uint64_t bar_full[pair_stages<BN>()];                // used in the leader only
  uint64_t bar_empty[pair_stages<BN>()];
  uint64_t bar_acc_full[kAccs];
  uint64_t bar_acc_empty[kAccs];                       // used in the leader only: an arrival for each epilogue warp that reads it, of both CTAs
  uint32_t tmem_base_slot;
  int abort_flag;
};

// A cluster's share of the work: whole tiles, then its part of the run of K blocks.  (A run has fewer than 2^31 K blocks.)
struct PairWork {
  int tile_next, u, u_end;
  __device__ PairWork(const BlockParams& p, int cluster) : tile_next(cluster), u(0), u_end(0) {
    if (cluster < p.sharers) {
      const int64_t run = (int64_t)(p.tiles_p * p.tiles_q - p.whole_tiles) * p.k_blocks;
      u = (int)(cluster * run / p.sharers);
      u_end = (int)((cluster + 1) * run / p.sharers);
    }
  }
  // The next tile and its K blocks [k0, k1).
  __device__ __forceinline__ bool next(const BlockParams& p, int& tile, int& k0, int& k1) {
    if (tile_next < p.whole_tiles) {
      tile = tile_next;
      tile_next += (int)(gridDim.x >> 1);
      k0 = 0;
      k1 = p.k_blocks;
      return true;
    }
    if (u >= u_end) return false;
    tile = u / p.k_blocks;
    k0 = u - tile * p.k_blocks;
    tile += p.whole_tiles;
    k1 = min(p.k_blocks, k0 + (u_end - u));
    u += k1 - k0;
    return true;
  }
};
// Which of `sharers` clusters of a run of `total` K blocks has block u in its share.
__device__ __forceinline__ int sharer_of(int64_t u, int64_t total, int sharers) { return (int)(((u + 1) * sharers - 1) / total); }

template <int BN>
__global__ void __launch_bounds__(kPairThreads, 1)
block_pair_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_w,
                  const __grid_constant__ CUtensorMap tm_out, const BlockParams prm) {
  extern __shared__ __align__(1024) uint8_t smem_pair[];
  constexpr int kStages = pair_stages<BN>(), kStageBytes = pair_stage_bytes<BN>();
  constexpr int kAccOf = BN / kAccCols, kRounds = kAccs / kAccOf;      // accumulators of a K block, K blocks' worth of them
  static_assert(kIssuers == 2 && kAccs % kIssuers == 0 && kStages % kIssuers == 0, "an issuer takes every second accumulator");
  constexpr int kCols = BN / 2, kLd = 32;              // columns of an epilogue warp, and of a load
  constexpr bool kAhead = BN == 256;
  PairShared<BN>& sh = *reinterpret_cast<PairShared<BN>*>(smem_pair);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* abort = &sh.abort_flag;
  const uint32_t abort_u32 = tc::smem_u32(&sh.abort_flag);
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  if (threadIdx.x == 0) {
    sh.abort_flag = 0;
    for (int s = 0; s < kStages; ++s) {
      tc::mbar_init(tc::smem_u32(&sh.bar_full[s]), 1);
      tc::mbar_init(tc::smem_u32(&sh.bar_empty[s]), kAccOf);
    }
    for (int b = 0; b < kAccs; ++b) {
      tc::mbar_init(tc::smem_u32(&sh.bar_acc_full[b]), 1);
      tc::mbar_init(tc::smem_u32(&sh.bar_acc_empty[b]), 16 / kAccOf);
    }
    tc::mbar_fence_init();
    tc::tma_prefetch_descriptor(&tm_a);
    tc::tma_prefetch_descriptor(&tm_w);
    tc::tma_prefetch_descriptor(&tm_out);
  }
  if (warp == 1) {
    tc::tmem_alloc_pair(tc::smem_u32(&sh.tmem_base_slot), 512);
    tc::tmem_relinquish_pair();
  }
  tc::fence_before_sync();
  __syncthreads();
  cluster_sync_all();                                  // both CTAs' barriers exist before anything signals them
  tc::fence_after_sync();
  const uint32_t tmem_base = sh.tmem_base_slot;
  pdl_wait();
  pdl_trigger();
  PairWork work(prm, (int)(blockIdx.x >> 1));               // (every role walks it for itself)
  int tile, k0, k1;

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(other_regs<BN>()));
    if (warp == 0) {
      if (lane == 0) {
        const uint32_t full0 = tc::cluster_addr(tc::smem_u32(&sh.bar_full[0]), 0u);
        int stage_i = 0;
        uint32_t phase = 0;
        bool ok = true;
        while (ok && work.next(prm, tile, k0, k1)) {
          int tp, tq;
          pair_tile_coords(tile, prm.tiles_p, prm.tiles_q, tp, tq);
          // of each accumulator's 128 weight rows a CTA brings 64
          const int row_a = tp * 2 * kBM + (int)rank * kBM, row_w = tq * BN + (int)rank * (kAccCols / 2);
          for (int it = k0; it < k1; ++it) {
            tc::mbar_wait_or_flag(tc::smem_u32(&sh.bar_empty[stage_i]), phase ^ 1u, abort_u32);
            if (leader) tc::mbar_arrive_expect_tx(tc::smem_u32(&sh.bar_full[stage_i]), 2u * kStageBytes);
            const uint32_t full = full0 + (uint32_t)stage_i * 8u;
            const uint32_t sp = tc::smem_u32(sh.tiles + stage_i * kStageBytes);
            tc::tma_load_2d_pair(sp, &tm_a, full, it * kRowBytes, row_a);
#pragma unroll
            for (int h = 0; h < kAccOf; ++h)
              tc::tma_load_2d_pair(sp + (kBM + h * (kAccCols / 2)) * kRowBytes, &tm_w, full, it * kRowBytes, row_w + h * kAccCols);
            if (++stage_i == kStages) { stage_i = 0; phase ^= 1u; }
          }
          if (*abort) ok = false;
        }
      }
    } else if (warp <= kIssuers) {
      if (leader) {
        // two accumulators a K block: this warp's is the w-th of every block; one: every second block's, from the w-th on
        constexpr int kStep = kAccOf == 2 ? 1 : kIssuers;
        const int w = warp - 1;
        int stage_i = kAccOf == 2 ? 0 : w, acc_i = w, skip = kAccOf == 2 ? 0 : w;       // skip: blocks of the segment ahead of this warp's first
        uint32_t phase = 0, acc_phase = 0;
        while (work.next(prm, tile, k0, k1)) {
          int left = k1 - k0 - skip;
          if (kStep == 2) skip = (skip + k1 - k0) & 1;
          for (; left > 0; left -= kStep) {
            tc::mbar_wait_or_flag(tc::smem_u32(&sh.bar_acc_empty[acc_i]), acc_phase ^ 1u, abort_u32);
            tc::mbar_wait_or_flag(tc::smem_u32(&sh.bar_full[stage_i]), phase, abort_u32);
            __syncwarp();
            tc::fence_after_sync();
            const uint32_t sp = tc::smem_u32(sh.tiles + stage_i * kStageBytes), d = tmem_base + (uint32_t)(acc_i * kAccCols);
            const uint64_t da = tc::smem_desc_k_major_sw128(sp);
            const uint64_t db = tc::smem_desc_k_major_sw128(sp + (kBM + (kAccOf == 2 ? w * (kAccCols / 2) : 0)) * kRowBytes);
            if (tc::elect_one()) {
#pragma unroll
              for (int j = 0; j < kRowBytes / 32; ++j)
                tc::mma_ss_pair<tc::MMA_F8>(d, da + (uint64_t)(2 * j), db + (uint64_t)(2 * j), prm.idesc, j > 0 ? 1u : 0u);
              tc::mma_commit_pair(tc::smem_u32(&sh.bar_acc_full[acc_i]));
              tc::mma_commit_pair(tc::smem_u32(&sh.bar_empty[stage_i]));
            }
            __syncwarp();
            if ((stage_i += kStep) >= kStages) { stage_i -= kStages; phase ^= 1u; }
            if ((acc_i += kIssuers) >= kAccs) { acc_i -= kAccs; acc_phase ^= 1u; }
          }
          if (tc::warp_aborted(abort)) break;
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(epilogue_regs<BN>()));
    // Two warps a lane quadrant, each taking half of the tile's columns: of one block of w_scale.
    const int quad = warp & 3, half = (warp - 4) >> 2;
    uint8_t* own = sh.out + (warp - 4) * kPairOutBytes;
    const uint32_t acc_empty0 = tc::cluster_addr(tc::smem_u32(&sh.bar_acc_empty[0]), 0u);
    const int acc_h = kAccOf == 2 ? half : 0;
    const uint32_t t_lane = tmem_base + ((uint32_t)(quad * 32) << 16) + (uint32_t)(half * kCols);
    int round = 0;
    uint32_t acc_phase = 0;
    while (work.next(prm, tile, k0, k1)) {
      int tp, tq;
      pair_tile_coords(tile, prm.tiles_p, prm.tiles_q, tp, tq);
      // Rows and columns behind the matrix take some valid scale: they are not written.
      const float* as = prm.a_scale + (int64_t)min(tp * 2 * kBM + (int)rank * kBM + quad * 32 + lane, prm.M - 1) * prm.k_blocks;
      const float* ws = prm.w_scale + (int64_t)min((tq * BN + half * kCols) / 128, (prm.N - 1) / 128) * prm.k_blocks;
      float a_next, w_next;
      load_now(as + k0, a_next);
      load_now(ws + k0, w_next);
      F2 acc[kCols / 2];
#pragma unroll
      for (int i = 0; i < kCols / 2; ++i) acc[i] = f2(0.f, 0.f);
      // 32 columns are multiplied while the next ones come; after a block's last ones its accumulator is free.  The wait for the next
      // block's takes 100 cycles even where it is complete.  With 256 columns it stands ahead of the last products, together
      // with the next first columns (behind them: 316 against 267 us without the scales); with 128, whether it is complete is
      // asked for ahead of the last columns (1000 x 4608 x 3584 21.8 us, like the other 23.3; with 256 it costs registers: 627
      // against 504 us for 4096 x 37888 x 3584).
      uint32_t r[2][kLd];
      bool ready = false;
      auto await = [&]() {
        if (!ready) tc::mbar_wait_or_flag(tc::smem_u32(&sh.bar_acc_full[round * kAccOf + acc_h]), acc_phase, abort_u32);
        __syncwarp();
        tc::fence_after_sync();
      };
      if (kAhead) {
        await();
        tc::tmem_ld_32x32(t_lane + (uint32_t)(round * BN), r[0]);
      }
#pragma unroll 1
      for (int kb = k0; kb < k1; ++kb) {
        if (!kAhead) await();
        const uint32_t taddr = t_lane + (uint32_t)(round * BN), empty = acc_empty0 + (uint32_t)(round * kAccOf + acc_h) * 8u;
        if (!kAhead) tc::tmem_ld_32x32(taddr, r[0]);
        const float s = __fmul_rn(a_next, w_next);
        const F2 ss = f2(s, s);
        load_now(as + min(kb + 1, k1 - 1), a_next);
        load_now(ws + min(kb + 1, k1 - 1), w_next);
        if (++round == kRounds) { round = 0; acc_phase ^= 1u; }
#pragma unroll
        for (int k = 0; k < kCols / kLd; ++k) {
          if (!kAhead && k + 1 == kCols / kLd) ready = tc::mbar_test_wait(tc::smem_u32(&sh.bar_acc_full[round * kAccOf + acc_h]), acc_phase);
          tc::tmem_ld_wait();
          if (k + 1 < kCols / kLd) {
            tc::tmem_ld_32x32(taddr + (uint32_t)(kLd * k + kLd), r[(k + 1) & 1]);
          } else {
            tc::fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster_relaxed(empty);
            if (kAhead && kb + 1 < k1) {
              await();
              tc::tmem_ld_32x32(t_lane + (uint32_t)(round * BN), r[0]);
            }
          }
#pragma unroll
          for (int c = 0; c < kLd; c += 2) acc[(kLd * k + c) / 2] = f2_fma(f2_of(r[k & 1][c], r[k & 1][c + 1]), ss, acc[(kLd * k + c) / 2]);
        }
      }
      // The clusters that share a tile are counted off warp by warp; the last of them finds the counter full, and sets it to zero.
      auto counted_off = [&](int c_first, int c_last) {
        __syncwarp();
        int before = 0;
        int* counter = prm.counters + ((tile - prm.whole_tiles) * 2 + (int)rank) * 8 + warp - 4;
        if (lane == 0) {
          before = atomicAdd(counter, 1);
          if (before == c_last - c_first) *counter = 0;
        }
        return __shfl_sync(0xffffffffu, before, 0) == c_last - c_first;
      };
      auto shared_by = [&](int& c_first, int& c_last) {
        const int64_t total = (int64_t)(prm.tiles_p * prm.tiles_q - prm.whole_tiles) * prm.k_blocks, u0 = (int64_t)(tile - prm.whole_tiles) * prm.k_blocks;
        c_first = sharer_of(u0, total, prm.sharers);
        c_last = sharer_of(u0 + prm.k_blocks - 1, total, prm.sharers);
        return total;
      };
      if (tc::warp_aborted(abort)) {
        // A wait has run out: the results are void, but the warp counts itself off all the same, here and for what is left of its share, so
        // that the next call finds the counters at zero.
        do {
          if (k1 - k0 < prm.k_blocks) {
            int c_first, c_last;
            shared_by(c_first, c_last);
            counted_off(c_first, c_last);
          }
        } while (work.next(prm, tile, k0, k1));
        break;
      }
      pair_tile_coords(tile, prm.tiles_p, prm.tiles_q, tp, tq);
      const int row0 = tp * 2 * kBM + (int)rank * kBM + quad * 32, x0 = tq * BN + half * kCols;
      if (k1 - k0 < prm.k_blocks) {
        // a tile of several clusters: this one's sums to the workspace, four columns of a row a store
        const int shared = tile - prm.whole_tiles;
        int c_first, c_last;
        const int64_t total = shared_by(c_first, c_last);
        const int64_t mine = (int64_t)((int)rank * 8 + warp - 4) * (kCols * 32);
        auto slot_of = [&](int c) {                    // a cluster has two slots: for the tile that its share begins with, and the last one
          const int begins = (int)(c * total / prm.sharers / prm.k_blocks);
          return prm.partials + (int64_t)(2 * c + (shared == begins ? 0 : 1)) * (2 * kBM * BN) + mine + lane * 4;
        };
        float* dst = slot_of((int)(blockIdx.x >> 1));
#pragma unroll
        for (int i = 0; i < kCols / 4; ++i) {
          float4 v;
          f2_split(acc[2 * i], v.x, v.y);
          f2_split(acc[2 * i + 1], v.z, v.w);
          __stcg(reinterpret_cast<float4*>(dst + i * 128), v);
        }
        __threadfence();
        if (!counted_off(c_first, c_last)) continue;   // another cluster will finish the tile
        __threadfence();
#pragma unroll
        for (int i = 0; i < kCols / 2; ++i) acc[i] = f2(0.f, 0.f);
        for (int c = c_first; c <= c_last; ++c) {
          const float* src = slot_of(c);
#pragma unroll
          for (int i = 0; i < kCols / 4; ++i) {
            const float4 v = __ldcg(reinterpret_cast<const float4*>(src + i * 128));
            acc[2 * i] = f2_add(acc[2 * i], f2(v.x, v.y));
            acc[2 * i + 1] = f2_add(acc[2 * i + 1], f2(v.z, v.w));
          }
        }
      }
      // 64 columns at a time through the warp's staging tile, 16-byte unit u of row r at u ^ (r & 7)
#pragma unroll
      for (int c0 = 0; c0 < kCols; c0 += 64) {
        const int cols = prm.N - x0 - c0;              // columns left of the matrix (may be <= 0)
        if (prm.tma_out && lane == 0) tma_stores_read();
        __syncwarp();
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          uint32_t v[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float lo, hi;
            f2_split(acc[(c0 + 8 * k) / 2 + e], lo, hi);
            if (prm.bias) {
              const int n = x0 + c0 + 8 * k + 2 * e;
              if (n < prm.N) lo += load_as_f32(prm.bias, n, prm.bias_dtype);
              if (n + 1 < prm.N) hi += load_as_f32(prm.bias, n + 1, prm.bias_dtype);
            }
            v[e] = pack16(lo, hi, prm.bf16);
          }
          *reinterpret_cast<uint4*>(own + lane * 128 + ((k ^ (lane & 7)) << 4)) = make_uint4(v[0], v[1], v[2], v[3]);
        }
        if (prm.tma_out) {
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0 && row0 < prm.M && cols > 0) tma_store_2d(&tm_out, tc::smem_u32(own), x0 + c0, row0);
        } else {                                       // rows of the output that do not begin on 16 bytes
          __syncwarp();
          for (int q = 0; q < min(32, prm.M - row0); ++q) {
            uint16_t* dst = reinterpret_cast<uint16_t*>(prm.out) + (int64_t)(row0 + q) * prm.ldo + x0 + c0;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int c = h * 32 + lane;
              if (c < cols) dst[c] = *reinterpret_cast<const uint16_t*>(own + q * 128 + (((c >> 3) ^ (q & 7)) << 4) + (c & 7) * 2);
            }
          }
          __syncwarp();
        }
      }
    }
    if (prm.tma_out && lane == 0) tma_stores_done();
  }

  tc::fence_before_sync();
  __syncthreads();
  if (sh.abort_flag) {
    const uint64_t t0 = tc::global_timer_ns();
    while (tc::global_timer_ns() - t0 < 100000ull) __nanosleep(1000);
  }
  cluster_sync_all();                                  // nobody leaves while its peer may still signal it
  if (warp == 1) {
    tc::fence_after_sync();
    tc::tmem_dealloc_pair(tmem_base, 512);
  }
  if (threadIdx.x == 0 && sh.abort_flag && prm.status) *prm.status = 1u;
}

// ---- host side ---------------------------------------------------------------------------------------

template <typename Kern>
cudaLaunchConfig_t config(Kern, int grid, int cluster, int threads, int smem, cudaStream_t st, cudaLaunchAttribute* attr) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid, 1, 1);
  cfg.blockDim = dim3((unsigned)threads, 1, 1);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = st;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (pdl_enabled()) {
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = 2;
  }
  return cfg;
}
// How many clusters of 1 .. kMaxCluster CTAs of a kernel can be resident at once (asked once per device and kernel).
template <typename Kern>
void ask_clusters(Kern kern, int threads, int smem, int lo, int hi, int* known) {
  if (ensure_dynamic_smem(reinterpret_cast<const void*>(kern), smem) != LLMQRT_OK) return;
  for (int c = lo; c <= hi; ++c) {
    cudaLaunchAttribute attr[2];
    cudaLaunchConfig_t cfg = config(kern, c, c, threads, smem, nullptr, attr);
    if (cudaOccupancyMaxActiveClusters(&known[c], kern, &cfg) != cudaSuccess) {
      cudaGetLastError();
      known[c] = 0;
    }
  }
}
template <int BN> const int* split_clusters() {
  static std::once_flag once[kMaxDevices];
  static int known[kMaxDevices][kMaxCluster + 1];
  static const int none[kMaxCluster + 1] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev >= kMaxDevices) return none;
  std::call_once(once[dev], [dev] { ask_clusters(block_split_kernel<BN>, split_threads<BN>(), split_smem<BN>(), 1, kMaxCluster, known[dev]); });
  return known[dev];
}
template <int BN> int pair_clusters() {
  static std::once_flag once[kMaxDevices];
  static int known[kMaxDevices][3];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev >= kMaxDevices) return 0;
  std::call_once(once[dev], [dev] { ask_clusters(block_pair_kernel<BN>, kPairThreads, (int)sizeof(PairShared<BN>), 2, 2, known[dev]); });
  return known[dev][2];
}

// The cluster that shares a reduction: rounds of co-resident clusters x (K blocks of a CTA + what a CTA costs beside them).  `active`:
// clusters at once with one CTA an SM (all that the runtime answers for kernels with tensor memory).  Where `shared`, twice as many do,
// at the price of the bandwidth they share and of their start: fitted to 15 layers, one to 64 tokens.  3584 x 18944, one token: eight CTAs
// a tile 14.8 us, four (one an SM) 17.0; 17920 x 1536: two 9.3, one 8.4; with 64 tokens a second CTA gains nothing.
int pick_splits(int64_t tiles, int k_blocks, const int* active, bool shared, int* waves) {
  const double fixed = 8., fixed_shared = 12., sms = sm_count();
  int splits = 1;
  *waves = (int)ceil_div(tiles, (int64_t)sms);
  double best = *waves * (k_blocks + fixed);
  for (int s = 2; s <= kMaxCluster && k_blocks >= s && tiles < sms; ++s) {
    if (active[s] <= 0) continue;
    int w = (int)ceil_div(tiles, (int64_t)active[s]);
    double t = w * ((double)k_blocks / s + fixed);
    if (shared && w == 2) {
      const double both = k_blocks * std::max(1. / s, tiles / sms) + fixed_shared;
      if (both < t) { t = both; w = 1; }
    }
    if (t <= best) { best = t; splits = s; *waves = w; }
  }
  return splits;
}

// How the pair kernel's tiles of 256 x BN are dealt out: `whole` of them one by one, the rest by K blocks among `sharers` clusters,
// and the estimated microseconds.  A tile has at most three shares.  Fitted to 200 sizes, M = 130 .. 2048, N = 300 .. 8960, K = 2048 ..
// 18944, with and without sharing: a K block takes 0.34 - 0.43 us (256 columns) or 0.23 - 0.27 (128), by how many clusters are at
// work; the sums through the workspace, and shares that begin anywhere in K and so find less of the operands in L2, cost
// 10 - 17 or 3 - 9.  256 x 300 x 18944: 29.7 us shared, 48.8 not; 2048 x 3584 x 18944 135 and 143; 333 x 3584 x 8960 28 and 23.
struct Deal {
  int64_t tiles, whole;
  int sharers;
  double us;
};
template <int BN> Deal deal_out(int64_t M, int64_t N, int64_t kb, bool workspace) {
  const int64_t clusters = sm_count() / 2, tiles = ceil_div(M, 2 * kBM) * ceil_div(N, BN), rest = tiles % clusters, waves = tiles / clusters;
  const double fill = std::min(1., (double)tiles / clusters);
  const double block = BN == 256 ? 0.335 + 0.09 * fill : 0.225 + 0.04 * fill;
  Deal d{tiles, tiles, 0, (BN == 256 ? 6.8 : 5.1) + (waves + (rest ? 1 : 0)) * (kb * block + 0.8)};
  if (!workspace || !rest || clusters > kMaxPairs || rest * 16 > LLMQRT_WS_NUM_COUNTERS || rest * kb > 0x7fffffffll) return d;
  const int64_t sharers = rest * 3 <= clusters ? rest * 3 : rest * 2 <= clusters ? rest * 2 : clusters;
  const int64_t share = ceil_div(rest * kb, sharers);
  const double saved = (kb - share) * block - (BN == 256 ? 10. + 0.1 * sharers : 2.5 + 0.08 * sharers);
  if (saved > 0. && share >= 4) d = Deal{tiles, tiles - rest, (int)sharers, d.us - saved};
  return d;
}

struct Operands {
  const void* a;
  const void* w;
  int64_t lda, ldw, K;
};

template <int BN>
int launch_split(const Operands& o, BlockParams prm, cudaStream_t st) {
  prm.tiles_p = (int)ceil_div(prm.N, kBM);
  prm.tiles_q = (int)ceil_div(prm.M, BN);
  prm.idesc = tc::instr_desc(1, 0, 0, kBM, BN);
  const int64_t tiles = (int64_t)prm.tiles_p * prm.tiles_q;
  LLMQRT_REQUIRE(tiles <= 0x7fffffffll / kMaxCluster, "fp8 block linear: too many tiles");
  int waves;
  prm.splits = pick_splits(tiles, prm.k_blocks, split_clusters<BN>(), BN <= 32, &waves);
  CUtensorMap tm_w, tm_a;
  if (int rc = make_operand_map(&tm_w, o.w, 1, prm.N, o.K, o.ldw, kBM)) return rc;
  if (int rc = make_operand_map(&tm_a, o.a, 1, prm.M, o.K, o.lda, BN)) return rc;
  auto kern = block_split_kernel<BN>;
  if (int rc = ensure_dynamic_smem(reinterpret_cast<const void*>(kern), split_smem<BN>())) return rc;
  const int64_t grid = prm.splits > 1 ? tiles * prm.splits : std::min(tiles, (int64_t)sm_count() * split_per_sm<BN>());
  cudaLaunchAttribute attr[2];
  cudaLaunchConfig_t cfg = config(kern, (int)grid, prm.splits, split_threads<BN>(), split_smem<BN>(), st, attr);
  LLMQRT_CUDA_OK(cudaLaunchKernelEx(&cfg, kern, tm_w, tm_a, prm));
  return check_launch("fp8 block linear");
}

template <int BN>
int launch_pair(const Operands& o, BlockParams prm, Deal deal, cudaStream_t st) {
  const int clusters = pair_clusters<BN>();
  if (clusters <= 0) return set_error(LLMQRT_ERR_CUDA, "fp8 block linear: no cluster of two CTAs fits on this device");
  prm.tiles_p = (int)ceil_div(prm.M, 2 * kBM);
  prm.tiles_q = (int)ceil_div(prm.N, BN);
  prm.idesc = tc::instr_desc(1, 0, 0, 2 * kBM, kAccCols);
  LLMQRT_REQUIRE(deal.tiles <= 0x7fffffffll, "fp8 block linear: too many tiles");
  if (deal.sharers > clusters) deal = Deal{deal.tiles, deal.tiles, 0, 0.};      // (a device that does not hold a cluster on every two SMs)
  prm.whole_tiles = (int)deal.whole;
  prm.sharers = deal.sharers;
  const int grid = (int)std::max((int64_t)deal.sharers, std::min(deal.whole, (int64_t)clusters));
  prm.tma_out = (reinterpret_cast<uintptr_t>(prm.out) & 15) == 0 && prm.ldo % 8 == 0;
  CUtensorMap tm_a, tm_w, tm_out;
  if (int rc = make_operand_map(&tm_a, o.a, 1, prm.M, o.K, o.lda, kBM)) return rc;
  if (int rc = make_operand_map(&tm_w, o.w, 1, prm.N, o.K, o.ldw, kAccCols / 2)) return rc;
  if (!prm.tma_out) tm_out = tm_a;                     // (not used)
  else if (int rc = make_output_map(&tm_out, prm.out, 2, prm.M, prm.N, prm.ldo)) return rc;
  static_assert(2 * kMaxPairs * sizeof(float) * 2 * kBM * BN <= LLMQRT_WS_PARTIAL_BYTES, "two partial tiles for each cluster");
  auto kern = block_pair_kernel<BN>;
  if (int rc = ensure_dynamic_smem(reinterpret_cast<const void*>(kern), (int)sizeof(PairShared<BN>))) return rc;
  cudaLaunchAttribute attr[2];
  cudaLaunchConfig_t cfg = config(kern, 2 * grid, 2, kPairThreads, (int)sizeof(PairShared<BN>), st, attr);
  LLMQRT_CUDA_OK(cudaLaunchKernelEx(&cfg, kern, tm_a, tm_w, tm_out, prm));
  return check_launch("fp8 block linear");
}

}  // namespace
}  // namespace llmqrt

using namespace llmqrt;

extern "C" int llmqrt_fp8_linear_block(const uint8_t* a, int64_t lda, const uint8_t* w, int64_t ldw, const void* bias, int bias_dtype,
                                       const float* a_scale, const float* w_scale, void* out, int out_dtype, int64_t ldo, int64_t M,
                                       int64_t N, int64_t K, void* workspace, llmqrt_stream_t stream, int flags) {
  LLMQRT_REQUIRE(M >= 0 && N > 0 && K > 0 && M < (1ll << 31) && N < (1ll << 31) && K < (1ll << 31),
                 "fp8 block linear: bad shape M=%lld N=%lld K=%lld", (long long)M, (long long)N, (long long)K);
  LLMQRT_REQUIRE(K % 16 == 0 && lda >= K && ldw >= K && lda % 16 == 0 && ldw % 16 == 0,
                 "fp8 block linear: K=%lld and leading dimensions must be multiples of 16, lda=%lld / ldw=%lld at least K", (long long)K,
                 (long long)lda, (long long)ldw);
  LLMQRT_REQUIRE(ldo >= N, "fp8 block linear: ldo=%lld < N", (long long)ldo);
  LLMQRT_REQUIRE(out_dtype == LLMQRT_F16 || out_dtype == LLMQRT_BF16, "fp8 block linear: out must be fp16 or bf16");
  LLMQRT_REQUIRE(!bias || bias_dtype == LLMQRT_F16 || bias_dtype == LLMQRT_BF16 || bias_dtype == LLMQRT_F32, "fp8 block linear: bad bias dtype");
  LLMQRT_REQUIRE((flags & ~LLMQRT_GEMM_STATIC_WEIGHT) == 0, "fp8 block linear: unknown flags 0x%x", flags);
  if (M == 0) return LLMQRT_OK;
  LLMQRT_REQUIRE(a && w && a_scale && w_scale && out, "fp8 block linear: null pointer");
  LLMQRT_REQUIRE(((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(w)) & 15) == 0, "fp8 block linear: operands must be 16-byte aligned");
  BlockParams p{};
  p.a_scale = a_scale; p.w_scale = w_scale; p.bias = bias; p.bias_dtype = bias_dtype; p.out = out; p.ldo = ldo;
  p.bf16 = out_dtype == LLMQRT_BF16; p.M = (int)M; p.N = (int)N; p.k_blocks = (int)ceil_div(K, kRowBytes);
  p.early_w = flags & LLMQRT_GEMM_STATIC_WEIGHT ? 1 : 0;
  if (workspace) {
    p.status = ws_scalars(workspace) + 1;
    p.partials = reinterpret_cast<float*>(ws_partials(workspace));
    p.counters = ws_counters(workspace);
  }
  const Operands o{a, w, lda, ldw, K};
  cudaStream_t st = (cudaStream_t)stream;
  if (M <= 16) return launch_split<16>(o, p, st);
  if (M <= 32) return launch_split<32>(o, p, st);
  if (M <= 64) return launch_split<64>(o, p, st);
  if (M <= 128) return launch_split<128>(o, p, st);
  const Deal wide = deal_out<256>(M, N, p.k_blocks, workspace != nullptr), narrow = deal_out<128>(M, N, p.k_blocks, workspace != nullptr);
  const double pair = std::min(wide.us, narrow.us);
  // Few tiles and a long reduction: panels of 64 tokens with it shared out, where the last panel is not nearly empty (a box that lies
  // mostly behind the tokens comes slowly).  130 x 300 x 3584 7.7 us, in pairs 12.1; 512 x 1536 x 3584 15.8 and 11.6.
  if (M <= 512 && (M - 1) % 64 >= 15) {
    int waves;
    const int s = pick_splits(ceil_div(N, kBM) * ceil_div(M, 64), p.k_blocks, split_clusters<64>(), false, &waves);
    if (s > 1 && 6. + waves * (0.45 * p.k_blocks / s + 2.5) < pair) return launch_split<64>(o, p, st);
  }
  return wide.us < narrow.us ? launch_pair<256>(o, p, wide, st) : launch_pair<128>(o, p, narrow, st);
}
