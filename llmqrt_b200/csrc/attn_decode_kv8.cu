// Attention of the newest tokens of each sequence over a paged cache of 8-bit keys and values with a scale for each page and
// head (kv8.cuh), split over the keys.
//
//   S = (q . code_k) * k_scale[page] / sqrt(d)      O = sum_j softmax(S)_j * code_v * v_scale[page]
//
// HBM-bound: each code is read once, half the bytes of a 16-bit cache, so that what a key costs the schedulers counts:
// at 6.5 TB/s an SM takes a key and value row of 128 every 11 cycles.  Warps stream 16 keys a step through rings of their own in
// shared memory (cp.async, 16 keys always lie in one page), turn the codes into fp16, where both kinds are exact, and multiply
// with warp-level MMAs: keys (or columns of V) are the sixteen rows, the query heads that share the KV head the eight columns.
//   S^T = K Q^T     : a lane's K fragment is 16 contiguous bytes of two keys' rows; Q is loaded with the same permutation of d.
//   O^T += V^T P^T  : the fragment wants two keys a register: bytes of two rows are interleaved before they are converted.
// (With the query rows as the sixteen, half of them idle, it took twice the MMAs and accumulators, and 64 us where this took 58.)
// Scales stay out of the products: k_scale multiplies S; v_scale, over the greatest one of the pages so far (a second running
// reference beside the softmax's maximum), multiplies P.  A page whose scale is far from the reference (2^8 below it, or above 2^50,
// where the reference ends) has products of its own, which are scaled in fp32 as they join O, so that no scale, an infinity included, takes
// bits from the other pages or touches rows that do not see the page.  Q in fp16 is exact for fp16 and, its row multiplied by a power of two, for
// bf16.  For an fp16 result what the rounding of Q (rotated here) and of P to fp16 left over takes MMAs of its own, so that the
// result is off by its own rounding alone; bf16's own rounding is eight times as large.
//
// Grid.  Few short sequences: clusters of up to eight blocks, which have a sequence's keys between them and merge their parts through
// each other's shared memory.  Otherwise (blocks, Hkv * row tiles): as many blocks as fit at once, each with an equal piece of all
// sequences' keys laid end to end, whatever their lengths; sequences that several blocks have had a part of are merged from
// the workspace by a second kernel.  (Pieces of one length for all sequences: 64 ragged sequences took 60 to 71 us, now 48.)
// Page numbers outside the cache and rows behind the last key are not read (zeros take their place) and get no weight.
//
// Measured, HBM at 6.5 TB/s: 64 sequences of 750 .. 6000 keys, 28 heads on 4 of 128, 48 us (4.7 TB/s: beginning a sequence costs a
// block 4 us, the last blocks end 8 us behind the median, the merge takes 5); one sequence of 131072 keys and two tokens 32.5 us
// (4.1 TB/s; 20 us of it at 6.7, the merge 6); 32 sequences of up to 30000 keys and 8 KV heads 185 us (6.1 TB/s).  Five sequences of up to
// 300 keys 5.0 us.
#include <algorithm>
#include <map>
#include <mutex>
#include <utility>

#include "kv8.cuh"

namespace llmqrt {
namespace {

constexpr int kWarps = 4, kThreads = kWarps * 32, kStep = 16 * kWarps;
// Blocks an SM, and stages of a warp, 16 keys each.  (64 sequences, 8 query heads of 128: four blocks 48.4 us and spills, three 47.4, two
// with a longer ring 46.7 but 50 in fp16; one long sequence, 16 rows: three 33.2, two 32.)
template <int D, int ROWS> constexpr int kv8_per_sm() { return ROWS == 8 ? (D == 128 ? 3 : 4) : D == 128 ? 2 : 3; }
template <int D, int ROWS> constexpr int kv8_ring() { return D == 128 && ROWS == 8 ? 3 : 4; }
constexpr int kSpan = 4096;                            // keys whose page numbers and scales a block holds at a time
constexpr int kSwitch = 6;                             // what another sequence costs a block, in units of kStep keys (4: 54, 6 to 10: 51.6, 16: 52.5 us)
constexpr int kMaxBlocks = 1024;                       // that one KV head's keys are shared out to
constexpr int kMaxPages = kSpan / 16 + 1;              // pages that these touch
constexpr int kClusterMergeMaxLen = 8192;              // greatest bound on the lengths for which a sequence gets one cluster
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kHead = 0x1p24f;                       // parts of O are kept so much smaller: sums of values near fp32's end do not pass it

struct Kv8Args {
  const uint16_t* q;               // [B, Sq, Hq, D]
  int64_t q_batch_stride, q_token_stride;
  const uint8_t* k_cache;          // [pages, Hkv, page, D]
  const uint8_t* v_cache;
  int64_t page_stride, head_stride;
  const float* k_scale;            // [pages, Hkv]
  const float* v_scale;
  const int32_t* table;            // [B, width] with row stride table_stride
  int64_t table_stride;
  const int32_t* seqlens;          // [B], the newest tokens counted
  const float* cos_tab;            // [table_rows, D / 2] or null
  const float* sin_tab;
  uint16_t* out;                   // [B, Sq, Hq, D]
  float* part_o;                   // [Hkv * tiles, blocks, 2, ROWS, D]
  float* part_ml;                  // [Hkv * tiles, blocks, 2, ROWS, 2]
  int table_rows, B, Sq, Hq, Hkv, pages, page, max_len, tiles, cluster;
  float scale, softcap;
};

template <int OFF> __device__ __forceinline__ void cp_async_16(uint32_t dst_smem, const uint8_t* src) {
  asm volatile("cp.async.cg.shared.global [%0 + %2], [%1 + %2], 16;" ::"r"(dst_smem), "l"(src), "n"(OFF) : "memory");
}
template <int OFF> __device__ __forceinline__ void cp_async_16_or_zero(uint32_t dst_smem, const uint8_t* src, bool take) {
  asm volatile("cp.async.cg.shared.global [%0 + %3], [%1 + %3], 16, %2;" ::"r"(dst_smem), "l"(src), "r"(take ? 16 : 0), "n"(OFF) : "memory");
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint4 lds_16(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint2 lds_8(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
  return v;
}
// An 8 x 8 matrix of 16-bit values, row lane / 4, columns 2 (lane % 4) and + 1, turned over.
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t pack_half(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack_half(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
template <bool BF16> __device__ __forceinline__ uint32_t round_pair(float a, float b) {
  return BF16 ? pack_pair<__nv_bfloat16>(a, b) : pack_pair<__half>(a, b);
}
template <bool BF16> __device__ __forceinline__ uint16_t round_bits(float f) {
  if constexpr (BF16) return __bfloat16_as_ushort(__float2bfloat16_rn(f));
  else return __half_as_ushort(__float2half_rn(f));
}

// Units of kStep keys of a sequence; one without keys counts as one (its rows of zeros are written).
__device__ __forceinline__ int units_of(const Kv8Args& p, int b) { return max(1, (max(0, min(p.seqlens[b], p.max_len)) + kStep - 1) / kStep); }

// Where share k of the line begins, and the share that a place lies in (64-bit divisions take 100 instructions).
__device__ __forceinline__ int64_t share_begin(int k, int64_t total, int shares) {
  if (total < (1 << 21)) return (int64_t)((uint32_t)k * (uint32_t)total / (uint32_t)shares);      // k <= 1024
  return k * total / shares;
}
__device__ __forceinline__ int share_of(int64_t place, int64_t total, int shares) {
  if (total < (1 << 21)) return (int)((((uint32_t)place + 1) * (uint32_t)shares - 1) / (uint32_t)total);
  return (int)(((place + 1) * shares - 1) / total);
}

// Sequences lie on a line one after the other, each kSwitch places for the work that it costs to begin one and then its units; shares
// are pieces of the line.  Finds the block's piece and where it begins.  (In shared memory: the loop over the keys has no registers
// to spare for what is wanted after it.)
struct Share {
  int64_t total;                                       // the line's length
  int64_t at, end;                                     // what is left of the piece
  int64_t before;                                      // the length of the sequences before b
  int shares, b;
  int unit, unit_end, n_units;                         // what the block has of b, and how many there are
};
__device__ __forceinline__ void find_share(const Kv8Args& p, Share& share) {
  __shared__ int64_t scan[2][kWarps];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  auto weight = [&](int b) -> int64_t { return b < p.B ? units_of(p, b) + kSwitch : 0; };
  int64_t own = weight(tid), up_to = own, rest = 0;
  for (int b = tid + kThreads; b < p.B; b += kThreads) rest += weight(b);
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t v = __shfl_up_sync(0xffffffffu, up_to, o);
    if (lane >= o) up_to += v;
    rest += __shfl_xor_sync(0xffffffffu, rest, o);
  }
  if (lane == 31) {
    scan[0][warp] = up_to;
    scan[1][warp] = rest;
  }
  __syncthreads();
  int64_t total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) total += scan[0][w] + scan[1][w];
  const int shares = (int)min((int64_t)gridDim.x, total);
  const int64_t first = share_begin((int)blockIdx.x, total, shares);
  if (tid == 0) {
    share.total = total;
    share.shares = shares;
    share.at = first;
    share.end = (int)blockIdx.x < shares ? share_begin((int)blockIdx.x + 1, total, shares) : first;
  }
  int64_t before = 0;
  for (int b0 = 0;;) {
    int64_t base = before;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) base += scan[0][w];
      before += scan[0][w];
    }
    if (first >= base + up_to - own && first < base + up_to) {
      share.b = b0 + tid;
      share.before = base + up_to - own;
    }
    b0 += kThreads;
    if (first < before || b0 >= p.B) break;          // (the whole block)
    own = up_to = weight(b0 + tid);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t v = __shfl_up_sync(0xffffffffu, up_to, o);
      if (lane >= o) up_to += v;
    }
    __syncthreads();
    if (lane == 31) scan[0][warp] = up_to;
    __syncthreads();
  }
  __syncthreads();
}

// Where a 16-byte chunk of a key's or a value's row lies in its tile of 16 rows, so that the fragment loads below meet no bank
// twice.  d = 128: rows of eight chunks, K read at chunks 4j + t of rows g, V at chunk g of rows 2t.  d = 64: rows of four
// chunks; K needs nothing, V (8 bytes a lane) has its rows paired anew.
template <int D> __device__ __forceinline__ uint32_t k_offset(int row, int chunk) {
  if constexpr (D == 128) return (uint32_t)(row * 128 + ((chunk ^ ((row & 1) << 2)) << 4));
  return (uint32_t)(row * 64 + (chunk << 4));
}
template <int D> __device__ __forceinline__ uint32_t v_offset(int row, int chunk) {
  if constexpr (D == 128) return (uint32_t)(row * 128 + ((chunk ^ (((row >> 1) & 3) << 1)) << 4));
  return (uint32_t)((row ^ ((row >> 1) & 1)) * 64 + ((chunk ^ (((row >> 2) & 1) << 1)) << 4));
}

// ROWS: rows of queries that a block's tile holds, 8 or 16.
template <int D, bool INT8, bool BF16, int ROWS>
__global__ void __launch_bounds__(kThreads, kv8_per_sm<D, ROWS>()) attn_decode_kv8_kernel(const Kv8Args p) {
  constexpr int NJ = D / 64;                           // 16-byte pieces of a key's row a lane takes
  constexpr int NE = D / 8;                            // columns of the output a lane's V pieces hold
  constexpr int TILE = 16 * D, STAGE = 2 * TILE;
  constexpr bool REST = !BF16;                         // Q's and P's remainders take part
  constexpr int G = ROWS / 8;
  extern __shared__ __align__(16) uint8_t smem[];
  constexpr int kQPitch = D + 8;
  __shared__ int page_ids[kMaxPages];                  // -1: none
  __shared__ float2 page_scales[kMaxPages];            // keys', values'
  __shared__ __align__(16) uint16_t q_rows[(REST ? 2 : 1) * ROWS * kQPitch];      // Q's rows as fp16, and what that leaves over
  __shared__ float q_scale[ROWS];
  __shared__ int q_sees[ROWS];                         // keys that a row's token sees
  pdl_wait();
  // (The merge kernel begins when this one's blocks have ended: let in earlier, its blocks take the SMs unevenly from those of the next
  // call, 52 against 48 us for 64 sequences and 59 against 45 for 100 of 64-wide heads.)
  if (p.cluster > 1) pdl_trigger();
  const int hkv = blockIdx.y / p.tiles, tile = blockIdx.y % p.tiles;
  const int rep = p.Hq / p.Hkv, rows = p.Sq * rep;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  // The block's share: a cluster's blocks have a sequence's keys between them, otherwise the blocks of a KV head share out all
  // sequences' keys.
  __shared__ Share share;
  if (p.cluster == 1) find_share(p, share);
  do {
  if (p.cluster == 1 && share.at >= share.end) return; // (more blocks than places)
  const int b = p.cluster > 1 ? (int)blockIdx.z : share.b;
  const int L_raw = p.seqlens[b], L = max(0, min(L_raw, p.max_len)), n_units = units_of(p, b);
  int unit, unit_end;
  if (p.cluster > 1) {
    const int each = (n_units + p.cluster - 1) / p.cluster;
    unit = min((int)blockIdx.x * each, n_units);
    unit_end = min(unit + each, n_units);
  } else {
    const int64_t begins = share.before + kSwitch;     // where b's units do
    unit = (int)max((int64_t)0, share.at - begins);
    unit_end = (int)max((int64_t)0, min((int64_t)n_units, share.end - begins));
    if (tid == 0) {
      share.unit = unit;
      share.unit_end = unit_end;
      share.n_units = n_units;
    }
  }
  if (p.cluster > 1 || unit_end > unit) {
  const int key_begin = min(unit * kStep, L), key_end = min(L, unit_end * kStep);

  // ---- page numbers and scales of the keys from span_begin on ----
  const int shift = __ffs(p.page) - 1;
  int span_begin = key_begin, span_end = min(key_end, key_begin + kSpan), page0 = key_begin >> shift;
  auto span_pages = [&]() { return span_end > span_begin ? ((span_end - 1) >> shift) - page0 + 1 : 0; };
  auto page_id = [&](int i) { return i < span_pages() ? p.table[(int64_t)b * p.table_stride + page0 + i] : -1; };
  auto page_scale = [&](int id) {
    const bool good = id >= 0 && id < p.pages;
    return make_float2(good ? p.k_scale[(int64_t)id * p.Hkv + hkv] : 0.f, good ? p.v_scale[(int64_t)id * p.Hkv + hkv] : 0.f);
  };
  auto keep_page = [&](int i, int id, float2 scales) {
    page_ids[i] = id >= 0 && id < p.pages ? id : -1;
    page_scales[i] = scales;
  };
  auto load_pages = [&](int from) {
    for (int i = from; i < span_pages(); i += kThreads) {
      const int id = page_id(i);
      keep_page(i, id, page_scale(id));
    }
    __syncthreads();
  };
  const int first_id = page_id(tid);

  // ---- Q, turned, as fp16: sixteen threads a row, which have pairs of elements half a head apart ----
  // (Asked for before the first tiles, behind which the loads would take 4 us, and beside the pages' scales.  Every warp preparing its own fragments took 3 us of all warps' issue.)
  constexpr int NP = D / 32;                           // pairs of a thread
  using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
  uint32_t q_lo[G][NP / 2], q_hi[G][NP / 2];
  float2 q_cos[G][NP / 2], q_sin[G][NP / 2];
#pragma unroll
  for (int h = 0; h < G; ++h) {
    const int r = tile * ROWS + h * 8 + (tid >> 4), i0 = NP * (tid & 15);
    const bool on = r < rows;
    const int s = on ? r / rep : 0, head = hkv * rep + (on ? r - s * rep : 0), angle = L_raw - p.Sq + s;
    const bool turn = p.cos_tab != nullptr && angle >= 0 && angle < p.table_rows;
    const uint16_t* src = p.q + (int64_t)b * p.q_batch_stride + (int64_t)s * p.q_token_stride + (int64_t)head * D + i0;
    const int64_t from = (int64_t)angle * (D / 2) + i0;
#pragma unroll
    for (int i = 0; i < NP / 2; ++i) {
      q_lo[h][i] = on ? *reinterpret_cast<const uint32_t*>(src + 2 * i) : 0u;
      q_hi[h][i] = on ? *reinterpret_cast<const uint32_t*>(src + D / 2 + 2 * i) : 0u;
      q_cos[h][i] = turn ? *reinterpret_cast<const float2*>(p.cos_tab + from + 2 * i) : make_float2(1.f, 1.f);
      q_sin[h][i] = turn ? *reinterpret_cast<const float2*>(p.sin_tab + from + 2 * i) : make_float2(0.f, 0.f);
    }
    if ((tid & 15) == 0) q_sees[h * 8 + (tid >> 4)] = on ? min(L, L_raw - p.Sq + 1 + s) : 0;
  }
  const float2 first_scale = page_scale(first_id);
#pragma unroll
  for (int h = 0; h < G; ++h) {
    const int r_here = h * 8 + (tid >> 4), i0 = NP * (tid & 15);
    float lo[NP], hi[NP];
#pragma unroll
    for (int i = 0; i < NP; i += 2) {
      const float2 a = unpack_pair<T>(q_lo[h][i / 2]), e = unpack_pair<T>(q_hi[h][i / 2]), c = q_cos[h][i / 2], sn = q_sin[h][i / 2];
      lo[i] = a.x * c.x - e.x * sn.x; hi[i] = a.x * sn.x + e.x * c.x;
      lo[i + 1] = a.y * c.y - e.y * sn.y; hi[i + 1] = a.y * sn.y + e.y * c.y;
    }
    // fp16 keeps 11 bits between 2^-14 and 65504: the row's maximum goes to [2^13, 2^14)
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < NP; ++i) top = fmaxf(top, fmaxf(fabsf(lo[i]), fabsf(hi[i])));
#pragma unroll
    for (int o_ = 1; o_ < 16; o_ <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o_));
    const int ex = min(max((int)(__float_as_uint(top) >> 23) - 127, -100), 127);      // (an infinity or a NaN stays what it is)
    const float up = __uint_as_float((uint32_t)(13 - ex + 127) << 23);
    uint16_t* row = q_rows + r_here * kQPitch + i0;
#pragma unroll
    for (int i = 0; i < NP; i += 2)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float x = (c ? hi[i] : lo[i]) * up, y = (c ? hi[i + 1] : lo[i + 1]) * up;
        const uint32_t w = pack_half(x, y);
        *reinterpret_cast<uint32_t*>(row + c * (D / 2) + i) = w;
        if constexpr (REST) {
          const float2 f = unpack_half(w);
          *reinterpret_cast<uint32_t*>(row + ROWS * kQPitch + c * (D / 2) + i) = pack_half(x - f.x, y - f.y);
        }
      }
    if ((tid & 15) == 0) q_scale[r_here] = __uint_as_float((uint32_t)(ex - 13 + 127) << 23) * p.scale * (p.softcap != 0.f ? 1.f : kLog2e);
  }
  if (tid < span_pages()) keep_page(tid, first_id, first_scale);
  load_pages(tid + kThreads);

  // ---- the ring's first stages ----
  // A lane's pieces of a tile are 512 bytes apart in both memories; their swizzle is one of two.
  constexpr int kRing = kv8_ring<D, ROWS>();
  constexpr int CPR = D / 16, kPieces = CPR / 2;       // 16-byte pieces of a row, and of a lane
  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + (uint32_t)(warp * kRing * STAGE);
  const uint32_t k_dst = k_offset<D>(lane / CPR, lane % CPR);
  const uint32_t v_dst0 = v_offset<D>(lane / CPR, lane % CPR), v_dst1 = v_offset<D>(lane / CPR + 32 / CPR, lane % CPR) - 512u;
  auto issue = [&](int key0, int stage) {
    if (key0 < span_end) {
      const uint32_t base = ring + (uint32_t)(stage * STAGE);
      const int id = page_ids[(key0 >> shift) - page0];
      const int64_t from = (int64_t)max(id, 0) * p.page_stride + (int64_t)hkv * p.head_stride + (int64_t)(key0 & (p.page - 1)) * D + lane * 16;
      const uint8_t* ks = p.k_cache + from;
      const uint8_t* vs = p.v_cache + from;
      const uint32_t kd = base + k_dst, v0 = base + TILE + v_dst0, v1 = base + TILE + v_dst1;
      if (id >= 0 && key0 + 16 <= span_end) {
        cp_async_16<0>(kd, ks);
        cp_async_16<0>(v0, vs);
        cp_async_16<512>(kd, ks);
        cp_async_16<512>(v1, vs);
        if constexpr (kPieces == 4) {
          cp_async_16<1024>(kd, ks);
          cp_async_16<1024>(v0, vs);
          cp_async_16<1536>(kd, ks);
          cp_async_16<1536>(v1, vs);
        }
      } else {                                         // zeros for the rows that are not there
        const int left = id >= 0 ? span_end - key0 - lane / CPR : 0;
        cp_async_16_or_zero<0>(kd, ks, 0 < left);
        cp_async_16_or_zero<0>(v0, vs, 0 < left);
        cp_async_16_or_zero<512>(kd, ks, 32 / CPR < left);
        cp_async_16_or_zero<512>(v1, vs, 32 / CPR < left);
        if constexpr (kPieces == 4) {
          cp_async_16_or_zero<1024>(kd, ks, 64 / CPR < left);
          cp_async_16_or_zero<1024>(v0, vs, 64 / CPR < left);
          cp_async_16_or_zero<1536>(kd, ks, 96 / CPR < left);
          cp_async_16_or_zero<1536>(v1, vs, 96 / CPR < left);
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");          // (always: the groups are counted)
  };
  auto issue_first = [&]() {
#pragma unroll
    for (int s = 0; s < kRing - 1; ++s) issue(span_begin + warp * 16 + s * kStep, s);
  };
  issue_first();

  // ---- its fragments: row g; registers 2i, 2i + 1 of a piece are the MMA's k slots 2t and 2t + 8 of step i ----
  uint32_t qa[G][NJ][8], qr[G][NJ][8];
  float scale_q[G][2];                                 // of rows 2t and 2t + 1, which the lane has scores of
  int sees[G][2];
#pragma unroll
  for (int h = 0; h < G; ++h) {
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int i = 0; i < 8; i += 4) {
        const uint16_t* src = q_rows + (h * 8 + g) * kQPitch + 16 * (4 * j + t) + 2 * i;
        const uint4 v = *reinterpret_cast<const uint4*>(src);
        qa[h][j][i] = v.x; qa[h][j][i + 1] = v.y; qa[h][j][i + 2] = v.z; qa[h][j][i + 3] = v.w;
        if constexpr (REST) {
          const uint4 u = *reinterpret_cast<const uint4*>(src + ROWS * kQPitch);
          qr[h][j][i] = u.x; qr[h][j][i + 1] = u.y; qr[h][j][i + 2] = u.z; qr[h][j][i + 3] = u.w;
        }
      }
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      scale_q[h][c] = q_scale[h * 8 + 2 * t + c];
      sees[h][c] = q_sees[h * 8 + 2 * t + c];
    }
  }

  float o[NE / 2][G][4];                               // columns 2e and 2e + 1 of the lane's NE, rows 2t and 2t + 1 each
#pragma unroll
  for (int e = 0; e < NE / 2; ++e)
#pragma unroll
    for (int h = 0; h < G; ++h)
#pragma unroll
      for (int c = 0; c < 4; ++c) o[e][h][c] = 0.f;
  // The reference that a row's scores are taken against moves only when one exceeds it by more than 2^kSlack: P is then at most
  // that, fp16 rounds it all the same, and most steps need no maximum over the lanes and leave O and the sums alone.
  // (kLift takes P to the upper end of fp16's range, 2^15: with a share of 2^-8 all of its bits last down to 2^-15 of the greatest P.  The
  // reference stays within 2^-50 .. 2^50: fp32 holds O at either end, whatever scales the append makes, 2^-49 .. 2^120.)
  constexpr float kSlack = 6.f, kLift = 512.f, kNothing = -3.4028235e38f, kNear = 0x1p-8f, kRefLeast = 0x1p-50f, kRefMost = 0x1p50f;
  float m_run[G][2], l_run[G][2], v_ref = 0.f, v_inv = 0.f;
  int sees_all = 0x7fffffff;                           // keys that every row of the tile sees
#pragma unroll
  for (int h = 0; h < G; ++h)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      m_run[h][c] = kNothing;
      l_run[h][c] = 0.f;
      sees_all = min(sees_all, tile * ROWS + h * 8 + 2 * t + c < rows ? sees[h][c] : 0x7fffffff);
    }
#pragma unroll
  for (int o_ = 16; o_ > 0; o_ >>= 1) sees_all = min(sees_all, __shfl_xor_sync(0xffffffffu, sees_all, o_));

  for (;;) {
    int it = 0;
    for (int key0 = span_begin + warp * 16; key0 < span_end; key0 += kStep, ++it) {
      issue(key0 + (kRing - 1) * kStep, (it + kRing - 1) % kRing);
      asm volatile("cp.async.wait_group %0;" ::"n"(kRing - 1) : "memory");
      __syncwarp();
      const uint32_t st = ring + (uint32_t)((it % kRing) * STAGE);
      const int pi = (key0 >> shift) - page0;
      const float2 info = page_scales[pi];
      const float ks = info.x, vs = info.y;
      const bool good = page_ids[pi] >= 0;

      // ---- S^T = K Q^T: this lane gets keys g and g + 8 of rows 2t and 2t + 1 ----
      float s_acc[G][NJ][4];
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
#pragma unroll
        for (int h = 0; h < G; ++h)
#pragma unroll
          for (int c = 0; c < 4; ++c) s_acc[h][j][c] = 0.f;
        const uint4 k0 = lds_16(st + k_offset<D>(g, 4 * j + t)), k1 = lds_16(st + k_offset<D>(8 + g, 4 * j + t));
        const uint32_t w0[4] = {k0.x, k0.y, k0.z, k0.w}, w1[4] = {k1.x, k1.y, k1.z, k1.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t a0, a1, a2, a3;
          kv8_word_to_half<INT8>(w0[i], a0, a2);
          kv8_word_to_half<INT8>(w1[i], a1, a3);
#pragma unroll
          for (int h = 0; h < G; ++h) {
            mma_16816<false>(s_acc[h][j], a0, a1, a2, a3, qa[h][j][2 * i], qa[h][j][2 * i + 1]);
            if constexpr (REST) mma_16816<false>(s_acc[h][j], a0, a1, a2, a3, qr[h][j][2 * i], qr[h][j][2 * i + 1]);
          }
        }
      }

      // ---- running softmax ----
      float pv[G][2][2];                                 // [.][key g, key g + 8][row]
      bool beyond = false;
#pragma unroll
      for (int h = 0; h < G; ++h)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float f = ks * scale_q[h][c];
#pragma unroll
          for (int kb = 0; kb < 2; ++kb) {
            float s = s_acc[h][0][2 * kb + c];
            if constexpr (NJ == 2) s += s_acc[h][1][2 * kb + c];
            pv[h][kb][c] = s * f;
          }
        }
      if (p.softcap != 0.f) {
#pragma unroll
        for (int h = 0; h < G; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i) pv[h][i >> 1][i & 1] = p.softcap * tanhf(pv[h][i >> 1][i & 1] / p.softcap) * kLog2e;
      }
      if (!good || key0 + 16 > sees_all) {
#pragma unroll
        for (int h = 0; h < G; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (!good || key0 + 8 * (i >> 1) + g >= sees[h][i & 1]) pv[h][i >> 1][i & 1] = -INFINITY;
      }
#pragma unroll
      for (int h = 0; h < G; ++h)
#pragma unroll
        for (int c = 0; c < 2; ++c) beyond |= fmaxf(pv[h][0][c], pv[h][1][c]) > m_run[h][c] + kSlack;
      float v_share = vs * v_inv;
      bool far = false;
      const bool fits = fabsf(v_share) >= kLift * kNear && fabsf(v_share) <= kLift * 1.001f;      // (one ulp above it is the reference itself; NaN: no)
      if (__any_sync(0xffffffffu, beyond) || !fits) {
        // (the quick division, off by two units of fp32's last place where the reference rises: the rounded one costs five short sequences 0.3 us)
        const float ref = fminf(fmaxf(fabsf(vs), kRefLeast), kRefMost), ref_corr = ref > v_ref ? __fdividef(v_ref, ref) : 1.f;
        if (ref > v_ref) {
          v_ref = ref;
          v_inv = kLift / ref;
        }
        far = good && !(fabsf(vs) >= kNear * v_ref && fabsf(vs) <= v_ref);
        v_share = far ? kLift : vs * v_inv;
#pragma unroll
        for (int h = 0; h < G; ++h)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float mx = fmaxf(pv[h][0][c], pv[h][1][c]);
#pragma unroll
            for (int o_ = 4; o_ < 32; o_ <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o_));
            const float m_new = fmaxf(m_run[h][c], mx);
            float corr = ex2(m_run[h][c] - m_new);
            m_run[h][c] = m_new;
            l_run[h][c] *= corr;
            corr *= ref_corr;
#pragma unroll
            for (int e = 0; e < NE / 2; ++e) {
              o[e][h][c] *= corr;
              o[e][h][c + 2] *= corr;
            }
          }
      }
#pragma unroll
      for (int h = 0; h < G; ++h)
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const float e = ex2(pv[h][kb][c] - m_run[h][c]);
            l_run[h][c] += e;
            pv[h][kb][c] = e * v_share;
          }
      if (key0 + 16 > sees_all) {                        // (whatever the scale of a page that the row does not see)
#pragma unroll
        for (int h = 0; h < G; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (key0 + 8 * (i >> 1) + g >= sees[h][i & 1]) pv[h][i >> 1][i & 1] = 0.f;
      }
      uint32_t pa[G][2], pr[G][2];                       // of row g: keys 2t, 2t + 1 and 2t + 8, 2t + 9
      auto pack_p = [&]() {
#pragma unroll
        for (int h = 0; h < G; ++h)
#pragma unroll
          for (int kb = 0; kb < 2; ++kb) {
            const uint32_t whole_p = pack_half(pv[h][kb][0], pv[h][kb][1]);
            pa[h][kb] = transpose_8x8(whole_p);
            if constexpr (REST) {
              const float2 f = unpack_half(whole_p);
              pr[h][kb] = transpose_8x8(pack_half(pv[h][kb][0] - f.x, pv[h][kb][1] - f.y));
            }
          }
      };
      // A word of V of each of a lane's four keys, as the MMA's operands: columns 2e and 2e + 1 from b0[2e], b0[2e + 1], b1[2e], b1[2e + 1].
      auto unpack_v = [](uint32_t w0, uint32_t w1, uint32_t w2, uint32_t w3, uint32_t (&b0)[4], uint32_t (&b1)[4]) {
        kv8_word_to_half<INT8>(__byte_perm(w0, w1, 0x5140), b0[0], b0[1]);
        kv8_word_to_half<INT8>(__byte_perm(w0, w1, 0x7362), b0[2], b0[3]);
        kv8_word_to_half<INT8>(__byte_perm(w2, w3, 0x5140), b1[0], b1[1]);
        kv8_word_to_half<INT8>(__byte_perm(w2, w3, 0x7362), b1[2], b1[3]);
      };
      auto v_word = [&](int s, int w) {                  // word w of key 2t, 2t + 1, 2t + 8, 2t + 9
        const int r = 2 * t + (s & 1) + 8 * (s >> 1);
        const uint32_t at = D == 128 ? v_offset<D>(r, g) : v_offset<D>(r, g >> 1) + (uint32_t)((g & 1) * 8);
        uint32_t v;
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(st + TILE + at + 4u * (uint32_t)w));
        return INT8 ? v : v & ~__vcmpeq4(v & 0x7f7f7f7fu, 0x7f7f7f7fu);      // (a NaN is seen to below)
      };
      if (__builtin_expect(far, 0)) {
        pack_p();
        const float apart = vs / v_ref;
#pragma unroll
        for (int w = 0; w < NE / 4; ++w) {
          uint32_t b0[4], b1[4];
          unpack_v(v_word(0, w), v_word(1, w), v_word(2, w), v_word(3, w), b0, b1);
#pragma unroll
          for (int e = 0; e < 4; e += 2)
#pragma unroll
            for (int h = 0; h < G; ++h) {
              float n[4] = {0.f, 0.f, 0.f, 0.f};
              mma_16816<false>(n, b0[e], b0[e + 1], b1[e], b1[e + 1], pa[h][0], pa[h][1]);
              if constexpr (REST) mma_16816<false>(n, b0[e], b0[e + 1], b1[e], b1[e + 1], pr[h][0], pr[h][1]);
#pragma unroll
              for (int c = 0; c < 4; ++c)
                if (key0 < sees[h][c & 1]) o[2 * w + e / 2][h][c] += n[c] * apart;      // (0 * infinity is not 0)
            }
        }
#pragma unroll
        for (int h = 0; h < G; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i) pv[h][i >> 1][i & 1] = 0.f;
      }
      pack_p();

      // ---- O^T += V^T P^T: a lane holds d = NE g .. of keys 2t, 2t + 1, 2t + 8, 2t + 9 ----
      uint32_t vw[4][NE / 4];
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const int r = 2 * t + (s & 1) + 8 * (s >> 1);
        if constexpr (D == 128) {
          const uint4 v = lds_16(st + TILE + v_offset<D>(r, g));
          vw[s][0] = v.x; vw[s][1] = v.y; vw[s][2] = v.z; vw[s][3] = v.w;
        } else {
          const uint2 v = lds_8(st + TILE + v_offset<D>(r, g >> 1) + (uint32_t)((g & 1) * 8));
          vw[s][0] = v.x; vw[s][1] = v.y;
        }
      }
      __syncwarp();                                      // every lane has read the stage: it may be filled again
      // A NaN among the values is for the rows that see its key alone (0 * NaN is not 0): it leaves the product, and the rows and
      // columns that it belongs to are counted by a product of their own.
      if (!INT8 && key0 + 16 > sees_all) {
        uint32_t any = 0;
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
          for (int w = 0; w < NE / 4; ++w) any |= __vcmpeq4(vw[s][w] & 0x7f7f7f7fu, 0x7f7f7f7fu);
        if (__any_sync(0xffffffffu, any != 0)) {
          uint32_t seen[G][2];
#pragma unroll
          for (int h = 0; h < G; ++h)
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
              const int k = key0 + 8 * kb + g;
              seen[h][kb] = transpose_8x8((k < sees[h][0] ? 0x3c00u : 0u) | (k < sees[h][1] ? 0x3c000000u : 0u));
            }
#pragma unroll
          for (int w = 0; w < NE / 4; ++w) {
            uint32_t one[4], b0[4], b1[4];
#pragma unroll
            for (int s = 0; s < 4; ++s) {
              const uint32_t m = __vcmpeq4(vw[s][w] & 0x7f7f7f7fu, 0x7f7f7f7fu);
              one[s] = m & 0x38383838u;                  // (1 in e4m3)
              vw[s][w] &= ~m;
            }
            kv8_word_to_half<INT8>(__byte_perm(one[0], one[1], 0x5140), b0[0], b0[1]);
            kv8_word_to_half<INT8>(__byte_perm(one[0], one[1], 0x7362), b0[2], b0[3]);
            kv8_word_to_half<INT8>(__byte_perm(one[2], one[3], 0x5140), b1[0], b1[1]);
            kv8_word_to_half<INT8>(__byte_perm(one[2], one[3], 0x7362), b1[2], b1[3]);
#pragma unroll
            for (int e = 0; e < 4; e += 2)
#pragma unroll
              for (int h = 0; h < G; ++h) {
                float n[4] = {0.f, 0.f, 0.f, 0.f};
                mma_16816<false>(n, b0[e], b0[e + 1], b1[e], b1[e + 1], seen[h][0], seen[h][1]);
#pragma unroll
                for (int c = 0; c < 4; ++c)
                  if (n[c] > 0.f) o[2 * w + e / 2][h][c] = __int_as_float(0x7fffffff);
              }
          }
        }
      }
#pragma unroll
      for (int w = 0; w < NE / 4; ++w) {
        uint32_t b0[4], b1[4];
        unpack_v(vw[0][w], vw[1][w], vw[2][w], vw[3][w], b0, b1);
#pragma unroll
        for (int e = 0; e < 4; e += 2)
#pragma unroll
          for (int h = 0; h < G; ++h) {
            mma_16816<false>(o[2 * w + e / 2][h], b0[e], b0[e + 1], b1[e], b1[e + 1], pa[h][0], pa[h][1]);
            if constexpr (REST) mma_16816<false>(o[2 * w + e / 2][h], b0[e], b0[e + 1], b1[e], b1[e + 1], pr[h][0], pr[h][1]);
          }
      }
    }

    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();                                     // the rings are idle, nobody reads the pages
    if (span_end >= key_end) break;
    span_begin = span_end;
    span_end = min(key_end, span_begin + kSpan);
    page0 = span_begin >> shift;
    load_pages(tid);
    issue_first();
  }

  // ---- merge the warps ----
  // A lane has NE neighbouring columns of two rows; every other lane's have their quarters of 32 bytes the other way round, so
  // that eight lanes' 16 bytes meet no bank twice.
  constexpr int kPitch = D + 4;
  auto column = [](int dd) { return dd ^ ((dd / NE & 1) << 2); };
  float* sm_o = reinterpret_cast<float*>(smem);        // [kWarps][ROWS][kPitch]
  float* sm_m = sm_o + kWarps * ROWS * kPitch;         // [kWarps][ROWS]
  float* sm_l = sm_m + kWarps * ROWS;
  float* cl_o = sm_l + kWarps * ROWS;                  // [ROWS][D] and [ROWS][2]: for the cluster's merge
  float* cl_ml = cl_o + ROWS * D;
  const float unlift = v_ref * (1.f / (kLift * kHead));
#pragma unroll
  for (int h = 0; h < G; ++h)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
#pragma unroll
      for (int o_ = 4; o_ < 32; o_ <<= 1) l_run[h][c] += __shfl_xor_sync(0xffffffffu, l_run[h][c], o_);
      const int r = h * 8 + 2 * t + c;
      if (g == 0) {
        sm_m[warp * ROWS + r] = m_run[h][c] > kNothing ? m_run[h][c] : l_run[h][c] == 0.f ? -INFINITY : 0.f;      // (nothing but NaN stays NaN)
        sm_l[warp * ROWS + r] = l_run[h][c];
      }
      float* row = sm_o + (warp * ROWS + r) * kPitch;
#pragma unroll
      for (int e = 0; e < NE / 2; e += 2)
        *reinterpret_cast<float4*>(row + column(NE * g + 2 * e)) =
            make_float4(unlift * o[e][h][c], unlift * o[e][h][c + 2], unlift * o[e + 1][h][c], unlift * o[e + 1][h][c + 2]);
    }
  __syncthreads();
  const int here = min(ROWS, rows - tile * ROWS);      // rows of this tile
  auto out_row = [&](int r) -> int64_t {
    const int rr = tile * ROWS + r, s = rr / rep;
    return ((int64_t)b * p.Sq + s) * p.Hq + hkv * rep + (rr - s * rep);
  };
  const bool whole = p.cluster == 1 && share.unit == 0 && share.unit_end == share.n_units;
  // A part of a sequence goes to the workspace: one begun in the middle to the block's first slot, one begun at the start to the second.
  const int64_t slot = (((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 2 + (p.cluster == 1 && share.unit > 0 ? 0 : 1)) * ROWS;
  for (int i = tid; i < here * (D / 4); i += kThreads) {
    const int r = i / (D / 4), dd = i % (D / 4) * 4;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) M = fmaxf(M, sm_m[w * ROWS + r]);
    float lsum = 0.f;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    if (M > -INFINITY) {
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float f = ex2(sm_m[w * ROWS + r] - M);
        const float4 v = *reinterpret_cast<const float4*>(sm_o + (w * ROWS + r) * kPitch + column(dd));
        lsum += sm_l[w * ROWS + r] * f;
        sum.x += v.x * f; sum.y += v.y * f; sum.z += v.z * f; sum.w += v.w * f;
      }
    }
    if (whole) {
      const float inv = lsum == 0.f ? 0.f : kHead / lsum;
      *reinterpret_cast<uint2*>(p.out + out_row(r) * D + dd) = make_uint2(round_pair<BF16>(sum.x * inv, sum.y * inv), round_pair<BF16>(sum.z * inv, sum.w * inv));
    } else {
      float* po = p.cluster > 1 ? cl_o + r * D + dd : p.part_o + (slot + r) * D + dd;
      *reinterpret_cast<float4*>(po) = sum;
      if (dd == 0) *reinterpret_cast<float2*>(p.cluster > 1 ? cl_ml + 2 * r : p.part_ml + 2 * (slot + r)) = make_float2(M, lsum);
    }
  }
  if (p.cluster > 1) {
    cluster_arrive();
    cluster_wait();
    const uint32_t lo = (uint32_t)__cvta_generic_to_shared(cl_o), lml = (uint32_t)__cvta_generic_to_shared(cl_ml);
    for (int i = blockIdx.x * kThreads + tid; i < here * D; i += p.cluster * kThreads) {
      const int r = i / D, dd = i - r * D;
      float pm[8], pl[8], po[8], M = -INFINITY;
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        pm[c] = -INFINITY;
        pl[c] = po[c] = 0.f;
        if (c < p.cluster) {
          uint32_t ro, rml;
          asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(ro) : "r"(lo + 4u * (uint32_t)i), "r"((uint32_t)c));
          asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(rml) : "r"(lml + 8u * (uint32_t)r), "r"((uint32_t)c));
          asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(po[c]) : "r"(ro) : "memory");
          asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(pm[c]), "=f"(pl[c]) : "r"(rml) : "memory");
        }
        M = fmaxf(M, pm[c]);
      }
      float lsum = 0.f, osum = 0.f;
      if (M > -INFINITY) {
#pragma unroll
        for (int c = 0; c < 8; ++c) {                  // split order: the same sum on every run
          const float f = exp2f(pm[c] - M);
          lsum += pl[c] * f;
          osum += po[c] * f;
        }
      }
      p.out[out_row(r) * D + dd] = round_bits<BF16>(lsum == 0.f ? 0.f : osum / lsum * kHead);
    }
    cluster_arrive();                                  // nobody leaves while a peer may still read its partial
    cluster_wait();
    return;                                            // (a cluster's block has one sequence)
  }
  }
  __syncthreads();                                     // (all has been read: the memory is the rings')
  if (tid == 0) {
    share.before += share.n_units + kSwitch;
    share.at = share.before;
    ++share.b;
  }
  __syncthreads();
  } while (share.at < share.end);
}

// Merge of the sequences that several blocks have had a part of.  `each` warps (1 .. 16) add up a row's parts, every each-th one, and
// are joined in shared memory; a lane has D / 32 neighbouring outputs.  (In the main kernel, by the block that comes last, it took
// 10 us a stage for 12 parts: one block has too few loads under way.)
template <bool BF16, int D, int ROWS>
__global__ void __launch_bounds__(512) attn_decode_kv8_merge_kernel(const Kv8Args p, int blocks, int each) {
  constexpr int W = D / 32, kBatch = 10;
  __shared__ float sm_o[16][D];
  __shared__ float2 sm_ml[16];
  __shared__ int64_t scan[2][16];
  pdl_wait_then_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, part = warp & (each - 1);
  const int b = blockIdx.y, r = blockIdx.x * ((int)(blockDim.x >> 5) / each) + warp / each;
  // which blocks had a part
  int64_t before = 0, total = 0;
  for (int i = threadIdx.x; i < p.B; i += blockDim.x) {
    const int w = units_of(p, i) + kSwitch;
    total += w;
    before += i < b ? w : 0;
  }
  const int n_units = units_of(p, b);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    total += __shfl_xor_sync(0xffffffffu, total, o);
    before += __shfl_xor_sync(0xffffffffu, before, o);
  }
  if (lane == 0) {
    scan[0][warp] = total;
    scan[1][warp] = before;
  }
  __syncthreads();
  total = before = 0;
  for (int w = 0; w < (int)(blockDim.x >> 5); ++w) {
    total += scan[0][w];
    before += scan[1][w];
  }
  const int shares = (int)min((int64_t)blocks, total);
  const int64_t begins = before + kSwitch;
  const int first = share_of(begins, total, shares), last = share_of(begins + n_units - 1, total, shares);
  if (first == last) return;                           // (one: the result is there)
  const bool on = r < p.Sq * p.Hq;
  const int s = on ? r / p.Hq : 0, head = on ? r - s * p.Hq : 0, rep = p.Hq / p.Hkv, hkv = head / rep, tr = s * rep + head - hkv * rep;
  const int64_t column = (int64_t)(hkv * p.tiles + tr / ROWS) * blocks;
  const int in_middle = share_begin(first, total, shares) > begins ? 0 : 1;      // (the parts behind the first begin in the middle)
  float M = -INFINITY, lsum = 0.f, o[W];
#pragma unroll
  for (int j = 0; j < W; ++j) o[j] = 0.f;
  auto join = [&](float2 ml, const float* v) {
    const float Mn = fmaxf(M, ml.x);
    const float keep = M > -INFINITY ? ex2(M - Mn) : 0.f, f = ml.x > -INFINITY ? ex2(ml.x - Mn) : 0.f;
    M = Mn;
    lsum = lsum * keep + ml.y * f;
#pragma unroll
    for (int j = 0; j < W; ++j) o[j] = o[j] * keep + v[j] * f;
  };
  if (on) {
    for (int k0 = first + part; k0 <= last; k0 += kBatch * each) {       // in the blocks' order
      float2 ml[kBatch];
      float v[kBatch][W];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int k = k0 + i * each;
        if (k <= last) {
          const int64_t slot = ((column + k) * 2 + (k == first ? in_middle : 0)) * ROWS + tr % ROWS;
          ml[i] = __ldcg(reinterpret_cast<const float2*>(p.part_ml + 2 * slot));
          if constexpr (W == 4) *reinterpret_cast<float4*>(v[i]) = __ldcg(reinterpret_cast<const float4*>(p.part_o + slot * D + lane * W));
          else *reinterpret_cast<float2*>(v[i]) = __ldcg(reinterpret_cast<const float2*>(p.part_o + slot * D + lane * W));
        }
      }
#pragma unroll
      for (int i = 0; i < kBatch; ++i)
        if (k0 + i * each <= last) join(ml[i], v[i]);
    }
  }
  if (each > 1) {
#pragma unroll
    for (int j = 0; j < W; ++j) sm_o[warp][lane * W + j] = o[j];
    if (lane == 0) sm_ml[warp] = make_float2(M, lsum);
    __syncthreads();
    if (part != 0 || !on) return;
    const float2 mine = lane < each ? sm_ml[warp + lane] : make_float2(-INFINITY, 0.f);
    M = mine.x;
#pragma unroll
    for (int x = 8; x > 0; x >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, x));
    M = __shfl_sync(0xffffffffu, M, 0);
    const float f_mine = mine.x > -INFINITY ? ex2(mine.x - M) : 0.f;
    lsum = 0.f;
#pragma unroll
    for (int j = 0; j < W; ++j) o[j] = 0.f;
    for (int w = 0; w < each; ++w) {
      const float f = __shfl_sync(0xffffffffu, f_mine, w);
      lsum += __shfl_sync(0xffffffffu, mine.y, w) * f;
#pragma unroll
      for (int j = 0; j < W; ++j) o[j] += sm_o[warp + w][lane * W + j] * f;
    }
  }
  if (!on) return;
  const float inv = lsum == 0.f ? 0.f : kHead / lsum;
  uint16_t* dst = p.out + ((int64_t)b * p.Sq * p.Hq + r) * D + lane * W;
  if constexpr (W == 4) *reinterpret_cast<uint2*>(dst) = make_uint2(round_pair<BF16>(o[0] * inv, o[1] * inv), round_pair<BF16>(o[2] * inv, o[3] * inv));
  else *reinterpret_cast<uint32_t*>(dst) = round_pair<BF16>(o[0] * inv, o[1] * inv);
}

template <int D, int ROWS> constexpr int kv8_smem() { return kWarps * kv8_ring<D, ROWS>() * 2 * 16 * D; }

// Clusters of `cluster` blocks of a kernel that can be resident at once (asked once per device and kernel).
int max_active_clusters(const void* kern, int cluster, int smem) {
  static std::mutex mu;
  static std::map<std::pair<std::pair<int, int>, const void*>, int> known;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  std::lock_guard<std::mutex> lock(mu);
  auto it = known.find({{dev, cluster}, kern});
  if (it != known.end()) return it->second;
  int n = 0;
  if (ensure_dynamic_smem(kern, smem) == LLMQRT_OK) {
    cudaLaunchAttribute attr[1];
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)cluster, 1, 1);
    cfg.blockDim = dim3(kThreads, 1, 1);
    cfg.dynamicSmemBytes = (size_t)smem;
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess) {
      cudaGetLastError();
      n = 0;
    }
  }
  known[{{dev, cluster}, kern}] = n;
  return n;
}

template <int D, bool INT8, bool BF16, int ROWS>
int launch(Kv8Args a, int B, void* workspace, cudaStream_t st) {
  constexpr int smem = kv8_smem<D, ROWS>();
  static_assert(smem >= (kWarps * ROWS * (D + 4 + 2) + ROWS * (D + 2)) * 4, "the rings hold the merge tile");
  auto kern = attn_decode_kv8_kernel<D, INT8, BF16, ROWS>;
  a.tiles = (int)ceil_div((int64_t)a.Sq * (a.Hq / a.Hkv), ROWS);
  a.B = B;
  const int64_t columns = (int64_t)a.Hkv * a.tiles;    // blocks' shares are of one KV head and row tile each
  const int slots = std::max(1, max_active_clusters(reinterpret_cast<const void*>(kern), 1, smem));
  const int64_t units = ceil_div(a.max_len > 0 ? a.max_len : 1, kStep);
  if (int rc = ensure_dynamic_smem(reinterpret_cast<const void*>(kern), smem)) return rc;
  // Few sequences that are not long: up to eight blocks for each, a cluster that merges their parts.  Otherwise all blocks that fit at
  // once share the keys out evenly, whatever the lengths, and sequences with several parts are merged by a second kernel.
  const int cluster = (int)std::min<int64_t>(8, units);
  if (cluster > 1 && a.max_len <= kClusterMergeMaxLen && B * columns <= max_active_clusters(reinterpret_cast<const void*>(kern), cluster, smem)) {
    a.cluster = cluster;
    if (int rc = launch_chained(kern, dim3((unsigned)cluster, (unsigned)columns, (unsigned)B), dim3(kThreads), smem, st, cluster, a)) return rc;
    return check_launch("attn_decode_kv8");
  }
  a.cluster = 1;
  // (one wave of blocks; where a column has fewer than four of them, up to four waves, the last of which is rarely full)
  const int64_t waves = columns * 4 <= slots ? 1 : 4;
  const int blocks = (int)std::min<int64_t>({std::max<int64_t>(1, waves * slots / columns), B * (units + kSwitch), kMaxBlocks});
  if (blocks > 1 && !workspace) return set_error(LLMQRT_ERR_WORKSPACE, "attn_decode_kv8: split keys need the workspace");
  const size_t slots_all = (size_t)columns * blocks * 2;
  if (blocks > 1 && (slots_all * ROWS * (D + 2) * 4 > LLMQRT_WS_PARTIAL_BYTES ))
    return set_error(LLMQRT_ERR_UNSUPPORTED, "attn_decode_kv8: the blocks' partial results do not fit the workspace");
  a.part_o = blocks > 1 ? reinterpret_cast<float*>(ws_partials(workspace)) : nullptr;
  a.part_ml = a.part_o + slots_all * ROWS * D;
  if (int rc = launch_chained(kern, dim3((unsigned)blocks, (unsigned)columns, 1), dim3(kThreads), smem, st, 1, a)) return rc;
  if (int rc = check_launch("attn_decode_kv8")) return rc;
  if (blocks == 1) return LLMQRT_OK;
  int each = 1;                                        // warps a row: about eight parts each, one batch of loads
  while (each < 16 && each * 8 * B < blocks) each *= 2;
  const int warps = std::max(4, each);
  if (int rc = launch_chained(attn_decode_kv8_merge_kernel<BF16, D, ROWS>, dim3((unsigned)ceil_div(a.Sq * a.Hq, warps / each), (unsigned)B),
                              dim3(32 * (unsigned)warps), 0, st, 1, a, blocks, each))
    return rc;
  return check_launch("attn_decode_kv8_merge");
}

}  // namespace
}  // namespace llmqrt

using namespace llmqrt;

extern "C" int llmqrt_attn_decode_kv8(const void* q, int64_t q_batch_stride, int64_t q_token_stride, const void* k_cache,
                                      const void* v_cache, int cache_type, int64_t page_stride, int64_t head_stride,
                                      const float* k_scale, const float* v_scale, const int32_t* block_table, int64_t table_stride,
                                      int64_t width, const int32_t* seqlens, const float* cos_table, const float* sin_table,
                                      int64_t table_rows, void* out, int dtype, int64_t B, int64_t Sq, int64_t Hq, int64_t Hkv,
                                      int64_t d, int64_t pages, int64_t page, int64_t max_seqlen, float softcap, void* workspace,
                                      llmqrt_stream_t stream) {
  LLMQRT_REQUIRE(dtype == LLMQRT_F16 || dtype == LLMQRT_BF16, "attn_decode_kv8: dtype must be fp16 or bf16");
  LLMQRT_REQUIRE(cache_type == LLMQRT_E4M3 || cache_type == LLMQRT_I8, "attn_decode_kv8: the cache holds e4m3 or int8");
  LLMQRT_REQUIRE(d == 64 || d == 128, "attn_decode_kv8: head_dim must be 64 or 128 (got %lld)", (long long)d);
  LLMQRT_REQUIRE(page >= 16 && page <= 128 && (page & (page - 1)) == 0,
                 "attn_decode_kv8: pages hold 16, 32, 64 or 128 tokens (got %lld)", (long long)page);
  LLMQRT_REQUIRE(Hkv > 0 && Hq > 0 && Hq % Hkv == 0 && Hq / Hkv <= 16 && Hq <= 1024, "attn_decode_kv8: need Hq %% Hkv == 0 and at most 16 query heads per KV head");
  LLMQRT_REQUIRE(Sq >= 0 && Sq <= 16, "attn_decode_kv8: at most 16 query tokens a sequence (got %lld)", (long long)Sq);
  LLMQRT_REQUIRE(B >= 0 && B < 65536 && pages >= 0 && pages <= 0x7fffffffll && width >= 0 && table_stride >= width && max_seqlen >= 0,
                 "attn_decode_kv8: bad shape");
  LLMQRT_REQUIRE(head_stride >= page * d && page_stride >= Hkv * head_stride && head_stride % 16 == 0 && page_stride % 16 == 0,
                 "attn_decode_kv8: the cache is [pages, Hkv, page, d] with contiguous pages, strides multiples of 16");
  LLMQRT_REQUIRE((cos_table == nullptr) == (sin_table == nullptr), "attn_decode_kv8: cos and sin tables go together");
  if (B == 0 || Sq == 0) return LLMQRT_OK;
  LLMQRT_REQUIRE(q && seqlens && out && (width == 0 || block_table) && (pages == 0 || (k_cache && v_cache && k_scale && v_scale)),
                 "attn_decode_kv8: null pointer");
  LLMQRT_REQUIRE(q_token_stride >= Hq * d && q_batch_stride >= 0 && q_token_stride % 8 == 0 && q_batch_stride % 8 == 0 &&
                 ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache) |
                   reinterpret_cast<uintptr_t>(out)) & 15) == 0, "attn_decode_kv8: q, caches and out must be 16-byte aligned");
  LLMQRT_REQUIRE(!cos_table || (table_rows > 0 && table_rows <= 0x7fffffffll &&
                                ((reinterpret_cast<uintptr_t>(cos_table) | reinterpret_cast<uintptr_t>(sin_table)) & 15) == 0),
                 "attn_decode_kv8: rotary tables must be 16-byte aligned fp32 [table_rows, d/2]");
  Kv8Args a{};
  a.q = static_cast<const uint16_t*>(q); a.q_batch_stride = q_batch_stride; a.q_token_stride = q_token_stride;
  a.k_cache = static_cast<const uint8_t*>(k_cache); a.v_cache = static_cast<const uint8_t*>(v_cache);
  a.page_stride = page_stride; a.head_stride = head_stride; a.k_scale = k_scale; a.v_scale = v_scale;
  a.table = block_table; a.table_stride = table_stride; a.seqlens = seqlens; a.cos_tab = cos_table; a.sin_tab = sin_table;
  a.table_rows = (int)table_rows; a.out = static_cast<uint16_t*>(out);
  a.Sq = (int)Sq; a.Hq = (int)Hq; a.Hkv = (int)Hkv; a.pages = (int)pages; a.page = (int)page;
  const int64_t most = max_seqlen < width * page ? max_seqlen : width * page;
  LLMQRT_REQUIRE(most <= 0x7fff0000ll, "attn_decode_kv8: sequences too long");      // (keys a few steps ahead are 32-bit numbers)
  a.max_len = pages == 0 ? 0 : (int)most;
  a.scale = 1.0f / sqrtf((float)d);
  a.softcap = softcap;
  cudaStream_t st = (cudaStream_t)stream;
  const bool i8 = cache_type == LLMQRT_I8, bf = dtype == LLMQRT_BF16, wide = Sq * (Hq / Hkv) > 8;
#define LLMQRT_KV8(DD, I, BF, R) return launch<DD, I, BF, R>(a, (int)B, workspace, st)
#define LLMQRT_KV8_R(DD, I, BF) do { if (wide) LLMQRT_KV8(DD, I, BF, 16); LLMQRT_KV8(DD, I, BF, 8); } while (0)
#define LLMQRT_KV8_BF(DD, I) do { if (bf) LLMQRT_KV8_R(DD, I, true); else LLMQRT_KV8_R(DD, I, false); } while (0)
#define LLMQRT_KV8_I(DD) do { if (i8) LLMQRT_KV8_BF(DD, true); else LLMQRT_KV8_BF(DD, false); } while (0)
  if (d == 128) LLMQRT_KV8_I(128);
  LLMQRT_KV8_I(64);
#undef LLMQRT_KV8_I
#undef LLMQRT_KV8_BF
#undef LLMQRT_KV8_R
#undef LLMQRT_KV8
}
