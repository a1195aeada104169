// Attention of the newest tokens of each sequence over a paged cache of 8-bit keys and values with a scale for each page and
// head (kv8.cuh), split over the keys.
//
//   S = (q . code_k) * k_scale[page] / sqrt(d)      O = sum_j softmax(S)_j * code_v * v_scale[page]
//
// HBM-bound: each code is read once, half the bytes of a 16-bit cache, so that what a key costs the schedulers counts:
// at 6.5 TB/s an SM takes a key and value row of 128 every 11 cycles.  Warps stream 16 keys a step through rings of their own in
// shared memory (cp.async, 16 keys always lie in one page), turn the codes into fp16, where both kinds are exact, and multiply
// with warp-level MMAs, whose rows are the query heads that share the KV head.
//   S = Q K^T : a lane's K fragment is 16 contiguous bytes of a key's row; Q is loaded with the same permutation of d.
//   O += P V  : the fragment wants two keys a register: bytes of two rows are interleaved before they are converted.
// Scales stay out of the products: k_scale multiplies S; v_scale, over the greatest one of the pages so far (a second running
// reference beside the softmax's maximum), multiplies P, which thus never leaves [0, 1], where fp16 rounds it as it rounds the result.
// Q in fp16 is exact for fp16 and, its row multiplied by a power of two, for bf16.
// With at most eight rows the MMA's other eight hold what the rounding of Q (rotated here) and of P to fp16 left over, so that an
// fp16 result is off by its own rounding alone; with more rows these remainders take MMAs of their own (fp16 only: bf16's own
// rounding is eight times as large).
//
// Grid (splits, Hkv * row tiles, B).  A block merges its four warps in shared memory; splits of one sequence are merged by the
// thread-block cluster that they form, or, where there are more than eight, by a second kernel from the workspace.
// Page numbers outside the cache and rows behind the last key are not read (zeros take their place) and get no weight.
#include <cstdlib>
#include <map>
#include <mutex>
#include <utility>

#include "kv8.cuh"

namespace llmqrt {
namespace {

constexpr int kWarps = 4, kThreads = kWarps * 32, kStep = 16 * kWarps;
constexpr int kRing = 6;                               // stages of a warp, 16 keys each
constexpr int kSpan = 4096;                            // keys whose page numbers and scales a block holds at a time
constexpr int kMaxPages = kSpan / 16 + 1;              // pages that these touch
constexpr int kClusterMergeMaxLen = 8192;               // greatest bound whose splits a cluster merges although it would take more than eight
constexpr float kLog2e = 1.4426950408889634f;

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
  float* part_o;                   // [B * Sq * Hq, splits, D]
  float* part_ml;                  // [B * Sq * Hq, splits, 2]
  int table_rows, Sq, Hq, Hkv, pages, page, max_len, chunk, splits, tiles, cluster;
  float scale, softcap;
};

__device__ __forceinline__ void cp_async_16_or_zero(uint32_t dst_smem, const void* src, bool take) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst_smem), "l"(src), "r"(take ? 16 : 0) : "memory");
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
__device__ __forceinline__ uint32_t pack_half(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack_half(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
template <bool BF16> __device__ __forceinline__ uint16_t round_bits(float f) {
  if constexpr (BF16) return __bfloat16_as_ushort(__float2bfloat16_rn(f));
  else return __half_as_ushort(__float2half_rn(f));
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
__global__ void __launch_bounds__(kThreads) attn_decode_kv8_kernel(const Kv8Args p) {
  constexpr int NJ = D / 64;                           // 16-byte pieces of a key's row a lane takes
  constexpr int NE = D / 8;                            // columns of the output a lane's V pieces hold
  constexpr int TILE = 16 * D, STAGE = 2 * TILE;
  constexpr bool REST = !BF16;                         // Q's and P's remainders take part
  constexpr int G = ROWS / 8;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int page_id[kMaxPages];
  __shared__ float page_ks[kMaxPages], page_vs[kMaxPages];
  pdl_wait();
  pdl_trigger();
  const int split = blockIdx.x, hkv = blockIdx.y / p.tiles, tile = blockIdx.y % p.tiles, b = blockIdx.z;
  const int rep = p.Hq / p.Hkv, rows = p.Sq * rep;
  const int L_raw = p.seqlens[b], L = max(0, min(L_raw, p.max_len));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  // A cluster's blocks share out the sequence's own length: the bound may be many times as long.
  int chunk = p.chunk;
  if (p.cluster > 1) chunk = max(kStep, ((L + p.cluster - 1) / p.cluster + kStep - 1) / kStep * kStep);
  const int key_begin = min(split * chunk, L), key_end = min(L, key_begin + chunk);
  if (p.cluster == 1 && key_begin >= key_end && split > 0) return;
  const int n_splits = max(1, (L + chunk - 1) / chunk);

  // ---- page numbers and scales of the keys from span_begin on ----
  const int shift = __ffs(p.page) - 1;
  int span_begin = key_begin, span_end = min(key_end, key_begin + kSpan), page0 = key_begin >> shift;
  auto load_pages = [&]() {
    const int n = span_end > span_begin ? ((span_end - 1) >> shift) - page0 + 1 : 0;
    for (int i = tid; i < n; i += kThreads) {
      const int id = p.table[(int64_t)b * p.table_stride + page0 + i];
      const bool good = id >= 0 && id < p.pages;
      page_id[i] = good ? id : -1;
      page_ks[i] = good ? p.k_scale[(int64_t)id * p.Hkv + hkv] : 0.f;
      page_vs[i] = good ? p.v_scale[(int64_t)id * p.Hkv + hkv] : 0.f;
    }
    __syncthreads();
  };
  load_pages();

  // ---- the ring's first stages ----
  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + (uint32_t)(warp * kRing * STAGE);
  auto issue = [&](int key0, int stage) {
    if (key0 < span_end) {
      constexpr int CPR = D / 16;
      const uint32_t base = ring + (uint32_t)(stage * STAGE);
      const int id = page_id[(key0 >> shift) - page0];
      const int64_t at = (int64_t)max(id, 0) * p.page_stride + (int64_t)hkv * p.head_stride + (int64_t)(key0 & (p.page - 1)) * D;
#pragma unroll
      for (int i = 0; i < 16 * CPR / 32; ++i) {
        const int n = i * 32 + lane, r = n / CPR, c = n % CPR;
        const bool take = id >= 0 && key0 + r < span_end;
        cp_async_16_or_zero(base + k_offset<D>(r, c), p.k_cache + at + n * 16, take);
        cp_async_16_or_zero(base + TILE + v_offset<D>(r, c), p.v_cache + at + n * 16, take);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");          // (always: the groups are counted)
  };
  auto issue_first = [&]() {
#pragma unroll
    for (int s = 0; s < kRing - 1; ++s) issue(span_begin + warp * 16 + s * kStep, s);
  };
  issue_first();

  // ---- Q: rows g and g + 8 of the tile; register 2i, 2i + 1 of a piece are the MMA's k slots 2t and 2t + 8 of step i ----
  uint32_t qa[G][NJ][8], qr[G][NJ][8];                 // fp16 and what it leaves over
  float row_scale[G];
  int sees[G];                                         // keys that the row's token sees
#pragma unroll
  for (int h = 0; h < G; ++h) {
    const int r = tile * ROWS + h * 8 + g;
    const bool on = r < rows;
    const int s = on ? r / rep : 0, head = hkv * rep + (on ? r - s * rep : 0);
    sees[h] = on ? min(L, L_raw - p.Sq + 1 + s) : 0;
    const int angle = L_raw - p.Sq + s;
    const bool rotate = p.cos_tab != nullptr && angle >= 0 && angle < p.table_rows;
    const uint16_t* src = p.q + (int64_t)b * p.q_batch_stride + (int64_t)s * p.q_token_stride + (int64_t)head * D;
    using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
    float x[NJ][16], other[NJ][16];                    // this lane's elements 16 (4j + t) .. + 15, and those they are rotated with
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const int d0 = 16 * (4 * j + t), d1 = (d0 + D / 2) % D;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint4 v = make_uint4(0, 0, 0, 0), w = v;
        if (on) {
          v = *reinterpret_cast<const uint4*>(src + d0 + 8 * i);
          if (rotate) w = *reinterpret_cast<const uint4*>(src + d1 + 8 * i);
        }
        const uint32_t vw[4] = {v.x, v.y, v.z, v.w}, ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 a = unpack_pair<T>(vw[e]), c = unpack_pair<T>(ww[e]);
          x[j][8 * i + 2 * e] = a.x; x[j][8 * i + 2 * e + 1] = a.y;
          other[j][8 * i + 2 * e] = c.x; other[j][8 * i + 2 * e + 1] = c.y;
        }
      }
      if (rotate) {
        const bool low = d0 < D / 2;
        const float* cr = p.cos_tab + (int64_t)angle * (D / 2) + d0 % (D / 2);
        const float* sr = p.sin_tab + (int64_t)angle * (D / 2) + d0 % (D / 2);
#pragma unroll
        for (int e = 0; e < 16; ++e) x[j][e] = low ? x[j][e] * cr[e] - other[j][e] * sr[e] : other[j][e] * sr[e] + x[j][e] * cr[e];
      }
    }
    // fp16 keeps 11 bits between 2^-14 and 65504: the row's maximum goes to [2^13, 2^14)
    float top = 0.f;
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) top = fmaxf(top, fabsf(x[j][e]));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const int ex = min(max((int)(__float_as_uint(top) >> 23) - 127, -100), 127);      // (an infinity or a NaN stays what it is)
    const float up = __uint_as_float((uint32_t)(13 - ex + 127) << 23);
    row_scale[h] = __uint_as_float((uint32_t)(ex - 13 + 127) << 23) * p.scale;
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float a = x[j][2 * e] * up, c = x[j][2 * e + 1] * up;
        qa[h][j][e] = pack_half(a, c);
        if (REST) {
          const float2 f = unpack_half(qa[h][j][e]);
          qr[h][j][e] = pack_half(a - f.x, c - f.y);
        }
      }
  }

  float o[NE][4];                                      // ROWS 8: c0, c1 of P's fp16 part, c2, c3 of the rest; 16: rows g and g + 8
#pragma unroll
  for (int e = 0; e < NE; ++e)
#pragma unroll
    for (int c = 0; c < 4; ++c) o[e][c] = 0.f;
  float m_run[G], l_run[G], v_ref = 0.f;
#pragma unroll
  for (int h = 0; h < G; ++h) {
    m_run[h] = -INFINITY;
    l_run[h] = 0.f;
  }

  for (;;) {
    int it = 0;
    for (int key0 = span_begin + warp * 16; key0 < span_end; key0 += kStep, ++it) {
      issue(key0 + (kRing - 1) * kStep, (it + kRing - 1) % kRing);
      asm volatile("cp.async.wait_group %0;" ::"n"(kRing - 1) : "memory");
      __syncwarp();
      const uint32_t st = ring + (uint32_t)((it % kRing) * STAGE);
      const int pi = (key0 >> shift) - page0;
      const float ks = page_ks[pi], vs = page_vs[pi];
      const bool good = page_id[pi] >= 0;

      // ---- S = Q K^T for 16 keys: this lane gets keys 8 nb + 2t, + 1 of rows g (and g + 8) ----
      float s_acc[2][4];
#pragma unroll
      for (int nb = 0; nb < 2; ++nb) {
#pragma unroll
        for (int c = 0; c < 4; ++c) s_acc[nb][c] = 0.f;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          const uint4 kw = lds_16(st + k_offset<D>(8 * nb + g, 4 * j + t));
          const uint32_t w[4] = {kw.x, kw.y, kw.z, kw.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t lo, hi;
            kv8_word_to_half<INT8>(w[i], lo, hi);
            if constexpr (ROWS == 8) {
              mma_16816<false>(s_acc[nb], qa[0][j][2 * i], REST ? qr[0][j][2 * i] : 0u, qa[0][j][2 * i + 1], REST ? qr[0][j][2 * i + 1] : 0u, lo, hi);
            } else {
              mma_16816<false>(s_acc[nb], qa[0][j][2 * i], qa[1][j][2 * i], qa[0][j][2 * i + 1], qa[1][j][2 * i + 1], lo, hi);
              if (REST) mma_16816<false>(s_acc[nb], qr[0][j][2 * i], qr[1][j][2 * i], qr[0][j][2 * i + 1], qr[1][j][2 * i + 1], lo, hi);
            }
          }
        }
      }

      // ---- running softmax ----
      float pv[G][2][2], corr[G];
      const float ref_new = fmaxf(v_ref, vs), share = ref_new > 0.f ? __fdividef(vs, ref_new) : 0.f;
      bool moved = ref_new != v_ref;
      const float ref_corr = ref_new > 0.f ? __fdividef(v_ref, ref_new) : 0.f;
#pragma unroll
      for (int h = 0; h < G; ++h) {
        float mx = -INFINITY;
#pragma unroll
        for (int nb = 0; nb < 2; ++nb)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float s = ROWS == 8 ? (REST ? s_acc[nb][c] + s_acc[nb][c + 2] : s_acc[nb][c]) : s_acc[nb][2 * h + c];
            s *= ks * row_scale[h];
            if (p.softcap != 0.f) s = p.softcap * tanhf(s / p.softcap);
            s *= kLog2e;
            if (!good || key0 + 8 * nb + 2 * t + c >= sees[h]) s = -INFINITY;
            pv[h][nb][c] = s;
            mx = fmaxf(mx, s);
          }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float m_new = fmaxf(m_run[h], mx), m_use = m_new == -INFINITY ? 0.f : m_new;
        moved |= m_new != m_run[h];
        corr[h] = exp2f(m_run[h] - m_use);
        m_run[h] = m_new;
        float sum = 0.f;
#pragma unroll
        for (int nb = 0; nb < 2; ++nb)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            pv[h][nb][c] = exp2f(pv[h][nb][c] - m_use);
            sum += pv[h][nb][c];
            pv[h][nb][c] *= share;
          }
        l_run[h] = l_run[h] * corr[h] + sum;
        corr[h] *= ref_corr;
      }
      v_ref = ref_new;
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int e = 0; e < NE; ++e) {
          o[e][0] *= corr[0]; o[e][1] *= corr[0];
          if (ROWS == 16 || REST) { o[e][2] *= corr[G - 1]; o[e][3] *= corr[G - 1]; }
        }
      }
      uint32_t pa[G][2], pr[G][2];                       // key slots 2t, 2t + 1 and 2t + 8, 2t + 9
#pragma unroll
      for (int h = 0; h < G; ++h)
#pragma unroll
        for (int nb = 0; nb < 2; ++nb) {
          pa[h][nb] = pack_half(pv[h][nb][0], pv[h][nb][1]);
          if (REST) {
            const float2 f = unpack_half(pa[h][nb]);
            pr[h][nb] = pack_half(pv[h][nb][0] - f.x, pv[h][nb][1] - f.y);
          }
        }

      // ---- O += P V: a lane holds d = NE g .. of keys 2t, 2t + 1, 2t + 8, 2t + 9 ----
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
#pragma unroll
      for (int w = 0; w < NE / 4; ++w) {
        uint32_t b0[4], b1[4];
        kv8_word_to_half<INT8>(__byte_perm(vw[0][w], vw[1][w], 0x5140), b0[0], b0[1]);
        kv8_word_to_half<INT8>(__byte_perm(vw[0][w], vw[1][w], 0x7362), b0[2], b0[3]);
        kv8_word_to_half<INT8>(__byte_perm(vw[2][w], vw[3][w], 0x5140), b1[0], b1[1]);
        kv8_word_to_half<INT8>(__byte_perm(vw[2][w], vw[3][w], 0x7362), b1[2], b1[3]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float(&acc)[4] = o[4 * w + e];
          if constexpr (ROWS == 8) {
            mma_16816<false>(acc, pa[0][0], REST ? pr[0][0] : 0u, pa[0][1], REST ? pr[0][1] : 0u, b0[e], b1[e]);
          } else {
            mma_16816<false>(acc, pa[0][0], pa[1][0], pa[0][1], pa[1][1], b0[e], b1[e]);
            if (REST) mma_16816<false>(acc, pr[0][0], pr[1][0], pr[0][1], pr[1][1], b0[e], b1[e]);
          }
        }
      }
    }

    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();                                     // the rings are idle, nobody reads the pages
    if (span_end >= key_end) break;
    span_begin = span_end;
    span_end = min(key_end, span_begin + kSpan);
    page0 = span_begin >> shift;
    load_pages();
    issue_first();
  }

  // ---- merge the warps ----
  constexpr int kPitch = D + 4;                        // (rows of the tile start in different banks)
  float* sm_o = reinterpret_cast<float*>(smem);        // [kWarps][ROWS][kPitch]
  float* sm_m = sm_o + kWarps * ROWS * kPitch;         // [kWarps][ROWS]
  float* sm_l = sm_m + kWarps * ROWS;
  float* cl_o = sm_l + kWarps * ROWS;                  // [ROWS][D] and [ROWS][2]: for the cluster's merge
  float* cl_ml = cl_o + ROWS * D;
#pragma unroll
  for (int h = 0; h < G; ++h) {
    l_run[h] += __shfl_xor_sync(0xffffffffu, l_run[h], 1);
    l_run[h] += __shfl_xor_sync(0xffffffffu, l_run[h], 2);
    const int r = h * 8 + g;
    if (t == 0) {
      sm_m[warp * ROWS + r] = m_run[h];
      sm_l[warp * ROWS + r] = l_run[h];
    }
    float* row = sm_o + (warp * ROWS + r) * kPitch;
#pragma unroll
    for (int e = 0; e < NE; ++e) {
      const float a = ROWS == 16 ? o[e][2 * h] : REST ? o[e][0] + o[e][2] : o[e][0];
      const float c = ROWS == 16 ? o[e][2 * h + 1] : REST ? o[e][1] + o[e][3] : o[e][1];
      row[NE * (2 * t) + e] = a * v_ref;
      row[NE * (2 * t + 1) + e] = c * v_ref;
    }
  }
  __syncthreads();
  const int here = min(ROWS, rows - tile * ROWS);      // rows of this tile
  auto out_row = [&](int r) -> int64_t {
    const int rr = tile * ROWS + r, s = rr / rep;
    return ((int64_t)b * p.Sq + s) * p.Hq + hkv * rep + (rr - s * rep);
  };
  for (int i = tid; i < here * D; i += kThreads) {
    const int r = i / D, dd = i - r * D;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) M = fmaxf(M, sm_m[w * ROWS + r]);
    float lsum = 0.f, osum = 0.f;
    if (M > -INFINITY) {
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float f = exp2f(sm_m[w * ROWS + r] - M);
        lsum += sm_l[w * ROWS + r] * f;
        osum += sm_o[(w * ROWS + r) * kPitch + dd] * f;
      }
    }
    if (p.cluster > 1) {
      cl_o[i] = osum;
      if (dd == 0) {
        cl_ml[2 * r] = M;
        cl_ml[2 * r + 1] = lsum;
      }
    } else if (n_splits == 1) {
      p.out[out_row(r) * D + dd] = round_bits<BF16>(lsum > 0.f ? osum / lsum : 0.f);
    } else {
      const int64_t slot = out_row(r) * p.splits + split;
      p.part_o[slot * D + dd] = osum;
      if (dd == 0) {
        p.part_ml[2 * slot] = M;
        p.part_ml[2 * slot + 1] = lsum;
      }
    }
  }
  if (p.cluster > 1) {
    cluster_arrive();
    cluster_wait();
    const uint32_t lo = (uint32_t)__cvta_generic_to_shared(cl_o), lml = (uint32_t)__cvta_generic_to_shared(cl_ml);
    for (int i = split * kThreads + tid; i < here * D; i += p.cluster * kThreads) {
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
      p.out[out_row(r) * D + dd] = round_bits<BF16>(lsum > 0.f ? osum / lsum : 0.f);
    }
    cluster_arrive();                                  // nobody leaves while a peer may still read its partial
    cluster_wait();
  }
}

// Merge of the splits that the workspace holds: a thread adds up four neighbouring outputs.
template <bool BF16, int D>
__global__ void __launch_bounds__(128) attn_decode_kv8_merge_kernel(const Kv8Args p) {
  pdl_wait_then_trigger();
  const int b = blockIdx.y, u = blockIdx.x * 128 + threadIdx.x, units = p.Sq * p.Hq * (D / 4);
  const int n_splits = (max(0, min(p.seqlens[b], p.max_len)) + p.chunk - 1) / p.chunk;
  if (n_splits <= 1 || u >= units) return;             // (one split: the result is there)
  const int64_t row = (int64_t)b * p.Sq * p.Hq + u / (D / 4);
  const int dd = u % (D / 4) * 4;
  float M = -INFINITY, lsum = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = 0; s < n_splits; ++s) {                 // in split order
    const int64_t slot = row * p.splits + s;
    const float2 ml = __ldcg(reinterpret_cast<const float2*>(p.part_ml + 2 * slot));
    const float4 a = __ldcg(reinterpret_cast<const float4*>(p.part_o + slot * D + dd));
    const float Mn = fmaxf(M, ml.x);
    const float keep = M > -INFINITY ? exp2f(M - Mn) : 0.f, f = ml.x > -INFINITY ? exp2f(ml.x - Mn) : 0.f;
    M = Mn;
    lsum = lsum * keep + ml.y * f;
    o[0] = o[0] * keep + a.x * f; o[1] = o[1] * keep + a.y * f;
    o[2] = o[2] * keep + a.z * f; o[3] = o[3] * keep + a.w * f;
  }
  uint16_t e[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) e[j] = round_bits<BF16>(lsum > 0.f ? o[j] / lsum : 0.f);
  *reinterpret_cast<uint2*>(p.out + row * D + dd) = make_uint2(e[0] | ((uint32_t)e[1] << 16), e[2] | ((uint32_t)e[3] << 16));
}

template <int D> constexpr int kv8_smem() { return kWarps * kRing * 2 * 16 * D; }

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
  constexpr int smem = kv8_smem<D>();
  static_assert(smem >= (kWarps * ROWS * (D + 4 + 2) + ROWS * (D + 2)) * 4, "the rings hold the merge tile");
  auto kern = attn_decode_kv8_kernel<D, INT8, BF16, ROWS>;
  a.tiles = (int)ceil_div((int64_t)a.Sq * (a.Hq / a.Hkv), ROWS);
  const int64_t blocks = (int64_t)B * a.Hkv * a.tiles, slots = 2 * (int64_t)sm_count();
  const int most = a.max_len > 0 ? a.max_len : 1;
  int chunk = kStep;
  while (chunk < most && blocks * ceil_div(most, chunk) > slots) chunk *= 2;
  if (chunk > 2048 && most > 4096) chunk = 2048;       // (ragged lengths: the longest sequence would run alone at the end)
  int splits = (int)ceil_div(most, chunk);
  a.cluster = 1;
  if (splits > 1 && (splits <= 8 || most <= kClusterMergeMaxLen)) {
    const int c = splits < 8 ? splits : 8;
    if (blocks <= max_active_clusters(reinterpret_cast<const void*>(kern), c, smem)) {
      a.cluster = splits = c;
      chunk = (int)ceil_div(ceil_div(most, c), kStep) * kStep;
    }
  }
  const size_t rows = (size_t)B * a.Sq * a.Hq;
  while (a.cluster == 1 && splits > 1 && rows * splits * (D + 2) * 4 > LLMQRT_WS_PARTIAL_BYTES) {
    chunk *= 2;
    splits = (int)ceil_div(most, chunk);
  }
  a.chunk = chunk;
  a.splits = splits;
  if (splits > 1 && a.cluster == 1) {
    if (!workspace) return set_error(LLMQRT_ERR_WORKSPACE, "attn_decode_kv8: split keys need the workspace");
    a.part_o = reinterpret_cast<float*>(ws_partials(workspace));
    a.part_ml = a.part_o + rows * splits * D;
  }
  if (int rc = ensure_dynamic_smem(reinterpret_cast<const void*>(kern), smem)) return rc;
  if (int rc = launch_chained(kern, dim3((unsigned)splits, (unsigned)(a.Hkv * a.tiles), (unsigned)B), dim3(kThreads), smem, st, a.cluster, a))
    return rc;
  if (int rc = check_launch("attn_decode_kv8")) return rc;
  if (splits == 1 || a.cluster > 1) return LLMQRT_OK;
  const int units = a.Sq * a.Hq * (D / 4);
  if (int rc = launch_chained(attn_decode_kv8_merge_kernel<BF16, D>, dim3((unsigned)ceil_div(units, 128), (unsigned)B), dim3(128), 0, st, 1, a))
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
  LLMQRT_REQUIRE(most <= 0x7ffffff0ll, "attn_decode_kv8: sequences too long");
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
