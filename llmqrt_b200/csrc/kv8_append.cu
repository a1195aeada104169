// New keys and values into a paged 8-bit cache.
//
// The new tokens of a page are a run: consecutive tokens of the call whose slots follow one another within the page.  For
// each run and head, with a the run's greatest magnitude and s0 the page's scale if the page holds rows ahead of the run:
//   s1 = max(s0, scale(a));   rows ahead: code <- code * (s0 / s1) rounded, where s1 is greater;   new: code = x / s1 rounded.
// A page's scale thus only grows while it fills, and a page whose first row is written starts afresh.  Rows behind the run
// stay as they were.  Keys are rotated first, if tables are given; nothing is rounded in between.
//
// A team of warps does one run of one head, of the keys or of the values: eight lanes (d = 64: four) hold a row, sixteen elements
// each -- eight and the eight half a head away, the rotation's pairs.  The first rows (four a lane where teams share a run) are asked
// for before the run's length is known and stay in registers as they came; those behind them are read once for the maximum and
// again (from L1) for their codes.  Nobody else touches these codes or their scale, so there are no atomics and the result is the same
// on every run.
//
// A block looks for runs in a window of the call's tokens, one window for each head, keys and values.  A decode step's tokens are runs
// of their own: a warp each, four to a window (a run that is alone in its window gets all four).  Of many tokens a window has 32, and the block's two warps (four, where pages hold 64 or
// more) take each run together.
//
// Bound by its chain of loads (slots, rows and positions, angles; 18 warps an SM) and 17 instructions an element, at half of what the
// schedulers could issue: 17600 tokens of 4 heads of 128 take 17 us with their rows in L2 and 21 without, 58 MB at 2.7 TB/s of 6.5.
// (A warp a run: 33 us; four warps: 18 and 24; eight: 26, as what a run costs before its rows is paid by each of them.
// Pages of 128, 8 heads: four warps 39 us, two 46; pages of 64, 3000 tokens: 8 and 11. 1800 tokens of two prompts: 5.3, a warp a run 9.6.  A block that goes over all heads of a run with the
// next ones' rows on their way: 19.6 and 22.5.)
#include "kv8.cuh"

namespace llmqrt {
namespace {

constexpr int kWarps = 4;                              // a warp a run

struct AppendArgs {
  uint8_t* cache[2];               // keys, values: [pages, Hkv, page, d]
  float* scale[2];                 // [pages, Hkv]
  const void* fresh[2];            // [T, Hkv, d], heads and d contiguous
  int64_t token_stride[2];
  int64_t page_stride, head_stride;
  const int64_t* slots;            // [T]
  const float* cos_tab;            // [table_rows, d / 2] or null
  const float* sin_tab;
  const int32_t* positions;        // [T]
  int64_t num_slots;               // pages * page
  int T, Hkv, page, table_rows, window;
};

// TEAM: warps that share a run, all of the block's; 1: a warp a run, where the window has one alone all four.
template <typename T, int D, bool INT8, int TEAM>
__global__ void __launch_bounds__(TEAM > 1 ? TEAM * 32 : kWarps * 32, TEAM > 1 ? 20 / TEAM : 5) kv8_append_kernel(AppendArgs p) {
  constexpr int kLanes = D / 16, kBlockWarps = TEAM > 1 ? TEAM : kWarps;      // lanes of a row
  __shared__ float tops[2][kBlockWarps];
  pdl_wait_then_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, head = blockIdx.y, kind = blockIdx.z;
  const int piece = lane % kLanes;
  const int w0 = blockIdx.x * p.window, w1 = min(p.T, w0 + p.window);
  const int shift = __ffs(p.page) - 1;
  // the runs that begin in the window: one bit a token (a window has at most 32)
  bool begins = false;
  if (w0 + lane < w1) {
    const int64_t s = p.slots[w0 + lane], before = w0 + lane > 0 ? p.slots[w0 + lane - 1] : -2;
    begins = s >= 0 && s < p.num_slots && !(before + 1 == s && (s & (p.page - 1)) != 0);
  }
  unsigned runs = __ballot_sync(0xffffffffu, begins);
  const bool together = TEAM > 1 || __popc(runs) == 1;
  const int sub = lane / kLanes + (together ? warp * (32 / kLanes) : 0), rows = 32 / kLanes * (together ? kBlockWarps : 1);      // taken at once
  for (int nth = 0; runs; runs &= runs - 1, ++nth) {
    if (!together && nth % kWarps != warp) continue;
    const int t0 = w0 + __ffs(runs) - 1;
    const int64_t s0 = p.slots[t0];
    const int row0 = (int)(s0 & (p.page - 1));
    const int64_t page = s0 >> shift;
    uint8_t* tile = p.cache[kind] + page * p.page_stride + (int64_t)head * p.head_stride;
    float* scale = p.scale[kind] + page * p.Hkv + head;
    const bool rotated = kind == 0 && p.cos_tab != nullptr;
    auto load = [&](int i, bool on, uint4& lo, uint4& hi, int& at) {
      const T* src = static_cast<const T*>(p.fresh[kind]) + (int64_t)(t0 + i) * p.token_stride[kind] + head * D + piece * 8;
      lo = on ? *reinterpret_cast<const uint4*>(src) : make_uint4(0, 0, 0, 0);
      hi = on ? *reinterpret_cast<const uint4*>(src + D / 2) : make_uint4(0, 0, 0, 0);
      at = on && rotated ? p.positions[t0 + i] : -1;
    };
    auto turn = [&](const uint4& lo, const uint4& hi, int at, float (&x)[16]) {
      const uint32_t a[4] = {lo.x, lo.y, lo.z, lo.w}, b[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = unpack_pair<T>(a[j]), g = unpack_pair<T>(b[j]);
        x[2 * j] = f.x; x[2 * j + 1] = f.y;
        x[8 + 2 * j] = g.x; x[8 + 2 * j + 1] = g.y;
      }
      if (at >= 0 && at < p.table_rows) {              // (outside the table: not rotated)
        const float* cr = p.cos_tab + (int64_t)at * (D / 2) + piece * 8;
        const float* sr = p.sin_tab + (int64_t)at * (D / 2) + piece * 8;
#pragma unroll
        for (int j = 0; j < 8; j += 4) {
          const float4 c = *reinterpret_cast<const float4*>(cr + j), s = *reinterpret_cast<const float4*>(sr + j);
          const float cs[4] = {c.x, c.y, c.z, c.w}, sn[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {                // (two products and their sum, each rounded: no contraction)
            const float u = x[j + e], v = x[8 + j + e];
            x[j + e] = __fsub_rn(__fmul_rn(u, cs[e]), __fmul_rn(v, sn[e]));
            x[8 + j + e] = __fadd_rn(__fmul_rn(u, sn[e]), __fmul_rn(v, cs[e]));
          }
        }
      }
    };
    auto fetch = [&](int i, float (&x)[16]) {
      uint4 lo, hi;
      int at;
      load(i, true, lo, hi, at);
      turn(lo, hi, at, x);
    };
    // The first rows are asked for before the run's length is known, and kept.
    constexpr int kKeep = TEAM == 1 ? 2 : 4;
    const int most = min(p.page - row0, p.T - t0);
    const float was = row0 > 0 ? *scale : 0.f;
    uint4 lo[kKeep], hi[kKeep];
    int at[kKeep];
#pragma unroll
    for (int k = 0; k < kKeep; ++k) load(sub + k * rows, sub + k * rows < most, lo[k], hi[k], at[k]);
    // length of the run: to the end of the page, or as far as the slots follow one another
    int n = 1;
    while (n < most) {
      const int i = n + lane;
      const bool on = i < most && p.slots[t0 + i] == s0 + i;
      const unsigned gap = ~__ballot_sync(0xffffffffu, on);
      n += gap ? __ffs(gap) - 1 : 32;
      if (gap) break;
    }
    float top = 0.f;
#pragma unroll
    for (int k = 0; k < kKeep; ++k) {
      if (sub + k * rows >= n) continue;
      float x[16];
      turn(lo[k], hi[k], at[k], x);
#pragma unroll
      for (int j = 0; j < 16; ++j) top = fmaxf(top, fabsf(x[j]));
    }
#pragma unroll 2
    for (int i = sub + kKeep * rows; i < n; i += rows) {
      float x[16];
      fetch(i, x);
#pragma unroll
      for (int j = 0; j < 16; ++j) top = fmaxf(top, fabsf(x[j]));
    }
    top = warp_max(top);
    if (together) {                                    // (two sets in turn: one barrier a run is enough, and none reads the old scale behind it)
      if (lane == 0) tops[nth & 1][warp] = top;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kBlockWarps; ++w) top = fmaxf(top, tops[nth & 1][w]);
    }
    const float now = fmaxf(was, kv8_scale<INT8>(top)), inv = __fdiv_rn(1.f, now);
    // lane `piece` of a row holds elements 8 piece .. + 7 and D / 2 further: two 8-byte stores
    auto store = [&](int i, const float (&x)[16]) {
      const uint4 c = kv8_encode<INT8>(x, inv);
      uint8_t* dst = tile + (int64_t)(row0 + i) * D + piece * 8;
      *reinterpret_cast<uint2*>(dst) = make_uint2(c.x, c.y);
      *reinterpret_cast<uint2*>(dst + D / 2) = make_uint2(c.z, c.w);
    };
#pragma unroll
    for (int k = 0; k < kKeep; ++k)
      if (sub + k * rows < n) {                       // (turned once more: as fp32 they would take twice the registers)
        float x[16];
        turn(lo[k], hi[k], at[k], x);
        store(sub + k * rows, x);
      }
    for (int i = sub + kKeep * rows; i < n; i += rows) {
      float x[16];
      fetch(i, x);
      store(i, x);
    }
    if (now != was) {
      if (row0 > 0) {
        const float ratio = __fdiv_rn(was, now);
        for (int i = sub; i < row0; i += rows) {
          uint8_t* at = tile + (int64_t)i * D + piece * 16;
          float x[16];
          kv8_decode<INT8>(*reinterpret_cast<const uint4*>(at), x);
          *reinterpret_cast<uint4*>(at) = kv8_encode<INT8>(x, ratio);
        }
      }
      __syncwarp();                                    // (every lane has read the old scale)
      if (together ? threadIdx.x == 0 : lane == 0) *scale = now;
    }
  }
}

}  // namespace
}  // namespace llmqrt

using namespace llmqrt;

extern "C" int llmqrt_kv8_append(void* k_cache, void* v_cache, float* k_scale, float* v_scale, int cache_type, int64_t page_stride,
                                 int64_t head_stride, const void* k, int64_t k_token_stride, const void* v, int64_t v_token_stride,
                                 int dtype, const int64_t* slots, const float* cos_table, const float* sin_table, int64_t table_rows,
                                 const int32_t* positions, int64_t T, int64_t pages, int64_t page, int64_t Hkv, int64_t d,
                                 llmqrt_stream_t stream) {
  LLMQRT_REQUIRE(dtype == LLMQRT_F16 || dtype == LLMQRT_BF16, "kv8_append: dtype must be fp16 or bf16");
  LLMQRT_REQUIRE(cache_type == LLMQRT_E4M3 || cache_type == LLMQRT_I8, "kv8_append: the cache holds e4m3 or int8");
  LLMQRT_REQUIRE(d == 64 || d == 128, "kv8_append: head_dim must be 64 or 128 (got %lld)", (long long)d);
  LLMQRT_REQUIRE(page >= 16 && page <= 128 && (page & (page - 1)) == 0, "kv8_append: pages hold 16, 32, 64 or 128 tokens (got %lld)",
                 (long long)page);
  LLMQRT_REQUIRE(T >= 0 && T <= 0x7fffff00ll && Hkv > 0 && Hkv < 65536 && pages >= 0 && pages <= 0x7fffffffll, "kv8_append: bad shape");
  LLMQRT_REQUIRE(head_stride >= page * d && page_stride >= Hkv * head_stride && head_stride % 16 == 0 && page_stride % 16 == 0,
                 "kv8_append: the cache is [pages, Hkv, page, d] with contiguous pages, strides multiples of 16");
  LLMQRT_REQUIRE((cos_table == nullptr) == (sin_table == nullptr) && (!cos_table || positions || T == 0),
                 "kv8_append: cos, sin and positions go together");
  if (T == 0 || pages == 0) return LLMQRT_OK;
  LLMQRT_REQUIRE(k_cache && v_cache && k_scale && v_scale && k && v && slots, "kv8_append: null pointer");
  LLMQRT_REQUIRE(k_token_stride >= Hkv * d && v_token_stride >= Hkv * d && k_token_stride % 8 == 0 && v_token_stride % 8 == 0 &&
                 ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(k_cache) |
                   reinterpret_cast<uintptr_t>(v_cache)) & 15) == 0, "kv8_append: rows and caches must be 16-byte aligned");
  LLMQRT_REQUIRE(!cos_table || (table_rows > 0 && table_rows <= 0x7fffffffll &&
                                ((reinterpret_cast<uintptr_t>(cos_table) | reinterpret_cast<uintptr_t>(sin_table)) & 15) == 0),
                 "kv8_append: rotary tables must be 16-byte aligned fp32 [table_rows, d/2]");
  AppendArgs a{};
  a.cache[0] = static_cast<uint8_t*>(k_cache); a.cache[1] = static_cast<uint8_t*>(v_cache);
  a.scale[0] = k_scale; a.scale[1] = v_scale;
  a.fresh[0] = k; a.fresh[1] = v;
  a.token_stride[0] = k_token_stride; a.token_stride[1] = v_token_stride;
  a.page_stride = page_stride; a.head_stride = head_stride;
  a.slots = slots; a.cos_tab = cos_table; a.sin_tab = sin_table; a.positions = positions;
  a.num_slots = pages * page;
  a.T = (int)T; a.Hkv = (int)Hkv; a.page = (int)page; a.table_rows = (int)table_rows;
  // (64 tokens of a decode step: 2.6 us with a warp each)
  const int team = T <= 2048 ? 0 : page >= 64 ? 4 : 2;
  a.window = team ? 32 : kWarps;
  const dim3 grid((unsigned)ceil_div(T, a.window), (unsigned)Hkv, 2);
  auto go = [&](auto kern) { return launch_chained(kern, grid, dim3(team ? (unsigned)team * 32 : kWarps * 32), 0, (cudaStream_t)stream, 1, a); };
  const bool i8 = cache_type == LLMQRT_I8;
  auto pick = [&](auto tag) {
    using T_ = decltype(tag);
#define LLMQRT_APPEND(D_, I_) (team == 4 ? go(kv8_append_kernel<T_, D_, I_, 4>) : team == 2 ? go(kv8_append_kernel<T_, D_, I_, 2>) : go(kv8_append_kernel<T_, D_, I_, 1>))
    return d == 128 ? (i8 ? LLMQRT_APPEND(128, true) : LLMQRT_APPEND(128, false)) : (i8 ? LLMQRT_APPEND(64, true) : LLMQRT_APPEND(64, false));
#undef LLMQRT_APPEND
  };
  if (int rc = dtype == LLMQRT_F16 ? pick(__half()) : pick(__nv_bfloat16())) return rc;
  return check_launch("kv8_append");
}
