// Pages and slots of a serving step, from the requests' lengths, on the GPU.
//
// Request b holds context[b] tokens in ceil(context[b] / page) pages, named by the first entries of its row of the block
// table, and is to get new[b] more.  The pages that this takes come from the top of a stack of free page numbers, in the
// order of the requests; then every new token has a slot, page number * page + row, and a position.
//
// Latency-bound (a step of 64 requests touches 3 KB): one launch.  Each block adds up all requests for itself -- tokens and pages at
// once, the pages again where the first sum turns a request down -- and keeps the sums in shared memory; tokens and pages are then
// dealt out, each finding its request by bisection.  The stack's count and the lengths may be updated in place: the last block to
// have read them writes them.
// On the GPU 3.5 us for 64 requests of one token (four warps, which wait for one another less than sixteen: 5.6), 5.4 us for 131072
// tokens of 333 requests, 128 blocks (a cluster of eight, which the instructions of a token bound: 13 us), 16.5 us for 8192 requests.
#include <algorithm>

#include "common.cuh"

namespace llmqrt {
namespace {

constexpr int kPlanThreads = 512;
constexpr int kPlanMaxRequests = 8192;                 // three words each in shared memory

struct PlanArgs {
  const int32_t* context;          // [B]
  const int32_t* fresh;            // [B] new tokens
  int32_t* table;                  // [B, width] with row stride table_stride
  int64_t table_stride;
  const int32_t* free_pages;       // [pool]
  const int32_t* free_count;       // [1]
  int32_t* free_left;              // [1], may be free_count
  int32_t* seq;                    // [B], may be context
  int32_t* cu;                     // [B + 1]
  int64_t* slots;                  // [max_tokens]
  int32_t* positions;              // [max_tokens]
  int* counter;                    // zero between calls; with several blocks
  int B, width, pool, page, max_tokens;
};

// Exclusive sums over the block's threads in thread order, of two values at once; the totals come back beside them.
template <int THREADS> __device__ __forceinline__ void block_exclusive_sums(int64_t a, int64_t b, longlong2* warp_sums, longlong2& before, longlong2& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t s = a, r = b;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t m = __shfl_up_sync(0xffffffffu, s, o), n = __shfl_up_sync(0xffffffffu, r, o);
    if (lane >= o) {
      s += m;
      r += n;
    }
  }
  if (lane == 31) warp_sums[warp] = make_longlong2(s, r);
  __syncthreads();
  before = make_longlong2(s - a, r - b);
  total = make_longlong2(0, 0);
  if constexpr (THREADS <= 128) {
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
      const longlong2 v = warp_sums[w];
      if (w < warp) {
        before.x += v.x;
        before.y += v.y;
      }
      total.x += v.x;
      total.y += v.y;
    }
  } else {                                             // (32 words one after the other: 4 us with 32 warps at it)
    longlong2 v = lane < THREADS / 32 ? warp_sums[lane] : make_longlong2(0, 0);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t m = __shfl_up_sync(0xffffffffu, v.x, o), n = __shfl_up_sync(0xffffffffu, v.y, o);
      if (lane >= o) {
        v.x += m;
        v.y += n;
      }
    }
    total = make_longlong2(__shfl_sync(0xffffffffu, v.x, 31), __shfl_sync(0xffffffffu, v.y, 31));
    const int64_t m = __shfl_sync(0xffffffffu, v.x, (warp + 31) & 31), n = __shfl_sync(0xffffffffu, v.y, (warp + 31) & 31);
    if (warp > 0) {
      before.x += m;
      before.y += n;
    }
  }
  __syncthreads();                                     // (the words may be used again)
}

// EACH: neighbouring requests that a thread adds up; THREADS * EACH >= B.
template <int THREADS, int EACH> __global__ void __launch_bounds__(THREADS) plan_step_kernel(PlanArgs p) {
  extern __shared__ int32_t plan_smem[];
  __shared__ longlong2 warp_sums[THREADS / 32];
  int32_t* cu_s = plan_smem;                           // [B] first token of the request
  int32_t* ctx_s = cu_s + p.B;                         // [B] its context; one that gets nothing: ~context
  int32_t* off_s = ctx_s + p.B;                        // [B] its first new page's place below the stack's top (pages wanted before it)
  const int cl = gridDim.x, rank = blockIdx.x, shift = __ffs(p.page) - 1;
  pdl_wait_then_trigger();
  const int64_t count = min(max(*p.free_count, 0), p.pool);
  __shared__ int32_t taken;
  if (threadIdx.x == 0) taken = 0;
  __syncthreads();
  const int b1 = (int)threadIdx.x * EACH;
  int ctx[EACH], n[EACH];
#pragma unroll
  for (int j = 0; j < EACH; ++j) {
    ctx[j] = b1 + j < p.B ? max(p.context[b1 + j], 0) : 0;
    n[j] = b1 + j < p.B ? max(p.fresh[b1 + j], 0) : 0;
  }
  // pages that a request takes; -1: more than its row of the table has
  auto pages_of = [&](int j) {
    const int64_t have = ((int64_t)ctx[j] + p.page - 1) >> shift, all = ((int64_t)ctx[j] + n[j] + p.page - 1) >> shift;
    return all <= p.width ? (int)(all - have) : -1;
  };
  int64_t my_tokens = 0, my_pages = 0;
#pragma unroll
  for (int j = 0; j < EACH; ++j) {
    my_tokens += n[j];
    my_pages += max(pages_of(j), 0);
  }
  // (where no request is turned down for its tokens, the pages' sum need not wait for the tokens')
  longlong2 before, sum;
  block_exclusive_sums<THREADS>(my_tokens, my_pages, warp_sums, before, sum);
  const int64_t tokens = sum.x;
  int64_t cu = before.x, off = before.y;
  if (tokens > p.max_tokens) {
    my_pages = 0;
    int64_t end = cu;
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
      end += n[j];
      if (end <= p.max_tokens) my_pages += max(pages_of(j), 0);
    }
    longlong2 before_again, sum_again;
    block_exclusive_sums<THREADS>(my_pages, 0, warp_sums, before_again, sum_again);
    off = before_again.x;
  }
#pragma unroll
  for (int j = 0; j < EACH; ++j) {
    const int pages = pages_of(j);
    bool fits = pages >= 0 && cu + n[j] <= p.max_tokens;
    const int64_t need = fits ? pages : 0;
    fits = fits && (need == 0 || off + need <= count);
    // (the requests that get pages are the first ones that want any: their pages are the stack's topmost)
    if (fits && need) atomicMax(&taken, (int32_t)(off + need));
    if (b1 + j < p.B) {
      cu_s[b1 + j] = (int32_t)min(cu, (int64_t)0x7fffffff);
      ctx_s[b1 + j] = fits ? ctx[j] : ~ctx[j];
      off_s[b1 + j] = (int32_t)min(off, (int64_t)0x7fffffff);
    }
    cu += n[j];
    off += need;
  }
  __syncthreads();
  bool last = cl == 1;
  if (cl > 1) {
    if (threadIdx.x == 0) {
      int before;
      asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;" : "=r"(before) : "l"(p.counter) : "memory");
      last = before == cl - 1;
      if (last) *p.counter = 0;                        // as the next call wants it
    }
    last = __syncthreads_or(last);
  }
  if (last) {                                          // every block has read the lengths and the count
    for (int b = threadIdx.x; b < p.B; b += THREADS) {
      const int32_t next = b + 1 < p.B ? cu_s[b + 1] : (int32_t)min(tokens, (int64_t)0x7fffffff);
      p.cu[b + 1] = next;
      p.seq[b] = ctx_s[b] >= 0 ? ctx_s[b] + next - cu_s[b] : ~ctx_s[b];
    }
    if (threadIdx.x == 0) {
      p.cu[0] = 0;
      *p.free_left = (int32_t)(count - taken);
    }
  }
  const int lane = threadIdx.x & 31, warps = cl * (THREADS / 32);
  // The last request, from lo on, whose first token, or page, is at most i: strides that double, then bisection.
  auto last_at_most = [&](const int32_t* first, int64_t i, int lo) {
    int hi = p.B;
    for (int step = 1; lo + step < p.B; step *= 2) {
      if (first[lo + step] > i) {
        hi = lo + step;
        break;
      }
      lo += step;
    }
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (first[mid] <= i) lo = mid;
      else hi = mid;
    }
    return lo;
  };
  // A warp has consecutive tokens, 32 kBatch at a time: a lane looks for each one's request from the last one's on, and kBatch look-ups are
  // under way at once.
  constexpr int kBatch = 4;
  const int64_t all_tokens = min(tokens, (int64_t)p.max_tokens);
  const int64_t each = ((int64_t)p.max_tokens + warps * 32 - 1) / (warps * 32) * 32;
  const int64_t begin = (rank * (THREADS / 32) + (threadIdx.x >> 5)) * each, end = min(begin + each, (int64_t)p.max_tokens);
  int lo = 0;
  for (int64_t t0 = begin + lane; t0 < end; t0 += 32 * kBatch) {
    int32_t position[kBatch];
    int id[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int64_t t = t0 + 32 * i;
      position[i] = 0;
      id[i] = -1;
      if (t < all_tokens) {
        lo = last_at_most(cu_s, t, lo);
        const int ctx = ctx_s[lo];
        if (ctx >= 0) {
          position[i] = ctx + (int32_t)(t - cu_s[lo]);
          const int have = (int)(((int64_t)ctx + p.page - 1) >> shift), j = position[i] >> shift;
          // (a page taken in this step is read from the stack: another block may write the table's entry)
          id[i] = j < have ? p.table[(int64_t)lo * p.table_stride + j] : p.free_pages[count - 1 - off_s[lo] - (j - have)];
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int64_t t = t0 + 32 * i;
      if (t < end) {
        p.slots[t] = id[i] >= 0 ? ((int64_t)id[i] << shift) + (position[i] & (p.page - 1)) : -1;
        p.positions[t] = position[i];
      }
    }
  }
  for (int i = rank * THREADS + threadIdx.x; i < taken; i += cl * THREADS) {
    const int b = last_at_most(off_s, i, 0), have = (int)(((int64_t)ctx_s[b] + p.page - 1) >> shift);
    p.table[(int64_t)b * p.table_stride + have + i - off_s[b]] = p.free_pages[count - 1 - i];
  }
}

// Pages of the requests that `done` marks go back onto the stack, in the order of the requests and of their rows, and
// their lengths become zero.  One block: a step releases a few requests.
__global__ void __launch_bounds__(kPlanThreads)
release_kernel(const uint8_t* __restrict__ done, int32_t* __restrict__ lens, const int32_t* __restrict__ table,
               int64_t table_stride, int32_t* __restrict__ free_pages, int32_t* __restrict__ free_count, int B, int width, int pool,
               int page) {
  __shared__ longlong2 warp_sums[kPlanThreads / 32];
  __shared__ int32_t first[kPlanThreads];
  __shared__ int32_t pages[kPlanThreads];
  pdl_wait_then_trigger();
  const int shift = __ffs(page) - 1;
  int64_t count = min(max(*free_count, 0), pool);
  for (int b0 = 0; b0 < B; b0 += kPlanThreads) {
    const int b = b0 + threadIdx.x;
    const bool go = b < B && done[b] != 0;
    const int64_t n = go ? min((int64_t)(((int64_t)max(lens[b], 0) + page - 1) >> shift), (int64_t)width) : 0;
    longlong2 before, sum;
    block_exclusive_sums<kPlanThreads>(n, 0, warp_sums, before, sum);
    const int64_t at = count + before.x;
    first[threadIdx.x] = (int32_t)min(at, (int64_t)pool);
    pages[threadIdx.x] = (int32_t)n;
    if (go) lens[b] = 0;
    count = min(count + (int64_t)sum.x, (int64_t)pool);
    __syncthreads();
    for (int r = threadIdx.x >> 5; r < min(kPlanThreads, B - b0); r += kPlanThreads / 32)
      for (int j = threadIdx.x & 31; j < pages[r]; j += 32)
        if (first[r] + j < pool) free_pages[first[r] + j] = table[(int64_t)(b0 + r) * table_stride + j];
    __syncthreads();
  }
  if (threadIdx.x == 0) *free_count = (int32_t)count;
}

int check_table(const char* what, const void* table, int64_t table_stride, const void* free_pages, const void* free_count, int64_t B,
                int64_t width, int64_t pool, int64_t page) {
  LLMQRT_REQUIRE(page >= 16 && page <= 128 && (page & (page - 1)) == 0, "%s: pages hold 16, 32, 64 or 128 tokens (got %lld)", what,
                 (long long)page);
  LLMQRT_REQUIRE(B >= 0 && B <= kPlanMaxRequests, "%s: at most %d requests (got %lld)", what, kPlanMaxRequests, (long long)B);
  LLMQRT_REQUIRE(width >= 0 && pool >= 0 && width * page <= 0x7fffffffll && pool <= 0x7fffffffll && table_stride >= width,
                 "%s: bad table or pool", what);
  LLMQRT_REQUIRE(free_count && (free_pages || pool == 0) && (table || B == 0 || width == 0), "%s: null pointer", what);
  return LLMQRT_OK;
}

}  // namespace
}  // namespace llmqrt

using namespace llmqrt;

extern "C" {

int llmqrt_plan_step(const int32_t* context, const int32_t* new_tokens, int32_t* block_table, int64_t table_stride,
                     const int32_t* free_pages, const int32_t* free_count, int32_t* free_left, int32_t* seq_lens, int32_t* cu_new,
                     int64_t* slots, int32_t* positions, int64_t B, int64_t width, int64_t pool, int64_t page, int64_t max_tokens,
                     void* workspace, llmqrt_stream_t stream) {
  if (int rc = check_table("plan_step", block_table, table_stride, free_pages, free_count, B, width, pool, page)) return rc;
  LLMQRT_REQUIRE(max_tokens >= 0 && max_tokens < 0x7fffffffll, "plan_step: bad max_tokens");
  LLMQRT_REQUIRE(free_left && cu_new && (B == 0 || (context && new_tokens && seq_lens)) && (max_tokens == 0 || (slots && positions)),
                 "plan_step: null pointer");
  // (a decode step wants few warps that wait for one another, a large one many look-ups under way)
  const bool few = max_tokens <= 256 && B <= 128;
  const int blocks = few ? 1 : (int)std::min<int64_t>(128, std::max<int64_t>(1, ceil_div(std::max(max_tokens, 4 * B), 1024)));
  LLMQRT_REQUIRE(blocks == 1 || workspace, "plan_step: null workspace");
  PlanArgs p{context, new_tokens, block_table, table_stride, free_pages, free_count, free_left, seq_lens, cu_new, slots, positions,
             blocks > 1 ? ws_counters(workspace) + LLMQRT_WS_NUM_COUNTERS - 1 : nullptr, (int)B, (int)width, (int)pool, (int)page, (int)max_tokens};
  const int smem = (int)(3 * 4 * B), threads = few ? 128 : B <= 512 ? 512 : 1024;
  // (8192 requests of one token: 16.5 us with eight a thread, 36 in eight rounds)
  static_assert(1024 * 8 >= kPlanMaxRequests, "one round of a block");
  auto kern = few ? plan_step_kernel<128, 1> : B <= 512 ? plan_step_kernel<512, 1> : B <= 1024 ? plan_step_kernel<1024, 1> : plan_step_kernel<1024, 8>;
  if (int rc = ensure_dynamic_smem(reinterpret_cast<const void*>(kern), smem)) return rc;
  if (int rc = launch_chained(kern, dim3((unsigned)blocks), dim3((unsigned)threads), (size_t)smem, (cudaStream_t)stream, 1, p)) return rc;
  return check_launch("plan_step");
}

int llmqrt_release_pages(const uint8_t* done, int32_t* lens, const int32_t* block_table, int64_t table_stride, int32_t* free_pages,
                         int32_t* free_count, int64_t B, int64_t width, int64_t pool, int64_t page, llmqrt_stream_t stream) {
  if (int rc = check_table("release_pages", block_table, table_stride, free_pages, free_count, B, width, pool, page)) return rc;
  if (B == 0) return LLMQRT_OK;
  LLMQRT_REQUIRE(done && lens, "release_pages: null pointer");
  if (int rc = launch_chained(release_kernel, dim3(1), dim3(kPlanThreads), 0, (cudaStream_t)stream, 1, done, lens, block_table,
                              table_stride, free_pages, free_count, (int)B, (int)width, (int)pool, (int)page))
    return rc;
  return check_launch("release_pages");
}

}  // extern "C"
