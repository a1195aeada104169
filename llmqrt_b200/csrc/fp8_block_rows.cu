// Activations in e4m3 with an fp32 scale for each token and group of 128 features: the quantizer, and RMS norm with the
// residual's addition ahead of it.  What the block-scaled fp8 layers (gemm_fp8_block.cu) read.
//
//   scale[m, g] = max(max_{k in g} |y[m, k]|, 1e-12) / 448          q[m, k] = e4m3(y[m, k] * (448 / that maximum))
//
// A group is the sixteen units of eight features that half a warp holds: its maximum is four shuffles and the row stays in
// registers from its one load to its one store.
//
// The norm needs no rounding between it and the quantizer.  With h = T(x + residual) (what the next layer's addition sees)
// and t = h * w, a product of two 16-bit values and therefore exact in fp32, y = t / sqrt(mean(h^2) + eps): the root divides
// the group's maximum like every element of it and cancels, q = e4m3(t * (448 / max |t|)), and only the scale carries it.
// (glue.cu's norm rounds to T twice on the way, as the reference's does; its int8 scale is one per row.)
//
// HBM-bound where rows are many, once a lane works out the factor of one of its units only and passes it on (the divisions, of all
// of them in every lane, held the norm's schedulers at 3/4 of their rate: 37.7 us): 8191 rows of 3584 with a residual take 33 us back
// to back and 35 among others, 6.2 and 5.9 TB/s of 6.5 (7 bytes a feature); 64 rows take 2 us of the GPU, the call 6.5 with its three
// allocations.  The quantizer: 4096 rows of 18944 40 us, 8192 of 3584 15.3, 5.8 TB/s (52.7 and 22 with blocks that went over the units
// of all rows, whose places took the registers of the loads).
#include <type_traits>

#include "common.cuh"

namespace llmqrt {
namespace {

constexpr int kGroup = 128, kGroupUnits = kGroup / 8;
constexpr float kE4m3Max = 448.f, kFloor = 1e-12f;
constexpr int kMaxUnits = 4096;                        // units of eight features of a row that one block takes
constexpr int64_t kMaxWide = 8 * 256 * 65535ll;       // features of a row in pieces
template <int U> constexpr int row_threads() { return U == 1 ? 1024 : 512; }

__device__ __forceinline__ float half_warp_max(float v) {
#pragma unroll
  for (int o = kGroupUnits / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ uint2 to_e4m3x8(const float (&t)[8], float c) {
  uint32_t o[4];
#pragma unroll
  for (int p = 0; p < 4; ++p)                          // (saturating: t * c may round to just above 448)
    o[p] = __nv_cvt_float2_to_fp8x2(make_float2(__fmul_rn(t[2 * p], c), __fmul_rn(t[2 * p + 1], c)), __NV_SATFINITE, __NV_E4M3);
  return make_uint2(o[0] | (o[1] << 16), o[2] | (o[3] << 16));
}
template <typename T> __device__ __forceinline__ void unpack8(const uint4& v, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const float2 x = unpack_pair<T>(w[p]);
    f[2 * p] = x.x;
    f[2 * p + 1] = x.y;
  }
}

// Two sums, each rounded once to T.
template <typename T> __device__ __forceinline__ uint32_t add_pairs(uint32_t a, uint32_t b) {
  using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
  const T2 s = __hadd2(*reinterpret_cast<const T2*>(&a), *reinterpret_cast<const T2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&s);
}

// Blocks (threads of a row's piece, rows), grid (rows, pieces); unit k of a thread is threadIdx.x + k * blockDim.x of its piece.  A lane divides for the group of one
// of its units, and passes the factor on.
template <typename T, int U>
__global__ void __launch_bounds__(256)
quantize_fp8_block_kernel(const T* __restrict__ x, int64_t ldx, uint8_t* __restrict__ q, float* __restrict__ scale, int64_t M, int K,
                          int groups) {
  pdl_wait_then_trigger();
  const int units = K / 8, lane = threadIdx.x & 31, u0 = blockIdx.y * (blockDim.x * U) + threadIdx.x;
  const int64_t m = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  if (m >= M) return;                                  // (the whole warp)
  uint4 v[U];
#pragma unroll
  for (int k = 0; k < U; ++k) {
    const int u = u0 + k * blockDim.x;
    v[k] = u < units ? ldg_cg_16B(x + m * ldx + u * 8) : make_uint4(0, 0, 0, 0);
  }
  const int mine = lane & (U - 1);
  float top = 0.f;
#pragma unroll
  for (int k = 0; k < U; ++k) {
    const float top_k = half_warp_max(absmax8<T>(v[k], 0.f));
    if (k == mine) top = top_k;
  }
  top = fmaxf(top, kFloor);
  const float c_mine = __fdiv_rn(kE4m3Max, top);
  const int in_group = lane & (kGroupUnits - 1), u_mine = u0 - in_group + in_group * (int)blockDim.x;
  if (in_group < U && u_mine < units) scale[m * groups + u_mine / kGroupUnits] = __fdiv_rn(top, kE4m3Max);
#pragma unroll
  for (int k = 0; k < U; ++k) {
    const int u = u0 + k * blockDim.x;
    const float c = __shfl_sync(0xffffffffu, c_mine, lane - mine + k);
    float t[8];
    unpack8<T>(v[k], t);
    if (u < units) *reinterpret_cast<uint2*>(q + m * K + u * 8) = to_e4m3x8(t, c);
  }
}

// One block per row, U units of eight features a thread; unit k of a thread is threadIdx.x + k * blockDim.x.  The sum of
// squares goes up by a butterfly over each 32 units, whose results are added in the same order for every U: a row has the
// same bits at every batch size.
template <typename T, int U>
__global__ void __launch_bounds__(row_threads<U>())
rmsnorm_fp8_block_kernel(const T* __restrict__ x, int64_t ldx, const T* __restrict__ residual, int64_t ldr, T* __restrict__ h_out,
                         const T* __restrict__ weight, float eps, uint8_t* __restrict__ q, float* __restrict__ scale, int H,
                         int groups) {
  __shared__ float red[kMaxUnits / 32];
  pdl_wait_then_trigger();
  const int64_t m = blockIdx.x;
  const int units = H / 8, lane = threadIdx.x & 31, nwarps = blockDim.x >> 5;
  uint4 hv[U];
  {
    uint4 rv[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {                      // all loads first
      const int u = threadIdx.x + k * blockDim.x;
      hv[k] = rv[k] = make_uint4(0, 0, 0, 0);
      if (u < units) {
        hv[k] = ldg_cg_16B(x + m * ldx + u * 8);
        if (residual) rv[k] = ldg_cg_16B(residual + m * ldr + u * 8);
      }
    }
    if (residual) {
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const uint32_t a[4] = {hv[k].x, hv[k].y, hv[k].z, hv[k].w}, b[4] = {rv[k].x, rv[k].y, rv[k].z, rv[k].w};
        uint32_t s[4];
#pragma unroll
        for (int p = 0; p < 4; ++p) s[p] = add_pairs<T>(a[p], b[p]);
        hv[k] = make_uint4(s[0], s[1], s[2], s[3]);
        const int u = threadIdx.x + k * blockDim.x;
        if (u < units) *reinterpret_cast<uint4*>(h_out + m * H + u * 8) = hv[k];
      }
    }
  }
#pragma unroll
  for (int k = 0; k < U; ++k) {
    float f[8], ss = 0.f;
    unpack8<T>(hv[k], f);
#pragma unroll
    for (int j = 0; j < 8; ++j) ss = __fmaf_rn(f[j], f[j], ss);
    ss = warp_sum(ss);
    if (lane == 0) red[k * nwarps + (threadIdx.x >> 5)] = ss;
  }
  __syncthreads();
  float ss = 0.f;
  for (int w = lane; w < U * nwarps; w += 32) ss += red[w];
  const float rstd = rsqrtf(warp_sum(ss) / (float)H + eps);
  float t[U][8], top = 0.f;
  const int mine = lane & (U - 1);                     // the unit whose group's factor and scale the lane works out
#pragma unroll
  for (int k = 0; k < U; ++k) {
    const int u = threadIdx.x + k * blockDim.x;
    float w[8], top_k = 0.f;
    unpack8<T>(hv[k], t[k]);
    unpack8<T>(u < units ? *reinterpret_cast<const uint4*>(weight + u * 8) : make_uint4(0, 0, 0, 0), w);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      t[k][j] = __fmul_rn(t[k][j], w[j]);
      top_k = fmaxf(top_k, fabsf(t[k][j]));
    }
    top_k = half_warp_max(top_k);
    if (k == mine) top = top_k;
  }
  const float y = __fmul_rn(top, rstd);
  const bool above = y >= kFloor;                      // (no: a row with an infinity or a NaN, or a group of next to nothing)
  const float c_mine = above ? __fdiv_rn(kE4m3Max, top) : __fmul_rn(rstd, kE4m3Max / kFloor);
  const int in_group = lane & (kGroupUnits - 1), u_mine = (int)threadIdx.x - in_group + in_group * (int)blockDim.x;
  if (in_group < U && u_mine < units) scale[m * groups + u_mine / kGroupUnits] = __fdiv_rn(above ? y : kFloor, kE4m3Max);
#pragma unroll
  for (int k = 0; k < U; ++k) {
    const int u = threadIdx.x + k * blockDim.x;
    const float c = __shfl_sync(0xffffffffu, c_mine, lane - mine + k);
    if (u < units) *reinterpret_cast<uint2*>(q + m * H + u * 8) = to_e4m3x8(t[k], c);
  }
}

int check_rows(const char* what, const void* x, int64_t ldx, const void* q, const void* scale, int dtype, int64_t M, int64_t K, int64_t most) {
  LLMQRT_REQUIRE(dtype == LLMQRT_F16 || dtype == LLMQRT_BF16, "%s: dtype must be fp16 or bf16", what);
  LLMQRT_REQUIRE(M >= 0 && M <= 0x7fffffffll && K > 0 && K % 8 == 0 && K <= most,
                 "%s: rows must have a multiple of 8 features, at most %lld (got %lld)", what, (long long)most, (long long)K);
  if (M == 0) return LLMQRT_OK;
  LLMQRT_REQUIRE(x && q && scale, "%s: null pointer", what);
  LLMQRT_REQUIRE(ldx >= K && ldx % 8 == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0 && (reinterpret_cast<uintptr_t>(q) & 7) == 0,
                 "%s: rows must be 16-byte aligned (q: 8)", what);
  return LLMQRT_OK;
}

}  // namespace
}  // namespace llmqrt

using namespace llmqrt;

extern "C" {

int llmqrt_quantize_fp8_block(const void* x, int x_dtype, int64_t M, int64_t K, int64_t ldx, uint8_t* q, float* scale,
                              llmqrt_stream_t stream) {
  if (int rc = check_rows("quantize_fp8_block", x, ldx, q, scale, x_dtype, M, K, kMaxUnits * 8)) return rc;
  return llmqrt_quantize_fp8_block_wide(x, x_dtype, M, K, ldx, q, scale, stream);
}

int llmqrt_quantize_fp8_block_wide(const void* x, int x_dtype, int64_t M, int64_t K, int64_t ldx, uint8_t* q, float* scale,
                                   llmqrt_stream_t stream) {
  if (int rc = check_rows("quantize_fp8_block", x, ldx, q, scale, x_dtype, M, K, kMaxWide)) return rc;
  if (M == 0) return LLMQRT_OK;
  const int groups = (int)ceil_div(K, kGroup);
  // Four units a thread once that still leaves every SM its 2048 threads.
  const int units = (int)(K / 8), U = M * units >= (int64_t)sm_count() * 2048 * 4 ? 4 : 1;
  const int64_t pieces = ceil_div(units, 256 * U);
  const unsigned threads = (unsigned)ceil_div(ceil_div(units, pieces * U), 32) * 32, rows = U == 1 ? 256 / threads : 1;
  auto go = [&](auto kern, auto tag) {
    using T = decltype(tag);
    return launch_chained(kern, dim3((unsigned)ceil_div(M, (int64_t)rows), (unsigned)pieces), dim3(threads, rows), 0, (cudaStream_t)stream, 1,
                          static_cast<const T*>(x), ldx, q, scale, M, (int)K, groups);
  };
  const int rc = x_dtype == LLMQRT_F16 ? (U == 4 ? go(quantize_fp8_block_kernel<__half, 4>, __half()) : go(quantize_fp8_block_kernel<__half, 1>, __half()))
                 : U == 4 ? go(quantize_fp8_block_kernel<__nv_bfloat16, 4>, __nv_bfloat16())
                          : go(quantize_fp8_block_kernel<__nv_bfloat16, 1>, __nv_bfloat16());
  if (rc) return rc;
  return check_launch("quantize_fp8_block");
}

int llmqrt_rmsnorm_fp8_block(const void* x, int64_t ldx, const void* residual, int64_t ldr, void* h_out, const void* weight,
                             float eps, uint8_t* q, float* scale, int dtype, int64_t M, int64_t H, llmqrt_stream_t stream) {
  if (int rc = check_rows("rmsnorm_fp8_block", x, ldx, q, scale, dtype, M, H, kMaxUnits * 8)) return rc;
  if (M == 0) return LLMQRT_OK;
  LLMQRT_REQUIRE(weight && (reinterpret_cast<uintptr_t>(weight) & 15) == 0, "rmsnorm_fp8_block: weight must be 16-byte aligned");
  LLMQRT_REQUIRE((residual == nullptr) == (h_out == nullptr), "rmsnorm_fp8_block: residual and h_out go together");
  LLMQRT_REQUIRE(!residual || (ldr >= H && ldr % 8 == 0 &&
                               ((reinterpret_cast<uintptr_t>(residual) | reinterpret_cast<uintptr_t>(h_out)) & 15) == 0),
                 "rmsnorm_fp8_block: residual and h_out must have 16-byte aligned rows");
  const int units = (int)(H / 8), groups = (int)ceil_div(H, kGroup);
  int U = 1;
  while (U < 8 && (units > (U == 1 ? 1024 : 512 * U) || (M >= 2 * sm_count() && units > 256 * U))) U *= 2;
  const int threads = (int)ceil_div(ceil_div(units, U), 32) * 32;
  auto go = [&](auto kern, auto tag) {
    using T = decltype(tag);
    return launch_chained(kern, dim3((unsigned)M), dim3((unsigned)threads), 0, (cudaStream_t)stream, 1, static_cast<const T*>(x),
                          ldx, static_cast<const T*>(residual), ldr, static_cast<T*>(h_out), static_cast<const T*>(weight), eps, q,
                          scale, (int)H, groups);
  };
  auto pick = [&](auto tag) {
    using T = decltype(tag);
    return U == 1 ? go(rmsnorm_fp8_block_kernel<T, 1>, tag) : U == 2 ? go(rmsnorm_fp8_block_kernel<T, 2>, tag)
           : U == 4 ? go(rmsnorm_fp8_block_kernel<T, 4>, tag) : go(rmsnorm_fp8_block_kernel<T, 8>, tag);
  };
  const int rc = dtype == LLMQRT_F16 ? pick(__half()) : pick(__nv_bfloat16());
  if (rc) return rc;
  return check_launch("rmsnorm_fp8_block");
}

}  // extern "C"
