// Absorbed MLA decode attention over the 8-bit paged latent cache.
//
//   s_j = softmax_scale * scale_j * (q_lat . c8_j + q_rope . kr_j)
//   out = sum_j softmax(s)_j * scale_j * c8_j

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cmath>

#include "dsb_internal.h"
#include "dsb_ptx.cuh"
#include "mla_fp8.cuh"

namespace dsb {
namespace {

constexpr int kWarps = 8;

// One CTA per (sequence, head); a warp takes every 8th token with its own
// running maximum, sum and R / 32 output columns per lane; the warps' states
// are merged in shared memory.
template <int R, int P>
__global__ void __launch_bounds__(kWarps * 32)
    decode_fp8_kernel(const __nv_bfloat16* __restrict__ q_lat, const __nv_bfloat16* __restrict__ q_rope,
                      const uint8_t* __restrict__ cache, const float* __restrict__ scales, int64_t n_blocks,
                      const int32_t* __restrict__ block_table, int max_blocks, const int32_t* __restrict__ seq_lens,
                      int H, float scale_log2, __nv_bfloat16* __restrict__ out, int* __restrict__ status) {
  constexpr int NR = R / 32, NP = P / 32;
  pdl_wait();
  pdl_launch_dependents();
  const int b = blockIdx.x, h = blockIdx.y;
  const int lane = (int)lane_id(), warp = (int)warp_id();
  int len = seq_lens[b];
  if (len < 0 || len > (int64_t)max_blocks * kPageTok) {
    if (threadIdx.x == 0) atomicCAS(status, 0, kStatusBadInput);
    len = 0;
  }
  float q[NR + NP], o[NR];
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    q[i] = __bfloat162float(q_lat[((int64_t)b * H + h) * R + lane * NR + i]);
    o[i] = 0.0f;
  }
#pragma unroll
  for (int i = 0; i < NP; ++i) q[NR + i] = __bfloat162float(q_rope[((int64_t)b * H + h) * P + lane * NP + i]);
  float m = -INFINITY, l = 0.0f;
  for (int j = warp; j < len; j += kWarps) {
    const int64_t page = block_table[(int64_t)b * max_blocks + j / kPageTok];
    if (page < 0 || page >= n_blocks) {
      if (lane == 0) atomicCAS(status, 0, kStatusBadInput);
      continue;
    }
    const uint8_t* row = cache + (page * kPageTok + j % kPageTok) * (R + 2 * P);
    const float sc = scales[page * kPageTok + j % kPageTok];
    float k[NR];
    float dot = 0.0f;
#pragma unroll
    for (int i = 0; i < NR; i += 2) {
      const float2 f = unpack_half2(e4m3x2_to_half2(*reinterpret_cast<const uint16_t*>(row + lane * NR + i)));
      k[i] = f.x;
      k[i + 1] = f.y;
      dot += q[i] * f.x + q[i + 1] * f.y;
    }
#pragma unroll
    for (int i = 0; i < NP; ++i)
      dot += q[NR + i] * __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(row + R)[lane * NP + i]);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, d);
    const float s = dot * sc * scale_log2;
    const float mn = fmaxf(m, s);
    const float a = exp2f(m - mn), p = exp2f(s - mn);
    m = mn;
    l = l * a + p;
#pragma unroll
    for (int i = 0; i < NR; ++i) o[i] = o[i] * a + p * sc * k[i];
  }
  __shared__ float sm[kWarps], sl[kWarps], so[kWarps][R];
  if (lane == 0) {
    sm[warp] = m;
    sl[warp] = l;
  }
#pragma unroll
  for (int i = 0; i < NR; ++i) so[warp][lane * NR + i] = o[i];
  __syncthreads();
  float mt = -INFINITY, lt = 0.0f;
  for (int w = 0; w < kWarps; ++w) mt = fmaxf(mt, sm[w]);
  for (int w = 0; w < kWarps; ++w) lt += sm[w] == -INFINITY ? 0.0f : sl[w] * exp2f(sm[w] - mt);
  for (int i = threadIdx.x; i < R; i += kWarps * 32) {
    float acc = 0.0f;
    for (int w = 0; w < kWarps; ++w) acc += sm[w] == -INFINITY ? 0.0f : so[w][i] * exp2f(sm[w] - mt);
    out[((int64_t)b * H + h) * R + i] = __float2bfloat16_rn(lt > 0.0f ? acc / lt : 0.0f);
  }
}

}  // namespace
}  // namespace dsb

extern "C" int dsb_mla_decode_fp8(dsb_ctx* ctx, const void* q_lat, const void* q_rope, const void* cache,
                                  const float* scales, int64_t n_blocks, const int32_t* block_table, int max_blocks,
                                  const int32_t* seq_lens, int B, int H, int R, int P, float softmax_scale,
                                  void* out_lat) {
  using namespace dsb;
  if (ctx == nullptr) return DSB_EINVAL;
  if (q_lat == nullptr || q_rope == nullptr || cache == nullptr || scales == nullptr || block_table == nullptr ||
      seq_lens == nullptr || out_lat == nullptr)
    return fail(ctx, DSB_EINVAL, "dsb_mla_decode_fp8: null pointer argument");
  if (!cache_shape_ok(R, P))
    return fail(ctx, DSB_EUNSUPPORTED, "dsb_mla_decode_fp8: (R, P) = (%d, %d) not supported", R, P);
  if (B <= 0 || H <= 0 || H > 128 || max_blocks <= 0 || n_blocks <= 0 || n_blocks >= (1 << 25) ||
      !std::isfinite(softmax_scale))
    return fail(ctx, DSB_EINVAL, "dsb_mla_decode_fp8: bad arguments B=%d H=%d max_blocks=%d n_blocks=%lld scale=%g", B,
                H, max_blocks, (long long)n_blocks, softmax_scale);
  if ((reinterpret_cast<uintptr_t>(q_lat) | reinterpret_cast<uintptr_t>(q_rope) |
       reinterpret_cast<uintptr_t>(out_lat) | reinterpret_cast<uintptr_t>(cache)) & 15u)
    return fail(ctx, DSB_EINVAL, "dsb_mla_decode_fp8: pointers must be 16-byte aligned");
  DeviceScope scope(ctx->device);
  if (!scope.ok) return fail(ctx, DSB_ECUDA, "dsb_mla_decode_fp8: cudaSetDevice(%d) failed", ctx->device);
  auto run = [&](auto kernel) {
    DSB_CUDA_TRY(ctx, launch_pdl(kernel, dim3((unsigned)B, (unsigned)H), kWarps * 32, 0, ctx->stream,
                                 static_cast<const __nv_bfloat16*>(q_lat), static_cast<const __nv_bfloat16*>(q_rope),
                                 static_cast<const uint8_t*>(cache), scales, n_blocks, block_table, max_blocks,
                                 seq_lens, H, softmax_scale * 1.4426950408889634f,
                                 static_cast<__nv_bfloat16*>(out_lat), ctx->d_status));
    ctx->stats.kernel_launches++;
    ctx->stats.mla_calls++;
    return (int)DSB_OK;
  };
  return R == 512 ? run(decode_fp8_kernel<512, 64>) : run(decode_fp8_kernel<128, 32>);
}
