// Prompt attention in expanded form (the per-head attention of
// src/models/deepseek/mla.cpp:86-116 for whole chunks of query rows):
//   s_ij = ([q_nope_i | q_rope_i] . [k_nope_j | k_rope_j]) * scale
//   out_i = sum_j softmax_j(s_ij) v_j,  lse_i = ln sum_j exp(s_ij)

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cmath>

#include "dsb_internal.h"
#include "dsb_ptx.cuh"

namespace dsb {
namespace {

constexpr int kWarps = 8;

// One CTA per (query row of a sequence, head, sequence); a warp takes every
// 8th key.
template <int NOPE, int P, int VD>
__global__ void __launch_bounds__(kWarps * 32) prefill_kernel(dsb_mla_prefill_args a, int* __restrict__ status) {
  constexpr int NN = NOPE / 32, NP = P / 32, NV = VD / 32;
  pdl_wait();
  pdl_launch_dependents();
  const int b = blockIdx.z, h = blockIdx.y, i = blockIdx.x;
  const int lane = (int)lane_id(), warp = (int)warp_id();
  const int q0 = a.cu_q[b], k0 = a.cu_k[b];
  const int lq = a.cu_q[b + 1] - q0, lk = a.cu_k[b + 1] - k0;
  if (q0 < 0 || k0 < 0 || lq < 0 || lk < 0 || q0 + lq > a.Tq || k0 + lk > a.Tk || lq > a.max_q) {
    if (threadIdx.x == 0) atomicCAS(status, 0, kStatusBadInput);
    if (q0 < 0 || k0 < 0 || lq < 0 || lk < 0 || q0 + lq > a.Tq || k0 + lk > a.Tk) return;
  }
  if (i >= lq) return;
  const int64_t row = q0 + i;
  const auto* qn = static_cast<const __nv_bfloat16*>(a.q_nope) + row * a.ld_q_nope + h * a.hd_q_nope;
  const auto* qr = static_cast<const __nv_bfloat16*>(a.q_rope) + row * a.ld_q_rope + h * a.hd_q_rope;
  float q[NN + NP], o[NV];
  for (int e = 0; e < NN; ++e) q[e] = __bfloat162float(qn[lane + 32 * e]);
  for (int e = 0; e < NP; ++e) q[NN + e] = __bfloat162float(qr[lane + 32 * e]);
  for (int e = 0; e < NV; ++e) o[e] = 0.0f;
  const int n = a.causal ? max(0, min(lk, i + 1 + lk - lq)) : lk;
  const float scale_log2 = a.softmax_scale * 1.4426950408889634f;
  float m = -INFINITY, l = 0.0f;
  for (int j = warp; j < n; j += kWarps) {
    const int64_t kr = k0 + j;
    const auto* kn = static_cast<const __nv_bfloat16*>(a.k_nope) + kr * a.ld_k_nope + h * a.hd_k_nope;
    const auto* kp = static_cast<const __nv_bfloat16*>(a.k_rope) + kr * a.ld_k_rope;
    const auto* v = static_cast<const __nv_bfloat16*>(a.v) + kr * a.ld_v + h * a.hd_v;
    float dot = 0.0f;
    for (int e = 0; e < NN; ++e) dot += q[e] * __bfloat162float(kn[lane + 32 * e]);
    for (int e = 0; e < NP; ++e) dot += q[NN + e] * __bfloat162float(kp[lane + 32 * e]);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, d);
    const float s = dot * scale_log2, mn = fmaxf(m, s);
    const float c = exp2f(m - mn), p = exp2f(s - mn);
    m = mn;
    l = l * c + p;
    for (int e = 0; e < NV; ++e) o[e] = o[e] * c + p * __bfloat162float(v[lane + 32 * e]);
  }
  __shared__ float sm[kWarps], sl[kWarps], so[kWarps][VD];
  if (lane == 0) {
    sm[warp] = m;
    sl[warp] = l;
  }
  for (int e = 0; e < NV; ++e) so[warp][lane + 32 * e] = o[e];
  __syncthreads();
  float mt = -INFINITY, lt = 0.0f;
  for (int w = 0; w < kWarps; ++w) mt = fmaxf(mt, sm[w]);
  for (int w = 0; w < kWarps; ++w) lt += sm[w] == -INFINITY ? 0.0f : sl[w] * exp2f(sm[w] - mt);
  if (threadIdx.x < VD) {
    float acc = 0.0f;
    for (int w = 0; w < kWarps; ++w) acc += sm[w] == -INFINITY ? 0.0f : so[w][threadIdx.x] * exp2f(sm[w] - mt);
    static_cast<__nv_bfloat16*>(a.out)[row * a.ld_out + h * VD + threadIdx.x] =
        __float2bfloat16_rn(lt > 0.0f ? acc / lt : 0.0f);
  }
  if (threadIdx.x == 0 && a.lse != nullptr)
    a.lse[row * a.H + h] = lt > 0.0f ? mt * 0.6931471805599453f + logf(lt) : -INFINITY;
}

}  // namespace
}  // namespace dsb

extern "C" int dsb_mla_prefill(dsb_ctx* ctx, const dsb_mla_prefill_args* args) {
  using namespace dsb;
  if (ctx == nullptr) return DSB_EINVAL;
  if (args == nullptr) return fail(ctx, DSB_EINVAL, "dsb_mla_prefill: null arguments");
  const dsb_mla_prefill_args& a = *args;
  if (a.q_nope == nullptr || a.q_rope == nullptr || a.k_nope == nullptr || a.k_rope == nullptr || a.v == nullptr ||
      a.cu_q == nullptr || a.cu_k == nullptr || a.out == nullptr)
    return fail(ctx, DSB_EINVAL, "dsb_mla_prefill: null pointer argument");
  const bool big = a.nope == 128 && a.P == 64 && a.vd == 128, small = a.nope == 64 && a.P == 32 && a.vd == 64;
  if (!big && !small)
    return fail(ctx, DSB_EUNSUPPORTED, "dsb_mla_prefill: (nope, P, vd) = (%d, %d, %d) not supported", a.nope, a.P,
                a.vd);
  if (a.B <= 0 || a.B > 65535 || a.H <= 0 || a.H > 4096 || a.Tq < 0 || a.Tk < 0 || a.max_q < 0 ||
      !std::isfinite(a.softmax_scale))
    return fail(ctx, DSB_EINVAL, "dsb_mla_prefill: bad arguments B=%d H=%d Tq=%d Tk=%d max_q=%d scale=%g", a.B, a.H,
                a.Tq, a.Tk, a.max_q, a.softmax_scale);
  const int64_t ld[] = {a.ld_q_nope, a.ld_q_rope, a.ld_k_nope, a.ld_k_rope, a.ld_v, a.ld_out};
  const int64_t hd[] = {a.hd_q_nope, a.hd_q_rope, a.hd_k_nope, 0, a.hd_v, a.vd};
  const int dim[] = {a.nope, a.P, a.nope, a.P, a.vd, a.vd};
  for (int i = 0; i < 6; ++i) {
    const int64_t heads = i == 3 ? 1 : a.H;
    if (ld[i] % 8 != 0 || hd[i] % 8 != 0 || hd[i] < 0 || (heads > 1 && hd[i] < dim[i]) ||
        ld[i] < (heads - 1) * hd[i] + dim[i])
      return fail(ctx, DSB_EINVAL, "dsb_mla_prefill: tensor %d: token pitch %lld, head pitch %lld", i,
                  (long long)ld[i], (long long)hd[i]);
  }
  if ((reinterpret_cast<uintptr_t>(a.q_nope) | reinterpret_cast<uintptr_t>(a.q_rope) |
       reinterpret_cast<uintptr_t>(a.k_nope) | reinterpret_cast<uintptr_t>(a.k_rope) |
       reinterpret_cast<uintptr_t>(a.v) | reinterpret_cast<uintptr_t>(a.out)) & 15u)
    return fail(ctx, DSB_EINVAL, "dsb_mla_prefill: pointers must be 16-byte aligned");
  if (a.Tq == 0 || a.max_q == 0) return DSB_OK;
  DeviceScope scope(ctx->device);
  if (!scope.ok) return fail(ctx, DSB_ECUDA, "dsb_mla_prefill: cudaSetDevice(%d) failed", ctx->device);
  auto run = [&](auto kernel) {
    DSB_CUDA_TRY(ctx, launch_pdl(kernel, dim3((unsigned)a.max_q, (unsigned)a.H, (unsigned)a.B), kWarps * 32, 0,
                                 ctx->stream, a, ctx->d_status));
    ctx->stats.kernel_launches++;
    return (int)DSB_OK;
  };
  return big ? run(prefill_kernel<128, 64, 128>) : run(prefill_kernel<64, 32, 64>);
}
