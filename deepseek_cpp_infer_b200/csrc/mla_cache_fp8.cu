// The 8-bit paged latent cache: appending tokens (norm + RoPE + quantisation)
// and reading rows back.  Layout in include/dsb/dsb.h: per token
//   scale * [ latent, R x e4m3 | rope key, P x bf16 ],  scale a power of two.
//
// Both kernels move bytes and do little arithmetic; what bounds them is
// stated at each.
//
// No counterpart in the reference (it caches fp32 keys and values per head:
// src/models/deepseek/mla.cpp:16-39, 71-102).

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>

#include "dsb_internal.h"
#include "dsb_ptx.cuh"
#include "mla_fp8.cuh"

namespace dsb {
namespace {

constexpr int kWarps = 4;  // warps per CTA (against 8: a chunk's append 30 us instead of 36)

// theta^(-2k/P) / pi of every rope pair: the angle of position p in units of
// pi is p times this, kept in 64 bits because p reaches 10^5 and beyond and
// the angle is only used modulo 2.
struct RopeFreq {
  double f[32];
};

__device__ __forceinline__ void rope_cos_sin(double freq, int pos, float& c, float& s) {
  double t = (double)pos * freq;
  t -= 2.0 * rint(0.5 * t);  // [-1, 1]
  sincospif((float)t, &s, &c);
}

// Rotates the four interleaved pairs of eight bf16 values.
__device__ __forceinline__ uint4 rotate8(uint4 v, const float (&c)[4], const float (&s)[4]) {
  uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float a = bf16lo_to_f32(w[i]), b = bf16hi_to_f32(w[i]);
    w[i] = pack_bf16x2(a * c[i] - b * s[i], a * s[i] + b * c[i]);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// One warp per job; a row has `parts` jobs for its query heads and one for
// its cache row.  Query job: eight lanes hold a head's P = 64 rope values (16
// bytes each; four lanes at P = 32), so a warp turns 4 (8) heads per step with
// the cosines and sines of its lane's four pairs in registers.  Cache job: R
// / 32 latents per lane; sum of squares, norm and division in 64 bits (the
// FP64 pipe has room: the kernel is bound by its bytes), so that the e4m3
// codes do not depend on the summation order, the largest magnitude by
// shuffles, 4 codes per 32-bit store.
// Bound by HBM for a chunk (4 (R+P) + 4 HP + R + 2P + 4 bytes a row; 4059
// rows of 128 heads 28.2 us, 79% of the copy rate), by its launch for a
// decode batch (1 row 3.3 us, 32 rows 3.7).
template <int R, int P>
__global__ void __launch_bounds__(kWarps * 32)
    append_fp8_kernel(const float* __restrict__ kv_a, int64_t ld_kv, const float* __restrict__ w_norm,
                      const __nv_bfloat16* __restrict__ q, int64_t ldq, const int32_t* __restrict__ positions,
                      const int32_t* __restrict__ seq_ids, const int32_t* __restrict__ block_table, int n_seqs,
                      int max_blocks, int B, int H, int nope, float eps, const __grid_constant__ RopeFreq freq,
                      uint8_t* __restrict__ cache, float* __restrict__ scales, int64_t n_blocks,
                      __nv_bfloat16* __restrict__ q_rope, int parts, int* __restrict__ status) {
  static_assert(R % 128 == 0 && P % 8 == 0 && P <= 64, "layout");
  pdl_wait();
  pdl_launch_dependents();
  const int64_t job = (int64_t)blockIdx.x * kWarps + warp_id();
  const int b = (int)(job / (parts + 1)), part = (int)(job % (parts + 1));
  if (b >= B) return;
  const int lane = (int)lane_id();
  const int pos = positions[b];
  if (pos < 0) return;  // padding

  constexpr int LPH = P / 8;  // lanes per head
  const int k0 = (lane % LPH) * 4;
  float c[4], s[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) rope_cos_sin(freq.f[k0 + i], pos, c[i], s[i]);

  if (part < parts) {
    constexpr int HPW = 32 / LPH;  // heads per step
    const int h0 = (int)((int64_t)part * H / parts), h1 = (int)((int64_t)(part + 1) * H / parts);
    const __nv_bfloat16* src = q + (int64_t)b * ldq + nope + (lane % LPH) * 8;
    __nv_bfloat16* dst = q_rope + (int64_t)b * H * P + (lane % LPH) * 8;
    const int qh = nope + P;
    int h = h0 + lane / LPH;
    for (; h + 3 * HPW < h1; h += 4 * HPW) {  // four loads in flight
      uint4 v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = *reinterpret_cast<const uint4*>(src + (int64_t)(h + i * HPW) * qh);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<uint4*>(dst + (int64_t)(h + i * HPW) * P) = rotate8(v[i], c, s);
    }
    for (; h < h1; h += HPW)
      *reinterpret_cast<uint4*>(dst + (int64_t)h * P) =
          rotate8(*reinterpret_cast<const uint4*>(src + (int64_t)h * qh), c, s);
    return;
  }

  const int seq = seq_ids != nullptr ? seq_ids[b] : b;
  int64_t page = -1;
  if (seq >= 0 && seq < n_seqs && pos / kPageTok < max_blocks)
    page = block_table[(int64_t)seq * max_blocks + pos / kPageTok];
  if (page < 0 || page >= n_blocks) {
    if (lane == 0) atomicCAS(status, 0, kStatusBadInput);
    return;
  }
  const float* kv = kv_a + (int64_t)b * ld_kv;
  float4 x[R / 128];
  double ss = 0.0;
#pragma unroll
  for (int i = 0; i < R / 128; ++i) {
    x[i] = *reinterpret_cast<const float4*>(kv + i * 128 + lane * 4);
    ss += (double)x[i].x * x[i].x + (double)x[i].y * x[i].y + (double)x[i].z * x[i].z + (double)x[i].w * x[i].w;
  }
  const float2 kr_in = lane < P / 2 ? *reinterpret_cast<const float2*>(kv + R + 2 * lane) : make_float2(0.f, 0.f);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  const double inv = 1.0 / sqrt(ss / R + (double)eps);
  double y[R / 32];
  float amax = 0.0f;
#pragma unroll
  for (int i = 0; i < R / 128; ++i) {
    const float4 w = *reinterpret_cast<const float4*>(w_norm + i * 128 + lane * 4);
    y[4 * i + 0] = x[i].x * inv * w.x;
    y[4 * i + 1] = x[i].y * inv * w.y;
    y[4 * i + 2] = x[i].z * inv * w.z;
    y[4 * i + 3] = x[i].w * inv * w.w;
#pragma unroll
    for (int e = 0; e < 4; ++e) amax = fmaxf(amax, fabsf((float)y[4 * i + e]));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  const int e2 = row_scale_exponent(amax);
  const float scale = exp2i(e2), inv_scale = exp2i(-e2);

  uint8_t* row = cache + (page * kPageTok + pos % kPageTok) * (int64_t)(R + 2 * P);
#pragma unroll
  for (int i = 0; i < R / 128; ++i) {
    uint32_t code = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      code |= (uint32_t)__nv_cvt_float_to_fp8((float)(y[4 * i + e] * (double)inv_scale), __NV_SATFINITE, __NV_E4M3)
              << (8 * e);
    *reinterpret_cast<uint32_t*>(row + i * 128 + lane * 4) = code;
  }
  if (lane < P / 2) {
    float cl, sl;
    rope_cos_sin(freq.f[lane], pos, cl, sl);
    const uint32_t kr = pack_bf16x2(kr_in.x * cl - kr_in.y * sl, kr_in.x * sl + kr_in.y * cl);
    *reinterpret_cast<uint32_t*>(row + R + 4 * lane) =
        pack_bf16x2(bf16lo_to_f32(kr) * inv_scale, bf16hi_to_f32(kr) * inv_scale);
  }
  if (lane == 0) scales[page * kPageTok + pos % kPageTok] = scale;
}

// A warp reads kReadRows consecutive output rows: the sequence of the first
// by bisection of cu_seqlens, then forward.  All rows' loads are issued before
// the first conversion.  e4m3 -> fp16 is exact, fp16 * 2^k in fp32 is exact,
// and its four significant bits are exact in bf16.
// Bound by HBM: R + 2P + 4 bytes read, 2 (R + P) written a row.  98,000 rows
// of R = 512: 32.8 us, 81% of the copy rate (4 rows a warp 34.8, 8 rows 43).
constexpr int kReadRows = 2;

template <int R, int P>
__global__ void __launch_bounds__(kWarps * 32)
    read_fp8_kernel(const uint8_t* __restrict__ cache, const float* __restrict__ scales, int64_t n_blocks,
                    const int32_t* __restrict__ block_table, int max_blocks, const int32_t* __restrict__ cu, int B,
                    int64_t T, __nv_bfloat16* __restrict__ latent, int64_t ld_lat, __nv_bfloat16* __restrict__ k_rope,
                    int64_t ld_rope, int* __restrict__ status) {
  pdl_wait();
  pdl_launch_dependents();
  const int lane = (int)lane_id();
  const int64_t t0 = ((int64_t)blockIdx.x * kWarps + warp_id()) * kReadRows;
  const int64_t end = min(T, (int64_t)cu[B]);
  if (t0 == 0 && lane == 0 && cu[B] > T) atomicCAS(status, 0, kStatusBadInput);
  if (t0 >= end) return;
  int lo = 0, hi = B;  // the last sequence that starts at or before t0
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= t0) lo = mid;
    else hi = mid;
  }
  int b = lo;
  const uint8_t* src[kReadRows];
  float scale[kReadRows];
#pragma unroll
  for (int r = 0; r < kReadRows; ++r) {
    const int64_t t = t0 + r;
    src[r] = nullptr;
    scale[r] = 0.0f;
    if (t < end) {
      while (b + 1 < B && cu[b + 1] <= t) ++b;
      const int64_t i = t - cu[b];
      int64_t page = -1;
      if (i >= 0 && i / kPageTok < max_blocks) page = block_table[(int64_t)b * max_blocks + i / kPageTok];
      if (page < 0 || page >= n_blocks) {
        if (lane == 0) atomicCAS(status, 0, kStatusBadInput);
      } else {
        const int64_t row = page * kPageTok + i % kPageTok;
        src[r] = cache + row * (R + 2 * P);
        scale[r] = scales[row];
      }
    }
  }
  constexpr int LN = R / 16;  // lanes with 16 latents each
  uint4 lat[kReadRows], kr[kReadRows];
#pragma unroll
  for (int r = 0; r < kReadRows; ++r) {
    lat[r] = kr[r] = make_uint4(0, 0, 0, 0);
    if (src[r] != nullptr) {
      if (latent != nullptr && lane < LN) lat[r] = *reinterpret_cast<const uint4*>(src[r] + lane * 16);
      if (k_rope != nullptr && lane < P / 8) kr[r] = *reinterpret_cast<const uint4*>(src[r] + R + lane * 16);
    }
  }
#pragma unroll
  for (int r = 0; r < kReadRows; ++r) {
    if (src[r] == nullptr) continue;
    const int64_t t = t0 + r;
    if (latent != nullptr && lane < LN) {
      const uint32_t in[4] = {lat[r].x, lat[r].y, lat[r].z, lat[r].w};
      uint32_t out[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 a = unpack_half2(e4m3x2_to_half2(in[i] & 0xffffu)), d = unpack_half2(e4m3x2_to_half2(in[i] >> 16));
        out[2 * i] = pack_bf16x2(a.x * scale[r], a.y * scale[r]);
        out[2 * i + 1] = pack_bf16x2(d.x * scale[r], d.y * scale[r]);
      }
      uint4* dst = reinterpret_cast<uint4*>(latent + t * ld_lat + lane * 16);
      dst[0] = make_uint4(out[0], out[1], out[2], out[3]);
      dst[1] = make_uint4(out[4], out[5], out[6], out[7]);
    }
    if (k_rope != nullptr && lane < P / 8) {
      const uint32_t in[4] = {kr[r].x, kr[r].y, kr[r].z, kr[r].w};
      uint32_t out[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        out[i] = pack_bf16x2(bf16lo_to_f32(in[i]) * scale[r], bf16hi_to_f32(in[i]) * scale[r]);
      *reinterpret_cast<uint4*>(k_rope + t * ld_rope + lane * 8) = make_uint4(out[0], out[1], out[2], out[3]);
    }
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace
}  // namespace dsb

extern "C" int dsb_kv_norm_rope_append_fp8(dsb_ctx* ctx, const float* kv_a, int64_t ld_kv, const float* w_norm,
                                           const void* q, int64_t ldq, const int32_t* positions,
                                           const int32_t* seq_ids, const int32_t* block_table, int n_seqs,
                                           int max_blocks, int B, int H, int nope, int R, int P, float eps,
                                           float theta, void* cache, float* scales, int64_t n_blocks, void* q_rope) {
  using namespace dsb;
  if (ctx == nullptr) return DSB_EINVAL;
  if (kv_a == nullptr || w_norm == nullptr || q == nullptr || positions == nullptr || block_table == nullptr ||
      cache == nullptr || scales == nullptr || q_rope == nullptr)
    return fail(ctx, DSB_EINVAL, "dsb_kv_norm_rope_append_fp8: null pointer argument");
  if (!cache_shape_ok(R, P))
    return fail(ctx, DSB_EUNSUPPORTED, "dsb_kv_norm_rope_append_fp8: (R, P) = (%d, %d) not supported", R, P);
  if (B <= 0 || H <= 0 || H > 4096 || nope < 0 || nope % 8 != 0 || n_seqs <= 0 || max_blocks <= 0 || n_blocks <= 0 ||
      ld_kv < R + P || ld_kv % 4 != 0 || ldq < (int64_t)H * (nope + P) || ldq % 8 != 0)
    return fail(ctx, DSB_EINVAL,
                "dsb_kv_norm_rope_append_fp8: bad sizes B=%d H=%d nope=%d n_seqs=%d max_blocks=%d n_blocks=%lld "
                "ld_kv=%lld ldq=%lld",
                B, H, nope, n_seqs, max_blocks, (long long)n_blocks, (long long)ld_kv, (long long)ldq);
  if (seq_ids == nullptr && B > n_seqs)
    return fail(ctx, DSB_EINVAL, "dsb_kv_norm_rope_append_fp8: %d rows without seq_ids, %d sequences", B, n_seqs);
  if (!(theta > 0.0f) || !std::isfinite(theta) || !(eps >= 0.0f) || !std::isfinite(eps))
    return fail(ctx, DSB_EINVAL, "dsb_kv_norm_rope_append_fp8: theta=%g eps=%g", theta, eps);
  if (!aligned16(kv_a) || !aligned16(w_norm) || !aligned16(q) || !aligned16(q_rope) || !aligned16(cache))
    return fail(ctx, DSB_EINVAL, "dsb_kv_norm_rope_append_fp8: pointers must be 16-byte aligned");
  DeviceScope scope(ctx->device);
  if (!scope.ok) return fail(ctx, DSB_ECUDA, "dsb_kv_norm_rope_append_fp8: cudaSetDevice(%d) failed", ctx->device);
  RopeFreq freq{};
  for (int k = 0; k < P / 2; ++k) freq.f[k] = std::pow((double)theta, -2.0 * k / P) / 3.14159265358979323846;
  // About 64 query warps for every SM, one step of 4 heads each at least: a
  // decode batch spreads a row's heads over the GPU, a chunk of 4096 rows has
  // two warps a row (28.2 us; one 30.0, four 28.8) that keep its cosines and
  // sines in registers.
  const int steps = (H + 32 / (P / 8) - 1) / (32 / (P / 8));
  const int parts = std::max(1, std::min(steps, ctx->sm_count * 64 / B));
  const int64_t jobs = (int64_t)B * (parts + 1);
  auto run = [&](auto kernel) {
    DSB_CUDA_TRY(ctx, launch_pdl(kernel, dim3((unsigned)((jobs + kWarps - 1) / kWarps)), kWarps * 32, 0, ctx->stream,
                                 kv_a, ld_kv, w_norm, static_cast<const __nv_bfloat16*>(q), ldq, positions, seq_ids,
                                 block_table, n_seqs, max_blocks, B, H, nope, eps, freq, static_cast<uint8_t*>(cache),
                                 scales, n_blocks, static_cast<__nv_bfloat16*>(q_rope), parts, ctx->d_status));
    ctx->stats.kernel_launches++;
    return (int)DSB_OK;
  };
  return R == 512 ? run(append_fp8_kernel<512, 64>) : run(append_fp8_kernel<128, 32>);
}

extern "C" int dsb_mla_cache_read_fp8(dsb_ctx* ctx, const void* cache, const float* scales, int64_t n_blocks,
                                      const int32_t* block_table, int max_blocks, const int32_t* cu_seqlens, int B,
                                      int64_t T, int R, int P, void* latent, int64_t ld_lat, void* k_rope,
                                      int64_t ld_rope) {
  using namespace dsb;
  if (ctx == nullptr) return DSB_EINVAL;
  if (cache == nullptr || scales == nullptr || block_table == nullptr || cu_seqlens == nullptr)
    return fail(ctx, DSB_EINVAL, "dsb_mla_cache_read_fp8: null pointer argument");
  if (!cache_shape_ok(R, P))
    return fail(ctx, DSB_EUNSUPPORTED, "dsb_mla_cache_read_fp8: (R, P) = (%d, %d) not supported", R, P);
  if (B <= 0 || T < 0 || T > INT32_MAX || max_blocks <= 0 || n_blocks <= 0 ||
      (latent != nullptr && (ld_lat < R || ld_lat % 8 != 0)) ||
      (k_rope != nullptr && (ld_rope < P || ld_rope % 8 != 0)))
    return fail(ctx, DSB_EINVAL,
                "dsb_mla_cache_read_fp8: bad sizes B=%d T=%lld max_blocks=%d n_blocks=%lld ld_lat=%lld ld_rope=%lld", B,
                (long long)T, max_blocks, (long long)n_blocks, (long long)ld_lat, (long long)ld_rope);
  if (!aligned16(cache) || !aligned16(latent) || !aligned16(k_rope))
    return fail(ctx, DSB_EINVAL, "dsb_mla_cache_read_fp8: pointers must be 16-byte aligned");
  if (T == 0 || (latent == nullptr && k_rope == nullptr)) return DSB_OK;
  DeviceScope scope(ctx->device);
  if (!scope.ok) return fail(ctx, DSB_ECUDA, "dsb_mla_cache_read_fp8: cudaSetDevice(%d) failed", ctx->device);
  auto run = [&](auto kernel) {
    DSB_CUDA_TRY(ctx, launch_pdl(kernel, dim3((unsigned)((T + kWarps * kReadRows - 1) / (kWarps * kReadRows))),
                                 kWarps * 32, 0, ctx->stream, static_cast<const uint8_t*>(cache), scales, n_blocks,
                                 block_table, max_blocks, cu_seqlens, B, T, static_cast<__nv_bfloat16*>(latent),
                                 ld_lat, static_cast<__nv_bfloat16*>(k_rope), ld_rope, ctx->d_status));
    ctx->stats.kernel_launches++;
    return (int)DSB_OK;
  };
  return R == 512 ? run(read_fp8_kernel<512, 64>) : run(read_fp8_kernel<128, 32>);
}
