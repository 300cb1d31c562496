// RMS norm of every query and key head with the Neox position rotation in the same pass:
//     n_d = x_d / sqrt(mean(x^2) + eps) * w_d                       (left out where no weight is given)
//     y_d = n_d cos_d - n_{d+64} sin_d,  y_{d+64} = n_{d+64} cos_d + n_d sin_d      for d < 64
// in fp32, rounded once to bf16.
#pragma once

#include "dkv_common.cuh"

namespace dkv {

struct QkNormParams {
    const __nv_bfloat16* x[2];       // queries, keys: [T, heads, 128]
    __nv_bfloat16* y[2];
    long long x_stride[2], y_stride[2];   // elements per token
    const void* weight[2];           // [128] or [heads, 128]; nullptr: no norm
    int weight_f32[2];
    int weight_stride[2];            // 0 or 128
    int heads[2];
    const void* positions;           // [T] int32 or int64
    int pos64;
    const float* cos_sin;            // [max_pos, 128]; nullptr: no rotation
    int max_pos;
    float eps;
    long long n_tokens;
    unsigned int* status;
};

__device__ __forceinline__ void load_weight4(const void* w, int is_f32, int at, float (&o)[4]) {
    if (is_f32) {
        const float4 f = *reinterpret_cast<const float4*>(static_cast<const float*>(w) + at);
        o[0] = f.x, o[1] = f.y, o[2] = f.z, o[3] = f.w;
    } else {
        const uint2 u = *reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(w) + at);
        o[0] = bf16lo(u.x), o[1] = bf16hi(u.x), o[2] = bf16lo(u.y), o[3] = bf16hi(u.y);
    }
}

// Half a warp per (token, head): lane l of 16 holds dimensions 4l..4l+3 and 64+4l..64+4l+3.
__global__ void __launch_bounds__(256) qk_norm_rope_kernel(const QkNormParams p) {
    const int l = threadIdx.x & 15;
    const int heads = p.heads[0] + p.heads[1];
    const long long r = (static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x) >> 4;
    const bool live = r < p.n_tokens * heads;
    const long long tok = live ? r / heads : 0;
    int h = live ? static_cast<int>(r - tok * heads) : 0;
    const int which = h >= p.heads[0] ? 1 : 0;
    if (which) h -= p.heads[0];
    const __nv_bfloat16* x = p.x[which] + tok * p.x_stride[which] + h * 128 + l * 4;
    const uint2 a = *reinterpret_cast<const uint2*>(x), b = *reinterpret_cast<const uint2*>(x + 64);
    float lo[4] = {bf16lo(a.x), bf16hi(a.x), bf16lo(a.y), bf16hi(a.y)};
    float hi[4] = {bf16lo(b.x), bf16hi(b.x), bf16lo(b.y), bf16hi(b.y)};
    if (p.weight[which] != nullptr) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) ss += lo[i] * lo[i] + hi[i] * hi[i];
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const float inv = 1.f / sqrtf(ss * (1.f / 128.f) + p.eps);
        float wl[4], wh[4];
        const int at = h * p.weight_stride[which] + l * 4;
        load_weight4(p.weight[which], p.weight_f32[which], at, wl);
        load_weight4(p.weight[which], p.weight_f32[which], at + 64, wh);
#pragma unroll
        for (int i = 0; i < 4; ++i) lo[i] *= inv * wl[i], hi[i] *= inv * wh[i];
    }
    if (!live) return;
    if (p.cos_sin != nullptr) {
        const long long pos = p.pos64 ? static_cast<const long long*>(p.positions)[tok]
                                      : static_cast<long long>(static_cast<const int*>(p.positions)[tok]);
        if (pos >= 0 && pos < p.max_pos) {
            const float4 c4 = *reinterpret_cast<const float4*>(p.cos_sin + pos * 128 + l * 4);
            const float4 s4 = *reinterpret_cast<const float4*>(p.cos_sin + pos * 128 + 64 + l * 4);
            const float c[4] = {c4.x, c4.y, c4.z, c4.w}, s[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float u = lo[i], v = hi[i];
                lo[i] = u * c[i] - v * s[i];
                hi[i] = v * c[i] + u * s[i];
            }
        } else if (l == 0) {
            atomicOr(p.status, kStatusBadPosition);
        }
    }
    __nv_bfloat16* y = p.y[which] + tok * p.y_stride[which] + h * 128 + l * 4;
    *reinterpret_cast<uint2*>(y) = make_uint2(pack_bf16x2(lo[0], lo[1]), pack_bf16x2(lo[2], lo[3]));
    *reinterpret_cast<uint2*>(y + 64) = make_uint2(pack_bf16x2(hi[0], hi[1]), pack_bf16x2(hi[2], hi[3]));
}

}  // namespace dkv
