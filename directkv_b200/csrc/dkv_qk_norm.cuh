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

__device__ __forceinline__ void unpack8(const uint4& u, float (&o)[8]) {
    o[0] = bf16lo(u.x), o[1] = bf16hi(u.x), o[2] = bf16lo(u.y), o[3] = bf16hi(u.y);
    o[4] = bf16lo(u.z), o[5] = bf16hi(u.z), o[6] = bf16lo(u.w), o[7] = bf16hi(u.w);
}

__device__ __forceinline__ void load_f32x8(const float* p, float (&o)[8]) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    o[0] = a.x, o[1] = a.y, o[2] = a.z, o[3] = a.w, o[4] = b.x, o[5] = b.y, o[6] = b.z, o[7] = b.w;
}

__device__ __forceinline__ void load_weight8(const void* w, int is_f32, int at, float (&o)[8]) {
    if (is_f32) load_f32x8(static_cast<const float*>(w) + at, o);
    else unpack8(*reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(w) + at), o);
}

// Eight lanes per row: lane l holds dimensions 8 l .. 8 l + 7 and 64 + 8 l .. 64 + 8 l + 7, two 16-byte loads.  The eight
// lanes take R heads of one token, so that the angles (512 bytes per token, as much as two rows) and the weights are
// loaded once for all of them and R rows are on their way at a time.
template <int R>
__global__ void __launch_bounds__(256) qk_norm_rope_kernel(const QkNormParams p, int q_groups, int groups) {
    const int l = threadIdx.x & 7;
    const long long id = (static_cast<long long>(blockIdx.x) * 256 + threadIdx.x) >> 3;
    const bool live = id < p.n_tokens * groups;
    const long long tok = live ? (id < 0x7fffffff ? static_cast<unsigned>(id) / static_cast<unsigned>(groups) : id / groups) : 0;
    const int grp = live ? static_cast<int>(id - tok * groups) : 0;
    const int which = grp >= q_groups ? 1 : 0;
    const int h0 = (which ? grp - q_groups : grp) * R, n = live ? min(R, p.heads[which] - h0) : 0;
    const __nv_bfloat16* x = (which ? p.x[1] + tok * p.x_stride[1] : p.x[0] + tok * p.x_stride[0]) + h0 * 128 + l * 8;
    __nv_bfloat16* y = (which ? p.y[1] + tok * p.y_stride[1] : p.y[0] + tok * p.y_stride[0]) + h0 * 128 + l * 8;
    const void* weight = which ? p.weight[1] : p.weight[0];
    const int weight_f32 = which ? p.weight_f32[1] : p.weight_f32[0], weight_stride = which ? p.weight_stride[1] : p.weight_stride[0];
    uint4 a[R], b[R];
#pragma unroll
    for (int i = 0; i < R; ++i)
        if (i < n) {
            a[i] = __ldcs(reinterpret_cast<const uint4*>(x + i * 128));
            b[i] = __ldcs(reinterpret_cast<const uint4*>(x + i * 128 + 64));
        }
    float c[8], s[8], wl[8], wh[8];
    bool turn = false;
    if (p.cos_sin != nullptr && live) {
        const long long pos = p.pos64 ? static_cast<const long long*>(p.positions)[tok]
                                      : static_cast<long long>(static_cast<const int*>(p.positions)[tok]);
        turn = pos >= 0 && pos < p.max_pos;
        if (turn) {
            load_f32x8(p.cos_sin + pos * 128 + l * 8, c);
            load_f32x8(p.cos_sin + pos * 128 + 64 + l * 8, s);
        } else if (l == 0) {
            atomicOr(p.status, kStatusBadPosition);
        }
    }
    if (weight != nullptr && weight_stride == 0) {
        load_weight8(weight, weight_f32, l * 8, wl);
        load_weight8(weight, weight_f32, l * 8 + 64, wh);
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
        if (i >= n) a[i] = b[i] = make_uint4(0u, 0u, 0u, 0u);
        float lo[8], hi[8];
        unpack8(a[i], lo), unpack8(b[i], hi);
        if (weight != nullptr) {
            float ss = 0.f;
#pragma unroll
            for (int d = 0; d < 8; ++d) ss = fmaf(lo[d], lo[d], fmaf(hi[d], hi[d], ss));
            const unsigned eight = 0xffu << (threadIdx.x & 24);
#pragma unroll
            for (int o = 4; o > 0; o >>= 1) ss += __shfl_xor_sync(eight, ss, o);
            const float inv = 1.f / sqrtf(ss * (1.f / 128.f) + p.eps);
            if (weight_stride != 0 && i < n) {
                load_weight8(weight, weight_f32, (h0 + i) * weight_stride + l * 8, wl);
                load_weight8(weight, weight_f32, (h0 + i) * weight_stride + l * 8 + 64, wh);
            }
#pragma unroll
            for (int d = 0; d < 8; ++d) lo[d] *= inv * wl[d], hi[d] *= inv * wh[d];
        }
        if (turn) {
#pragma unroll
            for (int d = 0; d < 8; ++d) {
                const float u = lo[d], v = hi[d];
                lo[d] = u * c[d] - v * s[d];
                hi[d] = v * c[d] + u * s[d];
            }
        }
        if (i < n) {
            *reinterpret_cast<uint4*>(y + i * 128) =
                make_uint4(pack_bf16x2(lo[0], lo[1]), pack_bf16x2(lo[2], lo[3]), pack_bf16x2(lo[4], lo[5]), pack_bf16x2(lo[6], lo[7]));
            *reinterpret_cast<uint4*>(y + i * 128 + 64) =
                make_uint4(pack_bf16x2(hi[0], hi[1]), pack_bf16x2(hi[2], hi[3]), pack_bf16x2(hi[4], hi[5]), pack_bf16x2(hi[6], hi[7]));
        }
    }
}

}  // namespace dkv
