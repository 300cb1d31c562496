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

__device__ __forceinline__ uint64_t mul_f32x2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

// Four values as two pairs.
__device__ __forceinline__ void unpack4(const uint2& u, uint64_t (&o)[2]) {
    o[0] = f32x2(bf16lo(u.x), bf16hi(u.x)), o[1] = f32x2(bf16lo(u.y), bf16hi(u.y));
}

__device__ __forceinline__ void load_f32x4(const float* p, uint64_t (&o)[2]) {
    const float4 a = *reinterpret_cast<const float4*>(p);
    o[0] = f32x2(a.x, a.y), o[1] = f32x2(a.z, a.w);
}

__device__ __forceinline__ void load_weight4(const void* w, int is_f32, int at, uint64_t (&o)[2]) {
    if (is_f32) load_f32x4(static_cast<const float*>(w) + at, o);
    else unpack4(*reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(w) + at), o);
}

__device__ __forceinline__ uint2 pack4(const uint64_t (&v)[2]) {
    float a, b, c, d;
    f32x2_split(v[0], a, b);
    f32x2_split(v[1], c, d);
    return make_uint2(pack_bf16x2(a, b), pack_bf16x2(c, d));
}

// Half a warp per row: lane l holds dimensions 4 l .. 4 l + 3 and 64 + 4 l .. 64 + 4 l + 3.  The sixteen lanes take R heads of
// one token: the angles (512 bytes per token, as much as two rows) and the weights are loaded and
// multiplied with one another once for all of them, y = inv (u A - v B), inv (v C + u D), and R rows are on their way at a time.
// Bound by HBM once there are many tokens: 16384 tokens of 32 + 8 heads out of a fused projection take 61 us for 344 MB (5.7
// TB/s, 0.87 of the copy rate).  One head per half warp takes 109 us (angles and weights read for every row), four 75 us.
// Blocks of one warp end and begin at all times, so that loads, arithmetic and stores of different blocks overlap: 65 us with
// two warps, 70 us with eight.
template <int R, int BLOCKS>
__global__ void __launch_bounds__(32, BLOCKS) qk_norm_rope_kernel(const QkNormParams p, int q_groups, int groups) {
    grid_wait();
    grid_trigger();
    const int l = threadIdx.x & 15;
    const long long id = (static_cast<long long>(blockIdx.x) * 32 + threadIdx.x) >> 4;
    if (id >= p.n_tokens * groups) return;                // by halves of a warp
    const long long tok = id < 0x7fffffff ? static_cast<unsigned>(id) / static_cast<unsigned>(groups) : id / groups;
    const int grp = static_cast<int>(id - tok * groups);
    const int which = grp >= q_groups ? 1 : 0;
    const int h0 = (which ? grp - q_groups : grp) * R, n = min(R, p.heads[which] - h0);
    const __nv_bfloat16* x = (which ? p.x[1] + tok * p.x_stride[1] : p.x[0] + tok * p.x_stride[0]) + h0 * 128 + l * 4;
    uint2 a[R], b[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        if (i < n) {
            a[i] = *reinterpret_cast<const uint2*>(x + i * 128);
            b[i] = *reinterpret_cast<const uint2*>(x + i * 128 + 64);
        }
    }
    const void* weight = which ? p.weight[1] : p.weight[0];
    const int weight_f32 = which ? p.weight_f32[1] : p.weight_f32[0], weight_stride = which ? p.weight_stride[1] : p.weight_stride[0];
    uint64_t ca[2], cb[2], cc[2], cd[2];                  // A, -B, C, D
    bool turn = false;
    const uint64_t one = f32x2(1.f, 1.f);
#pragma unroll
    for (int d = 0; d < 2; ++d) ca[d] = cc[d] = one, cb[d] = cd[d] = 0;
    if (p.cos_sin != nullptr) {
        const long long pos = p.pos64 ? static_cast<const long long*>(p.positions)[tok]
                                      : static_cast<long long>(static_cast<const int*>(p.positions)[tok]);
        turn = pos >= 0 && pos < p.max_pos;
        if (turn) {
            load_f32x4(p.cos_sin + pos * 128 + l * 4, ca);
            load_f32x4(p.cos_sin + pos * 128 + 64 + l * 4, cd);
#pragma unroll
            for (int d = 0; d < 2; ++d) cc[d] = ca[d], cb[d] = cd[d] ^ 0x8000000080000000ull;
        } else if (l == 0) {
            atomicOr(p.status, kStatusBadPosition);
        }
    }
    uint64_t wl[2], wh[2];
    if (weight != nullptr && weight_stride == 0) {
        load_weight4(weight, weight_f32, l * 4, wl);
        load_weight4(weight, weight_f32, l * 4 + 64, wh);
#pragma unroll
        for (int d = 0; d < 2; ++d) {
            ca[d] = mul_f32x2(ca[d], wl[d]), cb[d] = mul_f32x2(cb[d], wh[d]);
            cc[d] = mul_f32x2(cc[d], wh[d]), cd[d] = mul_f32x2(cd[d], wl[d]);
        }
    }
    __nv_bfloat16* y = (which ? p.y[1] + tok * p.y_stride[1] : p.y[0] + tok * p.y_stride[0]) + h0 * 128 + l * 4;
    const unsigned half = 0xffffu << (threadIdx.x & 16);
#pragma unroll
    for (int i = 0; i < R; ++i) {
        if (i >= n) break;
        uint64_t lo[2], hi[2];
        unpack4(a[i], lo), unpack4(b[i], hi);
        uint64_t inv = one;
        if (weight != nullptr) {
            uint64_t sq = mul_f32x2(lo[0], lo[0]), sr = mul_f32x2(hi[0], hi[0]);
#pragma unroll
            for (int d = 1; d < 2; ++d) sq = fma_f32x2(lo[d], lo[d], sq), sr = fma_f32x2(hi[d], hi[d], sr);
            float ss, st;
            f32x2_split(add_f32x2(sq, sr), ss, st);
            ss += st;
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) ss += __shfl_xor_sync(half, ss, o);
            const float r = rsqrtf(ss * (1.f / 128.f) + p.eps);
            inv = f32x2(r, r);
            if (weight_stride != 0) {
                load_weight4(weight, weight_f32, (h0 + i) * weight_stride + l * 4, wl);
                load_weight4(weight, weight_f32, (h0 + i) * weight_stride + l * 4 + 64, wh);
#pragma unroll
                for (int d = 0; d < 2; ++d) lo[d] = mul_f32x2(lo[d], wl[d]), hi[d] = mul_f32x2(hi[d], wh[d]);
            }
        }
#pragma unroll
        for (int d = 0; d < 2; ++d) {
            const uint64_t u = mul_f32x2(lo[d], inv), v = mul_f32x2(hi[d], inv);
            lo[d] = mul_f32x2(u, ca[d]);
            hi[d] = mul_f32x2(v, cc[d]);
            if (turn) lo[d] = fma_f32x2(v, cb[d], lo[d]), hi[d] = fma_f32x2(u, cd[d], hi[d]);
        }
        __stcs(reinterpret_cast<uint2*>(y + i * 128), pack4(lo));
        __stcs(reinterpret_cast<uint2*>(y + i * 128 + 64), pack4(hi));
    }
}

}  // namespace dkv
