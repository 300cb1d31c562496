// K/V rows held in 4 bits: the format, and the kernels that write it (store) and read it back as bf16 (load).
//
// A row of 128 values is 8 blocks of 16 consecutive dimensions.  With y = x / pool_scale (a power of two, so the
// division is exact):
//     s    = e4m3(max |y| / 6), at least 2^-9 (the smallest e4m3), at most 448
//     code = e2m1(y / s), nearest, ties to the even code: magnitudes 0 .5 1 1.5 2 3 4 6 and a sign bit
//     x'   = code * s * pool_scale
// 64 bytes of codes (dimension 2i in the low, 2i + 1 in the high four bits of byte i) and 8 bytes of scales: 72
// bytes instead of 256.  code * s has at most 6 significant bits, so it is exact in bf16 and in fp16 alike.
// Codes have no infinity and no not-a-number: an infinity is stored as the largest value (6 * 448), a
// not-a-number as zero, and both are reported in the status word.
#pragma once

#include <cuda_fp16.h>

#include "dkv_common.cuh"

namespace dkv {

constexpr int kKv4CodeBytes = 64;    // per row of one head
constexpr int kKv4ScaleBytes = 8;

// Four bytes of codes to four fp16 pairs (lower dimension in the lower half).
__device__ __forceinline__ void e2m1x8_to_f16(uint32_t w, uint32_t (&h)[4]) {
    asm("{\n\t"
        ".reg .b8 b0, b1, b2, b3;\n\t"
        "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t"
        "}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(w));
}

// Eight values, already over the block's scale, to codes: byte i of the word holds values 2i (low) and 2i + 1.
__device__ __forceinline__ uint32_t f32_to_e2m1x8(const float* v) {
    uint32_t w;
    asm("{\n\t"
        ".reg .b8 b0, b1, b2, b3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
        "mov.b32 %0, {b0, b1, b2, b3};\n\t"
        "}"
        : "=r"(w)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return w;
}

// Two e4m3 bytes to an fp16 pair.
__device__ __forceinline__ uint32_t e4m3x2_to_f16(uint32_t two) {
    uint32_t h;
    asm("{\n\t.reg .b16 t;\n\tcvt.u16.u32 t, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, t;\n\t}" : "=r"(h) : "r"(two));
    return h;
}

__device__ __forceinline__ float e4m3_to_f32(uint32_t byte) {
    const uint32_t h = e4m3x2_to_f16(byte);
    return __half2float(__ushort_as_half(static_cast<unsigned short>(h & 0xffffu)));
}

__device__ __forceinline__ uint32_t f32_to_e4m3(float v) {
    uint32_t r;
    asm("{\n\t.reg .b16 t;\n\tcvt.rn.satfinite.e4m3x2.f32 t, %2, %1;\n\tcvt.u32.u16 %0, t;\n\t}" : "=r"(r) : "f"(v), "f"(0.f));
    return r & 0xffu;
}

struct Kv4StoreParams {
    const __nv_bfloat16* src[2];     // K rows, V rows: [n, nh, 128], token stride in elements
    long long src_stride[2];
    uint8_t* codes[2];
    uint8_t* scales[2];
    float inv_scale[2];              // 1 / pool scale
    const void* slots;               // [n] int32 or int64
    int slots64;
    long long n_rows;                // n * nh
    int nh;
    long long n_slots;
    unsigned int* status;
};

__device__ __forceinline__ long long kv4_slot(const void* slots, int slots64, long long i) {
    return slots64 ? static_cast<const long long*>(slots)[i] : static_cast<long long>(static_cast<const int*>(slots)[i]);
}

// One thread per block of 16 dimensions (8 threads per row), K rows first, then V rows.
__global__ void __launch_bounds__(256) kv4_store_kernel(const Kv4StoreParams p) {
    const long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
    const int which = blockIdx.y;
    const long long row = i >> 3;
    if (row >= p.n_rows) return;
    const int blk = static_cast<int>(i & 7);
    const long long tok = row / p.nh;
    const int head = static_cast<int>(row - tok * p.nh);
    const long long slot = kv4_slot(p.slots, p.slots64, tok);
    if (slot < 0 || slot >= p.n_slots) {
        if (blk == 0) atomicOr(p.status, kStatusBadSlot);
        return;
    }
    const uint4* src = reinterpret_cast<const uint4*>(p.src[which] + tok * p.src_stride[which] + head * 128 + blk * 16);
    const uint4 lo = src[0], hi = src[1];
    const uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    float y[16], top = 0.f;
    bool odd = false;                 // a value that is not finite
#pragma unroll
    for (int j = 0; j < 16; ++j) {
        const float x = (j & 1) ? bf16hi(w[j >> 1]) : bf16lo(w[j >> 1]);
        odd |= !(fabsf(x) <= 3.4e38f);
        y[j] = x == x ? fminf(fmaxf(x * p.inv_scale[which], -2688.f), 2688.f) : 0.f;
        top = fmaxf(top, fabsf(y[j]));
    }
    if (odd) atomicOr(p.status, kStatusNonFinite);
    // __fdiv_rn: a quotient that lies exactly between two scales (or two codes) must come out exactly there.
    uint32_t sb = f32_to_e4m3(__fdiv_rn(top, 6.f));
    sb = sb == 0 ? 1u : sb;           // 2^-9: never a division by zero below
    const float s = e4m3_to_f32(sb);
#pragma unroll
    for (int j = 0; j < 16; ++j) y[j] = __fdiv_rn(y[j], s);
    const long long at = (slot * p.nh + head) * 8 + blk;
    reinterpret_cast<uint2*>(p.codes[which])[at] = make_uint2(f32_to_e2m1x8(y), f32_to_e2m1x8(y + 8));
    p.scales[which][at] = static_cast<uint8_t>(sb);
}

struct Kv4LoadParams {
    const uint8_t* codes[2];
    const uint8_t* scales[2];
    float scale[2];                  // pool scale
    __nv_bfloat16* dst[2];           // [n, nh, 128] contiguous
    const void* slots;
    int slots64;
    long long n_rows;
    int nh;
    long long n_slots;
    unsigned int* status;
};

__global__ void __launch_bounds__(256) kv4_load_kernel(const Kv4LoadParams p) {
    const long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
    const int which = blockIdx.y;
    const long long row = i >> 3;
    if (row >= p.n_rows) return;
    const int blk = static_cast<int>(i & 7);
    const long long tok = row / p.nh;
    const int head = static_cast<int>(row - tok * p.nh);
    const long long slot = kv4_slot(p.slots, p.slots64, tok);
    uint2 c = make_uint2(0u, 0u);
    float s = 0.f;
    if (slot >= 0 && slot < p.n_slots) {
        const long long at = (slot * p.nh + head) * 8 + blk;
        c = reinterpret_cast<const uint2*>(p.codes[which])[at];
        s = e4m3_to_f32(p.scales[which][at]) * p.scale[which];
    } else if (blk == 0) {
        atomicOr(p.status, kStatusBadSlot);
    }
    uint32_t h[8], o[8];
    e2m1x8_to_f16(c.x, reinterpret_cast<uint32_t(&)[4]>(h[0]));
    e2m1x8_to_f16(c.y, reinterpret_cast<uint32_t(&)[4]>(h[4]));
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[j]));
        o[j] = pack_bf16x2(f.x * s, f.y * s);
    }
    uint4* dst = reinterpret_cast<uint4*>(p.dst[which] + row * 128 + blk * 16);
    dst[0] = make_uint4(o[0], o[1], o[2], o[3]);
    dst[1] = make_uint4(o[4], o[5], o[6], o[7]);
}

}  // namespace dkv
