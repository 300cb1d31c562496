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
constexpr int kKv4RowThreads = 128;  // of a block that stores or loads rows (8191 tokens of 32 heads both ways: 58.1 us; 62.0 with 256, 59.5 with 64)

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

// 32 bytes in one instruction; 32-byte aligned.
__device__ __forceinline__ void ld_global_v8(const void* p, uint32_t (&w)[8]) {
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                 : "l"(p));
}
__device__ __forceinline__ void st_global_v8(void* p, const uint32_t (&w)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]),
                 "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
}

// To 16 significant bits, to nearest.
__device__ __forceinline__ float snap16(float x) { return __uint_as_float((__float_as_uint(x) + 0x80u) & 0xffffff00u); }

struct Kv4RowsParams {
    const __nv_bfloat16 *k, *v;      // store: [n, nh, 128], token strides in elements
    long long k_stride, v_stride;
    __nv_bfloat16 *k_out, *v_out;    // load: [n, nh, 128] contiguous
    uint8_t *k_codes, *k_scales, *v_codes, *v_scales;
    float k_scale, v_scale;          // store: 1 / pool scale; load: pool scale
    const void* slots;               // [n] int32 or int64
    int slots64;
    int wide;                        // the bf16 rows are 32-byte aligned
    long long n;
    int nh;
    int per_block;                   // tokens of a block
    long long n_slots;
    unsigned int* status;
};

__device__ __forceinline__ long long kv4_slot(const Kv4RowsParams& p, long long i) {
    return p.slots64 ? static_cast<const long long*>(p.slots)[i] : static_cast<long long>(static_cast<const int*>(p.slots)[i]);
}

// Quantises 16 bf16 values.  Returns whether one of them is not finite.
//
// y / s decides between codes at borders of 2 significant bits times s (4 bits), and max|y| / 6 between scales at borders of
// 5 bits: a bf16 value (8 bits) lies on such a border or is at least 2^-8 of it away.  So a product with the rounded
// reciprocal (off by less than 2^-21), snapped to 16 bits, is on a border only where the true quotient is, and on the
// right side of it otherwise: the result is that of exact arithmetic, without a division per value.
__device__ __forceinline__ bool kv4_quantise(const uint32_t (&w)[8], float inv_scale, uint2* codes, uint32_t* scale) {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = __vmaxu2(m, w[j] & 0x7fff7fffu);
    m = max(m & 0xffffu, m >> 16);
    const bool odd = m >= 0x7f80u;
    float y[16];
    float top;
    if (!odd) {
        top = fminf(__uint_as_float(m << 16) * inv_scale, 2688.f);
    } else {                                              // infinities count as the largest value, not-a-numbers as zero
        top = 0.f;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const float x = (j & 1) ? bf16hi(w[j >> 1]) : bf16lo(w[j >> 1]);
            top = fmaxf(top, x == x ? fminf(fabsf(x) * inv_scale, 2688.f) : 0.f);
        }
    }
    uint32_t sb = f32_to_e4m3(snap16(top * (1.f / 6.f)));
    sb = max(sb, 1u);                                     // 2^-9 at least: the reciprocal exists
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(e4m3_to_f32(sb)));
    const float f = r * inv_scale;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
        const float x = (j & 1) ? bf16hi(w[j >> 1]) : bf16lo(w[j >> 1]);
        y[j] = snap16(x * f);
    }
    if (odd) {
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const float x = (j & 1) ? bf16hi(w[j >> 1]) : bf16lo(w[j >> 1]);
            y[j] = x == x ? snap16(fminf(fmaxf(x, -1e30f), 1e30f) * f) : 0.f;
            if (!(fabsf(x) <= 3.4e38f) && x == x) y[j] = copysignf(6.f, x);
        }
    }
    *codes = make_uint2(f32_to_e2m1x8(y), f32_to_e2m1x8(y + 8));
    *scale = sb;
    return odd;
}

__device__ __forceinline__ void kv4_read16(const __nv_bfloat16* src, int wide, uint32_t (&w)[8]) {
    if (wide) {
        ld_global_v8(src, w);
    } else {
        const uint4 a = reinterpret_cast<const uint4*>(src)[0], b = reinterpret_cast<const uint4*>(src)[1];
        w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w, w[4] = b.x, w[5] = b.y, w[6] = b.z, w[7] = b.w;
    }
}

// A thread takes one block of 16 dimensions of K and the same one of V: 32-byte reads, 8 + 1 byte stores.  Bound by HBM: 8191
// tokens of 32 heads stored and read back take 58 to 60 us for 344 MB (5.7 to 5.9 TB/s, 0.88 to 0.91 of the copy rate); with a division per value
// and 16-byte accesses 157 us.
__global__ void __launch_bounds__(kKv4RowThreads) kv4_store_kernel(const Kv4RowsParams p) {
    grid_wait();
    grid_trigger();
    const int units = p.nh * 8;                           // blocks of 16 per token
    for (int i = threadIdx.x; i < p.per_block * units; i += kKv4RowThreads) {
        const int t = i / units, u = i - t * units;
        const long long tok = static_cast<long long>(blockIdx.x) * p.per_block + t;
        if (tok >= p.n) return;
        const long long slot = kv4_slot(p, tok);
        uint32_t kw[8], vw[8];
        kv4_read16(p.k + tok * p.k_stride + u * 16, p.wide, kw);
        kv4_read16(p.v + tok * p.v_stride + u * 16, p.wide, vw);
        if (slot < 0 || slot >= p.n_slots) {                // (-1: no token)
            if (u == 0 && slot != -1) atomicOr(p.status, kStatusBadSlot);
            continue;
        }
        uint2 kc, vc;
        uint32_t ks, vs;
        bool odd = kv4_quantise(kw, p.k_scale, &kc, &ks);
        odd |= kv4_quantise(vw, p.v_scale, &vc, &vs);
        const long long at = slot * units + u;
        reinterpret_cast<uint2*>(p.k_codes)[at] = kc;
        reinterpret_cast<uint2*>(p.v_codes)[at] = vc;
        p.k_scales[at] = static_cast<uint8_t>(ks);
        p.v_scales[at] = static_cast<uint8_t>(vs);
        if (odd) atomicOr(p.status, kStatusNonFinite);
    }
}

__device__ __forceinline__ void kv4_write16(__nv_bfloat16* dst, uint2 codes, uint32_t scale, float pool_scale, int wide) {
    uint32_t h[8], o[8];
    e2m1x8_to_f16(codes.x, reinterpret_cast<uint32_t(&)[4]>(h[0]));
    e2m1x8_to_f16(codes.y, reinterpret_cast<uint32_t(&)[4]>(h[4]));
    const float s = e4m3_to_f32(scale) * pool_scale;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[j]));
        o[j] = pack_bf16x2(f.x * s, f.y * s);
    }
    if (wide) {
        st_global_v8(dst, o);
    } else {
        reinterpret_cast<uint4*>(dst)[0] = make_uint4(o[0], o[1], o[2], o[3]);
        reinterpret_cast<uint4*>(dst)[1] = make_uint4(o[4], o[5], o[6], o[7]);
    }
}

__global__ void __launch_bounds__(kKv4RowThreads) kv4_load_kernel(const Kv4RowsParams p) {
    grid_wait();
    grid_trigger();
    const int units = p.nh * 8;
    for (int i = threadIdx.x; i < p.per_block * units; i += kKv4RowThreads) {
        const int t = i / units, u = i - t * units;
        const long long tok = static_cast<long long>(blockIdx.x) * p.per_block + t;
        if (tok >= p.n) return;
        const long long slot = kv4_slot(p, tok);
        uint2 kc = make_uint2(0u, 0u), vc = make_uint2(0u, 0u);
        uint32_t ks = 0, vs = 0;
        if (slot >= 0 && slot < p.n_slots) {
            const long long at = slot * units + u;
            kc = reinterpret_cast<const uint2*>(p.k_codes)[at];
            vc = reinterpret_cast<const uint2*>(p.v_codes)[at];
            ks = p.k_scales[at], vs = p.v_scales[at];
        } else if (u == 0 && slot != -1) {
            atomicOr(p.status, kStatusBadSlot);
        }
        const long long at = (tok * units + u) * 16;
        kv4_write16(p.k_out + at, kc, ks, p.k_scale, p.wide);
        kv4_write16(p.v_out + at, vc, vs, p.v_scale, p.wide);
    }
}

}  // namespace dkv
