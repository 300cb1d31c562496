// Decode attention over a pool held in 4 bits (format: dkv_kv4.cuh).
//
// out[b, j, h] = sum_t p_t v_t with p = softmax over t < len_b - n_q + 1 + j of scale * q[b, j, h] . k_t; a row that
// attends nothing is zero with a log-sum-exp of -inf.
#pragma once

#include "dkv_kv4.cuh"

namespace dkv {

struct Kv4AttnParams {
    const __nv_bfloat16* q;          // row (b, j) at q + (b * n_q + j) * q_stride, [nh_q, 128]
    long long q_stride;
    __nv_bfloat16* out;
    long long out_stride;
    float* lse;                      // [batch, n_q, nh_q] or nullptr
    const int* seq_lens;             // [batch]
    const int* page_table;
    long long pt_stride;
    int pt_rows;                     // 0: unknown
    int max_pages;                   // entries of a row that may be read
    const int* row_map;              // [batch] or nullptr
    const uint8_t* k_codes;          // [n_slots, nh_kv, 64]
    const uint8_t* k_scales;         // [n_slots, nh_kv, 8]
    const uint8_t* v_codes;
    const uint8_t* v_scales;
    long long n_slots;
    int page_shift;
    int batch, n_q, nh_q, nh_kv;
    float scale_log2;                // softmax scale * k_scale * log2(e)
    float v_scale;
    unsigned int* status;
};

__device__ __forceinline__ void kv4_row4(const uint8_t* codes, const uint8_t* scales, long long at, int lane, float (&v)[4]) {
    // Whole words go into the conversion: fed a 16-bit load, the compiled conversion took its bytes from the wrong place.
    const uint32_t c = *reinterpret_cast<const uint32_t*>(codes + at * 64 + (lane >> 1) * 4);
    uint32_t h[4];
    e2m1x8_to_f16(c, h);
    const float s = e4m3_to_f32(scales[at * 8 + (lane >> 2)]);
    const uint32_t h0 = lane & 1 ? h[2] : h[0], h1 = lane & 1 ? h[3] : h[1];
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&h0));
    const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&h1));
    v[0] = a.x * s, v[1] = a.y * s, v[2] = b.x * s, v[3] = b.y * s;
}

// One block per (request, query token, head); every warp takes every fourth token, lane l dimensions 4l..4l+3.
__global__ void __launch_bounds__(128) kv4_attn_kernel(const Kv4AttnParams p) {
    __shared__ float sm[4][130];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int h = blockIdx.x, j = blockIdx.y, b = blockIdx.z;
    const int kvh = h / (p.nh_q / p.nh_kv);
    long long row = p.row_map != nullptr ? p.row_map[b] : b;
    int len = p.seq_lens[b];
    const long long room = static_cast<long long>(p.max_pages) << p.page_shift;
    if (row < 0 || (p.pt_rows > 0 && row >= p.pt_rows) || len > room || len < 0) {
        if (threadIdx.x == 0) atomicOr(p.status, kStatusBadPage);
        len = row < 0 || (p.pt_rows > 0 && row >= p.pt_rows) || len < 0 ? 0 : static_cast<int>(room);
    }
    const int n = len - p.n_q + 1 + j;
    const uint2 qw = *reinterpret_cast<const uint2*>(p.q + (static_cast<long long>(b) * p.n_q + j) * p.q_stride + h * 128 + lane * 4);
    const float q[4] = {bf16lo(qw.x), bf16hi(qw.x), bf16lo(qw.y), bf16hi(qw.y)};
    float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int t = w; t < n; t += 4) {
        const long long page = p.page_table[row * p.pt_stride + (t >> p.page_shift)];
        const long long slot = (page << p.page_shift) + (t & ((1 << p.page_shift) - 1));
        float k[4] = {0.f, 0.f, 0.f, 0.f}, v[4] = {0.f, 0.f, 0.f, 0.f};
        if (slot >= 0 && slot < p.n_slots) {
            kv4_row4(p.k_codes, p.k_scales, slot * p.nh_kv + kvh, lane, k);
            kv4_row4(p.v_codes, p.v_scales, slot * p.nh_kv + kvh, lane, v);
        } else if (lane == 0) {
            atomicOr(p.status, kStatusBadPage);
        }
        float s = q[0] * k[0] + q[1] * k[1] + q[2] * k[2] + q[3] * k[3];
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
        s *= p.scale_log2;
        const float m2 = fmaxf(m, s), c = exp2f(m - m2), e = exp2f(s - m2);
        l = l * c + e;
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = o[i] * c + e * v[i];
        m = m2;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) sm[w][lane * 4 + i] = o[i];
    if (lane == 0) sm[w][128] = m, sm[w][129] = l;
    __syncthreads();
    if (w != 0) return;
    float top = -INFINITY;
    for (int i = 0; i < 4; ++i) top = fmaxf(top, sm[i][128]);
    float total = 0.f, r[4] = {0.f, 0.f, 0.f, 0.f};
    for (int i = 0; i < 4; ++i) {
        if (sm[i][129] == 0.f) continue;
        const float c = exp2f(sm[i][128] - top);
        total += sm[i][129] * c;
        for (int d = 0; d < 4; ++d) r[d] += sm[i][lane * 4 + d] * c;
    }
    const float inv = total > 0.f ? p.v_scale / total : (total == 0.f ? 0.f : NAN);
    const long long at = static_cast<long long>(b) * p.n_q + j;
    *reinterpret_cast<uint2*>(p.out + at * p.out_stride + h * 128 + lane * 4) =
        make_uint2(pack_bf16x2(r[0] * inv, r[1] * inv), pack_bf16x2(r[2] * inv, r[3] * inv));
    if (p.lse != nullptr && lane == 0)
        p.lse[at * p.nh_q + h] = total > 0.f ? top * 0.6931471805599453f + logf(total) : (total == 0.f ? -INFINITY : NAN);
}

}  // namespace dkv
