// Decode attention over a pool held in 4 bits (format: dkv_kv4.cuh).
//
// out[b, j, h] = sum_t p_t v_t with p = softmax over t < len_b - n_q + 1 + j of scale * q[b, j, h] . k_t; a row that
// attends nothing is zero with a log-sum-exp of -inf.
//
// One pass over the rows with a running maximum and sum.  The (query token, head) pairs that share a KV head are the
// columns of two warp-level products (m16n8k16, fp16 in, fp32 out) per 16 tokens:
//     S [16 tokens x 8 columns] = K Q^T            O^T [128 dims x 8 columns] += V^T P^T
// so a row is decoded once for all of them.  code * block scale is exact in fp16.  A query row is scaled by a power of two
// that brings its largest value to 2^14 before it becomes fp16 (undone in the fp32 scores): exact for values down to 2^-31 of the
// largest, off by at most 2^-39 of it below.  P is rounded to fp16, scaled so that the largest one lies between 2^12 and 2^15: off by
// 2^-11 of itself, or where it is less than 2^-26 of the largest by 2^-37 of that.  Without the scaling weights below 2^-25 of
// the largest vanish from O, but not from the sum: with one strong token whose value row is zero the output loses whatever is
// that far below.  Scores, maximum, sum and O are fp32.
//
// What bounds it is bytes, 144 per token and KV head, and close behind them the instructions that turn codes into fp16: 64
// requests of 12000 to 20000 tokens, 32 query heads on 8, take 217 us (5.51 TB/s, 0.84 of the measured copy rate), copies
// alone 192 us; the arithmetic needs 115 cycles per 16 tokens and SM, HBM 100.  Under sustained load the power limit
// lowers the clock (1965 to 1762 MHz and less) and with it this kernel (243 to 260 us).  So the loop is written for few instructions: 32 tokens
// per step with one vote on the running maximum, table entries looked up for 16 steps at a time, one multiply-add per
// copy address.
//
// A warp brings its tokens in through its own ring of cp.async copies (any page size, device or host pool alike), so warps never
// wait for one another.  A block's warps take neighbouring heads of the same tokens, which makes the 64-byte rows of a
// token one contiguous read.
#pragma once

#include "dkv_attn_mma.cuh"
#include "dkv_kv4.cuh"

namespace dkv {

constexpr int kKv4Tile = 32;                             // tokens a warp takes in one step, as two halves of 16
constexpr int kKv4Stages = 2;
constexpr int kKv4HalfBytes = 2 * 1024 + 2 * 128;        // 16 tokens: K codes, V codes, K scales, V scales
constexpr int kKv4StageBytes = 2 * kKv4HalfBytes;
// Warps of a block and blocks per SM: 16 warps per SM with 8 columns (query fragments in registers), 12 with 16 (in shared
// memory, 68 B of them spilled; 16 drafts of up to 4096 tokens: 32 us; as 16 warps, which spill more, at the time, 48 us against 37).
template <int NT>
constexpr int kKv4Warps = NT == 1 ? 8 : 4;
template <int NT>
constexpr int kKv4BlocksPerSm = NT == 1 ? 2 : 3;
template <int NT>
constexpr int kKv4WarpBytes = kKv4Stages * kKv4StageBytes + (NT == 1 ? 0 : NT * 2048);
constexpr int kKv4MaxBatch = 4096;                       // of a call
constexpr int kKv4LaunchBatch = 1024;                    // of a launch: what leaves room for the blocks that share an SM
constexpr int kKv4RecFloats = 132;                       // O[128], m (log2 domain), l, 2 pad
constexpr float kKv4Low = -3e38f;                        // the running maximum before the first token
// What P is relative to lies 2^12 below the running maximum, and follows once a score is 2^15 above it: P <= 2^15 in fp16, the
// largest one 2^12 at least.
constexpr float kKv4Lift = 12.f, kKv4Lag = 15.f;

// Division of 0 .. 2^31 - 1 by a number that the host knows: with 2^(l-1) < d <= 2^l and m = ceil(2^(31+l) / d) < 2^32, the product
// n m / 2^(31+l) is less than 1 / d above n / d.  A division by a variable is some 150 cycles of latency, and the way from a launch to
// its first copy has several.
struct Kv4Div {
    unsigned m;
    int shift;
    Kv4Div() = default;
    explicit Kv4Div(unsigned d) {
        int l = 0;
        while ((1ull << l) < d) ++l;
        shift = 31 + l;
        m = static_cast<unsigned>(((1ull << shift) + d - 1) / d);
    }
    __device__ __forceinline__ int operator()(int n) const {
        return static_cast<int>((static_cast<unsigned long long>(static_cast<unsigned>(n)) * m) >> shift);
    }
};

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
    int room;                        // tokens that the entries of a row reach
    const int* row_map;              // [batch] or nullptr: row b + row0
    int row0;
    const uint8_t* k_codes;          // [n_slots, nh_kv, 64]
    const uint8_t* k_scales;         // [n_slots, nh_kv, 8]
    const uint8_t* v_codes;
    const uint8_t* v_scales;
    int page_shift;
    int n_pages;                     // pages that begin inside the pool
    int batch, n_q, nh_q, nh_kv, group;
    int cols;                        // n_q * group: columns of one KV head
    int whole;                       // no segment is split: the list has one entry per segment, and nothing is left to merge
    int n_cc;                        // column chunks of 8 * NT
    int hg, ts, n_hg;                // heads and token lanes of a block (hg * ts <= kKv4Warps<NT>), head groups
    int tile_shift;                  // log2 of kKv4Tile * ts (ts is a power of two): tokens of a tile
    Kv4Div by_seg, by_cc, by_hg, by_group, by_nh_q, by_n_q, by_grid;      // n_hg * n_cc, n_cc, ...
    float scale_log2;                // softmax scale * k_scale * log2(e)
    float v_scale;
    float* rec;                      // [blocks, 2, hg, 8 * NT, kKv4RecFloats]
    int* cum;                        // [batch + 1] tiles before each request
    unsigned int* status;
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async8(uint32_t dst, const void* src, uint32_t bytes) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async8(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}
// base + slot * row, in one instruction.
__device__ __forceinline__ const uint8_t* row_of(const uint8_t* base, unsigned slot, unsigned row) {
    const uint8_t* p;
    asm("mad.wide.u32 %0, %1, %2, %3;" : "=l"(p) : "r"(slot), "r"(row), "l"(base));
    return p;
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint32_t hmul2_f16(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
    uint32_t d;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    return d;
}
__device__ __forceinline__ uint32_t bit_select(uint32_t a, uint32_t b, uint32_t mask) {   // mask ? a : b
    uint32_t d;
    asm("lop3.b32 %0, %1, %2, %3, 0xCA;" : "=r"(d) : "r"(mask), "r"(a), "r"(b));
    return d;
}
// The same with zeros to add to.
__device__ __forceinline__ void mma_f16_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The flattened tile list (its length fits 31 bits, the host sees to that) is dealt out evenly: block i of n begins at its
// share, the first total % n blocks have one tile more.
struct Kv4Deal {
    int each, more;
    __device__ __forceinline__ Kv4Deal(int total, int n, int grid, Kv4Div by_grid) {
        each = n == grid ? by_grid(total) : static_cast<unsigned>(total) / static_cast<unsigned>(n);
        more = total - each * n;
    }
    __device__ __forceinline__ int share(int i) const { return each * i + min(i, more); }
    __device__ __forceinline__ int owner(int x) const {
        const int edge = more * (each + 1);
        return x < edge ? static_cast<unsigned>(x) / static_cast<unsigned>(each + 1) : more + static_cast<unsigned>(x - edge) / static_cast<unsigned>(each);
    }
};
// Blocks that take part.  Segments of up to 4 tiles on average that are enough to occupy an eighth of the grid are not cut
// finer than there are segments: what is gained in steps goes into merging (64 requests of 77 tokens in a wide table, 32 heads on
// 8: 10.5 us, 11.8 us with a block per tile).
__device__ __forceinline__ int kv4_blocks(int total, int segments, int grid) {
    return min(total <= 4ll * segments && 8ll * segments >= grid ? segments : total, grid);
}

// A request's length as far as the table reaches, and its row; a length or row outside is reported.
__device__ __forceinline__ int kv4_length(const Kv4AttnParams& p, int b, long long* row_out) {
    const long long row = p.row_map != nullptr ? p.row_map[b] : b + p.row0;
    *row_out = row;
    const int len = p.seq_lens[b];
    if (row < 0 || (p.pt_rows > 0 && row >= p.pt_rows) || len < 0) return -1;
    return len > p.room ? -2 : len;
}
__device__ __forceinline__ int kv4_clean_length(const Kv4AttnParams& p, int code) {
    return code >= 0 ? code : (code == -2 ? p.room : 0);
}

template <int NT>
struct Kv4State {
    float o[8][NT][4];
    float m[NT][2], l[NT][2];
};

// WIDE: pages of 16 tokens and more, so that 16 tokens lie in one page and one table entry serves the whole warp.
template <int NT, bool WIDE>
__global__ void __launch_bounds__(kKv4Warps<NT> * 32, kKv4BlocksPerSm<NT>) kv4_attn_kernel(const Kv4AttnParams p) {
    constexpr int C = 8 * NT, W = kKv4Warps<NT>;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ int sh_scan[W];
    int* cum = reinterpret_cast<int*>(smem + W * kKv4WarpBytes<NT>);
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int g = lane >> 2, c = lane & 3;
    const int tl = p.by_hg(w), hl = w - tl * p.hg;
    const bool active = tl < p.ts;
    auto tiles_of = [&](int len) { return static_cast<int>((static_cast<unsigned>(len) + (1u << p.tile_shift) - 1u) >> p.tile_shift); };

    grid_wait();
    const int per_tile = p.n_hg * p.n_cc;
    int total;
    if (p.whole) {
        total = p.batch * per_tile;                  // one entry per segment, whatever its length
    } else if (p.batch <= 32) {
        // Tiles (of 32 * ts tokens) before every request; a request without tokens has one, which writes its zeros.  Every warp
        // for itself: without the block's barriers the first copies leave 0.4 us earlier.
        cum += w * 33;
        int n = 0;
        if (lane < p.batch) {
            long long row;
            n = max(1, tiles_of(kv4_clean_length(p, kv4_length(p, lane, &row))));
        }
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, n, o);
            if (lane >= o) n += x;
        }
        cum[lane + 1] = n;
        if (lane == 0) cum[0] = 0;
        if (blockIdx.x == 0 && w == 0) {
            p.cum[lane + 1] = n;
            if (lane == 0) p.cum[0] = 0;
        }
        __syncwarp();
        total = __shfl_sync(0xffffffffu, n, 31) * per_tile;
    } else {
        if (threadIdx.x == 0) cum[0] = 0;
        int before = 0;
        for (int b0 = 0; b0 < p.batch; b0 += W * 32) {
            const int b = b0 + threadIdx.x;
            int n = 0;
            if (b < p.batch) {
                long long row;
                const int len = kv4_clean_length(p, kv4_length(p, b, &row));
                n = max(1, tiles_of(len));
            }
            int inc = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, inc, o);
                if (lane >= o) inc += x;
            }
            if (lane == 31) sh_scan[w] = inc;
            __syncthreads();
            int base = before;
            for (int i = 0; i < w; ++i) base += sh_scan[i];
            if (b < p.batch) cum[b + 1] = base + inc;
            for (int i = 0; i < W; ++i) before += sh_scan[i];
            __syncthreads();
        }
        if (blockIdx.x == 0)
            for (int b = threadIdx.x; b <= p.batch; b += blockDim.x) p.cum[b] = cum[b];
        total = before * per_tile;
    }
    const int blocks = kv4_blocks(total, p.batch * per_tile, gridDim.x);
    grid_trigger();
    if (static_cast<int>(blockIdx.x) >= blocks) return;
    const Kv4Deal deal(total, blocks, gridDim.x, p.by_grid);
    const int x0 = deal.share(blockIdx.x), x1 = deal.share(blockIdx.x + 1);

    uint8_t* const ring_ptr = smem + w * kKv4WarpBytes<NT>;
    uint4* const q_smem = reinterpret_cast<uint4*>(ring_ptr + kKv4Stages * kKv4StageBytes) + lane;
    const uint32_t ring = smem_u32(ring_ptr);
    const int tau = (g >> 1) + 4 * (g & 1);          // token of this lane's rows of the score tile: tau and tau + 8
    const int page_mask = (1 << p.page_shift) - 1;
    Kv4State<NT> st;

    for (int x = x0; x < x1;) {
        // Segment: one request, head group and column chunk.
        const int y = p.by_seg(x);                   // (n_hg * n_cc once more below: a register less through the loop)
        int b = y, entries = 1, seg = x - y * (p.n_hg * p.n_cc), tile0 = 0;
        if (!p.whole) {
            int lo = 0, hi = p.batch - 1;
            while (lo < hi) {
                const int mid = (lo + hi + 1) >> 1;
                if (cum[mid] <= y) lo = mid;
                else hi = mid - 1;
            }
            b = lo;
            entries = cum[b + 1] - cum[b];
            const int r = x - cum[b] * (p.n_hg * p.n_cc);
            seg = p.n_hg * p.n_cc == 1 ? 0 : static_cast<unsigned>(r) / static_cast<unsigned>(entries);
            tile0 = r - seg * entries;
        }
        long long row;
        const int code = kv4_length(p, b, &row), len = kv4_clean_length(p, code);
        if (code < 0 && threadIdx.x == 0) atomicOr(p.status, kStatusBadPage);
        const int taken = min(entries - tile0, x1 - x);
        const int n_tiles = p.whole ? tiles_of(len) : taken;
        const int hgi = p.by_cc(seg), cc = seg - hgi * p.n_cc;
        const bool whole = taken == entries;
        const int kvh = hgi * p.hg + hl;
        const int* table = p.page_table + row * p.pt_stride;

        if (active) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int k = 0; k < 4; ++k) st.o[i][n][k] = 0.f;
#pragma unroll
            for (int n = 0; n < NT; ++n) st.m[n][0] = st.m[n][1] = kKv4Low, st.l[n][0] = st.l[n][1] = 0.f;

            // ---- copies: of every 16 tokens this lane brings 16 bytes of K and V of tokens tau and tau + 8, and 8 bytes of scales
            const unsigned code_row = p.nh_kv * 64, scale_row = p.nh_kv * 8;                 // bytes per token
            const uint8_t* k_lane = p.k_codes + kvh * 64 + c * 16 + (WIDE ? tau * code_row : 0u);
            const uint8_t* v_lane = p.v_codes + kvh * 64 + c * 16 + (WIDE ? tau * code_row : 0u);
            const int s_tau = tau + (c & 1) * 8;
            const uint8_t* s_lane = ((c & 2) ? p.v_scales : p.k_scales) + kvh * 8 + (WIDE ? s_tau * scale_row : 0);
            const uint32_t k_dst = ring + lane * 16;
            const uint32_t v_dst = ring + 1024 + tau * 64 + ((c ^ ((g >> 1) & 2)) << 4);     // 16-byte pieces of rows 2, 3 mod 4 change places
            const uint32_t s_dst = ring + 2048 + (c & 2) * 64 + s_tau * 8;
            auto token0 = [&](int i) { return ((tile0 + i) * p.ts + tl) * kKv4Tile; };
            // Slots, looked up by the lanes together and handed round: WIDE the first slot of a half (lane l of a batch of
            // 16 steps has half l), else every token's (lane l of a step has token l).  -1: behind the length, or no page.
            int now = -1, next;
            auto look = [&](int i) {
                const int step = WIDE ? i + (lane >> 1) : i;
                const int t = token0(step) + (WIDE ? (lane & 1) * 16 : lane);
                int slot = -1;
                if (step < n_tiles && t < len) {
                    const int e = table[t >> p.page_shift];
                    if (static_cast<unsigned>(e) < static_cast<unsigned>(p.n_pages)) slot = (e << p.page_shift) + (t & page_mask);
                    else atomicOr(p.status, kStatusBadPage);
                }
                return slot;
            };
            auto issue = [&](int i) {
                if (!WIDE || (i & 15) == 0) {
                    now = next;
                    next = look(i + (WIDE ? 16 : 1));
                }
                const uint32_t at = (i & (kKv4Stages - 1)) * kKv4StageBytes;
                const uint32_t kd = k_dst + at, vd = v_dst + at, sd = s_dst + at;
                const int left = len - token0(i);
                if constexpr (WIDE) {
                    // A page lies in the pool as a whole: rows behind the length may be addressed, but are not read.
                    const int s0 = __shfl_sync(0xffffffffu, now, (2 * i) & 31), s1 = __shfl_sync(0xffffffffu, now, (2 * i + 1) & 31);
                    if (left >= kKv4Tile && (s0 | s1) >= 0) {
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            const unsigned first = half ? s1 : s0, h = half * kKv4HalfBytes;
                            cp_async16(kd + h, row_of(k_lane, first, code_row));
                            cp_async16(kd + h + 512, row_of(k_lane, first + 8, code_row));
                            cp_async16(vd + h, row_of(v_lane, first, code_row));
                            cp_async16(vd + h + 512, row_of(v_lane, first + 8, code_row));
                            cp_async8(sd + h, row_of(s_lane, first, scale_row));
                        }
                    } else {                              // the end of a request, or no page: what is not read is filled with zeros
#pragma unroll 1
                        for (int half = 0; half < 2; ++half) {
                            const int slot = half ? s1 : s0, n = slot < 0 ? 0 : left - half * 16;
                            const unsigned first = max(slot, 0), h = half * kKv4HalfBytes;
                            const uint32_t n0 = tau < n ? 16u : 0u, n1 = tau + 8 < n ? 16u : 0u;
                            cp_async16(kd + h, row_of(k_lane, first, code_row), n0);
                            cp_async16(kd + h + 512, row_of(k_lane, first + 8, code_row), n1);
                            cp_async16(vd + h, row_of(v_lane, first, code_row), n0);
                            cp_async16(vd + h + 512, row_of(v_lane, first + 8, code_row), n1);
                            cp_async8(sd + h, row_of(s_lane, first, scale_row), ((c & 1) ? n1 : n0) >> 1);
                        }
                    }
                } else {
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const int a = __shfl_sync(0xffffffffu, now, half * 16 + tau), b8 = __shfl_sync(0xffffffffu, now, half * 16 + tau + 8);
                        const uint32_t n0 = a < 0 ? 0u : 16u, n1 = b8 < 0 ? 0u : 16u;
                        const unsigned ua = static_cast<unsigned>(max(a, 0)), ub = static_cast<unsigned>(max(b8, 0));
                        const uint32_t h = half * kKv4HalfBytes;
                        cp_async16(kd + h, row_of(k_lane, ua, code_row), n0);
                        cp_async16(kd + h + 512, row_of(k_lane, ub, code_row), n1);
                        cp_async16(vd + h, row_of(v_lane, ua, code_row), n0);
                        cp_async16(vd + h + 512, row_of(v_lane, ub, code_row), n1);
                        cp_async8(sd + h, row_of(s_lane, (c & 1) ? ub : ua, scale_row), ((c & 1) ? n1 : n0) >> 1);
                    }
                }
            };
            next = look(0);
            issue(0);
            cp_async_commit();

            // ---- queries: column g of each 8, dimensions 32 c .. 32 c + 31, as fp16 scaled by a power of two
            uint32_t qf[NT == 1 ? 16 : 1];
            float mul[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const int col = cc * C + n * 8 + g;
                uint4 v[4];
                uint32_t top = 0;
                if (col < p.cols) {
                    const int j = p.by_group(col), h = kvh * p.group + (col - j * p.group);
                    const uint4* src = reinterpret_cast<const uint4*>(p.q + (static_cast<long long>(b) * p.n_q + j) * p.q_stride + h * 128 + c * 32);
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[i] = src[i];
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[i] = make_uint4(0u, 0u, 0u, 0u);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    top = __vmaxu2(top, __vmaxu2(__vmaxu2(v[i].x & 0x7fff7fffu, v[i].y & 0x7fff7fffu), __vmaxu2(v[i].z & 0x7fff7fffu, v[i].w & 0x7fff7fffu)));
                top = max(top & 0xffffu, top >> 16);
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
                int e = static_cast<int>(top >> 7);                                 // biased exponent of the largest value
                e = e == 255 ? 127 + 14 : max(e, 127 + 14 - 100);                   // not finite: as it is; tiny rows: at most 2^100
                const float f = __uint_as_float(static_cast<uint32_t>(127 + 14 - e + 127) << 23);
                const float undo = __uint_as_float(static_cast<uint32_t>(e - 14) << 23);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint4 h = make_uint4(pack_f16x2(bf16lo(v[i].x) * f, bf16hi(v[i].x) * f), pack_f16x2(bf16lo(v[i].y) * f, bf16hi(v[i].y) * f),
                                               pack_f16x2(bf16lo(v[i].z) * f, bf16hi(v[i].z) * f), pack_f16x2(bf16lo(v[i].w) * f, bf16hi(v[i].w) * f));
                    if constexpr (NT == 1) qf[4 * i] = h.x, qf[4 * i + 1] = h.y, qf[4 * i + 2] = h.z, qf[4 * i + 3] = h.w;
                    else q_smem[(n * 4 + i) * 32] = h;       // read back by this lane alone
                }
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    mul[n][k] = __shfl_sync(0xffffffffu, undo, (2 * c + k) * 4) * p.scale_log2;
                    if (mul[n][k] == 0.f) mul[n][k] = 1e-30f;                       // scores of zero all the same; masks need a sign
                }
            }
            const int full = len - p.n_q + 1;             // tokens that every column attends

            for (int i = 0; i < n_tiles; ++i) {
                cp_async_wait<0>();
                __syncwarp();
                if (i + 1 < n_tiles) issue(i + 1);
                cp_async_commit();
                const uint8_t* s0 = ring_ptr + (i & (kKv4Stages - 1)) * kKv4StageBytes;
                const int t0 = token0(i);
                if (t0 >= len) continue;

                // ---- scores
                float sc[2][NT][4];
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const uint8_t* s = s0 + half * kKv4HalfBytes;
                    const uint4 ka = *reinterpret_cast<const uint4*>(s + lane * 16), kb = *reinterpret_cast<const uint4*>(s + 512 + lane * 16);
                    const uint32_t ha = e4m3x2_to_f16(*reinterpret_cast<const uint16_t*>(s + 2048 + tau * 8 + c * 2));
                    const uint32_t hb = e4m3x2_to_f16(*reinterpret_cast<const uint16_t*>(s + 2048 + 64 + tau * 8 + c * 2));
                    const uint32_t aw[4] = {ka.x, ka.y, ka.z, ka.w}, bw[4] = {kb.x, kb.y, kb.z, kb.w};
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint32_t sa = __byte_perm(ha, ha, k < 2 ? 0x1010 : 0x3232), sb = __byte_perm(hb, hb, k < 2 ? 0x1010 : 0x3232);
                        uint32_t a[4], bq[4];
                        e2m1x8_to_f16(aw[k], a);
                        e2m1x8_to_f16(bw[k], bq);
#pragma unroll
                        for (int u = 0; u < 4; ++u) a[u] = hmul2_f16(a[u], sa), bq[u] = hmul2_f16(bq[u], sb);
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            uint4 q;
                            if constexpr (NT == 1) q = make_uint4(qf[4 * k], qf[4 * k + 1], qf[4 * k + 2], qf[4 * k + 3]);
                            else q = q_smem[(n * 4 + k) * 32];
                            if (k == 0) mma_f16_first(sc[half][n], a[0], bq[0], a[1], bq[1], q.x, q.y);
                            else mma_f16(sc[half][n], a[0], bq[0], a[1], bq[1], q.x, q.y);
                            mma_f16(sc[half][n], a[2], bq[2], a[3], bq[3], q.z, q.w);
                        }
                    }
                }
                if (t0 + kKv4Tile > full) {               // a token that some column does not attend: its score becomes -inf
#pragma unroll
                    for (int half = 0; half < 2; ++half)
#pragma unroll
                        for (int n = 0; n < NT; ++n)
#pragma unroll
                            for (int k = 0; k < 4; ++k)
                                if (t0 + half * 16 + tau + (k >> 1) * 8 >= full + min((cc * C + n * 8 + 2 * c + (k & 1)) / p.group, p.n_q - 1)) sc[half][n][k] = copysignf(INFINITY, -mul[n][k & 1]);
                }
                float e[2][NT][4];
                float high = kKv4Low;
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        e[0][n][k] = fmaf(sc[0][n][k], mul[n][k & 1], -st.m[n][k & 1]);
                        e[1][n][k] = fmaf(sc[1][n][k], mul[n][k & 1], -st.m[n][k & 1]);
                        high = fmax3(high, e[0][n][k], e[1][n][k]);
                    }
                if (__any_sync(0xffffffffu, high > kKv4Lag)) {
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            const float u = mul[n][k];
                            float top = fmaxf(fmaxf(sc[0][n][k] * u, sc[0][n][k + 2] * u), fmaxf(sc[1][n][k] * u, sc[1][n][k + 2] * u));
                            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                            const float m2 = fmaxf(st.m[n][k], top - kKv4Lift);
                            const float f = m2 == st.m[n][k] ? 1.f : ex2_approx(st.m[n][k] - m2);
                            st.m[n][k] = m2;
                            st.l[n][k] *= f;
#pragma unroll
                            for (int d = 0; d < 8; ++d) st.o[d][n][k] *= f, st.o[d][n][k + 2] *= f;
#pragma unroll
                            for (int half = 0; half < 2; ++half)
                                e[half][n][k] = fmaf(sc[half][n][k], u, -m2), e[half][n][k + 2] = fmaf(sc[half][n][k + 2], u, -m2);
                        }
                }
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    uint32_t pf[NT][2];
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        const float e0 = ex2_approx(e[half][n][0]), e1 = ex2_approx(e[half][n][1]), e2 = ex2_approx(e[half][n][2]), e3 = ex2_approx(e[half][n][3]);
                        st.l[n][0] += e0 + e2;
                        st.l[n][1] += e1 + e3;
                        // Rows of the score tile become the k index of the second product: tokens c, c + 4 and c + 8, c + 12 of lane c.
                        pf[n][0] = movmatrix_trans(pack_f16x2(e0, e1));
                        pf[n][1] = movmatrix_trans(pack_f16x2(e2, e3));
                    }

                    // ---- O^T += V^T P^T: this lane has dimensions 16 g .. 16 g + 15 of tokens c, c + 4, c + 8, c + 12
                    const uint8_t* s = s0 + half * kKv4HalfBytes;
                    const uint8_t* vp = s + 1024 + c * 64 + (((g >> 1) ^ (c & 2)) << 4) + (g & 1) * 8;
                    const uint2 v0 = *reinterpret_cast<const uint2*>(vp), v1 = *reinterpret_cast<const uint2*>(vp + 256), v2 = *reinterpret_cast<const uint2*>(vp + 512), v3 = *reinterpret_cast<const uint2*>(vp + 768);
                    const uint8_t* sp = s + 2048 + 128 + c * 8 + g;
                    const uint32_t sa = e4m3x2_to_f16(sp[0] | (static_cast<uint32_t>(sp[32]) << 8)), sb = e4m3x2_to_f16(sp[64] | (static_cast<uint32_t>(sp[96]) << 8));
#pragma unroll
                    for (int word = 0; word < 2; ++word) {
                        const uint32_t w0 = word ? v0.y : v0.x, w1 = word ? v1.y : v1.x, w2 = word ? v2.y : v2.x, w3 = word ? v3.y : v3.x;
                        uint32_t a[2][4], bq[2][4];       // [even / odd dimensions][pair]
                        e2m1x8_to_f16(bit_select(w0, w1 << 4, 0x0f0f0f0fu), a[0]);
                        e2m1x8_to_f16(bit_select(w0 >> 4, w1, 0x0f0f0f0fu), a[1]);
                        e2m1x8_to_f16(bit_select(w2, w3 << 4, 0x0f0f0f0fu), bq[0]);
                        e2m1x8_to_f16(bit_select(w2 >> 4, w3, 0x0f0f0f0fu), bq[1]);
#pragma unroll
                        for (int q = 0; q < 2; ++q)
#pragma unroll
                            for (int u = 0; u < 2; ++u) {
                                const uint32_t a0 = hmul2_f16(a[q][2 * u], sa), a1 = hmul2_f16(a[q][2 * u + 1], sa);
                                const uint32_t a2 = hmul2_f16(bq[q][2 * u], sb), a3 = hmul2_f16(bq[q][2 * u + 1], sb);
#pragma unroll
                                for (int n = 0; n < NT; ++n) mma_f16(st.o[word * 4 + q * 2 + u][n], a0, a1, a2, a3, pf[n][0], pf[n][1]);
                            }
                    }
                }
            }
            cp_async_wait<0>();
            __syncwarp();
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    st.l[n][k] += __shfl_xor_sync(0xffffffffu, st.l[n][k], 4);
                    st.l[n][k] += __shfl_xor_sync(0xffffffffu, st.l[n][k], 8);
                    st.l[n][k] += __shfl_xor_sync(0xffffffffu, st.l[n][k], 16);
                }
        }
        // ---- join the token lanes of a head (its ring is free by now)
        if (p.ts > 1) {
            if (active && tl > 0) {
#pragma unroll
                for (int i = 0; i < 8; ++i)
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int k = 0; k < 4; ++k) reinterpret_cast<float*>(ring_ptr)[(((i * NT + n) * 4 + k) * 32 + lane)] = st.o[i][n][k];
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        reinterpret_cast<float*>(ring_ptr)[((32 * NT + n * 4 + k) * 32 + lane)] = st.m[n][k];
                        reinterpret_cast<float*>(ring_ptr)[((32 * NT + n * 4 + 2 + k) * 32 + lane)] = st.l[n][k];
                    }
            }
            __syncthreads();
            if (active && tl == 0) {
                for (int t = 1; t < p.ts; ++t) {
                    const float* from = reinterpret_cast<const float*>(smem + (t * p.hg + hl) * kKv4WarpBytes<NT>);
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            const float om = from[((32 * NT + n * 4 + k) * 32 + lane)], ol = from[((32 * NT + n * 4 + 2 + k) * 32 + lane)];
                            const float m2 = fmaxf(st.m[n][k], om);
                            const float fa = st.m[n][k] == m2 ? 1.f : ex2_approx(st.m[n][k] - m2), fb = om == m2 ? 1.f : ex2_approx(om - m2);
                            st.m[n][k] = m2;
                            st.l[n][k] = st.l[n][k] * fa + ol * fb;
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                st.o[i][n][k] = st.o[i][n][k] * fa + from[(((i * NT + n) * 4 + k) * 32 + lane)] * fb;
                                st.o[i][n][k + 2] = st.o[i][n][k + 2] * fa + from[(((i * NT + n) * 4 + k + 2) * 32 + lane)] * fb;
                            }
                        }
                }
            }
            __syncthreads();
        }
        if (active && tl == 0) {
            // Dimension 16 g + d of column 2 c + k sits in st.o[(d >> 3) * 4 + (d & 1) * 2 + ((d >> 2) & 1)][n][k + (d & 2)].
            const int slot = tile0 == 0 ? 1 : 0;          // of this block's two records: the segment that began before it, or the one that goes on
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const int cl = n * 8 + 2 * c + k, col = cc * C + cl;
                    if (col >= p.cols) continue;
                    float v[16];
#pragma unroll
                    for (int d = 0; d < 16; ++d) v[d] = st.o[(d >> 3) * 4 + (d & 1) * 2 + ((d >> 2) & 1)][n][k + (d & 2)];
                    const float l = st.l[n][k], m = st.m[n][k];
                    if (whole) {
                        const int j = p.by_group(col), h = kvh * p.group + (col - j * p.group);
                        const long long at = static_cast<long long>(b) * p.n_q + j;
                        const float inv = l == 0.f ? 0.f : p.v_scale / l;          // a not-a-number goes through
                        uint4* dst = reinterpret_cast<uint4*>(p.out + at * p.out_stride + h * 128 + g * 16);
                        dst[0] = make_uint4(pack_bf16x2(v[0] * inv, v[1] * inv), pack_bf16x2(v[2] * inv, v[3] * inv),
                                            pack_bf16x2(v[4] * inv, v[5] * inv), pack_bf16x2(v[6] * inv, v[7] * inv));
                        dst[1] = make_uint4(pack_bf16x2(v[8] * inv, v[9] * inv), pack_bf16x2(v[10] * inv, v[11] * inv),
                                            pack_bf16x2(v[12] * inv, v[13] * inv), pack_bf16x2(v[14] * inv, v[15] * inv));
                        if (p.lse != nullptr && g == 0)
                            p.lse[at * p.nh_q + h] = l == 0.f ? -INFINITY : m * 0.6931471805599453f + logf(l);
                    } else {
                        float* rec = p.rec + (((static_cast<long long>(blockIdx.x) * 2 + slot) * p.hg + hl) * C + cl) * kKv4RecFloats;
                        float4* dst = reinterpret_cast<float4*>(rec + g * 16);
#pragma unroll
                        for (int i = 0; i < 4; ++i) dst[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
                        if (g == 0) *reinterpret_cast<float2*>(rec + 128) = make_float2(m, l);
                    }
                }
        }
        x += taken;
    }
}

// Joins the records of the segments that more than one block had a part of: one block of NW warps per output row.  Every warp folds
// its records four at a time, maximum, sum and O loaded together, and the warps' results meet in shared memory: one way to
// memory instead of two (maxima first), 1 us of the launch.
template <int NT, int NW>
__global__ void __launch_bounds__(NW * 32) kv4_merge_kernel(const Kv4AttnParams p, int grid) {
    constexpr int C = 8 * NT;
    __shared__ float part[NW][128];
    __shared__ float2 ml[NW];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    grid_wait();
    grid_trigger();
    const int token = p.by_nh_q(blockIdx.x), h = blockIdx.x - token * p.nh_q, b = p.by_n_q(token), j = token - b * p.n_q;
    const int kvh = p.by_group(h), col = j * p.group + (h - kvh * p.group);
    const int hgi = p.by_hg(kvh), hl = kvh - hgi * p.hg, cc = col / C, cl = col - cc * C;
    const int first = p.cum[b], tiles = p.cum[b + 1] - first, per_tile = p.n_hg * p.n_cc;
    const int total = p.cum[p.batch] * per_tile;
    const Kv4Deal deal(total, kv4_blocks(total, p.batch * per_tile, grid), grid, p.by_grid);
    const int s0 = first * per_tile + (hgi * p.n_cc + cc) * tiles;
    const int i0 = deal.owner(s0), n = deal.owner(s0 + tiles - 1) - i0 + 1;
    if (n == 1) return;
    // The segment's first block has it as the one that goes on behind its share; for the others it began before theirs.
    const long long step = 2ll * p.hg * C * kKv4RecFloats;
    const float* rec0 = p.rec + ((static_cast<long long>(i0) * 2 * p.hg + hl) * C + cl) * kKv4RecFloats;
    const long long goes_on = static_cast<long long>(p.hg) * C * kKv4RecFloats;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    float own = kKv4Low, own_sum = 0.f;
    for (int first_of_4 = w; first_of_4 < n; first_of_4 += 4 * NW) {
        float2 m[4];
        float4 v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int i = first_of_4 + u * NW;
            m[u] = make_float2(kKv4Low, 0.f), v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (i >= n) continue;
            const float* r = rec0 + i * step + (i == 0 ? goes_on : 0);
            m[u] = *reinterpret_cast<const float2*>(r + 128);
            v[u] = *reinterpret_cast<const float4*>(r + lane * 4);
        }
        const float t = fmaxf(fmaxf(fmaxf(m[0].x, m[1].x), fmaxf(m[2].x, m[3].x)), own), keep = ex2_approx(own - t);
        own = t;
        o.x *= keep, o.y *= keep, o.z *= keep, o.w *= keep, own_sum *= keep;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const float f = ex2_approx(m[u].x - t);
            o.x += v[u].x * f, o.y += v[u].y * f, o.z += v[u].z * f, o.w += v[u].w * f;
            own_sum += m[u].y * f;
        }
    }
    *reinterpret_cast<float4*>(&part[w][lane * 4]) = o;
    if (lane == 0) ml[w] = make_float2(own, own_sum);
    __syncthreads();
    const int d = threadIdx.x;
    if (d >= 128) return;
    float top = kKv4Low, sum = 0.f, acc = 0.f;
#pragma unroll
    for (int i = 0; i < NW; ++i) top = fmaxf(top, ml[i].x);
#pragma unroll
    for (int i = 0; i < NW; ++i) {
        const float f = ex2_approx(ml[i].x - top);
        acc += part[i][d] * f, sum += ml[i].y * f;
    }
    const float inv = sum == 0.f ? 0.f : p.v_scale / sum;
    const long long at = static_cast<long long>(b) * p.n_q + j;
    p.out[at * p.out_stride + h * 128 + d] = __float2bfloat16_rn(acc * inv);
    if (p.lse != nullptr && d == 0) p.lse[at * p.nh_q + h] = sum == 0.f ? -INFINITY : top * 0.6931471805599453f + logf(sum);
}

}  // namespace dkv
