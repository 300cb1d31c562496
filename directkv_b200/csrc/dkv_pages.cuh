// Page tables and slot maps from request lengths, on the GPU.
//
// The free pages are a stack in device memory: free_pages[0 .. n_free).  Request b (row r of the page table) has
// a_b tokens on ceil(a_b / P) pages and gets n_b more.  Pages are taken in request order, then in page order, from the
// top of the stack: the i-th page taken is free_pages[n_free - 1 - i].  The packed new tokens get their positions
// a_b + j and their slots page * P + position % P.  Places behind the last new token (a captured call has room for the most
// that it may get) hold no token: a slot there becomes -1, which store and load pass over, and a position 0; what is negative already
// is left.  Without that a later step would store its padding rows into the slots of an earlier one.  Release puts the pages of
// the tokens [keep_b, len_b) back so that
// a release of exactly what the last call took restores the stack.
//
// A call takes effect as a whole or not at all: too few pages, a row or length outside the table, or more tokens
// than the caller has room for leave stack, table and lengths as they were, give slots of -1, and set a status bit.  So do two
// requests that change one row (they would share its new pages, or free its old ones twice); requests that change nothing, the padding
// of a batch, may repeat a row.
#pragma once

#include "dkv_common.cuh"

namespace dkv {

constexpr int kPagesThreads = 512;
constexpr int kPagesMaxBatch = 4096;

struct PagesParams {
    int* page_table;
    long long pt_stride;
    int pt_rows;
    int max_pages;                   // pages a row of the table has room for
    const int* rows;                 // [batch] or nullptr
    const int* lens;                 // [batch] assign: tokens before; release: tokens before the release
    const int* more;                 // [batch] assign: new tokens; release: tokens that stay
    int batch;
    int page_shift;
    int* free_pages;
    int free_cap;
    int* n_free;
    int* slots;                      // assign only, [capacity]
    int* positions;                  // [capacity] or nullptr
    long long capacity;
    int fresh;                       // bit 0: slots, bit 1: positions hold nothing yet
    int vector;                      // slots and positions are 16-byte aligned
    int* seq_lens;                   // [batch]: lens + more
    int* cu_new;                     // [batch + 1]
    unsigned int* status;
    unsigned int* ticket;            // zero between launches
};

// Block-wide exclusive prefix of (a, b) pairs over the threads; totals in *ta, *tb.  All threads of the block.
__device__ __forceinline__ void block_scan2(long long& a, long long& b, long long* sh, long long* ta, long long* tb) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    long long ia = a, ib = b;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long xa = __shfl_up_sync(0xffffffffu, ia, o), xb = __shfl_up_sync(0xffffffffu, ib, o);
        if (lane >= o) ia += xa, ib += xb;
    }
    __syncthreads();
    if (lane == 31) sh[w] = ia, sh[32 + w] = ib;
    __syncthreads();
    long long pa = 0, pb = 0, sa = 0, sb = 0;
    for (int i = 0; i < kPagesThreads / 32; ++i) {
        if (i == w) pa = sa, pb = sb;
        sa += sh[i], sb += sh[32 + i];
    }
    a = pa + ia - a;
    b = pb + ib - b;
    *ta = sa, *tb = sb;
}

// Bound by latency: one scan, one search and one look-up per thread.  64 requests with one more token each and their release take
// 8.7 us in two launches, 256 prompts of 1.0 M tokens 15 us (8 MB of slots and positions; two blocks per SM, which scan the batch
// side by side, 17 us); the look for repeated rows is 0.3 and 0.7 us of a launch.
template <bool RELEASE>
__global__ void __launch_bounds__(kPagesThreads) pages_kernel(const PagesParams p) {
    __shared__ int cu_tok[2 * (kPagesMaxBatch + 1)]; // (release: first half unused)
    int* const cu_page = cu_tok + kPagesMaxBatch + 1;
    __shared__ long long sh[64];
    __shared__ int sh_last;
    grid_wait();
    grid_trigger();
    const int P = 1 << p.page_shift;
    const int top = *reinterpret_cast<const volatile int*>(p.n_free);
    bool bad = top < 0 || top > p.free_cap;
    if (p.rows != nullptr && p.batch > 1) {
        // The rows that change go into a hash table of at least twice as many places, in the room of the prefix sums.
        const int bits = 33 - __clz(p.batch - 1), mask = (1 << bits) - 1;
        for (int i = threadIdx.x; i <= mask; i += kPagesThreads) cu_tok[i] = -1;
        __syncthreads();
        for (int b = threadIdx.x; b < p.batch; b += kPagesThreads) {
            const int row = p.rows[b], x = p.more[b];
            const bool changes = RELEASE ? (p.lens[b] + P - 1ll) >> p.page_shift > (x + P - 1ll) >> p.page_shift : x > 0;
            if (!changes || row < 0) continue;
            for (unsigned at = (static_cast<unsigned>(row) * 0x9E3779B1u) >> (32 - bits);; at = (at + 1) & mask) {
                const int other = atomicCAS(&cu_tok[at], -1, row);
                bad |= other == row;
                if (other == row || other == -1) break;
            }
        }
        __syncthreads();
    }
    long long tok = 0, pages = 0;
    // Every block scans the whole batch (a few thousand integers at most): no launch and no hand-over between
    // the scan and the fill.
    for (int b0 = 0; b0 < p.batch; b0 += kPagesThreads) {
        const int b = b0 + threadIdx.x;
        long long n = 0, m = 0;
        if (b < p.batch) {
            const long long len = p.lens[b], x = p.more[b];
            const long long after = RELEASE ? x : len + x;
            const long long row = p.rows != nullptr ? p.rows[b] : b;
            bool wrong = len < 0 || x < 0 || row < 0 || row >= p.pt_rows || (RELEASE && x > len);
            const long long have = (len + P - 1) >> p.page_shift, need = (after + P - 1) >> p.page_shift;
            wrong |= (RELEASE ? have : need) > p.max_pages;
            bad |= wrong;
            if (!wrong) {
                n = RELEASE ? 0 : x;
                m = RELEASE ? have - need : need - have;
            }
        }
        long long tt, tp;
        block_scan2(n, m, sh, &tt, &tp);
        if (b < p.batch) {
            cu_tok[b] = static_cast<int>(tok + n);
            cu_page[b] = static_cast<int>(pages + m);
        }
        tok += tt, pages += tp;
    }
    bool short_of = false, full = false;
    if (RELEASE) full = top + pages > p.free_cap;
    else short_of = pages > top, full = tok > p.capacity;
    bad = __syncthreads_or(bad) != 0;
    const bool ok = !bad && !short_of && !full;
    if (threadIdx.x == 0) {
        cu_tok[p.batch] = static_cast<int>(tok);
        cu_page[p.batch] = static_cast<int>(pages);
    }
    __syncthreads();
    const long long stride = static_cast<long long>(gridDim.x) * blockDim.x;
    const long long me = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        if (bad) atomicOr(p.status, kStatusBadPage);
        if (short_of) atomicOr(p.status, kStatusOutOfPages);
        if (full) atomicOr(p.status, kStatusBadSlot);
    }
    if constexpr (!RELEASE) {
        if (!ok) {
            for (long long v = me; v < p.capacity; v += stride) {
                p.slots[v] = -1;
                if (p.positions != nullptr) p.positions[v] = 0;
            }
        } else {
            // Four tokens per thread: one search, and one look at the table or the stack as long as the page is the same.
            for (long long v0 = me * 4; v0 < tok; v0 += stride * 4) {
                int lo = 0, hi = p.batch - 1;         // largest b with cu_tok[b] <= v0 (empty requests fall out)
                while (lo < hi) {
                    const int mid = (lo + hi + 1) >> 1;
                    if (cu_tok[mid] <= v0) lo = mid;
                    else hi = mid - 1;
                }
                const int n = static_cast<int>(min(tok - v0, 4ll));
                int slot[4], where[4], len = 0, have = 0, page = -1, number = 0;
                int* line = nullptr;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (i >= n) break;
                    const int v = static_cast<int>(v0) + i;
                    while (v >= cu_tok[lo + 1]) ++lo, line = nullptr;
                    if (line == nullptr) {
                        len = p.lens[lo];
                        have = static_cast<int>((static_cast<long long>(len) + P - 1) >> p.page_shift);
                        line = p.page_table + (p.rows != nullptr ? p.rows[lo] : lo) * p.pt_stride;
                        page = -1;
                    }
                    const int pos = len + (v - cu_tok[lo]), pg = pos >> p.page_shift;
                    if (pg != page) {
                        page = pg;
                        number = pg >= have ? p.free_pages[top - 1 - (cu_page[lo] + pg - have)] : line[pg];
                        if (number < 0 || number > (0x7fffffff >> p.page_shift)) atomicOr(p.status, kStatusBadPage);   // no slot
                    }
                    if (pg >= have && (pos & (P - 1)) == 0) line[pg] = number;
                    slot[i] = number >= 0 && number <= (0x7fffffff >> p.page_shift) ? number * P + (pos & (P - 1)) : -1;
                    where[i] = pos;
                }
                if (n == 4 && p.vector) {
                    *reinterpret_cast<int4*>(p.slots + v0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
                    if (p.positions != nullptr) *reinterpret_cast<int4*>(p.positions + v0) = make_int4(where[0], where[1], where[2], where[3]);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (i >= n) break;
                        p.slots[v0 + i] = slot[i];
                        if (p.positions != nullptr) p.positions[v0 + i] = where[i];
                    }
                }
            }
            for (long long v = tok + me; v < p.capacity; v += stride) {
                if ((p.fresh & 1) || p.slots[v] >= 0) p.slots[v] = -1;
                if (p.positions != nullptr && ((p.fresh & 2) || p.positions[v] >= 0)) p.positions[v] = 0;
            }
        }
    } else if (ok) {
        for (long long i = me; i < pages; i += stride) {
            int lo = 0, hi = p.batch - 1;
            while (lo < hi) {
                const int mid = (lo + hi + 1) >> 1;
                if (cu_page[mid] <= i) lo = mid;
                else hi = mid - 1;
            }
            const int keep = static_cast<int>((static_cast<long long>(p.more[lo]) + P - 1) >> p.page_shift);
            const int pg = keep + static_cast<int>(i - cu_page[lo]);
            p.free_pages[top + pages - 1 - i] = p.page_table[(p.rows != nullptr ? p.rows[lo] : lo) * p.pt_stride + pg];
        }
    }
    // The stack's height and the lengths (which may be updated in place) change once every block has read them: the
    // block that finishes last writes them.
    if (gridDim.x > 1) {
        __syncthreads();
        if (threadIdx.x == 0) {
            __threadfence();
            sh_last = atomicAdd(p.ticket, 1u) == gridDim.x - 1;
        }
        __syncthreads();
        if (!sh_last) return;
    } else {
        __syncthreads();
    }
    if constexpr (!RELEASE) {
        for (int b = threadIdx.x; b <= p.batch; b += blockDim.x) {
            p.cu_new[b] = ok ? cu_tok[b] : 0;
            if (b < p.batch) p.seq_lens[b] = p.lens[b] + (ok ? p.more[b] : 0);
        }
    }
    if (threadIdx.x == 0) {
        if (ok) *p.n_free = RELEASE ? top + static_cast<int>(pages) : top - static_cast<int>(pages);
        if (gridDim.x > 1) *p.ticket = 0u;
    }
}

}  // namespace dkv
