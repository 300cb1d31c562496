// C entry points of the operators around a 4-bit paged cache: store, load and attention, head norms with rotation,
// page tables.  Part of dkv_capi.cu (it uses that file's context and error helpers).
#pragma once

namespace {

// Makes the context's device current for the launches of one call and puts the caller's back.
struct DeviceScope {
    int before = -1;
    cudaError_t err;
    explicit DeviceScope(int device) {
        err = cudaGetDevice(&before);
        if (err == cudaSuccess && before != device) err = cudaSetDevice(device);
        else before = -1;
    }
    ~DeviceScope() {
        if (before >= 0) cudaSetDevice(before);
    }
};

// Launches a kernel that begins with grid_wait() so that its set-up overlaps the end of the kernel before it.
template <typename... KernelArgs, typename... Args>
cudaError_t launch_overlapped(void (*kernel)(KernelArgs...), unsigned grid, unsigned block, size_t smem, cudaStream_t st, Args... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

#define DKV_ON_DEVICE(ctx)              \
    DeviceScope device_scope((ctx)->device); \
    DKV_CUDA(device_scope.err)

bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

int log2_of(int v) {
    int s = 0;
    while ((1 << s) < v) ++s;
    return s;
}

int check_kv4_pool(const dkv_context* ctx, const dkv_kv4_pool* pool) {
    DKV_REQUIRE(pool->resolved == ctx->device + 1, "the 4-bit pool was not resolved for device %d (dkv_kv4_pool_resolve)", ctx->device);
    return DKV_OK;
}

// How a launch cuts its work: heads (hg) and token lanes (ts) of a block of W warps, and whether segments are left whole.
//  - By default as many warps as the number of heads allows, and of the shapes that use them the one with the most
//    heads side by side, whose rows of a token are read together.
//  - Where the page table has room for a few steps only (`room` tokens), nothing is split: a second launch and the
//    records' way through memory cost more than a few steps one behind the other.  With blocks to spare, token lanes make it
//    fewer steps (32 query heads on 8, one request of 77 tokens: 4.7 us as one step of four lanes, 6.3 us split).  Two steps are
//    always left whole, four where the segments occupy a fifth of the grid (64 requests of 512 tokens: 12.6 us, split 18.6; of
//    1 to 512 tokens: 12.0, split 17.1; 8 of 1024 tokens: 9.2, split 10.9; but one request of 1024 tokens: 8.7, split 7.5), eight
//    of the plain shape with half a grid of segments (64 requests of 256 tokens, 32 heads: 20.9 us, split 26.6).
//  - Very few segments (one long request): two heads per block and the other warps as token lanes, joined in the block, leave
//    a quarter of the records to merge (131071 tokens: 38.0 us, 39.7 us with eight heads).
template <int NT>
void kv4_shape(int batch, int nh_kv, int n_cc, int64_t room, int grid, int* hg, int* ts, int* whole) {
    constexpr int W = kKv4Warps<NT>;
    int best = 0;
    for (int h = 1; h <= W; ++h) {
        if (nh_kv % h != 0) continue;
        const int t = W / h;
        if (h * t >= best) best = h * t, *hg = h, *ts = t;
    }
    auto segments = [&](int h) { return static_cast<int64_t>(batch) * (nh_kv / h) * n_cc; };
    auto steps = [&](int t) { return (room + static_cast<int64_t>(kKv4Tile) * t - 1) / (static_cast<int64_t>(kKv4Tile) * t); };
    *whole = 0;
    int h0 = *hg, t0 = *ts;
    for (int t = t0; t <= W; ++t) {                       // the fewest lanes that give the fewest steps
        const int h = W / t;
        if (h * t != W || nh_kv % h != 0 || segments(h) > grid) continue;
        if (steps(t) < steps(t0)) h0 = h, t0 = t;
    }
    if (steps(t0) <= 2 || (steps(t0) <= 4 && 5 * segments(h0) >= grid)) *hg = h0, *ts = t0, *whole = 1;
    else if (2 * segments(*hg) >= grid) *whole = steps(*ts) <= 8;
    else if (segments(*hg) <= 8 && *hg > 2 && nh_kv % 2 == 0) *hg = 2, *ts = W / 2;
}

constexpr size_t kKv4CumBytes = (kKv4LaunchBatch + 1) * sizeof(int) / 256 * 256 + 256;

template <int NT>
int kv4_grid(const dkv_context* ctx) {
    return ctx->sm_count * kKv4BlocksPerSm<NT>;
}

// One size for every call, so that any call (or registering a pool) makes room for all of them.
size_t kv4_workspace(const dkv_context* ctx) {
    const size_t cols = std::max(kv4_grid<1>(ctx) * kKv4Warps<1> * 8, kv4_grid<2>(ctx) * kKv4Warps<2> * 16);
    return kKv4CumBytes + cols * 2 * kKv4RecFloats * sizeof(float);
}

template <int NT>
int launch_kv4_attn(dkv_context* ctx, Kv4AttnParams& p, cudaStream_t st) {
    p.n_cc = (p.cols + 8 * NT - 1) / (8 * NT);
    const int full_grid = kv4_grid<NT>(ctx);
    kv4_shape<NT>(p.batch, p.nh_kv, p.n_cc, p.room, full_grid, &p.hg, &p.ts, &p.whole);
    p.n_hg = p.nh_kv / p.hg;
    p.tile_shift = log2_of(kKv4Tile * p.ts);
    const int64_t most_parts = p.room / (kKv4Tile * p.ts) + 1;
    const int64_t most_tiles = (p.whole ? 1 : most_parts) * p.batch * p.n_hg * p.n_cc;
    if (most_tiles > INT32_MAX)
        return fail(DKV_ERR_UNSUPPORTED, "%d requests of up to %lld tokens are too many for one call", p.batch, static_cast<long long>(p.room));
    const int grid = static_cast<int>(std::min<int64_t>(full_grid, most_tiles));
    p.by_seg = Kv4Div(p.n_hg * p.n_cc), p.by_cc = Kv4Div(p.n_cc), p.by_hg = Kv4Div(p.hg), p.by_grid = Kv4Div(grid);
    const size_t smem = kv4_smem<NT>(p.batch);
    const auto kernel = p.page_shift >= 4 ? kv4_attn_kernel<NT, true> : kv4_attn_kernel<NT, false>;
    DKV_CUDA(launch_overlapped(kernel, grid, kKv4Warps<NT> * 32, smem, st, p));
    ctx->launches += 1;
    if (p.whole) return DKV_OK;
    const unsigned rows = static_cast<unsigned>(p.batch) * p.n_q * p.nh_q;
    // Few rows: many blocks had a part of each.
    const bool few = rows <= static_cast<unsigned>(2 * ctx->sm_count) && most_parts > 16;
    DKV_CUDA(launch_overlapped(few ? kv4_merge_kernel<NT, 16> : kv4_merge_kernel<NT, 4>, rows, few ? 512 : 128, 0, st, p, grid));
    ctx->launches += 1;
    return DKV_OK;
}

}  // namespace

extern "C" {

int dkv_kv4_pool_resolve(dkv_context* ctx, dkv_kv4_pool* pool) {
    DKV_REQUIRE(ctx != nullptr && pool != nullptr, "ctx / pool is NULL");
    DKV_REQUIRE(pool->k_codes && pool->k_scales && pool->v_codes && pool->v_scales, "codes and scales must not be NULL");
    DKV_REQUIRE(pool->n_slots > 0 && pool->n_slots <= INT32_MAX && pool->nh_kv > 0 && pool->nh_kv <= 65535,
                "n_slots must be 1..2^31-1 and nh_kv 1..65535");
    DKV_REQUIRE(pool->page_size >= 1 && (pool->page_size & (pool->page_size - 1)) == 0, "page_size (%d) must be a power of two", pool->page_size);
    DKV_REQUIRE(pool->n_slots % pool->page_size == 0, "n_slots (%lld) must be a multiple of page_size (%d)", (long long)pool->n_slots, pool->page_size);
    for (float s : {pool->k_scale, pool->v_scale}) {
        int e = 0;
        DKV_REQUIRE(s > 0.f && frexpf(s, &e) == 0.5f && e >= -23 && e <= 25, "pool scales must be powers of two from 2^-24 to 2^24");
    }
    DKV_REQUIRE(aligned(pool->k_codes, 16) && aligned(pool->v_codes, 16) && aligned(pool->k_scales, 8) && aligned(pool->v_scales, 8),
                "codes must be 16-byte and scales 8-byte aligned");
    DKV_ON_DEVICE(ctx);
    dkv_kv4_pool r = *pool;
    void** parts[4] = {&r.k_codes, &r.k_scales, &r.v_codes, &r.v_scales};
    for (void** p : parts) {
        cudaPointerAttributes attr;
        DKV_CUDA(cudaPointerGetAttributes(&attr, *p));
        DKV_REQUIRE(attr.type != cudaMemoryTypeDevice || attr.device == ctx->device, "a part of the 4-bit pool lives on device %d, not on %d",
                    attr.device, ctx->device);
        int rc = device_pointer_of(*p, p, "a 4-bit pool");
        if (rc != DKV_OK) return rc;
    }
    int rc = ensure_buffer(ctx, &ctx->kv4, kv4_workspace(ctx), false, "workspace of the 4-bit attention");
    if (rc != DKV_OK) return rc;
    r.resolved = ctx->device + 1;
    *pool = r;
    return DKV_OK;
}

static int kv4_rows(dkv_context* ctx, const dkv_kv4_pool* pool, const void* slots, int64_t n_tokens) {
    DKV_REQUIRE(ctx != nullptr && pool != nullptr, "ctx / pool is NULL");
    int rc = check_kv4_pool(ctx, pool);
    if (rc != DKV_OK) return rc;
    DKV_REQUIRE(n_tokens >= 0 && n_tokens <= INT32_MAX, "n_tokens must be 0..2^31-1");
    DKV_REQUIRE(n_tokens == 0 || slots != nullptr, "slots must not be NULL");
    return DKV_OK;
}

static Kv4RowsParams kv4_rows_params(const dkv_context* ctx, const dkv_kv4_pool* pool, const void* slots, int slots64, int64_t n) {
    Kv4RowsParams p{};
    p.k_codes = static_cast<uint8_t*>(pool->k_codes), p.v_codes = static_cast<uint8_t*>(pool->v_codes);
    p.k_scales = static_cast<uint8_t*>(pool->k_scales), p.v_scales = static_cast<uint8_t*>(pool->v_scales);
    p.slots = slots, p.slots64 = slots64;
    p.n = n;
    p.nh = pool->nh_kv;
    p.per_block = std::max(1, kKv4RowThreads / (pool->nh_kv * 8));
    p.n_slots = pool->n_slots;
    p.status = ctx->status;
    return p;
}

int dkv_kv4_store(dkv_context* ctx, const dkv_kv4_pool* pool, const void* slots, int slots_int64, const void* k, int64_t k_stride,
                  const void* v, int64_t v_stride, int64_t n_tokens, void* stream) {
    int rc = kv4_rows(ctx, pool, slots, n_tokens);
    if (rc != DKV_OK || n_tokens == 0) return rc;
    DKV_REQUIRE(k != nullptr && v != nullptr && aligned(k, 16) && aligned(v, 16), "k / v must be 16-byte aligned device pointers");
    const int64_t row = static_cast<int64_t>(pool->nh_kv) * 128;
    DKV_REQUIRE(k_stride >= row && v_stride >= row && k_stride % 8 == 0 && v_stride % 8 == 0, "k / v strides too small or unaligned");
    Kv4RowsParams p = kv4_rows_params(ctx, pool, slots, slots_int64, n_tokens);
    p.k = static_cast<const __nv_bfloat16*>(k), p.v = static_cast<const __nv_bfloat16*>(v);
    p.k_stride = k_stride, p.v_stride = v_stride;
    p.k_scale = 1.f / pool->k_scale, p.v_scale = 1.f / pool->v_scale;
    p.wide = aligned(k, 32) && aligned(v, 32) && k_stride % 16 == 0 && v_stride % 16 == 0;
    DKV_ON_DEVICE(ctx);
    DKV_CUDA(launch_overlapped(kv4_store_kernel, static_cast<unsigned>((n_tokens + p.per_block - 1) / p.per_block), kKv4RowThreads, 0, static_cast<cudaStream_t>(stream), p));
    ctx->launches += 1;
    return DKV_OK;
}

int dkv_kv4_load(dkv_context* ctx, const dkv_kv4_pool* pool, const void* slots, int slots_int64, void* k, void* v, int64_t n_tokens,
                 void* stream) {
    int rc = kv4_rows(ctx, pool, slots, n_tokens);
    if (rc != DKV_OK || n_tokens == 0) return rc;
    DKV_REQUIRE(k != nullptr && v != nullptr && aligned(k, 16) && aligned(v, 16), "k / v must be 16-byte aligned device pointers");
    Kv4RowsParams p = kv4_rows_params(ctx, pool, slots, slots_int64, n_tokens);
    p.k_out = static_cast<__nv_bfloat16*>(k), p.v_out = static_cast<__nv_bfloat16*>(v);
    p.k_scale = pool->k_scale, p.v_scale = pool->v_scale;
    p.wide = aligned(k, 32) && aligned(v, 32);
    DKV_ON_DEVICE(ctx);
    DKV_CUDA(launch_overlapped(kv4_load_kernel, static_cast<unsigned>((n_tokens + p.per_block - 1) / p.per_block), kKv4RowThreads, 0, static_cast<cudaStream_t>(stream), p));
    ctx->launches += 1;
    return DKV_OK;
}

int dkv_decode_kv4(dkv_context* ctx, const dkv_kv4_pool* pool, const dkv_decode_kv4_args* a, void* stream) {
    DKV_REQUIRE(ctx != nullptr && pool != nullptr && a != nullptr, "ctx / pool / args is NULL");
    int rc = check_kv4_pool(ctx, pool);
    if (rc != DKV_OK) return rc;
    if (a->batch == 0) return DKV_OK;
    DKV_REQUIRE(a->batch > 0 && a->batch <= kKv4MaxBatch, "batch (%d) must be 0..%d", a->batch, kKv4MaxBatch);
    DKV_REQUIRE(a->n_q >= 1 && a->n_q <= 1024, "query tokens per request (%d) must be 1..1024", a->n_q);
    DKV_REQUIRE(a->nh_q > 0 && a->nh_q % pool->nh_kv == 0, "nh_q (%d) must be a multiple of nh_kv (%d)", a->nh_q, pool->nh_kv);
    DKV_REQUIRE(a->q && a->out && a->seq_lens && a->page_table, "q / out / seq_lens / page_table must not be NULL");
    const int64_t row = static_cast<int64_t>(a->nh_q) * 128;
    DKV_REQUIRE(a->q_stride >= row && a->q_stride % 8 == 0 && aligned(a->q, 16), "q must be 16-byte aligned with a token stride that is a multiple of 8");
    DKV_REQUIRE(a->out_stride >= row && a->out_stride % 8 == 0 && aligned(a->out, 16),
                "out must be 16-byte aligned with a token stride that is a multiple of 8");
    DKV_REQUIRE(a->max_pages >= 0 && a->pt_stride >= 0 && a->pt_rows >= 0, "bad page table sizes");
    DKV_REQUIRE(a->softmax_scale == a->softmax_scale, "softmax_scale is not a number");
    DKV_ON_DEVICE(ctx);
    Kv4AttnParams p{};
    p.q = static_cast<const __nv_bfloat16*>(a->q);
    p.q_stride = a->q_stride;
    p.out = static_cast<__nv_bfloat16*>(a->out);
    p.out_stride = a->out_stride;
    p.lse = a->lse_out;
    p.seq_lens = a->seq_lens;
    p.page_table = a->page_table;
    p.pt_stride = a->pt_stride;
    p.pt_rows = a->pt_rows;
    p.page_shift = log2_of(pool->page_size);
    p.room = std::min(a->max_pages, INT32_MAX >> p.page_shift) << p.page_shift;
    p.row_map = a->row_map;
    p.k_codes = static_cast<const uint8_t*>(pool->k_codes), p.v_codes = static_cast<const uint8_t*>(pool->v_codes);
    p.k_scales = static_cast<const uint8_t*>(pool->k_scales), p.v_scales = static_cast<const uint8_t*>(pool->v_scales);
    p.n_pages = static_cast<int>(pool->n_slots / pool->page_size);
    p.batch = a->batch, p.n_q = a->n_q, p.nh_q = a->nh_q, p.nh_kv = pool->nh_kv;
    p.group = a->nh_q / pool->nh_kv;
    p.cols = a->n_q * p.group;
    p.by_group = Kv4Div(p.group), p.by_nh_q = Kv4Div(a->nh_q), p.by_n_q = Kv4Div(a->n_q);
    p.scale_log2 = a->softmax_scale * pool->k_scale * 1.4426950408889634f;
    p.v_scale = pool->v_scale;
    p.status = ctx->status;
    DKV_REQUIRE(static_cast<int64_t>(a->batch) * a->n_q * a->nh_q <= INT32_MAX, "too many query rows");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    rc = ensure_buffer(ctx, &ctx->kv4, kv4_workspace(ctx), stream_is_capturing(st), "workspace of the 4-bit attention");
    if (rc != DKV_OK) return rc;
    p.cum = reinterpret_cast<int*>(ctx->kv4.ptr);
    p.rec = reinterpret_cast<float*>(ctx->kv4.ptr + kKv4CumBytes);
    for (int b0 = 0; b0 < a->batch && rc == DKV_OK; b0 += kKv4LaunchBatch) {
        Kv4AttnParams part = p;
        part.batch = std::min(a->batch - b0, kKv4LaunchBatch);
        part.row0 = b0;
        part.seq_lens += b0;
        if (part.row_map) part.row_map += b0;
        part.q += static_cast<int64_t>(b0) * p.n_q * p.q_stride;
        part.out += static_cast<int64_t>(b0) * p.n_q * p.out_stride;
        if (part.lse) part.lse += static_cast<int64_t>(b0) * p.n_q * p.nh_q;
        rc = p.cols <= 8 ? launch_kv4_attn<1>(ctx, part, st) : launch_kv4_attn<2>(ctx, part, st);
    }
    return rc;
}

int dkv_qk_norm_rope(dkv_context* ctx, const dkv_qk_norm_args* a, void* stream) {
    DKV_REQUIRE(ctx != nullptr && a != nullptr, "ctx / args is NULL");
    DKV_REQUIRE(a->n_tokens >= 0 && a->nh_q >= 0 && a->nh_k >= 0 && a->nh_q <= 65535 && a->nh_k <= 65535, "bad sizes");
    if (a->n_tokens == 0 || a->nh_q + a->nh_k == 0) return DKV_OK;
    const int64_t rows = a->n_tokens * (a->nh_q + a->nh_k);
    DKV_REQUIRE(rows <= static_cast<int64_t>(INT32_MAX) * 2, "too many rows");
    DKV_REQUIRE(a->cos_sin == nullptr || (a->positions != nullptr && a->max_pos > 0), "a rotation needs positions and a table");
    DKV_REQUIRE(a->cos_sin == nullptr || aligned(a->cos_sin, 16), "cos_sin must be 16-byte aligned");
    DKV_REQUIRE(a->eps >= 0.f, "eps must not be negative");
    QkNormParams p{};
    const void* x[2] = {a->q, a->k};
    void* y[2] = {a->q_out, a->k_out};
    const int64_t xs[2] = {a->q_stride, a->k_stride}, ys[2] = {a->q_out_stride, a->k_out_stride};
    const int nh[2] = {a->nh_q, a->nh_k};
    const void* w[2] = {a->q_weight, a->k_weight};
    const int wf[2] = {a->q_weight_f32, a->k_weight_f32}, wp[2] = {a->q_weight_per_head, a->k_weight_per_head};
    for (int i = 0; i < 2; ++i) {
        p.heads[i] = nh[i];
        if (nh[i] == 0) continue;
        DKV_REQUIRE(x[i] != nullptr && y[i] != nullptr && aligned(x[i], 16) && aligned(y[i], 16), "q / k and their outputs must be 16-byte aligned device pointers");
        DKV_REQUIRE(xs[i] >= static_cast<int64_t>(nh[i]) * 128 && xs[i] % 8 == 0 && ys[i] >= static_cast<int64_t>(nh[i]) * 128 && ys[i] % 8 == 0,
                    "q / k token strides too small or not a multiple of 8");
        DKV_REQUIRE(w[i] == nullptr || aligned(w[i], 16), "norm weights must be 16-byte aligned");
        p.x[i] = static_cast<const __nv_bfloat16*>(x[i]);
        p.y[i] = static_cast<__nv_bfloat16*>(y[i]);
        p.x_stride[i] = xs[i], p.y_stride[i] = ys[i];
        p.weight[i] = w[i], p.weight_f32[i] = wf[i], p.weight_stride[i] = wp[i] ? 128 : 0;
    }
    p.positions = a->positions, p.pos64 = a->positions_int64;
    p.cos_sin = a->cos_sin, p.max_pos = a->max_pos;
    p.eps = a->eps;
    p.n_tokens = a->n_tokens;
    p.status = ctx->status;
    DKV_ON_DEVICE(ctx);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    // Eight heads per half warp once that still gives every SM 32 warps, else one.
    const int qn = (a->nh_q + 7) / 8, gn = qn + (a->nh_k + 7) / 8;
    if (a->n_tokens * gn >= static_cast<int64_t>(ctx->sm_count) * 64)
        DKV_CUDA(launch_overlapped(qk_norm_rope_kernel<8, 24>, static_cast<unsigned>((a->n_tokens * gn + 1) / 2), 32, 0, st, p, qn, gn));
    else
        DKV_CUDA(launch_overlapped(qk_norm_rope_kernel<1, 32>, static_cast<unsigned>((rows + 1) / 2), 32, 0, st, p, a->nh_q, a->nh_q + a->nh_k));
    ctx->launches += 1;
    return DKV_OK;
}

static int pages_common(dkv_context* ctx, const dkv_pages_args* a, PagesParams* p) {
    DKV_REQUIRE(ctx != nullptr && a != nullptr, "ctx / args is NULL");
    DKV_REQUIRE(a->batch >= 0 && a->batch <= kPagesMaxBatch, "batch (%d) must be 0..%d", a->batch, kPagesMaxBatch);
    DKV_REQUIRE(a->page_size >= 1 && (a->page_size & (a->page_size - 1)) == 0, "page_size (%d) must be a power of two", a->page_size);
    DKV_REQUIRE(a->page_table && a->free_pages && a->n_free && (a->batch == 0 || (a->lens && a->more)), "NULL argument");
    DKV_REQUIRE(a->pt_rows >= 0 && a->max_pages >= 0 && a->pt_stride >= 0 && a->free_cap >= 0, "bad sizes");
    p->page_table = a->page_table;
    p->pt_stride = a->pt_stride;
    p->pt_rows = a->pt_rows;
    p->page_shift = log2_of(a->page_size);
    p->max_pages = std::min(a->max_pages, INT32_MAX >> p->page_shift);
    p->rows = a->rows, p->lens = a->lens, p->more = a->more;
    p->batch = a->batch;
    p->free_pages = a->free_pages, p->free_cap = a->free_cap, p->n_free = a->n_free;
    p->status = ctx->status;
    p->ticket = ctx->counters + kMaxCounters;
    return DKV_OK;
}

int dkv_assign_pages(dkv_context* ctx, const dkv_pages_args* a, int32_t* slots, int32_t* positions, int64_t capacity, int32_t* seq_lens,
                     int32_t* cu_new, void* stream) {
    return dkv_assign_pages_fresh(ctx, a, slots, positions, capacity, seq_lens, cu_new, 0, stream);
}

int dkv_assign_pages_fresh(dkv_context* ctx, const dkv_pages_args* a, int32_t* slots, int32_t* positions, int64_t capacity, int32_t* seq_lens,
                           int32_t* cu_new, int fresh, void* stream) {
    PagesParams p{};
    int rc = pages_common(ctx, a, &p);
    if (rc != DKV_OK) return rc;
    DKV_REQUIRE(capacity >= 0 && capacity <= INT32_MAX && (capacity == 0 || slots != nullptr), "slots must hold 0..2^31-1 tokens");
    DKV_REQUIRE(cu_new != nullptr && (a->batch == 0 || seq_lens != nullptr), "seq_lens / cu_new must not be NULL");
    p.slots = slots, p.positions = positions, p.capacity = capacity, p.fresh = fresh, p.seq_lens = seq_lens, p.cu_new = cu_new;
    DKV_ON_DEVICE(ctx);
    p.vector = aligned(slots, 16) && aligned(positions, 16);
    const int64_t want = (capacity + 4 * kPagesThreads - 1) / (4 * kPagesThreads);
    const int grid = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(want, ctx->sm_count)));
    DKV_CUDA(launch_overlapped(pages_kernel<false>, grid, kPagesThreads, 0, static_cast<cudaStream_t>(stream), p));
    ctx->launches += 1;
    return DKV_OK;
}

int dkv_release_pages(dkv_context* ctx, const dkv_pages_args* a, void* stream) {
    PagesParams p{};
    int rc = pages_common(ctx, a, &p);
    if (rc != DKV_OK || a->batch == 0) return rc;
    DKV_ON_DEVICE(ctx);
    const int64_t most = std::min<int64_t>(static_cast<int64_t>(a->batch) * p.max_pages, p.free_cap);
    const int64_t want = (most + kPagesThreads - 1) / kPagesThreads;
    const int grid = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(want, ctx->sm_count)));
    DKV_CUDA(launch_overlapped(pages_kernel<true>, grid, kPagesThreads, 0, static_cast<cudaStream_t>(stream), p));
    ctx->launches += 1;
    return DKV_OK;
}

}  // extern "C"
