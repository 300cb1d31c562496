"""4-bit pool on the GPU: the stored bytes, reading them back, and decode attention over them, against plain 64-bit forms."""

import math

import pytest
import torch

import kv4_ref as ref

pytestmark = pytest.mark.gpu

from directkv_b200 import kernel  # noqa: E402
from directkv_b200._lib import get_context  # noqa: E402

DEV = "cuda:0"
BAD_SLOT, BAD_PAGE, NONFINITE = 1 << 1, 1 << 5, 1 << 6


@pytest.fixture(autouse=True)
def _clean_status():
    get_context(0).read_status(clear=True)
    yield
    get_context(0).read_status(clear=True)


def _rows(n, nh, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(n, nh, 128, generator=g) * torch.exp(torch.randn(nh, 128, generator=g) * spread)).to(torch.bfloat16)


# ------------------------------------------------------------------------------------------------ store and load
@pytest.mark.parametrize("host", [False, True])
@pytest.mark.parametrize("n,nh,i64,ke,ve", [(1, 1, False, 0, 0), (5, 3, True, 3, -4), (257, 8, False, -2, 1), (64, 33, True, 0, 24)])
def test_store_writes_the_format_and_load_reads_it(n, nh, i64, ke, ve, host):
    pool = kernel.KV4Pool.empty(2 * n + 3, nh, device="cpu" if host else DEV, k_scale=2.0 ** ke, v_scale=2.0 ** ve)
    g = torch.Generator().manual_seed(n)
    slots = torch.randperm(2 * n + 3, generator=g)[:n].to(torch.int64 if i64 else torch.int32)
    k, v = _rows(n, nh, 1) * 2.0 ** ke, _rows(n, nh, 2, 2.0)
    k[0, 0, :16] = 0.0                                   # a block of zeros
    k[0, 0, 16:32] = 1e-30                               # a block below the smallest scale
    v[0, 0, :16] = 1e30                                  # a block above the largest
    kernel.store_kv4(pool, slots.to(DEV), k.to(DEV), v.to(DEV))
    got = kernel.load_kv4(pool, slots.to(DEV))
    torch.cuda.synchronize()
    for x, codes, scales, back, s in ((k, pool.k_codes, pool.k_scales, got[0], 2.0 ** ke), (v, pool.v_codes, pool.v_scales, got[1], 2.0 ** ve)):
        want_c, want_s = ref.quantise(x, s)
        c, sc = codes.cpu(), scales.cpu()
        assert torch.equal(sc[slots.long()], want_s)
        assert torch.equal(c[slots.long()], want_c)
        assert torch.equal(back.cpu().double(), ref.values(want_c, want_s, s))
        untouched = torch.ones(2 * n + 3, dtype=torch.bool)
        untouched[slots.long()] = False
        assert not c[untouched].any() and not sc[untouched].any()
    assert get_context(0).read_status() == 0


def test_store_rounds_ties_to_even_for_every_scale():
    """All borders between neighbouring codes, times every e4m3 scale that a block maximum of 6 * s gives."""
    scales = ref.E4M3[1:]
    borders = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5.0, -0.0], dtype=torch.float64)
    x = (scales[:, None] * borders).to(torch.bfloat16)
    assert torch.equal(x.double(), scales[:, None] * borders), "every border must be a bf16 value"
    rows = torch.zeros(16, 1, 128, dtype=torch.bfloat16)
    rows.view(-1, 16)[:126] = x
    pool = kernel.KV4Pool.empty(16, 1, device=DEV)
    kernel.store_kv4(pool, torch.arange(16, dtype=torch.int32, device=DEV), rows.to(DEV), rows.to(DEV))
    c, s = ref.quantise(rows)
    assert torch.equal(pool.k_scales.cpu(), s) and torch.equal(pool.v_codes.cpu(), c)


def test_store_takes_strided_rows_and_reports_bad_slots_and_odd_values():
    n, nh = 9, 2
    fused = _rows(n, 3 * nh, 3).to(DEV)
    k, v = fused[:, nh:2 * nh], fused[:, 2 * nh:]
    pool = kernel.KV4Pool.empty(20, nh, device=DEV)
    slots = torch.tensor([3, 20, 1, -1, 5, 2 ** 31 - 1, 7, 8, 0], dtype=torch.int32, device=DEV)
    kernel.store_kv4(pool, slots, k, v)
    assert get_context(0).read_status() == BAD_SLOT
    back = kernel.load_kv4(pool, slots)
    assert get_context(0).read_status() == BAD_SLOT
    for x, y in zip((k, v), back):
        want = ref.values(*ref.quantise(x.cpu()))
        want[[1, 3, 5]] = 0.0
        assert torch.equal(y.cpu().double(), want)
    odd = _rows(2, nh, 4)
    odd[0, 0, 3], odd[0, 1, 17], odd[1, 1, 127] = math.nan, math.inf, -math.inf
    s2 = torch.tensor([10, 11], dtype=torch.int64, device=DEV)
    kernel.store_kv4(pool, s2, odd.to(DEV), odd.to(DEV))
    assert get_context(0).read_status() == NONFINITE
    assert torch.equal(kernel.load_kv4(pool, s2)[0].cpu().double(), ref.values(*ref.quantise(odd)))


def test_empty_calls_do_nothing():
    pool = kernel.KV4Pool.empty(4, 2, device=DEV)
    none = torch.empty(0, dtype=torch.int32, device=DEV)
    z = torch.empty(0, 2, 128, dtype=torch.bfloat16, device=DEV)
    kernel.store_kv4(pool, none, z, z)
    assert kernel.load_kv4(pool, none)[0].shape == (0, 2, 128)
    out = kernel.decode_kv4(torch.empty(0, 4, 128, dtype=torch.bfloat16, device=DEV), pool, none, 1.0, torch.zeros(0, 1, dtype=torch.int32, device=DEV))
    assert out.shape == (0, 4, 128)
    assert get_context(0).read_status() == 0


# ------------------------------------------------------------------------------------------------ attention
@pytest.fixture(params=[0, 3000], ids=["narrow", "wide"])
def columns(request):
    """Page tables with room for the lengths alone, where nothing is split, and with room for many more tokens, where segments
    are cut and merged."""
    return request.param


def _widen(c, columns):
    c["table"] = torch.cat([c["table"], torch.zeros(c["table"].shape[0], columns, dtype=torch.int32)], 1)
    return c


def _case(lens, nh_q, nh_kv, page, n_q, seed, host=False, k_scale=1.0, v_scale=1.0, spread=0.7, q_std=1.0):
    g = torch.Generator().manual_seed(seed)
    counts = [-(-n // page) for n in lens]
    total = sum(counts)
    perm = torch.randperm(total, generator=g) + 1
    table = torch.zeros(len(lens), max(max(counts), 1) + 2, dtype=torch.int32)
    at = 0
    for b, c in enumerate(counts):
        table[b, :c] = perm[at:at + c]
        at += c
    n_slots = (total + 1) * page
    pool = kernel.KV4Pool.empty(n_slots, nh_kv, page, "cpu" if host else DEV, k_scale, v_scale)
    parts = []
    for i, (codes, scales) in enumerate(((pool.k_codes, pool.k_scales), (pool.v_codes, pool.v_scales))):
        c, s = ref.quantise(_rows(n_slots, nh_kv, seed + 10 + i, spread))
        codes.copy_(c), scales.copy_(s)
        parts.append((c, s))
    q = (torch.randn(len(lens), n_q, nh_q, 128, generator=g) * q_std).to(torch.bfloat16)
    return dict(pool=pool, parts=parts, table=table, q=q, lens=lens, page=page, n_q=n_q, nh_q=nh_q, nh_kv=nh_kv, scale=128 ** -0.5)


def _want(c, lens=None, rows=None):
    outs, lses, bounds = [], [], []
    for b, n in enumerate(lens if lens is not None else c["lens"]):
        row = b if rows is None else rows[b]
        at = ref.slots_of(c["table"][row].tolist(), n, c["page"])
        k = ref.values(c["parts"][0][0][at], c["parts"][0][1][at], c["pool"].k_scale)
        v = ref.values(c["parts"][1][0][at], c["parts"][1][1][at], c["pool"].v_scale)
        o, l, e = ref.attend(c["q"][b], k, v, n, c["scale"])
        outs.append(o), lses.append(l), bounds.append(e)
    return torch.stack(outs), torch.stack(lses), torch.stack(bounds)


def _check(c, out, lse=None, want=None):
    o, l, e = want if want is not None else _want(c)
    got = out.detach().cpu().double().reshape(o.shape)
    assert torch.isfinite(got).all()
    bad = (got - o).abs() > e
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} outside the bound, worst {((got - o).abs() / e).max():.2f} times it"
    if lse is not None:
        got_l = lse.cpu().double().reshape(l.shape)
        assert torch.equal(torch.isinf(got_l), torch.isinf(l))
        fin = torch.isfinite(l)
        # scores in fp32 (see attend's bound; 2^-14 covers sums of magnitudes up to 8), the sum and the logarithm in fp32
        assert ((got_l - l).abs()[fin] <= 2.0 ** -14 * (1 + l.abs()[fin])).all()


def _run(c, **kw):
    n = len(c["lens"])
    lse = torch.full((n, c["n_q"], c["nh_q"]), 7.0, device=DEV)
    out = kernel.decode_kv4(c["q"].to(DEV), c["pool"], torch.tensor(c["lens"], dtype=torch.int32, device=DEV), c["scale"], c["table"].to(DEV), lse_out=lse, **kw)
    torch.cuda.synchronize()
    return out, lse


RAGGED = [1, 0, 2, 15, 16, 17, 31, 33, 64, 65, 127, 128, 129, 300, 513]


@pytest.mark.parametrize("nh_q,nh_kv", [(4, 4), (8, 2), (8, 1), (6, 3), (7, 7), (12, 1), (16, 1), (40, 2), (34, 2), (9, 9), (20, 10), (32, 8), (33, 11), (17, 17)])
def test_head_groupings(nh_q, nh_kv, columns):
    c = _widen(_case(RAGGED, nh_q, nh_kv, 16, 1, 100 + nh_q), columns)
    _check(c, *_run(c))
    assert get_context(0).read_status() == 0


@pytest.mark.parametrize("page", [1, 2, 4, 8, 32, 64, 256])
@pytest.mark.parametrize("host", [False, True])
def test_page_sizes_and_pool_places(page, host, columns):
    c = _widen(_case([1, 5, 40, 0, 257, 300], 8, 2, page, 1, 200 + page, host=host), columns)
    _check(c, *_run(c))


@pytest.mark.parametrize("n_q", [2, 3, 4, 5, 8, 17, 64])
@pytest.mark.parametrize("nh_q,nh_kv", [(4, 4), (8, 2), (12, 1)])
def test_several_query_tokens(n_q, nh_q, nh_kv, columns):
    """Every query token attends its own prefix; lengths shorter than n_q leave the first rows without any token."""
    c = _widen(_case([n_q, 0, 1, n_q - 1, n_q + 1, 16 + n_q, 47, 100, 130], nh_q, nh_kv, 16, n_q, 300 + n_q), columns)
    _check(c, *_run(c))


def test_pool_scales_and_softmax_scale():
    for ke, ve, s in ((3, -4, 0.3), (-6, 5, 128 ** -0.5), (0, 0, 0.0), (0, 0, -0.1)):
        c = _case([70, 3, 200], 8, 4, 16, 1, 400 + ke, k_scale=2.0 ** ke, v_scale=2.0 ** ve)
        c["scale"] = s
        _check(c, *_run(c))


@pytest.mark.parametrize("q_std", [1e-30, 1e-3, 30.0])
def test_small_and_large_queries(q_std, columns):
    """Large scores make the softmax a choice of one token; the running maximum moves on the way there."""
    c = _widen(_case([1, 40, 333, 1025], 8, 2, 16, 1, 500, q_std=q_std), columns)
    _check(c, *_run(c))


def test_rising_scores_move_the_maximum_at_every_tile(columns):
    n = 700
    c = _widen(_case([n, n], 4, 2, 16, 1, 510), columns)
    k = torch.zeros((n // 16 + 1) * 16 * 2 + 16, 2, 128, dtype=torch.bfloat16)
    direction = torch.sign(torch.randn(128, generator=torch.Generator().manual_seed(1)))
    for b in range(2):
        at = ref.slots_of(c["table"][b].tolist(), n, 16)
        t = torch.arange(n).float() / n * 6
        k[at] = ((t if b == 0 else t.flip(0))[:, None, None] * direction).to(torch.bfloat16).expand(n, 2, 128)
    kc, ks = ref.quantise(k[: c["pool"].n_slots])
    c["pool"].k_codes.copy_(kc), c["pool"].k_scales.copy_(ks)
    c["parts"][0] = (kc, ks)
    c["q"] = (direction * 3).to(torch.bfloat16).expand(2, 1, 4, 128).clone()
    _check(c, *_run(c))


@pytest.mark.parametrize("nh_q,nh_kv,page,n_q", [(8, 2, 64, 1), (8, 8, 16, 1), (32, 8, 16, 2), (16, 4, 1, 3), (5, 5, 32, 1)])
def test_one_long_request(nh_q, nh_kv, page, n_q):
    c = _case([9001], nh_q, nh_kv, page, n_q, 520)
    _check(c, *_run(c))


def test_many_short_requests(columns):
    """More requests than blocks, and more than one launch takes."""
    _check2 = lambda c: _check(c, *_run(c))  # noqa: E731
    _check2(_widen(_case([1 + i % 37 for i in range(300)], 4, 2, 4, 1, 521), columns))
    _check2(_widen(_case([i % 23 for i in range(2000)], 2, 2, 16, 1, 522), columns))
    _check2(_widen(_case([40 + i % 90 for i in range(70)], 8, 8, 16, 1, 523), columns))


@pytest.mark.parametrize("batch,longest,nh_q,nh_kv", [(64, 480, 8, 8), (8, 992, 16, 8), (20, 1000, 8, 8)])
def test_several_steps_and_token_lanes_of_whole_segments(batch, longest, nh_q, nh_kv, columns):
    c = _widen(_case([longest] + [(i * 131) % (longest + 1) for i in range(batch - 1)], nh_q, nh_kv, 16, 1, 524), columns)
    _check(c, *_run(c))


@pytest.mark.parametrize("batch", [31, 32, 33, 257])
def test_batches_that_a_warp_or_a_block_scans(batch, columns):
    c = _widen(_case([(i * 77) % 400 for i in range(batch)], 4, 4, 16, 1, 525 + batch), columns)
    _check(c, *_run(c))
    assert get_context(0).read_status() == 0


def test_row_map_strides_and_2d_queries():
    c = _case([50, 0, 300, 17], 8, 2, 16, 1, 530)
    rows = [2, 0, 3]
    lens = [c["lens"][r] for r in rows]
    wide = torch.full((3, 24, 128), 9.0, dtype=torch.bfloat16, device=DEV)
    wide[:, 8:16] = c["q"][:3, 0].to(DEV)
    room = torch.full((3, 12, 128), 5.0, dtype=torch.bfloat16, device=DEV)
    kw = dict(row_map=torch.tensor(rows, dtype=torch.int32, device=DEV))
    lens_t = torch.tensor(lens, dtype=torch.int32, device=DEV)
    want = _want(c, lens, rows)
    big = torch.zeros(4, c["table"].shape[1] + 5, dtype=torch.int32, device=DEV)
    big[:, :c["table"].shape[1]] = c["table"].to(DEV)
    out = kernel.decode_kv4(wide[:, 8:16], c["pool"], lens_t, c["scale"], big[:, :c["table"].shape[1]], out=room[:, 2:10], **kw)
    _check(c, out, want=want)
    assert (room[:, :2] == 5).all() and (room[:, 10:] == 5).all()
    flat = kernel.decode_kv4(c["q"][:3].reshape(3, -1).to(DEV), c["pool"], lens_t, c["scale"], c["table"].to(DEV), **kw)
    assert flat.shape == (3, 8 * 128)
    _check(c, flat, want=want)


def test_tokens_behind_the_length_do_not_matter(columns):
    """Slots behind a request's length hold not-a-number scales; they are never part of a result."""
    c = _widen(_case([19, 40], 4, 2, 16, 2, 540), columns)
    for b, n in enumerate(c["lens"]):
        for t in range(n, -(-n // 16) * 16):
            slot = ref.slots_of(c["table"][b].tolist(), t + 1, 16)[t]
            c["pool"].k_scales[slot] = 0x7f
            c["pool"].v_scales[slot] = 0x7f
    _check(c, *_run(c))


def test_bad_pages_rows_and_lengths_are_reported_and_bounded():
    c = _case([40, 40, 40, 40], 4, 2, 16, 1, 550)
    good = _run(c)[0]
    assert get_context(0).read_status() == 0
    keep = c["table"].clone()
    for number in (-1, 10 ** 6, 2 ** 31 - 1):                    # a page outside the pool counts as zeros
        c["table"] = keep.clone()
        c["table"][1, 1] = number
        out = _run(c)[0]
        assert get_context(0).read_status() == BAD_PAGE
        assert torch.equal(out[[0, 2, 3]], good[[0, 2, 3]]) and torch.isfinite(out).all()
    c["table"] = keep
    lens = torch.tensor([40, -3, 10 ** 9, 40], dtype=torch.int32, device=DEV)
    out = kernel.decode_kv4(c["q"].to(DEV), c["pool"], lens, c["scale"], keep[:, :3].contiguous().to(DEV))
    assert get_context(0).read_status() == BAD_PAGE
    assert torch.equal(out[[0, 3]], good[[0, 3]]) and not out[1].any()
    rows = torch.tensor([0, 7, -1, 3], dtype=torch.int32, device=DEV)
    out = kernel.decode_kv4(c["q"].to(DEV), c["pool"], torch.full((4,), 40, dtype=torch.int32, device=DEV), c["scale"], keep.to(DEV), row_map=rows)
    assert get_context(0).read_status() == BAD_PAGE
    assert torch.equal(out[[0, 3]], good[[0, 3]]) and not out[1:3].any()


def test_not_a_number_in_a_query_stays_in_its_row(columns):
    c = _widen(_case([64, 64], 8, 2, 16, 2, 560), columns)
    want = _want(c)
    c["q"][0, 1, 3, 5] = math.nan
    out, lse = _run(c)
    got = out.cpu().double()
    assert torch.isnan(got[0, 1, 3]).all() and torch.isnan(lse[0, 1, 3])
    mask = torch.ones(2, 2, 8, dtype=torch.bool)
    mask[0, 1, 3] = False
    assert ((got - want[0]).abs() <= want[2])[mask].all()


@pytest.mark.parametrize("n_q", [1, 3])
def test_the_same_inputs_give_the_same_bits_on_another_stream_and_in_a_graph(n_q):
    c = _case([1, 77, 900, 0, 2500, 33], 16, 4, 16, n_q, 570)
    first, lse = _run(c)
    q, table = c["q"].to(DEV), c["table"].to(DEV)
    lens = torch.tensor(c["lens"], dtype=torch.int32, device=DEV)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        again = kernel.decode_kv4(q, c["pool"], lens, c["scale"], table)
    s.synchronize()
    assert torch.equal(again, first)
    out = torch.zeros_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kernel.decode_kv4(q, c["pool"], lens, c["scale"], table, out=out)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, first)
    shorter = [1, 50, 30, 0, 2000, 1]                             # new lengths, same graph
    lens.copy_(torch.tensor(shorter, dtype=torch.int32))
    graph.replay()
    torch.cuda.synchronize()
    _check(c, out, want=_want(c, shorter))
    assert get_context(0).read_status() == 0


def test_after_copies_fills_and_joined_streams_eager_and_captured():
    """What comes before a call in its stream need not be a kernel: every call sees what was enqueued before it."""
    c = _case([200, 77], 8, 2, 16, 1, 580)
    want = _run(c)[0]
    table, lens = c["table"].to(DEV), torch.tensor(c["lens"], dtype=torch.int32, device=DEV)
    q_new, q = c["q"].to(DEV), torch.zeros(2, 1, 8, 128, dtype=torch.bfloat16, device=DEV)
    rows = _rows(4, 2, 9).to(DEV)
    k_in, slots = torch.zeros_like(rows), torch.arange(4, dtype=torch.int32, device=DEV)      # the padding page: nobody attends it
    out = torch.zeros_like(q)
    got = [torch.zeros_like(rows) for _ in range(2)]
    side = torch.cuda.Stream()

    def step():
        q.copy_(q_new)                                   # a device-to-device copy just before the attention
        kernel.decode_kv4(q, c["pool"], lens, c["scale"], table, out=out)
        q.zero_()                                        # must not overtake it
        here = torch.cuda.current_stream()
        side.wait_stream(here)
        with torch.cuda.stream(side):
            k_in.copy_(rows)
        here.wait_stream(side)
        kernel.store_kv4(c["pool"], slots, k_in, k_in)   # after the join
        k_in.zero_()
        kernel.load_kv4(c["pool"], slots, *got)
        kernel.decode_kv4(q_new, c["pool"], lens, c["scale"], table)

    step()
    torch.cuda.synchronize()
    values = ref.values(*ref.quantise(rows.cpu()))
    assert torch.equal(out, want) and torch.equal(got[0].cpu().double(), values)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(20):
        for t in (out, *got, c["pool"].k_codes[:4], c["pool"].v_scales[:4]):
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(got[0].cpu().double(), values) and torch.equal(got[1].cpu().double(), values)


def test_rows_behind_four_gigabytes():
    n, nh = 8_500_000, 8                                  # 4.35 GB of codes
    codes, scales = torch.empty(n, nh, 64, dtype=torch.uint8, device=DEV), torch.empty(n, nh, 8, dtype=torch.uint8, device=DEV)
    for page in (16, 1):
        pool = kernel.KV4Pool(codes, scales, codes, scales, page_size=page)      # K and V are the same rows
        length = 40
        first = (n // 16 - 3) * 16
        slots = torch.arange(first, first + length, device=DEV)
        k = _rows(length, nh, 31).to(DEV)
        kernel.store_kv4(pool, slots, k, k)
        back = kernel.load_kv4(pool, slots)
        want = ref.values(*ref.quantise(k.cpu()))
        assert torch.equal(back[0].cpu().double(), want) and torch.equal(back[1].cpu().double(), want)
        table = (torch.arange(-(-length // page), dtype=torch.int32, device=DEV) + first // page)[None]
        q = torch.randn(1, 16, 128, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
        out = kernel.decode_kv4(q.to(DEV), pool, torch.tensor([length], dtype=torch.int32, device=DEV), 128 ** -0.5, table)
        o, _, e = ref.attend(q, want, want, length, 128 ** -0.5)
        assert ((out.cpu().double() - o).abs() <= e).all()
    assert get_context(0).read_status() == 0


def test_rows_that_are_aligned_to_16_bytes_only():
    n, nh = 37, 3
    flat = _rows(n, nh, 33).reshape(-1)
    buf = torch.zeros(flat.numel() + 8, dtype=torch.bfloat16, device=DEV)
    buf[8:] = flat.to(DEV)
    k = buf[8:].view(n, nh, 128)
    pool = kernel.KV4Pool.empty(n, nh, device=DEV)
    slots = torch.arange(n, dtype=torch.int32, device=DEV)
    kernel.store_kv4(pool, slots, k, k)
    outs = [torch.zeros(flat.numel() + 8, dtype=torch.bfloat16, device=DEV)[8:].view(n, nh, 128) for _ in range(2)]
    kernel.load_kv4(pool, slots, *outs)
    want = ref.values(*ref.quantise(flat.view(n, nh, 128)))
    assert torch.equal(outs[0].cpu().double(), want) and torch.equal(outs[1].cpu().double(), want)
    odd = torch.zeros(flat.numel() + 4, dtype=torch.bfloat16, device=DEV)[4:].view(n, nh, 128)
    with pytest.raises(RuntimeError, match="aligned"):
        kernel.store_kv4(pool, slots, odd, k)
    with pytest.raises(RuntimeError, match="aligned"):
        kernel.load_kv4(pool, slots, odd, outs[0])
