"""Page tables and slot maps built on the GPU, against Python lists; and the operators of a decode step over a 4-bit cache in a row."""

import pytest
import torch

import kv4_ref as ref

pytestmark = pytest.mark.gpu

from directkv_b200 import kernel, workloads  # noqa: E402
from directkv_b200._lib import get_context  # noqa: E402

DEV = "cuda:0"
BAD_SLOT, BAD_PAGE, OUT_OF_PAGES = 1 << 1, 1 << 5, 1 << 7


@pytest.fixture(autouse=True)
def _clean_status():
    get_context(0).read_status(clear=True)
    yield
    get_context(0).read_status(clear=True)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _setup(lens, page, spare_pages, max_pages, seed, n_rows=None):
    g = torch.Generator().manual_seed(seed)
    n_rows = n_rows or len(lens) + 2
    rows = torch.randperm(n_rows, generator=g)[:len(lens)].tolist()
    held = sum(-(-n // page) for n in lens)
    order = (torch.randperm(held + spare_pages, generator=g) + 1).to(torch.int32)
    table = torch.full((n_rows, max_pages), -7, dtype=torch.int32)
    at = spare_pages
    for r, n in zip(rows, lens):
        c = -(-n // page)
        table[r, :c] = order[at:at + c]
        at += c
    return rows, table, order, spare_pages


def _same(state, table, free, n_free):
    assert torch.equal(table.cpu(), state.table)
    assert int(n_free) == state.n
    assert free.cpu().tolist()[:state.n] == state.stack[:state.n]


@pytest.mark.parametrize("page", [1, 2, 16, 128])
@pytest.mark.parametrize("lens,new", [([0], [1]), ([5], [0]), ([0, 16, 15, 17, 1, 0], [1, 1, 1, 1, 1, 0]), ([0, 0, 0], [33, 0, 700]),
                                      ([3, 200, 31, 0, 64], [5000, 1, 0, 77, 64])])
def test_assign_and_release(page, lens, new):
    need = sum(-(-(a + n) // page) - -(-a // page) for a, n in zip(lens, new))
    max_pages = max(-(-(a + n) // page) for a, n in zip(lens, new)) + 1
    rows, table, order, spare = _setup(lens, page, need + 3, max_pages, 11)
    state = ref.Pages(table, order, spare, page)
    t, free, n_free = table.to(DEV), order.to(DEV), _i32([spare])
    room = sum(new) + 5
    slots, positions = torch.full((room,), -9, dtype=torch.int32, device=DEV), torch.full((room,), -9, dtype=torch.int32, device=DEV)
    got = kernel.assign_pages(t, _i32(lens), _i32(new), free, n_free, page, room, rows=_i32(rows), slots=slots, positions=positions)
    want = state.assign(rows, lens, new)
    total = sum(new)
    assert got[0] is slots and got[1] is positions
    assert slots.cpu().tolist() == want[0] + [-9] * 5 and positions.cpu().tolist() == want[1] + [-9] * 5
    assert got[2].cpu().tolist() == want[2] and got[3].cpu().tolist() == want[3]
    _same(state, t, free, n_free)
    assert total == want[3][-1]
    # the same tokens taken back: the stack is what it was before
    kernel.release_pages(t, got[2], _i32(lens), free, n_free, page, rows=_i32(rows))
    state.release(rows, want[2], lens)
    _same(state, t, free, n_free)
    assert int(n_free) == spare and torch.equal(free.cpu(), order)
    # all pages of every request
    room_list = torch.zeros(order.numel() + 4, dtype=torch.int32, device=DEV)
    room_list[:order.numel()] = free
    state.stack += [0] * 4
    kernel.release_pages(t, _i32(lens), _i32([0] * len(lens)), room_list, n_free, page, rows=_i32(rows))
    state.release(rows, lens, [0] * len(lens))
    _same(state, t, room_list, n_free)
    assert get_context(0).read_status() == 0


def test_many_requests_and_tokens():
    """More blocks than one and more requests than a block has threads; lengths updated in place, step after step."""
    g = torch.Generator().manual_seed(3)
    lens = torch.randint(0, 60, (1500,), generator=g).tolist()
    page = 16
    rows, table, order, spare = _setup(lens, page, 9000, 12, 12)
    state = ref.Pages(table, order, spare, page)
    t, free, n_free, lens_t = table.to(DEV), order.to(DEV), _i32([spare]), _i32(lens)
    for step in range(3):
        new = torch.randint(0, 40, (1500,), generator=g).tolist()
        got = kernel.assign_pages(t, lens_t, _i32(new), free, n_free, page, sum(new), rows=_i32(rows), seq_lens=lens_t)
        want = state.assign(rows, lens, new)
        for x, y in zip(got, want):
            assert x.cpu().tolist() == list(y)
        lens = want[2]
        _same(state, t, free, n_free)
    keep = [n // 3 for n in lens]
    kernel.release_pages(t, lens_t, _i32(keep), free, n_free, page, rows=_i32(rows))
    state.release(rows, lens, keep)
    _same(state, t, free, n_free)
    assert get_context(0).read_status() == 0


@pytest.mark.parametrize("what,status", [("pages", OUT_OF_PAGES), ("room", BAD_SLOT), ("row", BAD_PAGE), ("negative row", BAD_PAGE), ("table", BAD_PAGE),
                                         ("negative", BAD_PAGE), ("stack", BAD_PAGE)])
def test_assign_takes_effect_as_a_whole_or_not_at_all(what, status):
    lens, new, page = [5, 30, 0], [20, 3, 40], 16
    rows, table, order, spare = _setup(lens, page, 6, 4, 13)
    n_tokens = sum(new)
    if what == "pages":
        spare = 3
    if what == "room":
        n_tokens -= 1
    if what == "row":
        rows[1] = 5
    if what == "negative row":
        rows[1] = -1
    if what == "table":
        new[2] = 65
        n_tokens = sum(new)
    if what == "negative":
        new[0] = -1
        n_tokens = 43
    if what == "stack":
        spare = order.numel() + 1
    t, free, n_free = table.to(DEV), order.to(DEV), _i32([spare])
    got = kernel.assign_pages(t, _i32(lens), _i32(new), free, n_free, page, n_tokens, rows=_i32(rows))
    assert get_context(0).read_status() == status
    assert torch.equal(t.cpu(), table) and torch.equal(free.cpu(), order) and int(n_free) == spare
    assert (got[0] == -1).all() and (got[1] == 0).all() and got[2].cpu().tolist() == lens and not got[3].any()


def test_release_takes_effect_as_a_whole_or_not_at_all():
    lens, page = [50, 30, 1], 16
    for what, keep, room, status in (("stack", [0, 0, 0], 6, BAD_SLOT), ("longer", [0, 31, 0], 20, BAD_PAGE), ("negative", [-1, 0, 0], 20, BAD_PAGE)):
        rows, table, order, spare = _setup(lens, page, 2, 4, 14)
        free = torch.zeros(room, dtype=torch.int32)
        free[:2] = order[:2]
        f, n_free = free.to(DEV), _i32([2])
        kernel.release_pages(table.to(DEV), _i32(lens), _i32(keep), f, n_free, page, rows=_i32(rows))
        assert get_context(0).read_status() == status, what
        assert torch.equal(f.cpu(), free) and int(n_free) == 2


@pytest.mark.parametrize("batch", [2, 5, 513, 4096])
def test_one_row_twice(batch):
    """Two requests that change one row are refused as a whole; requests that change nothing may repeat it."""
    page, at = 16, [0, batch - 1]
    lens, rows = [page] * batch, list(range(batch))
    rows[at[1]] = rows[at[0]]
    table = torch.arange(batch, dtype=torch.int32)[:, None].repeat(1, 3).to(DEV)
    free, n_free = torch.arange(batch, 4 * batch, dtype=torch.int32, device=DEV), _i32([2 * batch])
    before = table.clone(), free.clone()
    got = kernel.assign_pages(table, _i32(lens), _i32([1] * batch), free, n_free, page, batch, rows=_i32(rows))
    assert (got[0] == -1).all() and got[2].tolist() == lens and got[3].tolist() == [0] * (batch + 1)
    kernel.release_pages(table, _i32(lens), _i32([0] * batch), free, n_free, page, rows=_i32(rows))
    assert torch.equal(table, before[0]) and torch.equal(free, before[1]) and int(n_free) == 2 * batch
    assert get_context(0).read_status(clear=True) == BAD_PAGE
    new = [1] * batch
    new[at[1]] = 0
    got = kernel.assign_pages(table, _i32(lens), _i32(new), free, n_free, page, batch, rows=_i32(rows))
    taken = torch.arange(3 * batch - 1, 2 * batch, -1)
    assert torch.equal(got[0][:batch - 1].cpu(), (taken * page).to(torch.int32)) and int(n_free) == batch + 1
    kernel.release_pages(table, got[2], _i32(lens), free, n_free, page, rows=_i32(rows))
    assert torch.equal(free, before[1]) and int(n_free) == 2 * batch
    assert get_context(0).read_status() == 0


def test_outputs_that_are_not_aligned():
    lens, new, page = [0, 30], [5, 3000], 16
    rows, table, order, spare = _setup(lens, page, 200, 200, 15)
    state = ref.Pages(table, order, spare, page)
    buf = torch.full((2, 3010), -9, dtype=torch.int32, device=DEV)
    slots, positions = buf[0, 1:3006], buf[1, 2:3007]
    kernel.assign_pages(table.to(DEV), _i32(lens), _i32(new), order.to(DEV), _i32([spare]), page, 3005, rows=_i32(rows), slots=slots, positions=positions)
    want = state.assign(rows, lens, new)
    assert slots.cpu().tolist() == want[0] and positions.cpu().tolist() == want[1]
    assert (buf[0, :1] == -9).all() and (buf[0, 3006:] == -9).all() and (buf[1, :2] == -9).all() and (buf[1, 3007:] == -9).all()


def test_no_requests():
    table, free, n_free = torch.zeros(2, 2, dtype=torch.int32, device=DEV), _i32([1, 2]), _i32([2])
    got = kernel.assign_pages(table, _i32([]), _i32([]), free, n_free, 16, 0)
    assert [x.numel() for x in got] == [0, 0, 0, 1] and int(got[3]) == 0 and int(n_free) == 2
    kernel.release_pages(table, _i32([]), _i32([]), free, n_free, 16)


def test_decode_steps_over_a_four_bit_cache():
    """What a serving loop runs, captured once and replayed: pages and slots, head norms with rotation, store, attention.
    Two graphs share the context's workspace and are replayed in turn; every step is checked against the plain forms."""
    batch, nh_q, nh_kv, page, steps = 5, 8, 2, 4, 6
    g = torch.Generator().manual_seed(21)
    cs = workloads.build_cos_sin(64, 10000.0)
    wq, wk = [(1 + 0.2 * torch.randn(128, generator=g)).to(torch.bfloat16) for _ in range(2)]
    pool = kernel.KV4Pool.empty(200, nh_kv, page, DEV)
    table, free, n_free = torch.zeros(batch, 12, dtype=torch.int32, device=DEV), torch.arange(1, 50, dtype=torch.int32, device=DEV), _i32([49])
    state = ref.Pages(table.cpu(), free.cpu(), 49, page)
    lens = torch.zeros(batch, dtype=torch.int32, device=DEV)
    w = dict(cos_sin=cs.to(DEV), q_weight=wq.to(DEV), k_weight=wk.to(DEV))
    n_q = {0: 1, 1: 3}                                   # one token per request, or three drafted ones
    graphs, bufs = {}, {}
    for i in n_q:
        n = batch * n_q[i]
        b = bufs[i] = dict(rows=torch.zeros(n, nh_q + 2 * nh_kv, 128, dtype=torch.bfloat16, device=DEV), new=_i32([n_q[i]] * batch),
                           slots=torch.zeros(n, dtype=torch.int32, device=DEV), pos=torch.zeros(n, dtype=torch.int32, device=DEV),
                           cu=torch.zeros(batch + 1, dtype=torch.int32, device=DEV), out=torch.zeros(batch, n_q[i], nh_q, 128, dtype=torch.bfloat16, device=DEV))

        def step(b=b, m=n_q[i]):
            q, k, v = b["rows"][:, :nh_q], b["rows"][:, nh_q:nh_q + nh_kv], b["rows"][:, nh_q + nh_kv:]
            kernel.assign_pages(table, lens, b["new"], free, n_free, page, batch * m, slots=b["slots"], positions=b["pos"], seq_lens=lens, cu_new=b["cu"])
            kernel.qk_norm_rope(q, k, b["pos"], w["cos_sin"], w["q_weight"], w["k_weight"], q_out=q, k_out=k)
            kernel.store_kv4(pool, b["slots"], k, v)
            kernel.decode_kv4(q.view(batch, m, nh_q, 128), pool, lens, 128 ** -0.5, table, out=b["out"])

        # one eager step on a copy of the state sizes the workspace, then the capture
        saved = [t.clone() for t in (table, free, n_free, lens)]
        step()
        torch.cuda.synchronize()
        for t, s in zip((table, free, n_free, lens), saved):
            t.copy_(s)
        graphs[i] = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graphs[i]):
            step()
    host = [0] * batch
    kv = {b: [torch.zeros(0, nh_kv, 128, dtype=torch.float64) for _ in range(2)] for b in range(batch)}
    for s in range(steps):
        i = s % 2
        m, b = n_q[i], bufs[i]
        rows = torch.randn(batch * m, nh_q + 2 * nh_kv, 128, generator=g).to(torch.bfloat16)
        b["rows"].copy_(rows)
        graphs[i].replay()
        torch.cuda.synchronize()
        slots, pos, host, cu = state.assign(range(batch), host, [m] * batch)
        assert b["slots"].cpu().tolist() == slots and b["pos"].cpu().tolist() == pos and lens.cpu().tolist() == host
        p = torch.tensor(pos)
        for x, wt, got in ((rows[:, :nh_q], wq, b["rows"][:, :nh_q]), (rows[:, nh_q:nh_q + nh_kv], wk, b["rows"][:, nh_q:nh_q + nh_kv])):
            y, e = ref.norm_rope(x, wt, p, cs, 1e-6)
            assert ((got.cpu().double() - y).abs() <= e).all()
        q, k, v = b["rows"][:, :nh_q].cpu(), b["rows"][:, nh_q:nh_q + nh_kv].cpu(), rows[:, nh_q + nh_kv:]
        for r in range(batch):
            at = slice(r * m, (r + 1) * m)
            for j, x in enumerate((k, v)):
                kv[r][j] = torch.cat([kv[r][j], ref.values(*ref.quantise(x[at]))])
            o, _, e = ref.attend(q[at], kv[r][0], kv[r][1], host[r], 128 ** -0.5)
            assert ((b["out"][r].cpu().double() - o).abs() <= e).all(), (s, r)
    assert get_context(0).read_status() == 0
    kernel.release_pages(table, lens, torch.zeros_like(lens), free, n_free, page)
    assert int(n_free) == 49 and sorted(free.cpu().tolist()) == list(range(1, 50))


@pytest.mark.parametrize("n_q", [1, 3])
def test_tables_and_queries_written_by_the_kernel_just_before(n_q):
    """assign_pages and qk_norm_rope directly before the attention: it reads the table and the queries that they have just written."""
    batch, nh_q, nh_kv, page, n = 40, 8, 2, 4, 60
    g = torch.Generator().manual_seed(31)
    pool = kernel.KV4Pool.empty(batch * 20 * page, nh_kv, page, DEV)
    parts = []
    for codes, scales in ((pool.k_codes, pool.k_scales), (pool.v_codes, pool.v_scales)):
        c, s = ref.quantise(torch.randn(*codes.shape[:2], 128, generator=g).to(torch.bfloat16))
        codes.copy_(c), scales.copy_(s)
        parts.append((c, s))
    cs = workloads.build_cos_sin(64, 10000.0).to(DEV)
    new, zero = _i32([n] * batch), _i32([0] * batch)
    pos = _i32([n - 1] * (batch * n_q))
    out = torch.zeros(batch, n_q, nh_q, 128, dtype=torch.bfloat16, device=DEV)
    for step in range(6):
        order = torch.randperm(batch * 20, generator=g).to(torch.int32)
        free, n_free, table = order.to(DEV), _i32([order.numel()]), torch.zeros(batch, 20, dtype=torch.int32, device=DEV)
        x = torch.randn(batch * n_q, nh_q, 128, generator=g).to(torch.bfloat16).to(DEV)
        q = torch.zeros_like(x)
        torch.cuda.synchronize()
        if step % 2:
            kernel.qk_norm_rope(x, None, pos, cs, q_out=q)
            _, _, lens, _ = kernel.assign_pages(table, zero, new, free, n_free, page, n * batch)
        else:
            _, _, lens, _ = kernel.assign_pages(table, zero, new, free, n_free, page, n * batch)
            kernel.qk_norm_rope(x, None, pos, cs, q_out=q)
        kernel.decode_kv4(q.view(batch, n_q, nh_q, 128), pool, lens, 128 ** -0.5, table, out=out)
        torch.cuda.synchronize()
        state = ref.Pages(torch.zeros(batch, 20, dtype=torch.int32), order, order.numel(), page)
        slots = torch.tensor(state.assign(range(batch), [0] * batch, [n] * batch)[0]).view(batch, n)
        for b in range(0, batch, 7):
            k, v = (ref.values(c[slots[b]], s[slots[b]]) for c, s in parts)
            o, _, e = ref.attend(q.view(batch, n_q, nh_q, 128)[b].cpu(), k, v, n, 128 ** -0.5)
            assert ((out[b].cpu().double() - o).abs() <= e).all(), (step, b)
    assert get_context(0).read_status() == 0


@pytest.mark.parametrize("room", [3, 64, 5000])
def test_places_behind_the_last_token_hold_no_slot(room):
    """n_tokens may be more than the tokens there are.  What the call allocates, and what an earlier call left in the caller's
    tensors, becomes no token: slot -1, position 0."""
    rows, table, order, spare = _setup([5, 0], 16, 400, 400, 16)
    t, free, n_free, lens = table.to(DEV), order.to(DEV), _i32([spare]), _i32([5, 0])
    for junk in (7, -123456):                            # what the allocator hands out again
        for n in (room, 2 * room + 5 + (-room & 3)):
            torch.full((n,), junk, dtype=torch.int32, device=DEV)
        got = kernel.assign_pages(t, lens, _i32([2, 1]), free, n_free, 16, room, rows=_i32(rows))
        assert (got[0][:3] >= 0).all() and got[1][:3].tolist() == [5, 6, 0] and (got[0][3:] == -1).all() and (got[1][3:] == 0).all()
        kernel.release_pages(t, got[2], lens, free, n_free, 16, rows=_i32(rows))
    slots, positions = _i32([9] * room), _i32([4] * room)
    kernel.assign_pages(t, lens, _i32([1, 0]), free, n_free, 16, room, rows=_i32(rows), slots=slots)
    got = kernel.assign_pages(t, _i32([6, 0]), _i32([0, 1]), free, n_free, 16, room, rows=_i32(rows), slots=slots, positions=positions)
    assert got[0] is slots and slots[0] >= 0 and (slots[1:] == -1).all() and (positions == 0).all()
    assert get_context(0).read_status() == 0


def test_a_replay_with_fewer_tokens_than_the_graph_has_room_for_changes_no_other_row():
    """A captured step of up to 8 tokens: bookkeeping, rotation, store, load.  Replayed with fewer it stores those alone."""
    nh, page, room = 2, 4, 8
    g = torch.Generator().manual_seed(33)
    cs = workloads.build_cos_sin(64, 10000.0).to(DEV)
    pool = kernel.KV4Pool.empty(80, nh, page, DEV)
    table, free, n_free = torch.zeros(3, 6, dtype=torch.int32, device=DEV), torch.arange(1, 19, dtype=torch.int32, device=DEV), _i32([18])
    state = ref.Pages(table.cpu(), free.cpu(), 18, page)
    lens, new, cu = _i32([0] * 3), _i32([0] * 3), _i32([0] * 4)
    slots, pos = _i32([-1] * room), _i32([0] * room)
    k, v = (torch.zeros(room, nh, 128, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    back = [torch.zeros_like(k) for _ in range(2)]

    def step():
        kernel.assign_pages(table, lens, new, free, n_free, page, room, slots=slots, positions=pos, seq_lens=lens, cu_new=cu)
        kernel.qk_norm_rope(None, k, pos, cs, k_out=k)
        kernel.store_kv4(pool, slots, k, v)
        kernel.load_kv4(pool, slots, *back)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    want = torch.zeros(80, nh, 128, dtype=torch.float64)
    host = [0] * 3
    for more in ([4, 3, 1], [1, 0, 1], [0, 0, 0], [0, 5, 0], [1, 1, 1]):
        rows = [torch.randn(room, nh, 128, generator=g).to(torch.bfloat16) for _ in range(2)]
        k.copy_(rows[0]), v.copy_(rows[1]), new.copy_(torch.tensor(more, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        at, where, host, _ = state.assign(range(3), host, more)
        n = sum(more)
        assert slots.tolist() == at + [-1] * (room - n) and pos.tolist() == where + [0] * (room - n)
        want[at] = ref.values(*ref.quantise(v.cpu()[:n]))
        got = kernel.load_kv4(pool, torch.arange(80, dtype=torch.int32, device=DEV))[1]
        assert torch.equal(got.cpu().double(), want)
        assert torch.equal(back[1].cpu().double()[:n], want[at]) and not back[1][n:].any()
    assert get_context(0).read_status() == 0


@pytest.mark.parametrize("number", [-1, -7, 2 ** 28])
@pytest.mark.parametrize("where", ["table", "stack"])
def test_page_numbers_that_give_no_slot_are_reported(where, number):
    """A slot of -1 means no token, which the store passes over in silence: a wrong page number must not look like that."""
    rows, table, order, spare = _setup([20, 3], 16, 4, 4, 17)
    if where == "table":
        table[rows[0], 1] = number
    else:
        order[spare - 1] = number
    got = kernel.assign_pages(table.to(DEV), _i32([20, 3]), _i32([2, 2]) if where == "table" else _i32([13, 0]), order.to(DEV), _i32([spare]), 16,
                              4 if where == "table" else 13, rows=_i32(rows))
    assert get_context(0).read_status() == BAD_PAGE
    assert got[0].tolist()[:2] == [-1, -1] if where == "table" else got[0].tolist()[12] == -1 and min(got[0].tolist()[:12]) >= 0
