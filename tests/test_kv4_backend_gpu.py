"""The attention backend over a token pool held in 4 bits: prefill (short, long, chunked) and decode steps, eager and as a
CUDA graph, against plain 64-bit attention over the values that the pool stands for."""

import pytest
import torch

import kv4_ref as ref
from fake_sglang import DECODE, EXTEND, FakeModel, make_batch, make_runner

pytestmark = pytest.mark.gpu

import directkv_b200  # noqa: E402
from directkv_b200._lib import get_context  # noqa: E402

DEV = "cuda:0"
H, NH_Q, NH_KV, D, LAYERS = 256, 8, 2, 128, 2


def _setup(location, ctx_len=1024):
    torch.manual_seed(0)
    model = FakeModel(LAYERS, H, NH_Q, NH_KV, None, ctx_len).to(DEV)
    runner = make_runner(model, H, NH_Q, NH_KV, LAYERS, DEV, max_reqs=8, context_len=ctx_len)
    be = directkv_b200.DirectKVSmpV2Backend(runner)
    pool = directkv_b200.DirectKV4BitTokenToKVPool(size=3000, page_size=1, dtype=torch.bfloat16, head_num=NH_KV, head_dim=D, layer_num=LAYERS,
                                                   start_layer=0, end_layer=LAYERS - 1, location=location)
    perm = (torch.randperm(3000, generator=torch.Generator().manual_seed(3)) + 1).int()
    for rid in range(8):
        runner.req_to_token_pool.req_to_token[rid, :300] = perm[rid * 300:(rid + 1) * 300].to(DEV)
    get_context(0).read_status(clear=True)
    return be, runner.req_to_token_pool, model.layers[1], pool


def _rows(g, n, nh, std=1.0):
    return (torch.randn(n, nh * D, generator=g) * std).to(torch.bfloat16)


class Mirror:
    """What the pool stands for, per request, in 64 bits."""

    def __init__(self):
        self.kv = {}

    def add(self, rid, k, v):
        old = self.kv.get(rid, (torch.zeros(0, NH_KV, D, dtype=torch.float64),) * 2)
        self.kv[rid] = tuple(torch.cat([o, ref.values(*ref.quantise(x.view(-1, NH_KV, D)))]) for o, x in zip(old, (k, v)))

    def check(self, rid, q, out, extend):
        k, v = self.kv[rid]
        o, _, bound = ref.attend(q.view(-1, NH_Q, D), k, v, k.shape[0], D ** -0.5)
        if extend:
            # The extend kernel rounds its probabilities to bf16 (2^-8 of each, once in the numerator): up to 2^-8 of sum p |v|,
            # which is at most the largest |v|; its sums run over the rounded ones or not, 2^-8 again.
            bound = bound + 2 * 2.0 ** -8 * v.abs().amax(0).repeat_interleave(NH_Q // NH_KV, 0)
        got = out.cpu().double().view(o.shape)
        assert ((got - o).abs() <= bound).all(), (rid, ((got - o).abs() / bound).max())


@pytest.mark.parametrize("location", ["host", "device"])
def test_prefill_and_decode_over_a_four_bit_token_pool(location):
    be, r2t, layer, pool = _setup(location)
    g = torch.Generator().manual_seed(11)
    ref_kv = Mirror()

    def extend(plan):
        n = sum(e for _, e, _ in plan)
        loc = torch.cat([r2t.req_to_token[rid, p:p + e] for rid, e, p in plan])
        fb = make_batch(EXTEND, [p + e for _, e, p in plan], [rid for rid, _, _ in plan], DEV, extend_lens=[e for _, e, _ in plan],
                        prefix_lens=[p for _, _, p in plan], token_pool=pool, req_to_token_pool=r2t, out_cache_loc=loc)
        be.init_forward_metadata(fb)
        q, k, v = _rows(g, n, NH_Q), _rows(g, n, NH_KV), _rows(g, n, NH_KV)
        out = be.forward_extend(q.to(DEV), k.to(DEV), v.to(DEV), layer.attn, fb)
        at = 0
        for rid, e, p in plan:
            ref_kv.add(rid, k[at:at + e], v[at:at + e])
            ref_kv.check(rid, q[at:at + e], out[at:at + e], extend=e * (NH_Q // NH_KV) >= 128)
            at += e

    extend([(2, 150, 0), (4, 7, 0), (5, 40, 0)])          # long, short, long
    extend([(2, 3, 150)])                                  # a short chunk on a long prefix
    extend([(4, 64, 7), (5, 1, 40)])
    have = {2: 153, 4: 71, 5: 41}

    def decode(rids, step, graph=None):
        loc = torch.stack([r2t.req_to_token[r, have[r]] for r in rids])
        q, k, v = _rows(g, len(rids), NH_Q), _rows(g, len(rids), NH_KV), _rows(g, len(rids), NH_KV)
        for r in rids:
            have[r] += 1
        out = step(rids, loc, q, k, v)
        for i, r in enumerate(rids):
            ref_kv.add(r, k[i:i + 1], v[i:i + 1])
            ref_kv.check(r, q[i:i + 1], out[i:i + 1], extend=False)

    def eager(rids, loc, q, k, v):
        fb = make_batch(DECODE, [have[r] for r in rids], rids, DEV, token_pool=pool, req_to_token_pool=r2t, out_cache_loc=loc)
        be.init_forward_metadata(fb)
        return be.forward_decode(q.to(DEV), k.to(DEV), v.to(DEV), layer.attn, fb)

    for _ in range(3):
        decode([2, 4, 5], eager)

    # the same step under a CUDA graph, with the hooks that refresh its lengths
    bs = 3
    be.init_cuda_graph_state(bs, bs)
    bufs = dict(q=torch.zeros(bs, NH_Q * D, dtype=torch.bfloat16, device=DEV), k=torch.zeros(bs, NH_KV * D, dtype=torch.bfloat16, device=DEV),
                v=torch.zeros(bs, NH_KV * D, dtype=torch.bfloat16, device=DEV), loc=torch.zeros(bs, dtype=torch.int32, device=DEV),
                rid=torch.tensor([2, 4, 5], dtype=torch.int64, device=DEV), lens=torch.ones(bs, dtype=torch.int64, device=DEV))
    be.init_forward_metadata_capture_cuda_graph(bs, bs, bufs["rid"], bufs["lens"], None, DECODE, None)
    fb = make_batch(DECODE, [1] * bs, [2, 4, 5], DEV, token_pool=pool, req_to_token_pool=r2t, out_cache_loc=bufs["loc"])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out_g = be.forward_decode(bufs["q"], bufs["k"], bufs["v"], layer.attn, fb)

    def replay(rids, loc, q, k, v):
        bufs["q"].copy_(q), bufs["k"].copy_(k), bufs["v"].copy_(v), bufs["loc"].copy_(loc)
        lens = torch.tensor([have[r] for r in rids])
        bufs["lens"].copy_(lens)
        be.init_forward_metadata_replay_cuda_graph(bs, bufs["rid"], bufs["lens"], int(lens.sum()), None, DECODE, None, seq_lens_cpu=lens)
        graph.replay()
        torch.cuda.synchronize()
        return out_g

    for _ in range(3):
        decode([2, 4, 5], replay)
    assert get_context(0).read_status() == 0
    graph.reset()


def test_pool_moves_keep_the_bytes():
    make = lambda where: directkv_b200.DirectKV4BitTokenToKVPool(size=63, page_size=1, dtype=torch.bfloat16, head_num=2, head_dim=128, layer_num=2,  # noqa: E731
                                                                 location=where)
    host, dev = make("host"), make("device")
    g = torch.Generator().manual_seed(5)
    k, v = _rows(g, 10, 2).view(10, 2, 128).to(DEV), _rows(g, 10, 2).view(10, 2, 128).to(DEV)
    loc = torch.arange(20, 30, device=DEV)
    for lid in (0, 1):
        dev.set_kv_buffer(None, loc, k, v, layer_id_override=lid)
    want = dev.load_rows(1, loc)
    dev.backup_to_host_all_layer(host, list(range(10)), loc, None)
    dev.move_kv_cache(torch.arange(40, 50), loc)
    dev.load_from_host_per_layer(host, list(range(10)), list(range(50, 60)), 1, None)
    for pool, at in ((host, range(10)), (dev, range(40, 50)), (dev, range(50, 60))):
        got = pool.load_rows(1, torch.tensor(list(at), device=DEV))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    with pytest.raises(ValueError, match="k_scale"):
        dev.set_kv_buffer(None, loc, k, v, k_scale=2.0, layer_id_override=0)
    with pytest.raises(NotImplementedError, match="4 bits"):
        dev.get_key_buffer(0)


@pytest.mark.parametrize("name", ["DirectKV4BitTokenToKVPool", "DirectKVTokenToKVPool"])
def test_a_fresh_pool_loads_rows_that_the_gpu_has_just_stored(name):
    make = lambda: getattr(directkv_b200, name)(size=127, page_size=1, dtype=torch.bfloat16, head_num=4, head_dim=128, layer_num=1,  # noqa: E731
                                                start_layer=0, end_layer=0)
    host, fresh = make(), make()
    g = torch.Generator().manual_seed(6)
    k, v = (torch.randn(64, 4, 128, generator=g).to(torch.bfloat16).to(DEV) for _ in range(2))
    loc, busy = torch.arange(64, device=DEV), torch.randn(4096, 4096, device=DEV)
    torch.cuda.synchronize()
    for _ in range(20):
        busy = busy @ busy * 1e-3                         # the store is still to come when the copy is asked for
    host.set_kv_buffer(None, loc, k, v, layer_id_override=0)
    fresh.load_from_host_per_layer(host, list(range(64)), list(range(30, 94)), 0, None)
    if name == "DirectKV4BitTokenToKVPool":
        got = fresh.load_rows(0, loc + 30)
        want = [ref.values(*ref.quantise(x.cpu())) for x in (k, v)]
        assert all(torch.equal(a.cpu().double(), b) for a, b in zip(got, want))
    else:
        assert torch.equal(fresh.k_buffer[0][30:94], k.cpu()) and torch.equal(fresh.v_buffer[0][30:94], v.cpu())


def test_long_prompts_of_unlike_lengths_are_not_padded_to_the_longest():
    """One prompt of 3000 tokens beside 12 short ones: what a call holds on the device stays near the rows themselves, and every request
    gets its own answer."""
    torch.manual_seed(0)
    ctx_len, n_req = 3000, 13
    model = FakeModel(LAYERS, H, NH_Q, NH_KV, None, ctx_len).to(DEV)
    runner = make_runner(model, H, NH_Q, NH_KV, LAYERS, DEV, max_reqs=n_req, context_len=ctx_len)
    be = directkv_b200.DirectKVBackend(runner)
    pool = directkv_b200.DirectKV4BitTokenToKVPool(size=5000, page_size=1, dtype=torch.bfloat16, head_num=NH_KV, head_dim=D, layer_num=LAYERS,
                                                   start_layer=0, end_layer=LAYERS - 1, location="device")
    lens = [40 + 5 * i for i in range(n_req)]
    lens[4] = ctx_len
    perm, at = (torch.randperm(5000, generator=torch.Generator().manual_seed(3)) + 1).int(), 0
    r2t = runner.req_to_token_pool
    for rid, n in enumerate(lens):
        r2t.req_to_token[rid, :n] = perm[at:at + n].to(DEV)
        at += n
    g = torch.Generator().manual_seed(12)
    n = sum(lens)
    q, k, v = _rows(g, n, NH_Q), _rows(g, n, NH_KV), _rows(g, n, NH_KV)
    loc = torch.cat([r2t.req_to_token[rid, :m] for rid, m in enumerate(lens)])
    fb = make_batch(EXTEND, lens, list(range(n_req)), DEV, extend_lens=lens, prefix_lens=[0] * n_req, token_pool=pool, req_to_token_pool=r2t, out_cache_loc=loc)
    be.init_forward_metadata(fb)
    qd, kd, vd = (x.to(DEV) for x in (q, k, v))
    for _ in range(2):                                    # (the first call sizes the library's own scratch)
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        out = be.forward_extend(qd, kd, vd, model.layers[1].attn, fb)
        torch.cuda.synchronize()
    row = NH_KV * D * 2
    queries = 4 * n * NH_Q * D * 2                        # out, its parts and gathered queries
    assert torch.cuda.max_memory_allocated() - before <= 2 * (2 * n * row) + queries + (1 << 20)
    ref_kv, at = Mirror(), 0
    for rid, m in enumerate(lens):
        if m < 200:
            ref_kv.add(rid, k[at:at + m], v[at:at + m])
            ref_kv.check(rid, q[at:at + m], out[at:at + m], extend=True)
        else:                                             # the last rows of the long one
            kk, vv = (ref.values(*ref.quantise(x[at:at + m].view(-1, NH_KV, D))) for x in (k, v))
            o, _, bound = ref.attend(q[at + m - 9:at + m].view(-1, NH_Q, D), kk, vv, m, D ** -0.5)
            bound = bound + 2 * 2.0 ** -8 * vv.abs().amax(0).repeat_interleave(NH_Q // NH_KV, 0)
            assert ((out[at + m - 9:at + m].cpu().double().view(o.shape) - o).abs() <= bound).all()
        at += m
    assert get_context(0).read_status() == 0


@pytest.mark.parametrize("of_runner", [False, True])
def test_a_served_model_keeps_its_cache_in_four_bits(of_runner):
    """The attention modules run, so that their hooks hand over the hidden states: prefill, eager steps and replays of a padded graph store to
    the 4-bit pool and attend it."""
    be, r2t, layer, pool = _setup("device")
    if of_runner:
        be._model_runner.token_to_kv_pool = pool
    g = torch.Generator().manual_seed(13)
    ref_kv = Mirror()
    lens = {2: 62, 4: 9, 5: 130}
    loc = torch.cat([r2t.req_to_token[r, :n] for r, n in lens.items()])
    n = sum(lens.values())
    fb = make_batch(EXTEND, list(lens.values()), list(lens), DEV, extend_lens=list(lens.values()), prefix_lens=[0] * 3, token_pool=pool, req_to_token_pool=r2t,
                    out_cache_loc=loc)
    be.init_forward_metadata(fb)
    q, k, v = _rows(g, n, NH_Q), _rows(g, n, NH_KV), _rows(g, n, NH_KV)
    layer(hidden_states=torch.randn(n, H, generator=g).to(torch.bfloat16).to(DEV))
    out = be.forward_extend(q.to(DEV), k.to(DEV), v.to(DEV), layer.attn, fb)
    at = 0
    for rid, m in lens.items():
        ref_kv.add(rid, k[at:at + m], v[at:at + m])
        ref_kv.check(rid, q[at:at + m], out[at:at + m], extend=m * (NH_Q // NH_KV) >= 128)
        at += m

    def decode(rids, run):
        loc = torch.stack([r2t.req_to_token[r, lens[r]] for r in rids])
        x, q, k, v = torch.randn(len(rids), H, generator=g).to(torch.bfloat16), _rows(g, len(rids), NH_Q), _rows(g, len(rids), NH_KV), _rows(g, len(rids), NH_KV)
        for r in rids:
            lens[r] += 1
        out = run(rids, loc, x, q, k, v)
        for i, r in enumerate(rids):
            ref_kv.add(r, k[i:i + 1], v[i:i + 1])
            ref_kv.check(r, q[i:i + 1], out[i:i + 1], extend=False)

    def eager(rids, loc, x, q, k, v):
        fb = make_batch(DECODE, [lens[r] for r in rids], rids, DEV, token_pool=pool, req_to_token_pool=r2t, out_cache_loc=loc)
        be.init_forward_metadata(fb)
        layer(hidden_states=x.to(DEV))
        return be.forward_decode(q.to(DEV), k.to(DEV), v.to(DEV), layer.attn, fb)

    decode([4, 2, 5], eager)
    bs = 4
    be.init_cuda_graph_state(bs, bs)
    b = dict(x=torch.zeros(bs, H, dtype=torch.bfloat16, device=DEV), q=torch.zeros(bs, NH_Q * D, dtype=torch.bfloat16, device=DEV),
             k=torch.zeros(bs, NH_KV * D, dtype=torch.bfloat16, device=DEV), v=torch.zeros(bs, NH_KV * D, dtype=torch.bfloat16, device=DEV),
             loc=torch.zeros(bs, dtype=torch.int32, device=DEV), rid=torch.zeros(bs, dtype=torch.int64, device=DEV), lens=torch.ones(bs, dtype=torch.int64, device=DEV))
    be.init_forward_metadata_capture_cuda_graph(bs, bs, b["rid"], b["lens"], None, DECODE, None)
    fb = make_batch(DECODE, [1] * bs, [0] * bs, DEV, token_pool=pool, req_to_token_pool=r2t, out_cache_loc=b["loc"])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer(hidden_states=b["x"])
        out_g = be.forward_decode(b["q"], b["k"], b["v"], layer.attn, fb)

    def replay(rids, loc, x, q, k, v):
        n = len(rids)
        for name, t in (("x", x), ("q", q), ("k", k), ("v", v), ("loc", loc)):
            b[name][:n].copy_(t)
        fill = be.get_cuda_graph_seq_len_fill_value()
        here = torch.tensor([lens[r] for r in rids] + [fill] * (bs - n))
        b["loc"][n:] = 0
        b["rid"].copy_(torch.tensor(list(rids) + [0] * (bs - n))), b["lens"].copy_(here)
        be.init_forward_metadata_replay_cuda_graph(bs, b["rid"], b["lens"], int(here.sum()), None, DECODE, None, seq_lens_cpu=here)
        graph.replay()
        torch.cuda.synchronize()
        return out_g

    for _ in range(3):                                    # request 2 reaches the fill length on the way
        decode([4, 5, 2], replay)
    assert lens[2] == 66 and get_context(0).read_status() == 0
    assert (be._pool is None) == of_runner
    graph.reset()
