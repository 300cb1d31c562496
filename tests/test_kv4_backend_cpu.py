"""Host logic of the attention backend over a token pool held in 4 bits: what it registers with the engine, and when.  The engine's
calls are recorded, so no GPU is needed."""

import types

import pytest
import torch

from fake_sglang import DECODE, EXTEND, FakeModel, make_batch, make_runner

import directkv_b200
from directkv_b200 import directkv_backend

H, NH_Q, NH_KV, D, LAYERS = 256, 8, 2, 128, 2
BF = torch.bfloat16


class Engine:
    """Stands in for the kernel module's entry points that the backend calls."""

    def __init__(self, monkeypatch):
        self.layers, self.calls, self.fail = {}, [], False
        for name in ("register_layer", "unregister_layer", "extend_ragged", "decode", "decode_kv4"):
            monkeypatch.setattr(directkv_backend.kernel, name, getattr(self, name))

    def register_layer(self, layer_id, k_pool, v_pool, *weights, page_size=1, row_stride=0, device=None):
        self.layers[layer_id] = (k_pool, v_pool, row_stride)

    def unregister_layer(self, layer_id, device=None):
        del self.layers[layer_id]

    def extend_ragged(self, layer_id, X, Q, s_new, past, rows, scale, is_causal=True, page_table=None, out=None):
        k, v, stride = self.layers[layer_id]
        self.calls.append(("extend", layer_id, list(s_new), list(past), k.numel() + v.numel()))
        if self.fail:
            raise RuntimeError("no room")
        if page_table is None:
            assert max(a + b for a, b in zip(s_new, past)) <= stride and max(rows) < k.shape[0] == v.shape[0]
            # a row's answer tells which request's rows were attended: their sum, and the query itself
            of = torch.cat([k.view(-1, stride, NH_KV, D)[r, :a + b].float().sum().expand(a) for r, a, b in zip(rows, s_new, past)])
            return (Q.float() + of[:, None, None]).to(BF)
        return torch.zeros_like(Q)

    def decode(self, layer_id, q, *a, **kw):
        assert layer_id in self.layers
        self.calls.append(("decode", layer_id))
        return torch.zeros_like(q)

    def decode_kv4(self, q, *a, **kw):
        self.calls.append(("decode_kv4",))
        return torch.zeros_like(q)


class FourBits(directkv_b200.DirectKV4BitTokenToKVPool):
    """Rows that come back are filled with the request's number (its slots begin at 100 times that)."""

    def set_kv_buffer(self, *a, **kw):
        pass

    def load_rows(self, layer_id, loc, k_out=None, v_out=None):
        assert k_out.shape[0] == loc.numel()
        k_out.copy_((loc.float() / 2 ** 20)[:, None, None].expand_as(k_out))
        v_out.zero_()


class Bf16(directkv_b200.DirectKVTokenToKVPool):
    def set_kv_buffer(self, *a, **kw):
        pass


def _pool(cls, size=64):
    return cls(size=size, page_size=1, dtype=BF, head_num=NH_KV, head_dim=D, layer_num=LAYERS, start_layer=0, end_layer=LAYERS - 1)


def _setup(monkeypatch, ctx_len=4096):
    engine = Engine(monkeypatch)
    model = FakeModel(LAYERS, H, NH_Q, NH_KV, None, ctx_len)
    runner = make_runner(model, H, NH_Q, NH_KV, LAYERS, "cpu", max_reqs=8, context_len=ctx_len)
    be = directkv_b200.DirectKVBackend(runner)
    return engine, be, runner.req_to_token_pool, model.layers[1]


def _extend(be, r2t, layer, pool, plan, q=None):
    n = sum(e for _, e, _ in plan)
    fb = make_batch(EXTEND, [p + e for _, e, p in plan], [r for r, _, _ in plan], "cpu", extend_lens=[e for _, e, _ in plan],
                    prefix_lens=[p for _, _, p in plan], token_pool=pool, req_to_token_pool=r2t, out_cache_loc=torch.zeros(n, dtype=torch.int64))
    be._fwd_meta = types.SimpleNamespace(seq_lens_cpu=[p + e for _, e, p in plan], req_pool_indices_cpu=[r for r, _, _ in plan],
                                         extend_seq_lens_cpu=[e for _, e, _ in plan], extend_prefix_lens_cpu=[p for _, _, p in plan])
    q = torch.zeros(n, NH_Q * D, dtype=BF) if q is None else q
    kv = torch.zeros(n, NH_KV * D, dtype=BF)
    return be._extend_token_pool(q, kv, kv, layer.attn, fb)


def test_a_long_prompt_leaves_another_pools_registration_alone(monkeypatch):
    engine, be, r2t, layer = _setup(monkeypatch)
    wide, four = _pool(Bf16), _pool(FourBits)
    _extend(be, r2t, layer, wide, [(1, 40, 0)])
    before = dict(engine.layers)
    assert len(before) == 1
    _extend(be, r2t, layer, four, [(1, 40, 0)])
    assert engine.layers == before                          # the rows of one call are gone, the bf16 pool is as it was
    _extend(be, r2t, layer, wide, [(1, 40, 0)])             # fails where its layer was taken away
    assert [c[1] for c in engine.calls if c[0] == "extend"][0::2] == [next(iter(before))] * 2


def test_a_long_prompt_that_fails_leaves_nothing_registered(monkeypatch):
    engine, be, r2t, layer = _setup(monkeypatch)
    engine.fail = True
    with pytest.raises(RuntimeError, match="no room"):
        _extend(be, r2t, layer, _pool(FourBits), [(1, 40, 0)])
    assert not engine.layers


def test_long_prompts_hold_at_most_twice_their_rows_in_bf16(monkeypatch):
    """One long request beside short ones: nobody is padded to its length, and every request gets its own answer."""
    engine, be, r2t, layer = _setup(monkeypatch)
    plan = [(1, 40, 20), (2, 50, 3000), (3, 32, 0), (4, 33, 0), (5, 64, 100), (6, 40, 0)]
    for rid, e, p in plan:
        r2t.req_to_token[rid, :p + e] = 100 * rid
    n = sum(e for _, e, _ in plan)
    q = torch.randn(n, NH_Q * D, generator=torch.Generator().manual_seed(1)).to(BF)
    out = _extend(be, r2t, layer, _pool(FourBits), plan, q=q)
    total = sum(e + p for _, e, p in plan)
    assert all(c[4] <= 2 * 2 * total * NH_KV * D for c in engine.calls), [c[4] for c in engine.calls]
    assert sorted(x for c in engine.calls for x in c[2]) == sorted(e for _, e, _ in plan)
    at = 0
    for rid, e, p in plan:
        of = torch.full((p + e, NH_KV, D), 100 * rid / 2 ** 20).to(BF).float().sum()
        want = (q[at:at + e].float() + of).to(BF)
        assert torch.equal(out[at:at + e], want), rid
        at += e
    assert not engine.layers
    # like lengths stay one call
    engine.calls.clear()
    _extend(be, r2t, layer, _pool(FourBits), [(1, 40, 20), (2, 50, 60), (3, 32, 0)])
    assert len(engine.calls) == 1


def _batch(mode, lens, rids, pool, r2t, ext=None, pre=None):
    n = sum(ext) if ext else len(lens)
    return make_batch(mode, lens, rids, "cpu", extend_lens=ext, prefix_lens=pre, token_pool=pool, req_to_token_pool=r2t, out_cache_loc=torch.zeros(n, dtype=torch.int64))


@pytest.mark.parametrize("of_runner", [False, True])
def test_a_running_model_uses_the_four_bit_pool(monkeypatch, of_runner):
    """The modules' hooks hand over hidden states, as in a served model: the steps store to the 4-bit pool and attend it all the same, and no
    request pool is made beside it."""
    engine, be, r2t, layer = _setup(monkeypatch)
    stored = []
    pool = _pool(FourBits)
    monkeypatch.setattr(pool, "set_kv_buffer", lambda layer, loc, k, v: stored.append(k.shape[0]), raising=False)
    be._model_runner.token_to_kv_pool = pool if of_runner else None
    given = None if of_runner else pool
    fb = _batch(EXTEND, [40, 7], [1, 2], given, r2t, [40, 7], [0, 0])
    be.init_forward_metadata(fb)
    layer(hidden_states=torch.zeros(47, H, dtype=BF))
    kv = torch.zeros(47, NH_KV * D, dtype=BF)
    be.forward_extend(torch.zeros(47, NH_Q * D, dtype=BF), kv, kv, layer.attn, fb)
    fb = _batch(DECODE, [41, 8], [1, 2], given, r2t)
    be.init_forward_metadata(fb)
    layer(hidden_states=torch.zeros(2, H, dtype=BF))
    be.forward_decode(torch.zeros(2, NH_Q * D, dtype=BF), kv[:2], kv[:2], layer.attn, fb)
    assert stored == [47, 2] and [c[0] for c in engine.calls] == ["extend", "decode_kv4", "decode_kv4"]
    assert be._pool is None and not be._hidden and not engine.layers


def test_graphs_over_a_four_bit_pool_keep_every_length(monkeypatch):
    """A replayed batch has the lengths and requests it is given, one of the fill length among them, whatever the request pool knows."""
    engine, be, r2t, layer = _setup(monkeypatch)
    monkeypatch.setattr(directkv_backend, "get_context", lambda dev: types.SimpleNamespace(reserve=lambda *a: None))
    pool = _pool(FourBits)
    be._model_runner.token_to_kv_pool = pool
    be.init_cuda_graph_state(4, 4)
    fill = be.get_cuda_graph_seq_len_fill_value()
    be.init_forward_metadata_capture_cuda_graph(3, 3, torch.tensor([0, 0, 0]), torch.ones(3), None, DECODE, None)
    layer(hidden_states=torch.zeros(3, H, dtype=BF))
    kv = torch.zeros(3, NH_KV * D, dtype=BF)
    be.forward_decode(torch.zeros(3, NH_Q * D, dtype=BF), kv, kv, layer.attn, _batch(DECODE, [fill] * 3, [0, 0, 0], pool, r2t))
    lens = torch.tensor([91, 5, fill])
    be.init_forward_metadata_replay_cuda_graph(3, torch.tensor([4, 2, 6]), lens, int(lens.sum()), None, DECODE, None, seq_lens_cpu=lens)
    assert be._fwd_meta.seq_lens_dev.tolist() == [91, 5, fill] and be._fwd_meta.req_idx_dev.tolist() == [4, 2, 6]
    assert be._fwd_meta.seq_lens_dev.data_ptr() == be._cg_seq_lens.data_ptr() and be._fwd_meta.req_idx_dev.data_ptr() == be._cg_req.data_ptr()
    assert be._pool is None and [c[0] for c in engine.calls] == ["decode_kv4"]
