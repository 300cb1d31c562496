"""Argument checks of the 4-bit cache's operators, their C structs, and the plain forms the GPU tests compare with: no GPU."""

import os
import re

import pytest
import torch

import kv4_ref as ref

from directkv_b200 import _lib, kernel

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BF = torch.bfloat16


def _pool(n=32, nh=2, **kw):
    return kernel.KV4Pool.empty(n, nh, device="cpu", **kw)


def _i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def test_struct_layouts_match_header_field_order():
    text = open(os.path.join(ROOT, "include", "directkv_b200.h")).read()
    for name, cls in (("dkv_kv4_pool", _lib.Kv4PoolDesc), ("dkv_decode_kv4_args", _lib.DecodeKv4Args), ("dkv_qk_norm_args", _lib.QkNormArgs),
                      ("dkv_pages_args", _lib.PagesArgs)):
        body = re.sub(r"/\*.*?\*/", "", re.search(r"typedef struct \{([^}]*)\} " + name + ";", text).group(1), flags=re.S)
        assert re.findall(r"([a-z_0-9]+)\s*;", body) == [f[0] for f in cls._fields_], name


def test_plain_form_of_the_format():
    """The format by hand: a block whose maximum is 6 has scale 1, and its values go to the nearest code."""
    x = torch.zeros(1, 128, dtype=BF)
    x[0, :8] = torch.tensor([6.0, 0.25, 0.75, -1.25, 2.5, 3.5, -5.0, 0.3])
    codes, scales = ref.quantise(x)
    assert scales[0, 0] == 0x38 and scales[0, 1] == 1
    assert ref.values(codes, scales)[0, :8].tolist() == [6.0, 0.0, 1.0, -1.0, 2.0, 4.0, -4.0, 0.5]
    assert codes[0, 0] == 0x07 and codes[0, 1] == 0xA2
    # what the format holds it keeps
    g = torch.Generator().manual_seed(0)
    y = ref.values(*ref.quantise(torch.randn(50, 128, generator=g).to(BF)))
    assert torch.equal(ref.values(*ref.quantise(y.to(BF))), y)
    assert torch.equal(torch.arange(1, 127).to(torch.uint8).view(torch.float8_e4m3fn).double(), ref.E4M3[1:])


def test_pool_checks():
    c, s = torch.zeros(8, 2, 64, dtype=torch.uint8), torch.zeros(8, 2, 8, dtype=torch.uint8)
    pool = kernel.KV4Pool(c, s, c.clone(), s.clone(), page_size=4, k_scale=0.25)
    assert (pool.n_slots, pool.nh_kv, pool.nbytes()) == (8, 2, 8 * 2 * 144)
    for kw in (dict(page_size=3), dict(page_size=0), dict(k_scale=3.0), dict(v_scale=0.0), dict(v_scale=-1.0), dict(k_scale=2.0 ** 25), dict(k_scale=float("nan"))):
        with pytest.raises(RuntimeError, match="power of two"):
            kernel.KV4Pool(c, s, c, s, **kw)
    for args in ((c[:, :, :32], s, c, s), (c, s[:4], c, s), (c, s, c.float(), s), (c, s, c[::2], s), (c, c, c, s), (c[0], s, c, s)):
        with pytest.raises(RuntimeError, match="k_codes|codes must|scales must"):
            kernel.KV4Pool(*args)


def test_store_and_load_refuse():
    pool = _pool()
    k = torch.zeros(3, 2, 128, dtype=BF)
    ok = _i32(3)
    for slots, kk, vv, why in ((_i32(2), k, k, "must be"), (ok.float(), k, k, "int32 or int64"), (_i32(6)[::2], k, k, "contiguous"), (_i32(3, 1), k, k, "1D"),
                               (ok, k[:, :1], k, "must be"), (ok, k.float(), k, "bfloat16"), (ok, k, k.transpose(1, 2).contiguous().transpose(1, 2), "next to each other"),
                               (ok, k[..., :64], k, "next to each other|must be"), (ok, k, k, "CUDA tensor")):
        with pytest.raises(RuntimeError, match=why):
            kernel.store_kv4(pool, slots, kk, vv)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        kernel.load_kv4(pool, ok)
    with pytest.raises(RuntimeError, match="int32 or int64"):
        kernel.load_kv4(pool, ok.short())


def test_decode_refuses():
    pool = _pool()
    q = torch.zeros(2, 4, 128, dtype=BF)
    lens, table = _i32(2), _i32(2, 3)
    cases = [
        (dict(q=q[:, :3]), "multiple of"), (dict(q=q.float()), "bfloat16"), (dict(q=torch.zeros(2, 500, dtype=BF)), "must be"),
        (dict(q=torch.zeros(2, 2, 2, 4, 128, dtype=BF)), "3D or 4D"), (dict(q=torch.zeros(4, 3, 4, 128, dtype=BF)[::2, :2]), "evenly spaced"),
        (dict(q=torch.zeros(2, 0, 4, 128, dtype=BF)), "at most"), (dict(q=torch.zeros(2, 1025, 4, 128, dtype=BF)), "at most"),
        (dict(q=torch.zeros(4097, 4, 128, dtype=BF), seq_lens=_i32(4097), page_table=_i32(4097, 1)), "at most"),
        (dict(seq_lens=_i32(3)), "seq_lens"), (dict(seq_lens=lens.long()), "seq_lens"), (dict(page_table=table.long()), "page_table"), (dict(page_table=_i32(6)), "page_table"),
        (dict(page_table=_i32(3, 2).t()), "page_table"), (dict(page_table=_i32(1, 3)), "rows for 2"), (dict(row_map=_i32(1)), "row_map"), (dict(lse_out=torch.zeros(2, 3)), "lse_out"),
        (dict(lse_out=torch.zeros(2, 4).double()), "lse_out"), ({}, "CUDA tensor"),
    ]
    for kw, why in cases:
        a = dict(q=q, pool=pool, seq_lens=lens, softmax_scale=1.0, page_table=table)
        a.update(kw)
        with pytest.raises(RuntimeError, match=why):
            kernel.decode_kv4(**a)


def test_qk_norm_rope_refuses():
    q, k, pos, cs, w = torch.zeros(3, 4, 128, dtype=BF), torch.zeros(3, 2, 128, dtype=BF), _i32(3), torch.zeros(9, 128), torch.ones(128, dtype=BF)
    cuda = "CUDA tensor"
    cases = [
        (dict(q=None, k=None), "must be given"), (dict(q=q[:2]), "must be"), (dict(k=k[0]), "must be"), (dict(q=q.float()), "bfloat16"), (dict(q=q[..., ::2]), "next to each other"),
        (dict(q_out=q[:, :2]), "shape of q"), (dict(q_out=q.float()), "bfloat16"), (dict(q_weight=w.half()), "q_weight|" + cuda), (dict(k_weight=torch.ones(3, 128, dtype=BF)), "k_weight|" + cuda),
        (dict(q_weight=torch.ones(64, dtype=BF)), "q_weight"), ({}, cuda),
    ]
    for kw, why in cases:
        a = dict(q=q, k=k, positions=pos, cos_sin=cs, q_weight=w, k_weight=w)
        a.update(kw)
        with pytest.raises(RuntimeError, match=why):
            kernel.qk_norm_rope(**a)


def test_pages_refuse():
    table, lens, free, n = _i32(4, 3), _i32(2), _i32(8), _i32(1)
    base = dict(page_table=table, lens=lens, new_lens=lens, free_pages=free, n_free=n, page_size=16, n_tokens=4)
    cases = [
        (dict(lens=lens.long()), "lens"), (dict(new_lens=_i32(3)), "new_lens"), (dict(rows=_i32(1)), "rows"), (dict(page_table=table.t()), "page_table"), (dict(page_table=_i32(4)), "page_table"),
        (dict(page_table=_i32(1, 3).expand(4, 3)), "overlap"), (dict(free_pages=free.long()), "free_pages"), (dict(free_pages=free[::2]), "free_pages"), (dict(n_free=_i32(2)), "n_free"),
        (dict(page_size=12), "power of two"), (dict(lens=_i32(4097), new_lens=_i32(4097)), "at most 4096"), ({}, "CUDA tensor"),
    ]
    for kw, why in cases:
        with pytest.raises(RuntimeError, match=why):
            kernel.assign_pages(**{**base, **kw})
    rel = {k: v for k, v in base.items() if k not in ("new_lens", "n_tokens")}
    for kw, why in (({}, "CUDA tensor"), (dict(keep_lens=_i32(1)), "keep_lens")):
        with pytest.raises(RuntimeError, match=why):
            kernel.release_pages(**{**rel, "keep_lens": lens, **kw})


def test_plain_pages_restore_the_stack():
    table = torch.zeros(2, 9, dtype=torch.int32)
    p = ref.Pages(table, torch.arange(1, 20), 19, 4)
    slots, pos, lens, cu = p.assign([0, 1], [0, 0], [5, 9])
    assert slots[:5] == [76, 77, 78, 79, 72] and pos[5:] == list(range(9)) and cu == [0, 5, 14] and p.n == 14
    p.release([0, 1], lens, [0, 0])
    assert p.stack == list(range(1, 20)) and p.n == 19


def test_packed_arguments_are_the_c_structs():
    """The wrappers pack the structs' bytes themselves: sizes and the place of every field agree with the declared ones."""
    import ctypes
    import struct

    for cls, fmt in ((_lib.DecodeKv4Args, "@iiiPqPqPPqiiPfP"), (_lib.QkNormArgs, "@qiiPqPqPqPqPPiiiiPiPif"), (_lib.PagesArgs, "@PqiiPPPiiPiP")):
        values = [float(i + 1) if f is ctypes.c_float else i + 1 for i, (_, f) in enumerate(cls._fields_)]
        packed = struct.pack(fmt, *values)
        assert len(packed) <= ctypes.sizeof(cls)
        back = cls.from_buffer_copy(packed + bytes(ctypes.sizeof(cls) - len(packed)))
        assert [getattr(back, n) for n, _ in cls._fields_] == values, cls


def test_four_bit_token_pool_checks():
    import directkv_b200

    args = dict(size=30, page_size=1, dtype=BF, head_num=2, head_dim=128, layer_num=3)
    pool = directkv_b200.DirectKV4BitTokenToKVPool(**args, start_layer=4, end_layer=6)
    assert pool.n_slots == 31 and pool.get_kv_size_bytes() == (3 * 31 * 2 * 72,) * 2
    assert pool.layer_pool(5).nh_kv == 2 and pool.layer_pool(5) is not pool.layer_pool(6)
    for kw, why in ((dict(dtype=torch.float16), "bfloat16"), (dict(head_dim=64), "head_dim"), (dict(location="disk"), "location")):
        with pytest.raises(ValueError, match=why):
            directkv_b200.DirectKV4BitTokenToKVPool(**{**args, **kw})
    rows = torch.zeros(2, 2, 128, dtype=BF)
    with pytest.raises(RuntimeError, match="no CPU quantiser"):
        pool.set_kv_buffer(None, torch.tensor([1, 2]), rows, rows, layer_id_override=4)
    with pytest.raises(ValueError, match="v_scale"):
        pool.set_kv_buffer(None, torch.tensor([1, 2]), rows, rows, v_scale=0.5, layer_id_override=4)
    for f in (pool.get_key_buffer, pool.get_value_buffer):
        with pytest.raises(NotImplementedError, match="4 bits"):
            f(4)


def test_outputs_like_a_slice_are_contiguous():
    """The wrappers allocate with empty_like and take the result's tokens to lie one behind the other."""
    rows = torch.zeros(6, 10, 128, dtype=BF)
    for x in (rows[:, 2:5], rows[:, 2:3], rows[:1, 2:5], rows[::2, :4], rows.view(3, 2, 10, 128)[:, :, 1:3], rows.view(6, 1, 10, 128)[:, :, 1:3]):
        assert kernel._heads_stride(x, "x") > 0 and torch.empty_like(x).is_contiguous()
    flat = torch.zeros(6, 1280, dtype=BF)[:, 128:512]
    assert torch.empty_like(flat).is_contiguous()


def test_decode_refuses_a_row_map_into_a_table_without_rows():
    """The library takes 0 rows for an unknown number and would follow the row map out of the table."""
    q, lens = torch.zeros(2, 4, 128, dtype=BF), _i32(2)
    with pytest.raises(RuntimeError, match="no rows"):
        kernel.decode_kv4(q, _pool(), lens, 1.0, _i32(0, 3), row_map=_i32(2))
    with pytest.raises(RuntimeError, match="CUDA tensor"):                    # no request, nothing to look up: only the device is wrong
        kernel.decode_kv4(q[:0], _pool(), lens[:0], 1.0, _i32(0, 3), row_map=_i32(0))


def test_kernels_that_overlap_the_one_before_use_plain_loads():
    """A kernel that begins with grid_wait() runs while the one before it still writes: read-only loads are not for such data."""
    csrc = os.path.join(ROOT, "directkv_b200", "csrc")
    seen = 0
    for name in sorted(os.listdir(csrc)):
        text = re.sub(r"//[^\n]*", "", open(os.path.join(csrc, name)).read())
        if "grid_wait();" in text:
            seen += 1
            assert "__ldg" not in text and ".nc" not in text and "__restrict__" not in text, name
    assert seen >= 4


@pytest.mark.parametrize("name", ["DirectKV4BitTokenToKVPool", "DirectKVTokenToKVPool"])
def test_moves_between_pools_wait_for_the_stores_of_both(name, monkeypatch):
    """set_kv_buffer of device tensors returns before the rows are written: the host copies afterwards, from either pool's side."""
    import directkv_b200

    waited = []
    monkeypatch.setattr(torch.cuda, "synchronize", waited.append)
    make = lambda: getattr(directkv_b200, name)(size=7, page_size=1, dtype=BF, head_num=1, head_dim=128, layer_num=1, start_layer=0, end_layer=0)  # noqa: E731
    for stored in ("one", "other", "both"):
        here, there = make(), make()
        if stored != "other":
            here._compute_device = torch.device("cuda", 1)
        if stored != "one":
            there._compute_device = torch.device("cuda", 2)
        want = {"one": [1], "other": [2], "both": [1, 2]}[stored]
        for move in (lambda: here.load_from_host_per_layer(there, [1, 2], [3, 4], 0, None), lambda: here.backup_to_host_all_layer(there, [1, 2], [3, 4], None)):
            waited.clear()
            move()
            assert sorted(d.index for d in waited) == want, (stored, waited)


def test_calls_keep_no_tensor_between_them():
    """A call under FakeTensorMode fails, and nothing of it may be left for the calls that follow."""
    from torch._subclasses.fake_tensor import FakeTensor, FakeTensorMode

    pool = _pool()
    with FakeTensorMode(), pytest.raises(RuntimeError):
        kernel.load_kv4(pool, torch.empty(3, dtype=torch.int32, device="cuda"))
    kept = [x for value in vars(kernel).values() for x in (value.values() if isinstance(value, dict) and value is not vars(kernel) else [value])]
    assert not [x for x in kept if isinstance(x, (FakeTensor, torch.Tensor))]
