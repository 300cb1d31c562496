"""Workloads of the operators around a paged KV cache that is held in 4 bits.

Four operators are measured, each as a serving program calls it:

  attend   decode attention over a 4-bit paged pool (one token per request, or a few drafted ones)
  store    quantising new K/V rows into a 4-bit pool and reading them back as bf16 (what a chunked prefill does)
  rotate   RMS norm of every query and key head with the Neox position rotation in the same pass
  pages    block tables and slot maps from request lengths, and the release of the same pages

``own`` chooses between the plain form (elementary torch operations) and the package's kernels.

The 4-bit form of a row of 128 values: blocks of 16 consecutive dimensions, one e4m3 scale per block
(s = e4m3(max|y| / 6), at least 2^-9), one e2m1 code per value (nearest of y / s, ties to the even code); two codes per byte, the
lower dimension in the lower four bits.  y is the value over the pool's power-of-two scale; not-a-number counts as zero, infinities
as the largest value that the form holds.
"""

import math
import random

import torch

own = False

DEV = "cuda"
D = 128
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)             # magnitudes of the e2m1 codes 0..7
MOST = 6.0 * 448.0


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # One chat request just after its prompt: a call whose latency counts, not its bytes.
        dict(name="attend 1 short", kind="attend", batch=1, low=77, high=77, nh_q=32, nh_kv=8, q_len=1, page=16, lens_seed=1),
        # An ordinary decode batch of a grouped-query layer, ragged lengths.
        dict(name="attend 32 ragged", kind="attend", batch=32, low=300, high=8000, nh_q=32, nh_kv=8, q_len=1, page=16, lens_seed=2),
        # One long document.
        dict(name="attend 1 long", kind="attend", batch=1, low=131071, high=131071, nh_q=32, nh_kv=8, q_len=1, page=64, lens_seed=3),
        # One query head per KV head, token-indexed pool (page size 1).
        dict(name="attend 8 mha tokens", kind="attend", batch=8, low=900, high=2048, nh_q=32, nh_kv=32, q_len=1, page=1, lens_seed=4),
        # Four drafted tokens per request, each attending its own prefix.
        dict(name="attend 16 drafts", kind="attend", batch=16, low=5, high=4096, nh_q=32, nh_kv=8, q_len=4, page=16, lens_seed=5),
        # A full batch at long context: the largest call.
        dict(name="attend 64 full", kind="attend", batch=64, low=12000, high=20000, nh_q=32, nh_kv=8, q_len=1, page=16, lens_seed=6),
        # The new tokens of a decode step.
        dict(name="store 16 tokens", kind="store", tokens=16, nh_kv=8, page=16, k_exp=0, v_exp=0),
        # A prefill chunk, odd size, many KV heads.
        dict(name="store 8191 mha", kind="store", tokens=8191, nh_kv=32, page=16, k_exp=1, v_exp=-2),
        # Queries and keys of a decode step ...
        dict(name="rotate 8 tokens", kind="rotate", tokens=8, nh_q=32, nh_kv=8, norm=True, fused=True, max_pos=8192),
        # ... and of a prefill chunk, read out of the fused projection's output.
        dict(name="rotate 16384 tokens", kind="rotate", tokens=16384, nh_q=32, nh_kv=8, norm=True, fused=True, max_pos=131072),
        # Bookkeeping of a decode step: one more token each.
        dict(name="pages 64 steps", kind="pages", batch=64, low=0, high=8000, new_low=1, new_high=1, page=16, lens_seed=7),
        # Admission of a batch of prompts.
        dict(name="pages 256 prompts", kind="pages", batch=256, low=0, high=0, new_low=17, new_high=8000, page=16, lens_seed=8),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(("attend", "attend", "store", "rotate", "pages"))
    if kind == "attend":
        nh_kv, group = rng.choice(((8, 4), (8, 1), (32, 1), (4, 8), (2, 16), (1, 12), (8, 5), (7, 2), (56, 1), (3, 3)))
        q_len = rng.choice((1, 1, 1, 2, 3, 5, 8))
        batch = _log(rng, 1, 200)
        high = _log(rng, 1, min(131072, 8_000_000 // (batch * nh_kv)))
        return dict(kind=kind, batch=batch, low=max(1, int(high * rng.uniform(0.02, 1.0))), high=high, nh_q=nh_kv * group, nh_kv=nh_kv,
                    q_len=q_len, page=rng.choice((1, 4, 16, 64, 256)), lens_seed=rng.randrange(1 << 20))
    if kind == "store":
        return dict(kind=kind, tokens=_log(rng, 1, 16000), nh_kv=rng.choice((1, 2, 3, 7, 8, 16, 32)), page=rng.choice((1, 16, 64)),
                    k_exp=rng.randrange(-3, 4), v_exp=rng.randrange(-3, 4))
    if kind == "rotate":
        nh_kv, group = rng.choice(((8, 4), (32, 1), (4, 8), (1, 5), (7, 4), (2, 1)))
        return dict(kind=kind, tokens=_log(rng, 1, 16000), nh_q=nh_kv * group, nh_kv=nh_kv, norm=rng.random() < 0.8, fused=rng.random() < 0.6,
                    max_pos=rng.choice((2048, 8192, 131072)))
    high = _log(rng, 1, 20000)
    batch = _log(rng, 1, 1000)
    new_high = _log(rng, 1, min(8000, 2_000_000 // batch))
    return dict(kind=kind, batch=batch, low=int(high * rng.random()), high=high, new_low=rng.randrange(0, new_high + 1),
                new_high=new_high, page=rng.choice((1, 8, 16, 64, 128)), lens_seed=rng.randrange(1 << 20))


def _lens(case):
    rng = random.Random(case["lens_seed"])
    return [rng.randint(case["low"], case["high"]) for _ in range(case["batch"])]


def _new_lens(case):
    rng = random.Random(case["lens_seed"] + 1)
    return [rng.randint(case["new_low"], case["new_high"]) for _ in range(case["batch"])]


def _up(n, page):
    return -(-n // page)


def work(case):
    kind = case["kind"]
    if kind == "attend":
        lens = _lens(case)
        pages = sum(_up(n, case["page"]) for n in lens)
        rows = case["batch"] * case["q_len"] * case["nh_q"]
        pairs = sum(max(0, n - case["q_len"] + 1 + j) for n in lens for j in range(case["q_len"]))
        return {"bytes": sum(lens) * case["nh_kv"] * 144 + rows * 512 + pages * 4 + case["batch"] * 4, "flops": 4 * D * case["nh_q"] * pairs}
    if kind == "store":
        rows = case["tokens"] * case["nh_kv"] * 2                              # K and V: bf16 in, 4 bits out, 4 bits in, bf16 out
        return {"bytes": rows * (256 + 72 + 72 + 256) + case["tokens"] * 8, "flops": rows * D * 6}
    if kind == "rotate":
        rows = case["tokens"] * (case["nh_q"] + case["nh_kv"])
        return {"bytes": rows * 512 + min(case["tokens"], case["max_pos"]) * 512 + case["tokens"] * 4, "flops": rows * D * 7}
    lens, new = _lens(case), _new_lens(case)
    pages = sum(_up(a + n, case["page"]) - _up(a, case["page"]) for a, n in zip(lens, new))
    return {"bytes": sum(new) * 8 + pages * 16 + case["batch"] * 24, "flops": sum(new) * 4}


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _normal(shape, g, std=1.0):
    return (torch.randn(shape, generator=g, device=DEV) * std).to(torch.bfloat16)


def _channel_scale(nh, g, spread):
    """Keys have a few strong channels; their positions and sizes differ from head to head."""
    return torch.exp(torch.randn(nh, D, generator=g, device=DEV) * spread)


def prepare(case, seed):
    g = _gen(seed)
    kind = case["kind"]
    state = dict(case=case)
    if kind == "attend":
        lens, page, nh = _lens(case), case["page"], case["nh_kv"]
        counts = [_up(n, page) for n in lens]
        total = sum(counts)
        order = torch.randperm(total, generator=g, device=DEV).to(torch.int32) + 1      # page 0 is the padding page
        table = torch.zeros(case["batch"], _up(case["high"], page), dtype=torch.int32, device=DEV)
        table[torch.arange(table.shape[1], device=DEV) < torch.tensor(counts, device=DEV)[:, None]] = order
        n_slots = (total + 1) * page
        parts = []
        for spread in (0.5, 0.2):
            codes = torch.empty(n_slots, nh, D // 2, dtype=torch.uint8, device=DEV)
            scales = torch.empty(n_slots, nh, D // 16, dtype=torch.uint8, device=DEV)
            chan = _channel_scale(nh, g, spread)
            step = max(1, (1 << 22) // nh // 16)
            for r in range(0, n_slots, step):
                x = torch.randn(min(step, n_slots - r), nh, D, generator=g, device=DEV) * chan
                codes[r:r + step], scales[r:r + step] = _quantise(x, 0)
            parts += [codes, scales]
        state.update(q=_normal((case["batch"], case["q_len"], case["nh_q"], D), g), parts=parts, table=table, n_slots=n_slots,
                     lens=torch.tensor(lens, dtype=torch.int32, device=DEV))
        k_exp = v_exp = 0
    elif kind == "store":
        n, nh = case["tokens"], case["nh_kv"]
        n_slots = (_up(n, case["page"]) * 2 + 1) * case["page"]
        state.update(k=(torch.randn(n, nh, D, generator=g, device=DEV) * _channel_scale(nh, g, 0.5)).to(torch.bfloat16),
                     v=_normal((n, nh, D), g, 0.7), slots=torch.randperm(n_slots, generator=g, device=DEV)[:n].to(torch.int32),
                     parts=[torch.zeros(n_slots, nh, w, dtype=torch.uint8, device=DEV) for w in (D // 2, D // 16, D // 2, D // 16)])
        k_exp, v_exp = case["k_exp"], case["v_exp"]
    elif kind == "rotate":
        n, hq, hk = case["tokens"], case["nh_q"], case["nh_kv"]
        if case["fused"]:                                                    # [q | k | v] rows of one projection
            rows = _normal((n, hq + 2 * hk, D), g, 1.3)
            q, k = rows[:, :hq], rows[:, hq:hq + hk]
        else:
            q, k = _normal((n, hq, D), g, 1.3), _normal((n, hk, D), g, 1.3)
        pos = torch.arange(case["max_pos"], device=DEV, dtype=torch.float64)
        angle = torch.outer(pos, 500000.0 ** (-torch.arange(D // 2, device=DEV, dtype=torch.float64) / (D // 2)))
        first = int(torch.randint(0, max(1, case["max_pos"] - n), (1,), generator=g, device=DEV))
        weights = [(1.0 + 0.2 * torch.randn(D, generator=g, device=DEV)).to(torch.bfloat16) if case["norm"] else None for _ in range(2)]
        state.update(q=q, k=k, cos_sin=torch.cat([angle.cos(), angle.sin()], 1).float().contiguous(), weights=weights,
                     positions=((torch.arange(n, device=DEV) + first) % case["max_pos"]).to(torch.int32))
    else:
        lens, new, page = _lens(case), _new_lens(case), case["page"]
        have = [_up(n, page) for n in lens]
        need = [_up(a + n, page) for a, n in zip(lens, new)]
        total = sum(need) + 7
        order = torch.randperm(total, generator=g, device=DEV).to(torch.int32) + 1
        rows = torch.randperm(case["batch"] + 3, generator=g, device=DEV)[:case["batch"]].to(torch.int32)
        table = torch.zeros(case["batch"] + 3, max(need) + 1, dtype=torch.int32, device=DEV)
        held = table[rows.long()]                                            # pages held already come off the far end of the list
        at = total - sum(have)
        held[torch.arange(table.shape[1], device=DEV) < torch.tensor(have, device=DEV)[:, None]] = order[at:]
        table[rows.long()] = held
        ints = dict(dtype=torch.int32, device=DEV)
        state.update(lens=torch.tensor(lens, **ints), new=torch.tensor(new, **ints), rows=rows, table=table, free=order.clone(),
                     n_free=torch.tensor([at], **ints), tokens=sum(new))
    if own and kind in ("attend", "store"):
        from directkv_b200 import kernel

        state["pool"] = kernel.KV4Pool(*state["parts"], page_size=case["page"], k_scale=2.0 ** k_exp, v_scale=2.0 ** v_exp)
    return state


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(state):
    from directkv_b200 import kernel

    case = state["case"]
    if case["kind"] == "attend":
        return kernel.decode_kv4(state["q"], state["pool"], state["lens"], D ** -0.5, state["table"])
    if case["kind"] == "store":
        kernel.store_kv4(state["pool"], state["slots"], state["k"], state["v"])
        return kernel.load_kv4(state["pool"], state["slots"])
    if case["kind"] == "rotate":
        return kernel.qk_norm_rope(state["q"], state["k"], state["positions"], state["cos_sin"], state["weights"][0], state["weights"][1], eps=1e-6)
    got = kernel.assign_pages(state["table"], state["lens"], state["new"], state["free"], state["n_free"], case["page"], state["tokens"],
                              rows=state["rows"])
    # The tokens are taken back (a rejected draft, a request that was withdrawn): the list is as it was before.
    kernel.release_pages(state["table"], got[2], state["lens"], state["free"], state["n_free"], case["page"], rows=state["rows"])
    return got + (state["table"], state["free"], state["n_free"])


def _quantise(x, exp):
    """Codes and scales of x [..., 128] (see the module's text)."""
    y = torch.nan_to_num(x.float() * 2.0 ** -exp, nan=0.0, posinf=MOST, neginf=-MOST).clamp(-MOST, MOST)
    y = y.reshape(*x.shape[:-1], D // 16, 16)
    s = (y.abs().amax(-1).double() / 6.0).float().to(torch.float8_e4m3fn).float().clamp_min(2.0 ** -9)
    # A border times s has at most 7 significant bits and y 8: the rounded quotient is on a border only where y / s is.
    r = y.abs() / s.unsqueeze(-1)
    mag = torch.where(r < 2.0, torch.round(2.0 * r), torch.where(r < 4.0, torch.round(r) + 2.0, torch.round(0.5 * r) + 4.0)).clamp_max(7.0)
    code = (mag.to(torch.uint8) | ((y < 0).to(torch.uint8) << 3)).reshape(*x.shape[:-1], D // 2, 2)
    return code[..., 0] | (code[..., 1] << 4), s.to(torch.float8_e4m3fn).view(torch.uint8)


def _values(codes, scales, exp):
    """fp32 values of codes [..., 64] and scales [..., 8]."""
    grid = torch.tensor(GRID + tuple(-v for v in GRID), device=codes.device)
    both = torch.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], D // 16, 16)
    out = grid[both.int()] * scales.view(torch.float8_e4m3fn).float().unsqueeze(-1)
    return out.reshape(*codes.shape[:-1], D) * 2.0 ** exp


def _run_plain(state):
    case = state["case"]
    kind = case["kind"]
    if kind == "attend":
        nh, group, n_q, page, batch = case["nh_kv"], case["nh_q"] // case["nh_kv"], case["q_len"], case["page"], case["batch"]
        lens = state["lens"].long()
        t = torch.arange(case["high"], device=DEV)
        slot = state["table"][:, t // page].long() * page + t % page                                # [batch, n]; padding page beyond a request's own
        kc, ks, vc, vs = state["parts"]
        q = state["q"].float().reshape(batch, n_q, nh, group, D).transpose(1, 2).reshape(batch, nh, n_q * group, D)
        s = torch.matmul(q, _values(kc[slot], ks[slot], 0).permute(0, 2, 3, 1)).reshape(batch, nh, n_q, group, -1) * D ** -0.5
        last = lens[:, None] - n_q + torch.arange(n_q, device=DEV)                                  # [batch, n_q]
        s = s.masked_fill((t > last[..., None])[:, None, :, None, :], -math.inf)
        top = s.amax(-1, keepdim=True)
        e = torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top))
        o = torch.matmul(e.reshape(batch, nh, n_q * group, -1), _values(vc[slot], vs[slot], 0).transpose(1, 2)).reshape(batch, nh, n_q, group, D)
        total = e.sum(-1, keepdim=True)
        out = torch.where(total > 0, o / total, torch.zeros_like(o)).transpose(1, 2).reshape(state["q"].shape).to(torch.bfloat16)
        return out
    if kind == "store":
        kc, ks, vc, vs = state["parts"]
        at = state["slots"].long()
        kc[at], ks[at] = _quantise(state["k"], case["k_exp"])
        vc[at], vs[at] = _quantise(state["v"], case["v_exp"])
        return _values(kc[at], ks[at], case["k_exp"]).to(torch.bfloat16), _values(vc[at], vs[at], case["v_exp"]).to(torch.bfloat16)
    if kind == "rotate":
        cs = state["cos_sin"][state["positions"].long()]
        cos, sin = cs[:, None, :D // 2], cs[:, None, D // 2:]
        outs = []
        for x, w in zip((state["q"], state["k"]), state["weights"]):
            x = x.float()
            if w is not None:
                x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w.float()
            lo, hi = x[..., :D // 2], x[..., D // 2:]
            outs.append(torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1).to(torch.bfloat16))
        return tuple(outs)
    page, lens, new, rows, table = case["page"], state["lens"].long(), state["new"].long(), state["rows"].long(), state["table"]
    have, more = (lens + page - 1) // page, (lens + new + page - 1) // page - (lens + page - 1) // page
    first = torch.cumsum(more, 0) - more
    cu = torch.cat([torch.zeros(1, dtype=torch.long, device=DEV), torch.cumsum(new, 0)])
    b = torch.repeat_interleave(torch.arange(len(more), device=DEV), new, output_size=state["tokens"])      # one entry per token
    pos = lens[b] + torch.arange(b.numel(), device=DEV) - cu[b]
    fresh = pos // page - have[b]                                                                   # >= 0: on a page taken now
    old = table[rows[b], pos // page]
    number = torch.where(fresh >= 0, state["free"][(state["n_free"].long() - 1 - first[b] - fresh).clamp(0, len(state["free"]) - 1)], old)
    table[rows[b], pos // page] = number
    slots = number.long() * page + pos % page
    total = lens + new
    # The release puts the same pages back in the same places of the list and leaves the table's entries.
    return tuple(x.to(torch.int32) for x in (slots, pos, total, cu)) + (table, state["free"], state["n_free"])


# ------------------------------------------------------------------------------------------------ 64 bits, from the definitions
def exact(case, seed):
    state = prepare(case, seed)
    kind = case["kind"]
    f64 = torch.float64
    powers = torch.tensor([2.0 ** i for i in range(-40, 41)], dtype=f64, device=DEV)

    def two(e):                                                              # exact, as a computed power need not be
        return powers[e.clamp(-40, 40).long() + 40]

    def of_scale(byte):                                                      # e4m3: 1.mmm * 2^(e - 7), 0.mmm * 2^-6 for e = 0
        e, m = (byte.long() >> 3) & 15, (byte.long() & 7).to(f64)
        return torch.where(e == 0, m * 2.0 ** -9, (1.0 + m / 8.0) * two(e - 7))

    def of_code(c):                                                          # e2m1: 1.m * 2^(e - 1), 0.m * 2^0 for e = 0
        e, m = (c.long() >> 1) & 3, (c.long() & 1).to(f64)
        mag = torch.where(e == 0, 0.5 * m, (1.0 + 0.5 * m) * two(e - 1))
        return torch.where((c & 8) != 0, -mag, mag)

    def rows_of(codes, scales):
        out = torch.empty(*codes.shape[:-1], D, dtype=f64, device=DEV)
        out[..., 0::2], out[..., 1::2] = of_code(codes & 15), of_code(codes >> 4)
        return out * of_scale(scales).repeat_interleave(16, -1)

    if kind == "attend":
        page, nh, group, n_q = case["page"], case["nh_kv"], case["nh_q"] // case["nh_kv"], case["q_len"]
        kc, ks, vc, vs = state["parts"]
        out = torch.zeros(case["batch"], n_q, case["nh_q"], D, dtype=f64, device=DEV)
        for b, n in enumerate(state["lens"].tolist()):
            pages = state["table"][b, :_up(n, page)].long()
            slot = (pages[:, None] * page + torch.arange(page, device=DEV)).reshape(-1)[:n]
            k, v = rows_of(kc[slot], ks[slot]), rows_of(vc[slot], vs[slot])
            for j in range(n_q):
                m = n - n_q + 1 + j
                if m > 0:
                    p = torch.softmax(torch.einsum("mhd,hgd->hgm", k[:m], state["q"][b, j].to(f64).view(nh, group, D)) / math.sqrt(D), -1)
                    out[b, j] = torch.einsum("hgm,mhd->hgd", p, v[:m]).reshape(nh * group, D)
        return out
    if kind == "store":
        outs = []
        for x, exp in ((state["k"], case["k_exp"]), (state["v"], case["v_exp"])):
            y = (x.to(f64) / 2.0 ** exp).reshape(*x.shape[:-1], D // 16, 16)
            want = y.abs().amax(-1, keepdim=True)
            want = want / torch.full_like(want, 6.0)                         # a true division: halves between two scales occur
            unit = two((torch.frexp(want).exponent - 1).clamp_min(-6) - 3)    # an eighth of the power of two below
            s = (torch.round(want / unit) * unit).clamp(2.0 ** -9, 448.0)    # torch.round: ties to even
            mag = torch.zeros_like(y)
            for at, upper, rise in ((0.25, False, 0.5), (0.75, True, 0.5), (1.25, False, 0.5), (1.75, True, 0.5), (2.5, False, 1.0), (3.5, True, 1.0),
                                    (5.0, False, 2.0)):                      # a value on a border goes to the code that is even
                mag += rise * ((y.abs() >= at * s) if upper else (y.abs() > at * s))
            outs.append((torch.sign(y) * mag * s * 2.0 ** exp).reshape(x.shape))
        return tuple(outs)
    if kind == "rotate":
        outs = []
        cs = state["cos_sin"].to(f64)[state["positions"].long()]
        turn = torch.complex(cs[:, :D // 2], cs[:, D // 2:])[:, None]
        for x, w in zip((state["q"], state["k"]), state["weights"]):
            x = x.to(f64)
            if w is not None:
                x = x / torch.sqrt(x.square().sum(-1, keepdim=True) / D + 1e-6) * w.to(f64)
            z = torch.complex(x[..., :D // 2].contiguous(), x[..., D // 2:].contiguous()) * turn
            outs.append(torch.cat([z.real, z.imag], -1))
        return tuple(outs)
    page, lens, new, rows = case["page"], _lens(case), _new_lens(case), state["rows"].tolist()
    free, n = state["free"].tolist(), int(state["n_free"])
    table = state["table"].cpu()
    slots, positions, cu = [], [], [0]
    for row, a, more in zip(rows, lens, new):
        line = table[row].tolist()
        for t in range(a, a + more):
            if t % page == 0:                                                # a new page starts here
                n -= 1
                line[t // page] = free[n]
            slots.append(line[t // page] * page + t % page)
            positions.append(t)
        table[row] = torch.tensor(line, dtype=torch.int32)
        cu.append(len(slots))
    as_int = [torch.tensor(x, dtype=torch.int32, device=DEV) for x in (slots, positions, [a + b for a, b in zip(lens, new)], cu)]
    return tuple(as_int) + (table.to(DEV), state["free"], state["n_free"])
