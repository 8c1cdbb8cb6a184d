"""Cases of the paged key/value cache operators: append with rotation, attention, and both over a cache in 4 bits.

``run`` computes them as elementary torch operations in 32 bits, or, with ``own``, through the package.
"""
import math
import random

import torch

own = False

_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _case(name, op, dtype="bf16", fmt="16bit", batch=1, q_len=1, kv_len=1024, ragged=False, heads=32, kv_heads=8,
          head_dim=128, page=16, layout="hnd", window=0, softcap=0.0, base=10000.0, lens_seed=1):
    c = dict(op=op, dtype=dtype, fmt=fmt, batch=batch, q_len=q_len, kv_len=kv_len, ragged=ragged, heads=heads,
             kv_heads=kv_heads, head_dim=head_dim, page=page, layout=layout, window=window, softcap=softcap, base=base,
             lens_seed=lens_seed)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # one decode step of 8 sequences far into their context: the smallest call, all latency
        _case("append_step_8", "append", batch=8, kv_len=131072, ragged=True, page=16, base=500000.0),
        # a prompt chunk of several sequences packed together
        _case("append_prompt_8192", "append", dtype="f16", batch=5, q_len=2731, kv_len=2731, ragged=True, page=64,
              layout="nhd"),
        # one sequence, one token, a short odd context: what a chat user waits for
        _case("attend_step_1x700", "attend", batch=1, kv_len=700),
        # a server's decode batch of uneven lengths
        _case("attend_step_64x8192", "attend", batch=64, kv_len=8192, ragged=True, page=32, lens_seed=3),
        # few sequences with long contexts
        _case("attend_step_8x65536", "attend", batch=8, kv_len=65536, page=64),
        # multi-head decode of 64-wide heads with a window and capped scores
        _case("attend_window_cap", "attend", dtype="f16", batch=24, kv_len=12000, ragged=True, heads=16, kv_heads=16,
              head_dim=64, page=16, layout="nhd", window=4096, softcap=50.0, lens_seed=5),
        # a whole prompt in one pass
        _case("attend_prompt_4096", "attend", q_len=4096, kv_len=4096, page=128),
        # prompt chunks of uneven lengths behind cached prefixes, capped scores
        _case("attend_chunks_cap", "attend", dtype="f16", batch=6, q_len=777, kv_len=3001, ragged=True, heads=24,
              kv_heads=8, page=16, softcap=30.0, lens_seed=7),
        # a decode step into a 4-bit cache, read back
        _case("append4_step_48", "append", fmt="nvfp4", batch=48, kv_len=20000, ragged=True, page=32, lens_seed=9),
        # a prompt into a 4-bit cache, read back
        _case("append4_prompt_6000", "append", fmt="nvfp4", batch=3, q_len=2500, kv_len=4100, ragged=True, page=64,
              layout="nhd", lens_seed=11),
        # a decode batch over the 4-bit cache
        _case("attend4_step_32x16384", "attend", fmt="nvfp4", batch=32, kv_len=16384, ragged=True, page=64,
              lens_seed=13),
        # prompt chunks over cached 4-bit prefixes
        _case("attend4_chunks", "attend", dtype="f16", fmt="nvfp4", batch=4, q_len=256, kv_len=5000, ragged=True,
              page=32, lens_seed=15),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op, fmt = rng.choice(("append", "attend")), rng.choice(("16bit", "nvfp4"))
    head_dim = rng.choice((64, 128))
    kv_heads = rng.choice((1, 2, 4, 5, 8))
    group = rng.choice((1, 2, 3, 4, 7, 8))
    common = dict(dtype=rng.choice(("bf16", "f16")), fmt=fmt, heads=kv_heads * group, kv_heads=kv_heads,
                  head_dim=head_dim, page=rng.choice((16, 32, 64, 128)), layout=rng.choice(("hnd", "nhd")),
                  ragged=rng.random() < 0.75, lens_seed=rng.randrange(1 << 20))
    if op == "append":
        if rng.random() < 0.5:
            batch, q_len = _log_int(rng, 1, 256), 1
            kv_len = _log_int(rng, 1, 131072 if batch < 32 else 16384)
        else:
            batch, q_len = rng.randint(1, 8), _log_int(rng, 2, 1000)
            kv_len = q_len + _log_int(rng, 1, 2000)
        return _case("", "append", batch=batch, q_len=q_len, kv_len=kv_len, base=rng.choice((10000.0, 500000.0)),
                     **common)
    window = rng.choice((0, 0, _log_int(rng, 1, 5000)))
    softcap = rng.choice((0.0, 0.0, 30.0, 50.0))
    if rng.random() < 0.6:
        batch, q_len = _log_int(rng, 1, 64), rng.choice((1, 1, 1, 2, 4))
        kv_len = _log_int(rng, 5, 262144 // batch if batch > 8 else 32768)
    else:
        batch, q_len = rng.randint(1, 5), _log_int(rng, 5, 900)
        kv_len = q_len + _log_int(rng, 1, 2500)
    return _case("", "attend", batch=batch, q_len=q_len, kv_len=kv_len, window=window, softcap=softcap, **common)


def _lens(case):
    """(tokens, cached length after them) of every sequence: the first has the largest of both."""
    rng = random.Random(case["lens_seed"])
    q, kv = [case["q_len"]], [max(case["q_len"], case["kv_len"])]
    for _ in range(case["batch"] - 1):
        n = rng.randint(max(1, case["q_len"] // 3), case["q_len"]) if case["ragged"] else case["q_len"]
        full = max(case["q_len"], case["kv_len"])
        q.append(n)
        kv.append(max(n, _log_int(rng, max(1, full // 8), full)) if case["ragged"] else full)
    return q, kv


def _dtype(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float16


def _pool(case, pages, last, dtype):
    """An empty pool, always indexed [page, kv head, slot, value]; "nhd" keeps the heads of a slot together."""
    hk, p = case["kv_heads"], case["page"]
    if case["layout"] == "nhd":
        return torch.zeros(pages, p, hk, last, dtype=dtype, device="cuda").permute(0, 2, 1, 3)
    return torch.zeros(pages, hk, p, last, dtype=dtype, device="cuda")


def _quantise(x):
    """Values in blocks of 16 along the last axis: (codes 0..15, e4m3 scales), scale = e4m3(amax / 6)."""
    b = x.reshape(*x.shape[:-1], x.shape[-1] // 16, 16)
    scale = (b.abs().amax(-1) / 6.0).clamp(max=448.0).to(torch.float8_e4m3fn)
    s = scale.float().unsqueeze(-1)
    y = torch.where(s > 0, b / s, torch.zeros_like(b))
    a = y.abs()
    code = ((a > 0.25).int() + (a >= 0.75).int() + (a > 1.25).int() + (a >= 1.75).int() + (a > 2.5).int()
            + (a >= 3.5).int() + (a > 5.0).int())
    code = code + 8 * torch.signbit(y).int()
    return code.reshape(x.shape), scale


def _pack(code):
    return (code[..., 0::2] + 16 * code[..., 1::2]).to(torch.uint8)


def _unpack(packed, scales):
    """The values that packed bytes [.., D/2] and e4m3 bytes [.., D/16] stand for, in 32 bits."""
    table = torch.tensor(_E2M1 + tuple(-v for v in _E2M1), dtype=torch.float32, device=packed.device)
    code = torch.stack((packed % 16, packed // 16), -1).flatten(-2)
    return table[code.int()] * scales.view(torch.float8_e4m3fn).float().repeat_interleave(16, -1)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, d, hk, h, p = _dtype(case), case["head_dim"], case["kv_heads"], case["heads"], case["page"]
    q_lens, kv_lens = _lens(case)
    tokens, batch = sum(q_lens), len(q_lens)
    need = [-(-n // p) for n in kv_lens]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(batch, max(need), dtype=torch.int32, device="cuda")
    at = 0
    for b in range(batch):
        table[b, :need[b]] = order[at:at + need[b]]
        at += need[b]
    cu = torch.tensor([sum(q_lens[:b]) for b in range(batch + 1)], dtype=torch.int32, device="cuda")
    st = dict(case=case, table=table, cu_q=cu, max_q=max(q_lens), scale=d ** -0.5,
              kv_lens=torch.tensor(kv_lens, dtype=torch.int32, device="cuda"))

    def rand(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dt)

    st["q"] = rand(tokens, h, d)
    if case["op"] == "append":
        qkv = rand(tokens, (h + 2 * hk) * d)   # a fused projection's rows
        st["q"] = qkv[:, :h * d].unflatten(-1, (h, d))
        st["k"] = qkv[:, h * d:(h + hk) * d].unflatten(-1, (hk, d))
        st["v"] = qkv[:, (h + hk) * d:].unflatten(-1, (hk, d))
        i = torch.arange(0, d, 2, dtype=torch.float64, device="cuda")
        st["inv_freq"] = (case["base"] ** (-i / d)).float()
        st["rows"] = [torch.empty(tokens, hk, d, dtype=dt, device="cuda") for _ in range(2)]
    st["out"] = torch.empty(tokens, h, d, dtype=dt, device="cuda")
    names = ("k_pool", "v_pool")
    for name in names:
        if case["fmt"] == "16bit":
            st[name] = _pool(case, pages, d, dt)
        else:
            st[name] = _pool(case, pages, d // 2, torch.uint8)
            st[name + "_scales"] = _pool(case, pages, d // 16, torch.uint8)
        for at in range(0, pages, 2048):   # the cached tokens, a slab of pages at a time
            part = st[name][at:at + 2048]
            x = torch.randn(part.shape[0], hk, p, d, generator=g, device="cuda", dtype=torch.float32)
            if case["fmt"] == "16bit":
                part.copy_(x)
            else:
                code, scale = _quantise(x)
                part.copy_(_pack(code))
                st[name + "_scales"][at:at + 2048].copy_(scale.view(torch.uint8))
    if own:
        from cutile_rs_b200 import api, launch, paged
        st["cache"] = paged.PagedKvCache(st["k_pool"], st["v_pool"], st.get("k_pool_scales"), st.get("v_pool_scales"))
        st["batch"] = paged.PagedBatch(st["table"], st["cu_q"], st["kv_lens"], st["max_q"])
        st["t"] = {n: api.from_torch(st[n]) for n in ("q", "k", "v", "inv_freq", "out") if n in st}
        if "rows" in st:
            st["t"]["rows"] = [api.from_torch(x) for x in st["rows"]]
        st["ws"] = launch.paged_attention_workspace(st["cache"], st["batch"], h)
    return st


def _places(st):
    """For every token its sequence, its position, and its page and slot in the pool."""
    p, cu = st["case"]["page"], st["cu_q"]
    t = torch.arange(st["q"].shape[0], device="cuda", dtype=torch.int32)
    seq = torch.bucketize(t, cu[1:], right=True)
    pos = st["kv_lens"][seq] - cu[1:][seq] + t
    return seq, pos, st["table"][seq, pos // p].long(), (pos % p).long()


def _rotate(x, cos, sin):
    lo, hi = x.float().chunk(2, -1)
    return torch.cat((lo * cos - hi * sin, hi * cos + lo * sin), -1)


def _append(st):
    _, pos, page, slot = _places(st)
    angle = pos.double().unsqueeze(-1) * st["inv_freq"].double()
    cos, sin = angle.cos().float().unsqueeze(1), angle.sin().float().unsqueeze(1)
    dt = st["q"].dtype
    q, k, v = _rotate(st["q"], cos, sin).to(dt), _rotate(st["k"], cos, sin), st["v"].float()
    if st["case"]["fmt"] == "16bit":
        st["k_pool"][page, :, slot] = k.to(dt)
        st["v_pool"][page, :, slot] = v.to(dt)
        return q, st["k_pool"], st["v_pool"]
    (kc, ks), (vc, vs) = _quantise(k), _quantise(v)
    st["k_pool"][page, :, slot], st["k_pool_scales"][page, :, slot] = _pack(kc), ks.view(torch.uint8)
    st["v_pool"][page, :, slot], st["v_pool_scales"][page, :, slot] = _pack(vc), vs.view(torch.uint8)
    k = _unpack(st["k_pool"][page, :, slot], st["k_pool_scales"][page, :, slot])
    v = _unpack(st["v_pool"][page, :, slot], st["v_pool_scales"][page, :, slot])
    return q, k.to(dt), v.to(dt)


def _dense(st, name):
    """The cached rows of every sequence, padded: [batch, kv head, position, value] in 32 bits."""
    pool = st[name][st["table"].long()]                                  # [batch, page, head, slot, value]
    x = pool.float() if st["case"]["fmt"] == "16bit" else _unpack(pool, st[name + "_scales"][st["table"].long()])
    return x.transpose(1, 2).flatten(2, 3)


def _attend(st):
    c = st["case"]
    h, hk, d, dt = c["heads"], c["kv_heads"], c["head_dim"], st["q"].dtype
    seq, pos, _, _ = _places(st)
    row = torch.arange(st["q"].shape[0], device="cuda") - st["cu_q"][seq]
    batch, width = st["table"].shape[0], st["max_q"]
    q = torch.zeros(batch, width, h, d, device="cuda")
    q[seq, row] = st["q"].float()
    q = q.unflatten(2, (hk, h // hk)).permute(0, 2, 1, 3, 4).flatten(2, 3)   # [batch, kv head, row x group, value]
    k, v = _dense(st, "k_pool"), _dense(st, "v_pool")
    s = (q @ k.transpose(2, 3)) * st["scale"]
    if c["softcap"]:
        s = c["softcap"] * torch.tanh(s / c["softcap"])
    where = torch.full((batch, width), -1, dtype=torch.int64, device="cuda")
    where[seq, row] = pos.long()
    key = torch.arange(k.shape[2], device="cuda")
    seen = key <= where.unsqueeze(-1)
    if c["window"]:
        seen &= key > where.unsqueeze(-1) - c["window"]
    seen = seen.repeat_interleave(h // hk, 1).unsqueeze(1)
    s = s.masked_fill(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(top.isfinite(), top, torch.zeros_like(top)))
    o = (e @ v) / e.sum(-1, keepdim=True)
    o = o.unflatten(2, (width, h // hk)).permute(0, 2, 1, 3, 4).flatten(2, 3)
    return o[seq, row].to(dt)


def run(state):
    c = state["case"]
    if own:
        from cutile_rs_b200 import launch
        t = state["t"]
        if c["op"] == "attend":
            launch.paged_attention(t["out"], t["q"], state["cache"], state["batch"], state["scale"],
                                   window=c["window"], softcap=c["softcap"], workspace=state["ws"])
            return state["out"]
        launch.paged_kv_append(state["cache"], state["batch"], t["k"], t["v"], q=t["q"], q_out=t["out"],
                               inv_freq=t["inv_freq"])
        if c["fmt"] == "16bit":
            return state["out"], state["k_pool"], state["v_pool"]
        launch.paged_kv_gather(t["rows"][0], t["rows"][1], state["cache"], state["batch"])
        return state["out"], state["rows"][0], state["rows"][1]
    return _append(state) if c["op"] == "append" else _attend(state)


def _pairs(case):
    """(query, key) pairs that the masks leave, and cached rows that at least one query sees."""
    pairs = rows = 0
    for n, kv in zip(*_lens(case)):
        first, w = kv - n, case["window"] or kv
        inside = min(max(0, w - first), n)                     # queries that see all keys up to their own
        pairs += inside * first + inside * (inside + 1) // 2 + (n - inside) * w
        rows += kv - max(0, first - w + 1)
    return pairs, rows


def work(case):
    d, h, hk = case["head_dim"], case["heads"], case["kv_heads"]
    tokens = sum(_lens(case)[0])
    row = d * 2 if case["fmt"] == "16bit" else d // 2 + d // 16   # bytes of one cached head vector
    if case["op"] == "append":
        moved = tokens * (2 * h * d * 2 + 2 * hk * d * 2 + 2 * hk * row)
        if case["fmt"] != "16bit":
            moved += tokens * 2 * hk * (row + d * 2)              # the rows read back
        return {"bytes": moved, "flops": 6 * tokens * (h + hk) * d}
    pairs, rows = _pairs(case)
    return {"bytes": 2 * tokens * h * d * 2 + 2 * rows * hk * row, "flops": 4 * d * h * pairs}


def _exact_quantised(x):
    """Values of the 4-bit blocks: the nearest e4m3 to amax / 6 and the nearest e2m1 to x / scale, ties to even."""
    grid = torch.arange(0, 127, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn).double()
    small = torch.tensor(_E2M1, dtype=torch.float64, device="cuda")

    def nearest(v, values):
        hi = torch.searchsorted(values, v).clamp(max=len(values) - 1)
        lo = (hi - 1).clamp(min=0)
        up, down = (values[hi] - v).abs(), (v - values[lo]).abs()
        return values[torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)]

    out = torch.empty_like(x)
    for j in range(0, x.shape[-1], 16):
        b = x[..., j:j + 16]
        s = nearest((b.abs().amax(-1, keepdim=True) / 6).contiguous(), grid)
        y = torch.where(s > 0, b.abs() / s, torch.zeros_like(b))
        out[..., j:j + 16] = torch.sign(b) * nearest(y, small) * s
    return out


def _exact_cached(st, name, b, n):
    """The first n cached rows of sequence b in 64 bits: [position, kv head, value]."""
    p = st["case"]["page"]
    pages = st["table"][b, :-(-n // p)].long()
    rows = st[name][pages].permute(0, 2, 1, 3).flatten(0, 1)[:n]
    if st["case"]["fmt"] == "16bit":
        return rows.double()
    code = torch.empty(*rows.shape[:-1], st["case"]["head_dim"], dtype=torch.int64, device="cuda")
    code[..., 0::2], code[..., 1::2] = (rows & 15).long(), (rows >> 4).long()
    value = torch.tensor(_E2M1, dtype=torch.float64, device="cuda")[code & 7] * (1.0 - 2.0 * (code >> 3))
    scale = st[name + "_scales"][pages].permute(0, 2, 1, 3).flatten(0, 1)[:n].contiguous()
    scale = scale.view(torch.float8_e4m3fn).double()
    return (value.unflatten(-1, (-1, 16)) * scale.unsqueeze(-1)).flatten(-2)


def exact(case, seed):
    st = prepare(case, seed)
    q_lens, kv_lens = _lens(case)
    h, hk, d, p = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    out = torch.empty(sum(q_lens), h, d, dtype=torch.float64, device="cuda")
    if case["op"] == "append":
        half = d // 2
        four = case["fmt"] != "16bit"
        pools = [torch.empty(sum(q_lens), hk, d, dtype=torch.float64, device="cuda") for _ in range(2)] if four else \
            [st["k_pool"].double(), st["v_pool"].double()]
        at = 0
        for b, (n, kv) in enumerate(zip(q_lens, kv_lens)):
            where = torch.arange(kv - n, kv, device="cuda")
            turn = torch.polar(torch.ones(n, half, dtype=torch.float64, device="cuda"),
                               where.double()[:, None] * st["inv_freq"].double()[None, :])[:, None, :]
            both = []
            for x in (st["q"][at:at + n], st["k"][at:at + n]):
                z = torch.complex(x[..., :half].double(), x[..., half:].double()) * turn
                both.append(torch.cat((z.real, z.imag), -1))
            out[at:at + n] = both[0]
            for pool, x in zip(pools, (both[1], st["v"][at:at + n].double())):
                if four:
                    pool[at:at + n] = _exact_quantised(x)
                else:
                    pool[st["table"][b, where // p].long(), :, where % p] = x
            at += n
        return out, pools[0], pools[1]
    if max(kv_lens) * sum(q_lens) * h > 6e9:
        return None
    at = 0
    for b, (n, kv) in enumerate(zip(q_lens, kv_lens)):
        k, v = _exact_cached(st, "k_pool", b, kv), _exact_cached(st, "v_pool", b, kv)
        where = torch.arange(kv - n, kv, device="cuda")[:, None]
        key = torch.arange(kv, device="cuda")[None, :]
        hidden = key > where
        if case["window"]:
            hidden = hidden | (where - key >= case["window"])
        for j in range(h):
            s = st["q"][at:at + n, j].double() @ k[:, j * hk // h].T / math.sqrt(d)
            if case["softcap"]:
                s = torch.tanh(s / case["softcap"]) * case["softcap"]
            w = torch.softmax(s.masked_fill(hidden, -math.inf), -1)
            out[at:at + n, j] = w @ v[:, j * hk // h]
        at += n
    return out
