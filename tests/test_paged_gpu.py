"""Paged key/value cache: append with rotation, attention and read-back, against 64-bit plain forms.

Pages are shuffled, the block table holds junk behind every sequence's pages, and slots that no sequence owns hold NaN
patterns: nothing of either may show in a result."""
import ctypes

import pytest
import torch

import paged_reference as ref
from cutile_rs_b200 import _lib, api, launch, paged
from cutile_rs_b200.tensor import KernelLaunchError

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16
SENTINEL = -77.0


def _status(b200):
    st = _lib.StatusC()
    rc = b200.b200tile_status(torch.cuda.current_stream().cuda_stream, ctypes.byref(st))
    return (st.code, st.site, st.aux) if rc in (_lib.OK, _lib.ERR_DEVICE) else (-rc, 0, 0)


def _attend(p, scale, **kw):
    out = torch.full((p.tokens, p.heads, p.d), SENTINEL, dtype=p.dtype, device="cuda")
    launch.paged_attention(api.from_torch(out), api.from_torch(p.q), p.cache, p.batch, scale, **kw)
    return out


def _check(p, scale, **kw):
    p.poison()
    got = _attend(p, scale, **kw)
    want, tol = ref.attention(p, scale, **kw)
    n = p.cu[-1]
    assert not torch.isnan(got).any()
    bad = (got[:n].double() - want[:n]).abs() > tol[:n]
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()}, worst {float(((got[:n].double() - want[:n]).abs() / tol[:n].clamp(min=1e-9)).max()):.2f} bounds"
    assert (got[n:] == SENTINEL).all()
    return got


FORMS = [("16bit", "hnd"), ("16bit", "nhd"), ("nvfp4", "hnd"), ("nvfp4", "nhd")]


@pytest.mark.parametrize("fmt,layout", FORMS)
@pytest.mark.parametrize("d,heads,kvh,page,dtype", [
    (128, 8, 2, 16, BF16), (64, 6, 2, 32, F16), (128, 4, 4, 64, F16), (64, 16, 1, 16, BF16), (128, 14, 2, 128, BF16),
])
def test_decode_lengths(b200, fmt, layout, d, heads, kvh, page, dtype):
    """One token per sequence, lengths from one to several hundred, on both sides of step and page ends; one sequence
    without tokens, one whose length is 0, rows behind the last sequence."""
    kv = [1, 2, 15, 16, 17, 31, 100, 128, 129, 0, 333, 700]
    q = [1] * 12
    q[6] = 0
    p = ref.Problem(q, kv, heads, kvh, d, page, dtype, fmt, layout, seed=d + heads, pad_tokens=3)
    got = _check(p, d ** -0.5)
    assert (got[p.cu[9]:p.cu[10]] == 0).all()          # the sequence of length 0
    assert _status(b200)[0] == 0


@pytest.mark.parametrize("keys", [0, ref.MANY_KEYS])
@pytest.mark.parametrize("fmt", ["16bit", "nvfp4"])
@pytest.mark.parametrize("causal,window,softcap", [(True, 0, 30.0), (True, 1, 0.0), (True, 33, 0.0), (True, 100, 5.0),
                                                   (False, 0, 0.0), (False, 0, 20.0)])
def test_masks_and_cap(b200, fmt, causal, window, softcap, keys):
    """Several tokens per sequence: causal edges inside a block of rows, windows, caps; a sequence shorter than its
    tokens, whose first rows see nothing."""
    p = ref.Problem([3, 5, 1, 4, 2], [3, 260, 77, 2, 130], 6, 2, 64, 16, F16, fmt, seed=window + 1, table_keys=keys)
    got = _check(p, 0.3, causal=causal, window=window, softcap=softcap)
    if causal:
        assert (got[p.cu[3]:p.cu[3] + 2] == 0).all()   # positions -2 and -1


@pytest.mark.parametrize("keys", [0, ref.MANY_KEYS])
@pytest.mark.parametrize("fmt,d,dtype", [("16bit", 128, BF16), ("16bit", 64, F16), ("nvfp4", 128, F16), ("nvfp4", 64, BF16)])
@pytest.mark.parametrize("heads,kvh,page,window,softcap", [(8, 2, 16, 0, 0.0), (6, 2, 128, 150, 25.0), (7, 1, 32, 0, 50.0),
                                                           (2, 2, 64, 40, 0.0)])
def test_prompt_chunks(b200, fmt, d, dtype, heads, kvh, page, window, softcap, keys):
    """Prompts and chunks behind cached prefixes in one call with decode steps."""
    p = ref.Problem([150, 1, 300, 64, 0, 17], [150, 200, 555, 70, 40, 400], heads, kvh, d, page, dtype, fmt,
                    seed=heads + page, pad_tokens=5, table_keys=keys)
    _check(p, d ** -0.5, window=window, softcap=softcap)
    assert _status(b200)[0] == 0


@pytest.mark.parametrize("keys", [0, ref.MANY_KEYS])
@pytest.mark.parametrize("fmt,d,dtype", [("16bit", 128, F16), ("16bit", 64, BF16), ("nvfp4", 128, BF16), ("nvfp4", 64, F16)])
@pytest.mark.parametrize("heads,kvh,page,causal,window,softcap", [(8, 1, 64, True, 0, 0.0), (4, 4, 256, True, 700, 0.0),
                                                                  (10, 2, 16, True, 130, 30.0), (4, 1, 32, False, 0, 0.0),
                                                                  (4, 2, 128, False, 0, 40.0)])
def test_long_prompts(b200, fmt, d, dtype, heads, kvh, page, causal, window, softcap, keys):
    """Several tiles per sequence, ends inside tiles, pages and steps, whole steps before the window, a first step in
    which early rows see nothing yet; a sequence shorter than its tokens."""
    p = ref.Problem([1000, 129, 257, 90], [1500, 129, 2999, 33], heads, kvh, d, page, dtype, fmt, "nhd" if page == 64 else "hnd",
                    seed=heads + page, table_keys=keys)
    got = _check(p, d ** -0.5, causal=causal, window=window, softcap=softcap)
    if causal:
        assert (got[p.cu[3]:p.cu[3] + 57] == 0).all()
    assert _status(b200)[0] == 0


def test_long_prompts_with_very_negative_scores(b200):
    """Windows whose first step is empty for late rows, with scores far below zero: the reference of the running
    exponent must come from keys that are seen."""
    for fmt in ("16bit", "nvfp4"):
        p = ref.Problem([400], [900], 2, 1, 128, 16, BF16, fmt, seed=30, table_keys=ref.MANY_KEYS)
        p.q.copy_(p.q.abs())
        if fmt == "16bit":
            p.pools[0].copy_(-p.pools[0].abs())
        else:
            p.pools[0].bitwise_or_(0x88)
        _check(p, 5.0, window=100)


def test_long_context_is_split(b200):
    """A few long sequences: every item is cut over many workers and merged."""
    for fmt in ("16bit", "nvfp4"):
        p = ref.Problem([1, 1], [20011, 5003], 8, 2, 128, 64, BF16, fmt, seed=5)
        a = _check(p, 128 ** -0.5)
        b = _attend(p, 128 ** -0.5)
        assert torch.equal(a, b)                        # no order that changes from run to run


def test_many_sequences(b200):
    """More sequences than a CTA has threads, most of them short."""
    kv = [1 + (37 * i) % 90 for i in range(700)]
    p = ref.Problem([1] * 700, kv, 4, 2, 64, 16, BF16, seed=9)
    _check(p, 0.125)
    p = ref.Problem([(i * 7) % 3 for i in range(700)], kv, 2, 1, 64, 16, F16, "nvfp4", seed=10)
    _check(p, 0.125)


@pytest.mark.parametrize("fmt,d", [("16bit", 128), ("16bit", 64), ("nvfp4", 128), ("nvfp4", 64)])
@pytest.mark.parametrize("window,softcap", [(0, 0.0), (70, 20.0)])
def test_many_steps_and_a_prompt(b200, fmt, d, window, softcap):
    """So many decode steps beside the prompts that each kernel takes its own sequences; call after call, which run into
    one another, with one workspace."""
    q_lens = [1] * 150 + [130, 0, 40, 3]
    kv_lens = [1 + (53 * i) % 400 for i in range(150)] + [300, 20, 40, 500]
    p = ref.Problem(q_lens, kv_lens, 8, 2, d, 16, BF16, fmt, seed=d, table_keys=ref.MANY_KEYS, pad_tokens=3)
    got = _check(p, d ** -0.5, window=window, softcap=softcap)
    ws = launch.paged_attention_workspace(p.cache, p.batch, 8)
    outs = [torch.full_like(p.q, SENTINEL) for _ in range(10)]
    for o in outs:
        launch.paged_attention(api.from_torch(o), api.from_torch(p.q), p.cache, p.batch, d ** -0.5, window=window,
                               softcap=softcap, workspace=ws)
    assert all(torch.equal(got, o) for o in outs)
    assert _status(b200)[0] == 0


def test_large_scores_and_infinities(b200):
    """Scores of a few thousand stay finite; an infinite key takes the whole row, the other rows keep theirs."""
    p = ref.Problem([1, 1], [90, 90], 4, 2, 128, 16, F16, seed=3)
    p.q.mul_(30)
    _check(p, 1.0)
    lone = int(p.table[0, 2])
    p.pools[0][lone, 0, 5, 0] = float("inf")
    p.q[0, :2, 0] = 0.5                                 # score +inf for the heads of K/V head 0
    got = _attend(p, 1.0)
    assert torch.isnan(got[0, :2]).all() and not torch.isnan(got[0, 2:]).any() and not torch.isnan(got[1]).any()


def test_small_queries_over_fp4(b200):
    """Query rows far below 1 and far above keep their precision over an NVFP4 cache."""
    for unit in (2.0 ** -30, 2.0 ** 14):
        p = ref.Problem([1, 2], [50, 300], 4, 2, 128, 16, BF16, "nvfp4", seed=4)
        p.q.mul_(unit)
        _check(p, 128 ** -0.5 / unit)


def test_global_factors_and_wide_scales(b200):
    p = ref.Problem([1, 3], [70, 41], 4, 2, 64, 16, F16, "nvfp4", seed=6, k_global=0.01, v_global=40.0)
    _check(p, 0.125)
    p.scales[1].copy_(torch.randint(1, 0x7f, p.scales[1].shape, device="cuda").to(torch.uint8))   # 2^-9 .. 448
    p = ref.Problem([1, 3], [70, 41], 4, 2, 64, 16, BF16, "nvfp4", seed=7)
    p.scales[1].copy_(torch.randint(1, 0x7f, p.scales[1].shape, device="cuda").to(torch.uint8))
    _check(p, 0.125)


def test_strided_rows(b200):
    """q inside a fused projection's rows, out inside a wider buffer, heads in reverse memory order of tokens."""
    for q_lens, kv_lens in (([1, 1, 2], [30, 200, 64]), ([130, 1, 40], [130, 50, 90])):
        p = ref.Problem(q_lens, kv_lens, 4, 2, 128, 16, BF16, seed=8, table_keys=ref.MANY_KEYS)
        p.poison()
        wide = torch.zeros(p.tokens, 8, 130, dtype=BF16, device="cuda")
        qv = wide[:, 2:6, :128]
        qv.copy_(p.q)
        ow = torch.full((4, p.tokens, 130), SENTINEL, dtype=BF16, device="cuda")
        ov = ow.permute(1, 0, 2)[:, :, :128]
        launch.paged_attention(api.from_torch(ov), api.from_torch(qv), p.cache, p.batch, 0.1)
        want, tol = ref.attention(p, 0.1)
        assert ((ov.double() - want).abs() <= tol).all()
        assert (ow[:, :, 128:] == SENTINEL).all()


@pytest.mark.parametrize("keys", [0, ref.MANY_KEYS])
@pytest.mark.parametrize("fmt,d,dtype", [("16bit", 128, BF16), ("16bit", 64, F16), ("nvfp4", 128, BF16), ("nvfp4", 64, F16)])
def test_caps_near_and_far_from_the_scores(b200, fmt, d, dtype, keys):
    """Scores that are a small part of the cap, about its size, and far beyond it, in one call: the capped score has one
    form for small arguments and one for all."""
    for cap in (1.0, 4.0, 300.0):
        p = ref.Problem([200, 3, 90], [260, 40, 90], 6, 2, d, 16, dtype, fmt, seed=40, table_keys=keys)
        p.q[:70].mul_(6)
        _check(p, d ** -0.5, softcap=cap)
        _check(p, d ** -0.5, softcap=cap, window=50)


@pytest.mark.parametrize("unit", [2.0 ** -30, 2.0 ** 13])
def test_prompts_of_small_and_large_queries_over_fp4(b200, unit):
    for softcap in (0.0, 20.0):
        p = ref.Problem([150, 20], [300, 33], 4, 2, 128, 16, BF16, "nvfp4", seed=41, table_keys=ref.MANY_KEYS)
        p.q[::3].mul_(2.0 ** -9)                        # rows of very different size in one tile
        p.q.mul_(unit)
        _check(p, 128 ** -0.5 / unit, softcap=softcap)


def test_many_heads_per_kv_head(b200):
    """More heads per K/V head than a tile has rows: row blocks take the prompt."""
    p = ref.Problem([3, 2], [40, 90], 260, 2, 64, 16, BF16, seed=42)
    _check(p, 0.125)
    p = ref.Problem([9, 1], [40, 90], 128, 1, 64, 16, F16, "nvfp4", seed=42, table_keys=ref.MANY_KEYS)
    _check(p, 0.125)


def test_decode_runs_and_clusters_agree(b200):
    """The same sequences behind a short block table (a cluster per item) and a long one (runs of the whole line)."""
    for fmt in ("16bit", "nvfp4"):
        for q_len in (1, 3):
            p = ref.Problem([q_len] * 3, [700, 300, 45], 8, 2, 128, 16, F16, fmt, seed=43)
            a = _check(p, 0.1)
            wide = torch.full((3, 6000), -1, dtype=torch.int32, device="cuda")
            wide[:, :p.table.shape[1]] = p.table
            p.table = wide
            p.batch = paged.PagedBatch(wide, p.cu_q, p.kv, q_len)
            b = _check(p, 0.1)
            assert (a.double() - b.double()).abs().max() <= 2.0 ** -9


def test_workspace_contents_do_not_matter(b200):
    for q_lens, kv_lens in (([1, 1], [30000, 17000]), ([100, 1], [5000, 600])):
        for fmt in ("16bit", "nvfp4"):
            p = ref.Problem(q_lens, kv_lens, 4, 2, 64, 64, BF16, fmt, seed=44, table_keys=ref.MANY_KEYS)
            ws = launch.paged_attention_workspace(p.cache, p.batch, 4)
            a = _attend(p, 0.1, workspace=ws)
            ws.fill_(255)                               # NaN everywhere, -1 in every descriptor
            assert torch.equal(a, _attend(p, 0.1, workspace=ws))
            ws.random_(0, 256)
            assert torch.equal(a, _attend(p, 0.1, workspace=ws))


def test_output_may_be_the_query_tensor(b200):
    for q_lens in ([1, 1, 2], [130, 1, 70]):
        p = ref.Problem(q_lens, [700, 40, 300], 4, 2, 128, 16, BF16, seed=45, table_keys=ref.MANY_KEYS)
        want = _attend(p, 0.1)
        t = api.from_torch(p.q.clone())
        launch.paged_attention(t, t, p.cache, p.batch, 0.1)
        assert torch.equal(want, t.storage)


def test_sequences_that_share_pages(b200):
    """A common prefix in common pages, read by all."""
    for fmt in ("16bit", "nvfp4"):
        p = ref.Problem([1, 1, 80], [200, 220, 240], 4, 2, 64, 16, F16, fmt, seed=46, table_keys=ref.MANY_KEYS)
        p.table[1:, :9] = p.table[0, :9]
        got = _attend(p, 0.2)
        want, tol = ref.attention(p, 0.2)
        assert ((got.double() - want).abs() <= tol).all()


def test_lengths_and_ranges_that_do_not_fit(b200):
    """Lengths beyond the block table, negative ones, token ranges beyond the tensors: what fits is computed, nothing else
    is touched."""
    for fmt in ("16bit", "nvfp4"):
        for q_lens in ([1, 1, 1], [100, 1, 90]):
            p = ref.Problem(q_lens, [150, 60, 120], 4, 2, 64, 16, BF16, fmt, seed=47,
                            table_keys=4096 if q_lens[0] > 1 else 0)   # the tile kernel / row blocks
            cap = p.table.shape[1] * 16
            p.table.clamp_(min=0)                       # every entry a page: positions up to the table's end exist
            p.kv[0] = cap + 37                          # keys behind the table are left out, positions keep counting
            got = _attend(p, 0.2)
            n = q_lens[0]
            k, v = p.rows(0, cap)
            pos = torch.arange(cap + 37 - n, cap + 37, device="cuda")[:, None]
            seen = torch.arange(cap, device="cuda")[None] <= pos
            s = (p.q[:n, 0].double() @ k[:, 0].T * 0.2).masked_fill(~seen, float("-inf"))
            want = torch.softmax(s, -1) @ v[:, 0]
            assert ((got[:n, 0].double() - want).abs() <= 2.0 ** -6).all()
            before = [x.clone() for x in p.pools]
            p.kv[1] = -5
            p.cu_q[3] = p.tokens + 1000                 # the last sequence's range reaches behind the tensors
            got = _attend(p, 0.2)
            assert (got[p.cu[1]:p.cu[2]] == 0).all() and not torch.isnan(got).any()
            p.kv[0] = cap + n                           # positions cap .. cap + n - 1: all behind the table
            p.cu_q[3] = p.tokens
            p.kv[2] = 0
            launch.paged_kv_append(p.cache, p.batch, api.from_torch(p.k), api.from_torch(p.v))
            assert all(torch.equal(a, b) for a, b in zip(before, p.pools))
    assert _status(b200)[0] == 0


@pytest.mark.parametrize("keys", [0, ref.MANY_KEYS])
def test_windows_longer_than_anything(b200, keys):
    """No window at all, whatever its size, also for a sequence shorter than its tokens."""
    for fmt in ("16bit", "nvfp4"):
        p = ref.Problem([60, 2, 40], [50, 1, 700], 4, 2, 64, 16, BF16, fmt, seed=51, table_keys=keys)
        want = _check(p, 0.2)
        for window in (701, 0x7ffffffe, 0x7fffffff, 1 << 40):
            assert torch.equal(want, _attend(p, 0.2, window=window))


@pytest.mark.parametrize("keys", [0, ref.MANY_KEYS])
def test_pages_outside_the_pool_in_prompts(b200, keys):
    """As for single tokens: zeros in their place, the sequence named in the status record."""
    for fmt in ("16bit", "nvfp4"):
        for bad in (-1, 1 << 20, -(1 << 31)):
            p = ref.Problem([40, 120], [40, 700], 4, 2, 64, 16, BF16, fmt, seed=52, table_keys=keys)
            p.table[1, 20] = bad
            got = _attend(p, 0.2)
            assert _status(b200)[:2] == (4, 1)
            _lib.check(b200.b200tile_status_reset(torch.cuda.current_stream().cuda_stream))
            for x in p.pools:
                x[p.free[0]] = 0
            p.table[1, 20] = int(p.free[0])
            assert torch.equal(got, _attend(p, 0.2))


@pytest.mark.parametrize("keys", [0, 8192])
def test_lengths_up_to_the_largest_integer(b200, keys):
    """Lengths and token ranges that no cache has: nothing outside the tensors is touched, nothing hangs."""
    for fmt in ("16bit", "nvfp4"):
        p = ref.Problem([40, 120], [40, 700], 4, 2, 64, 16, BF16, fmt, seed=53, table_keys=keys)
        p.table.clamp_(min=0)
        want = _attend(p, 0.2)
        for kv, cu, window in ((0x7fffffff, 40, 0), (-(1 << 31), 40, 100), (700, -(1 << 31), 0), (700, 0x7fffffff, 33)):
            p.kv[0], p.cu_q[0], p.cu_q[1] = kv, min(cu, 0), cu
            _attend(p, 0.2, window=window)
        p.kv[0], p.cu_q[0], p.cu_q[1] = 40, 0, 40
        assert torch.equal(want, _attend(p, 0.2))


def test_no_more_than_max_q_len_tokens(b200):
    p = ref.Problem([5, 2], [50, 60], 4, 2, 64, 16, BF16, seed=48, max_q=3)
    got = _attend(p, 0.2)
    want, tol = ref.attention(p, 0.2)
    rows = [0, 1, 2, 5, 6]
    assert ((got[rows].double() - want[rows]).abs() <= tol[rows]).all()
    assert (got[3:5] == SENTINEL).all()


def test_pools_beyond_four_gigabytes(b200):
    """Pages whose offsets pass 2^32 bytes and 2^31 elements, in both formats and both kernels, and append and gather on
    them."""
    g = torch.Generator(device="cuda").manual_seed(49)
    for fmt in ("16bit", "nvfp4"):
        d, kvh, page = 128, 8, 64
        row = d if fmt == "16bit" else d // 2
        per = kvh * page * row
        pages = (1 << 31) // per + 40 if fmt == "16bit" else (1 << 32) // per + 40
        dt = BF16 if fmt == "16bit" else torch.uint8
        pools = [torch.empty(pages, kvh, page, row, dtype=dt, device="cuda") for _ in range(2)]
        scales = [torch.empty(pages, kvh, page, d // 16, dtype=torch.uint8, device="cuda") for _ in range(2)] if fmt != "16bit" \
            else [None, None]
        p = ref.Problem([1, 100], [300, 200], 16, kvh, d, page, BF16, fmt, seed=50, table_keys=ref.MANY_KEYS)
        used = torch.arange(pages - 9, pages, device="cuda")
        for big, small, bs, ss in zip(pools, p.pools, scales, p.scales):
            big[used] = small[:9]
            if ss is not None:
                bs[used] = ss[:9]
        p.table[0, :5], p.table[1, :4] = used[:5].int(), used[5:].int()
        p.pools, p.scales, p.pages = pools, scales, pages
        p.cache = paged.PagedKvCache(*pools, *scales)
        launch.paged_kv_append(p.cache, p.batch, api.from_torch(p.k), api.from_torch(p.v))
        out = [torch.empty_like(p.k) for _ in range(2)]
        launch.paged_kv_gather(api.from_torch(out[0]), api.from_torch(out[1]), p.cache, p.batch)
        for b, n in enumerate(p.q_lens):
            for got, want in zip(out, p.rows(b, p.kv_lens[b])):
                assert torch.equal(got[p.cu[b]:p.cu[b + 1]].double(), want[-n:])
        if fmt == "16bit":
            assert torch.equal(out[0], p.k)
        want, tol = ref.attention(p, 0.1)
        for width in (p.table.shape[1], 6):              # tiles, row blocks
            p.batch = paged.PagedBatch(p.table[:, :width], p.cu_q, p.kv, 100)
            assert ((_attend(p, 0.1).double() - want).abs() <= tol).all()
        del pools, scales, p, out
        torch.cuda.empty_cache()


# ---- append ------------------------------------------------------------------------------------------------------
def _inv_freq(r, base=500000.0):
    i = torch.arange(0, r, 2, dtype=torch.float64, device="cuda")
    return (base ** (-i / r)).float()


def _append_case(p, rot, with_q=True, in_place=False):
    f = _inv_freq(rot) if rot else None
    q_in, k_in, v_in = p.q.clone(), p.k.clone(), p.v.clone()
    before = [x.clone() for x in p.pools + [s for s in p.scales if s is not None]]
    q_out = p.q if in_place else torch.full_like(p.q, SENTINEL)
    kw = dict(q=api.from_torch(p.q), q_out=api.from_torch(q_out)) if with_q else {}
    launch.paged_kv_append(p.cache, p.batch, api.from_torch(p.k), api.from_torch(p.v),
                           inv_freq=api.from_torch(f) if rot else None, **kw)
    return f if rot else torch.empty(0, device="cuda"), q_in, k_in, v_in, before, q_out


@pytest.mark.parametrize("fmt,layout", FORMS)
@pytest.mark.parametrize("d,rot,dtype,heads,kvh,page", [(128, 128, BF16, 8, 2, 16), (64, 64, F16, 3, 3, 32),
                                                        (128, 64, F16, 5, 1, 64), (64, 0, BF16, 4, 2, 16),
                                                        (128, 32, BF16, 32, 8, 128)])
def test_append(b200, fmt, layout, d, rot, dtype, heads, kvh, page):
    q_lens, kv_lens = [1, 7, 0, 33, 1, 3], [131071 // 4, 7, 20, 100, 1, 2]   # the last: one token before position 0
    p = ref.Problem(q_lens, kv_lens, heads, kvh, d, page, dtype, fmt, layout, seed=d + rot, pad_tokens=4)
    f, q, k, v, before, q_out = _append_case(p, rot)
    eps = torch.finfo(dtype).eps
    touched = torch.zeros(p.pages, page, dtype=torch.bool, device="cuda")
    for b, (n, kv) in enumerate(zip(q_lens, kv_lens)):
        if n == 0:
            continue
        lo, hi = p.cu[b], p.cu[b + 1]
        pos = torch.arange(kv - n, kv, device="cuda")
        # one rounding of the result, 32-bit cos, sin and products before it
        want = ref.rotate(q[lo:hi], pos, f)
        room = eps / 2 * want.abs() + 2.0 ** -21 * q[lo:hi].double().abs().amax()
        assert ((q_out[lo:hi].double() - want).abs() <= room).all()
        first = max(0, -(kv - n))
        at = pos[first:]
        pg, slot = p.table[b, at // page].long(), at % page
        touched[pg, slot] = True
        for i, x in ((0, ref.rotate(k[lo:hi], pos, f)[first:]), (1, v[lo:hi].double()[first:])):
            rows = p.pools[i].permute(0, 2, 1, 3)[pg, slot]
            if fmt == "16bit":
                room = eps / 2 * x.abs() + 2.0 ** -21 * x.abs().amax() if (i == 0 and rot and x.numel()) else torch.zeros_like(x)
                assert ((rows.double() - x).abs() <= room).all()
            else:
                got = ref.dequant(rows, p.scales[i].permute(0, 2, 1, 3)[pg, slot])
                value, scale, margin = ref.quantise(x)
                off = (got - value).abs() > 1e-12
                # a rotated value within 32-bit rounding of a border may take either side
                assert not (off & (margin > (2.0 ** -18 if i == 0 and rot else 0.0))).any()
                assert (off.double() * (got - value).abs() <= 2.01 * scale).all()
    assert (q_out[p.cu[-1]:] == SENTINEL).all()
    for old, new in zip(before, p.pools + [s for s in p.scales if s is not None]):
        a, c = old.permute(0, 2, 1, 3)[~touched], new.permute(0, 2, 1, 3)[~touched]
        assert torch.equal(a.view(torch.uint8), c.view(torch.uint8))
    assert _status(b200)[0] == 0


@pytest.mark.parametrize("fmt", ["16bit", "nvfp4"])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_append_rounds_as_the_formula_in_32_bits(b200, fmt, dtype):
    """Angles in 64 bits, cosine and sine rounded to 32, then two products and a sum, each rounded: the same bits."""
    p = ref.Problem([700, 1, 300], [700, 90000, 20300], 8, 2, 128, 64, dtype, fmt, seed=54)
    f, q, k, v, _, q_out = _append_case(p, 128)
    pos = torch.cat([torch.arange(kv - n, kv, device="cuda") for n, kv in zip(p.q_lens, p.kv_lens)])
    angle = pos.double()[:, None] * f.double()[None]
    c, s = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def turned(x):
        lo, hi = x[..., :64].float(), x[..., 64:].float()
        return torch.cat((lo * c - hi * s, hi * c + lo * s), -1)

    assert torch.equal(q_out, turned(q).to(dtype))
    at = 0
    for b, n in enumerate(p.q_lens):
        want = turned(k)[at:at + n]
        got = p.rows(b, p.kv_lens[b])[0][-n:]
        if fmt == "16bit":
            assert torch.equal(got, want.to(dtype).double())
        else:
            assert torch.equal(got, ref.quantise(want.double())[0])
        at += n


def test_append_without_q_and_in_place(b200):
    p = ref.Problem([5, 1], [40, 9], 4, 2, 128, 16, BF16, seed=1)
    f, q, k, v, _, q_out = _append_case(p, 128, in_place=True)
    want = ref.rotate(q, torch.tensor([35, 36, 37, 38, 39, 8], device="cuda"), f)
    assert ((p.q.double() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-5).all()
    once = [x.clone() for x in p.pools]
    _append_case(p, 128, with_q=False)
    assert all(torch.equal(a, b) for a, b in zip(once, p.pools))


def test_append_large_and_special_values_fp4(b200):
    """Blocks beyond 6 * 448, of zeros, of one value, below the smallest scale, and with infinities."""
    p = ref.Problem([6], [6], 2, 1, 64, 16, BF16, "nvfp4", seed=2)
    p.v[0] = 0.0
    p.v[1] = 1e6
    p.v[2] = 2.0 ** -20
    p.v[3, :, ::2] = 0.0
    p.v[3, :, 1::2] = -3.0
    p.v[4, :, 3] = float("inf")
    launch.paged_kv_append(p.cache, p.batch, api.from_torch(p.k), api.from_torch(p.v))
    k, v = p.rows(0, 6)
    assert (v[0] == 0).all() and (v[1] == 2688).all() and (v[2] == 0).all()
    assert torch.equal(v[3], p.v[3].double())           # scale 0.5 exactly
    assert v[4, 0, 3] == 2688 and torch.isfinite(v).all()


def test_append_of_extreme_values_with_extreme_factors_fp4(b200):
    """Quotients beyond 32 bits keep their sign and saturate; those below the smallest scale are zeros."""
    for glob in (2.0 ** -21, 2.0 ** 17):
        p = ref.Problem([5], [5], 2, 1, 64, 16, BF16, "nvfp4", seed=3, k_global=glob, v_global=glob)
        for i, unit in enumerate((2.0 ** 127, 2.0 ** 99, 2.0 ** 90, 2.0 ** 89, 2.0 ** -110)):
            p.v[i] = unit
            p.v[i, :, ::2] = -unit
        launch.paged_kv_append(p.cache, p.batch, api.from_torch(p.k), api.from_torch(p.v))
        k, v = p.rows(0, 5)
        assert torch.equal(v[:4], torch.sign(p.v[:4].double()) * 2688 * glob) and (v[4] == 0).all()


def test_gather_returns_what_append_wrote(b200):
    for fmt, dtype in (("16bit", BF16), ("16bit", F16), ("nvfp4", BF16), ("nvfp4", F16)):
        for d in (64, 128):
            p = ref.Problem([50, 17, 1], [50, 17, 1], 4, 2, d, 16, dtype, fmt, seed=d, pad_tokens=2)
            launch.paged_kv_append(p.cache, p.batch, api.from_torch(p.k), api.from_torch(p.v))
            p.poison()
            out = [torch.full_like(p.k, SENTINEL) for _ in range(2)]
            launch.paged_kv_gather(api.from_torch(out[0]), api.from_torch(out[1]), p.cache, p.batch)
            for b in range(3):
                for got, want in zip(out, p.rows(b, p.kv_lens[b])):
                    assert torch.equal(got[p.cu[b]:p.cu[b + 1]].double(), want)   # products of e2m1 and e4m3 are exact
            assert all((x[p.cu[-1]:] == SENTINEL).all() for x in out)
            if fmt == "16bit":
                assert torch.equal(out[0][:p.cu[-1]], p.k[:p.cu[-1]])


# ---- together, and around the calls ------------------------------------------------------------------------------
@pytest.mark.parametrize("fmt", ["16bit", "nvfp4"])
def test_prompt_then_steps(b200, fmt):
    """A prompt and a few decode steps as a server runs them: append, attend, append, attend; each against the 64-bit
    form over the cache as it stands, and the prompt also against dense attention over the rows read back."""
    d, heads, kvh, page = 128, 8, 2, 16
    lens = [70, 33, 1]
    p = ref.Problem([0, 0, 0], [96, 64, 32], heads, kvh, d, page, BF16, fmt, seed=11)   # pages for what is to come
    f = api.from_torch(_inv_freq(d))
    g = torch.Generator(device="cuda").manual_seed(1)
    for step in range(4):
        new = lens if step == 0 else [1, 1, 1]
        total = [n + step for n in lens]
        cu = [0, new[0], new[0] + new[1], sum(new)]
        p.q_lens, p.kv_lens, p.cu, p.tokens = new, total, cu, cu[-1]
        p.cu_q.copy_(torch.tensor(cu))
        p.kv.copy_(torch.tensor(total))
        batch = paged.PagedBatch(p.table, p.cu_q, p.kv, max(new))
        x = torch.randn(p.tokens, heads + 2 * kvh, d, generator=g, device="cuda").to(BF16)
        p.q = torch.empty(p.tokens, heads, d, dtype=BF16, device="cuda")
        launch.paged_kv_append(p.cache, batch, api.from_torch(x[:, heads:heads + kvh]), api.from_torch(x[:, heads + kvh:]),
                               q=api.from_torch(x[:, :heads]), q_out=api.from_torch(p.q), inv_freq=f)
        out = torch.empty_like(p.q)
        launch.paged_attention(api.from_torch(out), api.from_torch(p.q), p.cache, batch, d ** -0.5)
        want, tol = ref.attention(p, d ** -0.5)
        assert ((out.double() - want).abs() <= tol).all(), step
    # the first sequence's rows, read back, through the dense kernel: the last token's output again
    n = total[0]
    rows = [torch.empty(n, kvh, d, dtype=BF16, device="cuda") for _ in range(2)]
    whole = paged.PagedBatch(p.table[:1], torch.tensor([0, n], dtype=torch.int32, device="cuda"), p.kv[:1], n)
    launch.paged_kv_gather(api.from_torch(rows[0]), api.from_torch(rows[1]), p.cache, whole)
    kt, vt = (r.permute(1, 0, 2).contiguous() for r in rows)
    dense = torch.empty(1, heads, d, dtype=BF16, device="cuda")
    st = (ctypes.c_int64 * 2)
    _lib.check(b200.b200tile_fmha_fwd(b"bf16", p.q.data_ptr(), kt.data_ptr(), vt.data_ptr(), dense.data_ptr(), 1, heads,
                                      kvh, 1, n, d, st(d, heads * d), st(n * d, d), st(n * d, d), st(d, heads * d),
                                      d ** -0.5, 1, n - 1, torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    assert ((dense[0].double() - want[0]).abs() <= tol[0] + 2.0 ** -7).all()


def test_graph_replay_with_other_lengths_on_another_stream(b200):
    p = ref.Problem([1, 1, 1], [600, 50, 300], 8, 2, 128, 16, F16, seed=12)
    out = torch.zeros(3, 8, 128, dtype=F16, device="cuda")
    qo = torch.zeros_like(out)
    args = [api.from_torch(x) for x in (p.k, p.v, p.q, qo, _inv_freq(128), out)]
    s = torch.cuda.Stream()
    ws = launch.paged_attention_workspace(p.cache, p.batch, 8)
    torch.cuda.synchronize()

    def step():
        launch.paged_kv_append(p.cache, p.batch, args[0], args[1], q=args[2], q_out=args[3], inv_freq=args[4], stream=s)
        launch.paged_attention(args[5], args[3], p.cache, p.batch, 0.1, workspace=ws, stream=s)

    step()                                               # function attributes are set outside the capture
    s.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        step()
    for lens in ([600, 50, 300], [17, 50, 1], [599, 33, 256]):
        p.kv.copy_(torch.tensor(lens))
        p.kv_lens = lens
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        q, p.q = p.q, qo
        want, tol = ref.attention(p, 0.1)
        p.q = q
        assert ((out.double() - want).abs() <= tol).all(), lens


def test_two_calls_at_once(b200):
    """Two streams, a workspace each."""
    ps = [ref.Problem([1] * 9, [700 + 13 * i for i in range(9)], 8, 2, 128, 32, BF16, f, seed=20) for f in ("16bit", "nvfp4")]
    alone = [_attend(p, 0.1) for p in ps]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ps]
    outs = [torch.zeros_like(a) for a in alone]
    ws = [launch.paged_attention_workspace(p.cache, p.batch, 8) for p in ps]
    torch.cuda.synchronize()
    for _ in range(20):
        for p, s, o, w in zip(ps, streams, outs, ws):
            launch.paged_attention(api.from_torch(o), api.from_torch(p.q), p.cache, p.batch, 0.1, workspace=w, stream=s)
    torch.cuda.synchronize()
    assert all(torch.equal(a, o) for a, o in zip(alone, outs))


def test_nothing_to_do(b200):
    p = ref.Problem([1], [5], 2, 1, 64, 16, BF16)
    t = api.from_torch(torch.empty(0, 2, 64, dtype=BF16, device="cuda"))
    kv = api.from_torch(torch.empty(0, 1, 64, dtype=BF16, device="cuda"))
    launch.paged_attention(t, t, p.cache, p.batch, 0.1)
    launch.paged_kv_append(p.cache, p.batch, kv, kv)
    launch.paged_kv_gather(kv, kv, p.cache, p.batch)


def test_device_and_stream_of_the_call(b200):
    p = ref.Problem([1], [5], 2, 1, 64, 16, BF16)
    o = torch.empty_like(p.q)
    with pytest.raises(KernelLaunchError, match="cpu"):
        launch.paged_attention(api.from_torch(o), api.from_torch(p.q.cpu()), p.cache, p.batch, 0.1)
    with pytest.raises(KernelLaunchError, match="workspace"):
        launch.paged_attention(api.from_torch(o), api.from_torch(p.q), p.cache, p.batch, 0.1,
                               workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))


def test_page_numbers_outside_the_pool(b200):
    """Zeros are read and nothing is written; the sequence is named in the status record."""
    for fmt in ("16bit", "nvfp4"):
        for bad in (-1, 1 << 20):
            p = ref.Problem([1, 1], [40, 60], 4, 2, 64, 16, BF16, fmt, seed=13)
            good = p.table[1, 1].clone()
            p.table[1, 1] = bad
            got = _attend(p, 0.2)
            assert _status(b200)[:2] == (4, 1)
            _lib.check(b200.b200tile_status_reset(torch.cuda.current_stream().cuda_stream))
            for x in p.pools:                            # the same with a page of zeros in its place
                x[p.free[0]] = 0
            p.table[1, 1] = int(p.free[0])
            assert torch.equal(got, _attend(p, 0.2))
            p.table[1, 1] = good
            # append at a position on a bad page leaves the pools alone
            p.table[1, 3] = bad
            before = [x.clone() for x in p.pools]
            launch.paged_kv_append(p.cache, p.batch, api.from_torch(p.k), api.from_torch(p.v))
            assert _status(b200)[:2] == (4, 1)
            _lib.check(b200.b200tile_status_reset(torch.cuda.current_stream().cuda_stream))
            pg = int(p.table[0, 39 // 16])
            for a, x in zip(before, p.pools):
                a[pg, :, 39 % 16] = x[pg, :, 39 % 16]    # sequence 0's token was written
                assert torch.equal(a, x)
