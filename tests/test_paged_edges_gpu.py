"""Paged key/value cache at the ends of what its calls accept, against 64-bit plain forms."""
import math

import pytest
import torch

import paged_reference as ref
from cutile_rs_b200 import api, launch, paged

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16
FORMS = [("16bit", 128, BF16), ("16bit", 64, F16), ("nvfp4", 128, BF16), ("nvfp4", 64, F16)]


def _attend(p, scale, **kw):
    out = torch.full((p.tokens, p.heads, p.d), -77.0, dtype=p.dtype, device="cuda")
    launch.paged_attention(api.from_torch(out), api.from_torch(p.q), p.cache, p.batch, scale, **kw)
    return out


def _largest_score(p, scale):
    """The largest |score| and |v| that a sequence's rows meet."""
    s = v_max = 0.0
    for b, (n, kv) in enumerate(zip(p.q_lens, p.kv_lens)):
        k, v = p.rows(b, kv)
        k = k.repeat_interleave(p.heads // p.kvh, 1)
        q = p.q[p.cu[b]:p.cu[b + 1]].double()
        s = max(s, float(torch.einsum("qhd,khd->hqk", q, k).abs().max()) * scale)
        v_max = max(v_max, float(v.abs().max()))
    return s, v_max


@pytest.mark.parametrize("keys", [0, ref.MANY_KEYS])
@pytest.mark.parametrize("fmt,d,dtype", FORMS)
@pytest.mark.parametrize("cap", [2e3, 1e5, 1e6, 1e8, 1e30, 3e38])
def test_caps_far_above_the_scores(b200, fmt, d, dtype, keys, cap):
    """c tanh(s / c) is s when c is far above it.  The bound does not grow with the cap: that of the uncapped call, and
    2^-20 of the largest score in every exponent, which three times (numerator, sum, both weights) reaches the output:
    the polynomial is off by 4.5e-8 < 2^-24 of the score with seven roundings of 2^-24 behind it, the exponential form,
    taken from 0.38 c on, by c 2^-22 < 2^-20 of it."""
    p = ref.Problem([150, 3, 1], [260, 40, 300], 6, 2, d, 16, dtype, fmt, seed=60, table_keys=keys)
    scale = d ** -0.5
    got = _attend(p, scale, softcap=cap)
    want, _ = ref.attention(p, scale, softcap=cap)
    _, tol = ref.attention(p, scale)
    s, v = _largest_score(p, scale)
    assert s < cap / 100                                   # so far below that the bound without a cap holds to 1 %
    assert ((got.double() - want).abs() <= 1.01 * tol + 3 * 2.0 ** -20 * s * v).all()


@pytest.mark.parametrize("keys", [0, ref.MANY_KEYS])
@pytest.mark.parametrize("fmt,d,dtype", FORMS)
def test_capped_rows_do_not_depend_on_their_neighbours(b200, fmt, d, dtype, keys):
    """A token whose scores reach the cap beside tokens whose scores are a small part of it: those are held to the bound
    of their own scores."""
    cap, scale = 1e5, d ** -0.5
    p = ref.Problem([90, 2], [200, 40], 4, 2, d, 16, dtype, fmt, seed=61, table_keys=keys)
    calm = p.q.clone()
    want, _ = ref.attention(p, scale, softcap=cap)
    _, tol = ref.attention(p, scale)
    s, v = _largest_score(p, scale)
    p.q[40:90:4] *= 1.5e4                                  # scores to 1e5: f16 holds such queries
    p.q[91] *= 1.5e4
    loud = (p.q != calm).any(-1).any(-1)
    got = _attend(p, scale, softcap=cap)
    assert not torch.isnan(got).any()
    assert ((got.double() - want).abs() <= tol + 3 * 2.0 ** -20 * s * v)[~loud].all()


@pytest.mark.parametrize("keys", [0, ref.MANY_KEYS])
@pytest.mark.parametrize("fmt", ["16bit", "nvfp4"])
def test_caps_far_below_the_scores(b200, fmt, keys):
    """A cap near zero leaves scores of +-c: plain means, whatever the scores are, zero among them."""
    p = ref.Problem([40, 2], [60, 30], 4, 2, 64, 16, BF16, fmt, seed=62, table_keys=keys)
    p.q[3] = 0
    for cap in (1e-6, 1e-30, 1e-40):
        got = _attend(p, 0.125, softcap=cap)
        want, tol = ref.attention(p, 0.125, softcap=cap)
        # the scores are off by no more than 2 c: nothing; the bound without a cap holds them
        assert ((got.double() - want).abs() <= tol).all(), cap


@pytest.mark.parametrize("keys", [0, ref.MANY_KEYS])
@pytest.mark.parametrize("window", [0, 60])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_infinite_scores_under_a_cap(b200, dtype, window, keys):
    """c tanh(-inf) = -c and c tanh(inf) = c: a key with an infinite score takes part, whichever kernel looks at it."""
    cap = 4.0
    p = ref.Problem([70, 3, 40], [300, 40, 40], 4, 2, 64, 16, dtype, seed=63, table_keys=keys)
    p.q[..., 0] = 0.5
    for b, key in ((0, 250), (0, 100), (1, 5), (2, 0), (2, 17)):
        page, slot = int(p.table[b, key // 16]), key % 16
        p.pools[0][page, 0, slot, 0] = float("-inf")
        p.pools[0][page, 1, slot, 0] = float("inf")
    got = _attend(p, 0.125, softcap=cap, window=window)
    # the definition with stand-ins for the infinite values that are far beyond the cap, too
    q = ref.Problem([70, 3, 40], [300, 40, 40], 4, 2, 64, 16, dtype, seed=63, table_keys=keys)
    q.q[..., 0] = 0.5
    for b, key in ((0, 250), (0, 100), (1, 5), (2, 0), (2, 17)):
        page, slot = int(q.table[b, key // 16]), key % 16
        q.pools[0][page, 0, slot, 0] = -30000.0
        q.pools[0][page, 1, slot, 0] = 30000.0
    want, _ = ref.attention(q, 0.125, softcap=cap, window=window)
    # as ref.attention's bound, for the scores that are not at the cap (which are exact), against the largest |v|
    q.pools[0][q.pools[0].abs() == 30000.0] = 0.0
    eps, room = torch.finfo(dtype).eps, 0.0
    for b, kv in enumerate(p.kv_lens):
        k, v = q.rows(b, kv)
        qk = float(torch.einsum("qhd,khd->hqk", q.q[q.cu[b]:q.cu[b + 1]].double().abs(),
                                k.abs().repeat_interleave(2, 1)).max()) * 0.125
        terms = 3 * ((64 + 8) * 2.0 ** -24 * qk + cap * 2.0 ** -19) + eps / 2 + (kv + 16) * 2.0 ** -24 + 2.0 ** -20
        room = max(room, float(v.abs().max()) * (terms + 2.0 ** -25 * kv))
    assert not torch.isnan(got).any()
    assert ((got.double() - want).abs() <= eps / 2 * want.abs() + room).all()


@pytest.mark.parametrize("keys", [0, ref.MANY_KEYS])
@pytest.mark.parametrize("softcap", [0.0, 4.0, 1e4])
def test_nan_scores_stay_nan(b200, softcap, keys):
    """The rows that see a NaN key are NaN, for the heads that it belongs to; the others are numbers."""
    for dtype in (BF16, F16):
        p = ref.Problem([70, 3], [300, 40], 4, 2, 64, 16, dtype, seed=68, table_keys=keys)
        p.pools[0][int(p.table[0, 260 // 16]), 1, 260 % 16, 5] = float("nan")
        got = _attend(p, 0.125, softcap=softcap)
        want = torch.zeros_like(got, dtype=torch.bool)
        want[260 - 230:70, 2:] = True                      # positions 230 .. 299
        assert torch.equal(torch.isnan(got), want)


@pytest.mark.parametrize("fmt,d,dtype", [("16bit", 128, F16), ("16bit", 64, F16), ("nvfp4", 128, BF16), ("nvfp4", 64, F16),
                                         ("nvfp4", 128, F16)])
@pytest.mark.parametrize("q_len,batch", [(1, 150), (40, 20)])
def test_a_long_tail_of_small_probabilities(b200, fmt, d, dtype, q_len, batch):
    """One key that holds most of the weight, with a value of zero, and 2^18 that share the rest: their probabilities,
    2^-19.6 of the first's, are far below the normal range of 16-bit floats (20.45 of f16's smallest steps), their sum is
    not.  The tail's keys are all alike, so that the result is known.  So many sequences, over the same pages, that most
    items are not cut and a worker meets the first key and its tail."""
    kv, kvh = (1 << 18) + 1, 8
    x = 24 - math.log2(20.45)                              # log2 of the first key's weight over one of the tail
    p = ref.Problem([q_len], [kv], kvh, kvh, d, 256, dtype, fmt, seed=64)
    for pool, scales in zip(p.pools, p.scales):
        pool.zero_()
        if scales is not None:
            scales.fill_(0x38)                             # 1.0
    first = int(p.table[0, 0])
    if fmt == "16bit":
        p.pools[0][first, :, 0, 0] = 1.0
        p.pools[1].fill_(0.5)
        p.pools[1][first, :, 0] = 0.0
    else:
        p.pools[0][first, :, 0, 0] = 0x2                   # code of 1
        p.pools[1].fill_(0x11)                             # codes of 0.5
        p.pools[1][first, :, 0] = 0
    q = torch.zeros(batch * q_len, kvh, d, dtype=dtype, device="cuda")
    q[..., 0] = 1.0
    cu = torch.arange(batch + 1, dtype=torch.int32, device="cuda") * q_len
    batch_of = paged.PagedBatch(p.table.repeat(batch, 1), cu, p.kv.repeat(batch), q_len)
    out = torch.empty_like(q)
    launch.paged_attention(api.from_torch(out), api.from_torch(q), p.cache, batch_of, x * math.log(2.0))
    n = torch.arange(kv - q_len, kv, device="cuda", dtype=torch.float64).repeat(batch)     # keys of the tail a token sees
    tail = n * 2.0 ** -x
    want = 0.5 * tail / (1 + tail)
    # half a step of the type; weights handed over in one f16 piece, 2^-11, and their exponents, x 2^-22, above and below
    # the line; the sum of the weights: up to 2^18 / 8 terms a lane, each rounded by 2^-24 of a partial sum of 1 + tail at
    # most, that of the products: 2^18 / 16 steps, two products each, that drop up to 2^-23 of the sum
    eps = torch.finfo(dtype).eps
    room = (eps / 2 + 2.0 ** -11 + 2 * x * 2.0 ** -22 + 2.0 ** -9 + 2.0 ** -8) * want
    off = (out.double() - want[:, None, None]).abs()
    assert (off <= room[:, None, None]).all(), float((off / room[:, None, None]).max())


def test_factors_that_underflow_together(b200):
    """A scale times a factor of the pool below the smallest 32-bit number: every score is 0, masked keys stay out."""
    for keys in (0, ref.MANY_KEYS):
        for softcap in (0.0, 20.0):
            p = ref.Problem([70, 2], [90, 200], 4, 2, 64, 16, BF16, "nvfp4", seed=65, table_keys=keys)
            p.poison()
            p.kg = 1e-30
            p.cache = paged.PagedKvCache(*p.pools, *p.scales, 1e-30, 1.0)
            got = _attend(p, 1e-20, softcap=softcap)
            want, tol = ref.attention(p, 1e-20, softcap=softcap)
            assert not torch.isnan(got).any()
            assert ((got.double() - want).abs() <= tol).all()


def test_nan_on_the_way_into_nvfp4_stays_visible(b200):
    """A block that holds a NaN, among finite values, among zeros, among infinities or alone, reads back as NaN; the other
    blocks of its row keep their values; attention over it is NaN for the heads that see it."""
    for d, rot in ((64, 0), (128, 32), (128, 128)):
        p = ref.Problem([6], [6], 2, 1, d, 16, BF16, "nvfp4", seed=66)
        clean = [x.clone() for x in (p.k, p.v)]
        nan, inf = float("nan"), float("inf")
        p.v[0, 0, 3] = nan
        p.v[1, 0, :16] = 0.0
        p.v[1, 0, 7] = nan
        p.v[2, 0, 16:32] = nan
        p.v[3, 0, 16], p.v[3, 0, 17] = inf, nan
        p.v[4, 0, 31] = -nan
        p.k[5, 0, d - 1] = nan
        f = None
        if rot:
            i = torch.arange(0, rot, 2, dtype=torch.float64, device="cuda")
            f = api.from_torch((10000.0 ** (-i / rot)).float())
        launch.paged_kv_append(p.cache, p.batch, api.from_torch(p.k), api.from_torch(p.v), inv_freq=f)
        out = [torch.empty(6, 1, d, dtype=BF16, device="cuda") for _ in range(2)]
        launch.paged_kv_gather(api.from_torch(out[0]), api.from_torch(out[1]), p.cache, p.batch)
        k, v = out
        for t, block in ((0, 0), (1, 0), (2, 1), (3, 1), (4, 1)):
            want = torch.zeros(d // 16, dtype=torch.bool, device="cuda")
            want[block] = True
            assert torch.equal(torch.isnan(v[t, 0]).reshape(-1, 16).all(-1), want)
            assert torch.equal(torch.isnan(v[t, 0]).reshape(-1, 16).any(-1), want)
        lost = torch.isnan(k[5, 0]).reshape(-1, 16)
        turned = {d // 16 - 1} | ({d // 32 - 1} if rot == d else set())      # its partner in the rotation, too
        assert {i for i in range(d // 16) if lost[i].any()} == turned and all(lost[i].all() for i in turned)
        assert not torch.isnan(k[:5]).any() and not torch.isnan(v[5]).any()
        good = ~torch.isnan(v)
        q = ref.Problem([6], [6], 2, 1, d, 16, BF16, "nvfp4", seed=66)
        launch.paged_kv_append(q.cache, q.batch, api.from_torch(clean[0]), api.from_torch(clean[1]))
        assert torch.equal(p.rows(0, 6)[1][good], q.rows(0, 6)[1][good])


def test_decode_steps_keep_their_kernel_beside_anything(b200):
    """Single tokens over long tables go to the kernel of few rows, which hands probabilities over in two pieces, beside a
    prompt or under a max_q_len that allows far more tokens than there are.  Keys of two scores, whose values cancel: the
    output is small beside the sums, so that the rounding of one piece, up to 2^-9 of them, would show."""
    d, kv, page = 64, 4096, 64
    for prompts, max_q in (([], 4096), ([200], None), ([200, 300], None)):
        q_lens = [1] * 12 + prompts
        p = ref.Problem(q_lens, [kv] * len(q_lens), 16, 8, d, page, BF16, seed=67, table_keys=ref.MANY_KEYS, max_q=max_q)
        p.q.zero_()
        p.q[..., 0] = 1.0
        for pool in p.pools:
            pool.zero_()
        p.pools[0][:, :, ::2, 0] = 0.25                    # half of the keys score 0.25, the others 0
        p.pools[1][:, :, ::2] = 1.0
        p.pools[1][:, :, 1::2] = -1.28125
        want, _ = ref.attention(p, 1.0)
        got = _attend(p, 1.0)[:12].double()
        want = want[:12]
        weight = 1.15                                      # sum p |v| / sum p
        assert want.abs().max() < 0.01
        assert ((got - want).abs() <= 2.0 ** -9 * want.abs() + (2.0 ** -15 + 80 * 2.0 ** -24 + 4096 * 2.0 ** -24) * weight).all(), \
            float((got - want).abs().max())


@pytest.mark.parametrize("fmt", ["16bit", "nvfp4"])
@pytest.mark.parametrize("heads,kvh,n", [(5, 1, 3), (32, 8, 1), (32, 8, 2000), (128, 2, 40)])
def test_append_rotates_queries_in_place(b200, fmt, heads, kvh, n):
    """q_out may be q, also inside a fused projection's rows, with one or many warps to a token: the bits of a call with an
    output of its own."""
    p = ref.Problem([n, 1], [n + 100, 7], heads, kvh, 128, 16, BF16, fmt, seed=69)
    i = torch.arange(0, 128, 2, dtype=torch.float64, device="cuda")
    f = api.from_torch((10000.0 ** (-i / 128)).float())
    k, v = api.from_torch(p.k), api.from_torch(p.v)
    want = torch.empty_like(p.q)
    launch.paged_kv_append(p.cache, p.batch, k, v, q=api.from_torch(p.q), q_out=api.from_torch(want), inv_freq=f)
    pools = [x.clone() for x in p.pools]
    for _ in range(3):
        rows = torch.full((p.tokens, heads + 2 * kvh, 128), 5.0, dtype=BF16, device="cuda")
        q = rows[:, :heads]
        q.copy_(p.q)
        t = api.from_torch(q)
        launch.paged_kv_append(p.cache, p.batch, k, v, q=t, q_out=t, inv_freq=f)
        assert torch.equal(q, want) and (rows[:, heads:] == 5.0).all()
        assert all(torch.equal(a, b) for a, b in zip(pools, p.pools))


def test_wide_scales_in_f16(b200):
    """Scales over the whole of e4m3, 2^-9 to 448, with a factor that keeps the output inside f16."""
    for keys in (0, ref.MANY_KEYS):
        p = ref.Problem([1, 30], [70, 41], 4, 2, 64, 16, F16, "nvfp4", seed=71, table_keys=keys, v_global=2.0 ** -4)
        for x in p.scales[1:]:
            x.copy_(torch.randint(1, 0x7f, x.shape, device="cuda").to(torch.uint8))
        got = _attend(p, 0.125)
        want, tol = ref.attention(p, 0.125)
        assert not torch.isnan(got).any() and ((got.double() - want).abs() <= tol).all()


def _piece_bound(p, scale, rows):
    """ref.attention's bound for tokens that the kernel of few rows takes, whatever else is in the call: probabilities in
    two pieces, 2^-15 (one f16 piece, 2^-11, for bf16 over NVFP4)."""
    keep = p.batch
    p.batch = paged.PagedBatch(p.table, p.cu_q, p.kv, 1)    # the bound of a call of single tokens
    want, tol = ref.attention(p, scale)
    p.batch = keep
    return want[rows], tol[rows]


@pytest.mark.parametrize("fmt,d,dtype", FORMS + [("nvfp4", 128, F16)])
def test_steps_beside_prompts_are_held_to_their_own_bound(b200, fmt, d, dtype):
    """150 decode steps beside two prompts, where each kernel takes its own sequences, and short prompts behind a short
    table, which the kernel of few rows takes alone: two pieces in both."""
    q_lens = [1] * 150 + [130, 40]
    kv_lens = [1 + (53 * i) % 400 for i in range(150)] + [300, 500]
    p = ref.Problem(q_lens, kv_lens, 8, 2, d, 16, dtype, fmt, seed=72, table_keys=ref.MANY_KEYS)
    got = _attend(p, d ** -0.5)
    want, tol = _piece_bound(p, d ** -0.5, slice(0, 150))
    assert ((got[:150].double() - want).abs() <= tol).all()
    p = ref.Problem([40, 17, 1], [60, 40, 90], 8, 2, d, 16, dtype, fmt, seed=73)
    got = _attend(p, d ** -0.5)
    want, tol = _piece_bound(p, d ** -0.5, slice(None))
    assert ((got.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("fmt", ["16bit", "nvfp4"])
@pytest.mark.parametrize("steps,prompts,kv", [(150, [130, 40], 400), (3, [200, 90], 300), (40, [], 3000)])
def test_captured_calls_of_every_kernel_at_once(b200, fmt, steps, prompts, kv):
    """Decode steps beside prompts, prompts alone and steps alone, several calls to a graph, two graphs replayed on two
    streams at once with a workspace each and lengths that change between replays: the bits of eager calls."""
    q_lens = [1] * steps + prompts
    ps = []
    for seed in (80, 81):
        kv_lens = [kv - (53 * i) % (kv - 20) for i in range(steps)] + [n + 70 for n in prompts]
        ps.append(ref.Problem(q_lens, kv_lens, 8, 2, 64, 16, BF16, fmt, seed=seed, table_keys=ref.MANY_KEYS))
    first = [p.kv.clone() for p in ps]
    # everything a graph points to lives as long as the graph does: beginning a capture gives cached memory back
    spaces = [launch.paged_attention_workspace(p.cache, p.batch, 8) for p in ps]
    outs = [[torch.zeros_like(p.q) for _ in range(3)] for p in ps]
    streams = [torch.cuda.Stream() for _ in ps]
    torch.cuda.synchronize()

    def calls(p, ws, out, s):
        for o, cap in zip(out, (0.0, 20.0, 1e4)):
            launch.paged_attention(api.from_torch(o), api.from_torch(p.q), p.cache, p.batch, 0.125, softcap=cap,
                                   workspace=ws, stream=s)

    graphs = []
    for p, ws, out, s in zip(ps, spaces, outs, streams):
        calls(p, ws, out, s)
        s.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            calls(p, ws, out, s)
        graphs.append(g)
    for shorter in (0, 7, 19):
        want = []
        for p, lens in zip(ps, first):
            p.kv.copy_((lens - shorter).clamp(min=1))
            want.append([_attend(p, 0.125, softcap=cap) for cap in (0.0, 20.0, 1e4)])
        torch.cuda.synchronize()
        for _ in range(5):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for a, b in zip(want, outs):
            assert all(torch.equal(x, y) for x, y in zip(a, b))
