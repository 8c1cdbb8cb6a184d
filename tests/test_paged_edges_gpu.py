"""Paged key/value cache at the ends of what its calls accept, against 64-bit plain forms."""
import pytest
import torch

import paged_reference as ref
from cutile_rs_b200 import api, launch

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
