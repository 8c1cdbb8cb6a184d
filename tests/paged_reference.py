"""Plain 64-bit forms of the paged-cache operators, sequence by sequence, and builders of small problems."""
import math

import torch

MANY_KEYS = 1 << 17
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def pool(pages, kvh, page, last, dtype, layout, device="cuda"):
    if layout == "nhd":
        return torch.zeros(pages, page, kvh, last, dtype=dtype, device=device).permute(0, 2, 1, 3)
    return torch.zeros(pages, kvh, page, last, dtype=dtype, device=device)


def dequant(codes, scales, glob=1.0):
    """Packed bytes [.., D/2] and e4m3 bytes [.., D/16] -> the values they stand for, in 64 bits."""
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).long()
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), dtype=torch.float64, device=codes.device)
    s = scales.contiguous().view(torch.float8_e4m3fn).double() * glob
    return table[c] * s.repeat_interleave(16, -1)


class Problem:
    """Pools filled with random rows, a shuffled block table with junk behind every sequence's pages, ragged lengths.
    `table_keys` makes the block table that long at least: the choice of kernels goes by what a table could hold, so that
    MANY_KEYS has small problems of more than a few rows take the kernel of the large ones."""

    def __init__(self, q_lens, kv_lens, heads, kv_heads, d, page=16, dtype=torch.bfloat16, fmt="16bit", layout="hnd",
                 seed=0, extra_pages=3, k_global=1.0, v_global=1.0, pad_tokens=0, junk=-7, max_q=None, table_keys=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.q_lens, self.kv_lens, self.heads, self.kvh, self.d, self.page = q_lens, kv_lens, heads, kv_heads, d, page
        self.dtype, self.fmt, self.kg, self.vg = dtype, fmt, k_global, v_global
        need = [-(-max(n, 0) // page) for n in kv_lens]
        self.pages = sum(need) + extra_pages
        order = torch.randperm(self.pages, generator=g, device="cuda").int()
        self.table = torch.full((len(q_lens), max(max(need) + 2, 3, table_keys // page)), junk, dtype=torch.int32, device="cuda")
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.free = order[at:].long()                       # pages of no sequence
        cu = [0]
        for n in q_lens:
            cu.append(cu[-1] + n)
        self.cu = cu
        self.cu_q = torch.tensor(cu, dtype=torch.int32, device="cuda")
        self.kv = torch.tensor(kv_lens, dtype=torch.int32, device="cuda")
        self.tokens = cu[-1] + pad_tokens

        def rand(*shape):
            return torch.randn(*shape, generator=g, device="cuda")

        self.q = rand(self.tokens, heads, d).to(dtype)
        self.k = rand(self.tokens, kv_heads, d).to(dtype)
        self.v = rand(self.tokens, kv_heads, d).to(dtype)
        if fmt == "16bit":
            self.pools = [pool(self.pages, kv_heads, page, d, dtype, layout) for _ in range(2)]
            for p in self.pools:
                p.copy_(rand(*p.shape))
            self.scales = [None, None]
        else:
            self.pools = [pool(self.pages, kv_heads, page, d // 2, torch.uint8, layout) for _ in range(2)]
            self.scales = [pool(self.pages, kv_heads, page, d // 16, torch.uint8, layout) for _ in range(2)]
            for p, s, gl in zip(self.pools, self.scales, (k_global, v_global)):
                p.copy_(torch.randint(0, 256, p.shape, generator=g, device="cuda").to(torch.uint8))
                s.copy_((torch.rand(*s.shape, generator=g, device="cuda") * 0.6 / gl + 0.05 / gl)
                        .to(torch.float8_e4m3fn).view(torch.uint8))
        from cutile_rs_b200 import paged
        self.cache = paged.PagedKvCache(*self.pools, *self.scales, k_global, v_global)
        self.batch = paged.PagedBatch(self.table, self.cu_q, self.kv, max(max(q_lens), 1) if max_q is None else max_q)

    def rows(self, b, n):
        """First n cached rows of sequence b: K, V [n, kv_heads, d] in 64 bits."""
        pages = self.table[b, :-(-n // self.page)].long()
        out = []
        for p, s, gl in zip(self.pools, self.scales, (self.kg, self.vg)):
            x = p[pages].permute(0, 2, 1, 3).flatten(0, 1)[:n]
            if self.fmt != "16bit":
                x = dequant(x, s[pages].permute(0, 2, 1, 3).flatten(0, 1)[:n], gl)
            out.append(x.double())
        return out

    def unseen_slots(self):
        """Mask [pages, page] of the slots that belong to no sequence's rows."""
        m = torch.ones(self.pages, self.page, dtype=torch.bool, device="cuda")
        for b, n in enumerate(self.kv_lens):
            for j in range(-(-max(n, 0) // self.page)):
                m[self.table[b, j].long(), :min(self.page, n - j * self.page)] = False
        return m

    def poison(self):
        """NaN patterns in every slot that no sequence owns."""
        m = self.unseen_slots()
        for p, s in zip(self.pools, self.scales):
            if self.fmt == "16bit":
                p.permute(0, 2, 1, 3)[m] = float("nan")
            else:
                s.permute(0, 2, 1, 3)[m] = 0x7f


def attention(p, scale, causal=True, window=0, softcap=0.0):
    """(out, bound on |out - result|): the definition in 64 bits and what the kernel's arithmetic may add to it.

    Per row: the output's own rounding, half a step of its type; probabilities whose exponents are off by the scores'
    error (a 32-bit dot product of d terms, the score's scale and the exponential's argument: (d + 8) 2^-24 of
    sum |q k| scale, with a cap 2^-19 of it more) and which are handed over in two 16-bit pieces (2^-15 of p; one f16 piece, 2^-11,
    for bf16 over NVFP4; one piece of the type, half a step, in calls whose max_q_len allows more than 16 rows, 48 over NVFP4), all against sum p |v|; sums of n
    terms in 32 bits.  Pieces in f16 (f16 rows, and all rows over NVFP4) have no relative step below 2^-14: they are off by
    up to half of f16's smallest step, 2^-25, each, while the largest p is at least 1 and so is the sum they are divided by:
    2^-25 sum |v| over the keys seen."""
    out = torch.zeros(p.tokens, p.heads, p.d, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(out)
    group = p.heads // p.kvh
    eps = torch.finfo(p.dtype).eps
    small_pieces = p.dtype == torch.float16 or p.fmt != "16bit"
    few = 2.0 ** -11 if p.fmt != "16bit" and p.dtype == torch.bfloat16 else 2.0 ** -15
    for b, (n, kv) in enumerate(zip(p.q_lens, p.kv_lens)):
        if n == 0 or kv <= 0:
            continue
        piece = few if p.batch.max_q_len * group <= (16 if p.fmt == "16bit" else 48) else eps / 2
        k, v = p.rows(b, kv)
        pos = torch.arange(kv - n, kv, device="cuda")[:, None]
        key = torch.arange(kv, device="cuda")[None, :]
        seen = (key <= pos) if causal else torch.ones(n, kv, dtype=torch.bool, device="cuda")
        if window:
            seen = seen & (key > pos - window)
        for h in range(p.heads):
            q = p.q[p.cu[b]:p.cu[b + 1], h].double()
            kh, vh = k[:, h // group], v[:, h // group]
            s = q @ kh.T * scale
            ds = (p.d + 8) * 2.0 ** -24 * float((q.abs() @ kh.abs().T).max()) * scale
            if softcap:
                s = softcap * torch.tanh(s / softcap)
                ds += softcap * 2.0 ** -19
            s = s.masked_fill(~seen, -math.inf)
            top = s.amax(-1, keepdim=True)
            e = torch.exp(s - torch.where(top.isfinite(), top, torch.zeros_like(top)))
            l = e.sum(-1, keepdim=True)
            w = torch.where(l > 0, e / l.clamp(min=1e-300), torch.zeros_like(e))
            o = w @ vh
            out[p.cu[b]:p.cu[b + 1], h] = o
            tol[p.cu[b]:p.cu[b + 1], h] = eps / 2 * o.abs() + (3 * ds + piece + (kv + 16) * 2.0 ** -24 + 2.0 ** -20) * \
                (w @ vh.abs()) + (2.0 ** -25 * (seen.double() @ vh.abs()) if small_pieces else 0.0) + 1e-7
    return out, tol


def rotate(x, pos, inv_freq):
    """x [n, heads, d] turned by pos [n] in 64 bits, halves of the first 2 len(inv_freq) dimensions paired."""
    r = 2 * inv_freq.numel()
    a = pos.double()[:, None] * inv_freq.double()[None, :]
    c, s = a.cos()[:, None], a.sin()[:, None]
    lo, hi, rest = x[..., :r // 2].double(), x[..., r // 2:r].double(), x[..., r:].double()
    return torch.cat((lo * c - hi * s, hi * c + lo * s, rest), -1)


def quantise(x, glob=1.0):
    """NVFP4 blocks of x (64 bits): (value, scale * glob, distance to the nearest rounding border in steps of the scale)."""
    grid = torch.arange(0, 127, dtype=torch.uint8, device=x.device).view(torch.float8_e4m3fn).double()
    small = torch.tensor(E2M1, dtype=torch.float64, device=x.device)
    b = x.reshape(*x.shape[:-1], -1, 16)

    def nearest(v, values):
        hi = torch.searchsorted(values, v.contiguous()).clamp(max=len(values) - 1)
        lo = (hi - 1).clamp(min=0)
        up, down = (values[hi] - v).abs(), (v - values[lo]).abs()
        return values[torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)]

    want = b.abs().amax(-1, keepdim=True) / (6 * glob)
    s = nearest(want, grid) * glob
    y = torch.where(s > 0, b.abs() / s, torch.zeros_like(b))
    value = torch.sign(b) * nearest(y, small) * s
    borders = torch.tensor((0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0), dtype=torch.float64, device=x.device)
    margin = (y.unsqueeze(-1) - borders).abs().amin(-1)
    mids = (grid[1:] + grid[:-1]) / 2
    near = ((want.unsqueeze(-1) - mids).abs() / mids).amin(-1)
    return value.reshape(x.shape), s.expand_as(b).reshape(x.shape), torch.minimum(margin, near.expand_as(b)).reshape(x.shape)
