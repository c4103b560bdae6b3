"""The 8-bit cache's format and the attention over it, plainly, in 64 bits."""
import math

import numpy as np
import torch

HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}     # half a step, relative

# the 256 numbers of e4m3 by their code (0x7f and 0xff are NaN)
_E4M3 = [(-1.0) ** (c >> 7) * ((c & 7) * 2.0 ** -9 if (c >> 3) & 15 == 0
                               else (1 + (c & 7) / 8) * 2.0 ** (((c >> 3) & 15) - 7)) for c in range(256)]
_E4M3[0x7f] = _E4M3[0xff] = math.nan
E4M3 = torch.tensor(_E4M3, dtype=torch.float64)


def scale_exponent(most: float) -> int:
    """The smallest e with most <= 448 * 2^e, in [-100, 119]."""
    if most == 0.0:
        return -100
    e = math.ceil(math.log2(most / 448.0))
    while most <= 448.0 * 2.0 ** (e - 1):
        e -= 1
    while most > 448.0 * 2.0 ** e:
        e += 1
    return min(max(e, -100), 119)


def quantise_rows(x: torch.Tensor):
    """(codes, scale bytes, values) of the rows of x (any leading shape); a row that is not finite is
    codes of zero, byte 255 and NaNs."""
    flat = x.double().cpu().reshape(-1, x.shape[-1]).numpy()
    table = E4M3[:0x7f].numpy()                                   # 0 .. 448, ascending
    codes = np.zeros(flat.shape, dtype=np.uint8)
    scales = np.zeros(flat.shape[0], dtype=np.uint8)
    values = np.zeros(flat.shape)
    for i, row in enumerate(flat):
        if not np.isfinite(row).all():
            scales[i], values[i] = 255, math.nan
            continue
        e = scale_exponent(float(np.abs(row).max()))
        y = np.minimum(np.abs(row) * 2.0 ** -e, 448.0)
        hi = np.minimum(np.searchsorted(table, y), 0x7e)          # table[hi] >= y
        lo = np.maximum(hi - 1, 0)
        up, down = table[hi] - y, y - table[lo]
        pick = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
        pick = np.where(table[hi] == y, hi, pick)
        codes[i] = pick | (np.signbit(row).astype(np.uint8) << 7)
        scales[i] = e + 127
        values[i] = np.where(np.signbit(row), -1, 1) * table[pick] * 2.0 ** e
    shape = tuple(x.shape)
    return (torch.from_numpy(codes).reshape(shape), torch.from_numpy(scales).reshape(shape[:-1]),
            torch.from_numpy(values).reshape(shape))


def values_of(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """What codes (uint8 or float8) and scale bytes stand for, float64 on the CPU."""
    v = E4M3[codes.view(torch.uint8).cpu().long()] * torch.exp2(scales.cpu().double() - 127.0).unsqueeze(-1)
    return torch.where((scales.cpu() == 255).unsqueeze(-1), torch.full_like(v, math.nan), v)


class Case:
    """Requests with random cached rows on scrambled pages, and the queries of some of their tokens."""

    def __init__(self, lens_q, lens_kv, nq, nkv, hd, page, act, seed=0, window=0, keep=0, device="cuda:0", q_scale=1.5,
                 spare=3):
        g = torch.Generator().manual_seed(seed)
        self.lens_q, self.lens_kv = list(lens_q), list(lens_kv)
        self.nq, self.nkv, self.hd, self.page, self.act, self.window, self.keep = nq, nkv, hd, page, act, window, keep
        self.scale = hd ** -0.5
        n = len(lens_q)
        width = max(1, max(-(-k // page) for k in lens_kv))
        table = torch.full((n, width), -1, dtype=torch.int32)
        held = []
        for r in range(n):
            first = max(0, lens_kv[r] - lens_q[r] - window + 1) if window else 0
            held += [(r, p) for p in range(-(-lens_kv[r] // page)) if p >= first // page or p * page < keep]
        order = torch.randperm(len(held) + spare, generator=g)
        for i, (r, p) in enumerate(held):
            table[r, p] = order[i]
        pages = len(held) + spare
        rows = torch.randn(pages, 2, nkv, page, hd, generator=g) * torch.exp(
            0.5 * torch.randn(pages, 2, nkv, page, 1, generator=g))
        self.codes, self.scales, self.values = quantise_rows(rows)
        self.table = table
        tokens = sum(lens_q)
        self.q = (q_scale * torch.randn(tokens, nq * hd, generator=g)).to(act)
        self.req = [r for r in range(n) for _ in range(lens_q[r])]
        self.pos = [lens_kv[r] - lens_q[r] + i for r in range(n) for i in range(lens_q[r])]
        self.indptr = [sum(lens_q[:r]) for r in range(n + 1)]
        self.device = device

    def i32(self, v):
        return torch.as_tensor(v, dtype=torch.int32, device=self.device)

    def cache(self):
        return self.codes.to(self.device).view(torch.float8_e4m3fn), self.scales.to(self.device)

    def decode(self, out=None, q=None, max_len=None, cache=None):
        from mstar_b200 import ops

        q = self.q.to(self.device) if q is None else q
        out = torch.full((len(self.req), self.nq * self.hd), 7.0, dtype=self.act, device=self.device) if out is None else out
        codes, scales = cache or self.cache()
        ops.paged_decode_attention_kv8(q, out, codes, scales, self.table.to(self.device), self.i32(self.req),
                                       self.i32(self.pos), len(self.req), self.nq, self.nkv, self.hd, self.page,
                                       self.window, self.keep, self.scale, max_len or max(self.lens_kv))
        return out

    def prefill(self, out=None, q=None, first=0, entries=None, max_len=None, max_q=None, cache=None):
        from mstar_b200 import ops

        q = self.q.to(self.device) if q is None else q
        out = torch.full((len(self.req), self.nq * self.hd), 7.0, dtype=self.act, device=self.device) if out is None else out
        codes, scales = cache or self.cache()
        ops.paged_prefill_attention_kv8(
            q, out, codes, scales, self.table.to(self.device), self.i32(self.indptr), self.i32(self.lens_kv), first,
            len(self.lens_q) - first if entries is None else entries, max_q or max(self.lens_q), self.nq, self.nkv,
            self.hd, self.page, self.window, self.keep, self.scale, max_len or max(self.lens_kv))
        return out

    def plain(self):
        """(the output, the bound below which a kernel's output stays), [tokens, heads * dim] in float64.

        The bound, elementwise, with h half a step of the output's type and A = sum of weight * |value|:
        h |out| for the last rounding; weights rounded to the type of the product, 2^-8 relative in the
        16-bit mode (bfloat16 or finer), nothing in the 32-bit one; scores in float, each sum of D products
        off by at most (D + 8) u S with S = scale * sum |q k| and u = 2^-23 (tensor cores may cut instead of
        rounding), twice (numerator and denominator); exponentials and the n terms' sums (8 + n / 16 + 16) u
        relative (sums of tiles, at least 16 partial sums a row)."""
        T, G, hd = len(self.req), self.nq // self.nkv, self.hd
        q = self.q.double().view(T, self.nq, hd)
        out, bound = torch.zeros(T, self.nq, hd, dtype=torch.float64), torch.zeros(T, self.nq, hd, dtype=torch.float64)
        u, h = 2.0 ** -23, HALF[self.act]
        w = 2.0 ** -8 if self.act == torch.bfloat16 else 0.0
        for t in range(T):
            r, p = self.req[t], self.pos[t]
            keys = [k for k in range(p + 1) if not self.window or k > p - self.window or k < self.keep]
            if not keys:
                continue
            at = torch.tensor(keys)
            pages = self.table[r].long()[at // self.page]
            assert (pages >= 0).all()
            rows = self.values[pages, :, :, at % self.page]                 # [keys, 2, nkv, hd]
            for i in range(self.nq):
                k, v = rows[:, 0, i // G], rows[:, 1, i // G]
                s = (k @ q[t, i]) * self.scale
                p_ = torch.softmax(s, 0)
                out[t, i] = p_ @ v
                spread = (k.abs() @ q[t, i].abs()) * self.scale
                rel = 2 * (hd + 8) * u * float(spread.max()) + (24 + len(keys) / 16) * u + w
                bound[t, i] = h * out[t, i].abs() + rel * (p_ @ v.abs())
        return out.view(T, -1), 1.02 * bound.view(T, -1) + 1e-30

    def check(self, got):
        want, bound = self.plain()
        err = (got.double().cpu() - want).abs()
        worst = float((err / bound).nan_to_num(nan=math.inf).max())
        assert worst <= 1.0, f"off by {worst:.3g} times the bound (largest error {float(err.max()):.3g})"
