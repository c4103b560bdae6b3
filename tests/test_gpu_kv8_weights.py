"""How many bits the weights of the attention over the 8-bit cache keep: keys far below the largest, in score or in the
size of their values, in the features where the large ones have zeros, and the 32-bit mode's own roundings."""
import pytest
import torch

from kv8_util import HALF, Case, values_of

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F32, BF16 = torch.float32, torch.bfloat16


def case_of(rows, q, lens_q, lens_kv, nq, nkv, hd, page, act, window=0, keep=0):
    """A ``Case`` with the given numbers: rows [requests][tokens, 2, nkv, hd] (float64), rounded to the cache's format
    by torch's cast, and queries [tokens, nq * hd]."""
    c = Case.__new__(Case)
    c.lens_q, c.lens_kv = list(lens_q), list(lens_kv)
    c.nq, c.nkv, c.hd, c.page, c.act, c.window, c.keep, c.scale, c.device = nq, nkv, hd, page, act, window, keep, hd ** -0.5, DEV
    n, width = len(lens_q), max(-(-k // page) for k in lens_kv)
    c.table = torch.full((n, width), -1, dtype=torch.int32)
    order = torch.randperm(n * width, generator=torch.Generator().manual_seed(1)).int()
    codes = torch.zeros(n * width, 2, nkv, page, hd, dtype=torch.uint8)
    scales = torch.zeros(n * width, 2, nkv, page, dtype=torch.uint8)
    for r in range(n):
        pages = -(-lens_kv[r] // page)
        c.table[r, :pages] = order[r * width:r * width + pages]
        x = rows[r]
        mantissa, exponent = torch.frexp(x.abs().amax(-1))
        e = (exponent - 9 + (mantissa > 0.875).int()).clamp(-100, 119)
        e = torch.where(x.abs().amax(-1) > 0, e, torch.full_like(e, -100))
        code = (x * torch.exp2(-e.double())[..., None]).clamp(-448, 448).float().to(torch.float8_e4m3fn).view(torch.uint8)
        at = torch.arange(lens_kv[r])
        codes[c.table[r].long()[at // page], :, :, at % page] = code
        scales[c.table[r].long()[at // page], :, :, at % page] = (e + 127).to(torch.uint8)
    c.codes, c.scales = codes, scales
    c.q = q.to(act)
    c.req = [r for r in range(n) for _ in range(lens_q[r])]
    c.pos = [lens_kv[r] - lens_q[r] + i for r in range(n) for i in range(lens_q[r])]
    c.indptr = [sum(lens_q[:r]) for r in range(n + 1)]
    return c


def exact(c, w, rounded=lambda p: p, sums=None):
    """(the output, the bound below which a kernel's output stays), [tokens, heads * dim] in float64 on the GPU.

    The bound, elementwise, with h half a step of the output's type, A = sum of weight * |value| and u = 2^-23 (tensor cores
    may cut sums): h |out| for the last rounding; a score is off by 2^-22 of S = scale * sum |q k| for a query of two
    float16 parts (nothing more where it is a bfloat16 in two codes: 2^-17.8 of the row's largest number there, below) and
    by (D / 8 + 10) u S for the float sums of tiles of 16 features, its scaling and its difference to the maximum, in
    numerator and denominator; an exponential by 2^-21; a weight by ``w``; sums over n keys in steps of 16 and of
    three parts by (3 n / 16 + 24) u, or ``sums``.  Nothing is allowed in absolute terms: a key counts for what it weighs in every feature."""
    T, G, hd = len(c.req), c.nq // c.nkv, c.hd
    values = values_of(c.codes, c.scales).to(DEV)
    q = c.q.double().view(T, c.nq, hd).to(DEV)
    out, bound = torch.zeros(T, c.nq, hd, dtype=torch.float64, device=DEV), torch.zeros(T, c.nq, hd, dtype=torch.float64, device=DEV)
    u = 2.0 ** -23
    for t in range(T):
        at = torch.arange(c.pos[t] + 1)
        rows = values[c.table[c.req[t]].long()[at // c.page].to(DEV), :, :, (at % c.page).to(DEV)]
        for i in range(c.nq):
            k, v = rows[:, 0, i // G], rows[:, 1, i // G]
            p = torch.softmax((k @ q[t, i]) * c.scale, 0)
            out[t, i] = rounded(p) @ v
            spread = float((k.abs() @ q[t, i].abs()).max()) * c.scale
            codes = 2.0 ** -17.8 * float(q[t, i].abs().max() * k.abs().sum(-1).max()) * c.scale if c.act == BF16 else 0.0
            rel = 2 * ((2.0 ** -22 + (hd / 8 + 10) * u) * spread + codes + 2.0 ** -21) + w + ((3 * len(at) / 16 + 24) * u if sums is None else sums)
            bound[t, i] = HALF[c.act] * out[t, i].abs() + rel * (p @ v.abs())
    return out.view(T, -1), 1.02 * bound.view(T, -1)


def check(c, got, w):
    want, bound = exact(c, w)
    err = (got.double() - want).abs()
    assert torch.isfinite(got).all()
    worst = float((err / (bound + 1e-300)).max())
    assert worst <= 1.0, f"off by {worst:.3g} times the bound"


def weight_bits(act, hd, portion):
    """Half a step of a weight: float on CUDA cores; three bfloat16 parts in the 32-bit mode; one in the 16-bit mode's
    portions of heads of 64 and 128, two elsewhere."""
    if hd not in (64, 128, 256):
        return 0.0
    if act == F32:
        return 2.0 ** -24
    return 2.0 ** -8 if portion and hd <= 128 else 2.0 ** -16


def peaked(n, new, nq, nkv, hd, act, gap, ratio, seed=0):
    """One key in the middle whose score lies ``gap`` above the others' and whose value is ``ratio`` in one feature and zero
    in all others, where the others have a common direction; a second one that is like the rest follows behind it."""
    g = torch.Generator().manual_seed(seed)
    rows = torch.zeros(n, 2, nkv, hd, dtype=torch.float64)
    rows[:, 0] = torch.randn(n, nkv, hd, generator=g).double()
    rows[:, 1] = 0.7 + 0.2 * torch.randn(n, nkv, hd, generator=g).double()
    rows[:, 0, :, 0] = 0.0
    top = n // 3
    rows[top, 0] = 0.0
    rows[top, 0, :, 0] = 16.0
    rows[top, 1] = 0.0
    rows[top, 1, :, 5] = ratio
    q = 0.05 * torch.randn(new, nq, hd, generator=g)
    q[:, :, 0] = gap / 16.0 * hd ** 0.5
    return rows, q.view(new, nq * hd)


FAR = [(12.0, 1.0), (17.4, 1.0), (20.0, 1.0), (40.0, 1.0), (0.0, 2.0 ** 20), (0.0, 2.0 ** 24), (0.0, 2.0 ** 60), (0.0, 2.0 ** 100),
       (12.0, 2.0 ** -30), (20.0, 2.0 ** 30)]


@pytest.mark.parametrize("act", [F32, BF16])
@pytest.mark.parametrize("nq,nkv,hd", [(4, 2, 48), (6, 2, 64), (6, 2, 128), (8, 1, 128), (7, 1, 64), (2, 1, 256), (8, 1, 256)])
@pytest.mark.parametrize("gap,ratio", FAR)
def test_light_keys_count_where_heavy_ones_have_zeros(act, nq, nkv, hd, gap, ratio):
    n, page = 3001, 16
    for new, portion in ((1, False), (2, True), (40, True)):
        rows, q = peaked(n, new, nq, nkv, hd, act, gap, ratio, seed=hd + nq)
        c = case_of([rows], q, [new], [n], nq, nkv, hd, page, act)
        check(c, c.prefill() if portion else c.decode(), weight_bits(act, hd, portion))


@pytest.mark.parametrize("act", [F32, BF16])
@pytest.mark.parametrize("hd,page", [(64, 16), (128, 16), (128, 12)])
def test_many_light_keys(act, hd, page):
    """16,384 of them 17.4 below one: together 4.5e-4 of its weight, and all there is in the other features."""
    n = 16385
    rows, q = peaked(n, 1, 4, 2, hd, act, 17.4, 1.0, seed=3)
    c = case_of([rows], q, [1], [n], 4, 2, hd, page, act)
    check(c, c.decode(), weight_bits(act, hd, False))
    check(c, c.prefill(), weight_bits(act, hd, True))


@pytest.mark.parametrize("act", [F32, BF16])
@pytest.mark.parametrize("hd", [48, 64, 128, 256])
@pytest.mark.parametrize("exponent", [-90, 0, 7, 8, 60, 110])
def test_codes_of_every_kind(act, hd, exponent):
    """One key, and a few: subnormal codes, the largest one, zeros, at scales on both sides of each step."""
    g = torch.Generator().manual_seed(7)
    rows = []
    for n in (1, 37):
        x = torch.randint(-7, 8, (n, 2, 2, hd), generator=g).double() * 2.0 ** -9      # subnormal codes
        x[..., 1::4] = torch.randn(n, 2, 2, hd // 4, generator=g).double() * 16
        x[..., 0] = 448.0
        x[:, 1] *= 2.0 ** exponent
        x[:, 0, :, 0] = 2.0
        rows.append(x)
    for new, portion in ((1, False), (1, True)):
        q = 0.3 * torch.randn(2 * new, 4 * hd, generator=g)
        c = case_of(rows, q, [new, new], [1, 37], 4, 2, hd, 16, act)
        check(c, c.prefill() if portion else c.decode(), weight_bits(act, hd, portion))


@pytest.mark.parametrize("hd", [48, 64, 128, 256])
def test_the_32_bit_mode_keeps_its_bits(hd):
    """Small queries, so that scores cost little: the bound is below what one float16 a weight would be off by, which is
    shown with weights of the exact form rounded so."""
    g = torch.Generator().manual_seed(11)
    for lens_q, lens_kv in (([1, 1, 1], [2, 9, 60]), ([2, 20, 33], [2, 21, 60])):
        rows = [torch.randn(n, 2, 2, hd, generator=g).double() for n in lens_kv]
        q = 0.25 * torch.randn(sum(lens_q), 4 * hd, generator=g)
        c = case_of(rows, q, lens_q, lens_kv, 4, 2, hd, 16, F32)
        want, bound = exact(c, 2.0 ** -24)
        got = c.decode() if max(lens_q) == 1 else c.prefill()
        assert ((got.double() - want).abs() <= bound).all()
        rounded, _ = exact(c, 0.0, lambda p: p.half().double())
        assert float(((rounded - want).abs() / bound).max()) > 2.0


@pytest.mark.parametrize("nq,nkv,hd", [(4, 2, 64), (4, 2, 128), (2, 1, 256)])
@pytest.mark.parametrize("new", [1, 3, 40])
def test_long_sums_of_the_32_bit_mode_do_not_drift(nq, nkv, hd, new):
    """30,000 keys in one part, or one a warp, whose values have one sign: sums that are cut instead of rounded lose half a
    step of a float at every product of 16 keys, 7e-5 in all.  Allowed are a tile's sum of 12 products, cut (12 u), a rounded
    sum for every tile of 64 keys (of 16 with few rows, but a warp has a quarter of the keys then) of the outputs and of the
    normaliser (n / 64 halves of u each), and 16 u for a row's sum of a tile's weights and the joining of parts."""
    n, u = 30_000, 2.0 ** -23
    g = torch.Generator().manual_seed(17)
    rows = torch.randn(n, 2, nkv, hd, generator=g).double()
    rows[:, 1] = 1.0 + 0.1 * rows[:, 1]
    q = 0.02 * torch.randn(new, nq * hd, generator=g)
    c = case_of([rows], q, [new], [n], nq, nkv, hd, 16, F32)
    want, bound = exact(c, 2.0 ** -24, sums=(n / 64 + 12 + 16) * u)
    got = c.decode(max_len=1) if new == 1 else c.prefill(max_len=1)
    assert float((bound / want.abs()).max()) < 1e-4
    assert float(((got.double() - want).abs() / bound).max()) <= 1.0
