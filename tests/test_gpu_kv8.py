"""The 8-bit cache on the GPU: rows written and read back, attention of single tokens and of portions
against the plain forms in 64 bits, and the engine on such a cache."""
import math

import pytest
import torch

import plain_llama as P
from kv8_util import HALF, Case, quantise_rows, values_of

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F32, BF16 = torch.float32, torch.bfloat16


def i32(v):
    return torch.as_tensor(v, dtype=torch.int32, device=DEV)


def freqs(rot):
    return torch.tensor([10000.0 ** (-2.0 * j / rot) for j in range(rot // 2)], dtype=F32, device=DEV) if rot else None


def rotate64(x, pos, rot, inter):
    """Rotary encoding of x [tokens, heads, hd] in float64, from the float frequencies."""
    x = x.double().cpu().clone()
    if not rot:
        return x
    a = torch.as_tensor(pos, dtype=torch.float64)[:, None] * freqs(rot).double().cpu()
    c, s = a.cos()[:, None], a.sin()[:, None]
    lo, hi = (slice(0, rot, 2), slice(1, rot, 2)) if inter else (slice(0, rot // 2), slice(rot // 2, rot))
    x0, x1 = x[..., lo].clone(), x[..., hi].clone()
    x[..., lo], x[..., hi] = x0 * c - x1 * s, x1 * c + x0 * s
    return x


# ------------------------------------------------------------------ writing and reading back
WRITES = [  # nq, nkv, hd, rot, interleaved
    (6, 3, 48, 48, False), (5, 1, 32, 16, False), (4, 4, 16, 16, True), (2, 1, 64, 0, False), (8, 2, 128, 128, False),
    (3, 3, 24, 12, False), (4, 1, 256, 256, True), (7, 1, 200, 72, False), (24, 8, 128, 64, False), (1, 1, 8, 2, True)]


@pytest.mark.parametrize("act", [F32, BF16])
@pytest.mark.parametrize("nq,nkv,hd,rot,inter", WRITES)
@pytest.mark.parametrize("page,start", [(4, 6), (24, 99990)])
def test_write_and_read_back(act, nq, nkv, hd, rot, inter, page, start):
    """Queries, codes, scales; a request that goes on at ``start`` and one from 0, odd pages; nothing
    else in the cache changes, and qkv stays."""
    from mstar_b200 import ops

    req, pos = [0] * 7 + [1] * 4, [start + i for i in range(7)] + list(range(4))
    width = (start + 7 + page - 1) // page
    table = torch.full((2, width), -1, dtype=torch.int32)
    ids = [9, 2, 5, 0, 7]
    for k, logical in enumerate(sorted({p // page for p in pos[:7]})):
        table[0, logical] = ids[k]
    table[1, 0] = 11
    g = torch.Generator().manual_seed(3)
    qkv = (torch.randn(11, (nq + 2 * nkv) * hd, generator=g) * 3).to(act).to(DEV)
    codes = torch.full((13, 2, nkv, page, hd), 0x55, dtype=torch.uint8, device=DEV)
    scales = torch.full((13, 2, nkv, page), 99, dtype=torch.uint8, device=DEV)
    before = qkv.clone()
    q = ops.rope_kv8_write(qkv, i32(pos), i32(pos), i32(req), table.to(DEV), freqs(rot), codes.view(torch.float8_e4m3fn),
                           scales, nq, nkv, hd, rot, inter, page)
    assert torch.equal(qkv, before)
    x = before.view(11, nq + 2 * nkv, hd)
    want = rotate64(x[:, :nq], pos, rot, inter)
    # sine and cosine to 2 steps of the rotation's type, two products and a sum, and the last rounding
    size = torch.sqrt((want ** 2).sum(-1, keepdim=True))
    err = (q.view(11, nq, hd).double().cpu() - want).abs()
    assert (err <= HALF[act] * want.abs() + 6 * 2.0 ** -24 * size).all()
    rows = torch.stack([rotate64(x[:, nq:nq + nkv], pos, rot, inter), x[:, nq + nkv:].double().cpu()], 1)
    w_codes, w_scales, w_values = quantise_rows(rows)
    pages = table[req, torch.tensor(pos) // page].long().to(DEV)
    slots = torch.tensor(pos, device=DEV) % page
    got_codes, got_scales = codes[pages, :, :, slots].cpu(), scales[pages, :, :, slots].cpu()
    # values as they came: to the code
    assert torch.equal(got_codes[:, 1], w_codes[:, 1]) and torch.equal(got_scales[:, 1], w_scales[:, 1])
    if act == F32:      # the rotation is double there: no key lies within 2^-24 of a border here
        assert torch.equal(got_codes, w_codes) and torch.equal(got_scales, w_scales)
    else:               # a float rotation: the nearest code but for values next to a border
        assert (got_scales != w_scales).sum() == 0
        off = (values_of(got_codes, got_scales) - rows).abs()
        best = (w_values - rows).abs()
        assert (off <= best + 12 * 2.0 ** -24 * torch.sqrt((rows ** 2).sum(-1, keepdim=True))).all()
    # nothing else
    codes[pages, :, :, slots] = 0x55
    scales[pages, :, :, slots] = 99
    assert (codes == 0x55).all() and (scales == 99).all()


@pytest.mark.parametrize("act", [F32, BF16])
@pytest.mark.parametrize("inter", [False, True])
def test_rotated_keys_get_their_nearest_codes(act, inter):
    """Four million numbers, some of them next to the border of two codes.  The rotation is off by half a step of a
    float of the result (2^-24) and 2^-38 of the two products; what is held is then the nearest code's value: off by half
    a code's step of the exact result, and by that much."""
    from mstar_b200 import ops

    T, nkv, hd, page = 4096, 8, 128, 64
    g = torch.Generator(device=DEV).manual_seed(5)
    qkv = torch.randn(T, (1 + 2 * nkv) * hd, generator=g, device=DEV).to(act)
    pos, at, req = i32(range(90_000, 90_000 + T)), i32(range(T)), i32([0] * T)
    codes = torch.zeros(T // page, 2, nkv, page, hd, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)
    scales = torch.zeros(T // page, 2, nkv, page, dtype=torch.uint8, device=DEV)
    table = i32([list(range(T // page))])
    ops.rope_kv8_write(qkv, pos, at, req, table, freqs(hd), codes, scales, 1, nkv, hd, hd, inter, page)
    got = ops.kv8_read_rows(codes, scales, table, req, at, F32)[:, 0].double()
    x = qkv[:, hd:(1 + nkv) * hd].double().view(T, nkv, hd)
    angle = (pos.double()[:, None] * freqs(hd).double())[:, None]
    lo, hi = (slice(0, hd, 2), slice(1, hd, 2)) if inter else (slice(0, hd // 2), slice(hd // 2, hd))
    want, size = torch.empty_like(x), torch.empty_like(x)
    want[..., lo] = x[..., lo] * angle.cos() - x[..., hi] * angle.sin()
    want[..., hi] = x[..., hi] * angle.cos() + x[..., lo] * angle.sin()
    size[..., lo] = size[..., hi] = x[..., lo].abs() + x[..., hi].abs()
    unit = torch.exp2(scales[:, 0].permute(0, 2, 1).reshape(T, nkv, 1).double() - 127.0)
    step = unit * torch.exp2((want.abs() / unit).clamp(min=2.0 ** -6).log2().floor() - 3)
    off = (got - want).abs() - step / 2
    assert (off <= 2.0 ** -24 * want.abs() + 2.0 ** -38 * size).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("nkv,hd,page", [(2, 64, 16), (3, 24, 7), (1, 256, 64), (8, 128, 1)])
def test_read_rows(dtype, nkv, hd, page):
    """Any order of tokens, the same one twice, places without a page."""
    from mstar_b200 import ops

    c = Case([1, 1, 1], [40, 3, 65], 1 * nkv, nkv, hd, page, BF16, seed=5)
    codes, scales = c.cache()
    req, pos = [2, 0, 0, 1, 2, 2, 0], [64, 39, 39, 0, 0, 17, 5]
    got = ops.kv8_read_rows(codes, scales, c.table.to(DEV), i32(req), i32(pos), dtype)
    at = torch.tensor(pos)
    want = c.values[c.table[req, at // page].long(), :, :, at % page]
    assert got.dtype == dtype and torch.equal(got.double().cpu(), want)
    table = c.table.clone()
    table[0, 39 // page] = -1
    table[2, 0] = 10 ** 6
    got = ops.kv8_read_rows(codes, scales, table.to(DEV), i32(req + [0, 0, 1]), i32(pos + [-1, 10 ** 6, 2]), dtype)
    none = torch.tensor([r in (0, 2) and p // page == (39 // page if r == 0 else 0) for r, p in zip(req, pos)] + [True, True, False])
    assert (got.cpu()[none] == 0).all() and torch.equal(got.double().cpu()[:7][~none[:7]], want[~none[:7]])


def test_rows_at_the_ends_of_the_format():
    """Zeros, the largest and smallest numbers, borders of scales and codes, rows that are not finite."""
    from mstar_b200 import ops

    hd = 16
    rows = torch.zeros(12, hd)
    rows[1] = 448.0
    rows[2, 3] = 448.0 * 2.0 ** -20
    rows[3, 0], rows[3, 1] = math.nextafter(448.0, 0), -1e-3
    rows[4, 0] = torch.nextafter(torch.tensor(448.0), torch.tensor(1e9))
    rows[5] = 3.4e38
    rows[6] = 1e-38
    rows[7, :4] = torch.tensor([1.0, 1.0625, 1.1875, -1.0625])          # halfway between codes at scale 2^-8
    rows[8, 5] = math.nan
    rows[9, 7] = -math.inf
    rows[10, :2] = torch.tensor([448.0, 2.0 ** -10])                    # half the smallest code: to even, zero
    rows[11, :2] = torch.tensor([448.0, 3 * 2.0 ** -11])
    n = rows.shape[0]
    qkv = torch.zeros(n, 3 * hd)
    qkv[:, 2 * hd:] = rows
    codes = torch.zeros(2, 2, 1, 16, hd, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)
    scales = torch.zeros(2, 2, 1, 16, dtype=torch.uint8, device=DEV)
    at = i32(range(n))
    table = i32([[1]])
    ops.rope_kv8_write(qkv.to(DEV), at, at, i32([0] * n), table, None, codes, scales, 1, 1, hd, 0, False, 16)
    w_codes, w_scales, w_values = quantise_rows(rows)
    assert torch.equal(codes.view(torch.uint8)[1, 1, 0, :n].cpu(), w_codes)
    assert torch.equal(scales[1, 1, 0, :n].cpu(), w_scales)
    got = ops.kv8_read_rows(codes, scales, table, i32([0] * n), at, F32)[:, 1, 0].double().cpu()
    assert torch.equal(got.nan_to_num(nan=7.5), w_values.nan_to_num(nan=7.5))
    assert torch.isnan(got[8:10]).all() and (got[5] - 448.0 * 2.0 ** 119).abs().max() == 0


def test_write_leaves_pages_alone_that_are_not_there():
    """Tokens whose table has no page, places past the table or below 0: nothing is written."""
    from mstar_b200 import ops

    nq, nkv, hd, page = 2, 1, 64, 4
    codes = torch.full((3, 2, nkv, page, hd), 0x55, dtype=torch.uint8, device=DEV)
    scales = torch.full((3, 2, nkv, page), 99, dtype=torch.uint8, device=DEV)
    qkv = torch.randn(4, (nq + 2 * nkv) * hd, device=DEV)
    q = ops.rope_kv8_write(qkv, i32([0, 1, 2, 3]), i32([0, 4, 8, -1]), i32([0] * 4), i32([[-1, 3]]), freqs(hd),
                           codes.view(torch.float8_e4m3fn), scales, nq, nkv, hd, hd, False, page)
    assert (codes == 0x55).all() and (scales == 99).all() and torch.isfinite(q).all()


# ------------------------------------------------------------------ attention
SHAPES = [  # nq, nkv, hd, page
    (8, 2, 64, 16), (6, 2, 128, 16), (3, 1, 128, 64), (4, 4, 64, 8), (5, 1, 48, 4), (16, 1, 128, 32), (2, 1, 256, 16),
    (12, 1, 64, 24), (34, 2, 128, 16), (1, 1, 8, 3)]


@pytest.mark.parametrize("act", [F32, BF16])
@pytest.mark.parametrize("nq,nkv,hd,page", SHAPES)
@pytest.mark.parametrize("window,keep", [(0, 0), (21, 0), (70, 3)])
def test_decode(act, nq, nkv, hd, page, window, keep):
    lens = [1, 2, 17, 64, 65, 129, 300]
    c = Case([1] * len(lens), lens, nq, nkv, hd, page, act, seed=nq + hd, window=window, keep=keep)
    c.check(c.decode())


@pytest.mark.parametrize("act", [F32, BF16])
@pytest.mark.parametrize("nq,nkv,hd,page", SHAPES)
@pytest.mark.parametrize("window,keep", [(0, 0), (21, 0), (70, 3)])
def test_portions(act, nq, nkv, hd, page, window, keep):
    """Whole prompts, portions on cached keys, one token, several row tiles."""
    c = Case([1, 5, 40, 70, 2], [1, 5, 140, 70, 300], nq, nkv, hd, page, act, seed=nq + hd + 1, window=window, keep=keep)
    c.check(c.prefill())


@pytest.mark.parametrize("act", [F32, BF16])
@pytest.mark.parametrize("nq,nkv,hd,page", [(6, 2, 128, 4), (3, 1, 64, 5), (140, 1, 64, 16), (130, 1, 128, 7), (9, 3, 256, 1)])
@pytest.mark.parametrize("window,keep", [(0, 0), (40, 2)])
def test_odd_pages_and_many_heads_a_kv_head(act, nq, nkv, hd, page, window, keep):
    """Pages that groups of eight keys cross, and more query heads a kv head than a tile of the portions' kernel has rows."""
    c = Case([1, 1, 1], [1, 67, 300], nq, nkv, hd, page, act, seed=41, window=window, keep=keep)
    c.check(c.decode())
    c = Case([3, 1, 30], [3, 67, 150], nq, nkv, hd, page, act, seed=42, window=window, keep=keep)
    c.check(c.prefill())


@pytest.mark.parametrize("act", [F32, BF16])
@pytest.mark.parametrize("hd", [64, 128])
def test_one_long_request(act, hd):
    """Few rows on many keys: the keys are shared out over blocks and joined."""
    c = Case([1], [3001], 8, 2, hd, 16, act, seed=2)
    c.check(c.decode())
    c = Case([3], [2500], 8, 2, hd, 16, act, seed=3)
    c.check(c.prefill())
    c = Case([3, 30], [1500, 777], 8, 2, hd, 64, act, seed=4, window=900, keep=5)
    c.check(c.prefill())


@pytest.mark.parametrize("hd,window,keep", [(64, 0, 0), (128, 0, 0), (64, 1400, 2)])
def test_few_rows_on_many_keys_side_by_side(hd, window, keep):
    """Portions of one row tile in so many requests that a block walks ten key tiles and more: two at a time."""
    from mstar_b200 import ops
    from mstar_b200.ops.kv8 import kv8_tc_splits

    lens_q, lens_kv = [3] * 19, [3, 4, 60, 128, 129, 256, 257, 1500] + [70] * 11
    assert kv8_tc_splits(8 * 19, 1500, ops.num_sms(), True) == (2, True)
    c = Case(lens_q, lens_kv, 8, 8, hd, 16, BF16, seed=17, window=window, keep=keep)
    c.check(c.prefill(max_len=1500))


@pytest.mark.parametrize("act", [F32, BF16])
@pytest.mark.parametrize("hd", [64, 128])
def test_bounds_only_cut_the_work(act, hd):
    """Looser bounds on the lengths change how the keys are cut, not what comes out beyond rounding."""
    c = Case([1, 1], [130, 700], 4, 1, hd, 16, act, seed=6)
    c.check(c.decode(max_len=20000))
    c.check(c.decode(max_len=1))
    c = Case([20, 33], [130, 700], 4, 1, hd, 16, act, seed=6)
    c.check(c.prefill(max_len=20000, max_q=500))


@pytest.mark.parametrize("act", [F32, BF16])
def test_other_rows_stay(act):
    """Decoded tokens first, then portions, as a step has them: each call writes its own rows only."""
    c = Case([1, 1, 9, 33], [40, 41, 60, 333], 8, 2, 128, 16, act, seed=8)
    out = torch.full((44 + 5, 8 * 128), 3.0, dtype=act, device=DEV)
    q = torch.cat([c.q, torch.zeros(5, 8 * 128, dtype=act)]).to(DEV)
    c.prefill(out=out, q=q, first=2)
    assert (out[:2] == 3).all() and (out[44:] == 3).all()
    want, bound = c.plain()
    assert ((out[2:44].double().cpu() - want[2:]).abs() <= bound[2:]).all()
    part = torch.full_like(out, 3.0)
    c.prefill(out=part, q=q, first=2, entries=1)
    assert (part[:2] == 3).all() and (part[11:] == 3).all() and torch.equal(part[2:11], out[2:11])


@pytest.mark.parametrize("act", [F32, BF16])
@pytest.mark.parametrize("hd", [48, 64, 128])
def test_queries_inside_wider_rows(act, hd):
    """q as a view of a projection's output: rows with a stride, an offset of whole 16 bytes."""
    c = Case([1, 1, 1], [5, 70, 200], 4, 2, hd, 16, act, seed=9)
    wide = torch.full((3, 8 * hd + 16), math.nan, dtype=act, device=DEV)
    wide[:, 8:8 + 4 * hd] = c.q.to(DEV)
    assert torch.equal(c.decode(q=wide[:, 8:8 + 4 * hd]), c.decode())
    odd = torch.full((3, 4 * hd + 3), math.nan, dtype=act, device=DEV)
    odd[:, 1:1 + 4 * hd] = c.q.to(DEV)
    c.check(c.decode(q=odd[:, 1:1 + 4 * hd]))
    c = Case([3, 1, 12], [5, 70, 200], 4, 2, hd, 16, act, seed=9)
    odd = torch.full((16, 4 * hd + 3), math.nan, dtype=act, device=DEV)
    odd[:, 1:1 + 4 * hd] = c.q.to(DEV)
    c.check(c.prefill(q=odd[:, 1:1 + 4 * hd]))


@pytest.mark.parametrize("act", [F32, BF16])
@pytest.mark.parametrize("hd", [48, 64, 128])
def test_rows_that_are_not_finite_reach_only_who_sees_them(act, hd):
    """A bad key and a bad value in the middle of a portion: the tokens before them keep finite outputs, the
    tokens that see them give NaNs."""
    c = Case([40], [100], 4, 2, hd, 16, act, seed=10)
    codes, scales = c.cache()
    clean = c.prefill()
    for plane, place in ((0, 75), (1, 80)):
        s2, c2 = scales.clone(), codes.view(torch.uint8).clone()
        page = c.table[0, place // 16]
        s2[page, plane, 1, place % 16] = 255
        c2[page, plane, 1, place % 16] = 0
        out = c.prefill(cache=(c2.view(torch.float8_e4m3fn), s2)).view(40, 4, hd)
        row = place - 60
        assert torch.equal(out[:, :2], clean.view(40, 4, hd)[:, :2])          # the other kv head's queries
        assert torch.equal(out[:row, 2:], clean.view(40, 4, hd)[:row, 2:])
        assert torch.isnan(out[row:, 2:]).all()
        one = Case([1, 1], [place, 100], 4, 2, hd, 16, act, seed=10)
        one.table = torch.cat([c.table, c.table])
        got = one.decode(q=c.q[:2].to(DEV).contiguous(), cache=(c2.view(torch.float8_e4m3fn), s2)).view(2, 4, hd)
        assert torch.isfinite(got[0]).all() and torch.isnan(got[1, 2:]).all() and torch.isfinite(got[1, :2]).all()
    q = c.q.clone().to(DEV)
    q[7, :hd] = math.nan
    q[9, :hd] = math.inf
    out = c.prefill(q=q).view(40, 4, hd)
    assert torch.isnan(out[7, 0]).all() and torch.isnan(out[9, 0]).any()
    keep = torch.ones(40, 4, dtype=torch.bool)
    keep[7, 0] = keep[9, 0] = False
    assert torch.equal(out.cpu()[keep], clean.view(40, 4, hd).cpu()[keep])


@pytest.mark.parametrize("act", [F32, BF16])
@pytest.mark.parametrize("hd", [48, 128])
def test_rows_without_keys_and_sizes_far_apart(act, hd):
    """A place below 0 gives zeros; values of very different sizes and large scores stay exact enough."""
    c = Case([1, 1], [30, 30], 4, 2, hd, 16, act, seed=11)
    codes, scales = c.cache()
    from mstar_b200 import ops

    out = torch.full((2, 4 * hd), 7.0, dtype=act, device=DEV)
    ops.paged_decode_attention_kv8(c.q.to(DEV), out, codes, scales, c.table.to(DEV), i32([0, 1]), i32([-1, 29]), 2, 4, 2,
                                   hd, 16, 0, 0, c.scale, 30)
    assert (out[0] == 0).all() and torch.isfinite(out[1]).all()
    # more tokens than keys: the first have none
    out = torch.full((2, 4 * hd), 7.0, dtype=act, device=DEV)
    ops.paged_prefill_attention_kv8(c.q.to(DEV), out, codes, scales, c.table.to(DEV), i32([0, 2]), i32([1]), 0, 1, 2, 4, 2,
                                    hd, 16, 0, 0, c.scale, 30)
    assert (out[0] == 0).all() and torch.isfinite(out[1]).all() and (out[1] != 7).any()
    for lens_q in ([1, 1, 1], [4, 20, 30]):
        c = Case(lens_q, [40, 90, 200], 4, 2, hd, 16, act, seed=12, q_scale=6.0)
        g = torch.Generator().manual_seed(1)
        c.scales[:, 1] = (c.scales[:, 1].int() + torch.randint(-60, 60, c.scales[:, 1].shape, generator=g)).to(torch.uint8)
        c.values = values_of(c.codes, c.scales)
        c.check(c.decode() if max(lens_q) == 1 else c.prefill())


@pytest.mark.parametrize("act", [F32, BF16])
def test_bad_pages_read_inside_the_cache(act):
    """A table whose seen entries are -1 or far out: some page of the cache is read, nothing else."""
    for lens_q in ([1, 1], [9, 40]):
        c = Case(lens_q, [50, 90], 4, 2, 128, 16, act, seed=13)
        c.table[0, 1], c.table[1, 2], c.table[1, 0] = -1, 2 ** 31 - 1, -2 ** 31
        got = c.decode() if max(lens_q) == 1 else c.prefill()
        assert torch.isfinite(got).all()


@pytest.mark.parametrize("act", [F32, BF16])
def test_another_stream_and_graphs(act):
    """The operators together as a step has them, on a stream of their own and captured: two graphs of
    different sizes replayed in turn while lengths move on the device, and an eager call between."""
    from mstar_b200 import ops

    nq, nkv, hd, page = 8, 2, 128, 16
    c = Case([1, 1, 1], [200, 33, 7], nq, nkv, hd, page, act, seed=14)
    qkv = (torch.randn(3, (nq + 2 * nkv) * hd, generator=torch.Generator().manual_seed(2)) * 2).to(act).to(DEV)
    table, freq = c.table.to(DEV), freqs(hd)

    def step(codes, scales, pos, req, n):
        q = ops.rope_kv8_write(qkv[:n], pos, pos, req, table, freq, codes, scales, nq, nkv, hd, hd, False, page)
        out = torch.empty_like(q)
        ops.paged_decode_attention_kv8(q, out, codes, scales, table, req, pos, n, nq, nkv, hd, page, 0, 0, c.scale, 256)
        return out, ops.kv8_read_rows(codes, scales, table, req, pos, act)

    want = []
    for n, pos in ((3, [199, 32, 6]), (2, [150, 20]), (3, [180, 31, 0])):
        codes, scales = c.cache()
        want.append(step(codes, scales, i32(pos), i32([0, 1, 2][:n]), n))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        codes, scales = c.cache()
        got = step(codes, scales, i32([199, 32, 6]), i32([0, 1, 2]), 3)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want[0]))
    codes, scales = c.cache()
    fresh, fresh_s = codes.view(torch.uint8).clone(), scales.clone()
    graphs = []
    for n in (3, 2):
        pos, req = i32([0] * n), i32([0, 1, 2][:n])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(codes, scales, pos, req, n)
        graphs.append((graph, pos, out, req))      # (a graph reads its inputs where they were)
    for turn in range(2):
        for k, (which, pos) in enumerate(((0, [199, 32, 6]), (1, [150, 20]), (0, [180, 31, 0]))):
            graph, at, out, _ = graphs[which]
            codes.view(torch.uint8).copy_(fresh)
            scales.copy_(fresh_s)
            at.copy_(i32(pos))
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want[k]))


@pytest.mark.parametrize("act", [F32, BF16])
def test_the_same_call_twice_gives_the_same_bits(act):
    c = Case([1, 1], [2000, 900], 8, 2, 128, 16, act, seed=15)
    assert torch.equal(c.decode(), c.decode())
    c = Case([30, 90], [2000, 900], 8, 2, 128, 16, act, seed=16)
    assert torch.equal(c.prefill(), c.prefill())


@pytest.mark.parametrize("act", [F32, BF16])
@pytest.mark.parametrize("hd", [48, 64, 128])
def test_tables_that_are_part_of_wider_ones(act, hd):
    """A view of some columns: what lies beside them belongs to somebody else, and is neither written nor read."""
    from mstar_b200 import ops

    nq, nkv, page = 4, 2, 16
    c = Case([1, 1, 20], [30, 47, 60], nq, nkv, hd, page, act, seed=31)
    wide = torch.full((3, c.table.shape[1] + 3), 0, dtype=torch.int32)
    wide[:, 2:-1] = c.table
    view = wide.to(DEV)[:, 2:-1]
    codes, scales = c.cache()
    out = torch.full((22, nq * hd), 7.0, dtype=act, device=DEV)
    q = c.q.to(DEV)
    ops.paged_decode_attention_kv8(q, out, codes, scales, view, c.i32(c.req), c.i32(c.pos), 2, nq, nkv, hd, page, 0, 0,
                                   c.scale, 60)
    ops.paged_prefill_attention_kv8(q, out, codes, scales, view, c.i32(c.indptr), c.i32(c.lens_kv), 2, 1, 20, nq, nkv, hd,
                                    page, 0, 0, c.scale, 60)
    c.check(out)
    # places behind the view's last page: its neighbour in the wide table names page 0
    before = codes.view(torch.uint8).clone(), scales.clone()
    past = view.shape[1] * page
    ops.rope_kv8_write(torch.randn(2, (nq + 2 * nkv) * hd, device=DEV).to(act), i32([0, 1]), i32([past, past + 1]), i32([0, 2]),
                       view, None, codes, scales, nq, nkv, hd, 0, False, page)
    assert torch.equal(codes.view(torch.uint8), before[0]) and torch.equal(scales, before[1])
    assert not ops.kv8_read_rows(codes, scales, view, i32([0, 2]), i32([past, past + 1]), act).any()


@pytest.mark.parametrize("act", [F32, BF16])
@pytest.mark.parametrize("hd", [48, 64, 128])
@pytest.mark.parametrize("max_q", [1, 30])
def test_portions_longer_than_their_bound_stay_inside_the_parts(monkeypatch, act, hd, max_q):
    """``max_q_len`` below the tokens that an entry has: those beyond are not computed, and nothing is written behind
    the memory for the parts or into other rows."""
    from mstar_b200 import ops
    from mstar_b200.ops import kv8

    made = []

    def parts(q, tokens, heads, dim, splits):
        assert splits > 1
        n = tokens * heads * splits
        t = torch.full((n * (dim + 2) + 500_000,), 7.0, dtype=F32, device=DEV)
        made.append((t, n * (dim + 2)))
        return t, t.data_ptr(), t.data_ptr() + 4 * n * dim

    c = Case([40, 40], [900, 800], 4, 1, hd, 16, act, seed=33)
    monkeypatch.setattr(kv8, "_parts", parts)
    out = torch.full((80 + 3, 4 * hd), 3.0, dtype=act, device=DEV)
    q = torch.cat([c.q, torch.zeros(3, 4 * hd, dtype=act)]).to(DEV)
    c.prefill(out=out, q=q, max_q=max_q)
    torch.cuda.synchronize()
    assert made and all((t[n:] == 7).all() for t, n in made)
    assert (out[80:] == 3).all()
    want, bound = c.plain()
    good = (out[:max_q].double().cpu() - want[:max_q]).abs() <= bound[:max_q]
    assert good.all()


@pytest.mark.parametrize("act", [F32, BF16])
@pytest.mark.parametrize("hd,page", [(128, 64), (48, 64), (256, 4)])
def test_pages_more_than_four_gigabytes_apart(act, hd, page):
    """The same rows on the first and on the last pages of a cache of 4.5 GB: written, read back and attended to alike."""
    from mstar_b200 import ops

    nq, nkv, n, width = 8, 4, 130, -(-130 // page)
    pages = int(4.5e9) // (2 * nkv * page * hd)
    codes = torch.zeros(pages, 2, nkv, page, hd, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)
    scales = torch.zeros(pages, 2, nkv, page, dtype=torch.uint8, device=DEV)
    table = i32([list(range(width)), list(range(pages - width, pages))])
    assert int(table[1, 0]) * 2 * nkv * page * hd > 2 ** 32
    g = torch.Generator(device=DEV).manual_seed(3)
    qkv = torch.randn(n, (nq + 2 * nkv) * hd, generator=g, device=DEV).to(act)
    pos, rows, got = i32(range(n)), [], []
    for r in range(2):
        q = ops.rope_kv8_write(qkv, pos, pos, i32([r] * n), table, freqs(hd), codes, scales, nq, nkv, hd, hd, False, page)
        rows.append(ops.kv8_read_rows(codes, scales, table, i32([r] * n), pos, act))
        one, all_ = torch.empty(1, nq * hd, dtype=act, device=DEV), torch.empty(n, nq * hd, dtype=act, device=DEV)
        ops.paged_decode_attention_kv8(q[-1:], one, codes, scales, table, i32([r]), pos[-1:], 1, nq, nkv, hd, page, 0, 0,
                                       hd ** -0.5, n)
        ops.paged_prefill_attention_kv8(q, all_, codes, scales, table[r:r + 1], i32([0, n]), i32([n]), 0, 1, n, nq, nkv, hd,
                                        page, 0, 0, hd ** -0.5, n)
        got.append((one, all_))
    assert rows[0].abs().max() > 1 and torch.equal(*rows)
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
    assert torch.isfinite(got[0][1]).all()


def test_nothing_to_do():
    from mstar_b200 import ops

    c = Case([1], [5], 4, 2, 64, 16, F32)
    codes, scales = c.cache()
    none = torch.empty(0, dtype=torch.int32, device=DEV)
    assert ops.rope_kv8_write(torch.empty(0, 512, device=DEV), none, none, none, c.table.to(DEV), freqs(64), codes, scales,
                              4, 2, 64, 64, False, 16).shape == (0, 256)
    assert ops.kv8_read_rows(codes, scales, c.table.to(DEV), none, none, F32).shape == (0, 2, 2, 64)
    out = torch.full((3, 256), 3.0, device=DEV)
    ops.paged_decode_attention_kv8(out.clone(), out, codes, scales, c.table.to(DEV), none, none, 0, 4, 2, 64, 16, 0, 0, 1.0, 1)
    ops.paged_prefill_attention_kv8(out.clone(), out, codes, scales, c.table.to(DEV), i32([0]), none, 0, 0, 0, 4, 2, 64, 16,
                                    0, 0, 1.0, 1)
    assert (out == 3).all()


# ------------------------------------------------------------------ the engine on it
def test_engine_steps(model_folders, monkeypatch):
    """Steps cut three ways on an 8-bit cache, float, against the plain model whose attention gets its keys
    and values rounded to the cache's format.  A key next to a border may take the other code (1/16 of its
    value): of a row's 16 to 32 features one, which moves an attention output by at most 1/16 of one feature
    and a logit by some 1e-3; a wrong row moves logits by tenths."""
    from mstar_b200.engine.model import load_model
    from mstar_b200.engine.step import StepEntry, make_stepper

    real = P.plain_attention

    def rounded(q, k, v, **kw):
        return real(q, quantise_rows(k)[2], quantise_rows(v)[2], **kw)

    for name in ("tiny_a", "tiny_b"):
        folder, raw, tensors = model_folders[name]
        ids = torch.randint(0, raw["vocab_size"], (45,), generator=torch.Generator().manual_seed(4)).tolist()
        exact = P.plain_logits(tensors, raw, ids)
        monkeypatch.setattr(P, "plain_attention", rounded)
        want = P.plain_logits(tensors, raw, ids)
        monkeypatch.setattr(P, "plain_attention", real)
        moved = float((want - exact).abs().max())
        model = load_model(folder, dtype="float32")
        for cuts in ([45], [1] * 45, [30, 1, 1, 9, 1, 3]):
            st = make_stepper(model, page_size=8, max_tokens=256, kv_cache_dtype="float8_e4m3")
            st.add_request("r")
            got, at = [], 0
            for n in cuts:
                got.append(st.step([StepEntry("r", ids[at:at + n], range(n))]).double().cpu().clone())
                at += n
            err = (torch.cat(got) - want).abs()
            assert err.max() < 5e-3 and err.mean() < 2e-4, (float(err.max()), float(err.mean()))
        assert moved > 1e-2                     # the rounding itself shows


def test_engine_generates_and_sizes_its_pool(model_folders):
    """Several requests together against each alone, in both types; twice the pages of bfloat16, nearly."""
    from mstar_b200 import LLM, SamplingParams

    folder, raw, _ = model_folders["tiny_b"]
    prompts = [torch.randint(0, raw["vocab_size"], (n,), generator=torch.Generator().manual_seed(n)).tolist()
               for n in (3, 50, 17)]
    for dtype in ("float32", "bfloat16"):
        llm = LLM(str(folder), dtype=dtype, page_size=16, max_num_pages=64, kv_cache_dtype="float8_e4m3")
        assert llm.stepper.storage.kv[0].dtype == torch.float8_e4m3fn
        p = SamplingParams(temperature=0.0, max_output_tokens=12, ignore_eos=True)
        together = [r.token_ids for r in llm.generate(prompts, p)]
        assert llm.stepper.graph_replays > 0
        if dtype == "float32":
            assert together == [llm.generate(q, p).token_ids for q in prompts]
        assert all(len(t) == 12 for t in together)
    pages = [LLM(str(folder), dtype="bfloat16", page_size=16, kv_cache_memory_fraction=0.02, kv_cache_dtype=t
                 ).stepper.storage.group_configs[0].num_pages for t in ("auto", "float8_e4m3")]
    assert 1.7 < pages[1] / pages[0] < 2.0


def test_engine_keeps_first_keys_beside_a_window():
    """A windowed layer with kept first keys, whose 16-bit cache has another path, on the 8-bit one: portions
    and single tokens give what one portion gives."""
    from mstar_b200.config.layout import AttentionSpec, PositionSpec
    from mstar_b200.cache.storage import CacheStorage
    from mstar_b200.parts.base import Runtime, StepContext
    from mstar_b200.parts.registry import build_part, part_class

    spec = AttentionSpec(hidden_size=96, num_heads=4, num_kv_heads=2, head_dim=64, window=20, keep_first=3,
                         position=PositionSpec(head_dim=64, rotary_dim=64))
    g = torch.Generator().manual_seed(1)
    params = {n: (torch.randn(s.shape, generator=g) * s.shape[-1] ** -0.5).to(DEV)
              for n, s in part_class("mixer", spec).param_specs(spec).items()}
    part = build_part("mixer", spec, params, Runtime(F32, torch.device(DEV)))
    x = torch.randn(60, 96, generator=g).to(DEV)
    outs = []
    for cuts in ([60], [30, 1, 1, 20, 8], [1] * 60):
        st = CacheStorage([part.cache_need(spec)], F32, torch.device(DEV), 8, 16, 2, "float8_e4m3")
        st.manager.add_request("r")
        got, at = [], 0
        for n in cuts:
            st.manager.reserve(["r"], [n])
            b = st.manager.fill_batch(["r"], [n])
            one = 1 if n == 1 else 0
            ctx = StepContext(n, 1, i32(b.token_req), i32(b.positions), i32(b.cache_pos), i32(b.qo_indptr), i32(b.kv_len),
                              i32(b.slots), q_lens=[n], kv_lens=b.kv_len.tolist(), max_q_len=n,
                              max_kv_len=int(b.kv_len.max()), num_decode=one)
            got.append(part.forward(x[at:at + n], ctx, st.layer_cache(0, [i32(b.tables[0]).view(1, -1)])))
            st.manager.commit("r", n)
            at += n
        outs.append(torch.cat(got))
    # float throughout; a key at a code's border may fall the other way between cuts (see above)
    for o in outs[1:]:
        assert (o - outs[0]).abs().max() < 2e-2 and (o - outs[0]).abs().mean() < 1e-4
