"""Calls of the 8-bit cache's operators that the larger tests do not make."""
import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

from kv8_util import HALF, Case

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F32, BF16 = torch.float32, torch.bfloat16


def i32(v):
    return torch.as_tensor(v, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("act", [F32, BF16])
def test_modes_see_what_the_operators_allocate(act):
    """Outputs and the memory for parts come by torch's dispatcher, so that a mode around the calls sees them."""
    from mstar_b200 import ops

    class Sizes(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            out = func(*args, **(kwargs or {}))
            if isinstance(out, torch.Tensor):
                seen.append((tuple(out.shape), out.dtype))
            return out

    seen: list = []
    c = Case([3], [1500], 4, 2, 128, 16, act, seed=1)
    codes, scales = c.cache()
    qkv, pos, req, table = torch.randn(3, 8 * 128, device=DEV).to(act), i32([0, 1, 2]), i32([0] * 3), c.table.to(DEV)
    with Sizes():
        ops.rope_kv8_write(qkv, pos, pos, req, table, None, codes, scales, 4, 2, 128, 0, False, 16)
        assert seen.pop() == ((3, 4 * 128), act)
        ops.kv8_read_rows(codes, scales, table, req, pos, act)
        assert seen.pop() == ((3, 2, 2, 128), act)
        c.prefill()
    assert any(dtype == F32 and len(shape) == 1 and shape[0] >= 3 * 4 * 130 * 2 for shape, dtype in seen)


@pytest.mark.parametrize("act", [F32, BF16])
@pytest.mark.parametrize("hd", [48, 64, 128, 256])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 4, 2 ** 30])
def test_the_largest_windows_hide_nothing(act, hd, window):
    """More new tokens than keys (the first stand below place 0) under a window that no place passes: as without one."""
    for lens_q, lens_kv in (([9, 70], [3, 40]), ([40], [38])):
        c = Case([1] * len(lens_q), lens_kv, 4, 2, hd, 16, act, seed=2)
        tokens = sum(lens_q)
        c.q = torch.randn(tokens, 4 * hd, generator=torch.Generator().manual_seed(3)).to(act)
        c.lens_q, c.req, c.indptr = lens_q, [0] * tokens, [0] + [sum(lens_q[:r + 1]) for r in range(len(lens_q))]
        want = c.prefill()
        assert (want[:lens_q[0] - lens_kv[0]] == 0).all() and (want[lens_q[0] - 1] != 0).all()
        c.window, c.keep = window, 0
        assert torch.equal(c.prefill(), want)
        c.keep = 5
        assert torch.equal(c.prefill(), want)


@pytest.mark.parametrize("act", [F32, BF16])
@pytest.mark.parametrize("hd", [48, 64, 128, 256])
@pytest.mark.parametrize("scale", [2.0 ** -126, 1e-30, 1e-12])
def test_scales_next_to_zero_give_means(act, hd, scale):
    """All visible keys weigh the same, for zeros as for ordinary queries: sums of n <= 90 terms, each rounded once or twice."""
    for lens_q, lens_kv in (([1, 1], [3, 90]), ([3, 40], [3, 90])):
        c = Case(lens_q, lens_kv, 4, 2, hd, 16, act, seed=4)
        c.scale = scale
        c.q[::2] = 0
        got = (c.decode() if max(lens_q) == 1 else c.prefill()).double().cpu().view(len(c.req), 4, hd)
        for t, (r, p) in enumerate(zip(c.req, c.pos)):
            at = torch.arange(p + 1)
            v = c.values[c.table[r].long()[at // 16], 1, :, at % 16].repeat_interleave(2, dim=1)      # [keys, heads, hd]
            bound = HALF[act] * v.mean(0).abs() + (2.0 ** -17 + 2.0 ** -8 * (act == BF16)) * v.abs().mean(0)
            assert ((got[t] - v.mean(0)).abs() <= bound).all()


@pytest.mark.parametrize("act", [F32, BF16])
@pytest.mark.parametrize("nkv,hd,rot,inter", [(4, 128, 64, False), (4, 128, 32, True), (8, 64, 16, False), (3, 24, 12, False),
                                              (2, 200, 72, False), (2, 48, 48, True), (2, 48, 40, False), (2, 256, 128, False),
                                              (5, 8, 2, True)])
@pytest.mark.parametrize("shift", [0, 1])
def test_partly_rotated_and_odd_keys_get_their_nearest_codes(act, nkv, hd, rot, inter, shift):
    """A million numbers each, on the path of whole runs and on the scalar one (odd sizes, rows off 16 bytes): the rotation is
    off by half a step of a float (2^-24) and 2^-38 of its two products, and the angle by less than 2^-52 of itself, so that what is held is off by half a code's
    step of the exact result and by that much.  Numbers that are not turned have their nearest codes."""
    from mstar_b200 import ops

    T, page = max(1024, 2 ** 20 // (nkv * hd)), 16
    g = torch.Generator(device=DEV).manual_seed(hd + rot)
    width = (1 + 2 * nkv) * hd
    wide = torch.randn(T, width + 8, generator=g, device=DEV).to(act)
    qkv = wide[:, shift:shift + width]
    freq = torch.tensor([10000.0 ** (-2.0 * j / rot) for j in range(rot // 2)], dtype=F32, device=DEV)
    pos, at, req = i32(range(70_000, 70_000 + T)), i32(range(T)), i32([0] * T)
    pages = -(-T // page)
    codes = torch.zeros(pages, 2, nkv, page, hd, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)
    scales = torch.zeros(pages, 2, nkv, page, dtype=torch.uint8, device=DEV)
    table = i32([list(range(pages))])
    q = ops.rope_kv8_write(qkv, pos, at, req, table, freq, codes, scales, 1, nkv, hd, rot, inter, page)
    got = ops.kv8_read_rows(codes, scales, table, req, at, F32)[:, 0].double()
    x = qkv[:, :(1 + nkv) * hd].double().view(T, 1 + nkv, hd)
    angle = (pos.double()[:, None] * freq.double())[:, None]
    lo, hi = (slice(0, rot, 2), slice(1, rot, 2)) if inter else (slice(0, rot // 2), slice(rot // 2, rot))
    want, size = x.clone(), torch.zeros_like(x)
    want[..., lo] = x[..., lo] * angle.cos() - x[..., hi] * angle.sin()
    want[..., hi] = x[..., hi] * angle.cos() + x[..., lo] * angle.sin()
    size[..., lo] = size[..., hi] = x[..., lo].abs() + x[..., hi].abs()
    # (the angle, exact in double, becomes half-turns by a product with 1 / pi in double: the constant is off by 2^-54 of
    # itself and the product by 2^-53, together less than angle * 2^-52, which at 73,000 is 2^-35.8 of the two products)
    near = 2.0 ** -24 * want.abs() * (size > 0) + (2.0 ** -38 + 75_000 * 2.0 ** -52) * size
    err = (q.double() - want[:, 0]).abs()
    assert (err <= HALF[act] * want[:, 0].abs() + near[:, 0]).all()
    unit = torch.exp2(scales[:, 0].permute(0, 2, 1).reshape(-1, nkv, 1)[:T].double() - 127.0)
    want, near = want[:, 1:], near[:, 1:]
    step = unit * torch.exp2((want.abs() / unit).clamp(min=2.0 ** -6).log2().floor() - 3)
    assert ((got - want).abs() - step / 2 <= near).all()
