"""The 8-bit cache away from the GPU: its format, its storage, what its operators refuse."""
import dataclasses

import pytest
import torch

from kv8_util import E4M3, quantise_rows, scale_exponent, values_of
from mstar_b200 import ops
from mstar_b200.cache.storage import CacheStorage, bytes_per_page, plan_groups
from mstar_b200.config.layout import AttentionSpec, PositionSpec
from mstar_b200.parts.attention import Attention
from mstar_b200.parts.base import CacheNeed, KVNeed, StateNeed

POS = PositionSpec(head_dim=64, rotary_dim=64)
PLAIN = AttentionSpec(hidden_size=256, num_heads=4, num_kv_heads=2, head_dim=64, position=POS)


def test_plain_format():
    """The tests' own rounding against torch's cast, and the scale at the borders of its binades."""
    x = torch.randn(50, 32, generator=torch.Generator().manual_seed(1)) * 10
    codes, scales, values = quantise_rows(x)
    again = (x.double() * torch.exp2(127.0 - scales.double())[:, None]).float().to(torch.float8_e4m3fn)
    assert torch.equal(again.view(torch.uint8), codes) and torch.equal(values_of(codes, scales), values)
    assert (values - x.double()).abs().max() <= (x.abs() * 2.0 ** -4).max()
    assert [scale_exponent(v) for v in (448.0, 449.0, 224.0, 0.0, 1e-40, 3e38)] == [0, 1, -1, -100, -100, 119]
    assert torch.isnan(E4M3[[0x7f, 0xff]]).all() and E4M3[0x7e] == 448


def test_storage_holds_codes_and_scales():
    needs = [Attention.cache_need(PLAIN), Attention.cache_need(dataclasses.replace(PLAIN, window=8, keep_first=2))]
    st = CacheStorage(needs, torch.bfloat16, torch.device("cpu"), 16, [3, 5], 2, "float8_e4m3")
    assert [tuple(t.shape) for t in st.kv] == [(4, 2, 2, 16, 64), (6, 2, 2, 16, 64)]
    assert all(t.dtype == torch.float8_e4m3fn for t in st.kv)
    assert [tuple(t.shape) for t in st.kv_scales] == [(4, 2, 2, 16), (6, 2, 2, 16)]
    tables = [torch.zeros(1, 1, dtype=torch.int32)] * 2
    assert st.layer_cache(1, tables).kv_scales is st.kv_scales[1]
    _, group_of = plan_groups(needs)
    assert bytes_per_page(needs, group_of, 0, 16, torch.bfloat16, "float8_e4m3") == 2 * 2 * 16 * 65
    assert bytes_per_page(needs, group_of, 0, 16, torch.bfloat16, "auto") == 2 * 2 * 16 * 64 * 2
    plain = CacheStorage(needs, torch.bfloat16, torch.device("cpu"), 16, [3, 5], 2)
    assert plain.kv_scales == [None, None] and plain.layer_cache(0, tables).kv_scales is None


def test_storage_refuses_what_it_cannot_hold():
    dev = torch.device("cpu")
    capped = Attention.cache_need(dataclasses.replace(PLAIN, softcap=30.0))
    for needs in ([Attention.cache_need(PLAIN), capped], [CacheNeed(kv=KVNeed(1, 64, planes=1))],
                  [CacheNeed(state=StateNeed((4,)))], []):
        with pytest.raises(ValueError, match="kv_cache_dtype"):
            CacheStorage(needs, torch.bfloat16, dev, 16, 4, 2, "float8_e4m3")
    with pytest.raises(ValueError, match="not known"):
        CacheStorage([Attention.cache_need(PLAIN)], torch.bfloat16, dev, 16, 4, 2, "int3")
    assert not dataclasses.replace(PLAIN, bias=True).eight_bit and PLAIN.eight_bit


def args(name, **changes):
    """Arguments of an operator that only lack a GPU, with some replaced."""
    T, nq, nkv, hd, page, pages = 3, 4, 2, 64, 16, 5
    i32 = lambda *shape: torch.zeros(*shape, dtype=torch.int32)  # noqa: E731
    common = dict(kv_cache=torch.zeros(pages, 2, nkv, page, hd, dtype=torch.uint8).view(torch.float8_e4m3fn),
                  kv_scales=torch.zeros(pages, 2, nkv, page, dtype=torch.uint8), block_table=i32(2, 4), num_heads=nq,
                  num_kv_heads=nkv, head_dim=hd, page_size=page)
    own = {
        "rope_kv8_write": dict(qkv=torch.zeros(T, (nq + 2 * nkv) * hd), positions=i32(T), cache_pos=i32(T), token_req=i32(T),
                               inv_freq=torch.ones(hd // 2), rotary_dim=hd, interleaved=False),
        "kv8_read_rows": dict(token_req=i32(T), cache_pos=i32(T), dtype=torch.float32),
        "paged_decode_attention_kv8": dict(q=torch.zeros(T, nq * hd), out=torch.zeros(T, nq * hd), token_req=i32(T),
                                           cache_pos=i32(T), tokens=T, window=0, keep_first=0, scale=0.125, max_len=10),
        "paged_prefill_attention_kv8": dict(q=torch.zeros(T, nq * hd), out=torch.zeros(T, nq * hd), qo_indptr=i32(3),
                                            kv_len=i32(2), first_entry=0, entries=2, max_q_len=2, window=0, keep_first=0,
                                            scale=0.125, max_kv_len=10),
    }[name]
    if name == "kv8_read_rows":
        for k in ("num_heads", "num_kv_heads", "head_dim", "page_size"):
            common.pop(k)
    return {**common, **own, **changes}


F8 = torch.float8_e4m3fn
Z = torch.zeros
REFUSALS = [
    ("rope_kv8_write", dict(qkv=Z(3, 500)), "qkv"),
    ("rope_kv8_write", dict(qkv=Z(3, 512, dtype=torch.float16)), "dtype"),
    ("rope_kv8_write", dict(qkv=Z(512, 3).t()), "without gaps"),
    ("rope_kv8_write", dict(rotary_dim=63), "rotary_dim"),
    ("rope_kv8_write", dict(rotary_dim=66), "rotary_dim"),
    ("rope_kv8_write", dict(inv_freq=None), "inv_freq"),
    ("rope_kv8_write", dict(inv_freq=torch.ones(31)), "inv_freq"),
    ("rope_kv8_write", dict(kv_cache=Z(5, 2, 2, 16, 64, dtype=torch.bfloat16)), "codes"),
    ("rope_kv8_write", dict(kv_scales=Z(5, 2, 2, 8, dtype=torch.uint8)), "scales"),
    ("rope_kv8_write", dict(page_size=8), "shape"),
    ("rope_kv8_write", dict(positions=Z(3, dtype=torch.int64)), "index arrays"),
    ("rope_kv8_write", dict(cache_pos=Z(2, dtype=torch.int32)), "index arrays"),
    ("rope_kv8_write", dict(token_req=Z(6, dtype=torch.int32)[::2]), "index arrays"),
    ("rope_kv8_write", dict(block_table=Z(4, dtype=torch.int32)), "block table"),
    ("rope_kv8_write", {}, "CUDA"),
    ("kv8_read_rows", dict(dtype=torch.float16), "float32 or bfloat16"),
    ("kv8_read_rows", dict(kv_cache=Z(5, 2, 16, 64, dtype=torch.uint8).view(F8)), "shape"),
    ("kv8_read_rows", dict(cache_pos=Z(2, dtype=torch.int32)), "index arrays"),
    ("kv8_read_rows", {}, "CUDA"),
    ("paged_decode_attention_kv8", dict(num_heads=3), "multiple"),
    ("paged_decode_attention_kv8", dict(q=Z(2, 256)), "q "),
    ("paged_decode_attention_kv8", dict(q=Z(3, 200)), "q "),
    ("paged_decode_attention_kv8", dict(out=Z(3, 256, dtype=torch.bfloat16)), "out"),
    ("paged_decode_attention_kv8", dict(out=Z(3, 512)[:, :256]), "out"),
    ("paged_decode_attention_kv8", dict(window=-1), "negative"),
    ("paged_decode_attention_kv8", dict(keep_first=-1), "negative"),
    ("paged_decode_attention_kv8", dict(scale=0.0), "scale"),
    ("paged_decode_attention_kv8", dict(scale=float("nan")), "scale"),
    ("paged_decode_attention_kv8", dict(cache_pos=Z(2, dtype=torch.int32)), "index arrays"),
    ("paged_decode_attention_kv8", dict(head_dim=32), "q|shape|out"),
    ("paged_decode_attention_kv8", {}, "CUDA"),
    ("paged_prefill_attention_kv8", dict(first_entry=-1), "first_entry"),
    ("paged_prefill_attention_kv8", dict(entries=3), "block table"),
    ("paged_prefill_attention_kv8", dict(qo_indptr=Z(2, dtype=torch.int32)), "index arrays"),
    ("paged_prefill_attention_kv8", dict(kv_len=Z(2, dtype=torch.int64)), "index arrays"),
    ("paged_prefill_attention_kv8", dict(q=Z(2, 256)), "row"),
    ("paged_prefill_attention_kv8", {}, "CUDA"),
]


@pytest.mark.parametrize("name,changes,match", REFUSALS, ids=[f"{n}-{'-'.join(c) or 'cpu'}-{i}"
                                                             for i, (n, c, _) in enumerate(REFUSALS)])
def test_refusals(name, changes, match):
    with pytest.raises(ops.KernelError, match=match):
        getattr(ops, name)(**args(name, **changes))


@pytest.mark.parametrize("name", ["paged_decode_attention_kv8", "paged_prefill_attention_kv8"])
def test_refuses_outputs_off_the_boundary_and_tables_without_pages(name):
    out = Z(3 * 256 + 1)[1:].view(3, 256)
    with pytest.raises(ops.KernelError, match="16-byte"):
        getattr(ops, name)(**args(name, out=out))
    with pytest.raises(ops.KernelError, match="no pages"):
        getattr(ops, name)(**args(name, block_table=Z(2, 0, dtype=torch.int32)))


def test_shapes_of_the_decode_kernel():
    """Blocks of a pair times pairs fit the GPU at once wherever some shape does, and no warp is without a tile."""
    from mstar_b200.ops.kv8 import kv8_decode_shape

    for hd in (64, 128, 256):
        for few in (True, False):
            for keys in (1, 31, 33, 100, 1000, 100_000):
                for pairs in (1, 2, 7, 8, 16, 64, 100, 148, 149, 296, 500, 1000, 10 ** 5):
                    blocks, warps = kv8_decode_shape(pairs, keys, hd, few, 148)
                    tiles = -(-keys // 32)
                    assert blocks in (1, 2, 4, 8) and 1 <= warps <= (4 if hd == 256 else 8)
                    assert blocks <= tiles and (blocks - 1) * warps < tiles
                    assert pairs > 148 or pairs * blocks <= 148 * 4
    assert kv8_decode_shape(8, 16384, 128, True, 148) == (8, 8)
    assert kv8_decode_shape(512, 2048, 128, True, 148) == (1, 3)


def test_splits_of_the_tensor_core_kernels():
    from mstar_b200.ops.kv8 import kv8_mma_splits, kv8_tc_splits

    assert kv8_mma_splits(256, 220, 148, False) == 1 and kv8_mma_splits(152, 1000, 148, False) == 2
    assert kv8_mma_splits(8, 10 ** 6, 148, True) == 4 * 28 and kv8_mma_splits(8, 100, 148, True) == 4
    assert kv8_mma_splits(1, 10 ** 6, 148, False) == 64 and kv8_mma_splits(1, 10 ** 6, 148, True) == 256
    assert kv8_tc_splits(16, 20017, 148, True) == (18, True) and kv8_tc_splits(16, 20017, 148, False) == (9, False)
    assert kv8_tc_splits(16, 4000, 148, True) == (9, False) and kv8_tc_splits(200, 511, 148, True) == (1, False)


def test_refuses_head_sizes_that_have_no_form():
    for hd in (12, 264):
        assert not ops.kv8_supported(hd)
        cache = Z(5, 2, 2, 16, hd, dtype=torch.uint8).view(F8)
        with pytest.raises(ops.KernelError, match="head_dim"):
            ops.kv8_read_rows(cache, Z(5, 2, 2, 16, dtype=torch.uint8), Z(2, 4, dtype=torch.int32),
                              Z(3, dtype=torch.int32), Z(3, dtype=torch.int32), torch.float32)


def test_splits_fill_the_gpu_and_keep_parts_long():
    assert ops.kv8_splits(8, 16384, 148) == 37 and ops.kv8_splits(512, 2048, 148) == 1
    assert ops.kv8_splits(1, 100, 148) == 1 and ops.kv8_splits(1, 10 ** 6, 148) == 64


def test_deployment_may_name_the_type():
    from mstar_b200.cli.main import _deployed_kv_dtype

    assert _deployed_kv_dtype({}) is None and _deployed_kv_dtype({"dtype": "bfloat16"}) is None
    assert _deployed_kv_dtype({"dtype": "float8_e4m3"}) == "float8_e4m3"


def test_command_line_takes_the_type():
    from mstar_b200.cli.main import build_parser

    a = build_parser().parse_args(["generate", "m", "--kv-cache-dtype", "float8_e4m3"])
    assert a.kv_cache_dtype == "float8_e4m3"
    assert build_parser().parse_args(["generate", "m"]).kv_cache_dtype is None
    with pytest.raises(SystemExit):
        build_parser().parse_args(["generate", "m", "--kv-cache-dtype", "int3"])
