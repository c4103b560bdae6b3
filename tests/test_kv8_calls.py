"""Calls around the 8-bit cache that need no GPU: deployment files, refusals."""
import logging

import pytest
import torch

from mstar_b200 import ops
from mstar_b200.cli.main import _deployed_kv_dtype
from test_kv8 import args


@pytest.mark.parametrize("name", ["bfloat16", "bf16", "float32", "fp32", "f32", "float16", "fp16", "half", None])
def test_deployments_that_name_a_compute_type_run_in_it(name, caplog):
    with caplog.at_level(logging.WARNING):
        assert _deployed_kv_dtype({"dtype": name}) is None
    assert not caplog.records


@pytest.mark.parametrize("name", ["fp8", "float8_e5m2", "int8", 8, ["bf16"]])
def test_deployments_that_name_another_type_run_as_before_and_say_so(name, caplog):
    with caplog.at_level(logging.WARNING):
        assert _deployed_kv_dtype({"dtype": name}) is None
    assert "compute type" in caplog.text


@pytest.mark.parametrize("name", ["auto", "float8_e4m3"])
def test_deployments_may_name_the_caches_types(name):
    assert _deployed_kv_dtype({"dtype": name}) == name


FAR = 2 ** 31 + 8          # (tensors without memory: these are refused before their device matters)


def far_rows(rows, width, dtype):
    return torch.empty(rows, FAR, dtype=dtype, device="meta")[:, :width]


@pytest.mark.parametrize("name,argument,width,dtype", [
    ("rope_kv8_write", "qkv", 512, torch.float32), ("rope_kv8_write", "block_table", 4, torch.int32),
    ("kv8_read_rows", "block_table", 4, torch.int32),
    ("paged_decode_attention_kv8", "q", 256, torch.float32), ("paged_decode_attention_kv8", "block_table", 4, torch.int32),
    ("paged_prefill_attention_kv8", "q", 256, torch.float32), ("paged_prefill_attention_kv8", "block_table", 4, torch.int32)])
def test_rows_too_far_apart_are_refused(name, argument, width, dtype):
    """Their distance is a 32-bit number in the kernels."""
    with pytest.raises(ops.KernelError, match="apart"):
        getattr(ops, name)(**args(name, **{argument: far_rows(3, width, dtype)}))


def test_queries_beyond_the_tensor_core_kernels_reach_take_the_other():
    from mstar_b200.ops.kv8 import kv8_tc_reaches

    assert kv8_tc_reaches(2048, 6144) and kv8_tc_reaches(15, 2 ** 31 - 8)
    assert not kv8_tc_reaches(17, 2 ** 31 - 8) and not kv8_tc_reaches(2 ** 25, 1024)
    assert kv8_tc_reaches(2 ** 25, 1023) and (2 ** 25 * 1023) >> 3 < 0xffffffff       # (which stands for no row)


@pytest.mark.parametrize("name", ["paged_decode_attention_kv8", "paged_prefill_attention_kv8"])
@pytest.mark.parametrize("scale", [float("inf"), 1e39, 2.0 ** 127, 1e-39, 1e-320, -1.0])
def test_scales_that_are_no_ordinary_floats_are_refused(name, scale):
    with pytest.raises(ops.KernelError, match="scale"):
        getattr(ops, name)(**args(name, scale=scale))


def test_a_layer_says_whether_its_head_size_can_be_held():
    import dataclasses

    from mstar_b200.config.layout import PositionSpec
    from mstar_b200.parts.attention import Attention
    from test_kv8 import PLAIN

    for hd, able in ((64, True), (8, True), (256, True), (20, False), (264, False)):
        spec = dataclasses.replace(PLAIN, head_dim=hd, position=PositionSpec(head_dim=hd, rotary_dim=4))
        assert Attention.cache_need(spec).kv.eight_bit is able
    assert not Attention.cache_need(dataclasses.replace(PLAIN, softcap=30.0)).kv.eight_bit
