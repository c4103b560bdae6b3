"""Calls around the 8-bit cache that need no GPU: deployment files."""
import logging

import pytest

from mstar_b200.cli.main import _deployed_kv_dtype


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
