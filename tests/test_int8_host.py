"""Weights in 8-bit integers: what is refused before anything touches a GPU."""
import pytest
import torch

import tinyllama_c_b200 as tlc
from tinyllama_c_b200 import ops
from tinyllama_c_b200.cli.options import add_common
from tinyllama_c_b200.config import config_from_dict
from tinyllama_c_b200.weights import build_model

import configs


def test_weight_formats_that_do_not_exist_or_do_not_go_with_the_type(tmp_path):
    with pytest.raises(ValueError, match="int8"):
        tlc.load_model(str(tmp_path), weights="int4")
    with pytest.raises(ValueError, match="bfloat16"):
        tlc.load_model(str(tmp_path), dtype="float32", weights="int8")


def test_a_float32_model_keeps_its_weights():
    model = build_model(config_from_dict(dict(configs.TINY_A)))
    model.dtype = torch.float32
    with pytest.raises(ValueError, match="float32"):
        model.to_int8()


def test_there_is_no_cpu_path():
    x, w, s = torch.zeros(2, 32), torch.zeros(8, 32, dtype=torch.int8), torch.zeros(8)
    for call in (lambda: ops.rows_int8(x), lambda: ops.rmsnorm_int8(x, torch.ones(32), 1e-5), lambda: ops.weight_int8(x),
                 lambda: ops.linear_int8(x, w, s, torch.zeros(2, 8)), lambda: ops.linear_swiglu_int8(x, w, s, torch.zeros(2, 4))):
        with pytest.raises(ops.KernelError):
            call()


def test_the_programs_know_the_option():
    import argparse
    ap = argparse.ArgumentParser()
    add_common(ap, 1)
    assert ap.parse_args(["-m", "x"]).weights is None and ap.parse_args(["-m", "x", "--weights", "int8"]).weights == "int8"
