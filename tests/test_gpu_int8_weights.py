"""Models whose weights become 8-bit integers after they have been used."""
import pytest
import torch

import tinyllama_c_b200 as tlc
from tinyllama_c_b200 import ops

import configs
from helpers import make_model_dir, random_tokens

pytestmark = pytest.mark.gpu
D4 = dict(configs.TINY_D, num_hidden_layers=4)


@pytest.fixture(scope="module")
def folder(tmp_path_factory):
    return make_model_dir(tmp_path_factory.mktemp("models"), D4, seed=7, std=0.1)


def _tokens(llm, prompts):
    return [r.tokens for r in llm.generate(prompts, tlc.GREEDY, max_new_tokens=12, ignore_eos=True)]


@pytest.mark.parametrize("how", ["to_int8", "another LLM"])
def test_captured_steps_follow_the_model_to_8_bit_weights(folder, how):
    """An LLM that has captured decode steps of the 16-bit weights, whose memory is given to someone else afterwards."""
    llm = tlc.LLM(folder, max_tokens=1024, max_seqs=4)
    prompts = [random_tokens(llm.model.vocab, n, n) for n in (33, 5)]
    before = _tokens(llm, prompts)
    assert llm._graphs and _tokens(llm, prompts) == before
    if how == "to_int8":
        llm.model.to_int8()
    else:
        tlc.LLM(llm.model, max_tokens=256, max_seqs=2, weights="int8")
    rubbish = [torch.full((1 << n,), float("nan"), dtype=torch.bfloat16, device="cuda") for n in range(8, 22) for _ in range(4)]
    after = _tokens(llm, prompts)
    eager = tlc.LLM(llm.model, max_tokens=1024, max_seqs=4, use_graphs=False)
    assert after == _tokens(eager, prompts)
    fresh = tlc.LLM(folder, max_tokens=1024, max_seqs=4, weights="int8")
    assert after == _tokens(fresh, prompts)
    ops.check_errors()
    del rubbish
