"""launch_count() says how many kernels were launched: compared with the kernels of a captured graph."""
import pytest
import torch

import tinyllama_c_b200 as tlc
from tinyllama_c_b200 import ops
from tinyllama_c_b200.engine import StepEntry

import configs
from helpers import make_model_dir, random_tokens

pytestmark = pytest.mark.gpu
DEV = "cuda"


def kernels_of(calls):
    """(kernels of a captured graph of these calls, what launch_count() says of them)."""
    rt = pytest.importorskip("cuda.bindings.runtime")
    calls()                                                # (nothing is set up under capture)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    before = ops.launch_count()
    with torch.cuda.graph(graph):
        calls()
    said = ops.launch_count() - before
    raw = rt.cudaGraph_t(graph.raw_cuda_graph())
    _, _, n = rt.cudaGraphGetNodes(raw)
    _, nodes, n = rt.cudaGraphGetNodes(raw, n)
    kinds = [rt.cudaGraphNodeGetType(node)[1] for node in nodes[:n]]
    return sum(k == rt.cudaGraphNodeType.cudaGraphNodeTypeKernel for k in kinds), said


def test_products_in_8_bit_integers_and_routing():
    w, sw = ops.weight_int8(torch.randn(256, 128, device=DEV))
    gu, sgu = ops.weight_int8(torch.randn(8, 128, 128, device=DEV))
    d, sd = ops.weight_int8(torch.randn(8, 128, 64, device=DEV))
    want = []
    for T in (1, 2, 5, 8, 9, 40, 400):
        x, logits = torch.randn(T, 128, device=DEV), torch.randn(T, 8, device=DEV)
        out, y = torch.empty(T, 256, device=DEV), torch.empty(T, 3, 128, device=DEV)
        q, s = ops.rows_int8(x)
        routing = ops.moe_route(logits, 8, 3)
        for calls in (lambda: ops.linear_int8(x, w, sw, out), lambda: ops.linear_int8(q, w, sw, out, a_scale=s), lambda: ops.rows_int8(x, (q, s)),
                      lambda: ops.moe_route(logits, 8, 3),
                      lambda: ops.moe_experts_int8(x, gu, sgu, d, sd, routing, 3, y)):
            made, said = kernels_of(calls)
            assert made == said > 0
            want.append(made)
    assert len(set(want)) > 3                              # (one launch, two, four and five among them)


@pytest.mark.parametrize("weights", [None, "int8"])
def test_layers_from_a_table_count_as_those_one_by_one(tmp_path, weights):
    llm = tlc.LLM(make_model_dir(tmp_path, dict(configs.TINY_D, num_hidden_layers=4), seed=7, std=0.1), max_tokens=1024, max_seqs=4, weights=weights)
    assert llm.model.repeated is not None
    counts = []
    for repeated in (llm.model.repeated, None):
        llm.model.repeated = repeated
        slot = llm.cache.acquire()
        before = ops.launch_count()
        llm.step([StepEntry(slot, random_tokens(llm.model.vocab, 60, 1), [59])])
        counts.append(ops.launch_count() - before)
        llm.cache.release(slot)
    assert counts[0] == counts[1]
