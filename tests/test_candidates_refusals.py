"""More that the operators for several candidates of a request refuse (no GPU)."""
import pytest
import torch

from tinyllama_c_b200 import ops

from test_candidates_host import ints, maps

REFUSED = [
    (maps, dict(lengths=ints(2))), (maps, dict(lengths=torch.zeros(3))), (maps, dict(lengths=ints(6)[::2])),
]


@pytest.mark.parametrize("i", range(len(REFUSED)))
def test_refused(i):
    call, change = REFUSED[i]
    with pytest.raises(ops.KernelError) as e:
        call(**change)
    assert "CUDA device" not in str(e.value)             # refused for what is wrong with it, not for where it runs
