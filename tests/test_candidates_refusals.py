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


@pytest.mark.parametrize("n_slots,max_pages,B,refused", [(64, 1 << 25, 64, True), (4096, 1 << 19, 4096, True), (4096, 1 << 19, 4095, False), (63, 1 << 25, 4096, False),
                                                         (1 << 20, 4096, 4096, False)])
def test_pages_of_a_call_fit_32_bits(n_slots, max_pages, B, refused, monkeypatch):
    """The library refuses before it looks at anything; what it does not refuse fails here for want of a device, not by a launch."""
    if torch.cuda.is_available():
        pytest.skip("made-up addresses")
    lib = ops.library()
    code = lib.tlc_page_resize(None, n_slots, max_pages, None, 1 << 20, None, None, None, B, None, None)
    assert code != 0 and ("2^31" in lib.tlc_last_error().decode()) == refused


@pytest.mark.parametrize("args,blocks,rows", [((0, 1, 50, 4, 64, 8, 2, 128, 4096, 64), 296, 64), ((0, 1, 50, 1, 3, 4, 2, 64, 100, 3), 12, 16),
                                              ((0, 1, 50, 4, 64, 8, 2, 37, 4096, 64), 296, 64)])
def test_scratch_by_the_current_device(args, blocks, rows):
    """Asked anew in every call, a B200's 148 SMs where there is no device: two blocks of partial results to an SM at most, each two slots of
    `rows` rows of heads in fours and two statistics, and the 32-byte split."""
    hd = args[7]
    assert ops.library().tlc_tree_attention_scratch(*args) == blocks * (2 * rows * ((hd + 3) // 4 * 4 + 2) * 4 + 32)
    assert ops.library().tlc_beam_select_scratch(8, 151551) == 8 * 296 * 16 and ops.library().tlc_beam_select_scratch(8, 151552) == 8 * 74 * 16
