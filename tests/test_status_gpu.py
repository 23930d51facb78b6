"""The status words of the kernels' bounded waits: read after the work of every stream."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", ["jl_prefill_status", "jl_tree_status", "jl_head_status"])
def test_status_waits_for_other_streams(name):
    from jetlm.kernels import _native
    assert getattr(_native.lib(), name)() == 0        # (the first call may allocate, which waits for everything)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(100_000_000)                # some 50 ms
    assert not side.query()
    assert getattr(_native.lib(), name)() == 0
    assert side.query()
