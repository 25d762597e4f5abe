"""The kernels' barrier waits are bounded in time: one that nothing ends gives up after a second and says so, and waits after it
return at once."""
import pytest
import torch

from flexgemm_b200 import _cabi

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


@pytest.mark.parametrize("kind", [0, 1])
def test_wait_that_nothing_ends(kind):
    from flexgemm_b200.kernels import cuda as K
    K.check_status(DEV)
    first, second, complete, one_try = K.microbench_wait(kind, DEV)
    # a second, and what the 64 tries between two looks at the clock take
    assert 1_000_000_000 <= first <= 1_000_000_000 + 200 * max(one_try, 1000), (first, one_try)
    assert second <= 4 * max(one_try, 1000) and complete == 0
    with pytest.raises(RuntimeError, match="wait ran out"):
        K.check_status(DEV)
    assert (torch.ones(8, device=DEV) + 1).sum().item() == 16   # the context is as it was
    K.check_status(DEV)


def test_refusals():
    import ctypes
    out = (ctypes.c_uint64 * 4)()
    lib = _cabi.lib()
    assert lib.fgb_microbench_wait(2, out, 1 << 20, None) == -2 and lib.fgb_microbench_wait(-1, out, 1 << 20, None) == -2
    assert lib.fgb_microbench_wait(0, None, 1 << 20, None) == -1 and lib.fgb_microbench_wait(0, out, None, None) == -1
