"""GPU: the wait of a whole warp on an mbarrier, which its lanes leave together, whether the phase completes or the CTA gives up."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_lanes_leave_together(pkg, cuda):
    lib = pkg.load_library()
    cycles = torch.zeros(1, dtype=torch.int64, device=cuda)
    for limit in (200_000, 1_000_000):
        assert lib.ixk_selftest_bounded_wait(limit, cycles.data_ptr(), torch.cuda.current_stream().cuda_stream) == pkg.IXK_OK
        torch.cuda.synchronize()
        assert limit <= int(cycles.item()) < limit + 40_000_000      # (-1: lanes of one warp were given unlike answers)
        with pytest.raises(pkg.IxkError) as e:
            pkg.device_status()
        assert e.value.status == pkg.IXK_DEVICE_TIMEOUT and "901" in str(e.value)
        assert pkg.device_status() == 0
