"""The attention kernels' bounded waits: a call whose waits run out returns, says so, and
leaves the workspace usable."""
import pytest
import torch

from test_kv4_gpu import BF, _run, _setup

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lens,qs", [
    ([3000, 17], [1, 1]), ([60000], [1]), ([500] * 300, [1] * 300),      # decode
    ([300], [300]), ([9000, 700], [300, 200]), ([2500, 900, 40], [1, 600, 1]),
])
@pytest.mark.parametrize("D", [64, 128])
def test_waits_that_run_out(dip, lens, qs, D):
    """One poll a wait: whether that is enough depends on the hardware.  If it was, the result
    stands; if not, the error is reported; afterwards the same workspace gives the same bits."""
    take = torch.ops.dip_b200.take_device_error
    q, cache, table, cu = _setup(len(lens), lens, qs, 8, 2, D, 64, BF)
    ws = dip.kv4_workspace("cuda")
    want = _run(dip, q, cache, table, lens, cu, workspace=ws)
    torch.cuda.synchronize()
    assert take() == 0
    for _ in range(3):
        torch.ops.dip_b200.set_spin_limit(1)
        try:
            out, lse = _run(dip, q, cache, table, lens, cu, workspace=ws)
            torch.cuda.synchronize()
        finally:
            torch.ops.dip_b200.set_spin_limit(0)
        if take() == 0:
            assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
        again = _run(dip, q, cache, table, lens, cu, workspace=ws)
        torch.cuda.synchronize()
        assert take() == 0
        assert torch.equal(again[0], want[0]) and torch.equal(again[1], want[1])
