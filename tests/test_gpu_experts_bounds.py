"""Bounds of the experts' slots that go up and down: sets that would overlap. The launch is laid out for the given number of slots, so the
kernels may not make more work of the bounds than that: no wait runs out, nothing outside y is written."""
import pytest
import torch

from ffn_util import whole
from gpu_util import Guarded
from test_gpu_experts import Bank

pytestmark = pytest.mark.gpu


def _units(offsets, slots, nt, row_tiles):
    """Host model: units of work that the few-token kernel makes of the bounds."""
    at, most, total = [min(max(o, 0), slots) for o in offsets], 0, 0
    for lo, hi in zip(at, at[1:]):
        lo = max(lo, most)
        most = max(lo, hi)
        total += (most - lo + nt - 1) // nt * row_tiles
    return total


@pytest.mark.parametrize("E,slots", [(8, 8), (8, 30), (4, 100), (2, 700), (512, 8), (512, 500), (512, 4000), (512, 30000)])
@pytest.mark.parametrize("cols", [128, 512, 2048])
@pytest.mark.parametrize("gather", [True, False])
def test_bounds_that_go_up_and_down(pkg, E, slots, cols, gather):
    rows = 256
    bank = Bank(pkg, 2, rows, cols) if E > 2 else Bank(pkg, E, rows, cols)
    w = bank.w if E == 2 else pkg.experts_alloc(E, rows, cols)
    if E > 2:  # (every expert past the first takes the second's tensors)
        for e in range(E):
            pkg.awq_repack_into(pkg.experts_view(w, e), 0, *bank.disk[min(e, 1)])
    n = max(1, slots // 2)  # the first expert's slots, which are right in every row of bounds below
    x = whole((50 if gather else slots, cols), 4, 1)
    x_rows = (torch.arange(slots, dtype=torch.int32, device="cuda") % 50) if gather else None
    want = bank.layer64(0, x[x_rows[:n].long()] if gather else x[:n]).to(torch.bfloat16)
    out = Guarded((slots, rows), torch.bfloat16)
    for offsets in ([0, n] + [0, slots] * E, [0, n] + [n, -1, 2 ** 31 - 1, -2 ** 31] * E, [0, n] + list(range(slots, -1, -1)) + [0] * E):
        offsets = offsets[:E + 1]
        nt = 8 if slots <= 4 * E else 16
        most = (min(slots, E) + (slots - min(slots, E)) // nt) * (rows // 128)
        assert _units(offsets, slots, nt, rows // 128) <= most
        out.t.fill_(0)
        pkg.experts_linear(out.t, w, x, torch.tensor(offsets, dtype=torch.int32, device="cuda"), x_rows=x_rows)
        assert pkg.device_status() == 0 and out.intact()
        assert torch.equal(out.t[:n], want)
    if E > 2:
        pkg.experts_free(w)
    bank.free()
