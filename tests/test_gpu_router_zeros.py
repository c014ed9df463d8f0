"""The router's order at zero: -0 and +0 are equal logits, so the lower index comes first, whatever the signs."""
import pytest
import torch

from test_gpu_experts import _check_route

pytestmark = pytest.mark.gpu


def _zeros(T, E, seed):
    """Zeros of both signs among few other values: ties within a lane (experts 32 apart), between lanes and at the picks' border."""
    gen = torch.Generator().manual_seed(seed)
    logits = torch.where(torch.rand((T, E), generator=gen) < 0.5, -0.0, 0.0)
    logits[torch.rand((T, E), generator=gen) < 0.02] = 1.0
    logits[torch.rand((T, E), generator=gen) < 0.1] = -1.0
    logits[0] = -0.0
    logits[0, 1::2] = 0.0  # the lower of every two neighbours is -0
    logits[1] = 0.0
    logits[1, :(E + 1) // 2] = -0.0
    return logits


@pytest.mark.parametrize("E", [2, 33, 64, 65, 128, 129, 256, 257, 512])
@pytest.mark.parametrize("T", [3, 45])
def test_zeros_of_both_signs_are_a_tie(pkg, E, T):
    logits = _zeros(T, E, E + T).cuda()
    assert bool((logits[0, 0] == logits[0, 1])) and bool(torch.signbit(logits[0, 0])) and not bool(torch.signbit(logits[0, 1]))
    for kind in (torch.float32, torch.bfloat16):
        for k in (1, min(7, E)):
            _check_route(pkg, logits.to(kind), k)
        _check_route(pkg, logits.to(kind), min(16, E), renormalize=False)


def test_numbers_next_to_zero_keep_their_order(pkg):
    """The smallest numbers of either sign (subnormal) around the two zeros, and the largest."""
    tiny, big = 2.0 ** -149, torch.finfo(torch.float32).max
    row = torch.tensor([-tiny, -0.0, 0.0, tiny, -2 * tiny, 2 * tiny, -big, big, -2.0 ** -126, 2.0 ** -126])
    assert float(row[3]) > 0
    logits = torch.stack([row, row.flip(0), row.roll(3)]).cuda()
    _check_route(pkg, logits, 10)
    _check_route(pkg, logits[:1], 7, renormalize=False)
