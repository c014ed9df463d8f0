"""Layers with an epilogue whose CTAs take several tiles or units, one after another: the staging buffer's way round (residual in, finished
tile out, next residual in), the accumulator's phases, and units without K splits; then an expert's view through every matmul call."""
import pytest
import torch

from ffn_util import disk, whole
from test_gpu_experts import Bank
from test_gpu_linear_epilogue import _check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,cols,M", [(5120, 256, 1100), (2592, 384, 2500), (34816, 256, 500)])
@pytest.mark.parametrize("act", ["none", "swiglu"])
@pytest.mark.parametrize("in_place", [False, True])
def test_more_tiles_than_pairs(pkg, rows, cols, M, act, in_place):
    """148 SMs run 74 pairs at once; a tile is 256 rows x 256 tokens at most."""
    assert -(-rows // 256) * -(-M // 256) > 74
    _check(pkg, rows, cols, M, act, True, True, in_place=in_place)


@pytest.mark.parametrize("M", [9, 40, 80])
@pytest.mark.parametrize("act", ["none", "gelu", "swiglu"])
@pytest.mark.parametrize("in_place", [False, True])
def test_more_tiles_than_ctas(pkg, M, act, in_place):
    """Few tokens, a CTA alone per tile: 449 row tiles."""
    _check(pkg, 449 * 128 - 32, 256, M, act, True, True, in_place=in_place)


@pytest.mark.parametrize("rows,cols", [(64, 128), (352, 384), (2080, 128)])
@pytest.mark.parametrize("M", [1, 3, 8])
@pytest.mark.parametrize("act", ["none", "silu", "swiglu"])
@pytest.mark.parametrize("in_place", [False, True])
def test_few_tokens_without_splits(pkg, rows, cols, M, act, in_place):
    """One to three groups of k: nothing to share out."""
    _check(pkg, rows, cols, M, act, True, True, in_place=in_place)


@pytest.mark.parametrize("M", [1, 8])
@pytest.mark.parametrize("act", ["none", "swiglu"])
@pytest.mark.parametrize("cols", [128, 640])
def test_few_tokens_several_units_per_cta(pkg, M, act, cols):
    """Two CTAs on each of 148 SMs; 701 row tiles."""
    _check(pkg, 701 * 128 - 96, cols, M, act, True, True)


@pytest.mark.parametrize("rows,cols", [(272, 256), (1024, 1024)])
def test_a_view_goes_through_every_matmul_call(pkg, rows, cols):
    """Each call gives the bits that it gives for the same layer in a container of its own."""
    bank = Bank(pkg, 3, rows, cols, seed=4, exact=False)
    s = pkg.gemv_scratch_alloc(cols, rows, 128, 16)
    ws = pkg.gemm_workspace_alloc(1 << 20)
    x = torch.randn((300, cols), generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    ln = torch.ones(cols, dtype=torch.bfloat16, device="cuda")

    def outputs(w):
        y = [torch.empty((m, rows), dtype=torch.bfloat16, device="cuda") for m in (1, 1, 5, 300, 9, 9, 1, 40)]
        f, ids = torch.empty(rows, device="cuda"), torch.empty(3, dtype=torch.int32, device="cuda")
        pkg.gemv_w4a16(y[0], w, x, s)
        pkg.gemv_w4a16_f32(f, w, x, s)
        pkg.gemv_w4a16_static(y[1], w, x)
        pkg.gemm_small_w4a16(y[2], w, x, 5, s)
        pkg.gemm_w4a16(y[3], w, x, 300, ws)
        pkg.linear_fused(y[4], w, x, 9, s, ln_weight=ln)
        y[5].copy_(y[4])
        pkg.linear_fused(y[5], w, x, 9, s, epilogue=pkg.EPILOGUE_RESIDUAL)
        pkg.lm_head_argmax(ids, w, x, 3, s)
        pkg.linear_epilogue(y[6], w, x[:1], 1)
        pkg.linear_epilogue(y[7], w, x[:40], 40, activation=pkg.ACT_SILU)
        torch.cuda.synchronize()
        return [*y, f, ids]

    for e in (2, 0, 1):  # (the last expert's stream ends with the allocation)
        alone = pkg.awq_repack(*bank.disk[e])
        for got, want in zip(outputs(pkg.experts_view(bank.w, e)), outputs(alone)):
            assert torch.equal(got, want)
        pkg.awq_free(alone)
    assert pkg.device_status() == 0
    pkg.gemv_scratch_free(s)
    pkg.gemm_workspace_free(ws)
    bank.free()


def test_a_view_is_repacked_in_parts(pkg):
    """gate and up of one expert by two calls, beside the experts around it."""
    E, inter, cols = 3, 144, 256
    w = pkg.experts_alloc(E, 2 * inter, cols)
    x, y = whole((2, cols), 4, 1), torch.empty((2, inter), dtype=torch.bfloat16, device="cuda")
    halves = [[disk(inter, cols, 10 * e + h) for h in range(2)] for e in range(E)]
    for e in (1, 0, 2):
        for h in (1, 0):
            pkg.awq_repack_into_swiglu(pkg.experts_view(w, e), h * inter, *halves[e][h], inter)
    for e in range(E):
        alone = pkg.awq_alloc_fused(2 * inter, cols)
        pkg.awq_repack_into_swiglu(alone, 0, *[torch.cat([a, b]) for a, b in zip(*halves[e])], inter)
        want = torch.empty_like(y)
        pkg.linear_epilogue(want, alone, x, 2, activation=pkg.ACT_SWIGLU)
        pkg.linear_epilogue(y, pkg.experts_view(w, e), x, 2, activation=pkg.ACT_SWIGLU)
        assert torch.equal(y, want)
        pkg.awq_free(alone)
    pkg.experts_free(w)
