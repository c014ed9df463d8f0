"""The linear layer with bias, activation and residual in its epilogue, for any number of tokens: against 64 bits, at the sizes where
it can go wrong (one token, the borders of token chunks and tiles, row counts that are no multiple of a tile, one group)."""
import pytest
import torch

from ffn_util import activate64, assert_close_to_rounding, code, disk, weights64, whole
from gpu_util import Guarded
from test_gpu_prefill_tiles import _one_weight_per_output

pytestmark = pytest.mark.gpu

ACTS = ["none", "silu", "gelu", "gelu_tanh", "swiglu"]


def _layer(pkg, rows, cols, act, seed, exact=True):
    t = disk(rows, cols, seed, exact)
    w = pkg.awq_alloc_fused(rows, cols)
    if act == "swiglu":
        pkg.awq_repack_into_swiglu(w, 0, *t, rows // 2)
    else:
        pkg.awq_repack_into(w, 0, *t)
    return w, t


def _check(pkg, rows, cols, M, act, bias, residual, in_place=False):
    w, t = _layer(pkg, rows, cols, act, rows + cols + M)
    ny = rows // 2 if act == "swiglu" else rows
    x = whole((M, cols), 4, M)
    # an activation of exact but large values tells nothing: outputs of 2^0 .. 2^5
    b = whole((rows,), 64 if act == "none" else 4, 1) if bias else None
    r = whole((M, ny), 64, 2) if residual else None
    out = Guarded((M, ny), torch.bfloat16)
    if in_place:
        out.t.copy_(r)
    pkg.linear_epilogue(out.t, w, x, M, bias=b, activation=code(pkg, act), residual=out.t if in_place else r)
    assert pkg.device_status() == 0
    v = x.double() @ weights64(*t).T
    if bias:
        v += b.double()
    v = activate64(v, act)
    if residual and act == "none":
        v += r.double()
    elif residual:  # the sum is rounded once: the activation's error beside a residual that may cancel it
        err = (out.t.double() - (v + r.double())).abs()
        assert bool((err <= (v + r.double()).abs() * 2.0 ** -8 + v.abs() * 2.0 ** -15 + r.abs() * 2.0 ** -23 + 2.0 ** -100).all())
        assert out.intact()
        pkg.awq_free(w)
        return
    assert_close_to_rounding(out.t, v, act)
    assert out.intact()
    pkg.awq_free(w)


@pytest.mark.parametrize("M", [1, 2, 7, 8, 9, 15, 16, 17, 24, 31, 32, 33, 47, 64, 65, 100, 128, 129, 255, 256, 257, 300, 513])
def test_token_counts(pkg, M):
    _check(pkg, 272, 640, M, "none", True, True)


@pytest.mark.parametrize("rows,cols", [(16, 128), (32, 256), (128, 128), (144, 384), (1040, 128), (2048, 5120), (5120, 17408), (512, 17408)])
@pytest.mark.parametrize("M", [1, 9, 40, 200])
def test_layer_sizes(pkg, rows, cols, M):
    _check(pkg, rows, cols, M, "none", True, False)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("bias,residual", [(False, False), (True, False), (False, True), (True, True)])
@pytest.mark.parametrize("M", [1, 5, 20, 77, 260])
def test_epilogues(pkg, act, bias, residual, M):
    _check(pkg, 352, 512, M, act, bias, residual)


@pytest.mark.parametrize("act", ["none", "swiglu"])
@pytest.mark.parametrize("M", [1, 16, 50, 300])
def test_residual_in_place(pkg, act, M):
    _check(pkg, 2080, 1024, M, act, False, True, in_place=True)


@pytest.mark.parametrize("rows,cols,M", [(5120, 6144, 1), (34816, 5120, 9), (16384, 5120, 77), (5120, 17408, 777)])
def test_random_weights(pkg, rows, cols, M):
    """Weights and activations of real distributions. An fp32 sum on the tensor cores adds 16 products at a time and loses at most 2^-22 of the
    sum of magnitudes at each of the cols / 16 steps (and at the joins of at most 16 pieces); rounding the output adds 2^-8."""
    w, t = _layer(pkg, rows, cols, "none", 5, exact=False)
    x = torch.randn((M, cols), generator=torch.Generator().manual_seed(6)).to(torch.bfloat16).cuda()
    y = torch.empty((M, rows), dtype=torch.bfloat16, device="cuda")
    pkg.linear_epilogue(y, w, x, M)
    w64 = weights64(*t)
    ref, mass = x.double() @ w64.T, x.double().abs() @ w64.abs().T
    err = (y.double() - ref).abs()
    assert bool((err <= ref.abs() * 2.0 ** -8 + mass * ((cols / 16 + 16) * 2.0 ** -22)).all())
    # and the same bits again
    z = torch.empty_like(y)
    pkg.linear_epilogue(z, w, x, M)
    assert torch.equal(y, z)
    pkg.awq_free(w)


@pytest.mark.parametrize("M", [1, 9, 77])
def test_non_finite_activations_stay_in_their_token(pkg, M):
    w, t = _layer(pkg, 256, 512, "none", 3)
    x = whole((M, 512), 4, 4)
    clean = torch.empty((M, 256), dtype=torch.bfloat16, device="cuda")
    pkg.linear_epilogue(clean, w, x, M)
    bad = M // 2
    x[bad, 100] = float("nan")
    y = torch.empty_like(clean)
    pkg.linear_epilogue(y, w, x, M, activation=pkg.ACT_NONE)
    assert bool(y[bad].isnan().all())
    others = [m for m in range(M) if m != bad]
    assert torch.equal(y[others], clean[others])
    pkg.awq_free(w)


def test_large_gates_and_infinite_residuals(pkg):
    """SiLU at gates of +-2^12 is the gate and zero, not NaN; an infinite residual comes out as itself."""
    rows, cols = 64, 128
    packed = torch.full((rows, cols // 8), -1, dtype=torch.int32, device="cuda")  # q = 15
    scale = torch.ones((rows, 1), dtype=torch.bfloat16, device="cuda")
    zp = torch.zeros((rows // 8, 1), dtype=torch.int32, device="cuda")
    w = pkg.awq_repack(packed, scale, zp)
    x = torch.zeros((2, cols), dtype=torch.bfloat16, device="cuda")
    x[0, :32], x[1, :32] = 8.0, -8.0  # 32 * 8 * 15 = 3840
    y = torch.empty((2, rows), dtype=torch.bfloat16, device="cuda")
    r = torch.zeros((2, rows), dtype=torch.bfloat16, device="cuda")
    r[0, 3] = -float("inf")
    for act in (pkg.ACT_SILU, pkg.ACT_GELU, pkg.ACT_GELU_TANH):
        pkg.linear_epilogue(y, w, x, 2, activation=act, residual=r)
        assert bool((y[1] == 0).all()) and float(y[0, 3]) == -float("inf")
        assert bool((torch.cat([y[0, :3], y[0, 4:]]) == 3840).all())
    pkg.awq_free(w)


@pytest.mark.parametrize("M", [1, 8, 16, 77, 300])
def test_every_weight_by_itself(pkg, synth, M):
    """Scales of every kind (subnormal, largest, either sign), every code and zero point, and one power of two per token: an output is one
    weight times it, exactly, wherever that is a normal number."""
    N, K = 272, 384
    q, z, scale = _one_weight_per_output(N, K, seed=M)
    w = pkg.weights_from_numpy(synth.pack_weight(q), scale, synth.pack_zero_point(z))
    want = torch.empty((N, K), dtype=torch.bfloat16, device="cuda")
    pkg.w4a16_dequant_rows(want, w, 0, N)
    want = want.double()
    y = torch.empty((M, N), dtype=torch.bfloat16, device="cuda")
    for power in (2.0 ** 60, 2.0 ** -60):
        for k0 in range(0, K, M) if M > 1 else (0, 127, 128, 255, 383):
            n = min(M, K - k0)
            x = torch.zeros((M, K), dtype=torch.bfloat16, device="cuda")
            x[torch.arange(n), torch.arange(k0, k0 + n)] = power
            pkg.linear_epilogue(y, w, x, M)
            got, ref = y[:n].double().t(), want[:, k0:k0 + n] * power
            normal = (ref.abs() >= 2.0 ** -126) & (ref.abs() < 2.0 ** 128)
            assert torch.equal(got[normal], ref[normal])
            assert bool((got[ref == 0] == 0).all())
    assert pkg.device_status() == 0
    pkg.awq_free(w)


@pytest.mark.parametrize("M", [1, 40, 300])
def test_captured_replayed_and_on_another_stream(pkg, M):
    w, t = _layer(pkg, 1024, 2048, "none", 9)
    x = whole((M, 2048), 4, 1)
    y = torch.empty((M, 1024), dtype=torch.bfloat16, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    pkg.linear_epilogue(y, w, x, M, stream=side)
    side.synchronize()
    eager = y.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        pkg.linear_epilogue(y, w, x, M, residual=y)  # twice in a row in the graph: y = layer + layer of itself's residual
        pkg.linear_epilogue(y, w, x, M, residual=y)
    y.zero_()
    g.replay()
    torch.cuda.synchronize()
    ref = (x.double() @ weights64(*t).T).to(torch.bfloat16)
    assert torch.equal(eager, ref)
    once = (x.double() @ weights64(*t).T)
    assert torch.equal(y, (once + ref.double()).to(torch.bfloat16))
    assert pkg.device_status() == 0
    pkg.awq_free(w)


def test_right_behind_a_repack_and_beside_the_other_matmuls(pkg):
    """A layer that was just repacked on the same stream, and calls of the existing kernels in front and behind."""
    w, _ = _layer(pkg, 2048, 1024, "none", 1)
    s = pkg.gemv_scratch_alloc(1024, 2048, 128, 16)
    x = whole((1, 1024), 4, 2)
    a, b, c = (torch.empty((1, 2048), dtype=torch.bfloat16, device="cuda") for _ in range(3))
    for seed in range(20, 26):
        t = disk(2048, 1024, seed)
        pkg.awq_repack_into(w, 0, *t)
        pkg.linear_epilogue(a, w, x, 1)
        pkg.gemv_w4a16(b, w, x, s)
        pkg.linear_epilogue(c, w, x, 1, residual=b)
        ref = x.double() @ weights64(*t).T
        assert torch.equal(a, ref.to(torch.bfloat16)) and torch.equal(b, a)
        assert torch.equal(c, (ref + b.double()).to(torch.bfloat16))
    pkg.gemv_scratch_free(s)
    pkg.awq_free(w)


def test_no_tokens(pkg):
    w, _ = _layer(pkg, 128, 128, "none", 1)
    y = torch.empty((0, 128), dtype=torch.bfloat16, device="cuda")
    pkg.linear_epilogue(y, w, torch.empty((0, 128), dtype=torch.bfloat16, device="cuda"), 0)
    pkg.awq_free(w)


def test_refusals(pkg):
    w, _ = _layer(pkg, 144, 128, "none", 1)
    x = whole((4, 128), 4, 1)
    y = torch.zeros((4, 144), dtype=torch.bfloat16, device="cuda")
    both = torch.zeros(4 * 144 + 4 * 128, dtype=torch.bfloat16, device="cuda")

    def refused(*a, **k):
        with pytest.raises(pkg.W4A16Error) as e:
            pkg.linear_epilogue(*a, **k)
        assert e.value.code == -1
        return str(e.value)

    assert "activation" in refused(y, w, x, 4, activation=7)
    assert "multiple of 32" in refused(y.view(-1)[:4 * 72].view(4, 72), w, x, 4, activation=pkg.ACT_SWIGLU)
    assert "overlaps x" in refused(both[:4 * 144].view(4, 144), w, both[4 * 128:8 * 128].view(4, 128), 4)
    assert "not y" in refused(both[:576].view(4, 144), w, x, 4, residual=both[8:584].view(4, 144))
    assert "overlaps bias" in refused(y, w, x, 4, bias=y[1])
    assert "aligned" in refused(both[1:577].view(4, 144), w, x, 4)
    assert "x:" in refused(y, w, x[:, ::2], 4)
    assert "x:" in refused(y, w, x.float(), 4)
    assert "residual:" in refused(y, w, x, 4, residual=x)
    assert "y:" in refused(y.cpu(), w, x, 4)
    assert "x:" in refused(y, w, x, 5)
    pkg.awq_free(w)
