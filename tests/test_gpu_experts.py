"""Layers of experts: the router, the products grouped by expert and the combination of the experts' outputs, each against 64 bits,
and run together as a decoder layer runs them."""
import math

import pytest
import torch

from ffn_util import activate64, assert_close_to_rounding, code, disk, weights64, whole
from gpu_util import Guarded

pytestmark = pytest.mark.gpu


class Bank:
    """A container of experts with its checkpoint tensors."""

    def __init__(self, pkg, E, rows, cols, act="none", seed=0, exact=True):
        self.pkg, self.act = pkg, act
        self.disk = [disk(rows, cols, seed * 1000 + e, exact) for e in range(E)]
        self.w = pkg.experts_alloc(E, rows, cols)
        for e, t in enumerate(self.disk):
            view = pkg.experts_view(self.w, e)
            if act == "swiglu":
                pkg.awq_repack_into_swiglu(view, 0, *t, rows // 2)
            else:
                pkg.awq_repack_into(view, 0, *t)

    def layer64(self, e, x, bias=None):
        v = x.double() @ weights64(*self.disk[e]).T
        return activate64(v if bias is None else v + bias.double(), self.act)

    def free(self):
        self.pkg.experts_free(self.w)


def _offsets(counts):
    at = [0]
    for n in counts:
        at.append(at[-1] + n)
    return at, torch.tensor(at, dtype=torch.int32, device="cuda")


def _check(pkg, counts, rows, cols, act="none", bias=False, gather=True, spare=0, tokens=13):
    """Ragged counts per expert; `spare` rows behind the last slot have to stay as they were."""
    E = len(counts)
    bank = Bank(pkg, E, rows, cols, act)
    at, offsets = _offsets(counts)
    slots = at[-1] + spare
    ny = rows // 2 if act == "swiglu" else rows
    x = whole((tokens if gather else max(slots, 1), cols), 4, 1)
    gen = torch.Generator().manual_seed(2)
    x_rows = torch.randint(0, tokens, (slots,), generator=gen).to(torch.int32).cuda() if gather else None
    b = whole((E, rows), 4, 3) if bias else None
    out = Guarded((slots, ny), torch.bfloat16)
    out.t.fill_(7)
    pkg.experts_linear(out.t, bank.w, x, offsets, x_rows=x_rows, bias=b, activation=code(pkg, act))
    assert pkg.device_status() == 0
    for e in range(E):
        lo, hi = at[e], at[e + 1]
        if lo < hi:
            xe = x[x_rows[lo:hi].long()] if gather else x[lo:hi]
            assert_close_to_rounding(out.t[lo:hi], bank.layer64(e, xe, b[e] if bias else None), act)
    assert bool((out.t[at[-1]:] == 7).all()) and out.intact()
    bank.free()


@pytest.mark.parametrize("counts", [
    [1], [0, 1], [1, 0], [0, 0, 3, 0, 0], [1] * 8, [0] * 20 + [5], [7, 8, 9, 15, 16, 17, 31, 32, 33], [0, 64, 0, 1, 0, 65],
    [100, 1, 0, 130], [224, 225, 3, 0, 260, 1], [2] * 70, [0] * 300 + [3] + [0] * 200 + [1], [600]])
@pytest.mark.parametrize("gather", [True, False])
def test_ragged_counts(pkg, counts, gather):
    _check(pkg, counts, 144, 384, gather=gather, bias=True, spare=3)


@pytest.mark.parametrize("rows,cols", [(16, 128), (32, 128), (128, 256), (2048, 5120), (5120, 1024), (528, 640)])
@pytest.mark.parametrize("counts", [[1, 0, 2, 1], [9, 0, 20, 3], [40, 70, 0, 90]])
def test_layer_sizes(pkg, rows, cols, counts):
    _check(pkg, counts, rows, cols)


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh", "swiglu"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("counts", [[1, 0, 2], [12, 30, 0, 5], [100, 0, 180, 66]])
def test_activations(pkg, act, bias, counts):
    _check(pkg, counts, 352, 512, act=act, bias=bias)


@pytest.mark.parametrize("counts", [[3200] + [0] * 400 + [5] * 111, [0] * 511 + [40], [0, 2, 1, 15] * 128, [0] * 511 + [6000], [0, 25, 3, 70] * 128])
@pytest.mark.parametrize("gather", [True, False])
def test_as_many_experts_as_a_container_takes(pkg, counts, gather):
    """Tables of 512 sets beside each kernel's stages; expert 511's rows."""
    _check(pkg, counts, 144, 256, gather=gather, bias=True, spare=2)


@pytest.mark.parametrize("n", [3, 40, 3500])
def test_experts_past_four_gigabytes_of_weights(pkg, n):
    E, rows, cols = 512, 34816, 512
    w = pkg.experts_alloc(E, rows, cols)
    t = disk(rows, cols, 5)
    pkg.awq_repack_into(pkg.experts_view(w, E - 1), 0, *t)
    x = whole((n, cols), 4, 1)
    y = torch.empty((n, rows), dtype=torch.bfloat16, device="cuda")
    pkg.experts_linear(y, w, x, torch.tensor([0] * E + [n], dtype=torch.int32, device="cuda"))
    assert torch.equal(y, (x.double() @ weights64(*t).T).to(torch.bfloat16))
    pkg.experts_free(w)


@pytest.mark.parametrize("gather", [True, False])
def test_rows_past_four_gigabytes(pkg, gather):
    """Inputs and outputs whose offsets pass 32 bits, in bytes and in elements."""
    n, tokens, K, N = 140000, 80, 128, 17408
    bank = Bank(pkg, 3, N, K)
    at, offsets = _offsets([n - 50, 0, 50])
    x = whole((tokens if gather else n, K), 4, 1)
    rows = (torch.arange(n, dtype=torch.int32, device="cuda") % tokens) if gather else None
    y = torch.empty((n, N), dtype=torch.bfloat16, device="cuda")
    pkg.experts_linear(y, bank.w, x, offsets, x_rows=rows)
    for e, lo, hi in ((0, 0, 300), (0, n - 400, n - 50), (2, n - 50, n)):
        xe = x[rows[lo:hi].long()] if gather else x[lo:hi]
        assert torch.equal(y[lo:hi], bank.layer64(e, xe).to(torch.bfloat16))
    # and as inputs: the last rows, of 17408 columns
    back = Bank(pkg, 3, 128, N, seed=1)
    y[n - 400:].copy_(whole((400, N), 4, 2))
    last = torch.arange(n - 1, n - 41, -1, dtype=torch.int32, device="cuda")
    z = torch.empty((40, 128), dtype=torch.bfloat16, device="cuda")
    off = torch.tensor([0, 0, 30, 40], dtype=torch.int32, device="cuda")
    for count in (12, 40):  # few rows and many
        pkg.experts_linear(z[:count], back.w, y, off.clamp(max=count), x_rows=last[:count])
        for e, lo, hi in ((1, 0, min(30, count)), (2, 30, 40)):
            if hi <= count:
                assert torch.equal(z[lo:hi], back.layer64(e, y[last[lo:hi].long()]).to(torch.bfloat16))
    bank.free()
    back.free()


def test_no_slots_at_all(pkg):
    _check(pkg, [0, 0, 0], 128, 128, spare=4)
    _check(pkg, [0, 0, 0], 128, 128)


def test_random_weights_many_tokens(pkg):
    """Real distributions; the tolerance of the dense layer's test."""
    E, rows, cols = 6, 1024, 2048
    bank = Bank(pkg, E, rows, cols, exact=False)
    at, offsets = _offsets([300, 0, 31, 700, 5, 129])
    x = torch.randn((400, cols), generator=torch.Generator().manual_seed(6)).to(torch.bfloat16).cuda()
    x_rows = torch.randint(0, 400, (at[-1],), generator=torch.Generator().manual_seed(7)).to(torch.int32).cuda()
    y = torch.empty((at[-1], rows), dtype=torch.bfloat16, device="cuda")
    pkg.experts_linear(y, bank.w, x, offsets, x_rows=x_rows)
    for e in range(E):
        xe, w64 = x[x_rows[at[e]:at[e + 1]].long()].double(), weights64(*bank.disk[e])
        ref, mass = xe @ w64.T, xe.abs() @ w64.abs().T
        assert bool(((y[at[e]:at[e + 1]].double() - ref).abs() <= ref.abs() * 2.0 ** -8 + mass * ((cols / 16 + 16) * 2.0 ** -22)).all())
    z = torch.empty_like(y)
    pkg.experts_linear(z, bank.w, x, offsets, x_rows=x_rows)
    assert torch.equal(y, z)
    bank.free()


def test_offsets_and_rows_out_of_range_stay_inside_the_buffers(pkg):
    """Bounds and rows that make no sense are clamped on the device: nothing outside y is written and what is right comes out right."""
    bank = Bank(pkg, 4, 128, 128)
    x = whole((5, 128), 4, 1)
    out = Guarded((12, 128), torch.bfloat16)
    for offsets, rows in (([0, 3, 3, 2 ** 30, 2 ** 30], [0] * 12), ([-5, 3, 3, 12, 4], [0] * 12),
                          ([0, 3, 3, 9, 12], [0, 1, 2, -7, 2 ** 31 - 1, 5] + [-2 ** 31] * 6)):
        pkg.experts_linear(out.t, bank.w, x, torch.tensor(offsets, dtype=torch.int32, device="cuda"),
                           x_rows=torch.tensor(rows, dtype=torch.int32, device="cuda"))
        assert pkg.device_status() == 0 and out.intact()
        ref = bank.layer64(0, x[torch.tensor(rows[:3], device="cuda")]).to(torch.bfloat16)
        assert torch.equal(out.t[:3], ref)
    bank.free()


def test_a_view_is_a_layer_of_its_own(pkg):
    bank = Bank(pkg, 3, 272, 256)
    deq = torch.empty((272, 256), dtype=torch.bfloat16, device="cuda")
    for e in (2, 0, 1):
        pkg.w4a16_dequant_rows(deq, pkg.experts_view(bank.w, e), 0, 272)
        assert torch.equal(deq.double(), weights64(*bank.disk[e]))
    x, y = whole((3, 256), 4, 1), torch.empty((3, 272), dtype=torch.bfloat16, device="cuda")
    pkg.linear_epilogue(y, pkg.experts_view(bank.w, 1), x, 3)
    assert torch.equal(y, bank.layer64(1, x).to(torch.bfloat16))
    with pytest.raises(pkg.W4A16Error):
        pkg.awq_free(pkg.experts_view(bank.w, 0))
    with pytest.raises(pkg.W4A16Error):
        pkg.experts_view(bank.w, 3)
    bank.free()


@pytest.mark.parametrize("counts", [[2, 0, 1], [50, 0, 30]])
def test_right_behind_a_repack(pkg, counts):
    """Experts repacked on the same stream without a wait in between, read as a group and by themselves."""
    E, rows, cols = 3, 1024, 512
    w = pkg.experts_alloc(E, rows, cols)
    at, offsets = _offsets(counts)
    x = whole((at[-1], cols), 4, 1)
    y, z = torch.empty((at[-1], rows), dtype=torch.bfloat16, device="cuda"), torch.empty((counts[2], rows), dtype=torch.bfloat16, device="cuda")
    for seed in range(30, 50, 4):
        tensors = [disk(rows, cols, seed + e) for e in range(E)]
        for e, t in enumerate(tensors):
            pkg.awq_repack_into(pkg.experts_view(w, e), 0, *t)
        pkg.experts_linear(y, w, x, offsets)
        pkg.linear_epilogue(z, pkg.experts_view(w, 2), x[at[2]:], counts[2])
        want = torch.cat([x[at[e]:at[e + 1]].double() @ weights64(*t).T for e, t in enumerate(tensors)]).to(torch.bfloat16)
        assert torch.equal(y, want) and torch.equal(z, want[at[2]:])
    pkg.experts_free(w)


# ------------------------------------------------------------------ router
def _route_reference(logits, k, renormalize):
    """By the definition, on the host in 64 bits."""
    T, E = logits.shape
    ids, weights = [[-1] * k for _ in range(T)], [[0.0] * k for _ in range(T)]
    biggest = torch.finfo(torch.float32).max
    for t, row in enumerate(logits.float().tolist()):
        row = [-math.inf if v != v else min(v, biggest) for v in row]
        picks = [e for e in sorted(range(E), key=lambda e: (-row[e], e))[:k] if row[e] > -math.inf]
        if picks:
            top = row[picks[0]]
            over = picks if renormalize else [e for e in range(E) if row[e] > -math.inf]
            total = sum(math.exp(row[e] - top) for e in over)
            for j, e in enumerate(picks):
                ids[t][j], weights[t][j] = e, math.exp(row[e] - top) / total
    by_expert = [[(t, j) for t in range(T) for j in range(k) if ids[t][j] == e] for e in range(E)]
    offsets, slots, rows = [0], [[-1] * k for _ in range(T)], []
    for picks in by_expert:
        for t, j in picks:
            slots[t][j] = len(rows)
            rows.append(t)
        offsets.append(len(rows))
    return ids, weights, offsets, slots, rows


def _check_route(pkg, logits, k, renormalize=True):
    T, E = logits.shape
    r = pkg.route_alloc(T + 5, E, k)
    for t in (r.ids, r.slots, r.rows, r.offsets):
        t.fill_(-9)
    pkg.route(r, logits, renormalize=renormalize)
    ids, weights, offsets, slots, rows = _route_reference(logits, k, renormalize)
    assert r.ids[:T].tolist() == ids
    assert r.offsets.tolist() == offsets
    assert r.slots[:T].tolist() == slots
    assert r.rows[:len(rows)].tolist() == rows
    # behind the last slot and the last token: untouched
    assert bool((r.rows[len(rows):] == -9).all()) and bool((r.ids[T:] == -9).all()) and bool((r.slots[T:] == -9).all())
    # exp (2 units and the rounding of its argument: |l| < 64 -> 2^-18), a sum of up to 512 terms, a division
    want = torch.tensor(weights, dtype=torch.float64).reshape(T, k)
    got = r.weights[:T].double().cpu()
    assert bool(((got - want).abs() <= want * 2.0 ** -16 + 1e-30).all())


@pytest.mark.parametrize("T", [1, 2, 31, 32, 33, 64, 65, 200, 1000])
@pytest.mark.parametrize("E,k", [(64, 8), (5, 2)])
def test_route_token_counts(pkg, T, E, k):
    _check_route(pkg, torch.randn((T, E), generator=torch.Generator().manual_seed(T)).cuda() * 2, k)


@pytest.mark.parametrize("E,k", [(1, 1), (2, 2), (8, 8), (31, 3), (32, 4), (33, 5), (65, 1), (127, 16), (129, 7), (256, 8), (257, 6), (512, 16)])
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("T", [3, 70])
def test_route_sizes(pkg, E, k, renormalize, T):
    logits = torch.randn((T, E), generator=torch.Generator().manual_seed(E)).cuda() * 3
    _check_route(pkg, logits, k, renormalize)
    _check_route(pkg, logits.to(torch.bfloat16), k, renormalize)


@pytest.mark.parametrize("T,E,k", [(1184, 64, 8), (1185, 64, 8), (4000, 12, 3), (8192, 20, 2), (8193, 20, 2), (250, 512, 16), (513, 512, 4), (300, 5, 5), (40, 1, 1)])
def test_route_borders_of_its_launches(pkg, T, E, k):
    """Eight tokens to a block or 32, counts added up by every block or in between."""
    _check_route(pkg, torch.randn((T, E), generator=torch.Generator().manual_seed(T)).cuda(), k)


def test_route_many_tokens(pkg):
    _check_route(pkg, torch.randn((9000, 40), generator=torch.Generator().manual_seed(1)).cuda().to(torch.bfloat16), 4)


@pytest.mark.parametrize("T", [6, 100])
def test_route_ties_and_masked_logits(pkg, T):
    """Equal logits go to the lowest index; -inf, NaN, rows with too few experts or none, +inf, the largest finite values of either sign."""
    inf, nan, big = math.inf, math.nan, torch.finfo(torch.float32).max
    E = 40
    logits = torch.randint(-2, 3, (T, E), generator=torch.Generator().manual_seed(3)).float()
    logits[0] = -inf
    logits[1, 2:] = -inf
    logits[2, ::2] = nan
    logits[3] = -big
    logits[3, 7] = -inf
    logits[4, 5], logits[4, 9] = inf, inf
    logits[5] = nan
    logits = logits.cuda()
    _check_route(pkg, logits, 6)
    _check_route(pkg, logits, 6, renormalize=False)


def test_route_no_tokens_and_refusals(pkg):
    r = pkg.route_alloc(40, 8, 2)
    r.offsets.fill_(5)
    pkg.route(r, torch.empty((0, 8), device="cuda"))
    assert r.offsets.tolist() == [0] * 9
    for bad in (torch.zeros((41, 8), device="cuda"), torch.zeros((4, 9), device="cuda"), torch.zeros((4, 8), device="cuda").half(),
                torch.zeros((8, 8), device="cuda").t()[:4], torch.zeros((4, 8))):
        with pytest.raises(pkg.W4A16Error):
            pkg.route(r, bad)
    with pytest.raises(pkg.W4A16Error):
        pkg.route(pkg.route_alloc(4, 8, 9), torch.zeros((4, 8), device="cuda"))
    r.workspace_bytes, r.workspace = 4, r.workspace[:1]
    with pytest.raises(pkg.W4A16Error) as e:
        pkg.route(r, torch.zeros((40, 8), device="cuda"))
    assert e.value.code == -3


# ------------------------------------------------------------------ combination
@pytest.mark.parametrize("T,k,H", [(1, 1, 8), (1, 8, 5120), (3, 9, 1032), (70, 2, 16), (513, 8, 2048), (5, 16, 8200), (2500, 5, 2056), (4000, 8, 1288), (9000, 3, 520), (1000, 2, 5120)])
@pytest.mark.parametrize("residual", [None, "apart", "in place"])
def test_combine(pkg, T, k, H, residual):
    """fp32 sums of k + 1 terms, each rounding at most 2^-24 of the sum of magnitudes (products by fma), then one to bf16."""
    gen = torch.Generator().manual_seed(T + k + H)
    parts = torch.randn((T * k + 3, H), generator=gen).to(torch.bfloat16).cuda()
    slots = torch.randperm(T * k + 3, generator=gen)[:T * k].to(torch.int32).view(T, k)
    empty = torch.rand((T, k), generator=gen) < 0.2
    slots[empty] = -1
    slots, weights = slots.cuda(), torch.rand((T, k), generator=gen).cuda()
    r = torch.randn((T, H), generator=gen).to(torch.bfloat16).cuda() if residual else None
    ref = torch.where(slots.unsqueeze(-1) >= 0, parts[slots.clamp(min=0).long()].double(), 0.0) * weights.double().unsqueeze(-1)
    mass = ref.abs().sum(1) + (r.double().abs() if residual else 0)
    ref = ref.sum(1) + (r.double() if residual else 0)
    out = Guarded((T, H), torch.bfloat16)
    if residual == "in place":
        out.t.copy_(r)
        r = out.t
    pkg.experts_combine(out.t, parts, slots, weights, residual=r)
    assert out.intact()
    assert bool(((out.t.double() - ref).abs() <= ref.abs() * 2.0 ** -8 + mass * ((k + 1) * 2.0 ** -24)).all())


def test_combine_past_four_gigabytes(pkg):
    T, H = 450000, 5120
    parts = torch.empty((T, H), dtype=torch.bfloat16, device="cuda")
    parts[:9], parts[-9:] = whole((9, H), 4, 1), whole((9, H), 4, 2)
    slots = torch.full((T, 2), -1, dtype=torch.int32, device="cuda")
    slots[-4:] = torch.tensor([[0, T - 1], [T - 2, T - 9], [8, -1], [T - 3, T]], dtype=torch.int32)
    y = torch.empty((T, H), dtype=torch.bfloat16, device="cuda")
    pkg.experts_combine(y, parts, slots, torch.ones((T, 2), device="cuda"))
    p = parts[[0, T - 1, T - 2, T - 9, 8, T - 3]].float()
    assert torch.equal(y[-4:].float(), torch.stack([p[0] + p[1], p[2] + p[3], p[4], p[5]]))
    assert int(torch.count_nonzero(y[:-4])) == 0


def test_combine_empty_picks_read_nothing(pkg):
    """A token without picks is its residual, whatever the parts hold; slots outside parts are empty."""
    parts = torch.full((4, 64), float("nan"), dtype=torch.bfloat16, device="cuda")
    r = whole((2, 64), 64, 1)
    y = torch.empty_like(r)
    slots = torch.tensor([[-1, -1], [4, 2 ** 31 - 1]], dtype=torch.int32, device="cuda")
    pkg.experts_combine(y, parts, slots, torch.ones((2, 2), device="cuda"), residual=r)
    assert torch.equal(y, r)
    pkg.experts_combine(y, parts[:0], slots, torch.ones((2, 2), device="cuda"))
    assert bool((y == 0).all())


def test_combine_and_experts_refusals(pkg):
    def refused(fn, *a, **k):
        with pytest.raises(pkg.W4A16Error) as e:
            fn(*a, **k)
        assert e.value.code == -1
        return str(e.value)

    parts = torch.zeros((4, 64), dtype=torch.bfloat16, device="cuda")
    y, slots, weights = parts[:2].clone(), torch.zeros((2, 2), dtype=torch.int32, device="cuda"), torch.ones((2, 2), device="cuda")
    assert "overlaps parts" in refused(pkg.experts_combine, parts[:2], parts, slots, weights)
    assert "multiple of 8" in refused(pkg.experts_combine, y[:, :60].contiguous(), parts[:, :60].contiguous(), slots, weights)
    assert "slots" in refused(pkg.experts_combine, y, parts, slots.long(), weights)
    assert "weights" in refused(pkg.experts_combine, y, parts, slots, weights.double())
    assert "weights" in refused(pkg.experts_combine, y, parts, slots, weights[:1])
    wide = torch.zeros((2, 17), dtype=torch.int32, device="cuda")
    assert "top_k" in refused(pkg.experts_combine, y, parts, wide, wide.float())
    bank = Bank(pkg, 2, 32, 128)
    x, out = whole((4, 128), 4, 1), torch.zeros((4, 32), dtype=torch.bfloat16, device="cuda")
    off, rows = torch.tensor([0, 2, 4], dtype=torch.int32, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    assert "offsets" in refused(pkg.experts_linear, out, bank.w, x, off[:2])
    assert "x_rows" in refused(pkg.experts_linear, out, bank.w, x, off, x_rows=rows[:3])
    assert "without x_rows" in refused(pkg.experts_linear, out, bank.w, x[:3].contiguous(), off)
    assert "activation" in refused(pkg.experts_linear, out, bank.w, x, off, activation=-1)
    assert "overlaps x" in refused(pkg.experts_linear, x.view(-1)[:128].view(4, 32), bank.w, x, off)
    assert "empty" in refused(pkg.experts_linear, out, bank.w, x[:0], off, x_rows=rows)
    assert "bias" in refused(pkg.experts_linear, out, bank.w, x, off, bias=out)
    bank.free()
    for E, rows_, cols in ((0, 32, 128), (513, 32, 128), (2, 24, 128), (2, 32, 100)):
        refused(pkg.experts_alloc, E, rows_, cols)


# ------------------------------------------------------------------ together
def _block(pkg, r, bank1, bank2, x, logits, mid, parts, y):
    pkg.route(r, logits)
    pkg.experts_linear(mid, bank1.w, x, r.offsets, x_rows=r.rows, activation=pkg.ACT_SWIGLU)
    pkg.experts_linear(parts, bank2.w, mid, r.offsets)
    pkg.experts_combine(y, parts, r.slots, r.weights, residual=x)


@pytest.mark.parametrize("T", [1, 13, 150, 700])
def test_a_layer_of_experts(pkg, T):
    """route -> gate|up with SwiGLU -> down -> combine, eagerly, and captured and replayed on other logits, with padded tokens, against the
    chain in 64 bits that rounds where the operators do. What an operator's rounding (2^-8) does to the next one's input adds up over
    the sums: relative to the outputs' deviation 2^-8 for the intermediate, 2^-8 for the parts, 2^-8 for the result, in all under 3 * 2^-8 in
    the 2-norm."""
    E, k, H, I = 12, 4, 512, 256
    bank1, bank2 = Bank(pkg, E, 2 * I, H, "swiglu", 1, False), Bank(pkg, E, H, I, "none", 2, False)
    gen = torch.Generator().manual_seed(T)
    r = pkg.route_alloc(T, E, k)
    mid = torch.full((T * k, I), float("nan"), dtype=torch.bfloat16, device="cuda")
    parts = torch.full((T * k, H), float("nan"), dtype=torch.bfloat16, device="cuda")
    x = torch.randn((T, H), generator=gen).to(torch.bfloat16).cuda()
    logits = torch.empty((T, E), device="cuda")
    y = torch.empty((T, H), dtype=torch.bfloat16, device="cuda")

    def new_logits():
        v = torch.randn((T, E), generator=gen)
        if T > 1:
            v[torch.rand(T, generator=gen) < 0.2] = -math.inf
            v[:, 3] = -math.inf  # an expert that nobody picks
        logits.copy_(v)

    def check():
        assert pkg.device_status() == 0
        ids, weights, *_ = _route_reference(logits.cpu(), k, True)
        ids, weights = torch.tensor(ids, device="cuda"), torch.tensor(weights, dtype=torch.float64, device="cuda")
        ref = torch.zeros((T, H), dtype=torch.float64, device="cuda")
        for e in range(E):
            t, j = (ids == e).nonzero(as_tuple=True)
            if len(t):
                ref.index_add_(0, t, weights[t, j].unsqueeze(1) * bank2.layer64(e, bank1.layer64(e, x[t])))
        moe = y.double() - x.double()
        padded = (ids < 0).all(1)
        assert torch.equal(y[padded], x[padded])
        assert float((moe - ref).norm()) <= 3 * 2.0 ** -8 * float((ref + x.double()).norm())
        return y.clone()

    new_logits()
    _block(pkg, r, bank1, bank2, x, logits, mid, parts, y)
    check()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        _block(pkg, r, bank1, bank2, x, logits, mid, parts, y)
    for _ in range(3):
        new_logits()
        g.replay()
        torch.cuda.synchronize()
        replayed = check()
        _block(pkg, r, bank1, bank2, x, logits, mid, parts, y)
        torch.cuda.synchronize()
        assert torch.equal(y, replayed)
    bank1.free()
    bank2.free()


def test_two_layers_of_experts_on_two_streams(pkg):
    """Two calls in flight at once, each with its own plan and buffers."""
    E, k, H, I, T = 8, 2, 512, 256, 40
    bank1, bank2 = Bank(pkg, E, 2 * I, H, "swiglu", 1, False), Bank(pkg, E, H, I, "none", 2, False)
    sets = []
    for i in range(2):
        gen = torch.Generator().manual_seed(i)
        bufs = [torch.empty(s, dtype=torch.bfloat16, device="cuda") for s in ((T * k, I), (T * k, H), (T, H))]
        x, logits = torch.randn((T, H), generator=gen).to(torch.bfloat16).cuda(), torch.randn((T, E), generator=gen).cuda()
        sets.append((pkg.route_alloc(T, E, k), x, logits, *bufs))
    want = []
    for r, x, logits, mid, parts, y in sets:
        _block(pkg, r, bank1, bank2, x, logits, mid, parts, y)
        want.append(y.clone())
        y.zero_()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):
        for stream, (r, x, logits, mid, parts, y) in zip(streams, sets):
            with torch.cuda.stream(stream):
                _block(pkg, r, bank1, bank2, x, logits, mid, parts, y)
    torch.cuda.synchronize()
    assert all(torch.equal(s[5], w) for s, w in zip(sets, want))
    bank1.free()
    bank2.free()
