"""Refusals of the feed-forward operators that the library makes before it touches a device, and the sizes it states."""
import ctypes as C

import test_ring_handback


def _weights(pkg, rows=128, cols=256):
    w = pkg.Weights()
    w.qweight = w.scale = w.zp = 4096  # never read: every call below is refused or empty
    w.out_f, w.in_f, w.group_size, w.num_groups = rows, cols, 128, cols // 128
    return w


def _experts(pkg, **fields):
    w = pkg.Experts(4096, 4, 128, 256, 128, 2)
    for name, v in fields.items():
        setattr(w, name, v)
    return w


def test_one_lane_arrives_behind_a_syncwarp(monkeypatch):
    monkeypatch.setattr(test_ring_handback, "HANDED_OVER", ("ready_a", "empty_a"))
    seen = list(test_ring_handback._arrivals("ragged.cu"))
    assert [bar for _, bar, _ in seen] == ["ready_a", "empty_a"] and all(before == "__syncwarp();" for *_, before in seen)


def test_struct_layout(pkg):
    assert C.sizeof(pkg.Experts) == 32  # pointer + 5 ints (+ pad)


def test_linear_epilogue_refusals(pkg):
    L, w = pkg.lib(), _weights(pkg)
    y, x = 1 << 20, 1 << 24

    def call(y=y, w=w, x=x, M=4, bias=None, act=0, residual=None):
        return L.w4a16_linear_epilogue(y, C.byref(w), x, M, bias, act, residual, None)

    assert call(M=0) == 0
    assert call(M=-1) == -1 and b"M = -1" in L.w4a16_last_error()
    assert call(act=5) == -1 and b"activation" in L.w4a16_last_error()
    assert call(act=-1) == -1
    assert call(w=_weights(pkg, 144), act=4) == -1 and b"multiple of 32" in L.w4a16_last_error()
    assert call(x=None) == -1 and call(y=None) == -1
    assert call(x=x + 8) == -1 and call(y=y + 2) == -1 and call(residual=y + 4) == -1 and call(bias=x + 1) == -1
    assert call(x=y + 4 * 128 * 2 - 16) == -1 and b"overlaps x" in L.w4a16_last_error()
    assert call(residual=y + 16) == -1 and b"is not y" in L.w4a16_last_error()
    assert call(bias=y + 2) == -1 and b"overlaps bias" in L.w4a16_last_error()
    w.group_size = 64
    assert call() == -1


def test_experts_refusals(pkg):
    L = pkg.lib()
    w = pkg.Experts()
    for E, rows, cols, group in ((0, 128, 256, 128), (513, 128, 256, 128), (4, 100, 256, 128), (4, 128, 200, 128), (4, 128, 256, 32), (4, 128, 256, 0), (4, 0, 256, 128)):
        assert L.w4a16_experts_alloc(C.byref(w), E, rows, cols, group, None) == -1
    assert L.w4a16_experts_alloc(None, 1, 128, 128, 128, None) == -1
    view = pkg.Weights()
    good = _experts(pkg)
    assert L.w4a16_experts_view(C.byref(good), 3, C.byref(view)) == 0
    block = 8576 * 2
    assert view.qweight == 4096 + 3 * block and (view.out_f, view.in_f, view.num_groups) == (128, 256, 2)
    assert L.w4a16_weights_free(C.byref(view)) == -1 and b"view" in L.w4a16_last_error()
    assert L.w4a16_experts_view(C.byref(good), 4, C.byref(view)) == -1
    assert L.w4a16_experts_view(C.byref(good), -1, C.byref(view)) == -1
    assert L.w4a16_experts_view(C.byref(_experts(pkg, qweight=None)), 0, C.byref(view)) == -1

    def call(w=good, y=1 << 20, x=1 << 24, tokens=8, rows=None, offsets=1 << 28, slots=8, bias=None, act=0):
        return L.w4a16_experts_linear(y, C.byref(w), x, tokens, rows, offsets, slots, bias, act, None)

    assert call(slots=0) == 0
    assert call(offsets=None) == -1
    assert call(slots=-1) == -1 and call(tokens=-1) == -1
    assert call(slots=9) == -1 and b"x_rows" in L.w4a16_last_error()
    assert call(offsets=(1 << 28) + 2) == -1 and call(rows=(1 << 28) + 1) == -1
    assert call(tokens=0, rows=1 << 29) == -1
    assert call(act=9) == -1
    assert call(w=_experts(pkg, num_experts=0)) == -1 and call(w=_experts(pkg, num_groups=3)) == -1
    assert call(w=_experts(pkg, out_f=112), act=4) == -1
    assert call(offsets=(1 << 20) + 16) == -1 and b"overlaps offsets" in L.w4a16_last_error()
    assert call(rows=(1 << 20) - 28) == -1 and b"x_rows" in L.w4a16_last_error()


def test_route_and_combine_refusals(pkg):
    L = pkg.lib()
    assert L.w4a16_route_workspace(32, 64) == 2 * 64 * 4 and L.w4a16_route_workspace(33, 64) == 3 * 64 * 4
    assert L.w4a16_route_workspace(10, 0) == 0 and L.w4a16_route_workspace(10, 513) == 0 and L.w4a16_route_workspace(-1, 8) == 0
    p = 1 << 20

    def route(ids=p, weights=p, offsets=p, slots=p, rows=p, logits=p, f32=1, T=4, E=8, k=2, ws=p, nbytes=1 << 16):
        return L.w4a16_route(ids, weights, offsets, slots, rows, logits, f32, T, E, k, 1, ws, nbytes, None)

    assert route(E=0) == -1 and route(E=513) == -1
    assert route(k=0) == -1 and route(k=9) == -1 and route(E=64, k=17) == -1
    assert route(T=-1) == -1 and route(T=2 ** 31 - 1) == -1
    assert route(offsets=None, T=0) == -1
    for name in ("ids", "weights", "slots", "rows", "logits"):
        assert route(**{name: None}) == -1
        assert route(**{name: p + 2}) == -1
    assert route(logits=p + 1, f32=0) == -1
    assert route(T=33, nbytes=2 * 8 * 4) == -3 and route(T=33, ws=None) == -3
    assert L.w4a16_route_workspace(2 ** 31 - 1, 8) == (2 ** 26 + 1) * 8 * 4 and route(T=2 ** 31 - 1, k=1) == -3

    def combine(y=p, parts=1 << 24, n=8, slots=1 << 26, weights=1 << 27, residual=None, T=4, k=2, H=64):
        return L.w4a16_experts_combine(y, parts, n, slots, weights, residual, T, k, H, None)

    assert combine(T=0) == 0
    assert combine(T=-1) == -1 and combine(n=-1) == -1 and combine(k=0) == -1 and combine(k=17) == -1
    assert combine(H=60) == -1 and combine(H=0) == -1
    assert combine(y=None) == -1 and combine(slots=None) == -1 and combine(weights=None) == -1 and combine(parts=None) == -1
    assert combine(y=p + 8) == -1 and combine(parts=(1 << 24) + 2) == -1 and combine(slots=p + 2) == -1
    assert combine(parts=p + 4 * 64 * 2 - 16) == -1 and combine(residual=p + 16) == -1
    assert combine(slots=p - 4) == -1 and b"overlaps slots" in L.w4a16_last_error()
    assert combine(weights=p + 508) == -1 and b"overlaps slots" in L.w4a16_last_error()
