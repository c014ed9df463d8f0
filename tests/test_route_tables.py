"""Where the router's Python call writes: into memory that its Route owns, whatever a caller does with the tensors that show it. On the
CPU, with the library's call replaced by one that notes its arguments."""
import copy

import pytest
import torch


@pytest.fixture
def route(pkg, monkeypatch):
    """make(...) -> a Route on the CPU; calls: the five addresses of every call."""
    real, zeros, calls = pkg.lib(), torch.zeros, []

    class Noting:
        w4a16_route_workspace = real.w4a16_route_workspace

        @staticmethod
        def w4a16_route(*args):
            calls.append(args[:5])
            return 0

    monkeypatch.setattr(torch, "zeros", lambda *a, device=None, **k: zeros(*a, **k))
    monkeypatch.setattr(pkg, "lib", lambda: Noting)
    monkeypatch.setattr(pkg, "_device", lambda: -1)
    monkeypatch.setattr(pkg, "_stream_of", lambda stream, dev: None)
    for name, kind in (("_BF16", torch.bfloat16), ("_F32", torch.float32), ("_I32", torch.int32)):
        monkeypatch.setattr(pkg, name, kind)
    return pkg.route_alloc, calls


def _tables(r):
    return [r.ids, r.weights, r.offsets, r.slots, r.rows]


@pytest.mark.parametrize("tokens,E,k", [(1, 1, 1), (5, 7, 3), (33, 64, 8), (0, 8, 2)])
def test_tables_are_apart_and_the_call_gets_them(pkg, route, tokens, E, k):
    make, calls = route
    r = make(tokens, E, k)
    assert [tuple(t.shape) for t in _tables(r)] == [(tokens, k), (tokens, k), (E + 1,), (tokens, k), (tokens * k,)]
    assert r.weights.dtype == torch.float32 and all(t.dtype == torch.int32 for t in (r.ids, r.offsets, r.slots, r.rows))
    for i, t in enumerate(_tables(r)):
        t.fill_(i + 1)
    assert all(bool((t == i + 1).all()) and t.is_contiguous() for i, t in enumerate(_tables(r)))
    pkg.route(r, torch.zeros((tokens, E)))
    for t, address in zip(_tables(r), calls[-1]):
        assert t.numel() == 0 or t.data_ptr() == address
        assert address % 16 == r._memory.data_ptr() % 16


@pytest.mark.parametrize("name", ["ids", "weights", "offsets", "slots", "rows"])
def test_another_tensor_in_a_tables_place_is_refused(pkg, route, name):
    make, calls = route
    r = make(5, 7, 3)
    before = getattr(r, name)
    with pytest.raises(pkg.W4A16Error) as e:
        setattr(r, name, before * 2)
    assert e.value.code == -1 and name in str(e.value)
    with pytest.raises(pkg.W4A16Error):
        setattr(r, name, None)
    assert getattr(r, name) is before
    pkg.route(r, torch.zeros((5, 7)))
    assert [t.data_ptr() for t in _tables(r)] == list(calls[-1])


def test_its_sizes_stay(pkg, route):
    make, _ = route
    r = make(5, 7, 3)
    for name, value in (("max_tokens", 500), ("num_experts", 70), ("top_k", 4)):
        with pytest.raises(pkg.W4A16Error):
            setattr(r, name, value)
    with pytest.raises(pkg.W4A16Error):
        pkg.route(r, torch.zeros((6, 7)))


def test_contents_may_be_changed_in_place(pkg, route):
    make, calls = route
    r = make(5, 7, 3)
    r.weights.fill_(3)
    r.weights *= 2
    r.weights[1:2] += 1
    assert float(r.weights[0, 0]) == 6 and float(r.weights[1, 0]) == 7
    pkg.route(r, torch.zeros((5, 7)))
    assert calls[-1][1] == r.weights.data_ptr()


def test_a_table_with_other_memory_leaves_the_calls_where_they_were(pkg, route):
    """Even a tensor whose storage is swapped or grown: the call writes into what the Route holds at that time."""
    make, calls = route
    for spoil in (lambda r: setattr(r.weights, "data", torch.ones(1)), lambda r: r.rows.resize_(10 ** 6), lambda r: delattr(r, "ids")):
        r = make(5, 7, 3)
        spoil(r)
        pkg.route(r, torch.zeros((5, 7)))
        lo, size = r._memory.data_ptr(), r._memory.numel() * 4
        assert all(lo <= address and address + 4 * n <= lo + size for address, n in zip(calls[-1], (15, 15, 8, 15, 15)))


def test_another_device_is_refused(pkg, route, monkeypatch):
    """Whatever logits and workspace are handed over there."""
    make, calls = route
    r = make(5, 7, 3)
    monkeypatch.setattr(pkg, "_device", lambda: 1)
    monkeypatch.setattr(pkg, "_want", lambda *a: None)
    with pytest.raises(pkg.W4A16Error) as e:
        pkg.route(r, torch.zeros((5, 7)))
    assert "device" in str(e.value) and not calls


def test_copies_have_memory_of_their_own(pkg, route):
    make, calls = route
    r = make(5, 7, 3)
    other = copy.deepcopy(r)
    pkg.route(other, torch.zeros((5, 7)))
    assert [t.data_ptr() for t in _tables(other)] == list(calls[-1]) and other.ids.data_ptr() != r.ids.data_ptr()


def test_sizes_that_make_no_sense(pkg, route):
    make, _ = route
    for sizes in ((-1, 8, 2), (4, 0, 1), (4, 8, 0)):
        with pytest.raises(pkg.W4A16Error):
            make(*sizes)
