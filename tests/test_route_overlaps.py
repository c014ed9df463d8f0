"""The router's tables, its logits and its workspace have to be apart: its second launch takes experts and counts for indices. Refused on the
host, before a device is touched."""
import pytest

TABLES = ("ids", "weights", "offsets", "slots", "rows", "logits", "workspace")
T, E, K = 40, 16, 2  # (two blocks of tokens: the workspace is used)
SIZES = {"ids": T * K * 4, "weights": T * K * 4, "offsets": (E + 1) * 4, "slots": T * K * 4, "rows": T * K * 4, "logits": T * E * 4,
         "workspace": 3 * E * 4}


def _call(pkg, where, tokens=T, f32=1):
    return pkg.lib().w4a16_route(*[where[n] for n in ("ids", "weights", "offsets", "slots", "rows", "logits")], f32, tokens, E, K, 1,
                                 where["workspace"], SIZES["workspace"], None)


@pytest.mark.parametrize("one", TABLES)
@pytest.mark.parametrize("other", TABLES)
def test_overlaps_are_refused(pkg, one, other):
    if one == other:
        return
    for shift in (0, 4, SIZES[other] - 4, 4 - SIZES[one]):  # one begins in the other, or ends in it
        where = {n: (i + 1) << 20 for i, n in enumerate(TABLES)}
        where[one] = where[other] + shift
        assert _call(pkg, where) == -1, (one, other, shift)
        assert b"overlap" in pkg.lib().w4a16_last_error()


def test_bf16_logits_are_half_as_long(pkg):
    where = {n: (i + 1) << 20 for i, n in enumerate(TABLES)}
    where["ids"] = where["logits"] + T * E * 2 - 4
    assert _call(pkg, where, f32=0) == -1 and b"logits" in pkg.lib().w4a16_last_error()
