"""CPU: what fwb_beam_reorder_dev says of states whose bytes meet, before any device work."""
import pytest

from fwb import native

PTR = 1 << 20   # an address that is never read: the parents' is misaligned, which is refused after the overlaps
ARGS = dict(src=PTR, dst=PTR, parent=PTR + 2, n_outer=2, n_group=1, n_beam=4, n_inner=3, run=64, so=4096, ss=1024, si=128,
            do=4096, ds=1024, di=128)


@pytest.fixture(scope="module")
def lib(built):
    return native.product()


@pytest.mark.parametrize("state", [
    dict(ss=0), dict(ss=32), dict(si=0), dict(si=63), dict(so=0), dict(so=1024), dict(ss=128, si=1024, so=300),
    dict(so=1 << 63), dict(ss=256),
], ids=lambda d: ",".join(f"{k}={v}" for k, v in d.items()))
@pytest.mark.parametrize("place", ["in", "out"])
def test_a_destination_that_overlaps_itself(lib, state, place):
    """An expanded view, or rows nearer than they are long: threads would write the same bytes."""
    bad = {**state, **{"d" + k[1]: v for k, v in state.items()}}
    if place == "out":
        bad = {**{k: v for k, v in bad.items() if k[0] == "d"}, "dst": PTR << 20}
    assert lib.fwb_beam_reorder_dev(*{**ARGS, **bad}.values(), None) == -1
    assert "overlap one another" in lib.fwb_last_error().decode()


def touched(base, a):
    return {base + o * a["so"] + s * a["ss"] + i * a["si"] + b for o in range(a["n_outer"])
            for s in range(a["n_group"] * a["n_beam"]) for i in range(a["n_inner"]) for b in range(a["run"])}


@pytest.mark.parametrize("layout", [
    dict(n_outer=2, n_beam=3, n_inner=2, run=4, so=60, ss=20, si=8), dict(n_outer=3, n_beam=2, n_inner=1, run=4, so=16, ss=8, si=0),
    dict(n_outer=2, n_beam=3, n_inner=2, run=4, so=8, ss=48, si=20), dict(n_outer=1, n_beam=4, n_inner=3, run=8, so=0, ss=64, si=16),
], ids=str)
def test_states_in_each_others_gaps(lib, layout):
    """Refused exactly where a byte is shared; the others come to the parents' address."""
    a = {**ARGS, **layout}
    a.update(do=a["so"], ds=a["ss"], di=a["si"])
    mine = touched(0, a)
    seen = set()
    for off in range(-200, 201):
        if off == 0:
            continue
        meet = bool(mine & touched(off, a))
        assert lib.fwb_beam_reorder_dev(*{**a, "dst": PTR + off}.values(), None) == -1
        assert ("overlap" in lib.fwb_last_error().decode()) == meet, off
        seen.add(meet)
    assert seen == {False, True}
