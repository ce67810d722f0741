"""More refusals of include/spiky_lm_tokens.h's entries, which need no device."""
import pytest

from spiky_amd import _native


def refuse(status, message):
    with pytest.raises(ValueError, match=message):
        _native.check_lm(status)


@pytest.mark.parametrize("change", [dict(out_search=32), dict(out_beam=16), dict(out_run=12), dict(in_run=0)])
def test_reorder_in_place_has_one_layout(change):
    """Equal pointers mean in place, where other strides would let one beam's store pass another's load."""
    same = dict(runs=2, run_bytes=8, in_search=48, out_search=48, in_beam=8, out_beam=8, in_run=24, out_run=24)
    s = _native.LmState(**{"in": 16, "out": 16, **same, **change})
    refuse(_native.lib().spiky_lm_reorder(s, 1, 16, 1, 2, 3, 3, None), "both strides must be the same")
    # strides of one index alone are not used
    s = _native.LmState(**{"in": 16, "out": 16, **same, "out_search": 1, "out_beam": 2, "run_bytes": 0})
    assert _native.lib().spiky_lm_reorder(s, 1, 16, 1, 1, 1, 1, None) == 0
