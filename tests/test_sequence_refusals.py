"""Calls of the sequence operators that are refused before anything reaches a device."""
import pytest

import arraymancer_amd as am
from arraymancer_amd import _lib
from test_sequence import attention_args, backward_args


@pytest.mark.parametrize("sfx", ["f32", "f64"])
@pytest.mark.parametrize("entry,args,change", [("decay_attention", attention_args, dict(ot=7)), ("decay_attention", attention_args, dict(ot=-1)),
                                               ("decay_attention_backward", backward_args, dict(dqt=7)), ("decay_attention_backward", backward_args, dict(dkt=-7)),
                                               ("decay_attention_backward", backward_args, dict(dvt=1))], ids=str)
def test_results_whose_tokens_overlap(entry, args, change, sfx):
    """Rows of 8 elements nearer to each other than that."""
    assert getattr(am.load_library(), f"am_hip_{entry}_{sfx}")(*args(**change)) == _lib.AM_E_SHAPE
    assert "overlap" in _lib.last_error()
