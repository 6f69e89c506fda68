"""What the host layer keeps between the pieces of one call (no GPU needed)."""
import pytest
import torch

from hils_attention_b200 import _lib


def test_a_refused_type_leaves_no_devices_behind():
    """The devices of a call that was given up are not the next call's, which may run elsewhere."""
    for t in (torch.zeros(2, dtype=torch.float16), torch.zeros(2, dtype=torch.float64)):
        _lib._pending().append(torch.device("cuda:1"))
        with pytest.raises(TypeError):
            _lib.dtype_code(t)
        assert _lib._pending() == []


def test_a_refused_call_is_not_counted_as_launched():
    before = _lib.launch_count()
    with pytest.raises(_lib.HilsError) as e:
        _lib.call("hils_draft_positions", None, None, None, 1, 65, None)
    assert e.value.status == -1 and _lib.launch_count() == before
    _lib.call("hils_draft_positions", None, None, None, 0, 4, None)
    assert _lib.launch_count() == before + 1
