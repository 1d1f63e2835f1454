"""Uses of the packed attention and the relative position bias at the edge of
what they accept, without a GPU."""
import types

import pytest
import torch


def _check_status(monkeypatch, word):
    import mergenet_b200 as mn
    from mergenet_b200.model import MergeNetSmall
    monkeypatch.setattr(mn.attention, "attention_status", lambda device=None, reset=False: word)
    MergeNetSmall.check_status(types.SimpleNamespace(), torch.zeros(1, dtype=torch.int32))


def test_bad_offsets_of_another_call_are_not_the_models_error(monkeypatch):
    from mergenet_b200 import _lib as L
    _check_status(monkeypatch, 0)
    _check_status(monkeypatch, L.MN_STATUS_BAD_LENGTHS)


@pytest.mark.parametrize("more", [0, 512])
def test_a_models_status_names_the_timeout(monkeypatch, more):
    from mergenet_b200 import _lib as L
    with pytest.raises(RuntimeError, match="0x100 .*gave up"):
        _check_status(monkeypatch, L.MN_STATUS_TC_TIMEOUT | more)
    with pytest.raises(RuntimeError, match="unknown"):
        _check_status(monkeypatch, 1 << 20 | more)
