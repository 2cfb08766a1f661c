"""Refusals of the Python side that need no GPU."""
import pytest
import torch


def test_from_winners_refuses_what_is_not_on_a_gpu():
    from sdr_amd import SDRBatch
    ids = torch.zeros(2, 3, dtype=torch.int32)
    for weights in (None, torch.zeros(2, 3)):
        with pytest.raises(ValueError):
            SDRBatch.from_winners(ids, weights, width=9)
    for bad in (ids[0], ids.long()):
        with pytest.raises(ValueError):
            SDRBatch.from_winners(bad)
    with pytest.raises(ValueError):
        SDRBatch.from_winners(ids, torch.zeros(2, 4))
