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


def test_an_output_that_is_its_input_is_refused():
    """by the library, before any device work: gradients of winners would be read from the zeros that they are written over"""
    from sdr_amd import _lib
    from sdr_amd._lib import Dense, Rows, WinnersSpec
    lib, at, other = _lib.load(), 0x1000, 0x9000
    m, apart, r, spec = Dense(at, 4, 16, 16, 0), Dense(other, 4, 16, 16, 0), Rows(4, 8, None, other, None, 32), WinnersSpec(2, 0, 0, 1, 1, 1, 1.0, None)
    for rc, name in ((lambda: lib.sdrb_lookup(0, r, m, 1.0, m, None, 0, None), b"table"),
                     (lambda: lib.sdrb_lookup_grad_table(0, r, m, 1.0, 0, m, other, 1 << 40, None), b"grad"),
                     (lambda: lib.sdrb_winners_grad(0, m, spec, other, other, m, None), b"scores")):
        assert rc() == -1
        assert b"out is " + name + b" itself" in lib.sdrb_last_error()
    # no refusal where one of them holds nothing
    none = Dense(at, 0, 16, 16, 0)
    assert lib.sdrb_lookup(0, Rows(0, 0, None, None, None, 32), m, 1.0, none, None, 0, None) == 0
    # and what lies apart comes as far as the next check
    assert lib.sdrb_lookup_grad_table(0, r, m, 1.0, 0, apart, None, 0, None) == -1 and b"scratch" in lib.sdrb_last_error()
