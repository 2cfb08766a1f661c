"""Refusals of the operators between sparse rows and dense matrices: every one is made on the host, before any device work."""
import ctypes as C

import pytest
import torch

from sdr_amd import _lib
from sdr_amd._lib import Dense, Rows, WinnersSpec

INVALID, UNSUPPORTED, OVERFLOW = -1, -5, -6
AT = 0x1000   # an address that no refused call follows


def rows(n_rows=4, n_elems=8, offsets=None, ids=AT, weights=None, bits=32):
    return Rows(n_rows, n_elems, offsets, ids, weights, bits)


def dense(n_rows=4, n_cols=16, ld=16, type=0, data=AT):
    return Dense(data, n_rows, n_cols, ld, type)


def spec(k=2, score=0, renormalise=0, groups=1, top_groups=1, group_top=1, scale=1.0, bias=None):
    return WinnersSpec(k, score, renormalise, groups, top_groups, group_top, scale, bias)


BAD_ROWS = [(rows(bits=16), INVALID), (rows(ids=None), INVALID), (rows(n_rows=3), INVALID), (rows(n_rows=0), INVALID),
            (rows(n_rows=2 ** 31), OVERFLOW), (rows(n_elems=2 ** 32), OVERFLOW)]
BAD_DENSE = [(dict(type=3), INVALID), (dict(type=-1), INVALID), (dict(data=None), INVALID), (dict(ld=15), INVALID), (dict(data=AT + 1), INVALID),
             (dict(type=2, data=AT + 1), INVALID), (dict(n_cols=2 ** 24 + 1, ld=2 ** 25), OVERFLOW), (dict(n_rows=2 ** 31), OVERFLOW),
             (dict(ld=2 ** 41), OVERFLOW)]


def refused(rc, code, lib):
    assert rc == code, lib.sdrb_last_error()
    assert lib.sdrb_last_error()


@pytest.mark.parametrize("bad,code", BAD_ROWS)
def test_rows_are_checked(bad, code):
    lib, n = _lib.load(), C.c_size_t()
    table, out = dense(100), dense(bad.n_rows if bad.n_rows < 2 ** 31 else 4)
    refused(lib.sdrb_lookup_scratch(bad, 16, n), code, lib)
    refused(lib.sdrb_lookup(0, bad, table, 1.0, out, None, 0, None), code, lib)
    refused(lib.sdrb_lookup_grad_table_scratch(bad, 100, 16, n), code, lib)
    refused(lib.sdrb_lookup_grad_table(0, bad, out, 1.0, 0, table, AT, 1 << 40, None), code, lib)
    refused(lib.sdrb_lookup_grad_weights(0, bad, out, table, 1.0, AT, None), code, lib)


@pytest.mark.parametrize("bad,code", BAD_DENSE)
def test_matrices_are_checked(bad, code):
    lib = _lib.load()
    m, good = dense(**bad), dense()
    refused(lib.sdrb_lookup(0, rows(), m, 1.0, good, None, 0, None), code, lib)
    refused(lib.sdrb_lookup(0, rows(), good, 1.0, m, None, 0, None), code, lib)
    refused(lib.sdrb_lookup_grad_table(0, rows(), m, 1.0, 0, good, AT, 1 << 40, None), code, lib)
    refused(lib.sdrb_lookup_grad_table(0, rows(), good, 1.0, 0, m, AT, 1 << 40, None), code, lib)
    refused(lib.sdrb_lookup_grad_weights(0, rows(), m, good, 1.0, AT, None), code, lib)
    refused(lib.sdrb_lookup_grad_weights(0, rows(), good, m, 1.0, AT, None), code, lib)
    refused(lib.sdrb_winners(0, m, spec(), AT, AT, None), code, lib)
    refused(lib.sdrb_winners_grad(0, m, spec(), AT, AT, good, None), code, lib)
    refused(lib.sdrb_winners_grad(0, good, spec(), AT, AT, m, None), code, lib)


def test_null_structures_shapes_and_outputs():
    lib, n = _lib.load(), C.c_size_t()
    r, m = rows(), dense()
    for rc in (lib.sdrb_lookup(0, None, m, 1.0, m, None, 0, None), lib.sdrb_lookup(0, r, None, 1.0, m, None, 0, None),
               lib.sdrb_lookup(0, r, m, 1.0, None, None, 0, None), lib.sdrb_lookup_scratch(None, 4, n), lib.sdrb_lookup_scratch(r, 4, None),
               lib.sdrb_lookup_scratch(r, 2 ** 24 + 1, n), lib.sdrb_lookup_grad_table_scratch(r, 2 ** 31, 4, n),
               lib.sdrb_lookup_grad_table(0, r, None, 1.0, 0, m, AT, 1 << 40, None), lib.sdrb_lookup_grad_weights(0, r, m, m, 1.0, None, None),
               lib.sdrb_winners(0, None, spec(), AT, AT, None), lib.sdrb_winners(0, m, None, AT, AT, None),
               lib.sdrb_winners(0, m, spec(), None, AT, None), lib.sdrb_winners(0, m, spec(), AT, None, None),
               lib.sdrb_winners_grad(0, m, spec(), None, AT, m, None), lib.sdrb_winners_grad(0, m, spec(), AT, None, m, None),
               lib.sdrb_batch_rows(None, r),
               # shapes that do not belong together
               lib.sdrb_lookup(0, r, m, 1.0, dense(5), None, 0, None), lib.sdrb_lookup(0, r, m, 1.0, dense(4, 15), None, 0, None),
               lib.sdrb_lookup_grad_table(0, r, dense(5), 1.0, 0, m, AT, 1 << 40, None),
               lib.sdrb_lookup_grad_table(0, r, dense(4, 15), 1.0, 0, m, AT, 1 << 40, None),
               lib.sdrb_lookup_grad_weights(0, r, dense(5), m, 1.0, AT, None), lib.sdrb_lookup_grad_weights(0, r, dense(4, 15), m, 1.0, AT, None),
               lib.sdrb_winners_grad(0, m, spec(), AT, AT, dense(5), None), lib.sdrb_winners_grad(0, m, spec(), AT, AT, dense(4, 15), None)):
        refused(rc, INVALID, lib)


@pytest.mark.parametrize("bad,code", [(dict(k=0), INVALID), (dict(k=17), INVALID), (dict(score=2), INVALID), (dict(score=-1), INVALID),
                                      (dict(groups=0), INVALID), (dict(groups=3), INVALID), (dict(groups=4, top_groups=5), INVALID),
                                      (dict(groups=4, top_groups=0), INVALID), (dict(group_top=0), INVALID), (dict(group_top=3), INVALID),
                                      (dict(k=1025), UNSUPPORTED), (dict(groups=257), UNSUPPORTED)])
def test_the_winners_spec_is_checked(bad, code):
    lib, m = _lib.load(), dense()
    refused(lib.sdrb_winners(0, m, spec(**bad), AT, AT, None), code, lib)
    refused(lib.sdrb_winners_grad(0, m, spec(**bad), AT, AT, m, None), code, lib)
    refused(lib.sdrb_winners(0, dense(4, 16385, 16385), spec(), AT, AT, None), UNSUPPORTED, lib)


def test_scratch_is_asked_for_and_checked():
    lib, n = _lib.load(), C.c_size_t(7)
    assert lib.sdrb_lookup_scratch(rows(), 16, n) == 0 and n.value == 0
    long_rows = rows(n_rows=3, n_elems=100_000, offsets=AT)
    assert lib.sdrb_lookup_scratch(long_rows, 16, n) == 0 and n.value > 0
    refused(lib.sdrb_lookup(0, long_rows, dense(9), 1.0, dense(3), None, 0, None), INVALID, lib)
    refused(lib.sdrb_lookup(0, long_rows, dense(9), 1.0, dense(3), AT, n.value - 1, None), INVALID, lib)
    refused(lib.sdrb_lookup(0, long_rows, dense(9), 1.0, dense(3), AT + 4, n.value, None), INVALID, lib)
    assert lib.sdrb_lookup_grad_table_scratch(rows(), 50, 16, n) == 0 and n.value > 0
    refused(lib.sdrb_lookup_grad_table(0, rows(), dense(), 1.0, 0, dense(50), None, 0, None), INVALID, lib)
    refused(lib.sdrb_lookup_grad_table(0, rows(), dense(), 1.0, 0, dense(50), AT, n.value - 1, None), INVALID, lib)


def test_nothing_to_do_is_no_error():
    lib = _lib.load()
    none = rows(n_rows=0, n_elems=0, ids=None)
    assert lib.sdrb_lookup(0, none, dense(), 1.0, dense(0, data=None), None, 0, None) == 0
    assert lib.sdrb_lookup_grad_weights(0, none, dense(0, data=None), dense(), 1.0, None, None) == 0
    assert lib.sdrb_lookup_grad_table(0, rows(), dense(), 1.0, 0, dense(0, data=None), None, 0, None) == 0
    assert lib.sdrb_winners(0, dense(0, data=None), spec(), None, None, None) == 0


def test_python_refuses_tensors_that_are_not_on_a_gpu():
    import sdr_amd
    ids, t = torch.zeros(3, dtype=torch.int32), torch.zeros(4, 5)
    for call in (lambda: sdr_amd.lookup(ids, t), lambda: sdr_amd.lookup_grad_table(ids, torch.zeros(3, 5), 4),
                 lambda: sdr_amd.lookup_grad_weights(ids, torch.zeros(3, 5), t), lambda: sdr_amd.winners(t, 2),
                 lambda: sdr_amd.winners_grad(t, ids.view(1, 3), torch.zeros(1, 3))):
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("k", [1, 2, 63, 64])
def test_rows_of_up_to_64_ids_need_no_scratch(k):
    """where they have equal lengths: calls with the ids of winners, or of tokens, rely on it"""
    lib, n = _lib.load(), C.c_size_t(1)
    for n_rows in (1, 3, 64, 65, 4096, 100_000, 60_000_000):
        if n_rows * k < 2 ** 32:
            assert lib.sdrb_lookup_scratch(rows(n_rows=n_rows, n_elems=n_rows * k), 2048, n) == 0 and n.value == 0
