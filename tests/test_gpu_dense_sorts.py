"""The table's gradient on both sides of every choice of its sort: one block or many, one pass or two, sums over runs or over ids,
with elements that contribute nothing -- and whatever the scratch held before the call.  Gradients and weights are small integers,
so that sums in binary32 are exact and results have to be equal."""
import ctypes as C

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DIM = 20


def _elements(g, form, n, n_table):
    """(ids, offsets, row of every element or -1, rows): a sixth of the ids lie outside the table, on either side"""
    ids = (torch.rand(n, generator=g) ** 3 * n_table).long()
    stray = torch.rand(n, generator=g)
    ids = torch.where(stray < 0.1, -1, torch.where(stray > 0.95, n_table + torch.randint(0, 3, (n,), generator=g), ids))
    if form == "tokens":
        return ids, None, torch.arange(n), n
    if form == "rows":
        k = next(k for k in (16, 17, 11, 13, 7, 1) if n % k == 0)
        return ids.view(-1, k), None, torch.arange(n) // k, n // k
    before, behind, lens = 37, 61, []
    while sum(lens) < n - before - behind:   # ragged rows, some of them empty, and elements that no row holds
        lens.append(int(torch.randint(0, 9, (1,), generator=g)))
    lens[-1] -= sum(lens) - (n - before - behind)
    offsets = torch.tensor([before] + [before + int(m) for m in np.cumsum(lens)], dtype=torch.int32)
    row = torch.full((n,), -1)
    row[before:n - behind] = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor(lens))
    return ids, offsets, row, len(lens)


def _want(ids, row, weights, grad, n_table):
    ids = ids.reshape(-1)
    on = (ids >= 0) & (ids < n_table) & (row >= 0)
    terms = grad.double()[row[on]] * (1.0 if weights is None else weights.reshape(-1)[on].double()[:, None])
    return torch.zeros(n_table, grad.shape[1], dtype=torch.float64).index_add_(0, ids[on], terms)


def _by_c(ids, offsets, weights, grad, out, accumulate, fill):
    """the C call, its scratch filled by `fill`"""
    from sdr_amd import _lib
    lib, need = _lib.load(), C.c_size_t()
    n_rows = offsets.numel() - 1 if offsets is not None else ids.shape[0]
    rows = _lib.Rows(n_rows, ids.numel(), None if offsets is None else offsets.data_ptr(), ids.data_ptr(),
                     None if weights is None else weights.data_ptr(), 64 if ids.dtype == torch.int64 else 32)
    g = _lib.Dense(grad.data_ptr(), *grad.shape, grad.shape[1], 0)
    o = _lib.Dense(out.data_ptr(), *out.shape, out.shape[1], 0)
    _lib.check(lib.sdrb_lookup_grad_table_scratch(rows, out.shape[0], out.shape[1], need))
    words = (need.value + 3) // 4
    scratch = fill(words).to(torch.int32).cuda()
    _lib.check(lib.sdrb_lookup_grad_table(0, rows, g, 1.0, int(accumulate), o, scratch.data_ptr(), need.value,
                                          torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    return out


@pytest.mark.parametrize("form", ["tokens", "rows", "ragged"])
@pytest.mark.parametrize("n_table", [1365, 1400, 2048, 3000, 4095, 4096, 4097])
@pytest.mark.parametrize("n", [4096, 4097, 8000, 8193, 12287])
def test_elements_that_contribute_nothing_at_every_choice_of_the_sort(n, n_table, form):
    import sdr_amd
    g = torch.Generator().manual_seed(n * 7 + n_table)
    ids, offsets, row, n_rows = _elements(g, form, n, n_table)
    grad = torch.randint(-40, 40, (n_rows, DIM), generator=g).float()
    weights = torch.randint(-3, 4, ids.shape, generator=g).float()
    start = torch.randint(-9, 9, (n_table, DIM), generator=g).float()
    on_gpu = (ids.cuda(), None if offsets is None else offsets.cuda())
    for w in (None, weights):
        w_gpu = None if w is None else w.cuda()
        want = _want(ids, row, w, grad, n_table)
        got = sdr_amd.lookup_grad_table(on_gpu[0], grad.cuda(), n_table, w_gpu, offsets=on_gpu[1])
        assert torch.equal(got.cpu().double(), want)
        into = start.cuda()
        sdr_amd.lookup_grad_table(on_gpu[0], grad.cuda(), weights=w_gpu, offsets=on_gpu[1], out=into, accumulate=True)
        assert torch.equal(into.cpu().double(), want + start.double())


FILLS = {"zeros": lambda words: torch.zeros(words), "a valid key": lambda words: torch.full((words,), 1234),
         "the last key": lambda words: torch.full((words,), 1399), "ones": lambda words: torch.full((words,), -1),
         "rising keys": lambda words: torch.arange(words) * 1400 // words}


@pytest.mark.parametrize("fill", sorted(FILLS))
@pytest.mark.parametrize("n,n_table", [(4000, 1400), (4097, 1400), (8000, 3000), (8192, 4096), (12287, 4096), (9000, 5000), (16000, 1400)])
def test_the_scratch_may_hold_anything(n, n_table, fill):
    g = torch.Generator().manual_seed(n + n_table)
    for form in ("tokens", "ragged"):
        ids, offsets, row, n_rows = _elements(g, form, n, n_table)
        grad = torch.randint(-40, 40, (n_rows, DIM), generator=g).float()
        weights = torch.randint(-3, 4, ids.shape, generator=g).float()
        want = _want(ids, row, weights, grad, n_table)
        for accumulate in (False, True):
            out = torch.ones(n_table, DIM, device="cuda")
            _by_c(ids.int().cuda(), None if offsets is None else offsets.cuda(), weights.cuda(), grad.cuda(), out, accumulate, FILLS[fill])
            assert torch.equal(out.cpu().double(), want + 1 if accumulate else want)


def test_one_scratch_for_full_and_padded_calls_in_turn():
    """a graph's scratch holds what its last replay left: a step of padded tokens follows one without padding"""
    import sdr_amd
    g = torch.Generator().manual_seed(4)
    n, n_table = 8192, 4096
    grad = torch.randint(-40, 40, (n, DIM), generator=g).float().cuda()
    ids = torch.zeros(n, dtype=torch.int64, device="cuda")
    steps = []
    for padded in (0, 64, 0, 200, 512):
        drawn = torch.randint(0, n_table, (n,), generator=g)
        steps.append(torch.where(torch.arange(n) % 512 >= 512 - padded, -1, drawn))
    sdr_amd.lookup_grad_table(ids, grad, n_table)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = sdr_amd.lookup_grad_table(ids, grad, n_table)
    for step in steps:
        ids.copy_(step)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.cpu().double(), _want(step, torch.arange(n), None, grad.cpu(), n_table))
