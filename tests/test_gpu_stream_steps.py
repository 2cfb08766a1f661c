"""Calls made of several steps on an explicit stream: torch's own steps between the kernels belong to that stream as well.  The
stream is behind by other work when the calls are made, and the current stream idle."""
import numpy as np
import pytest
import torch

from util import ragged_rows

pytestmark = pytest.mark.gpu


def _pair(kind):
    from sdr_amd import SDRBatch
    made = []
    for seed in (1, 2):
        rng = np.random.default_rng(seed)
        off, ids = ragged_rows(rng, 300, 500, 40)[:2]
        ids = np.asarray(ids, dtype=np.int32)
        data = None if kind == "empty" else rng.random(len(ids)).astype(np.float32)
        made.append(SDRBatch.from_csr(off, ids, data, width=500, kind=kind))
    return made


def _late_stream():
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        a = torch.randn(4096, 4096, device="cuda", dtype=torch.bfloat16)
        for _ in range(200):
            a = (a @ a) * 2.0 ** -12
    return stream


def _equal(a, b):
    return all((x is None and y is None) or np.array_equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("by_handle", [False, True])
@pytest.mark.parametrize("kind", ["unit", "arith"])
def test_rmi_with_a_combiner(kind, by_handle):
    combine = lambda t, a: t * 0.5 - a * 0.25  # noqa: E731
    mine, other = _pair(kind)
    want, _ = _pair(kind)
    want.rmi(other, combine=combine)
    torch.cuda.synchronize()
    stream = _late_stream()
    mine.rmi(other, combine=combine, stream=stream.cuda_stream if by_handle else stream)
    torch.cuda.synchronize()
    assert (mine.n_rows, mine.nnz) == (want.n_rows, want.nnz)
    assert torch.equal(mine.to_wire(), want.to_wire())


@pytest.mark.parametrize("few", [False, True])
@pytest.mark.parametrize("ret", ["empty", "unit"])
def test_results_of_another_type(ret, few):
    from sdr_amd import SDRBatch
    q, d = _pair("empty" if ret == "unit" else "unit")
    if few:
        rows = [[1, 5, 9, 300], list(range(0, 500, 7)), []]
        q = SDRBatch.from_rows(rows, width=500) if ret == "unit" else SDRBatch.from_rows(
            [(r, [0.5] * len(r)) for r in rows], with_data=True, width=500)
    want = [op(d, ret=ret).to_host() for op in (q.ande, q.ore, q.xore)]
    for k, op in enumerate((q.ande, q.ore, q.xore)):
        torch.cuda.synchronize()
        stream = _late_stream()
        got = op(d, ret=ret, stream=stream)
        stream.synchronize()
        assert _equal(got.to_host(), want[k])
