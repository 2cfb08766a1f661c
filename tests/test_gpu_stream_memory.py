"""Results of calls on an explicit stream are that stream's memory: one that is dropped while its call still runs must not be
handed to work on another stream."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _batch():
    from sdr_amd import SDRBatch
    rng = np.random.default_rng(5)
    rows = [np.sort(rng.choice(512, 12, replace=False)).astype(np.int32) for _ in range(40)]
    return SDRBatch.from_csr(np.arange(0, 12 * 40 + 1, 12), np.concatenate(rows), width=512)


CALLS = {
    "ands": lambda q, s: q.ands(q, stream=s),
    "ands_u8": lambda q, s: _torch_u8(q, s),
    "ande": lambda q, s: q.ande(q, stream=s).ids_buffer,
    "rme": lambda q, s: q.rme(q, stream=s).ids_buffer,
    "andv": lambda q, s: q.andv(q, stream=s).this_pos,
    "range_size": lambda q, s: q.range_size([3, 5], [90, 100], stream=s),
    "point_query": lambda q, s: q.point_query([3, 5], stream=s),
    "allpairs_topk": lambda q, s: q.allpairs_topk(q, 4, stream=s)[0],
    "equals": lambda q, s: q.equals(q, stream=s),
}


def _torch_u8(q, s):
    import torch
    return q.ands(q, dtype=torch.uint8, stream=s)


@pytest.mark.parametrize("name", sorted(CALLS))
def test_dropped_results_stay_with_their_stream(name):
    import torch
    q = _batch()
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    result = CALLS[name](q, stream)
    at, size = result.untyped_storage().data_ptr(), result.untyped_storage().nbytes()
    del result
    others = [torch.empty(size, dtype=torch.uint8, device="cuda") for _ in range(4)]   # of the current stream
    stream.synchronize()
    assert all(x.data_ptr() != at for x in others)
