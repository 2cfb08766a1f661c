"""A result of a call on an explicit stream may be used on the stream that was current at the call and dropped there: its memory
is not handed to the next call on the explicit stream while that work is still to come.  Addresses alone are compared."""
import pytest
import torch

from test_gpu_dense import BF16, matrix, rng, score_matrix
from test_gpu_stream_memory import CALLS, _batch

pytestmark = pytest.mark.gpu


def _dense_calls():
    import sdr_amd
    g = rng(2)
    ids = torch.randint(0, 100, (300, 5), generator=g).cuda()
    t, go, s = matrix(g, 100, 64, BF16), matrix(g, 300, 64, BF16), score_matrix(g, 300, 64, BF16)
    won, w = sdr_amd.winners(s, 5)
    return {"lookup": lambda q, st: sdr_amd.lookup(ids, t, stream=st), "lookup_grad_table": lambda q, st: sdr_amd.lookup_grad_table(ids, go, 100, stream=st),
            "lookup_grad_weights": lambda q, st: sdr_amd.lookup_grad_weights(ids, go, t, stream=st),
            "winners": lambda q, st: sdr_amd.winners(s, 5, stream=st)[1], "winners_grad": lambda q, st: sdr_amd.winners_grad(s, won, w, stream=st)}


DENSE = ["lookup", "lookup_grad_table", "lookup_grad_weights", "winners", "winners_grad"]


@pytest.mark.parametrize("by_handle", [False, True])
@pytest.mark.parametrize("name", sorted(CALLS) + DENSE)
def test_memory_waits_for_the_stream_that_was_current(name, by_handle):
    call = CALLS[name] if name in CALLS else _dense_calls()[name]
    q = _batch()
    own = torch.cuda.Stream()
    stream = own.cuda_stream if by_handle else own
    a = torch.randn(8192, 8192, device="cuda", dtype=BF16)
    call(q, stream)   # what a first call builds is there
    torch.cuda.synchronize()
    result = call(q, stream)
    own.synchronize()
    storage = result.untyped_storage()
    at, end = storage.data_ptr(), storage.data_ptr() + storage.nbytes()
    del storage
    for _ in range(150):
        a = (a @ a) * 2.0 ** -13      # (some 150 ms of the current stream)
    seen = result.clone()             # behind all that
    del result
    busy = torch.cuda.Event()
    busy.record()
    assert not busy.query(), "the current stream was to be busy when the next call asks for memory"
    later = call(q, stream)
    storage = later.untyped_storage()
    apart = storage.data_ptr() >= end or storage.data_ptr() + storage.nbytes() <= at
    assert apart or busy.query()      # (a call that waits for the device in between may have the same memory again)
    torch.cuda.synchronize()
    written = getattr(q, name)(q).total if name in ("ande", "rme") else seen.shape[0]   # (buffers sized by a bound hold anything behind)
    assert torch.equal(seen[:written], later[:written])   # (the same call)
    del storage, later


def test_memory_of_a_call_on_the_current_stream_is_handed_on_at_once():
    q = _batch()
    for stream in (torch.cuda.current_stream(), torch.cuda.current_stream().cuda_stream):
        addresses = set()
        for _ in range(20):
            addresses.add(q.ands(q, stream=stream).untyped_storage().data_ptr())
        assert len(addresses) <= 2


def test_a_captured_step_on_a_stream_of_its_own():
    """calls on a second stream inside a capture, their results used and dropped on the first one"""
    import sdr_amd
    g = rng(3)
    ids = torch.randint(0, 100, (300, 5), generator=g).cuda()
    t, s = matrix(g, 100, 64, BF16), score_matrix(g, 300, 100, BF16)
    side = torch.cuda.Stream()

    def step(stream):
        won, w = sdr_amd.winners(s, 5, stream=stream)
        return sdr_amd.lookup(won, t, w, stream=stream), sdr_amd.lookup(ids, t, stream=stream)

    def whole(stream=None):
        here = torch.cuda.current_stream()
        if stream is not None:
            stream.wait_stream(here)
        both = step(stream)
        if stream is not None:
            here.wait_stream(stream)
        return both[0] + both[1]

    whole(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = whole(side)
    for r in range(3):
        s.copy_(score_matrix(g, 300, 100, BF16))
        t.copy_(matrix(g, 100, 64, BF16))
        want = whole()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
