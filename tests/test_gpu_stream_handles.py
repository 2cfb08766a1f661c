"""Calls that name their stream by its handle run on that stream: the default stream's handle is 0."""
import pytest
import torch

from test_gpu_dense import BF16, F32, matrix, rng, score_matrix

pytestmark = pytest.mark.gpu


def test_handle_of_the_default_stream():
    from sdr_amd import batch
    default = torch.cuda.default_stream()
    assert default.cuda_stream == 0
    assert batch._torch_stream(0, 0) == default
    other = torch.cuda.Stream()
    with torch.cuda.stream(other):   # whichever stream is current
        assert batch._torch_stream(0, 0) == default
        assert batch._torch_stream(0, other.cuda_stream).cuda_stream == other.cuda_stream


def test_results_follow_inputs_that_the_default_stream_still_makes():
    """inputs come from long work on the default stream; the calls name it by its handle and wait for nothing"""
    import sdr_amd
    g = rng(21)
    ids = torch.randint(0, 1000, (3000, 9), generator=g).cuda()
    t, go, s = matrix(g, 1000, 128, BF16), matrix(g, 3000, 128, BF16), score_matrix(g, 3000, 200, F32)
    a = torch.randn(4096, 4096, device="cuda")

    def step(**on):
        won, w = sdr_amd.winners(s, 7, **on)
        return (won, w, sdr_amd.lookup(ids, t, **on), sdr_amd.lookup_grad_table(ids, go, 1000, **on),
                sdr_amd.lookup_grad_weights(ids, go, t, **on), sdr_amd.winners_grad(s, won, w, **on))

    for _ in range(3):
        for _ in range(20):
            a = (a @ a).tanh()
        t.add_(1)
        go.mul_(2)
        s.neg_()
        got = step(stream=torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        for x, y in zip(got, step()):
            assert torch.equal(x, y)
