"""Weights and gradients of winners far below the largest score keep binary32's precision: their error does not grow with the
distance.  Bounds count half steps of binary32 (2^-24 of the value):
an exponential 2 of the hardware's, 1 of the last fma, and its argument's second part's own roundings, below 1 together; a sigmoid that,
1 of 1 + e, 3 of e again, 2 of the reciprocal, 1 of the product; a sum its additions and its terms' errors -- over a whole row those of the fast
exponential, 3 d + 4 of a term d below the largest, weighed by the terms --, then its reciprocal 2, and two products."""
import numpy as np
import pytest
import torch

import dense_oracle as plain
from test_gpu_dense import BF16, F32, SPECS, rng

pytestmark = pytest.mark.gpu


def _scores(g, n, n_ids, dtype):
    """spread over 70 below and around several heights, so that differences of two scores are rounded"""
    s = -70 * torch.rand(n, n_ids, generator=g) + torch.tensor([0.3, 37.3, -19.7, 1000.1])[torch.arange(n) % 4, None]
    s[:, n_ids // 2] += 5
    return s.to(dtype).cuda()


def _steps(s, ids, spec):
    """half steps that each row's weights may be off by"""
    x, ids = s.cpu().double().numpy(), ids.cpu().numpy()
    out = []
    for r in range(x.shape[0]):
        if spec.get("renormalise"):
            over = x[r][ids[r][ids[r] >= 0]]
            terms = 10.0 if spec["score"] == "sigmoid" else 4.0
        elif spec["score"] == "softmax":
            over = x[r]
            d = over.max() - over
            terms = float((np.exp(-d) * (3 * d + 4)).sum() / np.exp(-d).sum())
        else:
            over, terms = x[r][:1], 0.0
        out.append(10.0 + terms + over.size / 16 + 10 + 2 + 2)   # (additions: a thread's, 16 at least a row, and over them)
    return np.array(out)[:, None]


@pytest.mark.parametrize("spec", SPECS)
@pytest.mark.parametrize("n,n_ids,k,dtype", [(40, 64, 50, F32), (40, 256, 64, F32), (4100, 200, 16, F32), (12, 2048, 64, BF16), (8, 3000, 1024, F32), (5, 16384, 1000, F32)])
def test_weights_far_below_the_largest_score(n, n_ids, k, dtype, spec):
    import sdr_amd
    s = _scores(rng(n_ids + k), n, n_ids, dtype)
    for bias in (None, torch.where(torch.arange(n_ids) % 3 == 0, 2.0, 0.0).cuda()):   # (the bias makes small shares win)
        ids, w = sdr_amd.winners(s, k, bias=bias, **spec)
        rows = slice(0, 24)
        want = plain.winners(s[rows], k, bias=bias, **spec)
        assert np.array_equal(ids[rows].cpu().numpy(), want[0])
        off = np.abs(w[rows].cpu().double().numpy() - want[1])
        tol = np.abs(want[1]) * _steps(s[rows], ids[rows], spec) * plain.U32 + 2.0 ** -126 * spec.get("scale", 1.0)
        assert (off <= tol).all(), float((off / np.maximum(np.abs(want[1]), 1e-37)).max() / plain.U32)


@pytest.mark.parametrize("spec", SPECS)
@pytest.mark.parametrize("n,n_ids,k", [(40, 64, 50), (4100, 200, 16), (8, 2048, 100), (4, 16384, 1000)])
def test_gradients_of_winners_far_below_the_largest_score(n, n_ids, k, spec):
    """the values at the winners: a share's error, their dot product's, and a sigmoid's slope beside them"""
    import sdr_amd
    g = rng(n_ids + k)
    s = _scores(g, n, n_ids, F32)
    bias = torch.where(torch.arange(n_ids) % 3 == 0, 2.0, 0.0).cuda()
    ids, _ = sdr_amd.winners(s, k, bias=bias, **spec)
    gw = torch.randn(n, k, generator=g).cuda()
    got = sdr_amd.winners_grad(s, ids, gw, **spec)
    rows = slice(0, 24)
    want, size = plain.winners_grad(s[rows], ids[rows], gw[rows], **spec)
    steps = 2 * _steps(s[rows], ids[rows], spec) + k / 16 + 20   # (of the share, of the sum that dot is divided by; dot's own; slope and products)
    off = np.abs(got[rows].cpu().double().numpy() - want)
    chosen = np.zeros(off.shape, bool)
    np.put_along_axis(chosen, ids[rows].cpu().numpy().astype(np.int64), True, 1)
    tol = size * steps * plain.U32 + 2.0 ** -124
    assert (off <= tol)[chosen].all(), float((off / np.maximum(size, 1e-37))[chosen].max() / plain.U32)
