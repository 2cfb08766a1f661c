"""Winners under biases without bounds: ids that a bias of +inf forces, more of them than a row's list of candidates holds."""
import numpy as np
import pytest
import torch

import dense_oracle as plain
from test_gpu_dense import F32, assert_winners, rng, score_matrix, weight_bound

pytestmark = pytest.mark.gpu
INF = float("inf")


def _biases(n_ids, k):
    """ids that are sure to win: none, one, fewer than win, more, every other one, all but one, all"""
    at = torch.arange(n_ids)
    yield torch.zeros(n_ids)
    for forced in (at == n_ids // 3, at % 7 == 1, at % 2 == 0, at % 2 == 1, at != n_ids - 2, at >= n_ids // 3, at >= 0):
        yield torch.where(forced, INF, 0.0)
    low = torch.where(at % 2 == 0, INF, 0.25)
    low[::5] = -INF
    yield low


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("n,n_ids,k", [(4099, 60, 5), (4099, 128, 16), (4097, 256, 3), (9, 64, 6), (9, 128, 100), (9, 256, 8), (9, 2048, 40), (5, 4096, 100),
                                       (5, 5000, 200), (5, 1000, 300), (3, 16384, 1024)])
def test_more_ids_forced_than_a_list_holds(n, n_ids, k, score):
    import sdr_amd
    g = rng(n_ids + k)
    s = score_matrix(g, n, n_ids, F32)
    s[0], s[2], s[3:5, ::2] = 0.5, -1.0, -INF     # rows whose other ids are alike stand beside rows whose are not
    bound = weight_bound(s, n_ids, k)
    for bias in _biases(n_ids, k):
        for renormalise in (False, True):
            got = sdr_amd.winners(s, k, score=score, bias=bias.cuda(), renormalise=renormalise)
            rows = torch.cat([torch.arange(min(n, 40)), torch.arange(max(n - 8, min(n, 40)), n)])   # (the statement is slow)
            want = plain.winners(s[rows], k, score=score, bias=bias, renormalise=renormalise)
            assert_winners(tuple(x[rows] for x in got), want, bound)
            ids = got[0].cpu().numpy()
            assert ids.min() >= -1 and ids.max() < n_ids and (np.diff(ids, axis=1) > 0)[ids[:, 1:] >= 0].all()


@pytest.mark.parametrize("n,n_ids,k,groups,top", [(4099, 64, 6, 4, 2), (9, 2048, 40, 8, 3), (5, 250, 20, 10, 4), (3, 16384, 300, 16, 5)])
def test_forced_ids_in_groups(n, n_ids, k, groups, top):
    import sdr_amd
    g = rng(n_ids + k)
    s = score_matrix(g, n, n_ids, F32)
    s[0], s[2] = 0.5, -1.0
    for bias in _biases(n_ids, k):
        for group_top in (1, 2):
            more = dict(score="sigmoid", bias=bias, groups=groups, top_groups=top, group_top=group_top)
            want = plain.winners(s[:20], k, **more)
            more["bias"] = bias.cuda()
            assert_winners(tuple(x[:20] for x in sdr_amd.winners(s, k, **more)), want, weight_bound(s, n_ids, k))
