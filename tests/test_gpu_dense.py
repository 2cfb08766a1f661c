"""Lookups into dense tables, their gradients, the winners of dense scores and their gradient, through the public entry points,
against plain statements in 64 bits (dense_oracle.py)."""
import numpy as np
import pytest
import torch

import dense_oracle as plain

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def rng(seed):
    return torch.Generator().manual_seed(seed)


def matrix(g, n, m, dtype, scale=1.0, pad=0, shift=0):
    """[n, m] on the GPU; rows `pad` elements apart and the first one `shift` elements into its buffer"""
    full = (torch.randn(n, m + pad, generator=g) * scale).to(dtype)
    buf = torch.zeros(n * (m + pad) + shift, dtype=dtype, device="cuda")
    buf[shift:] = full.reshape(-1).cuda()
    return torch.as_strided(buf, (n, m), (m + pad, 1), shift)


def some_rows(g, form, n, n_table, id_type):
    """(ids, offsets): tokens with padding, rows of five, or ragged rows, some of them empty"""
    def draw(*shape):
        ids = torch.randint(0, n_table, shape, generator=g)
        stray = torch.rand(*shape, generator=g)
        ids = torch.where(stray < 0.1, torch.tensor(-1), ids)
        return torch.where(stray > 0.95, torch.tensor(n_table), ids).to(id_type)
    if form == "tokens":
        return draw(n).cuda(), None
    if form in ("fives", "sixteens"):
        return draw(n, 5 if form == "fives" else 16).cuda(), None
    lens = torch.randint(0, 9, (n,), generator=g) * (torch.rand(n, generator=g) < 0.7)
    offsets = torch.zeros(n + 1, dtype=torch.int32)
    offsets[1:] = lens.cumsum(0)
    return draw(int(offsets[-1])).cuda(), offsets.cuda()


# ---- lookup -----------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("form", ["tokens", "fives", "ragged"])
@pytest.mark.parametrize("table,out,dim,pad,shift", [
    (F32, F32, 1, 0, 0), (F32, BF16, 3, 1, 1), (F16, F16, 7, 0, 1), (F16, F32, 8, 0, 0), (BF16, BF16, 9, 2, 1), (BF16, F32, 64, 0, 0),
    (BF16, F16, 100, 1, 3), (F32, F16, 1001, 0, 0), (BF16, BF16, 1024, 8, 8), (F16, BF16, 1537, 0, 0), (F32, F32, 255, 0, 0)])
def test_lookup(form, table, out, dim, pad, shift):
    import sdr_amd
    g = rng(dim + len(form))
    n_table = 53
    t = matrix(g, n_table, dim, table, pad=pad, shift=shift)
    for weighted in (False, True):
        ids, offsets = some_rows(g, form, 37, n_table, torch.int64 if dim % 2 else torch.int32)
        w = torch.randn(ids.shape, generator=g).cuda() if weighted else None
        got = sdr_amd.lookup(ids, t, w, offsets=offsets, scale=0.75, dtype=out)
        assert got.dtype == out
        plain.assert_sum(got, *plain.lookup(ids, t, w, offsets, 0.75), f"{form} weighted={weighted}")
        # into rows of a wider buffer: what lies beside them is left as it was
        wide = torch.full((got.shape[0], dim + 5), 7.0, dtype=out, device="cuda")
        sdr_amd.lookup(ids, t, w, offsets=offsets, scale=0.75, out=wide[:, 2:dim + 2])
        assert torch.equal(wide[:, 2:dim + 2], got) and (wide[:, :2] == 7).all() and (wide[:, dim + 2:] == 7).all()


@pytest.mark.parametrize("dim,dtype", [(5, F32), (64, BF16), (520, F16)])
@pytest.mark.parametrize("lens", [[5000], [0, 129, 0, 128, 1, 0], [3, 2000, 0, 0, 700, 1, 1, 4097], [127] * 40 + [40_000], [1]])
def test_lookup_of_long_rows(lens, dim, dtype):
    import sdr_amd
    g = rng(sum(lens) + dim)
    offsets = torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32).cuda()
    ids = torch.randint(-1, 300, (sum(lens),), generator=g, dtype=torch.int32).cuda()
    t = matrix(g, 300, dim, dtype)
    w = torch.rand(ids.shape, generator=g).cuda()
    for weights in (None, w):
        got = sdr_amd.lookup(ids, t, weights, offsets=offsets, dtype=F32)
        plain.assert_sum(got, *plain.lookup(ids, t, weights, offsets))
        assert torch.equal(got, sdr_amd.lookup(ids, t, weights, offsets=offsets, dtype=F32))
    if len(lens) == 1:   # the same row without offsets
        assert torch.equal(got, sdr_amd.lookup(ids.view(1, -1), t, w.view(1, -1), dtype=F32))


def test_lookup_without_rows_ids_or_columns():
    import sdr_amd
    t = torch.randn(4, 6, device="cuda")
    empty = torch.zeros(0, dtype=torch.int32, device="cuda")
    assert sdr_amd.lookup(empty, t).shape == (0, 6)
    assert sdr_amd.lookup(empty, t, offsets=torch.zeros(1, dtype=torch.int32, device="cuda")).shape == (0, 6)
    assert not sdr_amd.lookup(empty, t, offsets=torch.zeros(4, dtype=torch.int32, device="cuda")).any()
    assert not sdr_amd.lookup(empty.view(3, 0), torch.full((4, 6), float("nan"), device="cuda")).any()
    assert sdr_amd.lookup(torch.zeros(3, dtype=torch.int32, device="cuda"), t[:, :0]).shape == (3, 0)
    ids = torch.tensor([0, -5, 2 ** 33, 4, 3], device="cuda")
    assert torch.equal(sdr_amd.lookup(ids, t), torch.stack([t[0], t[0] * 0, t[0] * 0, t[0] * 0, t[3]]).abs() * torch.stack([t[0], t[0], t[0], t[0], t[3]]).sign())
    assert not sdr_amd.lookup(ids, t[:0]).any()   # a table without rows
    # a padded place adds nothing, whatever stands beside it
    w = torch.tensor([1.0, float("nan"), float("inf"), float("nan"), 1.0], device="cuda")
    assert torch.equal(sdr_amd.lookup(ids, t, w)[[0, 4]], t[[0, 3]]) and not sdr_amd.lookup(ids, t, w)[1:4].any()


def test_lookup_beyond_32_bit_offsets():
    """a table of 5 GB: rows whose first element lies beyond 2^31 elements and 2^32 bytes"""
    import sdr_amd
    rows, dim = 620_000, 4096
    t = torch.zeros(rows, dim, dtype=BF16, device="cuda")
    ids = torch.tensor([0, 262_143, 262_144, 524_287, 524_288, rows - 1], device="cuda")
    t[ids] = torch.randn(ids.numel(), dim, device="cuda").to(BF16)
    assert torch.equal(sdr_amd.lookup(ids, t), t[ids])
    assert torch.equal(sdr_amd.lookup(ids.view(2, 3), t, dtype=F32), t[ids].float().view(2, 3, dim).sum(1))


def test_more_threads_than_one_launch_takes():
    """a launch has fewer than 2^32 threads: rows on both sides of where the next one begins, and the last ones"""
    import sdr_amd
    blocks = (2 ** 32 - 1) // 256 // 64 * 64
    g = rng(3)
    ends = torch.arange(-70, 70, device="cuda")
    t = matrix(g, 53, 7, BF16)
    n = 32 * blocks + 1000   # eight lanes a row of seven columns
    ids = torch.arange(n, dtype=torch.int32, device="cuda").remainder_(53)
    out = torch.full((n, 7), float("nan"), dtype=BF16, device="cuda")
    sdr_amd.lookup(ids, t, out=out)
    for r in (32 * blocks + ends, n - 1 - ends.abs()):
        assert torch.equal(out[r], t[ids[r].long()])
    del out, ids
    n = 16 * blocks + 100    # sixteen lanes a row
    even = torch.arange(n, dtype=torch.int32, device="cuda").remainder_(2)
    s = torch.stack([1 - even, even], 1).to(BF16)
    won, w = sdr_amd.winners(s, 1, score="sigmoid")
    gone = sdr_amd.winners_grad(s, won, w, score="sigmoid")
    for r in (16 * blocks + ends, n - 1 - ends.abs()):
        assert torch.equal(won[r, 0], even[r])
        assert (w[r] - 0.7310586).abs().max() < 1e-6
        assert torch.equal(gone[r] != 0, s[r] == 1)
    del won, w, gone, s, even
    n = 128 * blocks + 4096
    ids = torch.arange(n, dtype=torch.int32, device="cuda").remainder_(3).view(1, n)
    t, go = matrix(g, 3, 8, F32), matrix(g, 1, 8, F32)
    got = sdr_amd.lookup_grad_weights(ids, go, t)
    for r in (128 * blocks + ends, n - 1 - ends.abs()):
        plain.assert_sum(got[0, r].view(1, -1), *(x.view(1, -1) for x in plain.lookup_grad_weights(ids[:, r], go, t)), 8)
    del got, ids
    torch.cuda.empty_cache()   # (some 30 GB)


def test_lookup_of_non_finite_values():
    import sdr_amd
    t = torch.tensor([[1.0, float("inf"), float("nan"), 65504.0], [1.0, float("-inf"), 1.0, 65504.0], [0.0, 1.0, 1.0, 1.0]], device="cuda")
    ids = torch.tensor([[0, 2], [0, 1], [2, 2]], dtype=torch.int32, device="cuda")
    want = t[ids.long()].sum(1)
    got = sdr_amd.lookup(ids, t)
    assert torch.equal(got.nan_to_num(3, 4, 5), want.nan_to_num(3, 4, 5))
    assert torch.isinf(sdr_amd.lookup(ids, t, dtype=F16)[1, 3])   # 131008 rounds to infinity in fp16


# ---- its gradients ----------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("form", ["tokens", "fives", "ragged"])
@pytest.mark.parametrize("grad,out,dim,n,n_table", [
    (F32, F32, 1, 40, 5), (F16, F32, 7, 300, 17), (BF16, F32, 64, 500, 255), (BF16, BF16, 100, 700, 256), (F32, F16, 33, 900, 257),
    (F16, F16, 520, 100, 65_537), (BF16, F32, 24, 3000, 70_000), (F32, F32, 8, 1, 1), (BF16, F32, 136, 2500, 3)])
def test_lookup_grad_table(form, grad, out, dim, n, n_table):
    import sdr_amd
    g = rng(dim + n)
    ids, offsets = some_rows(g, form, n, n_table, torch.int64 if n % 2 else torch.int32)
    w = torch.randn(ids.shape, generator=g).cuda() if form != "tokens" else None
    go = matrix(g, n, dim, grad, pad=dim % 3, shift=dim % 2)
    want = plain.lookup_grad_table(ids, go, n_table, w, offsets, 1.5)
    got = sdr_amd.lookup_grad_table(ids, go, n_table, w, offsets=offsets, scale=1.5, dtype=out)
    plain.assert_sum(got, *want, form)
    assert torch.equal(got, sdr_amd.lookup_grad_table(ids, go, n_table, w, offsets=offsets, scale=1.5, dtype=out))
    # added to what is there; rows that no id names keep their bits, a NaN among them
    into = matrix(g, n_table, dim, out, pad=1)
    free = (want[2] == 0).all(1).nonzero()[:, 0]
    if free.numel():
        into[free[0]] = float("nan")
    before = into.clone()
    sdr_amd.lookup_grad_table(ids, go, weights=w, offsets=offsets, scale=1.5, out=into, accumulate=True)
    assert torch.equal(into[free.cuda()].view(torch.int32 if out == F32 else torch.int16), before[free.cuda()].view(torch.int32 if out == F32 else torch.int16))
    on = (want[2] > 0).all(1)
    plain.assert_sum(into.cpu()[on], (want[0] + before.cpu().double())[on], (want[1] + before.cpu().double().abs())[on], want[2][on] + 1, form)


@pytest.mark.parametrize("n", [1, 63, 64, 65, 1023, 1025, 2049, 16_384, 16_385, 40_000])
@pytest.mark.parametrize("ids_of", ["one", "two", "all_padding", "distinct", "skewed"])
@pytest.mark.parametrize("n_table", [None, 100, 70_000])
def test_lookup_grad_table_of_shared_ids(n, ids_of, n_table):
    """ids that many rows hold, and the order of additions: integers in fp32 add exactly"""
    import sdr_amd
    g = rng(n)
    n_table = max(n, 9) if n_table is None else n_table
    ids = {"one": torch.full((n,), 7), "two": torch.arange(n) % 2 * 5 + 2, "all_padding": torch.full((n,), -1), "distinct": torch.randperm(n, generator=g),
           "skewed": (torch.rand(n, generator=g) ** 8 * n).long()}[ids_of].cuda()
    ids = torch.where(ids < n_table, ids, -1)
    go = torch.randint(-50, 50, (n, 12), generator=g).float().cuda()
    want = torch.zeros(n_table + 1, 12).index_add_(0, torch.where(ids < 0, n_table, ids).cpu(), go.cpu())[:-1]
    assert torch.equal(sdr_amd.lookup_grad_table(ids, go, n_table).cpu(), want)
    assert torch.equal(sdr_amd.lookup_grad_table(ids.int(), go, n_table, scale=2.0).cpu(), want * 2)


def test_lookup_grad_table_of_many_ids():
    """more than 2^24 ids: three passes of the sort of many elements"""
    import sdr_amd
    g = rng(24)
    n, n_table = 30_000, 2 ** 24 + 5
    ids = torch.randint(0, n_table, (n,), generator=g).cuda()
    ids[::7] = 2 ** 24 + 4
    ids[1::7] = 3
    go = torch.randint(-50, 50, (n, 3), generator=g).float().cuda()
    want = torch.zeros(n_table, 3, device="cuda").index_add_(0, ids, go)
    assert torch.equal(sdr_amd.lookup_grad_table(ids, go, n_table), want)
    assert torch.equal(sdr_amd.lookup_grad_table(ids[:9000], go[:9000], n_table), torch.zeros(n_table, 3, device="cuda").index_add_(0, ids[:9000], go[:9000]))


@pytest.mark.parametrize("form", ["tokens", "fives", "sixteens", "ragged"])
@pytest.mark.parametrize("grad,table,dim", [(F32, F32, 1), (F16, F32, 7), (BF16, BF16, 64), (F32, BF16, 100), (F16, F16, 1001), (BF16, F16, 2048)])
def test_lookup_grad_weights(form, grad, table, dim):
    import sdr_amd
    g = rng(dim)
    n_table = 91
    ids, offsets = some_rows(g, form, 77, n_table, torch.int64 if dim % 2 else torch.int32)
    go, t = matrix(g, 77, dim, grad, pad=3), matrix(g, n_table, dim, table, shift=1)
    got = sdr_amd.lookup_grad_weights(ids, go, t, offsets=offsets, scale=0.3)
    assert got.shape == ids.shape and got.dtype == F32
    want, size = plain.lookup_grad_weights(ids, go, t, offsets, 0.3)
    plain.assert_sum(got, want, size, torch.tensor(float(dim)))
    stray = (ids < 0) | (ids >= n_table)
    assert not got[stray].any()


@pytest.mark.parametrize("scale", [1, 40, 1500])
def test_lookup_gradients_of_ragged_rows_with_gaps(scale):
    """runs of empty rows, elements before the first row and behind the last one; short lists and long ones"""
    import sdr_amd
    g = rng(scale)
    lens = [0] * 70 + [3] + [0] * 63 + [1] + [0] * 64 + [2] + [0] * 200 + [17, 0, 1, 1, 1, 9, 0, 0] + [0] * 65
    lens = [m * scale for m in lens]
    before, behind, dim, n_table = 5, 11, 72, 90
    offsets = torch.tensor([before] + [before + int(m) for m in np.cumsum(lens)], dtype=torch.int32).cuda()
    total = int(offsets[-1]) + behind
    ids = torch.randint(-1, n_table + 1, (total,), generator=g, dtype=torch.int32).cuda()
    t, go = matrix(g, n_table, dim, BF16), matrix(g, len(lens), dim, F32)
    w = torch.rand(total, generator=g).cuda()
    inside = slice(before, total - behind)
    own, at = ids[inside], (offsets - before).contiguous()
    plain.assert_sum(sdr_amd.lookup_grad_table(ids, go, n_table, w, offsets=offsets), *plain.lookup_grad_table(own, go, n_table, w[inside], at))
    got = sdr_amd.lookup_grad_weights(ids, go, t, offsets=offsets)
    plain.assert_sum(got[inside], *plain.lookup_grad_weights(own, go, t, at), dim)
    assert not got[:before].any() and not got[total - behind:].any()


def test_lookup_gradients_against_differences():
    """the sum of result * r changes by its gradients; it is linear in table and weights, so a step of 1 has no curvature"""
    import sdr_amd
    g = rng(3)
    ids, offsets = some_rows(g, "ragged", 11, 13, torch.int32)
    t, r = matrix(g, 13, 6, F32), matrix(g, 11, 6, F32)
    w = torch.rand(ids.shape, generator=g).cuda()
    loss = lambda t_, w_: float((sdr_amd.lookup(ids, t_, w_, offsets=offsets, scale=0.5).double() * r.double()).sum())  # noqa: E731
    d_table = sdr_amd.lookup_grad_table(ids, r, 13, w, offsets=offsets, scale=0.5)
    d_w = sdr_amd.lookup_grad_weights(ids, r, t, offsets=offsets, scale=0.5)
    for v, c in ((0, 0), (5, 3), (12, 5)):
        up, down = t.clone(), t.clone()
        up[v, c] += 1
        down[v, c] -= 1
        assert abs((loss(up, w) - loss(down, w)) / 2 - float(d_table[v, c])) < 1e-4
    for e in (0, ids.numel() // 2, ids.numel() - 1):
        step = torch.zeros_like(w)
        step[e] = 1
        assert abs((loss(t, w + step) - loss(t, w - step)) / 2 - float(d_w[e])) < 1e-4


# ---- winners ----------------------------------------------------------------------------------------------------------


def score_matrix(g, n, m, dtype, masked=0.0, pad=0):
    s = matrix(g, n, m, dtype, scale=2.0, pad=pad)
    if masked:
        s[torch.rand(n, m, generator=g).cuda() < masked] = float("-inf")
    return s


def weight_bound(scores, n_ids, k):
    """relative error of a share: two exponentials whose arguments are off by half a step of at most the range of the scores,
    some steps of the functions themselves (2 of exp, 1 of each of log1p, division and product, on both sides), and a sum of
    positive terms, 64 lanes wide"""
    finite = scores[torch.isfinite(scores)].double()
    spread = float(finite.max() - finite.min()) if finite.numel() else 0.0
    return (2 * spread + 16 + n_ids / 64 + 6) * plain.U32


def assert_winners(got, want, bound):
    ids, weights = got
    assert np.array_equal(ids.cpu().numpy(), want[0])
    off = np.abs(weights.cpu().double().numpy() - want[1])
    assert (off <= np.abs(want[1]) * bound + 2.0 ** -126).all(), float((off / np.maximum(np.abs(want[1]), 1e-30)).max())


SPECS = [dict(score="softmax"), dict(score="sigmoid", renormalise=True, scale=2.5), dict(score="softmax", renormalise=True),
         dict(score="sigmoid", scale=0.5)]


@pytest.mark.parametrize("spec", SPECS)
@pytest.mark.parametrize("n,n_ids,k,dtype,masked,pad", [
    (1, 1, 1, F32, 0, 0), (3, 8, 8, F32, 0, 1), (70, 64, 6, BF16, 0, 0), (33, 63, 5, F16, 0.3, 0), (65, 65, 2, F32, 0, 3), (9, 256, 8, F32, 0, 0),
    (5, 257, 40, BF16, 0.5, 0), (4, 1000, 33, F32, 0.9, 0), (7, 2048, 40, BF16, 0, 0), (3, 4097, 64, F16, 0.1, 1), (2, 16384, 328, F32, 0, 0),
    (2, 5000, 1024, BF16, 0.5, 0), (300, 16, 3, F32, 0.2, 0), (129, 128, 128, F32, 0.1, 0)])
def test_winners(spec, n, n_ids, k, dtype, masked, pad):
    import sdr_amd
    g = rng(n_ids + k)
    s = score_matrix(g, n, n_ids, dtype, masked, pad)
    bound = weight_bound(s, n_ids, k)
    got = sdr_amd.winners(s, k, **spec)
    assert_winners(got, plain.winners(s, k, **spec), bound)
    bias = torch.randn(n_ids, generator=g).cuda() * 0.3
    assert_winners(sdr_amd.winners(s, k, bias=bias, **spec), plain.winners(s, k, bias=bias, **spec), bound)


@pytest.mark.parametrize("spec", SPECS)
@pytest.mark.parametrize("n,n_ids,k,groups,top,dtype,masked", [
    (40, 256, 8, 8, 4, F32, 0), (31, 64, 6, 8, 3, BF16, 0), (7, 160, 6, 8, 3, F32, 0.4), (5, 96, 4, 96, 10, F32, 0.3), (6, 512, 24, 2, 1, F16, 0),
    (11, 33, 2, 3, 2, F32, 0.8), (3, 4096, 64, 256, 9, BF16, 0.2), (2, 16384, 100, 128, 64, F32, 0), (9, 64, 60, 4, 2, F32, 0)])
def test_winners_in_groups(spec, n, n_ids, k, groups, top, dtype, masked):
    import sdr_amd
    g = rng(n_ids + groups)
    s = score_matrix(g, n, n_ids, dtype, masked)
    bias = torch.randn(n_ids, generator=g).cuda() * 0.1
    for group_top in (1, 2):
        for b in (None, bias):
            more = dict(bias=b, groups=groups, top_groups=top, group_top=group_top, **spec)
            assert_winners(sdr_amd.winners(s, k, **more), plain.winners(s, k, **more), weight_bound(s, n_ids, k))


@pytest.mark.parametrize("n_ids,k", [(8, 3), (64, 8), (200, 40), (4096, 17)])
def test_winners_ties_go_to_the_lowest_id(n_ids, k):
    import sdr_amd
    g = rng(n_ids)
    few = torch.randint(0, 3, (20, n_ids), generator=g).float().cuda()   # many equal scores
    few[0] = 1.0
    few[1] = 0.0
    few[1, -1] = -0.0   # zeros of either sign are equal
    zero = torch.zeros(n_ids, device="cuda")
    for bias in (None, zero):
        for score in ("softmax", "sigmoid"):
            assert_winners(sdr_amd.winners(few, k, score=score, bias=bias), plain.winners(few, k, score=score, bias=bias), weight_bound(few, n_ids, k))
            more = dict(score=score, bias=bias, groups=4, top_groups=2, group_top=2)
            k2 = min(k, n_ids // 2)
            assert_winners(sdr_amd.winners(few, k2, **more), plain.winners(few, k2, **more), weight_bound(few, n_ids, k))


@pytest.mark.parametrize("n,n_ids,k,groups,top", [(4100, 152, 11, 4, 2), (4100, 250, 16, 10, 1), (4100, 60, 16, 1, 1), (30, 2000, 60, 8, 1), (9, 16000, 300, 1, 1),
                                                  (5, 9000, 900, 3, 2), (5, 1500, 1024, 1, 1)])
@pytest.mark.parametrize("dtype", [F32, F16])
def test_winners_that_few_threads_hold(n, n_ids, k, groups, top, dtype):
    """the largest scores side by side, in few groups, or more of them than a threshold over the threads' largest finds"""
    import sdr_amd
    g = rng(n_ids + k)
    s = score_matrix(g, n, n_ids, dtype)
    s[: n // 2, n_ids // 3: n_ids // 3 + 2 * k] += 9
    for bias in (None, torch.randn(n_ids, generator=g).cuda() * 0.1, torch.zeros(n_ids, device="cuda")):
        for spec in (dict(score="softmax"), dict(score="sigmoid", renormalise=True)):
            more = dict(spec, bias=bias, groups=groups, top_groups=top, group_top=2)
            assert_winners(sdr_amd.winners(s, k, **more), plain.winners(s, k, **more), weight_bound(s, n_ids, k))


@pytest.mark.parametrize("n,n_ids,k", [(4100, 40, 5), (4100, 256, 16), (5, 250, 20), (5, 2048, 64), (5, 5000, 7), (5, 16384, 1024)])
def test_winners_of_many_equal_keys(n, n_ids, k):
    import sdr_amd
    g = rng(n_ids * k)
    s = torch.randint(0, 2, (n, n_ids), generator=g).float().cuda()
    s[0], s[1], s[2, 3:] = 0.0, -7.5, float("-inf")
    s[3] = torch.linspace(-1e-6, 1e-6, n_ids)           # not one of them equal, all within an error of binary32
    s[4, ::2], s[4, 1::2] = 0.5, 0.5 + 2.0 ** -23       # two values within one
    two = torch.where(torch.arange(n_ids) % 3 == 0, 0.25, -0.25).cuda()
    for bias in (None, torch.zeros(n_ids, device="cuda"), two):
        for score in ("softmax", "sigmoid"):
            for more in (dict(), dict(groups=n_ids // 5, top_groups=n_ids // 10, group_top=2)) if n_ids == 250 else (dict(),):
                got = sdr_amd.winners(s, k, score=score, bias=bias, **more)
                assert_winners(got, plain.winners(s, k, score=score, bias=bias, **more), weight_bound(s, n_ids, k))


def test_winners_of_close_keys():
    """sigmoids that differ by less than a step of binary32, and shares that a bias brings within one of each other"""
    import sdr_amd
    s = torch.full((4, 64), -1.0)
    s[0, 10:30] = 15.0 + torch.arange(20) * 2.0 ** -15      # sigmoids within 1e-8 of one another
    s[1, :] = 17.5
    s[1, 40] = 17.75                                         # both are 1 in binary32
    s[2] = torch.linspace(-1e-6, 1e-6, 64)
    s[3] = torch.linspace(1e-6, -1e-6, 64)
    s = s.cuda()
    bias = torch.zeros(64, device="cuda")
    for score in ("softmax", "sigmoid"):
        for b in (None, bias):
            for more in (dict(), dict(groups=8, top_groups=2, group_top=2)):
                assert_winners(sdr_amd.winners(s, 5, score=score, bias=b, **more), plain.winners(s, 5, score=score, bias=b, **more), weight_bound(s, 64, 5))


def test_winners_of_masked_and_extreme_scores():
    import sdr_amd
    inf, nan, low = float("inf"), float("nan"), torch.finfo(F32).min
    s = torch.zeros(10, 70)
    s[0] = -inf                                  # nothing left
    s[1] = -inf
    s[1, 66] = 3.0                               # one left
    s[2] = low                                   # masked by the type's lowest value: still candidates, of equal shares
    s[3, ::2] = nan
    s[3, 1] = -inf
    s[4] = low
    s[4, 5] = 1.0
    s[5, [3, 69]] = inf                          # shared by the infinite ones
    s[6] = torch.linspace(-300, -100, 70)        # sigmoids that underflow binary32
    s[7] = torch.linspace(80, 900, 70)
    s[8] = nan
    s[9] = torch.linspace(-1e30, 1e30, 70)
    want_row_1 = np.array([66, -1, -1, -1])
    for spec in SPECS:
        ids, w = sdr_amd.winners(s.cuda(), 4, **spec)
        assert_winners((ids, w), plain.winners(s, 4, **spec), 1e-3)   # (rows with a spread of 300: 2 * 300 * 2^-24 = 4e-5; 1e30 decides by 0 or 1)
        assert (ids[0] == -1).all() and not w[0].any() and (ids[8] == -1).all() and np.array_equal(ids[1].cpu(), want_row_1)
        assert torch.isfinite(w).all()
    # a bias of -inf or NaN bars an id, one of +inf makes it win
    bias = torch.zeros(70)
    bias[0], bias[1], bias[2] = -inf, nan, inf
    s = torch.ones(1, 70)
    assert sdr_amd.winners(s.cuda(), 3, bias=bias.cuda(), score="sigmoid")[0].tolist() == [[2, 3, 4]]
    # an id is chosen for its bias although its share is nothing beside the others'
    s[0, 60:63] = torch.tensor([-200.0, -201.0, -400.0])
    bias = torch.zeros(70)
    bias[60:63] = 5
    for spec in SPECS:
        got = sdr_amd.winners(s.cuda(), 3, bias=bias.cuda(), **spec)
        assert_winners(got, plain.winners(s, 3, bias=bias, **spec), 1e-3)


def grad_bound(scores, want, size, n_ids, dtype):
    return size * weight_bound(scores, n_ids, 1) * 2 + np.abs(want) * plain.half_step(dtype) * (1 + 2.0 ** -7) + plain.tiny(dtype) + 2.0 ** -126


@pytest.mark.parametrize("spec", SPECS)
@pytest.mark.parametrize("n,n_ids,k,dtype,out,masked", [
    (1, 1, 1, F32, F32, 0), (3, 8, 8, F32, BF16, 0.2), (70, 64, 6, BF16, BF16, 0), (33, 63, 5, F16, F32, 0.3), (5, 257, 40, BF16, F32, 0.5),
    (4, 1000, 33, F32, F32, 0.97), (7, 2048, 40, BF16, BF16, 0.1), (3, 4097, 64, F16, F16, 0.1), (2, 16384, 328, F32, F32, 0), (300, 16, 3, F32, F32, 0.2),
    (2, 3000, 1024, F32, F32, 0)])
def test_winners_grad(spec, n, n_ids, k, dtype, out, masked):
    import sdr_amd
    g = rng(n_ids + k)
    s = score_matrix(g, n, n_ids, dtype, masked)
    bias = torch.randn(n_ids, generator=g).cuda() * 0.3
    ids, w = sdr_amd.winners(s, k, bias=bias, **spec)
    gw = torch.randn(n, k, generator=g).cuda()
    gw[ids < 0] = float("nan")   # places without an id are not read as gradients
    got = sdr_amd.winners_grad(s, ids, gw, dtype=out, **spec)
    want, size = plain.winners_grad(s, ids, gw, **spec)
    assert got.dtype == out
    off = np.abs(got.cpu().double().numpy() - want)
    assert (off <= grad_bound(s, want, size, n_ids, out)).all(), float(off.max())
    # nothing flows to ids that play no part
    idle = torch.isinf(s) if spec == SPECS[0] else torch.ones(n, n_ids + 1, dtype=torch.bool, device="cuda").scatter(1, torch.where(ids < 0, n_ids, ids).long(), False)[:, :-1]
    assert not got[idle].any()


@pytest.mark.parametrize("spec", SPECS)
def test_winners_grad_against_differences(spec):
    """(w(s + h) - w(s - h)) / 2h: off by h^2 / 6 times a third derivative of at most 1, and by the weights' rounding over h"""
    import sdr_amd
    g = rng(5)
    s = score_matrix(g, 1, 40, F32)
    ids, w = sdr_amd.winners(s, 6, **spec)
    r = torch.randn(1, 6, generator=g).cuda()
    d = sdr_amd.winners_grad(s, ids, r, **spec)
    h = 2.0 ** -7
    gap = torch.sort(s[0], descending=True).values
    assert float(gap[5] - gap[6]) > 2 * h   # the choice stays
    for e in range(40):
        step = torch.zeros_like(s)
        step[0, e] = h
        up, down = sdr_amd.winners(s + step, 6, **spec), sdr_amd.winners(s - step, 6, **spec)
        assert torch.equal(up[0], ids) and torch.equal(down[0], ids)
        slope = float(((up[1].double() - down[1].double()) * r.double()).sum()) / (2 * h)
        size = float(spec.get("scale", 1.0) * r.abs().sum())
        assert abs(slope - float(d[0, e])) < size * (h * h / 6 + 40 * plain.U32 / h)


def test_winners_grad_of_masked_and_extreme_scores():
    import sdr_amd
    inf, low = float("inf"), torch.finfo(F32).min
    s = torch.zeros(6, 70)
    s[0] = -inf
    s[1] = -inf
    s[1, 66] = 3.0
    s[2] = low
    s[3] = torch.linspace(-300, -100, 70)
    s[4] = torch.linspace(80, 900, 70)
    s[5, ::3] = float("nan")
    for spec in SPECS:
        ids, w = sdr_amd.winners(s.cuda(), 4, **spec)
        r = torch.randn(6, 4, generator=rng(1)).cuda()
        got = sdr_amd.winners_grad(s.cuda(), ids, r, **spec)
        want, size = plain.winners_grad(s, ids, r, **spec)
        assert torch.isfinite(got).all() and not got[0].any()
        off = np.abs(got.cpu().double().numpy() - want)
        assert (off <= size * 1e-3 + 2.0 ** -126).all()


# ---- together ---------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("n,n_ids,k,dim,dtype", [(50, 96, 7, 40, F32), (130, 2048, 40, 65, F32)])
def test_a_memory_layer_and_its_gradients(n, n_ids, k, dim, dtype):
    """scores -> winners -> weighted lookup, and back to the table and the scores, against torch's autograd in 64 bits"""
    import sdr_amd
    g = rng(n)
    s, t, go = score_matrix(g, n, n_ids, dtype), matrix(g, n_ids, dim, dtype), matrix(g, n, dim, dtype)
    for spec in SPECS:
        ids, w = sdr_amd.winners(s, k, **spec)
        out = sdr_amd.lookup(ids, t, w)
        d_table = sdr_amd.lookup_grad_table(ids, go, n_ids, w)
        d_w = sdr_amd.lookup_grad_weights(ids, go, t)
        d_s = sdr_amd.winners_grad(s, ids, d_w, **spec)
        s64, t64 = s.cpu().double().requires_grad_(), t.cpu().double().requires_grad_()
        at = ids.cpu().long()
        if spec.get("renormalise"):
            chosen = s64.gather(1, at)
            w64 = torch.softmax(chosen if spec["score"] == "softmax" else torch.nn.functional.logsigmoid(chosen), 1)
        else:
            w64 = (torch.softmax(s64, 1) if spec["score"] == "softmax" else torch.sigmoid(s64)).gather(1, at)
        o64 = ((w64 * spec.get("scale", 1.0))[..., None] * t64[at]).sum(1)
        o64.backward(go.cpu().double())
        for got, want in ((out, o64.detach()), (d_table, t64.grad), (d_s, s64.grad)):
            assert float((got.cpu().double() - want).abs().max()) <= 1e-4 * float(want.abs().max())   # k * dim sums of 2^-24 each


def test_batches_take_the_same_operators():
    import sdr_amd
    from sdr_amd import SDRBatch, SdrbError
    g = rng(8)
    rows = [np.unique(np.random.default_rng(r).integers(0, 500, r % 23)) for r in range(90)]
    off = np.concatenate([[0], np.cumsum([r.size for r in rows])])
    ids = np.concatenate(rows).astype(np.int32)
    data = np.random.default_rng(1).random(ids.size).astype(np.float32)
    t, go = matrix(g, 500, 72, BF16), matrix(g, 90, 72, BF16)
    off_t, ids_t, data_t = torch.from_numpy(off.astype(np.int32)).cuda(), torch.from_numpy(ids).cuda(), torch.from_numpy(data).cuda()
    for kind, d in (("empty", None), ("unit", data), ("arith", data)):
        w = None if d is None else data_t
        b = SDRBatch.from_csr(off, ids, d, width=500, kind=kind)
        assert torch.equal(b.lookup(t, scale=2.0), sdr_amd.lookup(ids_t, t, w, offsets=off_t, scale=2.0))
        plain.assert_sum(b.lookup(t, dtype=F32), *plain.lookup(ids_t, t, w, off_t))
        assert torch.equal(b.lookup_grad_table(go), sdr_amd.lookup_grad_table(ids_t, go, 500, w, offsets=off_t))
        assert torch.equal(b.lookup_grad_data(go, t), sdr_amd.lookup_grad_weights(ids_t, go, t, offsets=off_t))
        # a batch's transpose looked up in the gradient is the table's gradient too
        assert torch.equal(b.transpose().lookup(go, dtype=F32), b.lookup_grad_table(go))
    wide = SDRBatch.from_csr(off, ids.astype(np.int64), None)
    assert torch.equal(wide.lookup(t), sdr_amd.lookup(ids_t, t, offsets=off_t))
    with pytest.raises(ValueError):
        wide.lookup_grad_table(go)
    with pytest.raises(SdrbError):
        SDRBatch(0, 10).lookup(t)


def test_a_batch_without_a_width_adds_to_the_rows_it_is_given():
    from sdr_amd import SDRBatch
    g = rng(9)
    b = SDRBatch.from_rows([[1, 4], [], [0, 4, 6]])
    go = matrix(g, 3, 24, F32)
    want = b.lookup_grad_table(go, 9)
    into = torch.ones(9, 24, device="cuda")
    assert b.lookup_grad_table(go, out=into, accumulate=True) is into
    plain.assert_sum(into, want.cpu().double() + 1, want.cpu().double().abs() + 1, torch.tensor(3.0))
    with pytest.raises(ValueError):
        b.lookup_grad_table(go)


def test_winners_become_a_batch():
    import sdr_amd
    from sdr_amd import SDRBatch
    s = score_matrix(rng(2), 40, 300, F32, masked=0.97)
    ids, w = sdr_amd.winners(s, 20, renormalise=True)
    b = SDRBatch.from_winners(ids, w, width=300)
    assert b.n_rows == 40 and b.nnz == int((ids >= 0).sum())
    t = matrix(rng(4), 300, 33, F32)
    plain.assert_sum(b.lookup(t), *plain.lookup(ids, t, w))
    codes = SDRBatch.from_winners(ids, width=300)   # overlaps of the codes, by the set algebra
    hot = torch.zeros(40, 301, device="cuda").scatter(1, torch.where(ids < 0, 300, ids).long(), 1.0)[:, :-1]
    assert torch.equal(codes.ands(codes).float(), hot @ hot.T)


def test_captured_and_replayed_on_new_values():
    """the whole step in one graph, replayed over changed inputs with eager work between the replays"""
    import sdr_amd
    g = rng(11)
    n, n_ids, k, dim = 300, 512, 12, 96
    s, t, go = score_matrix(g, n, n_ids, F32), matrix(g, n_ids, dim, BF16), matrix(g, n, dim, BF16)

    def step():
        ids, w = sdr_amd.winners(s, k, score="sigmoid", renormalise=True)
        return (ids, w, sdr_amd.lookup(ids, t, w), sdr_amd.lookup_grad_table(ids, go, n_ids, w),
                sdr_amd.winners_grad(s, ids, sdr_amd.lookup_grad_weights(ids, go, t), score="sigmoid", renormalise=True))

    step()
    graphs = []
    for _ in range(2):   # two graphs of the same step: their scratch is their own
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        graphs.append((graph, outs))
    for r in range(4):
        s.copy_(score_matrix(g, n, n_ids, F32, masked=0.2 * r))
        t.copy_(matrix(g, n_ids, dim, BF16))
        want = step()
        for graph, outs in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for graph, outs in graphs:
            for a, b in zip(outs, want):
                assert torch.equal(a, b)


def test_another_stream_and_two_at_once():
    import sdr_amd
    g = rng(12)
    ids = torch.randint(0, 1000, (4000, 9), generator=g).cuda()
    t, go = matrix(g, 1000, 128, BF16), matrix(g, 4000, 128, BF16)
    want = (sdr_amd.lookup(ids, t), sdr_amd.lookup_grad_table(ids, go, 1000))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = [(sdr_amd.lookup(ids, t, stream=st), sdr_amd.lookup_grad_table(ids, go, 1000, stream=st.cuda_stream)) for st in streams for _ in range(4)]
    torch.cuda.synchronize()
    for a, b in got:
        assert torch.equal(a, want[0]) and torch.equal(b, want[1])
