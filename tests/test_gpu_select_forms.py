"""Block selection in each of its forms: head sizes, heads a group, rows a CTA, CTAs a list, and scores of any spread."""
import numpy as np
import pytest
import torch

import long_context_reference as L
from test_gpu_attention import context, generator, ints, numbers, rows_of
from test_gpu_blocks import mean_places, random_means

pytestmark = pytest.mark.gpu


def check(ctx, lengths, rows, blocks, first=1, last=1, width=0, spread=None, gone=(), none=(), seed=5):
    """Lists against the statement; block table rows `width` entries wide, `spread` the means' factors, `gone` blocks of every request on pages outside
    the cache, `none` blocks whose mean is NaN."""
    gen, page, kv = generator(seed), ctx.pageTokens, ctx.kvHeads
    used = [-(-n // page) for n in lengths]
    ids = np.random.RandomState(seed).permutation(sum(used) + 1)
    table, at = np.zeros((len(lengths), max(used + [1, width])), dtype=np.int64), 0
    for r, n in enumerate(used):
        table[r, :n] = ids[at:at + n]
        at += n
    means = random_means(gen, sum(used) + 1, ctx)
    if spread is not None:
        means = (means.float() * spread(means.shape[:3], gen)[..., None]).bfloat16()
    q = rows_of(gen, sum(rows), ctx.heads, ctx.headDim)
    q[: len(q) // 3] *= -1.0
    for r, n in enumerate(lengths):
        for b in none:
            if b < n // 64:
                where, place = mean_places(ctx, table, r, b)
                means[int(where), :, int(place)] = float("nan")
    held = numbers(means)
    of = []
    for r, n in enumerate(lengths):
        places = [mean_places(ctx, table, r, b) for b in range(n // 64)]
        of.append(np.stack([held[w, :, p] for w, p in places]) if places else np.zeros((0, kv, ctx.headDim)))
    shown = table.copy()
    for b in gone:
        shown[:, (b * 64 + 63) // page] = 1 << 30
    start = np.concatenate([[0], np.cumsum(rows)])
    got = ctx.selectBlocks(q, means, ints(shown), ints(start), ints(lengths), blocks, first=first, last=last).cpu().numpy()
    want = L.select(numbers(q), of, lengths, rows, kv, blocks, first, last)
    if not gone:
        assert np.array_equal(got, want) and ctx.info().deviceErrorFlag == 0
    return got, want


GROUPS = [1, 2, 3, 4, 5, 7, 8, 9, 16, 17, 24, 33, 64]


# enough lists that some rows share a CTA (more than four an SM), over the ends of requests
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("group", GROUPS)
def test_many_rows(dim, group):
    ctx = context(heads=4 * group, kvHeads=4, dim=dim, page=32, requests=6, tokens=512)
    check(ctx, [1000, 1500, 640, 0, 2000, 300], [3, 101, 1, 0, 2, 62], 6)


# rows of the block table so wide that scores leave a CTA room for four, two rows and one
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("group", [1, 2, 5, 8, 16, 24, 64])
@pytest.mark.parametrize("keys", [1 << 18, 1 << 19, 1 << 20, 1 << 21])
def test_many_rows_of_wide_tables(dim, group, keys):
    ctx = context(heads=4 * group, kvHeads=4, dim=dim, page=256, requests=3, tokens=512)
    check(ctx, [1000, 9000, 70], [5, 155, 1], 5, width=keys // 256)


def test_many_rows_of_a_long_context():
    ctx = context(heads=2, kvHeads=2, dim=64, page=256, requests=2, tokens=512)
    check(ctx, [1 << 18, 5000], [300, 3], 40, 2, 3)


# a cluster of CTAs a list
@pytest.mark.parametrize("heads,kvHeads,dim,rows", [(16, 1, 64, 1), (3, 1, 64, 2), (8, 8, 128, 1), (24, 2, 128, 2), (7, 1, 256, 2), (64, 1, 256, 1), (34, 2, 256, 1), (40, 8, 128, 5), (32, 8, 256, 9)])
def test_few_rows_of_a_long_context(heads, kvHeads, dim, rows):
    ctx = context(heads=heads, kvHeads=kvHeads, dim=dim, page=128, requests=2, tokens=16)
    check(ctx, [1 << 17, 100], [rows, 1], 60, 1, 4)


# many requests of a row or two: a CTA a list
@pytest.mark.parametrize("heads,kvHeads,dim", [(8, 2, 64), (32, 2, 128), (4, 2, 256)])
def test_many_requests(heads, kvHeads, dim):
    rng = np.random.RandomState(dim)
    ctx = context(heads=heads, kvHeads=kvHeads, dim=dim, page=64, requests=400, tokens=1024)
    check(ctx, rng.randint(0, 1500, 400).tolist(), rng.randint(0, 3, 400).tolist(), 5)


def few_loud(shape, gen):
    """A few far above the rest."""
    return torch.where(torch.rand(shape, generator=gen, device="cuda") < 0.02, 2.0 ** 30, 1.0)


def of_any_size(shape, gen):
    """Even in their logarithm."""
    return 2.0 ** torch.randint(-50, 50, shape, generator=gen, device="cuda")


def nearly_none(shape, gen):
    """Most of them zero, equal then."""
    return torch.where(torch.rand(shape, generator=gen, device="cuda") < 0.05, 1.0, 0.0)


@pytest.mark.parametrize("spread", [few_loud, of_any_size, nearly_none])
@pytest.mark.parametrize("lengths,rows", [([1 << 17], [1]), ([1 << 15, 30000, 70], [4, 2, 1]), ([20000, 3000], [300, 40])])
@pytest.mark.parametrize("blocks", [3, 30, 40])
def test_scores_of_any_spread(spread, lengths, rows, blocks):
    ctx = context(heads=8, kvHeads=2, dim=128, page=64, requests=4, tokens=512)
    check(ctx, lengths, rows, blocks, spread=spread)


@pytest.mark.parametrize("lengths,rows", [([1 << 15], [1]), ([9000, 4000], [300, 40])])
def test_means_that_are_no_number_or_nowhere(lengths, rows):
    """Blocks of no number come first; those that lie nowhere last: a list that has room for others names none of them."""
    ctx = context(heads=8, kvHeads=2, dim=64, page=64, requests=4, tokens=512)
    check(ctx, lengths, rows, 20, none=(3, 17, 40))
    got, want = check(ctx, lengths, rows, 20, gone=(5, 9, 33))
    full = (got >= 0).all(-1)
    assert ctx.info().deviceErrorFlag == 16 and full.any()
    # a row has 20 blocks or more beside those three where it sees 23 blocks and more
    start = np.concatenate([[0], np.cumsum(rows)])
    for r, n in enumerate(lengths):
        for i in range(rows[r]):
            seen = (n - rows[r] + i) // 64 + 1
            if seen >= 24:
                assert not np.isin(got[start[r] + i], (5, 9, 33)).any()
                for h in range(2):
                    assert len(set(got[start[r] + i, h])) == 20 and set(want[start[r] + i, h]) - {5, 9, 33} <= set(got[start[r] + i, h])
