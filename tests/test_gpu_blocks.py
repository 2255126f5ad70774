"""Block means and block selection over the INT4 cache, and page books with shared pages, against plain statements."""
import numpy as np
import pytest
import torch

import attention_reference as R
import long_context_reference as L
from test_gpu_attention import context, generator, ints, numbers, rows_of

pytestmark = pytest.mark.gpu


def cache_of(ctx, lengths, loud=1.0, seed=3, spare=2, tables=None):
    """(pages, table, width) of a written cache: every request's pages in no order."""
    gen = generator(seed)
    page = ctx.pageTokens
    used = [-(-n // page) for n in lengths]
    count = sum(used) + spare
    ids = np.random.RandomState(seed).permutation(count)
    width = max(used + [1])
    table, at = np.full((len(lengths), width), 0), 0
    for r, n in enumerate(used):
        table[r, :n] = ids[at:at + n]
        at += n
    pages = ctx.newCache(count)
    slots = ints(np.random.RandomState(seed + 1).permutation(count * page))
    for a in range(0, count * page, ctx.maxTokens):
        part = slots[a:a + ctx.maxTokens]
        k = rows_of(gen, len(part), ctx.kvHeads, ctx.headDim, loud)
        ctx.append(None, k, rows_of(gen, len(part), ctx.kvHeads, ctx.headDim), None, part, part, pages)
    return pages, table


def slots_of(table, lengths, page):
    return [[table[r, p // page] * page + p % page for p in range(n)] for r, n in enumerate(lengths)]


def mean_places(ctx, table, r, b):
    last = b * 64 + 63
    return table[r, last // ctx.pageTokens], last % ctx.pageTokens // 64


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_means_of_completed_blocks(dim, page):
    ctx = context(dim=dim, page=page, requests=8, tokens=2048)
    old = [0, 63, 64, 0, 100, 500, 130, 7]
    new = [64, 64, 127, 0, 40, 700, 130, 63]
    pages, table = cache_of(ctx, [max(a, b) for a, b in zip(old, new)], loud=3.0)
    means = ctx.newMeans(len(pages))
    means.fill_(9.0)
    ctx.blockMeans(pages, ints(table), ints(old), ints(new), means)
    keys, _ = R.unpack(pages.cpu().numpy(), ctx.kvHeads, dim, page)
    want = np.full(tuple(means.shape), 9.0)
    for r, at in enumerate(slots_of(table, new, page)):
        for b in range(old[r] // 64, new[r] // 64):
            where, place = mean_places(ctx, table, r, b)
            for h in range(ctx.kvHeads):
                want[where, h, place] = L.block_mean(keys[at[b * 64:b * 64 + 64], h])
    assert (want != 9.0).any()
    assert np.array_equal(numbers(means), want)
    assert ctx.info().deviceErrorFlag == 0


@pytest.mark.parametrize("requests", [300, 1025])
def test_means_of_many_requests(requests):
    ctx = context(heads=1, kvHeads=1, page=64, requests=requests, tokens=4096)
    rng = np.random.RandomState(requests)
    old = rng.randint(0, 130, requests)
    new = np.where(rng.rand(requests) < 0.3, rng.randint(0, 200, requests), old)
    pages, table = cache_of(ctx, np.maximum(old, new))
    means = ctx.newMeans(len(pages))
    ctx.blockMeans(pages, ints(table), ints(old), ints(new), means)
    keys, _ = R.unpack(pages.cpu().numpy(), 1, 64, 64)
    want = np.zeros(tuple(means.shape))
    for r, at in enumerate(slots_of(table, new, 64)):
        for b in range(old[r] // 64, new[r] // 64):
            want[table[r, b], 0, 0] = L.block_mean(keys[at[b * 64:b * 64 + 64], 0])
    assert np.array_equal(numbers(means), want)


def test_means_at_the_ends_of_range_and_of_no_number():
    """Blocks of zeros, of tiny and huge keys, of opposite signs, and with a key that stands for NaN."""
    ctx = context(heads=1, kvHeads=1, page=64, requests=1, tokens=1024)
    x = torch.zeros((7 * 64, 1, 64), device="cuda")
    gen = generator()
    x[64:128] = 2.0 ** -70 * torch.randn((64, 1, 64), generator=gen, device="cuda")
    x[128:192] = 2.0 ** 90 * torch.randn((64, 1, 64), generator=gen, device="cuda")
    x[192:256] = torch.randn((64, 1, 64), generator=gen, device="cuda")
    x[224:256] = -x[192:224]
    x[256:320] = 1.0
    x[300, 0, 5] = float("inf")
    x[320:384] = torch.randn((64, 1, 64), generator=gen, device="cuda")
    x[330] *= 2.0 ** 30
    x[384:] = -(2.0 ** -20)
    pages = ctx.newCache(7)
    slots = ints(range(7 * 64))
    ctx.append(None, x.bfloat16(), x.bfloat16(), None, slots, slots, pages)
    means = ctx.newMeans(7)
    ctx.blockMeans(pages, ints([list(range(7))]), ints([0]), ints([448]), means)
    keys, _ = R.unpack(pages.cpu().numpy(), 1, 64, 64)
    want = np.stack([L.block_mean(np.where(np.isnan(keys[b * 64:b * 64 + 64, 0]), np.nan, keys[b * 64:b * 64 + 64, 0])) for b in range(7)])
    got = numbers(means)[:, 0, 0]
    assert np.isnan(got[4]).all() and not np.isnan(got[[0, 1, 2, 3, 5, 6]]).any()
    assert np.array_equal(got, want, equal_nan=True)


@pytest.mark.parametrize("dim", [64, 256])
def test_means_of_keys_whose_sum_passes_32_bits(dim):
    """Finite keys near the end of bf16's range: equal ones, which lie in the biases, and others of either sign, which lie in the scales too."""
    ctx = context(heads=1, kvHeads=1, dim=dim, page=64, requests=1, tokens=1024)
    gen = generator(8)
    parts = [torch.full((64, 1, dim), sign * 2.0 ** e, device="cuda") for e, sign in ((115, 1), (117, -1), (118, 1), (121, -1), (122, 1), (127, -1))]
    parts += [2.0 ** e * (2 * torch.rand((64, 1, dim), generator=gen, device="cuda") - 1) for e in (112, 119, 120, 121, 122, 124, 126)]  # (a group's width stays below 2^128)
    parts += [2.0 ** e * torch.rand((64, 1, dim), generator=gen, device="cuda") for e in (120, 122, 127)]
    x = torch.cat(parts).bfloat16()
    blocks = len(parts)
    pages, slots = ctx.newCache(blocks), ints(range(blocks * 64))
    for a in range(0, blocks * 64, 1024):
        ctx.append(None, x[a:a + 1024], x[a:a + 1024], None, slots[a:a + 1024], slots[a:a + 1024], pages)
    means = ctx.newMeans(blocks)
    ctx.blockMeans(pages, ints([list(range(blocks))]), ints([0]), ints([blocks * 64]), means)
    keys, _ = R.unpack(pages.cpu().numpy(), 1, dim, 64)
    assert np.isfinite(keys).all()
    want = np.stack([L.block_mean(keys[b * 64:b * 64 + 64, 0]) for b in range(blocks)])
    assert np.array_equal(numbers(means)[:, 0, 0], want) and ctx.info().deviceErrorFlag == 0


def test_means_past_the_table_and_the_cache():
    ctx = context(heads=1, kvHeads=1, page=16, requests=1, tokens=256)
    pages, _ = cache_of(ctx, [256])
    means = ctx.newMeans(len(pages))
    means.fill_(9.0)
    ctx.blockMeans(pages, ints([[0, 1, 2, 3, 4]]), ints([0]), ints([256]), means)  # a row for 80 keys
    got = numbers(means)[:, 0, 0, 0]
    assert got[3] != 9.0 and (got[[0, 1, 2, 4, 5, 6, 7]] == 9.0).all()
    assert ctx.info().deviceErrorFlag == 14
    ctx.resetDeviceError()
    means.fill_(9.0)
    ctx.blockMeans(pages, ints([[0, 99999, 2, 3, 4, 5, 6, -1]]), ints([0]), ints([128]), means)
    got = numbers(means)
    assert (got[3] == 0.0).all() and (np.delete(got, 3, 0) == 9.0).all()
    assert ctx.info().deviceErrorFlag == 16


def random_means(gen, pages, ctx, loud=1.0):
    x = loud * numbers(torch.randn((pages, ctx.kvHeads, max(1, ctx.pageTokens // 64), ctx.headDim), generator=gen, device="cuda"))
    return torch.from_numpy(L.held(x, np.clip(L.exponent(x), -60, 60))).to("cuda").bfloat16()


def select_case(ctx, lengths, rows, blocks, first, last, spare=0, means=None, q=None, seed=5):
    gen = generator(seed)
    page = ctx.pageTokens
    used = [-(-n // page) for n in lengths]
    ids = np.random.RandomState(seed).permutation(sum(used) + 1)
    table, at = np.zeros((len(lengths), max(used + [1])), dtype=np.int64), 0
    for r, n in enumerate(used):
        table[r, :n] = ids[at:at + n]
        at += n
    means = random_means(gen, sum(used) + 1, ctx) if means is None else means
    tokens = sum(rows) + spare
    q = rows_of(gen, tokens, ctx.heads, ctx.headDim) if q is None else q
    start = np.concatenate([[0], np.cumsum(rows)])
    got = ctx.selectBlocks(q, means, ints(table), ints(start), ints(lengths), blocks, first=first, last=last).cpu().numpy()
    held = numbers(means)
    meansOf = []
    for r, n in enumerate(lengths):
        places = [mean_places(ctx, table, r, b) for b in range(n // 64)]
        meansOf.append(np.stack([held[w, :, p] for w, p in places]) if places else np.zeros((0, ctx.kvHeads, ctx.headDim)))
    want = L.select(numbers(q), meansOf, lengths, rows, ctx.kvHeads, blocks, first, last)
    return got, want


@pytest.mark.parametrize("heads,kvHeads", [(2, 2), (4, 2), (8, 2), (14, 2), (16, 1), (24, 2), (64, 1), (3, 1)])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_select_against_exact_scores(heads, kvHeads, dim):
    ctx = context(heads=heads, kvHeads=kvHeads, dim=dim, page=32, requests=8, tokens=512)
    lengths, rows = [900, 63, 64, 0, 2000, 700, 1300, 1], [3, 1, 1, 0, 1, 40, 0, 1]
    got, want = select_case(ctx, lengths, rows, 7, 1, 2)
    assert np.array_equal(got, want)
    assert ctx.info().deviceErrorFlag == 0


@pytest.mark.parametrize("page", [16, 64, 128, 256])
@pytest.mark.parametrize("blocks,first,last", [(1, 0, 1), (2, 1, 1), (4, 0, 1), (20, 3, 5), (40, 0, 40), (39, 2, 1), (600, 1, 1)])
def test_select_of_list_sizes(page, blocks, first, last):
    ctx = context(heads=4, kvHeads=2, page=page, requests=4, tokens=512)
    got, want = select_case(ctx, [2600, 65, 2559, 0], [2, 1, 5, 0], blocks, first, last)
    assert np.array_equal(got, want)


@pytest.mark.parametrize("heads,kvHeads,rows", [(4, 4, 300), (8, 4, 301), (16, 4, 200)])
def test_select_of_many_rows(heads, kvHeads, rows):
    """Several rows a CTA, over the ends of requests."""
    ctx = context(heads=heads, kvHeads=kvHeads, page=16, requests=6, tokens=1024)
    got, want = select_case(ctx, [1000, 1500, 640, 0, 2000, 300], [3, rows, 1, 0, 2, 290], 6, 1, 1)
    assert np.array_equal(got, want)


def test_select_rows_of_no_request():
    ctx = context(requests=3, tokens=64)
    got, want = select_case(ctx, [1000, 0, 500], [2, 0, 3], 4, 1, 1, spare=5)
    assert np.array_equal(got, want) and (got[5:] == -1).all()


def test_select_equal_scores_take_the_first():
    ctx = context(heads=2, kvHeads=1, page=64, requests=1, tokens=8)
    means = torch.zeros((61, 1, 1, 64), device="cuda", dtype=torch.bfloat16)
    got, want = select_case(ctx, [59 * 64 + 1], [1], 9, 2, 3, means=means)
    assert np.array_equal(got, want) and got[0, 0].tolist() == [0, 1, 2, 3, 4, 5, 57, 58, 59]
    # some of two values
    means[::7] = 1.0
    q = torch.ones((1, 2, 64), device="cuda").bfloat16()
    got, want = select_case(ctx, [59 * 64 + 1], [1], 7, 0, 1, means=means, q=q)
    assert np.array_equal(got, want)


def test_select_of_queries_and_means_at_the_ends_of_range():
    ctx = context(heads=4, kvHeads=1, page=64, requests=1, tokens=16)
    gen = generator(11)
    n = 40
    means = random_means(gen, n + 2, ctx)
    factors = 2.0 ** torch.randint(-58, 50, (n + 2, 1, 1, 1), generator=gen, device="cuda")
    means = (means.float() * factors).bfloat16()
    means[5] = float("nan")
    q = rows_of(gen, 8, 4, 64)
    scales = torch.tensor([[0, 0, 0, 0], [-130, -130, -131, -126], [110, 0, 100, -100], [0, -70, 0, -61], [100, 110, 120, 40], [0, 0, 0, 0], [0, 0, 0, 0],
                           [-100, -40, -140, 3]], device="cuda")
    q = (q.double() * 2.0 ** scales[:, :, None].double()).bfloat16()
    q[5] = 0
    q[6, 1, 7] = float("inf")
    q[6, 2, 9] = float("nan")
    for first in (0, 1):
        got, want = select_case(ctx, [n * 64 + 1], [8], 6, first, 1, means=means, q=q)
        assert np.array_equal(got, want)


def test_select_of_a_long_context():
    ctx = context(heads=2, kvHeads=1, dim=64, page=256, requests=1, tokens=8)
    got, want = select_case(ctx, [1 << 20], [2], 100, 4, 4)
    assert np.array_equal(got, want)
    got, want = select_case(ctx, [(1 << 21) - 5], [1], 1000, 4, 4)
    assert np.array_equal(got, want)


def test_select_past_the_table_and_the_cache():
    ctx = context(heads=2, kvHeads=1, page=64, requests=2, tokens=8)
    means = random_means(generator(), 12, ctx)
    q = rows_of(generator(), 2, 2, 64)
    table = np.arange(12).reshape(1, 12)
    got = ctx.selectBlocks(q, means, ints(table), ints([0, 2]), ints([5000]), 5).cpu().numpy()
    held = numbers(means)
    want = L.select(numbers(q), [held[:, :, 0]], [5000], [2], 1, 5, 1, 1, most=12)
    assert np.array_equal(got, want) and ctx.info().deviceErrorFlag == 14
    ctx.resetDeviceError()
    table[0, [3, 5]] = [99, -1]
    got = ctx.selectBlocks(q, means, ints(table), ints([0, 2]), ints([12 * 64]), 10).cpu().numpy()
    assert (got == [0, 1, 2, 4, 6, 7, 8, 9, 10, 11]).all()  # of the pages outside, which come last, none
    assert ctx.info().deviceErrorFlag == 16


def test_select_of_row_starts_that_go_back():
    ctx = context(heads=2, kvHeads=1, page=64, requests=3, tokens=8)
    means = random_means(generator(), 30, ctx)
    q = rows_of(generator(), 6, 2, 64)
    table = np.arange(30).reshape(3, 10)
    got = ctx.selectBlocks(q, means, ints(table), ints([0, 4, 2, 6]), ints([600, 600, 600]), 3).cpu().numpy()
    assert ((got >= -1) & (got < 10)).all() and ctx.info().deviceErrorFlag == 15


def test_select_strided_queries_on_another_stream_and_captured():
    ctx = context(heads=4, kvHeads=2, page=64, requests=2, tokens=64)
    gen = generator()
    means = random_means(gen, 41, ctx)
    wide = rows_of(gen, 6, 8, 64)
    q = wide[:, 2:6]
    table, start, lengths = ints(np.arange(40).reshape(2, 20)), ints([0, 2, 6]), ints([1280, 1200])
    want = ctx.selectBlocks(q.contiguous(), means, table, start, lengths, 5)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    got = ctx.selectBlocks(q, means, table, start, lengths, 5, stream=stream)
    stream.synchronize()
    assert torch.equal(got, want)
    ids = torch.empty_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ctx.selectBlocks(q, means, table, start, lengths, 5, ids=ids)
    for _ in range(3):
        ids.fill_(77)
        wide.copy_(rows_of(gen, 6, 8, 64))
        graph.replay()
        assert torch.equal(ids, ctx.selectBlocks(q.contiguous(), means, table, start, lengths, 5))


def test_refusals():
    from ane_fieldfare_b200.attention import FieldfareError

    ctx = context(heads=4, kvHeads=2, page=64, requests=2, tokens=8)
    means, table, start, lengths, q = ctx.newMeans(4), ints([[0, 1]]), ints([0, 1]), ints([100]), rows_of(generator(), 1, 4, 64)
    pages = ctx.newCache(4)
    for kw, says in [(dict(blocks=0), "blocks a list"), (dict(blocks=4, last=0), "own block"), (dict(blocks=4, first=4), "more than a list"),
                     (dict(blocks=4, first=1, last=4), "more than a list")]:
        with pytest.raises(FieldfareError, match=says):
            ctx.selectBlocks(q, means, table, start, lengths, **kw)
    for kw in [dict(blocks=-1), dict(blocks=4, first=-1), dict(blocks=4, last=1 << 32)]:
        with pytest.raises(ValueError):
            ctx.selectBlocks(q, means, table, start, lengths, **kw)
    with pytest.raises(FieldfareError, match="2\\^21 keys"):
        ctx.selectBlocks(q, means, ints(np.zeros((1, 32769))), start, lengths, 4)
    with pytest.raises(FieldfareError, match="maxRequests"):
        ctx.selectBlocks(q, means, ints(np.zeros((3, 2))), ints([0, 1, 1, 1]), ints([9, 9, 9]), 4)
    with pytest.raises(FieldfareError, match="maxTokens"):
        ctx.selectBlocks(rows_of(generator(), 9, 4, 64), means, table, start, lengths, 4)
    for bad in [dict(means=means.float()), dict(means=means[:, :, :, :32].contiguous()), dict(q=q.half()), dict(start=ints([0, 1, 1])), dict(table=ints([0, 1])),
                dict(ids=ints([[1, 2, 3, 4]])), dict(lengths=lengths.long()), dict(table=table.cpu())]:
        a = dict(q=q, means=means, table=table, start=start, lengths=lengths, ids=None) | bad
        with pytest.raises(ValueError):
            ctx.selectBlocks(a["q"], a["means"], a["table"], a["start"], a["lengths"], 4, ids=a["ids"])
    with pytest.raises(ValueError, match="number of pages"):
        ctx.blockMeans(pages, table, lengths, lengths, ctx.newMeans(3))
    with pytest.raises(ValueError, match="number of requests"):
        ctx.blockMeans(pages, table, ints([1, 2]), lengths, means)
    with pytest.raises(ValueError):
        ctx.blockMeans(pages.float(), table, lengths, lengths, means)
    assert ctx.selectBlocks(q[:0], means, table, ints([0, 0]), lengths, 4).shape == (0, 2, 4)
    ctx.blockMeans(pages, table[:0], lengths[:0], lengths[:0], means)


# ---- shared pages in the book-keeping -------------------------------------------------------------


def test_plan_with_shared_pages_page_by_page():
    """Every request's table row begins with pages of another's; they stay whatever its length does."""
    rng = np.random.RandomState(2)
    requests, page, pages, width = 12, 16, 90, 9
    ctx = context(page=page, requests=requests, tokens=2000)
    owner = 0
    sharedPages = np.array([0] + [4] * 6 + [2] * 4 + [0])
    table, free, count = np.full((requests, width), -1), np.full(pages, -1), pages
    free[:] = rng.permutation(pages)

    def step(old, new):
        nonlocal table, free, count
        rows = int(np.maximum(0, new - old).sum()) + 2
        out = dict(table=ints(table), free=ints(free), count=ints([count]), start=ints([0] * (requests + 1)), positions=ints([7] * rows), slots=ints([7] * rows))
        ctx.plan(ints(old), ints(new), out["table"], out["free"], out["count"], out["count"], out["start"], out["positions"], out["slots"], heldPages=ints(sharedPages))
        got = {k: v.cpu().numpy() for k, v in out.items()}
        stack, want = list(free[:count]), table.copy()
        up = lambda n, r: max(-(-n // page), sharedPages[r])  # noqa: E731
        for r in range(requests):
            stack += [int(p) for p in table[r, up(new[r], r):up(old[r], r)]]
        slots = []
        for r in range(requests):
            for i in range(up(old[r], r), up(new[r], r)):
                want[r, i] = stack.pop()
            slots += [want[r, p // page] * page + p % page if p // page >= sharedPages[r] else -1 for p in range(old[r], new[r])]
        assert np.array_equal(got["table"], want) and got["count"][0] == len(stack) and list(got["free"][:len(stack)]) == stack
        assert list(got["slots"]) == slots + [-1] * (rows - len(slots))
        table, free, count = got["table"], got["free"], len(stack)

    zero = np.zeros(requests, dtype=int)
    now = zero.copy()
    now[owner] = 70
    step(zero, now)
    table[1:, :4] = table[owner, :4]  # the caller's part
    before, now = now, now.copy()
    before = before.copy()
    before[1:] = sharedPages[1:] * page
    now[1:] = before[1:] + rng.randint(0, 60, requests - 1)
    step(before, now)
    for _ in range(6):
        then = np.where(rng.rand(requests) < 0.5, np.minimum(now + rng.randint(1, 20, requests), width * page), np.maximum(sharedPages * page, now - rng.randint(0, 30, requests)))
        then[owner] = 70
        step(now, then)
        now = then
    assert ctx.info().deviceErrorFlag == 0
    then = np.where(np.arange(requests) == owner, 70, 0)
    step(now, then)
    step(then, zero)
    assert count == pages and sorted(free) == list(range(pages))
    step(zero, np.where(np.arange(requests) == 3, 70, 0))  # new tokens on shared pages have no slot
    assert ctx.info().deviceErrorFlag == 20


def test_plan_refuses_shared_pages_of_another_number():
    ctx = context(page=16, requests=2)
    a = [ints([0, 0]), ints([0, 0]), ints([[0], [1]]), ints([2, 3]), ints([2]), ints([2]), ints([0, 0, 0]), ints([0]), ints([0])]
    for bad in (ints([0]), torch.zeros(2, device="cuda")):
        with pytest.raises(ValueError):
            ctx.plan(*a, heldPages=bad)
