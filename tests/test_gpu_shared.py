"""Attention of requests that share prefixes over the INT4 cache: against the plain statement in 64 bits, which knows of no sharing."""
import numpy as np
import pytest
import torch

from test_gpu_attention import SHAPES, Batch, context, generator, ints, numbers, rows_of

pytestmark = pytest.mark.gpu


class Shared(Batch):
    """A batch whose requests groups[g] .. groups[g + 1] - 1 have the pages of the first of them for their first prefix[g] keys."""

    def __init__(self, heads, kvHeads, dim, page, lengths, rows, groups, prefix, **more):
        super().__init__(heads, kvHeads, dim, page, lengths, rows, **more)
        self.groups, self.prefix = list(groups), list(prefix)
        for g, n in enumerate(prefix):
            pages = n // page
            for r in range(groups[g], groups[g + 1]):
                have = min(pages, -(-self.lengths[r] // page))
                self.table[r, :have] = self.table[groups[g], :have]
        self.slots = [[int(self.table[r, p // page]) * page + p % page for p in range(n)] for r, n in enumerate(self.lengths)]

    def shared(self, scale=None, maxRows=None, always=True, **more):
        start = np.concatenate([[0], np.cumsum(self.rows)])
        return self.ctx.attendShared(self.q, self.cache, ints(self.table), ints(start), ints(self.lengths), max(self.rows + [1]) if maxRows is None else maxRows,
                                     ints(self.groups), ints(self.prefix), scale=scale, always=always, **more)


# few columns in both launches, many in the first alone, many in both
ROWS = [[1, 1, 1], [1, 2, 1, 0, 1, 2], [1] * 20, [3, 16, 5, 1, 0, 16], [40, 130, 1, 33]]


@pytest.mark.parametrize("heads,kvHeads,dim,page", SHAPES)
@pytest.mark.parametrize("rows", ROWS)
def test_one_group(heads, kvHeads, dim, page, rows):
    prefix = 512
    lengths = [prefix + m + 37 * i % 150 for i, m in enumerate(rows)]
    b = Shared(heads, kvHeads, dim, page, lengths, rows, [0, len(rows)], [prefix])
    b.check(b.shared())


@pytest.mark.parametrize("dim,page", [(64, 16), (128, 32), (256, 256)])
@pytest.mark.parametrize("rows", [1, 5, 30])
@pytest.mark.parametrize("prefix", [[0, 256, 1024], [768, 64, 63], [1024, 1024, 1], [256, 512, 300]])
def test_groups_and_requests_of_none(dim, page, rows, prefix):
    """Three groups of unequal sizes, one of a single request; requests in front of and behind the groups; prefixes that are no whole page."""
    requests, groups = 10, [1, 3, 4, 8]
    whole = [n // page * page for n in prefix]
    lengths = [300, *[whole[0] + 70 + i for i in range(2)], whole[1] + 100, *[whole[2] + 64 * i + 40 for i in range(4)], 90, 1000]
    many = [min(n, rows + r % 2) for r, n in enumerate(lengths)]
    b = Shared(4, 2, dim, page, lengths, many, groups, whole)
    b.check(b.shared())


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("rows", [[1] * 12, [1, 1], [20, 7, 90]])
def test_a_long_prefix_is_split_and_joined(dim, rows):
    prefix = 6400
    b = Shared(4, 2, dim, 64, [prefix + m + 10 * i for i, m in enumerate(rows)], rows, [0, len(rows)], [prefix])
    want = b.shared().clone()
    b.check(want)
    for _ in range(10):
        assert torch.equal(b.shared(), want)


@pytest.mark.parametrize("rows", [1, 9, 40])
def test_long_requests_behind_a_prefix_are_split_and_joined(rows):
    b = Shared(8, 2, 128, 64, [4000, 3500], [rows, rows], [0, 2], [640])
    b.check(b.shared())


@pytest.mark.parametrize("rows", [1, 6, 40])
def test_rows_inside_the_prefix(rows):
    """Requests that have not come to the prefix's end, or just so: their rows see what they see, no more."""
    prefix = 256
    lengths = [prefix + 100, prefix, prefix + 1, prefix - 1, 200, rows, prefix + rows, prefix + rows - 1]
    b = Shared(4, 2, 64, 64, lengths, [rows] * 8, [0, 8], [prefix])
    b.check(b.shared())


@pytest.mark.parametrize("rows", [[1, 1, 0], [5, 16, 0], [30, 2, 0]])
def test_rows_without_keys_and_of_no_request_are_zero(rows):
    b = Shared(4, 2, 128, 16, [140, 133, 0], rows, [0, 1], [128], extraRows=5)
    b.lengths[1] = rows[1] - 1  # its first row stands at position -1 and sees nothing
    out = b.shared(out=torch.full_like(b.q, 7.0))
    assert not out[sum(rows):].any() and not out[rows[0]].any() and out[:rows[0]].any()
    b.check(out)
    out = b.ctx.attendShared(b.q, b.cache, ints(np.zeros((0, 3))), ints([0]), ints([]), 1, ints([0]), ints([]), out=torch.full_like(b.q, 7.0))
    assert not out.any() and b.ctx.info().deviceErrorFlag == 0


def test_no_group_is_the_attention_of_the_requests():
    b = Shared(4, 2, 64, 16, [100, 300], [1, 3], [0], [])
    b.check(b.shared())
    assert torch.equal(b.shared(), b.attend())
    b = Shared(4, 2, 64, 16, [100, 300], [20, 33], [1, 1, 1], [64, 64])  # groups of no request
    assert torch.equal(b.shared(), b.attend())


def test_the_bound_on_a_requests_rows():
    b = Shared(4, 2, 64, 16, [200, 230], [3, 9], [0, 2], [128])
    for bound in (9, 100, 10 ** 12):
        b.check(b.shared(maxRows=bound))
    out = b.shared(maxRows=5)
    assert not out[8:].any() and b.ctx.info().deviceErrorFlag == 15


@pytest.mark.parametrize("rows", [1, 4, 33])
@pytest.mark.parametrize("where", ["prefix", "suffix", "both"])
def test_a_key_that_is_not_a_number_reaches_the_rows_that_see_it(rows, where):
    b = Shared(4, 2, 64, 16, [200, 190 + rows, 150], [rows, rows, rows], [0, 2], [128])
    want = b.shared().clone()
    bad = torch.full((1, 2, 64), float("nan"), device="cuda").bfloat16()
    for slot in ([b.slots[0][70]] if where != "suffix" else []) + ([b.slots[0][129]] if where != "prefix" else []):
        b.ctx.append(None, bad, bad, None, ints([0]), ints([slot]), b.cache)
    got = b.shared()
    assert torch.isnan(got[:rows]).all()
    assert torch.isnan(got[rows:2 * rows]).all() if where != "suffix" else torch.equal(got[rows:2 * rows], want[rows:2 * rows])
    assert torch.equal(got[2 * rows:], want[2 * rows:])


@pytest.mark.parametrize("rows", [1, 4, 33])
@pytest.mark.parametrize("loud", [["prefix"], ["suffix"]])
def test_one_part_far_above_the_other(rows, loud):
    """The logits of one part exceed the other's by hundreds."""
    b = Shared(4, 2, 64, 16, [200 + rows] * 3, [rows] * 3, [0, 3], [128])
    many = len(b.k)
    at = np.arange(many) % (200 + rows)
    strong = torch.from_numpy((at < 128) if loud == ["prefix"] else (at >= 128)).to("cuda")[:, None, None]
    b.k = torch.where(strong, b.k.float() * 300, b.k.float()).bfloat16()
    writer = context(4, 2, 64, 16, tokens=many)
    flat = [int(s) for r in range(3) for s in b.slots[r]]
    writer.append(None, b.k, b.v, None, ints([0] * many), ints([s if (r == 0 or p >= 128) else -1 for r in range(3) for p, s in enumerate(b.slots[r])]), b.cache)
    assert len(flat) == many
    b.check(b.shared(scale=1.0), scale=1.0)


@pytest.mark.parametrize("rows", [1, 33])
@pytest.mark.parametrize("power", [-60, 40, 100])
def test_keys_and_values_of_any_size(rows, power):
    factor = 2.0 ** power
    b = Shared(4, 2, 128, 16, [330, 300 + rows], [rows, rows], [0, 2], [256])
    writer, many = context(4, 2, 128, 16, tokens=1024), len(b.k)
    held = [s for mine in b.slots for s in mine]
    keep = [s if held.index(s) == i else -1 for i, s in enumerate(held)]
    writer.append(None, (b.k.float() * factor).bfloat16(), (b.v.float() / factor).bfloat16(), None, ints([0] * many), ints(keep), b.cache)
    b.check(b.shared(scale=128 ** -0.5 / factor), scale=128 ** -0.5 / factor)


@pytest.mark.parametrize("rows", [1, 40])
def test_pages_outside_the_cache_are_not_read(rows):
    b = Shared(4, 2, 64, 16, [300, 290], [rows, rows], [0, 2], [256])
    page = b.table[0, 2]
    b.table[0, 2] = b.pageCount
    assert torch.isfinite(b.shared()).all() and b.ctx.info().deviceErrorFlag == 16
    b.ctx.resetDeviceError()
    b.table[0, 2] = page
    b.prefix = [10 ** 6]  # longer than a row of the table
    b.shared()
    b.ctx.resetDeviceError()
    b.prefix = [256]
    b.check(b.shared())


def test_a_prefix_longer_than_what_the_requests_hold():
    """No row comes behind it: every request by itself."""
    b = Shared(4, 2, 64, 16, [300, 290], [2, 3], [0, 2], [256], tableExtra=60)
    b.prefix = [640]
    b.check(b.shared())


@pytest.mark.parametrize("rows", [1, 40])
def test_row_starts_and_groups_that_go_back_are_reported(rows):
    b = Shared(4, 2, 64, 16, [200, 190, 180], [rows] * 3, [0, 3], [128])
    for start, groups in (([0, 2 * rows, rows, 3 * rows], [0, 3]), ([0, rows, 2 * rows, 3 * rows], [2, 0, 3])):
        out = b.ctx.attendShared(b.q, b.cache, ints(b.table), ints(start), ints(b.lengths), 2 * rows, ints(groups), ints([128] * (len(groups) - 1)), always=True, out=torch.full_like(b.q, 7.0))
        assert not out.any() and b.ctx.info().deviceErrorFlag == 15
        b.ctx.resetDeviceError()
    b.check(b.shared())
    b.groups = [0, 99]  # more requests than there are
    b.check(b.shared())


@pytest.mark.parametrize("rows", [1, 40])
def test_more_work_than_a_call_counts_is_reported(rows):
    """1024 heads over a prefix of 2^31 keys, none of them there: 2^35 tiles in the first launch, few in the second."""
    ctx = context(1024, 1024, 64, 16, requests=1, tokens=rows)
    q = rows_of(generator(), rows, 1024, 64)
    table = torch.full((1, 1 << 27), -1, dtype=torch.int32, device="cuda")
    out = ctx.attendShared(q, ctx.newCache(1), table, ints([0, rows]), ints([2 ** 31 - 1]), rows, ints([0, 1]), ints([2 ** 31 - 1 - rows]), always=True, out=torch.full_like(q, 7.0))
    assert not out.any()
    assert ctx.info().deviceErrorFlag == 19


@pytest.mark.parametrize("rows", [1, 20])
def test_strides_streams_and_graphs(rows):
    heads, kvHeads, dim, page = 8, 2, 128, 64
    b = Shared(heads, kvHeads, dim, page, [700, 600 + rows, 650], [rows, rows, 1], [0, 3], [576])
    want = b.shared().clone()
    b.check(want)
    tokens = 2 * rows + 1
    wide = torch.zeros((tokens, 3 * heads, dim), device="cuda").bfloat16()
    wide[:, heads:2 * heads] = b.q
    out = torch.full((tokens, 2 * heads, dim), 7.0, device="cuda").bfloat16()
    args = ints(b.table), ints([0, rows, 2 * rows, tokens]), ints(b.lengths), rows, ints(b.groups), ints(b.prefix)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    b.ctx.attendShared(wide[:, heads:2 * heads], b.cache, *args, always=True, out=out[:, :heads], stream=stream)
    stream.synchronize()
    assert torch.equal(out[:, :heads], want) and (out[:, heads:] == 7.0).all()
    out = torch.empty_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.ctx.attendShared(b.q, b.cache, *args, always=True, out=out)
    for lengths, prefix in (([700, 600 + rows, 650], [576]), ([650, 600, 640], [512]), ([576 + rows, 600, 10], [576])):
        b.lengths = lengths
        b.slots = [[int(b.table[r, p // page]) * page + p % page for p in range(n)] for r, n in enumerate(lengths)]
        args[2].copy_(ints(lengths))
        args[5].copy_(ints(prefix))
        b.q.copy_(rows_of(generator(lengths[0]), tokens, heads, dim))
        graph.replay()
        b.check(out)


@pytest.mark.parametrize("dim,page", [(64, 64), (128, 16), (128, 64), (256, 64)])
def test_many_rows_are_the_same_every_time(dim, page):
    """Logits that pass the maximum again and again: outputs are rescaled between products that run ahead of the rows."""
    b = Shared(16, 2, dim, page, [1500, 700], [260, 130], [0, 2], [512], loud=3.0)
    want, alone = b.shared().clone(), b.attend().clone()
    b.check(want)
    b.check(alone)
    for _ in range(150):
        assert torch.equal(b.shared(), want) and torch.equal(b.attend(), alone)


def test_many_requests():
    """More requests than a CTA has threads, in groups of five."""
    requests = 1000
    b = Shared(2, 1, 64, 64, [70 + r % 60 for r in range(requests)], [1 if r % 3 else 0 for r in range(requests)], list(range(0, requests + 1, 5)), [64] * 200)
    b.check(b.shared())


# by the rule of ff_attention.cu, 0.1 ns saved eight heads of 40 times 64 keys: 40 requests of one row (40 * 20 - 2 * 62) * 40 * 8 = 216320, 12 of
# nine (12 * 44 - 4 * 62) * 40 * 8 = 89600, 30 of nine (30 * 44 - 9 * 62) * 40 * 8 = 243840; 200000 are needed
@pytest.mark.parametrize("requests,rows,shares", [(2, 1, False), (40, 1, True), (12, 9, False), (30, 9, True), (3, 200, False)])
def test_where_sharing_is_chosen_by_its_cost(requests, rows, shares):
    prefix = 2560
    b = Shared(32, 8, 128, 64, [prefix + rows + 11 * r % 60 for r in range(requests)], [rows] * requests, [0, requests], [prefix], tableExtra=0)
    want = numbers(b.attend())
    for bound in (None, prefix, 64, 0, 10 ** 12):
        before = b.ctx.info().kernelLaunches
        got = numbers(b.shared(always=False, maxPrefix=bound))
        assert b.ctx.info().kernelLaunches - before == (3 if shares and bound not in (64, 0) else 1)
        assert np.linalg.norm(got - want) <= 5e-3 * np.linalg.norm(want)  # (either is within 2.5e-3 of the exact rows, as the other tests hold)
    assert b.ctx.info().deviceErrorFlag == 0


def test_refusals():
    from ane_fieldfare_b200.attention import FieldfareError

    b = Shared(4, 2, 64, 16, [100, 100], [1, 1], [0, 2], [64])
    table, start, lengths, groups, prefix = ints(b.table), ints([0, 1, 2]), ints([100, 100]), ints([0, 2]), ints([64])
    call = lambda **kw: b.ctx.attendShared(**(dict(q=b.q, pages=b.cache, blockTable=table, rowStart=start, lengths=lengths, maxRows=1, groupStart=groups, prefixLengths=prefix) | kw))  # noqa: E731
    for kw in [dict(groupStart=prefix), dict(prefixLengths=groups), dict(groupStart=groups.long()), dict(prefixLengths=prefix.cpu()), dict(maxRows=-1), dict(maxPrefix=-1), dict(rowStart=lengths),
               dict(q=b.q.float()), dict(out=torch.empty_like(b.q).float()), dict(blockTable=table[0]), dict(pages=b.cache[:, :1].contiguous())]:
        with pytest.raises(ValueError):
            call(**kw)
    for kw, says in [(dict(scale=0.0), "scale"), (dict(maxRows=0), "maxRows"), (dict(groupStart=ints([0, 1, 2, 2]), prefixLengths=ints([64] * 3)), "more groups"),
                     (dict(blockTable=ints(np.zeros((3, 3))), rowStart=ints([0, 1, 1, 1]), lengths=ints([1, 1, 1])), "maxRequests")]:
        with pytest.raises(FieldfareError, match=says):
            call(**kw)
    assert call(q=b.q[:0], rowStart=ints([0, 0, 0])).shape == (0, 4, 64)
    assert numbers(call()).shape == (2, 4, 64)


def test_a_step_without_rows_may_say_so_in_its_bound():
    """As `attend` has it: nothing to do, whatever maxRows is."""
    b = Shared(4, 2, 64, 16, [100, 100], [1, 1], [0, 2], [64])
    none = ints([0, 0, 0])
    for always in (False, True):
        assert b.ctx.attendShared(b.q[:0], b.cache, ints(b.table), none, ints(b.lengths), 0, ints(b.groups), ints(b.prefix), always=always).shape == (0, 4, 64)
    assert b.ctx.attend(b.q[:0], b.cache, ints(b.table), none, ints(b.lengths), 0).shape == (0, 4, 64)


def test_memory_is_taken_where_prefixes_are_shared_alone():
    """Room for the rows' results over the prefixes, 32 bits each, is needed only by calls that share."""
    b = Shared(8, 2, 128, 64, [900] * 2, [400, 400], [0, 2], [64])
    want = b.shared(always=False, maxPrefix=64).clone()
    out = torch.empty_like(want)

    def peak(**kw):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        b.shared(out=out, **kw)
        return torch.cuda.max_memory_allocated() - before

    small = 1 << 16  # (the step's lists)
    assert peak(always=False, maxPrefix=64) < small and torch.equal(out, want)
    assert peak(always=True) >= 800 * 8 * (128 * 4 + 8)
    b.check(out)


def test_more_groups_than_threads():
    """In either kernel over the prefixes; in the one of few rows most requests have none."""
    b = Shared(2, 1, 64, 64, [66 + r % 60 for r in range(2200)], [1] * 2200, list(range(0, 2201, 2)), [64] * 1100)
    b.check(b.shared())
    rows = [1 if r % 90 == 7 else 0 for r in range(700)]
    b = Shared(2, 1, 64, 64, [130 + r % 60 for r in range(700)], rows, [*range(0, 698, 2), 700], [128] * 349)
    assert sum(rows) * 2 <= 16
    b.check(b.shared())
