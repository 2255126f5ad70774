"""Attention over listed blocks of the INT4 cache against the plain statement in 64 bits."""
import numpy as np
import pytest
import torch

import attention_reference as R
import long_context_reference as L
from test_gpu_attention import SHAPES, Batch, context, generator, ints, numbers, rows_of

pytestmark = pytest.mark.gpu


def lists(b, blocks, seed=1, kind="chosen"):
    """Lists [tokens][kvHeads][blocks]: chosen: ascending, the row's own last, -1 behind; any: any order, some twice, some none."""
    rng, kvHeads = np.random.RandomState(seed), b.shape[1]
    out = np.full((b.tokens, kvHeads, blocks), -1, dtype=np.int64)
    at = 0
    for n, m in zip(b.lengths, b.rows):
        for i in range(m):
            p = n - m + i
            for h in range(kvHeads):
                seen = p // 64 + 1 if p >= 0 else 0
                if kind == "chosen":
                    mine = sorted(rng.permutation(max(0, seen - 1))[:blocks - 1].tolist()) + ([seen - 1] if seen else [])
                else:
                    mine = rng.randint(-1, seen + 2, blocks).tolist()
                out[at + i, h, :len(mine)] = mine
        at += m
    return out


def attend(b, ids, **more):
    start = np.concatenate([[0], np.cumsum(b.rows)])
    return b.ctx.attendSelected(b.q, b.cache, ints(b.table), ints(start), ints(b.lengths), ints(ids), **more)


def check(b, got, ids, scale=None):
    heads, kvHeads, dim, page = b.shape
    keys, values = R.unpack(b.cache.cpu().numpy(), kvHeads, dim, page)
    counted = ids.copy()  # of a list the first p / 64 + 1 entries
    at = 0
    for n, m in zip(b.lengths, b.rows):
        for i in range(m):
            counted[at + i, :, (n - m + i) // 64 + 1 if n - m + i >= 0 else 0:] = -1
        at += m
    want, bound = L.attention_listed(numbers(b.q), keys, values, b.slots, b.lengths, b.rows, counted, dim ** -0.5 if scale is None else scale)
    got = numbers(got)
    assert np.isfinite(got).all()
    # a rounding of a bf16 result, and what 11-bit operands leave
    assert np.all(np.abs(got - want) <= 2.0 ** -8 * np.abs(want) + bound)
    assert np.linalg.norm(got - want) <= 2.5e-3 * np.linalg.norm(want) + 1e-30
    assert b.ctx.info().deviceErrorFlag == 0


@pytest.mark.parametrize("heads,kvHeads,dim,page", SHAPES)
@pytest.mark.parametrize("blocks", [1, 2, 5, 40])
@pytest.mark.parametrize("kind", ["chosen", "any"])
def test_rows_of_a_batch(heads, kvHeads, dim, page, blocks, kind):
    b = Batch(heads, kvHeads, dim, page, [1, 2, 15, 63, 64, 65, 0, 200, 833, 700], [1, 1, 1, 2, 1, 3, 0, 1, 1, 20])
    if kind == "any":  # a row without a key would be zeros, which the last check is not made for
        b.lengths[6] = 0
    ids = lists(b, blocks, kind=kind)
    check(b, attend(b, ids), ids)


@pytest.mark.parametrize("heads,kvHeads", [(2, 2), (64, 1), (24, 2)])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_all_blocks_are_the_attention_over_all_keys(heads, kvHeads, dim):
    b = Batch(heads, kvHeads, dim, 64, [300, 64, 1, 1000], [3, 1, 1, 5])
    ids = np.full((b.tokens, kvHeads, 16), -1, dtype=np.int64)
    at = 0
    for n, m in zip(b.lengths, b.rows):
        for i in range(m):
            seen = (n - m + i) // 64 + 1
            ids[at + i, :, :seen] = np.arange(seen)
        at += m
    b.check(attend(b, ids))


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_one_row_of_many_blocks_is_split_and_joined(dim):
    b = Batch(4, 2, dim, 64, [9000], [1])
    ids = lists(b, 130)
    want = attend(b, ids).clone()
    check(b, want, ids)
    for _ in range(10):
        assert torch.equal(attend(b, ids), want)


@pytest.mark.parametrize("rows", [161, 400, 900])
def test_many_rows(rows):
    """More rows than a CTA has threads."""
    b = Batch(4, 2, 64, 16, [1000, 70, 0, 500], [rows, 3, 0, 11])
    ids = lists(b, 3)
    check(b, attend(b, ids), ids)


def test_many_requests():
    """More requests than the kernel keeps in shared memory, most of them idle."""
    requests = 700
    b = Batch(2, 1, 64, 16, [100] * requests, [1 if r % 3 == 0 else 0 for r in range(requests)])
    ids = lists(b, 2)
    check(b, attend(b, ids), ids)


def test_rows_without_keys_and_of_no_request_are_zero():
    b = Batch(4, 2, 128, 16, [40, 33, 0], [1, 3, 0], extraRows=5)
    b.lengths[1] = 2  # its first row stands at position -1
    ids = np.zeros((9, 2, 3), dtype=np.int64)
    ids[0] = -1
    out = attend(b, ids, out=torch.full_like(b.q, 7.0))
    assert not out[:2].any() and not out[4:].any() and out[2:4].any()
    # rows in front of the first request, and no request
    out = b.ctx.attendSelected(b.q, b.cache, ints(b.table), ints([2, 3, 4, 4]), ints(b.lengths), ints(np.zeros((9, 2, 3))), out=torch.full_like(b.q, 7.0))
    assert not out[:2].any() and out[2].any() and not out[4:].any()
    out = b.ctx.attendSelected(b.q, b.cache, ints(np.zeros((0, 3))), ints([0]), ints([]), ints(np.zeros((9, 2, 3))), out=torch.full_like(b.q, 7.0))
    assert not out.any() and b.ctx.info().deviceErrorFlag == 0


def test_a_block_that_is_named_twice_counts_twice():
    b = Batch(2, 1, 64, 64, [300], [1])
    ids = np.array([[[0, 2, 2, 2, -1]]])
    check(b, attend(b, ids), ids)
    ids = np.array([[[-1, 1 << 25, 3, 3, 2 ** 31 - 1]]])
    check(b, attend(b, ids), ids)


def test_a_key_that_is_not_a_number_reaches_the_rows_that_name_its_block():
    b = Batch(4, 2, 64, 16, [200, 190], [2, 1])
    ids = np.array([[[0, 3], [1, 3]], [[1, 3], [2, 3]], [[0, 2], [0, 2]]])
    want = attend(b, ids).clone()
    bad = torch.full((1, 2, 64), float("nan"), device="cuda").bfloat16()
    b.ctx.append(None, bad, bad, None, ints([0]), ints([b.slots[0][70]]), b.cache)
    got = attend(b, ids)
    assert torch.isnan(got[0, 2:]).all() and torch.isnan(got[1, :2]).all()
    assert torch.equal(got[0, :2], want[0, :2]) and torch.equal(got[1, 2:], want[1, 2:]) and torch.equal(got[2], want[2])


def test_the_length_ends_inside_the_last_block():
    """What lies behind a row in its own block is not seen, whatever it is."""
    b = Batch(4, 2, 64, 64, [130], [3])
    ids = np.array([[[0, 2], [1, 2]]] * 3)
    check(b, attend(b, ids), ids)


def test_pages_outside_the_cache_and_the_table():
    b = Batch(4, 2, 64, 16, [300], [1])
    ids = np.array([[[0, 2, 4], [1, 3, 4]]])
    page = b.table[0, 2]
    b.table[0, 2] = b.pageCount
    assert torch.isfinite(attend(b, ids)).all() and b.ctx.info().deviceErrorFlag == 16
    b.ctx.resetDeviceError()
    b.table = b.table[:, :10].copy()
    b.table[0, 2] = page
    assert torch.isfinite(attend(b, ids)).all() and b.ctx.info().deviceErrorFlag == 14


def test_row_starts_that_go_back_are_reported():
    b = Batch(4, 2, 64, 16, [100, 90, 80], [2] * 3)
    out = b.ctx.attendSelected(b.q, b.cache, ints(b.table), ints([0, 4, 2, 6]), ints(b.lengths), ints(np.zeros((6, 2, 1))), out=torch.full_like(b.q, 7.0))
    assert not out.any() and b.ctx.info().deviceErrorFlag == 15


@pytest.mark.parametrize("length", [-1, 2 ** 31 - 1])
def test_lengths_that_are_none(length):
    b = Batch(2, 1, 64, 16, [200], [2])
    b.lengths = [length]
    ids = np.array([[[0, 1, 2]], [[0, 2, -1]]])
    got = numbers(attend(b, ids))
    keys, values = R.unpack(b.cache.cpu().numpy(), 1, 64, 16)
    want, bound = L.attention_listed(numbers(b.q), keys, values, b.slots, [200], [2], ids, 0.125)
    assert np.all(np.abs(got - want) <= 2.0 ** -8 * np.abs(want) + bound)


def test_strides_streams_and_graphs():
    heads, kvHeads, dim, page = 8, 2, 128, 64
    b = Batch(heads, kvHeads, dim, page, [700, 300], [1, 2])
    ids = lists(b, 4)
    want = attend(b, ids).clone()
    wide = torch.zeros((3, 3 * heads, dim), device="cuda").bfloat16()
    wide[:, heads:2 * heads] = b.q
    out = torch.full((3, 2 * heads, dim), 7.0, device="cuda").bfloat16()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    args = ints(b.table), ints([0, 1, 3]), ints(b.lengths), ints(ids)
    b.ctx.attendSelected(wide[:, heads:2 * heads], b.cache, *args, out=out[:, :heads], stream=stream)
    stream.synchronize()
    assert torch.equal(out[:, :heads], want) and (out[:, heads:] == 7.0).all()
    out, args = torch.empty_like(want), args
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.ctx.attendSelected(b.q, b.cache, *args, out=out)
    for seed in range(3):
        ids = lists(b, 4, seed=seed)
        args[3].copy_(ints(ids))
        b.q.copy_(rows_of(generator(seed), 3, heads, dim))
        graph.replay()
        check(b, out, ids)


def test_select_and_attend_one_behind_the_other():
    """append, block means, selection and attention over what it lists, as a decode step makes them."""
    heads, kvHeads, dim, page = 4, 2, 64, 32
    b = Batch(heads, kvHeads, dim, page, [64 * 9 + 3, 400], [1, 1])
    b.ctx = context(heads, kvHeads, dim, page, requests=2, tokens=2)
    means = b.ctx.newMeans(b.pageCount)
    table, lengths, start = ints(b.table), ints(b.lengths), ints([0, 1, 2])
    b.ctx.blockMeans(b.cache, table, ints([0, 0]), lengths, means)
    ids = b.ctx.selectBlocks(b.q, means, table, start, lengths, 4)
    got = b.ctx.attendSelected(b.q, b.cache, table, start, lengths, ids)
    check(b, got, ids.cpu().numpy().astype(np.int64))
    keys, _ = R.unpack(b.cache.cpu().numpy(), kvHeads, dim, page)
    meansOf = [np.stack([[L.block_mean(keys[mine[c * 64:c * 64 + 64], h]) for h in range(kvHeads)] for c in range(len(mine) // 64)]) for mine in b.slots]
    assert np.array_equal(ids.cpu().numpy(), L.select(numbers(b.q), meansOf, b.lengths, b.rows, kvHeads, 4, 1, 1))


def test_refusals():
    from ane_fieldfare_b200.attention import FieldfareError

    b = Batch(4, 2, 64, 16, [100], [1])
    ids, table, start, lengths = ints(np.zeros((1, 2, 3))), ints(b.table), ints([0, 1]), ints([100])
    call = lambda **kw: b.ctx.attendSelected(**(dict(q=b.q, pages=b.cache, blockTable=table, rowStart=start, lengths=lengths, ids=ids) | kw))  # noqa: E731
    for kw in [dict(ids=ids[:, :1].contiguous()), dict(ids=ids[0]), dict(ids=ids.long()), dict(ids=ids.cpu()), dict(rowStart=lengths), dict(q=b.q.float()),
               dict(out=torch.empty_like(b.q).float()), dict(pages=b.cache[:, :1].contiguous()), dict(blockTable=table[0])]:
        with pytest.raises(ValueError):
            call(**kw)
    for kw, says in [(dict(ids=ids[:, :, :0].contiguous()), "blocks a list"), (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale"),
                     (dict(blockTable=ints(np.zeros((2, 3))), rowStart=ints([0, 1, 1]), lengths=ints([1, 1])), "maxRequests")]:
        with pytest.raises(FieldfareError, match=says):
            call(**kw)
    assert call(q=b.q[:0], ids=ids[:0], rowStart=ints([0, 0])).shape == (0, 4, 64)


@pytest.mark.parametrize("rows", [1, 20])
def test_pages_behind_four_gigabytes(rows):
    """Means, selected blocks and a shared prefix of keys whose pages lie past what 32 bits reach."""
    heads, kvHeads, dim, page = 2, 2, 256, 256
    ctx = context(heads, kvHeads, dim, page, requests=2, tokens=1300)
    pages = (1 << 32) // ctx.pageBytes + 8
    cache = torch.empty((pages, kvHeads, ctx.pageBytes // kvHeads), dtype=torch.uint8, device="cuda")
    table = np.array([[pages - 1, 0, pages - 2, pages - 3], [pages - 1, 0, pages - 4, pages - 5]])
    lengths, prefix = [900, 700], 512
    gen = generator()
    slots = [[int(table[r, p // page]) * page + p % page for p in range(n)] for r, n in enumerate(lengths)]
    flat = slots[0] + slots[1][prefix:]
    k, v, q = rows_of(gen, len(flat), kvHeads, dim), rows_of(gen, len(flat), kvHeads, dim), rows_of(gen, 2 * rows, heads, dim)
    ctx.append(None, k, v, None, ints([0] * len(flat)), ints(flat), cache)
    means = ctx.newMeans(pages)
    start, held = ints([0, rows, 2 * rows]), ints(lengths)
    ctx.blockMeans(cache, ints(table), ints([0, 0]), held, means)
    kHeld, vHeld = R.quantized(numbers(k))[3], R.quantized(numbers(v))[3]
    place = {s: i for i, s in enumerate(flat)}
    at = [[place[s] for s in mine] for mine in slots]
    meansOf = [np.stack([[L.block_mean(kHeld[mine[b * 64:b * 64 + 64], h]) for h in range(kvHeads)] for b in range(len(mine) // 64)]) for mine in at]
    ids = ctx.selectBlocks(q, means, ints(table), start, held, 5)
    chosen = ids.cpu().numpy().astype(np.int64)
    assert np.array_equal(chosen, L.select(numbers(q), meansOf, lengths, [rows, rows], kvHeads, 5, 1, 1))
    got = numbers(ctx.attendSelected(q, cache, ints(table), start, held, ids))
    want, bound = L.attention_listed(numbers(q), kHeld, vHeld, at, lengths, [rows, rows], chosen, dim ** -0.5)
    assert np.all(np.abs(got - want) <= 2.0 ** -8 * np.abs(want) + bound)
    got = numbers(ctx.attendShared(q, cache, ints(table), start, held, rows, ints([0, 2]), ints([prefix]), always=True))
    want, bound = R.attention(numbers(q), kHeld, vHeld, at, lengths, [rows, rows], 0, 0, dim ** -0.5)
    assert np.all(np.abs(got - want) <= 2.0 ** -8 * np.abs(want) + bound)
    assert ctx.info().deviceErrorFlag == 0
