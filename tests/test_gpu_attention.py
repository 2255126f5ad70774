"""The INT4 key/value cache and its attention on the GPU against plain statements in 64 bits."""
import numpy as np
import pytest
import torch

import attention_reference as R

pytestmark = pytest.mark.gpu


def context(heads=4, kvHeads=2, dim=64, page=16, requests=16, tokens=1024):
    from ane_fieldfare_b200 import attention

    return attention.AttentionContext(heads=heads, kvHeads=kvHeads, headDim=dim, pageTokens=page, maxRequests=requests, maxTokens=tokens)


def ints(values):
    return torch.tensor(np.asarray(values, dtype=np.int64).astype(np.int32), device="cuda")


def numbers(t):
    return t.detach().float().cpu().numpy().astype(np.float64)


def rows_of(gen, tokens, heads, dim, loud=1.0):
    return (loud * torch.randn((tokens, heads, dim), generator=gen, device="cuda")).bfloat16()


def generator(seed=7):
    return torch.Generator(device="cuda").manual_seed(seed)


# ---- book-keeping ------------------------------------------------------------------------------


def run_plan(ctx, old, new, table, free, count, rows):
    out = dict(table=ints(table), free=ints(free), count=ints([count]), start=ints([0] * (len(old) + 1)), positions=ints([7] * rows),
               slots=ints([7] * rows))
    ctx.plan(ints(old), ints(new), out["table"], out["free"], out["count"], out["count"], out["start"], out["positions"], out["slots"])
    return {k: v.cpu().numpy() for k, v in out.items()}


@pytest.mark.parametrize("requests,page,most,extra", [(1, 16, 1, 0), (1, 64, 200, 5), (7, 16, 60, 0), (33, 32, 500, 3), (1025, 16, 90, 1), (3000, 256, 900, 17)])
def test_plan_is_the_book_keeping_page_by_page(requests, page, most, extra):
    rng = np.random.RandomState(requests)
    old = rng.randint(0, most + 1, requests)
    new = np.where(rng.rand(requests) < 0.5, np.maximum(0, old + rng.randint(-40, 41, requests)), old)
    new = np.where(rng.rand(requests) < 0.1, 0, new)
    width = -(-int(max(old.max(), new.max(), 1)) // page)
    used = -(-old // page)
    pages = int(used.sum()) + requests * 3 + 2
    ids = rng.permutation(pages)
    table, free, at = np.full((requests, width), -1), np.full(pages, -1), 0
    for r in range(requests):
        table[r, :used[r]] = ids[at:at + used[r]]
        at += used[r]
    free[:pages - at] = ids[at:]
    rows = int(np.maximum(0, new - old).sum()) + extra
    ctx = context(page=page, requests=requests, tokens=max(1, rows))
    want = R.plan(old.tolist(), new.tolist(), table, free, pages - at, page, rows)
    got = run_plan(ctx, old, new, table, free, pages - at, rows)
    assert np.array_equal(got["table"], want[0])
    assert np.array_equal(got["free"], want[1])
    assert got["count"][0] == want[2]
    assert got["start"].tolist() == want[3]
    assert got["positions"].tolist() == want[4]
    assert got["slots"].tolist() == want[5]
    assert ctx.info().deviceErrorFlag == 0


def test_plan_gives_returned_pages_to_the_requests_that_grow():
    ctx = context(page=16)
    got = run_plan(ctx, [40, 0, 16], [0, 33, 17], [[5, 6, 7], [9, 9, 9], [4, 9, 9]], [3, -1, -1, -1, -1, -1, -1, -1], 1, 34)
    assert got["table"].tolist() == [[5, 6, 7], [7, 6, 5], [4, 3, 9]]
    assert got["count"][0] == 0
    assert got["start"].tolist() == [0, 0, 33, 34]
    assert got["slots"][[0, 32, 33]].tolist() == [112, 80, 48]


def test_plan_without_pages_or_room_says_so_and_stays_inside():
    ctx = context(page=16)
    got = run_plan(ctx, [0, 16], [40, 17], [[5, 5], [2, 5]], [0, 1, -1], 2, 41)
    # a request of three pages and a table row of two; then none is left
    assert got["table"].tolist() == [[1, 0], [2, -1]]
    assert got["slots"][:32].tolist() == list(range(16, 32)) + list(range(16))
    assert got["count"][0] == 0
    assert ctx.info().deviceErrorFlag in (13, 14)
    assert (got["slots"][32:] == -1).all()
    ctx.resetDeviceError()
    assert ctx.info().deviceErrorFlag == 0
    run_plan(ctx, [0], [5], [[0]], [3], 1, 4)
    assert ctx.info().deviceErrorFlag == 15


@pytest.mark.parametrize("requests,pages,most,steps", [(2, 4, 64, 12), (5, 9, 100, 30), (40, 70, 90, 12), (1500, 900, 40, 6)])
def test_plan_after_the_pages_ran_out(requests, pages, most, steps):
    """Requests that found no page shrink, end and grow again: every page is in one place all the time, and none is lost."""
    page, width, rng = 16, -(-most // 16), np.random.RandomState(requests)
    ctx = context(page=page, requests=requests, tokens=requests * most)
    table, free, count, old = np.full((requests, width), -1), np.full(pages, -1), pages, np.zeros(requests, dtype=int)
    free[:] = rng.permutation(pages)
    ranOut = 0
    for step in range(steps):
        new = np.where(rng.rand(requests) < 0.7, rng.randint(0, most + 1, requests), old)
        if step % 3 == 2:
            new = np.where(rng.rand(requests) < 0.5, 0, np.minimum(new, old))
        if step == steps - 1:
            new[:] = 0
        got = run_plan(ctx, old, new, table, free, count, requests * most)
        has = [list(table[r, :-(-old[r] // page)]) for r in range(requests)]
        stack = list(free[:count])
        for r in range(requests):
            while len(has[r]) > -(-new[r] // page):
                has[r].pop()
        for r in range(requests):  # given back in order of their places
            stack += [p for p in table[r, len(has[r]):-(-old[r] // page)] if p >= 0]
        short = False
        for r in range(requests):
            while len(has[r]) < -(-new[r] // page):
                has[r].append(stack.pop() if stack else -1)
                short |= has[r][-1] < 0
        assert [list(got["table"][r, :len(has[r])]) for r in range(requests)] == has
        assert got["count"][0] == len(stack) and list(got["free"][:len(stack)]) == stack
        held = [p for mine in has for p in mine if p >= 0]
        assert sorted(held + stack) == list(range(pages))
        slots = [has[r][p // page] * page + p % page if has[r][p // page] >= 0 else -1 for r in range(requests) for p in range(old[r], new[r])]
        assert list(got["slots"][:len(slots)]) == slots
        assert ctx.info().deviceErrorFlag == (13 if short else 0)
        ctx.resetDeviceError()
        ranOut += short
        table, free, count, old = got["table"], got["free"], len(stack), new
    assert ranOut and sorted(free) == list(range(pages))


def test_plan_does_not_hand_out_what_is_no_page():
    ctx = context(page=16)
    got = run_plan(ctx, [0], [40], [[7, 7, 7]], [2, 99, 0, -1], 3, 40)
    assert got["table"].tolist() == [[0, -1, 2]]
    assert got["slots"].tolist() == list(range(16)) + [-1] * 16 + list(range(32, 40))
    assert ctx.info().deviceErrorFlag == 13


@pytest.mark.parametrize("requests", [4, 1500])
def test_plan_of_lengths_that_are_none(requests):
    """Words of -1 in a batch: their requests end with their table rows, and the arrays with themselves."""
    ctx = context(page=16, requests=requests)
    new = [5] + [-1] * (requests - 2) + [7]
    pages = 2 * requests
    got = run_plan(ctx, [0] * requests, new, np.full((requests, 2), 99999), np.arange(pages), pages, 48)
    want = np.arange(pages)[::-1]
    assert got["table"].tolist() == [[want[0], 99999]] + [[want[1 + 2 * r], want[2 + 2 * r]] for r in range(requests - 2)] + [[want[2 * requests - 3], 99999]]
    assert got["count"][0] == 2
    assert got["positions"].tolist() == list(range(5)) + list(range(43))
    slot = lambda r, p: -1 if p >= 32 else got["table"][r, p // 16] * 16 + p % 16  # noqa: E731
    assert got["slots"].tolist() == [slot(0, p) for p in range(5)] + [slot(1, p) for p in range(43)]
    assert got["start"][:2].tolist() == [0, 5] and (got["start"][2:] >= 48).all()
    assert ctx.info().deviceErrorFlag in (14, 15)


# ---- rotary positions and append -----------------------------------------------------------------


def turned(x, table, rotary, interleaved):
    out = x.copy()
    for i in range(rotary // 2):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rotary // 2)
        c, s = table[:, i, 0][:, None], table[:, i, 1][:, None]
        out[..., a], out[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
    return out


@pytest.mark.parametrize("scaling", ["none", "linear", "byParts"])
def test_rotary_table_against_64_bits(scaling):
    ctx = context(dim=128)
    table = numbers(ctx.ropeTable(5000, base=500000.0, rotaryDim=96, scaling=scaling, factor=8.0, lowTurns=1.0, highTurns=4.0,
                                  originalContext=1000.0, amplitude=1.25))
    freq = 500000.0 ** (-2.0 * np.arange(48) / 96)
    if scaling == "linear":
        freq = freq / 8
    if scaling == "byParts":
        kept = np.clip((1000 * freq / (2 * np.pi) - 1) / 3, 0, 1)
        freq = freq * kept + freq / 8 * (1 - kept)
        assert 0 < np.sum((kept > 0) & (kept < 1)) < 48
    angle = np.arange(5000)[:, None] * freq
    # the angle's own error: pow to 2 ulp of 64 bits, times 5000; then one rounding to 32 bits
    assert np.abs(table - 1.25 * np.stack([np.cos(angle), np.sin(angle)], -1)).max() <= 1.25 * (2.0 ** -24 + 5000 * 2.0 ** -50)


@pytest.mark.parametrize("dim,rotary", [(64, 64), (64, 16), (128, 128), (128, 96), (256, 256), (256, 64), (256, 0)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_turns_pairs_and_rounds_once(dim, rotary, interleaved):
    ctx = context(dim=dim)
    gen = generator()
    x = rows_of(gen, 13, 5, dim)
    at = ints([0, 1, 2, 3, 700, 701, 99, 98, 5, 5, 5, 1023, 512])
    table = ctx.ropeTable(1024, rotaryDim=rotary) if rotary else None
    y = ctx.rope(x, table, at, interleaved=interleaved) if rotary else x.clone()
    want = turned(numbers(x), numbers(table)[at.cpu().numpy()], rotary, interleaved) if rotary else numbers(x)
    # two products and a sum rounded to 32 bits, then bf16
    assert np.all(np.abs(numbers(y) - want) <= 2.0 ** -8 * np.abs(want) + 2.0 ** -22 * 12)
    assert np.array_equal(numbers(y)[..., rotary:], numbers(x)[..., rotary:])
    if rotary:
        ctx.rope(x, table, at, x, interleaved=interleaved)  # in place
        assert torch.equal(x, y)


@pytest.mark.parametrize("dim,heads", [(64, 5), (256, 3)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_heads_that_do_not_rotate_pass_through_the_kernel(dim, heads, interleaved):
    """No rotary table: bit for bit what came in, NaN and all, at other strides."""
    ctx = context(dim=dim)
    x = torch.randint(-32768, 32768, (9, heads, dim), device="cuda", generator=generator()).to(torch.int16).view(torch.bfloat16)
    y = torch.zeros((9, heads + 2, dim), dtype=torch.bfloat16, device="cuda")
    before = ctx.info().kernelLaunches
    ctx.rope(x, None, ints([4_000_000_000 - (1 << 32)] * 9), y[:, 1:-1], interleaved=interleaved)
    assert torch.equal(y[:, 1:-1].contiguous().view(torch.int16), x.view(torch.int16)) and not y[:, 0].any() and not y[:, -1].any()
    assert ctx.info().kernelLaunches == before + 1 and ctx.info().deviceErrorFlag == 0


def test_a_position_outside_the_table_is_reported():
    ctx = context()
    x = rows_of(generator(), 2, 4, 64)
    y = ctx.rope(x, ctx.ropeTable(8), ints([7, 8]))
    assert ctx.info().deviceErrorFlag == 18
    assert torch.equal(y[1], x[1])  # turned as position 0


@pytest.mark.parametrize("dim,kvHeads,heads,page,tokens", [(64, 2, 14, 16, 1), (64, 1, 3, 32, 37), (128, 8, 32, 64, 50), (128, 3, 3, 16, 3),
                                                            (256, 8, 16, 64, 65), (256, 1, 16, 128, 2), (64, 5, 5, 256, 301)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_append_quantizes_what_the_definition_says(dim, kvHeads, heads, page, tokens, interleaved):
    ctx = context(heads, kvHeads, dim, page, tokens=tokens)
    gen = generator(tokens)
    qkv = rows_of(gen, tokens, heads + 2 * kvHeads, dim)  # one product's rows: strides of all three
    q, k, v = qkv.split([heads, kvHeads, kvHeads], dim=1)
    pages = -(-tokens // page) + 2
    cache = torch.full((pages, kvHeads, ctx.pageBytes // kvHeads), 0xA5, dtype=torch.uint8, device="cuda")
    slots = torch.randperm(pages * page, generator=gen, device="cuda")[:tokens].int()
    live = np.ones(tokens, dtype=bool)
    if tokens > 4:
        slots[3::7] = -1
        live[3::7] = False
    table = ctx.ropeTable(3000, rotaryDim=dim // 2)
    at = torch.arange(tokens, device="cuda", dtype=torch.int32) + 2000
    before = cache.clone()
    qOut = ctx.append(q, k, v, table, at, slots, cache, interleaved=interleaved)
    assert torch.equal(qOut, ctx.rope(q, table, at, interleaved=interleaved))
    kTurned = numbers(ctx.rope(k, table, at, interleaved=interleaved))
    keys, values = R.unpack(cache.cpu().numpy(), kvHeads, dim, page)
    held = slots.cpu().numpy()[live]
    assert np.array_equal(keys[held], R.quantized(kTurned)[3][live])
    assert np.array_equal(values[held], R.quantized(numbers(v))[3][live])
    # and half a step of each group's own scale away from what came in, where that did not lose its top
    codes, scale, low, value = R.quantized(kTurned)
    step = np.repeat(scale, 64, -1).reshape(kTurned.shape)
    assert np.all(np.abs(value - kTurned) <= step * (0.5 + 15 * 2.0 ** -8))
    # nothing else was written
    oldKeys, oldValues = R.unpack(before.cpu().numpy(), kvHeads, dim, page)
    others = np.setdiff1d(np.arange(pages * page), held)
    assert np.array_equal(keys[others], oldKeys[others], equal_nan=True) and np.array_equal(values[others], oldValues[others], equal_nan=True)
    kBack, vBack = ctx.read(cache, slots)
    want = R.to_bf16(np.where(live[:, None, None], keys[np.maximum(slots.cpu().numpy(), 0)], 0))
    assert np.array_equal(numbers(kBack), want)
    assert np.array_equal(numbers(vBack), R.to_bf16(np.where(live[:, None, None], values[np.maximum(slots.cpu().numpy(), 0)], 0)))
    assert ctx.info().deviceErrorFlag == 0


def test_append_of_constant_tiny_huge_and_broken_groups():
    ctx = context(2, 2, 128, 16, tokens=8)
    x = torch.zeros((8, 2, 128), device="cuda")
    x[0] = 3.25                                      # no range: the bias is the value
    x[1] = torch.linspace(-1, 1, 128, device="cuda") * 2.0 ** -120
    x[2] = torch.linspace(-1, 1, 128, device="cuda") * 2.0 ** 125
    x[3, 0, 5], x[4, 1, 100], x[5, 0, 70] = float("inf"), float("nan"), -float("inf")
    x[6, :, :64], x[6, :, 64:] = 3.0e38, -3.0e38
    x[7, 0, ::2], x[7, 0, 1::2] = 3.0e38, -3.0e38    # a range that 32 bits do not hold
    x = x.bfloat16()
    cache = ctx.newCache(1)
    slots = torch.arange(8, device="cuda", dtype=torch.int32)
    ctx.append(None, x, x, None, slots, slots, cache)
    keys, values = R.unpack(cache.cpu().numpy(), 2, 128, 16)
    want = R.quantized(numbers(x))[3]
    assert np.array_equal(keys[:8], want, equal_nan=True) and np.array_equal(values[:8], want, equal_nan=True)
    assert np.isnan(want[3, 0, :64]).all() and np.isfinite(want[3, 0, 64:]).all() and np.isnan(want[7, 0]).all()
    assert np.array_equal(keys[0], np.full((2, 128), 3.25))


def test_slots_outside_the_cache_are_reported_and_left_out():
    ctx = context(2, 2, 64, 16)
    x = rows_of(generator(), 2, 2, 64)
    cache = ctx.newCache(2)
    ctx.append(None, x, x, None, ints([0, 0]), ints([32, 3]), cache)
    assert ctx.info().deviceErrorFlag == 16
    keys, _ = R.unpack(cache.cpu().numpy(), 2, 64, 16)
    assert np.count_nonzero(np.abs(keys).sum((1, 2))) == 1
    assert not ctx.read(cache, ints([32]))[0].any()


# ---- attention -----------------------------------------------------------------------------------


class Batch:
    """Requests with filled caches, on shuffled pages, their rows' queries, and garbage wherever no key is."""

    def __init__(self, heads, kvHeads, dim, page, lengths, rows, *, seed=3, extraRows=0, loud=1.0, spare=3, tableExtra=1):
        self.shape = (heads, kvHeads, dim, page)
        self.lengths, self.rows, self.tokens = list(lengths), list(rows), sum(rows) + extraRows
        self.ctx = context(heads, kvHeads, dim, page, requests=len(lengths), tokens=max(1, self.tokens))
        gen, rng = generator(seed), np.random.RandomState(seed)
        used = [-(-n // page) for n in lengths]
        self.pageCount = sum(used) + spare
        ids = rng.permutation(self.pageCount)
        table, at = np.full((len(lengths), max(used + [0]) + tableExtra), -1), 0
        for r, u in enumerate(used):
            table[r, :u] = ids[at:at + u]
            at += u
        self.table = table
        # a word of NaN scales wherever nothing was written
        self.cache = torch.full((self.pageCount, kvHeads, self.ctx.pageBytes // kvHeads), 0xFF, dtype=torch.uint8, device="cuda")
        self.slots = [[int(table[r, p // page]) * page + p % page for p in range(n)] for r, n in enumerate(lengths)]
        flat = [s for mine in self.slots for s in mine]
        self.k, self.v = rows_of(gen, max(1, len(flat)), kvHeads, dim, loud), rows_of(gen, max(1, len(flat)), kvHeads, dim)
        for a in range(0, len(flat), 1024):  # (a handle takes as many rows at a time as it was made for)
            b = min(len(flat), a + 1024)
            with_room = context(heads, kvHeads, dim, page, tokens=1024)
            with_room.append(None, self.k[a:b], self.v[a:b], None, ints([0] * (b - a)), ints(flat[a:b]), self.cache)
        self.q = rows_of(gen, self.tokens, heads, dim)

    def attend(self, window=0, sinks=0, scale=None, maxRows=None, **more):
        start = np.concatenate([[0], np.cumsum(self.rows)])
        return self.ctx.attend(self.q, self.cache, ints(self.table), ints(start), ints(self.lengths),
                               max(self.rows + [1]) if maxRows is None else maxRows, window=window, sinks=sinks, scale=scale, **more)

    def check(self, got, window=0, sinks=0, scale=None):
        heads, kvHeads, dim, page = self.shape
        keys, values = R.unpack(self.cache.cpu().numpy(), kvHeads, dim, page)
        scale = dim ** -0.5 if scale is None else scale
        want, bound = R.attention(numbers(self.q), keys, values, self.slots, self.lengths, self.rows, window, sinks, scale)
        got = numbers(got)
        assert np.isfinite(got).all()
        assert np.all(np.abs(got - want) <= 2.0 ** -8 * np.abs(want) + bound)
        # bf16 rounding alone is 1.65e-3 of random values; operands of 11 bits add about a quarter of that
        assert np.linalg.norm(got - want) <= 2.5e-3 * np.linalg.norm(want) + 1e-30
        assert self.ctx.info().deviceErrorFlag == 0


SHAPES = [(4, 2, 64, 16), (14, 2, 64, 32), (8, 2, 128, 64), (3, 3, 128, 16), (4, 2, 256, 64), (16, 1, 256, 128), (40, 1, 64, 256)]


@pytest.mark.parametrize("heads,kvHeads,dim,page", SHAPES)
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (30, 3), (64, 100)])
def test_decode_rows(heads, kvHeads, dim, page, window, sinks):
    b = Batch(heads, kvHeads, dim, page, [1, 2, 15, 16, 17, 63, 64, 65, 0, 200, 333], [1] * 8 + [0, 1, 1])
    b.check(b.attend(window, sinks), window, sinks)


@pytest.mark.parametrize("heads,kvHeads,dim,page", SHAPES)
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 1), (40, 4)])
def test_verify_rows(heads, kvHeads, dim, page, window, sinks):
    b = Batch(heads, kvHeads, dim, page, [16, 16, 70, 5, 0, 129, 300, 31], [16, 1, 7, 2, 0, 16, 3, 16])
    b.check(b.attend(window, sinks), window, sinks)


@pytest.mark.parametrize("heads,kvHeads,dim,page", SHAPES)
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (50, 4), (200, 70)])
def test_prefill_rows(heads, kvHeads, dim, page, window, sinks):
    b = Batch(heads, kvHeads, dim, page, [17, 64, 65, 300, 1, 0, 193, 129], [17, 64, 1, 130, 1, 0, 40, 128])
    b.check(b.attend(window, sinks), window, sinks)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("rows", [1, 9, 40])
def test_one_long_request_is_split_and_joined(dim, rows):
    b = Batch(4, 2, dim, 64, [5000], [rows])
    b.check(b.attend())
    b.check(b.attend(700, 5), 700, 5)


@pytest.mark.parametrize("dim,page", [(64, 16), (64, 64), (128, 16), (256, 16)])
def test_many_tiles_a_cta(dim, page):
    """The rings of the kernel for many rows go round several times, with tiles whose pieces lie on several pages."""
    b = Batch(16, 2, dim, page, [1500, 700], [260, 130])
    want = b.attend().clone()
    b.check(want)
    for _ in range(20):
        assert torch.equal(b.attend(), want)


@pytest.mark.parametrize("rows", [[1, 1, 0], [5, 16, 0], [30, 2, 0]])
def test_rows_without_keys_and_spare_rows_are_zero(rows):
    b = Batch(4, 2, 128, 16, [40, 33, 0], rows, extraRows=5)
    b.lengths[1] = rows[1] - 1  # its first row stands at position -1 and sees nothing
    out = b.attend(out=torch.full_like(b.q, 7.0))
    assert not out[sum(rows):].any()
    assert not out[rows[0]].any()
    assert out[:rows[0]].any()
    b.check(out)


@pytest.mark.parametrize("rows", [1, 4, 33])
def test_what_is_masked_may_hold_anything(rows):
    """Keys of the cache that no row sees: NaN, infinities and the largest numbers, in pages that rows do see."""
    b = Batch(4, 2, 64, 16, [100, 150], [rows, rows])
    want = b.attend(20, 2).clone()
    gone = [s for r, n in enumerate(b.lengths) for s in b.slots[r][2:n - rows - 20]]
    keys = torch.zeros((len(gone), 2, 64), device="cuda")
    keys[0::3], keys[1::3], keys[2::3, :, ::2] = float("nan"), float("inf"), 3.3e38
    keys = keys.bfloat16()
    context(4, 2, 64, 16).append(None, keys, keys, None, ints([0] * len(gone)), ints(gone), b.cache)
    assert torch.equal(b.attend(20, 2), want)


@pytest.mark.parametrize("rows", [1, 4, 33])
def test_a_key_that_is_not_a_number_reaches_the_rows_that_see_it_and_no_other(rows):
    b = Batch(4, 2, 64, 16, [100, 90], [rows, rows])
    want = b.attend().clone()
    bad = torch.full((1, 2, 64), float("nan"), device="cuda").bfloat16()
    b.ctx.append(None, bad, bad, None, ints([0]), ints([b.slots[0][10]]), b.cache)
    got = b.attend()
    assert torch.isnan(got[:rows]).all()
    assert torch.equal(got[rows:], want[rows:])


@pytest.mark.parametrize("rows", [1, 4, 33])
@pytest.mark.parametrize("power", [-60, -14, 13, 40, 100])
def test_keys_and_values_of_any_size(rows, power):
    """The cache's scale follows a model's; what is scaled by a power of two gives the scaled result."""
    b = Batch(4, 2, 128, 16, [130], [rows])
    factor = 2.0 ** power
    b.ctx, many = context(4, 2, 128, 16, tokens=256), len(b.k)
    b.ctx.append(None, (b.k.float() * factor).bfloat16(), (b.v.float() / factor).bfloat16(), None, ints([0] * many), ints(b.slots[0]), b.cache)
    b.check(b.attend(scale=128 ** -0.5 / factor), scale=128 ** -0.5 / factor)


@pytest.mark.parametrize("rows", [1, 4, 33])
@pytest.mark.parametrize("power", [-100, -20, 20, 100])
def test_queries_of_any_size(rows, power):
    b = Batch(4, 2, 128, 16, [130], [rows])
    b.q = (b.q.float() * 2.0 ** power).bfloat16()
    b.check(b.attend(scale=128 ** -0.5 / 2.0 ** power), scale=128 ** -0.5 / 2.0 ** power)


@pytest.mark.parametrize("rows", [1, 4, 33])
@pytest.mark.parametrize("window,sinks", [(0, 0), (20, 2)])
@pytest.mark.parametrize("which", ["all zero", "one zero", "tiny", "zero keys"])
@pytest.mark.parametrize("power", [0, -80])
def test_rows_whose_logits_vanish(rows, window, sinks, which, power):
    """Queries of zero, or so small that no logit differs from zero: the mean of the visible values; their neighbours stay."""
    b = Batch(4, 2, 128, 16, [150, 70], [rows, max(1, rows - 3)])
    if which == "all zero":
        b.q.zero_()
    elif which == "one zero":
        b.q[rows // 2, 1] = 0
        b.q[rows] = 0
    elif which == "tiny":
        b.q = (b.q.float() * 2.0 ** -125).bfloat16()
    else:
        b.q = (b.q.float() * 2.0 ** -60).bfloat16()
        many = 220
        b.k[:130] = 0
        b.ctx = context(4, 2, 128, 16, tokens=many)
        b.ctx.append(None, b.k, b.v, None, ints([0] * many), ints([s for mine in b.slots for s in mine]), b.cache)
    scale = 128 ** -0.5 * 2.0 ** power
    b.check(b.attend(window, sinks, scale=scale), window, sinks, scale=scale)


@pytest.mark.parametrize("rows", [1, 6, 50])
def test_sharp_logits(rows):
    """One key far above the rest: the running maximum moves, weights vanish."""
    b = Batch(4, 2, 64, 16, [400], [rows], loud=12.0)
    b.check(b.attend(scale=1.0), scale=1.0)


@pytest.mark.parametrize("rows", [1, 6, 50])
def test_values_of_very_different_sizes(rows):
    b = Batch(4, 2, 64, 16, [300], [rows])
    v = b.v.float()
    v[::7] *= 2.0 ** 12
    v[128:192] *= 2.0 ** -12
    b.ctx = context(4, 2, 64, 16, tokens=300)
    b.ctx.append(None, b.k, v.bfloat16(), None, ints([0] * 300), ints(b.slots[0]), b.cache)
    b.check(b.attend())


@pytest.mark.parametrize("rows,length", [(1, 300), (6, 300), (50, 300), (1, 4000), (30, 4000)])
@pytest.mark.parametrize("small", [0.0, 2.0 ** -90])
@pytest.mark.parametrize("power", [26, 60, 110])
@pytest.mark.parametrize("where", ["first", "last", "between"])
def test_weights_of_small_values_count_beside_large_ones(rows, length, small, power, where):
    """Tiles of values that are zero or tiny among large ones: their weights are in the sum all the same."""
    b = Batch(4, 2, 64, 16, [length], [rows])
    v = b.v.float() * 2.0 ** power
    third = length // 3
    v[{"first": slice(0, third), "last": slice(2 * third, length), "between": slice(third, 2 * third)}[where]] *= small / 2.0 ** power
    for a in range(0, length, 1024):
        c = min(length, a + 1024)
        context(4, 2, 64, 16, tokens=1024).append(None, b.k[a:c], v[a:c].bfloat16(), None, ints([0] * (c - a)), ints(b.slots[0][a:c]), b.cache)
    b.check(b.attend())


@pytest.mark.parametrize("rows", [1, 12, 70])
def test_strides_streams_and_repeats(rows):
    b = Batch(8, 2, 128, 32, [500, 77, 1200], [rows] * 3)
    want = b.attend()
    wide = torch.zeros((b.tokens, 20, 128), dtype=torch.bfloat16, device="cuda")
    wide[:, 3:11] = b.q
    out = torch.full((b.tokens, 11, 128), 5.0, dtype=torch.bfloat16, device="cuda")
    b.q = wide[:, 3:11]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = b.attend(out=out[:, 2:10], stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    assert (out[:, :2] == 5).all() and (out[:, 10:] == 5).all()
    for _ in range(20):  # the same bits, whatever the order in which CTAs end
        assert torch.equal(b.attend(), want)


def test_outputs_are_memory_of_the_stream_that_writes_them():
    """What a call allocates for a stream is not what the current stream may still be using."""
    b = Batch(4, 2, 64, 16, [5000], [1000], seed=5)
    table, at, slots = b.ctx.ropeTable(64), ints([5] * 1000), ints(b.slots[0][:1000])
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    calls = [((1000, 4, 64), lambda: [b.attend(stream=side)]), ((1000, 4, 64), lambda: [b.ctx.rope(b.q, table, at, stream=side)]),
             ((1000, 4, 64), lambda: [b.ctx.append(b.q, b.k[:1000], b.v[:1000], table, at, slots, b.cache, stream=side)]),
             ((1000, 2, 64), lambda: b.ctx.read(b.cache, slots, stream=side)), ((4000, 2, 64), lambda: [b.ctx.ropeTable(4000, rotaryDim=64, stream=side)])]
    for shape, run in calls:
        torch.cuda.synchronize()
        used = [torch.empty(shape, dtype=torch.bfloat16, device="cuda") for _ in range(3)]
        held = {t.data_ptr() for t in used}
        del used  # (the current stream's work on them may be in flight)
        out = run()
        torch.cuda.synchronize()
        assert not held & {t.data_ptr() for t in out}


@pytest.mark.parametrize("rows,bound", [(1, 16), (1, 400), (9, 16), (9, 100), (100, 4096)])
def test_the_bound_on_a_requests_rows_may_be_loose(rows, bound):
    b = Batch(4, 2, 128, 16, [400, 111], [rows, 1])
    b.check(b.attend(maxRows=bound))


def test_a_step_in_a_graph_follows_the_lengths():
    """plan, append and attend captured once; the lengths change between replays."""
    heads, kvHeads, dim, page = 4, 2, 64, 16
    ctx = context(heads, kvHeads, dim, page, requests=3, tokens=8)
    cache, table, free, count = ctx.newCache(40), ints(np.zeros((3, 12))), ints(np.arange(40)), ints([40])
    old, new, start = ints([0, 0, 0]), ints([0, 0, 0]), ints([0] * 4)
    at, slots = ints([0] * 8), ints([0] * 8)
    gen = generator()
    q, k, v = rows_of(gen, 8, heads, dim), rows_of(gen, 8, kvHeads, dim), rows_of(gen, 8, kvHeads, dim)
    rope = ctx.ropeTable(200)
    qOut, out = torch.empty_like(q), torch.empty_like(q)

    def step():
        ctx.plan(old, new, table, free, count, count, start, at, slots)
        ctx.append(q, k, v, rope, at, slots, cache, qOut)
        ctx.attend(qOut, cache, table, start, new, 4, out=out)

    step()  # no row yet
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    have = [0, 0, 0]
    held = [[], [], []]
    for want in ([3, 0, 4], [4, 1, 8], [4, 4, 9], [2, 5, 0], [5, 6, 4]):
        old.copy_(ints(have))
        new.copy_(ints(want))
        for t in (q, k, v):
            t.copy_(rows_of(gen, 8, t.shape[1], dim))
        graph.replay()
        torch.cuda.synchronize()
        row = 0
        for r in range(3):
            held[r] = held[r][:want[r]]
            for p in range(have[r], want[r]):
                held[r].append((numbers(ctx.rope(k, rope, at))[row], numbers(v)[row]))
                row += 1
        rows = [max(0, b - a) for a, b in zip(have, want)]
        flat = [kv for mine in held for kv in mine]
        keys = R.quantized(np.array([kv[0] for kv in flat]))[3]
        values = R.quantized(np.array([kv[1] for kv in flat]))[3]
        ends = np.cumsum([0] + [len(mine) for mine in held])
        exact, bound = R.attention(numbers(qOut), keys, values, [list(range(ends[r], ends[r + 1])) for r in range(3)],
                                   [n if m else 0 for n, m in zip(want, rows)], rows, 0, 0, dim ** -0.5)
        assert np.all(np.abs(numbers(out) - exact) <= 2.0 ** -8 * np.abs(exact) + bound)
        assert int(count) == 40 - sum(-(-n // page) for n in want)
        have = want
    assert ctx.info().deviceErrorFlag == 0


@pytest.mark.parametrize("rows", [1, 20])
def test_pages_behind_four_gigabytes(rows):
    heads, kvHeads, dim, page = 2, 2, 256, 256
    ctx = context(heads, kvHeads, dim, page, tokens=600)
    pages = (1 << 32) // ctx.pageBytes + 3
    cache = torch.empty((pages, kvHeads, ctx.pageBytes // kvHeads), dtype=torch.uint8, device="cuda")
    table = ints([[pages - 1, 0, pages - 2]])
    gen = generator()
    slots = [[int(table[0, p // page]) * page + p % page for p in range(600)]]
    k, v, q = rows_of(gen, 600, kvHeads, dim), rows_of(gen, 600, kvHeads, dim), rows_of(gen, rows, heads, dim)
    ctx.append(None, k, v, None, ints([0] * 600), ints(slots[0]), cache)
    kBack, vBack = ctx.read(cache, ints(slots[0]))
    kHeld, vHeld = R.quantized(numbers(k))[3], R.quantized(numbers(v))[3]
    assert np.array_equal(numbers(kBack), R.to_bf16(kHeld)) and np.array_equal(numbers(vBack), R.to_bf16(vHeld))
    got = numbers(ctx.attend(q, cache, table, ints([0, rows]), ints([600]), rows))
    want, bound = R.attention(numbers(q), kHeld, vHeld, [list(range(600))], [600], [rows], 0, 0, dim ** -0.5)
    assert np.all(np.abs(got - want) <= 2.0 ** -8 * np.abs(want) + bound)


@pytest.mark.parametrize("rows", [1, 40])
def test_pages_outside_the_cache_are_not_read(rows):
    b = Batch(4, 2, 64, 16, [100], [rows])
    b.table[0, 2] = b.pageCount
    out = b.attend()
    assert torch.isfinite(out).all()
    assert b.ctx.info().deviceErrorFlag == 16
    b.ctx.resetDeviceError()
    b.table = b.table[:, :5].copy()  # a row of the table that ends before the request does
    b.table[0, 2] = 0
    b.attend()
    assert b.ctx.info().deviceErrorFlag == 14


@pytest.mark.parametrize("rows", [1, 7, 40])
@pytest.mark.parametrize("requests,length", [(1, 113), (1, 100_000), (3, -1), (64, -1)])
def test_a_length_past_the_table_row_ends_with_it(rows, requests, length):
    """The keys that the table has room for are seen, those behind it do not exist and take no time."""
    heads, kvHeads, dim, page = 8, 8, 64, 16
    b = Batch(heads, kvHeads, dim, page, [112] * requests, [rows] * requests, tableExtra=0)
    keys, values = R.unpack(b.cache.cpu().numpy(), kvHeads, dim, page)
    b.lengths = [length] * requests
    for window, sinks in ((0, 0), (1 << 30, 3), (64, 3)):
        p = [(length if length > 0 else 2 ** 31 - 1) - rows + i for i in range(rows)] * requests
        mine = [b.slots[n // rows] for n in range(requests * rows)]
        seen = [[s for j, s in enumerate(mine[n]) if j <= p[n] and (not window or j > p[n] - window or j < sinks)] for n in range(requests * rows)]
        want, bound = R.attention(numbers(b.q), keys, values, seen, [len(s) for s in seen], [1] * len(seen), 0, 0, dim ** -0.5)
        got = numbers(b.attend(window, sinks))
        assert np.all(np.abs(got - want) <= 2.0 ** -8 * np.abs(want) + bound)
        assert b.ctx.info().deviceErrorFlag == 14
        b.ctx.resetDeviceError()


@pytest.mark.parametrize("rows", [1, 40])
def test_row_starts_that_go_back_are_reported(rows):
    b = Batch(4, 2, 64, 16, [100, 90, 80], [rows] * 3)
    args = ints(b.table), ints([0, 2 * rows, rows, 3 * rows]), ints(b.lengths), 2 * rows
    out = b.ctx.attend(b.q, b.cache, *args, out=torch.full_like(b.q, 7.0))
    assert not out.any()
    assert b.ctx.info().deviceErrorFlag == 15
    b.ctx.resetDeviceError()
    b.check(b.attend())


@pytest.mark.parametrize("rows", [1, 40])
def test_more_work_than_a_call_counts_is_reported(rows):
    """1024 heads over a table of 2^31 keys, none of them there: 2^35 tiles."""
    ctx = context(1024, 1024, 64, 16, requests=1, tokens=rows)
    q = rows_of(generator(), rows, 1024, 64)
    table = torch.full((1, 1 << 27), -1, dtype=torch.int32, device="cuda")
    out = ctx.attend(q, ctx.newCache(1), table, ints([0, rows]), ints([2 ** 31 - 1]), rows, out=torch.full_like(q, 7.0))
    assert not out.any()
    assert ctx.info().deviceErrorFlag == 19


@pytest.mark.parametrize("rows", [1, 40])
def test_a_reset_clears_what_a_call_that_gave_up_leaves(rows):
    """The counts of parts that have arrived: no call leaves them but one that gave up a wait, so they are set from outside."""
    import ctypes

    class Handle(ctypes.Structure):  # FFAttention of csrc/ff_attention.cuh, up to the counts
        _fields_ = [("device", ctypes.c_int), ("smCount", ctypes.c_int), ("config", ctypes.c_uint32 * 6), ("errorFlag", ctypes.c_void_p),
                    ("planCount", ctypes.c_void_p), ("rowsCtas", ctypes.c_uint32), ("partials", ctypes.c_void_p), ("stats", ctypes.c_void_p),
                    ("arrived", ctypes.c_void_p)]

    class Words:
        def __init__(self, pointer, count):
            self.__cuda_array_interface__ = {"shape": (count,), "typestr": "<i4", "data": (pointer, False), "version": 3}

    b = Batch(4, 2, 64, 16, [3000], [rows])
    handle = ctypes.cast(b.ctx.handle, ctypes.POINTER(Handle)).contents
    assert list(handle.config)[:4] == [4, 2, 64, 16] and handle.rowsCtas == 2 * handle.smCount
    arrived = torch.as_tensor(Words(handle.arrived, 3 * handle.rowsCtas), device="cuda")
    planned = torch.as_tensor(Words(handle.planCount, 1), device="cuda")
    assert not arrived.any() and not planned.any()
    arrived.fill_(1)
    planned.fill_(1)
    b.ctx.resetDeviceError()
    assert not arrived.any() and not planned.any()
    b.check(b.attend())


# ---- refusals --------------------------------------------------------------------------------------


def test_arguments_that_the_library_refuses():
    from ane_fieldfare_b200.attention import FieldfareError

    b = Batch(4, 2, 64, 16, [40, 40], [1, 1])
    ctx, start = b.ctx, ints([0, 1, 2])
    good = dict(q=b.q, pages=b.cache, blockTable=ints(b.table), rowStart=start, lengths=ints(b.lengths), maxRows=1)
    for change, error, says in [
            (dict(q=b.q.float()), ValueError, "bf16"),
            (dict(q=b.q[:, :3]), ValueError, "4"),
            (dict(q=b.q.transpose(1, 2).contiguous().transpose(1, 2)), ValueError, "side by side"),
            (dict(q=b.q.cpu()), ValueError, "bf16 on"),
            (dict(pages=b.cache[:, :1]), ValueError, "bytes a page"),
            (dict(blockTable=ints(b.table).long()), ValueError, "int32"),
            (dict(lengths=ints([1])), ValueError, "number of requests"),
            (dict(maxRows=0), FieldfareError, "maxRows"),
            (dict(window=-1), ValueError, "negative"),
            (dict(sinks=2), FieldfareError, "sinks need a window"),
            (dict(scale=0.0), FieldfareError, "scale"),
            (dict(scale=float("nan")), FieldfareError, "scale"),
            (dict(q=torch.zeros((3, 4, 64), dtype=torch.bfloat16, device="cuda")), FieldfareError, "maxTokens")]:
        args = {**good, **change}
        with pytest.raises(error, match=says):
            ctx.attend(args.pop("q"), args.pop("pages"), args.pop("blockTable"), args.pop("rowStart"), args.pop("lengths"), args.pop("maxRows"), **args)
    wide = torch.zeros((2, 4 * 64 + 4), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(FieldfareError, match="16-byte"):
        ctx.attend(wide[:, 4:].unflatten(1, (4, 64)), b.cache, ints(b.table), start, ints(b.lengths), 1)
    with pytest.raises(FieldfareError, match="rotaryDim"):
        ctx.rope(b.q, torch.zeros((4, 12, 2), device="cuda"), ints([0, 1]))
    with pytest.raises(FieldfareError, match="rotaryDim"):
        ctx.ropeTable(4, rotaryDim=72)
    with pytest.raises(FieldfareError, match="factor"):
        ctx.ropeTable(4, scaling="linear", factor=0.0)
    with pytest.raises(ValueError, match="one position"):
        ctx.append(b.q, b.k[:2], b.v[:2], None, ints([0]), ints([0, 1]), b.cache)
    with pytest.raises(FieldfareError, match="maxRequests"):
        ctx.plan(ints([0] * 3), ints([0] * 3), ints(np.zeros((3, 2))), ints([0]), ints([0]), ints([0]), ints([0] * 4), ints([0]), ints([0]))
    assert ctx.attend(b.q[:0], b.cache, ints(b.table), ints([0, 0, 0]), ints(b.lengths), 1).shape == (0, 4, 64)


def test_numbers_past_32_bits_are_not_cut():
    """Rows further apart than 2^32 elements are refused; windows, sinks and bounds on rows past 2^32 are what they say."""
    b = Batch(4, 2, 64, 16, [300, 200], [2, 2])
    far = torch.empty((1 << 32) + 4096, dtype=torch.bfloat16, device="cuda")
    q = far.as_strided((4, 4, 64), ((1 << 32) // 3 // 8 * 8, 64, 1))  # below 2^32, the last row past it
    q.copy_(b.q)
    b.check(b.ctx.attend(q, b.cache, ints(b.table), ints([0, 2, 4]), ints(b.lengths), 2))
    q = far.as_strided((2, 4, 64), ((1 << 32) + 256, 64, 1))
    q.copy_(b.q[:2])
    one = ints(b.table[:1]), ints([0, 2]), ints(b.lengths[:1])
    with pytest.raises(ValueError, match="apart"):
        b.ctx.attend(q, b.cache, *one, 2)
    with pytest.raises(ValueError, match="apart"):
        b.ctx.attend(b.q[:2], b.cache, *one, 2, out=q)
    del far, q
    want = b.attend()
    assert torch.equal(b.attend(window=(1 << 32) + 5), want)
    assert torch.equal(b.attend(window=1 << 32, sinks=(1 << 32) + 3), want)
    assert torch.equal(b.attend(window=7, sinks=(1 << 32) + 3), want)
    assert torch.equal(b.ctx.attend(b.q, b.cache, ints(b.table), ints([0, 2, 4]), ints(b.lengths), (1 << 32) + 2),
                       b.ctx.attend(b.q, b.cache, ints(b.table), ints([0, 2, 4]), ints(b.lengths), 4))


def test_a_table_that_is_too_large_to_count_is_refused():
    from ane_fieldfare_b200.attention import FieldfareError
    from ane_fieldfare_b200.binding import call

    ctx, word = context(requests=4), ints([0] * 8)
    with pytest.raises(FieldfareError, match="2\\^30"):
        call("ff_cache_plan", ctx.handle, word.data_ptr(), word.data_ptr(), 4, word.data_ptr(), (1 << 28) + 1, word.data_ptr(), 1, word.data_ptr(),
             word.data_ptr(), word.data_ptr(), word.data_ptr(), word.data_ptr(), 1, None)


def test_kernels_are_counted():
    b = Batch(4, 2, 64, 16, [40], [1])
    before = b.ctx.info().kernelLaunches
    b.attend()
    assert b.ctx.info().kernelLaunches > before
    b.ctx.close()
    with pytest.raises(Exception, match="destroyed"):
        b.attend()
