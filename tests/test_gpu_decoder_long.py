"""Shared prefixes and selected blocks in the decoder put together from the operators."""
import numpy as np
import pytest
import torch

import attention_reference as R
import long_context_reference as L

pytestmark = pytest.mark.gpu


def numbers(t):
    return t.detach().float().cpu().numpy().astype(np.float64)


def run(book, unit, x, steps):
    """Attention rows of the layer, [request][token] -> row, over steps of lengths; x(request, token) its input."""
    out = {}
    for want in steps:
        have, step = list(book.lengths), book.step(want)
        rows = [(r, p) for r, (a, b) in enumerate(zip(have, want)) for p in range(a, b)]
        if rows:
            got = unit.attend(torch.stack([x[r][p] for r, p in rows]), step)
            for i, at in enumerate(rows):
                out[at] = got[i]
    return out


def inputs(requests, tokens, shared, seed=3):
    """Inputs of requests whose first `shared` tokens are the same."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((requests, tokens, 256), generator=gen, device="cuda").bfloat16()
    x[:, :shared] = x[0, :shared]
    return x


def exact(book, unit, x, lengths, r, listed=None):
    """The layer's attention rows of request r in 64 bits, over all of its keys or (row, head) -> blocks."""
    att, n = book.attention, lengths[r]
    qkv = (x[r][:n] @ unit.weights.qkv.T).unflatten(1, (-1, att.headDim))
    at = torch.arange(n, device="cuda", dtype=torch.int32)
    q = numbers(att.rope(qkv[:, :att.heads], unit.ropeTable, at))
    k = numbers(att.rope(qkv[:, att.heads:att.heads + att.kvHeads], unit.ropeTable, at))
    held = [R.quantized(t)[3] for t in (k, numbers(qkv[:, att.heads + att.kvHeads:]))]
    if listed is None:
        return R.attention(q, held[0], held[1], [list(range(n))], [n], [n], 0, 0, att.headDim ** -0.5)[0]
    return L.attention_listed(q, held[0], held[1], [list(range(n))], [n], [n], listed, att.headDim ** -0.5)[0]


def near(got, want):
    # (a product's rows may be rounded otherwise in a step of other size: see test_gpu_decoder.py)
    assert np.linalg.norm(got - want) <= 2e-2 * np.linalg.norm(want)


@pytest.mark.parametrize("always", [False, True])
def test_requests_that_share_a_prompt(always, monkeypatch):
    from ane_fieldfare_b200 import attention, decoder

    if always:
        plain = attention.AttentionContext.attendShared
        monkeypatch.setattr(attention.AttentionContext, "attendShared", lambda self, *a, **kw: plain(self, *a, **(kw | {"always": True})))
    book, stack = decoder.small_decoder(requests=5, pages=80)
    unit, x = stack[0], inputs(5, 400, 140)
    x[4] = inputs(1, 400, 0, seed=9)[0]
    run(book, unit, x, [[140, 0, 0, 0, 20]])
    assert book.share(0, [1, 2, 3], 140) == 128  # pages of 16
    free = int(book.freeCount)
    steps = [[140, 150, 131, 200, 21], [141, 151, 132, 201, 30], [160, 145, 133, 202, 31], [161, 146, 140, 203, 31]]
    got = run(book, unit, x, steps)
    assert book.attention.info().deviceErrorFlag == 0
    # a page of its own for every sixteen tokens behind the prefix
    assert free - int(book.freeCount) == sum(-(-(n - 128) // 16) for n in (146, 140, 203)) + (-(-161 // 16) - 9) + (-(-31 // 16) - 2)
    for r in range(5):
        want = exact(book, unit, x, steps[-1], r)
        near(np.stack([numbers(got[r, p]) for p in range(steps[-1][r]) if (r, p) in got]), want[[p for p in range(steps[-1][r]) if (r, p) in got]])
    # one ends and its place is taken by a request of its own; then all end
    got = run(book, unit, x, [[161, 147, 0, 204, 31], [161, 148, 40, 205, 31]])
    near(np.stack([numbers(got[2, p]) for p in range(40)]), exact(book, unit, x, [0, 0, 40], 2))
    near(numbers(got[3, 204])[None], exact(book, unit, x, [0, 0, 0, 205], 3)[204:])
    run(book, unit, x, [[161, 0, 0, 0, 0], [0, 0, 0, 0, 0]])
    assert int(book.freeCount) == 80 and sorted(book.freePages.tolist()) == list(range(80))
    assert book.attention.info().deviceErrorFlag == 0


def test_groups_of_the_requests_that_share():
    from ane_fieldfare_b200 import decoder

    book, _ = decoder.small_decoder(requests=9, pages=80)
    book.step([40, 0, 0, 70, 0, 0, 0, 0, 10])
    book.share(0, [1, 2], 40)
    book.share(3, [4, 6, 7], 64)
    step = book.step([40, 33, 34, 70, 65, 1, 66, 67, 10])
    assert step.groupStart.tolist() == [0, 3, 5, 6, 8] and step.prefixLengths.tolist() == [32, 64, 0, 64] and step.maxPrefix == 64
    step = book.step([40, 0, 0, 70, 66, 2, 0, 67, 10])
    assert step.groupStart.tolist() == [3, 5] and step.prefixLengths.tolist() == [64]
    step = book.step([40, 0, 0, 70, 0, 2, 0, 68, 10])
    assert step.groupStart is None
    assert book.attention.info().deviceErrorFlag == 0


def test_a_prefix_is_not_taken_from_those_who_share_it():
    from ane_fieldfare_b200 import decoder

    book, _ = decoder.small_decoder(requests=4, pages=40)
    book.step([40, 0, 10, 0])
    with pytest.raises(ValueError, match="holds 40"):
        book.share(0, [1], 41)
    with pytest.raises(ValueError, match="no tokens"):
        book.share(0, [2], 40)
    with pytest.raises(ValueError, match="no tokens"):
        book.share(0, [0], 40)
    assert book.share(0, [1], 15) == 0 and book.share(0, [], 40) == 0
    assert book.share(0, [1], 40) == 32
    with pytest.raises(ValueError, match="itself"):
        book.share(1, [3], 32)
    with pytest.raises(ValueError, match="request 1 shares its first 32"):
        book.step([40, 31, 10, 0])
    with pytest.raises(ValueError, match="tokens of request 0"):
        book.step([31, 33, 10, 0])
    book.step([32, 33, 10, 0])
    book.step([0, 0, 10, 0])
    assert int(book.freeCount) == 39


def test_requests_that_share_are_named_by_their_numbers():
    """-1 for the last one would be another owner than itself: kept from giving its own pages back once those who shared them had ended."""
    from ane_fieldfare_b200 import decoder

    book, _ = decoder.small_decoder(requests=3, pages=40)
    book.step([0, 0, 40])
    for owner, requests in [(-1, [0]), (2, [-3]), (2, [0, 3]), (3, [0])]:
        with pytest.raises(ValueError, match="0 .. 2"):
            book.share(owner, requests, 40)
    assert book.share(2, [0, 1], 40) == 32
    book.step([33, 34, 41])
    book.step([0, 0, 41])
    book.step([0, 0, 10])
    assert int(book.freeCount) == 39 and book.attention.info().deviceErrorFlag == 0


def test_selected_blocks_of_a_layer():
    """Of a prompt all keys; of the decode steps behind it the blocks that the definition chooses."""
    from ane_fieldfare_b200 import decoder

    choice = decoder.Selection(blocks=3, maxRows=4)
    book, stack = decoder.small_decoder(requests=3, pages=120, selected=choice)
    unit, x = stack[0], inputs(3, 600, 0)
    steps = [[400, 0, 0], [500, 127, 0], [501, 128, 1], [505, 130, 3], [503, 129, 3], [506, 133, 4]]
    got = run(book, unit, x, steps)
    att = book.attention
    assert att.info().deviceErrorFlag == 0
    for r, n in enumerate(steps[-1]):
        dense = exact(book, unit, x, steps[-1], r)
        near(np.stack([numbers(got[r, p]) for p in range(steps[1][r])]), dense[:steps[1][r]]) if steps[1][r] else None
        # the layer's own keys' means, and its queries, through the definition
        qkv = (x[r][:n] @ unit.weights.qkv.T).unflatten(1, (-1, att.headDim))
        at = torch.arange(n, device="cuda", dtype=torch.int32)
        q, k = numbers(att.rope(qkv[:, :att.heads], unit.ropeTable, at)), numbers(att.rope(qkv[:, att.heads:att.heads + att.kvHeads], unit.ropeTable, at))
        held = R.quantized(k)[3]
        means = np.stack([[L.block_mean(held[b * 64:b * 64 + 64, h]) for h in range(att.kvHeads)] for b in range(n // 64)]) if n >= 64 else np.zeros((0, att.kvHeads, att.headDim))
        ids = L.select(q, [means], [n], [n], att.kvHeads, 3, 1, 1)
        rows = [p for p in range(steps[1][r], n)]
        want = exact(book, unit, x, steps[-1], r, ids)
        # (rows whose products were rounded otherwise may choose another block where two score alike: most rows are held to the definition)
        off = [np.linalg.norm(numbers(got[r, p]) - want[p]) <= 5e-2 * np.linalg.norm(want[p]) for p in rows]
        assert sum(off) >= len(rows) - 1


def test_whole_layers_with_both_and_the_demonstration(capsys):
    from ane_fieldfare_b200 import decoder

    book, stack = decoder.small_decoder(requests=4, pages=100, selected=decoder.Selection(blocks=2))
    gen = torch.Generator(device="cuda").manual_seed(4)
    for at, want in enumerate([(200, 0, 0, 33), (200, 200, 201, 34), (201, 205, 203, 35), (202, 192, 204, 0), (0, 0, 0, 0)]):
        if at == 1:
            assert book.share(0, [1, 2], 200) == 192
        hidden = torch.randn((sum(max(0, b - a) for a, b in zip(book.lengths, want)), 256), device="cuda", generator=gen).bfloat16()
        step = book.step(want)
        for layer in stack:
            layer.forward(hidden, step)
        assert torch.isfinite(hidden).all()
    assert int(book.freeCount) == 100 and book.attention.info().deviceErrorFlag == 0 and stack[0].moe.info().deviceErrorFlag == 0
    with pytest.raises(ValueError, match="window"):
        decoder.DecoderLayer(stack[1].moe, book.attention, 1, stack[1].weights, stack[1].ropeTable, 10, window=4, selected=decoder.Selection(blocks=2))
    decoder.main()
    said = capsys.readouterr().out
    assert said.count("error flag: 0") == 2 and "288 tokens" in said


def spied(monkeypatch, unit):
    """(rows, lengths, queries, ids) of every call that selects blocks, each checked against the definition."""
    from ane_fieldfare_b200 import attention

    calls, plain = [], attention.AttentionContext.selectBlocks

    def select(self, q, means, table, start, lengths, blocks, **kw):
        ids = plain(self, q, means, table, start, lengths, blocks, **kw)
        rows, n, held, pages = torch.diff(start).tolist(), lengths.tolist(), numbers(means), table.tolist()
        size = self.pageTokens
        of = [np.stack([held[pages[r][(b * 64 + 63) // size], :, (b * 64 + 63) % size // 64] for b in range(m // 64)]) if m >= 64
              else np.zeros((0, self.kvHeads, self.headDim)) for r, m in enumerate(n)]
        assert np.array_equal(ids.cpu().numpy(), L.select(numbers(q), of, n, rows, self.kvHeads, blocks, kw["first"], kw["last"]))
        calls.append((rows, n, ids.cpu().numpy()))
        return ids

    monkeypatch.setattr(attention.AttentionContext, "selectBlocks", select)
    return calls


def test_a_prompt_in_the_step_leaves_the_other_requests_their_blocks(monkeypatch):
    """Requests with few rows attend to their blocks, requests with many to all keys, in whatever order and whatever else the step has."""
    from ane_fieldfare_b200 import decoder

    book, stack = decoder.small_decoder(requests=5, pages=160, selected=decoder.Selection(blocks=3, maxRows=4))
    unit, x = stack[0], inputs(5, 600, 0)
    calls = spied(monkeypatch, unit)
    steps = [[400, 0, 0, 430, 0], [401, 40, 0, 433, 70], [402, 41, 30, 434, 71], [408, 42, 31, 438, 75], [412, 43, 31, 470, 80]]
    few = [[], [0, 3], [0, 1, 3, 4], [1, 2, 3, 4], [0, 1]]
    run(book, unit, x, [[400, 0, 0, 0, 0], steps[0]])
    assert not calls
    for before, want, chosen in zip(steps, steps[1:], few[1:]):
        calls.clear()
        got = run(book, unit, x, [want])
        rows = [b - a for a, b in zip(before, want)]
        (ran, lengths, ids), = calls
        assert ran == [rows[r] for r in chosen] and lengths == [want[r] for r in chosen]
        at = 0
        for r, n in enumerate(want):
            if not rows[r]:
                continue
            listed = None
            if r in chosen:
                listed = np.full((n, *ids.shape[1:]), -1)
                listed[n - rows[r]:] = ids[at:at + rows[r]]
                at += rows[r]
            near(np.stack([numbers(got[r, p]) for p in range(n - rows[r], n)]), exact(book, unit, x, want, r, listed)[n - rows[r]:])
    assert book.attention.info().deviceErrorFlag == 0
    # a bound that has to be the same for several steps decides for all requests
    calls.clear()
    step = book.step([413, 44, 31, 471, 80], maxRows=16)
    unit.attend(torch.stack([x[0][412], x[1][43], x[3][470]]), step)
    assert not calls
    unit.attend(torch.stack([x[0][413], x[1][44], x[3][471]]), book.step([414, 45, 31, 472, 80], maxRows=4))
    assert len(calls) == 1


@pytest.mark.parametrize("always", [False, True])
def test_prompts_behind_a_shared_prefix_beside_single_tokens(always, monkeypatch):
    from ane_fieldfare_b200 import attention, decoder

    plain, shared = attention.AttentionContext.attendShared, []

    def attend(self, q, pages, table, start, lengths, most, groups, prefixes, **kw):
        shared.append((groups.tolist(), prefixes.tolist(), lengths.tolist()))
        return plain(self, q, pages, table, start, lengths, most, groups, prefixes, **(kw | {"always": always}))

    monkeypatch.setattr(attention.AttentionContext, "attendShared", attend)
    book, stack = decoder.small_decoder(requests=8, pages=200, selected=decoder.Selection(blocks=2, maxRows=4))
    unit, x = stack[0], inputs(8, 400, 140)
    x[5:] = inputs(3, 400, 80, seed=9)
    calls = spied(monkeypatch, unit)
    run(book, unit, x, [[140, 0, 0, 0, 30, 90, 0, 0]])
    assert book.share(0, [1, 2, 3], 140) == 128 and book.share(5, [6, 7], 80) == 80
    #                 single, few, many, many, single, many, few, many
    steps = [[141, 130, 160, 150, 31, 120, 82, 110], [142, 150, 161, 170, 40, 121, 83, 111], [143, 151, 181, 171, 41, 122, 84, 112]]
    got = run(book, unit, x, steps)
    assert shared == [([0, 2, 4], [128, 80], [160, 150, 120, 110]), ([0, 2, 3], [128, 0], [150, 170, 40])]
    assert [c[0] for c in calls] == [[1, 2, 1, 2], [1, 1, 1, 1, 1], [1, 1, 1, 1, 1, 1, 1]]
    for r, p0, p1 in [(2, 128, 160), (3, 128, 150), (5, 90, 120), (7, 80, 110), (1, 130, 150), (3, 150, 170), (4, 31, 40), (2, 161, 181)]:
        near(np.stack([numbers(got[r, p]) for p in range(p0, p1)]), exact(book, unit, x, steps[-1], r)[p0:p1])
    assert book.attention.info().deviceErrorFlag == 0


def test_a_mixed_step_is_captured_at_first_sight():
    from ane_fieldfare_b200 import decoder

    book, stack = decoder.small_decoder(requests=6, pages=160, selected=decoder.Selection(blocks=20, maxRows=4))
    unit, x = stack[0], inputs(6, 300, 64)
    run(book, unit, x, [[200, 0, 0, 100, 0, 0]])
    assert book.share(0, [1, 2], 64) == 64
    have, want = list(book.lengths), [201, 104, 100, 140, 3, 0]  # blocks enough for all keys: whatever the split, every row sees all
    step = book.step(want)
    rows = torch.stack([x[r][p] for r in range(6) for p in range(have[r], want[r])])
    torch.cuda.synchronize()
    graph, out = torch.cuda.CUDAGraph(), None
    with torch.cuda.graph(graph):
        out = unit.attend(rows, step)
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    captured = out.clone()
    assert torch.equal(unit.attend(rows, step), captured) and torch.equal(unit.attend(rows, step), captured)
    graph.replay()
    assert torch.equal(out, captured)
    at = 0
    for r in range(6):
        n = want[r] - have[r]
        if n:
            near(numbers(captured[at:at + n]), exact(book, unit, x, want, r)[have[r]:])
        at += n
    assert book.attention.info().deviceErrorFlag == 0
