"""A decoder layer put together from the operators: its attention against the statement in 64 bits, whatever the steps in which a
request's rows arrive; its MoE half against the operators called one by one elsewhere (tests/test_gpu_stack.py)."""
import numpy as np
import pytest
import torch

import attention_reference as R

pytestmark = pytest.mark.gpu


def numbers(t):
    return t.detach().float().cpu().numpy().astype(np.float64)


@pytest.mark.parametrize("steps", [[(50, 20)], [(30, 1), (40, 17), (41, 18), (50, 20)], [(20, 5), (28, 9), (23, 9), (24, 10), (50, 20)]])
@pytest.mark.parametrize("layer", [0, 1])
def test_attention_of_a_layer_does_not_depend_on_the_steps(steps, layer):
    """Rows of two requests in one step, in several, and with rows taken back on the way."""
    from ane_fieldfare_b200 import decoder

    book, stack = decoder.small_decoder()
    att, unit = book.attention, stack[layer]
    x = torch.randn((2, 50, 256), generator=torch.Generator(device="cuda").manual_seed(3), device="cuda").bfloat16()
    got = torch.zeros((2, 50, att.heads, att.headDim), dtype=torch.bfloat16, device="cuda")
    have = [0, 0]
    for want in steps:
        spans = [(r, a, b) for r, (a, b) in enumerate(zip(have, want)) if b > a]
        step = book.step(want)
        if spans:
            out = unit.attend(torch.cat([x[r, a:b] for r, a, b in spans]), step)
            at = 0
            for r, a, b in spans:
                got[r, a:b] = out[at:at + b - a]
                at += b - a
        have = list(want)
    torch.cuda.synchronize()
    assert att.info().deviceErrorFlag == 0
    # the same rows in one go, from their products on
    for r, n in enumerate(have):
        qkv = (x[r, :n] @ unit.weights.qkv.T).unflatten(1, (-1, att.headDim))
        at = torch.arange(n, device="cuda", dtype=torch.int32)
        q = numbers(att.rope(qkv[:, :att.heads], unit.ropeTable, at))
        k = numbers(att.rope(qkv[:, att.heads:att.heads + att.kvHeads], unit.ropeTable, at))
        held = [R.quantized(t)[3] for t in (k, numbers(qkv[:, att.heads + att.kvHeads:]))]
        want, bound = R.attention(q, held[0], held[1], [list(range(n))], [n], [n], unit.window, unit.sinks, att.headDim ** -0.5)
        off = np.abs(numbers(got[r, :n]) - want)
        # a product's rows may be rounded otherwise in a step of other size: a bf16 step here and there in q, k and v, which moves
        # a code by one; what that is worth is bounded for the rows as a whole
        assert np.linalg.norm(off) <= 2e-2 * np.linalg.norm(want)


def test_steps_through_whole_layers():
    from ane_fieldfare_b200 import decoder

    book, stack = decoder.small_decoder()
    have, outputs = [0, 0], []
    gen = torch.Generator(device="cuda").manual_seed(4)
    for want in [(70, 33), (78, 41), (73, 36), (74, 37), (75, 0)]:
        rows = sum(max(0, b - a) for a, b in zip(have, want))
        hidden = torch.randn((rows, 256), device="cuda", generator=gen).bfloat16()
        before, step = hidden.clone(), book.step(want)
        for layer in stack:
            layer.forward(hidden, step)
        assert torch.isfinite(hidden).all() and (rows == 0 or not torch.equal(hidden, before))
        assert int(book.freeCount) == 64 - sum(-(-n // 16) for n in want)
        outputs.append(hidden)
        have = want
    assert stack[0].moe.info().deviceErrorFlag == 0 and book.attention.info().deviceErrorFlag == 0


def test_the_demonstration_runs(capsys):
    from ane_fieldfare_b200 import decoder

    decoder.main()
    assert "error flag: 0" in capsys.readouterr().out
