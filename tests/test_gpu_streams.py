"""Results that a call allocates for a stream are that stream's memory, not what the current one may still be using."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_outputs_are_memory_of_the_stream_that_writes_them():
    from ane_fieldfare_b200 import hotpath, workload

    layer = workload.make_layer(3, 0, experts=16, d=256, f=128, sharedF=192, topK=8, router_bias="normal")
    ctx = hotpath.HotpathContext(layers=1, experts=16, d=256, f=128, sharedF=192, topK=8, maxTokens=512)
    workload.load_layer(ctx, 0, layer)
    x = torch.randn((512, 256), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).bfloat16()
    groups = torch.randint(0, 16, (512, 8), device="cuda", dtype=torch.int32)
    torch.cuda.synchronize()
    want = [ctx.moeLayer(0, x), ctx.moeStack(0, 1, x), ctx.rmsnorm(x, None, 1e-6)]
    pairs = hotpath.PrefillGroupedRoutedMoE(ctx).sortRoutesOnDevice(None, groups, 16)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    calls = [(lambda: [ctx.moeLayer(0, x, stream=side)], want[:1]), (lambda: [ctx.moeStack(0, 1, x, stream=side)], want[1:2]),
             (lambda: [ctx.rmsnorm(x, None, 1e-6, stream=side)], want[2:]),
             (lambda: hotpath.PrefillGroupedRoutedMoE(ctx).sortRoutesOnDevice(side, groups, 16), pairs)]
    for run, expected in calls:
        used = [torch.empty_like(t) for t in expected for _ in range(3)]
        held = {t.data_ptr() for t in used}
        del used
        out = run()
        torch.cuda.synchronize()
        assert not held & {t.data_ptr() for t in out}
        assert all(torch.equal(a, b) for a, b in zip(out, expected))
