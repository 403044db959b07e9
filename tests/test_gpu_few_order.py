"""The few-token layer's hand-overs inside a kernel: hidden activations from the CTAs that made them to those that read them,
scales from the lanes that asked for them to the whole warp, finished items through a ring of 64 places."""
import pytest

from test_gpu_few_tokens import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("weights", ["16", "8", "4"])
def test_many_calls_give_the_same_bits(weights):
    """Scales that differ from step to step and experts whose hidden activations come from many CTAs: what is read too early is
    another number."""
    import torch
    c = Case(12, 40, 4, 1024, 1024, 2, weights, std=0.03, seed=3)
    if weights == "8":
        g = torch.Generator(device="cuda")
        g.manual_seed(1)
        for m in c.s:
            c.s[m] *= torch.exp2(torch.randint(-6, 7, c.s[m].shape, device="cuda", generator=g).float())
    want = c.run()
    c.check(want)
    for _ in range(100):
        got = c.run()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("weights,n", [("16", 40), ("8", 40), ("16", 6)])
def test_more_finished_items_than_wait_to_be_counted(weights, n):
    """64 experts (n = 6: some 40 of them) of 4096 / 16 blocks of rows: over a hundred (70) up items per CTA, each a step or two long,
    go through the 64 places between the warp that adds and the warp that counts. A place that were written again before it
    was counted would start one expert's down projection early and another's never."""
    import torch
    c = Case(n, 64, 8, 128, 4096, 2, weights, std=0.05, seed=n)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = c.run(dev_status=status)
    assert int(status) == 0
    c.check(got)
    for _ in range(10):
        assert all(torch.equal(a, b) for a, b in zip(c.run(), got))
