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
