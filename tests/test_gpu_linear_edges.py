"""The output head where its parts meet: launches on one another's heels."""
import numpy as np  # noqa: F401
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def s(lib):
    from born_b200 import Sampler
    with Sampler(device=0, max_batch=64, max_vocab=65536) as h:
        yield h


def whole(shape, seed, lo=-2, hi=3):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(lo, hi, shape, generator=g, device="cuda").to(torch.bfloat16)


# (pairs of one, two and many slices, with K in one part and in several, and lone CTAs between them)
@pytest.mark.parametrize("shapes", [[(100, 64, 300), (65, 128, 257)], [(128, 2048, 2000), (100, 64, 300), (3, 72, 500)],
                                    [(256, 264, 900), (255, 520, 700), (200, 2048, 1000)], [(65, 136, 18945), (128, 2048, 2000)]])
def test_launches_that_overlap(s, shapes):
    """A launch begins while the one before it ends: whatever is on its way into a CTA has to arrive before that CTA ends, or it
    arrives at the next one's barriers."""
    import torch
    calls = []
    for i, (M, K, V) in enumerate(shapes):
        x, w = whole((M, K), i), whole((V, K), 10 + i)
        calls.append((s.prepare_linear(x, w), (x.double() @ w.double().t()).float()))
    torch.cuda.synchronize()
    wrong = torch.zeros((), dtype=torch.int64, device="cuda")
    for turn in range(60):
        for call, _ in calls:
            call.out.fill_(-1.0)
        for _ in range(4):
            for call, _ in calls:
                call.run()
        for call, want in calls:
            wrong += (call.out != want).sum()
    s.check_error()
    assert int(wrong) == 0
