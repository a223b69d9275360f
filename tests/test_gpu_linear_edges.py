"""The output head where its parts meet: launches on one another's heels."""
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


def test_gelu_far_below_zero(s):
    """0.5 y erfc(-y/sqrt 2) to a relative bound: 1/sqrt 2 and its product with y are rounded (2 * 2^-24), which erfc enlarges by
    y^2 + 1 at most (t erfc'(t)/erfc(t) <= 2t^2 + 1), erfcf is within 4 ulp (8 * 2^-24), the product and the result round once each;
    below 2^-126 the same ulps are 2^-149."""
    import torch
    V = 30000
    y = torch.linspace(-14.0, 14.0, V, device="cuda")
    x, w = torch.zeros((2, 64), dtype=torch.bfloat16, device="cuda"), torch.zeros((V, 64), dtype=torch.bfloat16, device="cuda")
    got = s.linear(x, w, bias=y, activation="gelu").double()
    d = y.double()
    want = 0.5 * d * torch.special.erfc(-d / 2 ** 0.5)
    most = want.abs() * 2.0 ** -24 * (2 * (d * d + 1) + 10) + (4 * d.abs() + 2) * 2.0 ** -149
    assert ((got - want).abs() <= most).all()
    low = s.linear(x, w, bias=y, activation="gelu", out_dtype=torch.bfloat16).double()
    assert ((low - want).abs() <= most + want.abs() * 2.0 ** -8 + 2.0 ** -134).all()


def test_gelu_of_what_is_no_number(s):
    import torch
    y = torch.tensor([float("inf"), float("nan"), float("-inf"), 0.0, 1e30, -1e30, 3e38, -3e38, -30.0, 30.0], device="cuda")
    x, w = torch.zeros((1, 64), dtype=torch.bfloat16, device="cuda"), torch.zeros((len(y), 64), dtype=torch.bfloat16, device="cuda")
    got = s.linear(x, w, bias=y, activation="gelu")[0].tolist()
    assert got[0] == float("inf") and got[1] != got[1] and got[2] != got[2]  # (the formula's -inf * 0)
    f32 = torch.tensor([0.0, 1e30, 0.0, 3e38, 0.0, 0.0, 30.0], device="cuda").tolist()
    assert got[3:] == f32


def test_more_rows_than_a_tiles_width_may_be_added_to(s):
    """2.14e9 rows of 8, one feature: as many as an int holds beside the tiles' number."""
    import torch
    M = 2_140_000_000
    x = torch.zeros((M, 8), dtype=torch.bfloat16, device="cuda")
    x[-3:] = whole((3, 8), 1)
    x[123_456_789] = 1
    w = whole((1, 8), 2, 1, 4)
    out = s.linear(x, w)
    assert torch.equal(out[-3:], (x[-3:].double() @ w.double().t()).float())
    assert out[123_456_789].item() == w.double().sum().item()
    assert sum(int((part != 0).sum()) for part in out.split(1 << 28)) <= 4
    s.check_error()


@pytest.mark.parametrize("M,K,V", [(1, 4096, 2000), (64, 8192, 1000), (200, 4096, 3000), (256, 8192, 2000)])
def test_sums_of_512_products(s, M, K, V):
    """Cut off 32 times at most, before registers add the next ones, rounded.  A partial sum of j steps of 16 has the root mean square
    sqrt(j/32) of the 512's and is cut off by less than 2^-23 of itself: sum_j sqrt(j/32) 2^-23 = 21.8 * 2^-23 of the result if all go
    one way.  The additions round by half of 2^-23 of their partial sums.  (One sum over 4096 products was off by 4.3e-6 = 36 * 2^-23.)"""
    import torch
    g = torch.Generator(device="cuda").manual_seed(K + M)
    x = torch.randn((M, K), generator=g, device="cuda").to(torch.bfloat16)
    w = torch.randn((V, K), generator=g, device="cuda").to(torch.bfloat16)
    want = x.double() @ w.double().t()
    rms = lambda v: float(v.square().mean().sqrt())  # noqa: E731
    chunks = K // 512
    most = sum((j / 32) ** 0.5 for j in range(1, 33)) + 0.5 * sum((i / chunks) ** 0.5 for i in range(1, chunks + 1))
    assert rms(s.linear(x, w).double() - want) <= most * 2.0 ** -23 * rms(want)
