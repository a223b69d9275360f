"""Beam search at the edges of its arguments' ranges, against the definition in 64 bits (np_beam.py)."""
import math

import numpy as np
import pytest

from tests import np_beam as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def s(lib):
    from born_b200 import Sampler
    with Sampler(device=0, max_batch=512, max_vocab=262144) as h:
        yield h


def test_beams_that_go_on_are_normalised_as_the_pool(s):
    """score / length^length_penalty in 64 bits, rounded once: equal scores are equal wherever they come from."""
    import torch
    from born_b200 import BeamConfig, BeamSearch
    N, K, V = 32, 16, 300
    z = torch.randn((N * K, V), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    for penalty in (1.0, 0.7):
        search = BeamSearch(s, N, K, 3, V, BeamConfig(length_penalty=penalty))
        search.begin()
        for _ in range(3):
            search.step(z)
        got = search.result()["scores"].cpu().numpy()
        norm = np.float64(3) ** np.float64(np.float32(penalty))
        want = (search.scores.cpu().numpy().astype(np.float64) / norm).astype(np.float32).reshape(N, K)
        assert np.array_equal(got, -np.sort(-want, axis=1))


def test_length_penalties_beyond_all_numbers(s):
    """length^length_penalty is infinite: every score is (negative) zero, the beams keep their order."""
    import torch
    from born_b200 import BeamConfig, BeamSearch
    N, K, V = 2, 4, 100
    search = BeamSearch(s, N, K, 4, V, BeamConfig(length_penalty=600.0))
    search.begin()
    for t in range(4):
        search.step(torch.randn((N * K, V), device="cuda"))
    found = search.result()
    assert (found["scores"] == 0).all() and (found["lens"] == 4).all()
    assert torch.equal(found["tokens"][:, :, 3], search.tokens.view(N, K))


def dev(x, dtype=None):
    import torch
    t = torch.from_numpy(np.ascontiguousarray(x)).cuda()
    return t.to(torch.bfloat16) if dtype == "bf16" else t


def bits_of(allowed):
    r, v = allowed.shape
    pad = np.zeros((r, (v + 31) // 32 * 32), bool)
    pad[:, :v] = allowed
    return np.packbits(pad, axis=1, bitorder="little").view(np.uint32).view(np.int32).copy()


def normaliser_error(score):
    """A normaliser is off by at most 11 * 2^-24: an exponential by ex2's 2^-22, 2^-25 of its exponent's fraction and a little
    for that fraction's second part (half of 2^-24 allows for it and for the 64-bit remainder), a sum of 32 of them by six rounded
    additions.  The reported score is rounded once."""
    return 11 * 2.0 ** -24 + np.abs(score) * 2.0 ** -24


def check(out, rows, scores, K, T=0.0):
    """Tokens, parents and statuses as the definition has them, scores within normaliser_error.  rows: fp32 logits, -inf where masked."""
    got = {k: v.cpu().numpy() for k, v in out.items()}
    for n in range(len(rows) // K):
        sl = slice(n * K, (n + 1) * K)
        want = R.step([r.astype(np.float32) for r in rows[sl]], scores[sl], (), T)
        for k in ("status", "token", "parent"):
            assert got[k][sl].tolist() == want[k], (k, n, got[k][sl], want[k])
        a, b = got["score"][sl].astype(np.float64), np.array(want["score"], dtype=np.float64)
        assert (np.isinf(a) == np.isinf(b)).all()
        f = np.isfinite(b)
        assert (np.abs(a[f] - b[f]) <= normaliser_error(b[f])).all(), (n, (a - b)[f] * 2.0 ** 24)


@pytest.mark.parametrize("T", [1e30, 2e30, 4e36, 6e36, 2e37, 1e38, 3.4e38])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("masked", ["mask", "-inf", "history"])
def test_large_temperatures(s, T, dtype, masked):
    """Every finite temperature counts a token that is masked or at -inf for nothing, however near the others' weights are."""
    import torch
    from born_b200 import BeamConfig
    rng = np.random.default_rng(int(math.log2(T)))
    N, K, V = 4, 3, 1500
    z = (rng.standard_normal((N * K, V)) * np.float32(3e37)).astype(np.float32)
    if masked != "history":
        z[::2] = 2.0  # (all weights alike, all tokens equal: z/T of unequal ones would be lost in 64 bits beside the score)
    if dtype == "bf16":
        z = torch.from_numpy(z).to(torch.bfloat16).float().numpy()
    allowed = rng.random((N * K, V)) < 0.4
    rows = np.where(allowed, z, np.float32(-np.inf))
    scores = (-20 - 3 * rng.random(N * K)).astype(np.float32)
    kw, cfg = {}, BeamConfig(temperature=T)
    if masked == "-inf":
        z = rows
    else:
        kw["mask"] = dev(bits_of(allowed))
    if masked == "history":
        pen = dict(presence=2.0)
        history = rng.integers(0, V, (N * K, 40)).astype(np.int32)
        rows = np.stack([np.where(allowed[b], R.penalised(z[b], history[b], **pen), np.float32(-np.inf)) for b in range(N * K)])
        kw["history"], cfg.presence_penalty = dev(history), 2.0
    out = s.beam_step(dev(z, dtype), dev(scores), K, config=cfg, **kw)
    check(out, rows, scores, K, T)


def test_a_wait_that_runs_out(s, lib):
    """A copy that never comes fails the rows that its CTA had in hand (the hook checks which, and the other groups' tokens) and leaves
    nothing behind: neither tickets nor an error for the next step."""
    from born_b200 import _lib as L
    for _ in range(2):
        rc = lib.born_debug_expire_wait(s._h, None)
        assert rc == L.ERR_DEVICE_TIMEOUT, (rc, lib.born_last_error(s._h))
    for N, K, V in ((3, 5, 1000), (1, 4, 32000), (40, 4, 9000)):
        rng = np.random.default_rng(V)
        z = (rng.standard_normal((N * K, V)) * 2).astype(np.float32)
        scores = (-20 - 3 * rng.random(N * K)).astype(np.float32)
        check(s.beam_step(dev(z), dev(scores), K), z, scores, K)
    s.check_error()


def lone_scores(s, z, T=0.0, **kw):
    """Every row a group of one beam at score 0: (reported score, the definition's in 64 bits); -inf logits weigh nothing."""
    import torch
    from born_b200 import BeamConfig
    cfg = BeamConfig(temperature=T, presence_penalty=kw.pop("presence", 0.0))
    rows = kw.pop("rows", z).double()
    out = s.beam_step(z, torch.zeros(z.shape[0], device="cuda"), 1, config=cfg, **kw)
    assert (out["status"] == 0).all()
    x = (rows - rows.max(1, keepdim=True).values) / float(np.float32(T or 1.0))
    return out["score"].cpu().numpy().astype(np.float64), -torch.log(torch.exp(x).sum(1)).cpu().numpy()


def near(got, want):
    return (np.abs(got - want) <= normaliser_error(want)).all(), float((np.abs(got - want) * 2.0 ** 24).max())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("T", [0.0, 0.37, 1.7, 30.0])
@pytest.mark.parametrize("V", [1000, 4096, 50001])
def test_normalisers_of_equal_logits(s, V, T, dtype):
    """All terms of a row are the same number: whatever its exponential is off by, and its sums' roundings, go one way."""
    import torch
    z = (torch.rand((512, 1), generator=torch.Generator(device="cuda").manual_seed(V), device="cuda") * 60 - 30).expand(512, V)
    z = z.to(torch.bfloat16 if dtype == "bf16" else torch.float32).contiguous()
    ok, worst = near(*lone_scores(s, z, T))
    assert ok, worst


@pytest.mark.parametrize("border", [72.6817, -72.6817, 70.0, 5000.0])
@pytest.mark.parametrize("V", [1000, 20000])
def test_normalisers_at_the_largest_exponents(s, V, border):
    """|z/T| log2 e just below and above 2^20 (72.68 at T = 1e-4), where the logits begin to be taken relative to the maximum; tokens
    lie a few steps of fp32 apart, so that all of them weigh."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(V)
    step = 2.0 ** (math.floor(math.log2(abs(border))) - 23)
    near_it = border + (torch.randint(-40, 41, (512, 1), generator=g, device="cuda") * 2.0 ** 5 * step)
    z = (near_it.double() - torch.randint(0, 8, (512, V), generator=g, device="cuda") * step).float()
    ok, worst = near(*lone_scores(s, z, 1e-4))
    assert ok, worst


def test_normalisers_of_histories(s):
    """All of a row's mass comes from tokens of the history, and they come in any order."""
    import torch
    V = 700
    g = torch.Generator(device="cuda").manual_seed(9)
    z = torch.randn((512, V), generator=g, device="cuda")
    history = torch.stack([torch.randperm(V, generator=g, device="cuda") for _ in range(512)]).to(torch.int32)
    ok, worst = near(*lone_scores(s, z, 0.0, presence=1.5, history=history, rows=z - 1.5))
    assert ok, worst


@pytest.mark.parametrize("V", [128256, 262144])
def test_normalisers_of_long_rows(s, V):
    import torch
    z = torch.randn((200, V), generator=torch.Generator(device="cuda").manual_seed(V), device="cuda")
    z[:100] = z[:100].abs() * -0.01  # many terms near the largest
    ok, worst = near(*lone_scores(s, z))
    assert ok, worst


def test_the_states_of_a_single_beam(s):
    """One group of one beam: nothing moves, whatever the layout; pieces that overlap are still refused."""
    import torch
    from born_b200 import BeamSearch, InvalidArgument
    p = torch.zeros(1, dtype=torch.int32, device="cuda")
    lens = torch.tensor([3], dtype=torch.int32, device="cuda")
    for shape, dim in (((1, 2, 5, 8), 2), ((1, 5, 2, 8), 1), ((1, 3, 2, 5, 4), 3), ((1, 7), None), ((1,), None)):
        x = torch.randn(shape, device="cuda")
        y = x.clone()
        s.beam_reorder([x], p, 1, lens=None if dim is None else lens, position_dim=dim)
        assert torch.equal(x, y)
    call = s.prepare_beam_reorder([torch.randn((1, 2, 5, 8), device="cuda")], p, 1, position_dim=2)
    call.args.plane_stride -= 4
    with pytest.raises(InvalidArgument):
        call.run()
    cache = torch.randn((1, 2, 5, 8), device="cuda")
    search = BeamSearch(s, 1, 1, 5, 100)
    search.begin()
    search.step(torch.randn((1, 100), device="cuda"), states=[cache], lens=lens, position_dim=2)
    assert search.tokens.item() >= 0


def test_strides_whose_multiples_are_beyond_64_bits(s):
    """Rows and pieces overlap, however the product of a stride and a number of them wraps round."""
    import torch
    from born_b200 import InvalidArgument
    p = torch.zeros(8, dtype=torch.int32, device="cuda")
    for rows, planes in ((2 ** 61, 2 ** 61), (2 ** 62, 2 ** 61), (2 ** 61, 2 ** 62), (2 ** 61 + 8, 2 ** 62 + 8), (2 ** 62, 2 ** 62 - 64)):
        call = s.prepare_beam_reorder([torch.zeros((8, 8, 5, 8), device="cuda")], p, 4, position_dim=2)
        call.args.row_stride, call.args.plane_stride = rows, planes
        with pytest.raises(InvalidArgument):
            call.run()


@pytest.mark.parametrize("N,K,V", [(1, 1, 2_000_001), (1, 4, 1_000_000), (1, 16, 700_001), (2, 3, 600_000)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("kind", ["random", "sorted", "history"])
def test_rows_of_more_records_than_a_warp_holds(lib, N, K, V, dtype, kind):
    """A long row is shared by more CTAs than a warp has lanes: the merge goes over their records in several turns."""
    import torch
    from born_b200 import BeamConfig, Sampler
    rng = np.random.default_rng(V + K)
    z = (rng.standard_normal((N * K, V)) * 2).astype(np.float32)
    if kind == "sorted":
        z.sort(axis=1)  # (the best tokens lie together)
    if dtype == "bf16":
        z = torch.from_numpy(z).to(torch.bfloat16).float().numpy()
    scores = (-20 - 3 * rng.random(N * K)).astype(np.float32)
    kw, rows = {}, z
    if kind == "history":
        history = np.argsort(-z, axis=1)[:, :50].astype(np.int32)
        kw, rows = dict(history=dev(history)), np.stack([R.penalised(z[b], history[b], presence=1.5) for b in range(N * K)])
    with Sampler(device=0, max_batch=N * K, max_vocab=V) as s:
        out = s.beam_step(dev(z, dtype), dev(scores), K, config=BeamConfig(presence_penalty=1.5 if kw else 0.0), **kw)
        check(out, rows, scores, K)
        s.check_error()


def test_groups_that_are_done_at_large_temperatures(s):
    import torch
    from born_b200 import BeamConfig, _lib as L
    N, K, V = 3, 4, 900
    rng = np.random.default_rng(8)
    z = (rng.standard_normal((N * K, V)) * np.float32(3e37)).astype(np.float32)
    scores = (-20 - 3 * rng.random(N * K)).astype(np.float32)
    pool = s.beam_pool(N, K)
    pool.done[1] = 1
    out = s.beam_step(dev(z), dev(scores), K, config=BeamConfig(temperature=1e38), pool=pool)
    assert (out["status"][K:2 * K] == L.ROW_FINISHED).all() and (out["token"][K:2 * K] == -1).all()
    keep = [r for r in range(N * K) if not K <= r < 2 * K]
    check({k: v[torch.tensor(keep, device="cuda")] for k, v in out.items()}, z[keep], scores[keep], K, 1e38)


@pytest.mark.parametrize("T", [1e18, 1e28, 1e34])
def test_values_that_64_bits_do_not_tell_apart(s, T):
    """z/T is lost beside the score: all tokens of a row have one value.  The candidates are the row's best by their logits all the same,
    in the order of their indices."""
    from born_b200 import BeamConfig
    N, K, V = 3, 5, 2000
    rng = np.random.default_rng(4)
    z = rng.permuted(np.tile(np.arange(V, dtype=np.float32) * 0.01 - 5, (N * K, 1)), axis=1)
    scores = np.tile(np.float32([-7, -3, -9, -4, -5]), N)  # (of each group the second beam's are ahead of all others')
    out = {k: v.cpu().numpy() for k, v in s.beam_step(dev(z), dev(scores), K, config=BeamConfig(temperature=T)).items()}
    for n in range(N):
        assert out["token"][n * K:(n + 1) * K].tolist() == sorted(np.argsort(-z[n * K + 1])[:K].tolist())
        assert (out["parent"][n * K:(n + 1) * K] == 1).all()
