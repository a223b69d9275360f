"""Beam search on the GPU against its definition in 64 bits (np_beam.py).

Tokens, parents and statuses are equal.  A reported score is the definition's rounded once to fp32
(2^-24 of its size), from a normaliser that is off by at most half of what the host allows two rows
together before it recomputes them in 64 bits: 3 roundings of 2^-24 of an exponent that weighs at most
log2(V) + 8, 8 * 2^-24 for the exponentials and one rounding per turn of a thread (V / 4096 + 12 of them at
most) -- score_error below.
"""
import math

import numpy as np
import pytest

from tests import np_beam as R

pytestmark = pytest.mark.gpu


def score_error(V):
    u = 2.0 ** -24
    return 3 * u * (math.log2(V) + 8) * math.log(2) + 8 * u + (V / 4096 + 12) * u


@pytest.fixture(scope="module")
def s(lib):
    from born_b200 import Sampler
    with Sampler(device=0, max_batch=512, max_vocab=262144) as h:
        yield h


def bits_of(allowed):
    """[R, V] bool -> [R, ceil(V/32)] uint32 as int32."""
    r, v = allowed.shape
    pad = np.zeros((r, (v + 31) // 32 * 32), bool)
    pad[:, :v] = allowed
    return np.packbits(pad, axis=1, bitorder="little").view(np.uint32).view(np.int32).copy()


def to_bf16(z):
    import torch
    return torch.from_numpy(z).to(torch.bfloat16).float().numpy()


def check(out, z, scores, K, stops=(), temperature=0.0, keep=False, allowed=None, history=None, lens=None, pen=None):
    """Holds a step's outputs against the definition, group by group."""
    V, N = z.shape[1], z.shape[0] // K
    got = {k: v.cpu().numpy() for k, v in out.items()}
    for n in range(N):
        rows = []
        for b in range(n * K, (n + 1) * K):
            r = z[b].astype(np.float32)
            if history is not None:
                ids = history[b][:len(history[b]) if lens is None else max(0, min(len(history[b]), lens[b]))]
                r = R.penalised(r, ids, **pen)
            if allowed is not None:
                r = np.where(allowed[b], r, np.float32(-np.inf))
            rows.append(r)
        want = R.step(rows, scores[n * K:(n + 1) * K], stops, temperature, keep)
        sl = slice(n * K, (n + 1) * K)
        for k in ("status", "token", "parent"):
            assert got[k][sl].tolist() == want[k], (k, n, got[k][sl], want[k])
        pairs = [(got["score"][sl], want["score"])]
        if "end_token" in got:
            assert got["end_token"][n].tolist() == want["end_token"], n
            assert got["end_parent"][n].tolist() == want["end_parent"], n
            pairs.append((got["end_score"][n], want["end_score"]))
        for a, b in pairs:
            b = np.array(b)
            assert (np.isinf(a) == np.isinf(b)).all()
            f = np.isfinite(b)
            assert (np.abs(a[f] - b[f]) <= score_error(V) + np.abs(b[f]) * 2.0 ** -24).all(), (a, b)


def inputs(seed, N, K, V, dtype="f32"):
    rng = np.random.default_rng(seed)
    z = (rng.standard_normal((N * K, V)) * 2).astype(np.float32)
    if dtype == "bf16":
        z = to_bf16(z)
    scores = (-20 - 3 * rng.random(N * K)).astype(np.float32)
    return rng, z, scores


def dev(x, dtype=None):
    import torch
    t = torch.from_numpy(np.ascontiguousarray(x)).cuda()
    return t.to(torch.bfloat16) if dtype == "bf16" else t


@pytest.mark.parametrize("N,K,V", [(1, 1, 1), (1, 4, 2), (2, 16, 7), (1, 3, 33), (3, 5, 1000), (1, 4, 32000), (5, 4, 8191),
                                   (9, 7, 50257), (64, 4, 4096), (2, 16, 128256), (1, 1, 262144), (100, 2, 1024), (512, 1, 515)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_shapes(s, N, K, V, dtype):
    from born_b200 import BeamConfig
    _, z, scores = inputs(N * 31 + K * 7 + V, N, K, V, dtype)
    stops = (V // 2, 0) if V > 1 else ()
    out = s.beam_step(dev(z, dtype), dev(scores), K, config=BeamConfig(stop_tokens=stops))
    check(out, z, scores, K, stops)


@pytest.mark.parametrize("seed", range(12))
def test_everything_at_once(s, seed):
    from born_b200 import BeamConfig
    rng = np.random.default_rng(1000 + seed)
    K, N, V = int(rng.integers(1, 17)), int(rng.integers(1, 9)), int(rng.integers(60, 40000))
    dtype = ["f32", "bf16"][seed % 2]
    _, z, scores = inputs(seed, N, K, V, dtype)
    scores[rng.random(N * K) < 0.2] = -np.inf
    stops = tuple(int(t) for t in rng.integers(0, V, int(rng.integers(0, 9))))
    for t in stops:
        z[:, t] = 6.0 + (rng.random(N * K) < 0.5) * 4.0
    if dtype == "bf16":
        z = to_bf16(z)
    allowed = (rng.random((N * K, V)) < [0.05, 0.5, 1.0][seed % 3]) if seed % 4 else None
    H = int(rng.integers(1, 1025))
    history = rng.integers(-3, V + 3, (N * K, H)).astype(np.int32)
    history[:, ::3] = np.argsort(-z, axis=1)[:, :1]  # the likeliest token many times
    if stops:
        history[:, 1::7] = stops[0]
    lens = rng.integers(0, H + 4, N * K).astype(np.int32)
    pen = dict(repetition=1.3) if seed % 3 == 0 else dict(frequency=0.25, presence=0.5) if seed % 3 == 1 else dict(repetition=0.7, frequency=-0.1)
    T = [0.0, 0.6, 1.7][seed % 3]
    keep = bool(seed % 2)
    cfg = BeamConfig(temperature=T, repetition_penalty=pen.get("repetition", 0.0), frequency_penalty=pen.get("frequency", 0.0),
                     presence_penalty=pen.get("presence", 0.0), stop_tokens=stops, keep_slots=keep)
    out = s.beam_step(dev(z, dtype), dev(scores), K, config=cfg, mask=None if allowed is None else dev(bits_of(allowed)),
                      history=dev(history), history_len=dev(lens))
    check(out, z, scores, K, stops, T, keep, allowed, history, lens, pen)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("offset,extra", [(0, 0), (1, 0), (3, 5), (7, 1)])
def test_strides_and_alignment(s, dtype, offset, extra):
    import torch
    N, K, V = 3, 4, 9001
    _, z, scores = inputs(offset * 10 + extra, N, K, V, dtype)
    rng = np.random.default_rng(5)
    allowed = rng.random((N * K, V)) < 0.3
    big = torch.full((N * K * (V + extra) + offset + 16,), math.nan, dtype=torch.float32 if dtype == "f32" else torch.bfloat16, device="cuda")
    view = big[offset:offset + N * K * (V + extra)].view(N * K, V + extra)[:, :V]
    view.copy_(dev(z, dtype))
    check(s.beam_step(view, dev(scores), K), z, scores, K)
    check(s.beam_step(view, dev(scores), K, mask=dev(bits_of(allowed))), z, scores, K, allowed=allowed)
    history = rng.integers(0, V, (N * K, 300)).astype(np.int32)
    history[:, :4] = [0, 1, V - 1, V - 2]
    from born_b200 import BeamConfig
    out = s.beam_step(view, dev(scores), K, config=BeamConfig(presence_penalty=1.0), mask=dev(bits_of(allowed)), history=dev(history))
    check(out, z, scores, K, allowed=allowed, history=history, pen=dict(presence=1.0))


def test_offsets_past_32_bits(s):
    import torch
    K, V, stride = 4, 5000, 1 << 30
    _, z, scores = inputs(3, 1, K, V, "bf16")
    big = torch.empty((K - 1) * stride + V, dtype=torch.bfloat16, device="cuda")
    view = big.as_strided((K, V), (stride, 1))
    view.copy_(dev(z, "bf16"))
    check(s.beam_step(view, dev(scores), K), z, scores, K)


def test_rows_without_candidates(s):
    """Masked rows, rows at -inf, NaN and infinities in allowed and in masked places, dead beams; all in one call."""
    K, V = 8, 3000
    _, z, scores = inputs(4, 3, K, V)
    allowed = np.ones((3 * K, V), bool)
    allowed[1] = False                  # nothing allowed
    z[2] = -np.inf                      # nothing above -inf
    z[3, 70] = np.nan
    z[4, 71], allowed[4, 71] = np.nan, False    # masked: not seen
    z[5, 72] = np.inf
    z[6, 73], allowed[6, 73] = np.inf, False
    z[7, ::2] = -np.inf
    scores[0] = -np.inf
    allowed[K:2 * K] = False            # a group without any candidate
    z[2 * K:, 10:] = -np.inf            # fewer candidates than the other rows have
    scores[2 * K + 1], scores[2 * K + 2] = np.nan, np.inf
    from born_b200 import BeamConfig
    for keep in (False, True):
        out = s.beam_step(dev(z), dev(scores), K, config=BeamConfig(keep_slots=keep, stop_tokens=(5,)), mask=dev(bits_of(allowed)))
        check(out, z, scores, K, (5,), keep=keep, allowed=allowed)


@pytest.mark.parametrize("low", [np.finfo(np.float32).min, -1e30])
def test_lowest_values_are_candidates(s, low):
    K, V = 4, 2000
    _, z, scores = inputs(5, 2, K, V)
    z[:, 3:] = low                      # a mask of the type's lowest value: three tokens are left, then ties
    z[K + 1] = low
    check(s.beam_step(dev(z), dev(scores), K), z, scores, K)


@pytest.mark.parametrize("dtype,offset", [("f32", 0), ("f32", 1), ("bf16", 0), ("bf16", 3)])
def test_equal_rows_and_values_go_by_index(s, dtype, offset):
    """Equal logits, equal rows and equal scores: the lowest beam, then the lowest token, however rows are aligned."""
    import torch
    N, K, V = 2, 6, 20001
    rng = np.random.default_rng(6)
    row = np.round(rng.standard_normal(V)).astype(np.float32)
    z = np.tile(row, (N * K, 1))
    z[K:] = 0.5
    scores = np.full(N * K, -7.25, np.float32)
    big = torch.empty(N * K * V + offset, dtype=torch.float32 if dtype == "f32" else torch.bfloat16, device="cuda")
    view = big[offset:].view(N * K, V)
    view.copy_(dev(z, dtype))
    check(s.beam_step(view, dev(scores), K), z, scores, K)


def test_near_ties_of_different_rows(s):
    """Rows that hold the same values in different places, and scores 1e-10 apart: only 64 bits tell them apart."""
    from born_b200 import BeamConfig
    N, K, V, H = 4, 8, 128256, 40
    rng = np.random.default_rng(7)
    z = np.empty((N * K, V), np.float32)
    scores = np.empty(N * K, np.float32)
    for n in range(N):
        row = (rng.standard_normal(V) * 2).astype(np.float32)
        for b in range(K):
            z[n * K + b] = rng.permutation(row)
        base = np.float32(-1e-3)
        step = np.spacing(base)
        scores[n * K:(n + 1) * K] = base + step * rng.permutation(K)
    check(s.beam_step(dev(z), dev(scores), K), z, scores, K)
    # ... with histories, whose tokens enter the normaliser penalised, and a mask
    history = np.stack([np.argsort(-z[r])[:H] for r in range(N * K)]).astype(np.int32)
    history[:, 1::2] = history[:, ::2]
    allowed = z > -1.0
    out = s.beam_step(dev(z), dev(scores), K, config=BeamConfig(frequency_penalty=0.25, temperature=0.8), mask=dev(bits_of(allowed)),
                      history=dev(history))
    check(out, z, scores, K, temperature=0.8, allowed=allowed, history=history, pen=dict(frequency=0.25))


@pytest.mark.parametrize("order", ["ascending", "descending"])
def test_sorted_rows(s, order):
    K, V = 5, 30000
    _, z, scores = inputs(8, 2, K, V)
    z.sort(axis=1)
    if order == "descending":
        z = z[:, ::-1].copy()
    check(s.beam_step(dev(z), dev(scores), K), z, scores, K)


def test_stop_tokens_outside_and_twice(s):
    from born_b200 import BeamConfig
    K, V = 4, 1000
    _, z, scores = inputs(9, 2, K, V)
    z[:, 17] = 9.0
    out = s.beam_step(dev(z), dev(scores), K, config=BeamConfig(stop_tokens=(17, -1, V, 17, 5)))
    check(out, z, scores, K, (17, 5))


def test_scores_in_place(s):
    K, V = 4, 12000
    _, z, scores = inputs(10, 6, K, V)
    t = dev(scores)
    out = s.beam_step(dev(z), t, K, out={"score": t})
    assert out["score"] is t
    check(out, z, scores, K)


def test_results_do_not_depend_on_the_run(s):
    from born_b200 import BeamConfig
    N, K, V = 8, 8, 60000
    _, z, scores = inputs(11, N, K, V)
    hist = dev(np.random.default_rng(1).integers(0, V, (N * K, 500)).astype(np.int32))
    zt, st = dev(z), dev(scores)
    first = None
    for _ in range(5):
        out = s.beam_step(zt, st, K, config=BeamConfig(repetition_penalty=1.1, stop_tokens=(1, 2)), history=hist)
        got = {k: v.cpu().numpy().copy() for k, v in out.items()}
        if first is not None:
            assert all((got[k] == first[k]).all() for k in got)
        first = got


# ---- pool ---------------------------------------------------------------------------------
@pytest.mark.parametrize("alpha,early", [(0.0, False), (1.0, False), (0.6, True), (-0.5, False)])
def test_pool_over_steps(s, alpha, early):
    """Eight steps over logits in which stop tokens are likely: pool, done and what done groups return."""
    from born_b200 import BeamConfig
    N, K, V, steps, stops = 5, 4, 700, 12, (3, 9)
    rng = np.random.default_rng(12)
    cfg = BeamConfig(stop_tokens=stops, length_penalty=alpha, early_stop=early)
    pool = s.beam_pool(N, K)
    want = [R.Pool(K) for _ in range(N)]
    scores = np.full(N * K, -np.inf, np.float32)
    scores[::K] = 0
    for t in range(steps):
        z = (rng.standard_normal((N * K, V)) * 2).astype(np.float32)
        z[:, 3] = 4 + 3 * rng.random(N * K)
        z[:, 9] = 3 + 3 * rng.random(N * K)
        if t == 9:
            z[:K] = -np.inf  # no beam of the first group goes on
        out = s.beam_step(dev(z), dev(scores), K, config=cfg, pool=pool, step=t)
        got = {k: v.cpu().numpy() for k, v in out.items()}
        for n in range(N):
            sl = slice(n * K, (n + 1) * K)
            if want[n].done:
                assert (got["token"][sl] == -1).all() and (got["score"][sl] == -np.inf).all()
                assert got["parent"][sl].tolist() == list(range(K)) and (got["status"][sl] == R.FINISHED).all()
                assert (got["end_token"][n] == -1).all()
                continue
            ref = R.step(list(z[sl]), scores[sl], stops)
            assert got["token"][sl].tolist() == ref["token"] and got["end_token"][n].tolist() == ref["end_token"]
            want[n].add(ref, t, alpha, early)
        done = pool.done.cpu().numpy()
        held = {k: getattr(pool, k).cpu().numpy() for k in ("score", "step", "parent", "token")}
        for n in range(N):
            assert bool(done[n]) == want[n].done, (t, n)
            k = len(want[n].items)
            assert (held["step"][n][k:] == -1).all() and (held["score"][n][k:] == -np.inf).all()
            for i, (v, st, p, tok) in enumerate(want[n].items):
                assert (held["step"][n][i], held["parent"][n][i], held["token"][n][i]) == (st, p, tok)
                assert abs(held["score"][n][i] - v) <= (score_error(V) * steps + abs(v) * 2.0 ** -22) * max(1, (st + 1) ** -alpha)
        # (the next step starts from the reported scores, so that errors do not add up in the comparison)
        scores = got["score"].copy()
    assert any(w.done for w in want) and any(w.items for w in want)


# ---- device-resident history -----------------------------------------------------------------
def test_next_moves_the_histories(s):
    from born_b200 import BeamConfig
    N, K, V, cap = 4, 5, 3000, 24
    rng = np.random.default_rng(13)
    cfg = BeamConfig(repetition_penalty=1.5, presence_penalty=0.5, stop_tokens=(7,), keep_slots=True)
    prompt = rng.integers(0, V, (N * K, 10)).astype(np.int32)
    s.history_create(cap)
    s.history_reset(dev(prompt))
    text = [list(p) for p in prompt]
    scores = np.full(N * K, -np.inf, np.float32)
    scores[::K] = 0
    pen = dict(repetition=1.5, presence=0.5)
    for t in range(30):
        z = (rng.standard_normal((N * K, V)) * 2).astype(np.float32)
        if t == 11:
            z[K:2 * K] = -np.inf  # no beam of the second group goes on: its histories stay
        out = s.beam_next(dev(z), dev(scores), K, config=cfg)
        history = np.full((N * K, cap), -1, np.int32)
        lens = np.array([min(len(x), cap) for x in text], np.int32)
        for r, x in enumerate(text):
            history[r, :lens[r]] = x[-cap:]
        check(out, z, scores, K, (7,), keep=True, history=history, lens=lens, pen=pen)
        parent, token = out["parent"].cpu().numpy(), out["token"].cpu().numpy()
        text = [text[r // K * K + parent[r]] + ([int(token[r])] if token[r] >= 0 else []) for r in range(N * K)]
        scores = out["score"].cpu().numpy()
        ring, total, finished = s.history_read(N * K, cap)
        assert not finished.any()
        for r, x in enumerate(text):
            assert total[r] == len(x)
            for i in range(max(0, len(x) - cap), len(x)):
                assert ring[r, i % cap] == x[i], (t, r, i)


# ---- reordering -----------------------------------------------------------------------------
def expected(x, parents, K, lens, position_dim):
    r = x.shape[0]
    ok = (parents >= 0) & (parents < K)
    src = np.where(ok, np.arange(r) // K * K + parents, np.arange(r))
    y = x.copy()
    for i in range(r):
        if lens is None:
            y[i] = x[src[i]]
        else:
            n = max(0, min(int(lens[i // K]), x.shape[position_dim]))
            sel = [slice(None)] * (x.ndim - 1)
            sel[position_dim - 1] = slice(0, n)
            y[i][tuple(sel)] = x[src[i]][tuple(sel)]
    return y


@pytest.mark.parametrize("shape,position_dim", [((12, 2, 50, 64), 2), ((12, 50, 3, 16), 1), ((12, 1, 1, 1), 2), ((12, 4099), None),
                                                ((12, 3, 7, 5), 2), ((12, 2, 3, 129, 24), 3), ((12,), None), ((12, 5, 1), None)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "int32", "uint8"])
@pytest.mark.parametrize("K", [1, 3, 4, 12])
def test_reorder(s, shape, position_dim, dtype, K):
    import torch
    rng = np.random.default_rng(len(shape) * 100 + K)
    N = 12 // K
    raw = [rng.integers(0, 120, shape) for _ in range(3)]
    states = [torch.from_numpy(x).to(getattr(torch, dtype)).cuda() for x in raw]
    parents = np.concatenate([rng.permutation(K) if n % 2 else rng.integers(0, K, K) for n in range(N)]).astype(np.int32)
    lens = rng.integers(-1, shape[position_dim] + 3, N).astype(np.int32) if position_dim is not None else None
    s.beam_reorder(states, dev(parents), K, lens=None if lens is None else dev(lens), position_dim=position_dim)
    for x, t in zip(raw, states):
        assert (t.cpu().to(torch.float32).numpy() == expected(x, parents, K, lens, position_dim)).all()


@pytest.mark.parametrize("parents", [[1, 2, 3, 0] * 2, [3, 3, 3, 3, 0, 1, 2, 3], [0, 1, 2, 9, -1, 0, 0, 7], [1, 0, 3, 2, 0, 0, 1, 1]])
@pytest.mark.parametrize("offset", [0, 1, 2, 5])
def test_reorder_permutations_and_alignment(s, parents, offset):
    """Cycles, everybody's child, parents that do not exist; bytes on both sides of the rows stay."""
    import torch
    rng = np.random.default_rng(offset)
    buf = rng.integers(0, 250, 8 * 700 + 64).astype(np.uint8)
    t = torch.from_numpy(buf).cuda()
    rows = t[offset:offset + 8 * 700].view(8, 700)[:, :633]
    x = rows.cpu().numpy().copy()
    p = np.array(parents, np.int32)
    s.beam_reorder([rows], dev(p), 4)
    want = buf.copy()
    want[offset:offset + 8 * 700].reshape(8, 700)[:, :633] = expected(x, p, 4, None, None)
    assert (t.cpu().numpy() == want).all()


def test_reorder_pieces_outside_rows(s):
    """A cache of [layers, rows, positions, width] is one call: layers are the pieces of a row."""
    import torch
    rng = np.random.default_rng(2)
    x = rng.standard_normal((5, 8, 33, 8)).astype(np.float32)
    t = torch.from_numpy(x).cuda()
    p = np.array([2, 0, 0, 3, 1, 1, 1, 0], np.int32)
    lens = np.array([20, 33], np.int32)
    s.beam_reorder([t.transpose(0, 1)], dev(p), 4, lens=dev(lens), position_dim=2)
    want = expected(x.transpose(1, 0, 2, 3).copy(), p, 4, lens, 2)
    assert (t.cpu().numpy().transpose(1, 0, 2, 3) == want).all()


def test_reorder_past_32_bits(s):
    import torch
    t = torch.zeros((4, 1500, 1024, 1024), dtype=torch.uint8, device="cuda")  # 1.5 GB a row
    t[:, ::100, 3, 5] = torch.arange(4, device="cuda", dtype=torch.uint8)[:, None] + 1
    p = np.array([0, 0, 3, 2], np.int32)
    s.beam_reorder([t], dev(p), 4)
    assert t[:, ::100, 3, 5].cpu().numpy().T.tolist() == [[1, 1, 4, 3]] * 15


# ---- sequences ---------------------------------------------------------------------------------
@pytest.mark.parametrize("N,K,T,H", [(1, 1, 1, 1), (2, 4, 2, 4), (3, 16, 255, 16), (1, 5, 256, 3), (2, 8, 257, 8), (4, 3, 1000, 5), (1, 16, 16384, 2), (1, 2, 70001, 2), (2, 4, 512, 4), (2, 4, 513, 4), (80, 4, 2049, 4), (3, 9, 5000, 2), (150, 2, 1500, 3)])
@pytest.mark.parametrize("broken", [False, True])
def test_sequences(s, N, K, T, H, broken):
    rng = np.random.default_rng(T)
    tokens = rng.integers(0, 100000, (T, N * K)).astype(np.int32)
    parents = rng.integers(0, K, (T, N * K)).astype(np.int32)
    parents[0] = -5  # nothing lies before the first step
    if broken:
        parents[rng.integers(0, T, 3), rng.integers(0, N * K, 3)] = [-1, K, 1 << 20]
    es = rng.integers(-2, T + 2, (N, H)).astype(np.int32)
    es[0, 0] = T - 1
    ep = rng.integers(0, K, (N, H)).astype(np.int32)
    if broken:
        ep[N - 1, H - 1] = K
    et = rng.integers(0, 100000, (N, H)).astype(np.int32)
    out = s.beam_sequences(dev(tokens), dev(parents), dev(es), dev(ep), dev(et), K, pad=-7)
    got, lens = out["tokens"].cpu().numpy(), out["lens"].cpu().numpy()
    for n in range(N):
        for h in range(H):
            want, e, b = [-7] * T, int(es[n, h]), int(ep[n, h])
            ok = 0 <= e < T and 0 <= b < K
            if ok:
                want[e] = int(et[n, h])
                for t in range(e - 1, -1, -1):
                    want[t] = int(tokens[t, n * K + b])
                    b = int(parents[t, n * K + b])
                    if t > 0 and not 0 <= b < K:
                        ok = False
                        break
            if not ok:
                want, e = [-7] * T, -1
            assert lens[n, h] == e + 1 and got[n, h].tolist() == want, (n, h)


# ---- the loop ---------------------------------------------------------------------------------
def run_loop(s, table, N, K, steps, stops, stream=None, graph=False):
    """A search over a model whose logits depend on the last token alone; every row's state is the sum of its tokens."""
    import torch
    from born_b200 import BeamConfig
    V = table.shape[1]
    cfg = BeamConfig(stop_tokens=stops, length_penalty=1.0, keep_slots=True)
    tab = dev(table)
    d = tab.device
    last = torch.zeros(N * K, dtype=torch.int64, device=d)
    last.copy_(torch.arange(N, device=d).repeat_interleave(K) + 11)
    scores = torch.full((N * K,), -math.inf, device=d)
    scores[::K] = 0
    tokens = torch.full((steps, N * K), -1, dtype=torch.int32, device=d)
    parents = torch.zeros((steps, N * K), dtype=torch.int32, device=d)
    total = torch.zeros((N * K, 3, 4, 2), dtype=torch.int32, device=d)
    logits = torch.empty((N * K, V), device=d)
    pool = s.beam_pool(N, K)

    def steps_of():
        raw = torch.cuda.current_stream().cuda_stream
        for t in range(steps):
            torch.index_select(tab, 0, last, out=logits)
            s.beam_step(logits, scores, K, config=cfg, pool=pool, step=t, stream=raw,
                        out={"token": tokens[t], "parent": parents[t], "score": scores})
            s.beam_reorder([total], parents[t], K, stream=raw)
            last.copy_(tokens[t].clamp(min=0))
            total.add_(tokens[t].clamp(min=0)[:, None, None, None])
        return s.beam_sequences(tokens, parents, pool.step, pool.parent, pool.token, K, stream=raw)

    side = stream or torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    if graph:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            seq = steps_of()
        g.replay()
    else:
        with torch.cuda.stream(side):
            seq = steps_of()
    torch.cuda.synchronize()
    return pool, seq, total.cpu().numpy(), tokens.cpu().numpy(), parents.cpu().numpy()


@pytest.mark.parametrize("graph", [False, True])
def test_loop_finds_what_the_definition_finds(s, graph):
    N, K, V, steps, stops = 3, 4, 400, 14, (5, 6)
    rng = np.random.default_rng(21)
    table = (rng.standard_normal((V, V)) * 2.5).astype(np.float32)
    table[:, 5] += 2.0
    pool, seq, total, tokens, parents = run_loop(s, table, N, K, steps, stops, graph=graph)
    got, lens = seq["tokens"].cpu().numpy(), seq["lens"].cpu().numpy()
    held = {k: getattr(pool, k).cpu().numpy() for k in ("score", "step")}
    for n in range(N):
        # the definition's search, with whole sequences in place of tables
        beams = [([], 0.0)] + [([], -np.inf)] * (K - 1)
        ref, kept = R.Pool(K), []
        for t in range(steps):
            if ref.done:
                break
            rows = [table[b[0][-1] if b[0] else n + 11] for b in beams]
            out = R.step(rows, [np.float32(b[1]) for b in beams], stops, keep_slots=True)
            before = list(ref.items)
            ref.add(out, t, 1.0, False)
            kept += [((t, p, k), beams[p][0] + [k]) for p, k in zip(out["end_parent"], out["end_token"]) if k >= 0]
            beams = [((beams[p][0] + [k]) if k >= 0 else beams[p][0], v) for p, k, v in zip(out["parent"], out["token"], out["score"])]
            del before
        kept = dict(kept)
        for i, (v, t, p, k) in enumerate(ref.items):
            want = kept[(t, p, k)]
            assert held["step"][n, i] == t and lens[n, i] == len(want)
            assert got[n, i, :len(want)].tolist() == want and (got[n, i, len(want):] == -1).all()
            # each of the steps rounds the running score once
            assert abs(held["score"][n, i] - v) <= steps * (score_error(V) + abs(v) * (t + 1) * 2.0 ** -24) / (t + 1) + abs(v) * 2.0 ** -24
        if not ref.done:
            for b in range(K):
                assert (total[n * K + b] == sum(beams[b][0])).all()


def test_two_handles_on_two_streams(s):
    import torch
    from born_b200 import Sampler
    rng = np.random.default_rng(22)
    table = (rng.standard_normal((300, 300)) * 2.5).astype(np.float32)
    with Sampler(device=0, max_batch=64, max_vocab=512) as other:
        a = run_loop(s, table, 2, 4, 10, (5,), stream=torch.cuda.Stream())
        b = run_loop(other, table, 2, 4, 10, (5,), stream=torch.cuda.Stream())
    assert (a[3] == b[3]).all() and (a[4] == b[4]).all()


# ---- refusals ----------------------------------------------------------------------------------
def test_refusals(s):
    import torch
    from born_b200 import BeamConfig, InvalidArgument, SamplerError, _lib as L
    K, V = 4, 100
    z, sc = torch.zeros((8, V), device="cuda"), torch.zeros(8, device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")

    def bad(error, code, f, *a, **kw):
        with pytest.raises(error) as e:
            f(*a, **kw)
        assert e.value.code == code, e.value

    inv, uns = (InvalidArgument, L.ERR_INVALID_ARGUMENT), (SamplerError, L.ERR_UNSUPPORTED)
    bad(*inv, s.beam_step, z, sc, 3)                         # rows are no multiple of the beams
    bad(*inv, s.beam_step, z, sc, 0)
    bad(*inv, s.beam_step, z.cpu(), sc, K)
    bad(*inv, s.beam_step, z, sc.cpu(), K)
    bad(*inv, s.beam_step, z, sc.double(), K)
    bad(*inv, s.beam_step, z, sc[:4], K)
    bad(*inv, s.beam_step, z.half(), sc, K)
    bad(*inv, s.beam_step, z.t(), torch.zeros(V, device="cuda"), K)
    bad(*inv, s.beam_step, z[0], sc, K)
    bad(*inv, s.beam_step, z, sc, K, mask=torch.zeros((8, 3), **i32))
    bad(*inv, s.beam_step, z, sc, K, mask=torch.zeros((4, 4), **i32))
    bad(*inv, s.beam_step, z, sc, K, history=torch.zeros((8, 3), device="cuda"))
    bad(*inv, s.beam_step, z, sc, K, history_len=torch.zeros(8, **i32))
    bad(*inv, s.beam_step, z, sc, K, config=BeamConfig(stop_tokens=tuple(range(9))))
    bad(*inv, s.beam_step, z, sc, K, config=BeamConfig(temperature=-1.0))
    bad(*inv, s.beam_step, z, sc, K, config=BeamConfig(temperature=math.nan))
    bad(*inv, s.beam_step, z, sc, K, pool=s.beam_pool(4, 2))
    bad(*inv, s.beam_step, z, sc, K, pool=s.beam_pool(2, 4), step=-1)
    bad(*inv, s.beam_step, z, sc, K, pool=s.beam_pool(2, 4), config=BeamConfig(length_penalty=math.inf))
    bad(*uns, s.beam_step, torch.zeros((17, V), device="cuda"), torch.zeros(17, device="cuda"), 17)
    bad(*uns, s.beam_step, z, sc, K, history=torch.zeros((8, 1025), **i32))
    bad(*inv, s.beam_step, torch.zeros((520, V), device="cuda"), torch.zeros(520, device="cuda"), K)
    bad(*inv, s.beam_next, z, sc, K, history=torch.zeros((8, 3), **i32))
    call = s.prepare_beam_step(z, sc, K)
    for field, value, err in [("struct_size", 8, inv), ("memory", L.MEM_HOST, uns), ("memory", 9, inv), ("groups", 0, inv),
                              ("logits_row_stride", V - 1, inv), ("logits_dtype", 7, inv), ("out_parent", None, inv),
                              ("scores", None, inv), ("n_stop", 9, inv), ("flags", 8, inv), ("vocab", 0, inv),
                              ("out_end_token", 16, inv), ("done", 16, inv), ("logits", z.data_ptr() + 1, inv)]:
        keep = getattr(call.args, field)
        setattr(call.args, field, value)
        bad(*err, call.run)
        setattr(call.args, field, keep)
    call.args.params.top_k = 5
    bad(*uns, call.run)

    p = torch.zeros(8, **i32)
    bad(*inv, s.beam_reorder, [], p, K)
    bad(*inv, s.beam_reorder, [z, sc], p, K)
    bad(*inv, s.beam_reorder, [z.cpu()], p, K)
    bad(*inv, s.beam_reorder, [z], p.long(), K)
    bad(*inv, s.beam_reorder, [z], p[:4], K)
    bad(*inv, s.beam_reorder, [z], p, K, lens=torch.zeros(2, **i32))
    bad(*inv, s.beam_reorder, [z], p, K, lens=torch.zeros(3, **i32), position_dim=1)
    bad(*inv, s.beam_reorder, [z], p, K, position_dim=2)
    bad(*inv, s.beam_reorder, [z[:1].expand(8, V)], p, K)          # rows that overlap
    bad(*inv, s.beam_reorder, [torch.zeros((8, 6, 4), device="cuda").transpose(1, 2)], p, K, position_dim=1)
    bad(*inv, s.beam_reorder, [torch.zeros((8, 3, 4, 5, 6), device="cuda").transpose(1, 2)[:, :, :2]], p, K, position_dim=3)
    bad(*uns, s.beam_reorder, [z] * 129, p, K)

    t = torch.zeros((5, 8), **i32)
    e = torch.zeros((2, 4), **i32)
    bad(*inv, s.beam_sequences, t, t[:4], e, e, e, K)
    bad(*inv, s.beam_sequences, t, t, e, e, e[:1], K)
    bad(*inv, s.beam_sequences, t, t, e[:1], e, e, K)
    bad(*inv, s.beam_sequences, t.long(), t, e, e, e, K)
    e17 = torch.zeros((2, 17), **i32)
    bad(*uns, s.beam_sequences, t, t, e17, e17, e17, K)


# ---- the search path --------------------------------------------------------------------------
@pytest.mark.parametrize("history", [0, 16])
@pytest.mark.parametrize("side", [False, True])
def test_search_path(s, history, side):
    """BeamSearch over a head: hidden states are rows of a table picked by the last token, so that the definition can
    follow; whole numbers in the table and the head make the logits exact."""
    import torch
    from born_b200 import BeamConfig, BeamSearch, Head
    N, K, V, D, steps, stops = 3, 4, 300, 64, 12, (5, 6)
    rng = np.random.default_rng(31)
    hid = rng.integers(-3, 4, (V, D)).astype(np.float32)
    w = rng.integers(-3, 4, (V, D)).astype(np.float32)
    bias = (rng.standard_normal(V) * 8 - 60).astype(np.float32)
    bias[list(stops)] += 30
    T = 7.0
    pen = dict(repetition=1.3, presence=2.0) if history else {}
    cfg = BeamConfig(temperature=T, stop_tokens=stops, length_penalty=0.8, keep_slots=True,
                     repetition_penalty=pen.get("repetition", 0.0), presence_penalty=pen.get("presence", 0.0))
    head = Head(dev(w).to(torch.bfloat16), dev(bias))
    table = dev(hid).to(torch.bfloat16)
    st = torch.cuda.Stream() if side else torch.cuda.default_stream()
    raw = st.cuda_stream if side else None
    prompts = rng.integers(0, V, (N, 5)).astype(np.int32)
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        search = BeamSearch(s, N, K, steps, V, cfg, head=head, history=history)
        cache = torch.zeros((N * K, 2, steps, 3), device="cuda")
        flat = torch.zeros((N * K, 7), device="cuda", dtype=torch.int32)
        search.begin(dev(prompts) if history else None, stream=raw)
        last = torch.arange(N, device="cuda").repeat_interleave(K) + 11
        for t in range(steps):
            cache[:, :, t] = last.float()[:, None, None]
            used = torch.full((N,), t + 1, dtype=torch.int32, device="cuda")
            search.step(table[last], states=[cache], lens=used, position_dim=2, stream=raw)
            s.beam_reorder([flat], search.parent_table[t], K, stream=raw)
            last = search.tokens.clamp(min=0).long()
        found = search.result(stream=raw)
    torch.cuda.synchronize()
    got = {k: v.cpu().numpy() for k, v in found.items()}
    cache = cache.cpu().numpy()
    for n in range(N):
        beams = [([], 0.0)] + [([], -np.inf)] * (K - 1)
        ref, kept = R.Pool(K), {}
        fed = [[] for _ in range(K)]
        for t in range(steps):
            if ref.done:
                break
            rows = []
            for b in range(K):
                at = beams[b][0][-1] if beams[b][0] else n + 11
                row = (hid[at] @ w.T + bias).astype(np.float32)
                if history:
                    row = R.penalised(row, (list(prompts[n]) + beams[b][0])[-history:], **pen)
                rows.append(row)
            out = R.step(rows, [np.float32(b[1]) for b in beams], stops, T, True)
            fed = [fed[p] + [beams[p][0][-1] if beams[p][0] else n + 11] for p in out["parent"]]
            for p, k in zip(out["end_parent"], out["end_token"]):
                if k >= 0:
                    kept[(t, p, k)] = beams[p][0] + [k]
            ref.add(out, t, 0.8, False)
            beams = [((beams[p][0] + [k]) if k >= 0 else beams[p][0], v) for p, k, v in zip(out["parent"], out["token"], out["score"])]
        want = [(float(v), kept[(t, p, k)]) for v, t, p, k in ref.items]
        if not ref.done:
            want += [(v / steps ** np.float64(np.float32(0.8)), q) for q, v in beams if np.isfinite(v)]
            for b in range(K):  # the caches followed the beams that were fed
                assert cache[n * K + b, 0, :, 0].tolist() == fed[b], (n, b)
        want.sort(key=lambda x: -x[0])
        for i, (v, q) in enumerate(want[:K]):
            assert got["lens"][n, i] == len(q) and got["tokens"][n, i, :len(q)].tolist() == q, (n, i)
            # every step rounds the running score once, the normalised one is rounded twice
            assert abs(got["scores"][n, i] - v) <= steps * score_error(V) + (steps + 2) * abs(v) * len(q) * 2.0 ** -24
        for i in range(len(want), K):
            assert got["lens"][n, i] == 0 and got["scores"][n, i] == -np.inf


def test_search_refusals(s):
    import torch
    from born_b200 import BeamConfig, BeamSearch, Head, InvalidArgument
    with pytest.raises(InvalidArgument):
        BeamSearch(s, 2, 4, 5, 100, BeamConfig(presence_penalty=1.0))
    with pytest.raises(InvalidArgument):
        BeamSearch(s, 0, 4, 5, 100)
    with pytest.raises(InvalidArgument):
        BeamSearch(s, 2, 4, 5, 100, head=Head(torch.zeros((99, 64), dtype=torch.bfloat16, device="cuda")))
    b = BeamSearch(s, 2, 4, 1, 100)
    z = torch.zeros((8, 100), device="cuda")
    for f in (lambda: b.step(z), lambda: b.tokens, b.result):
        with pytest.raises(InvalidArgument):
            f()
    b.begin()
    with pytest.raises(InvalidArgument):
        b.step(z[:4])
    b.step(z)
    with pytest.raises(InvalidArgument):
        b.step(z)


def test_search_steps_allocate_nothing(s):
    """What a step writes must not be memory that the caller's other work gets while the kernel still runs."""
    import torch
    from born_b200 import BeamConfig, BeamSearch
    N, K, V = 2, 4, 600
    z = torch.randn((N * K, V), device="cuda")
    state = torch.zeros((N * K, 8), device="cuda")
    search = BeamSearch(s, N, K, 6, V, BeamConfig(stop_tokens=(3,)))
    search.begin()
    search.step(z, states=[state])
    before = torch.cuda.memory_stats()["allocation.all.allocated"]
    for _ in range(5):
        search.step(z, states=[state])
    assert torch.cuda.memory_stats()["allocation.all.allocated"] == before


def test_search_refuses_states_before_the_step(s):
    import torch
    from born_b200 import BeamSearch, InvalidArgument
    N, K, V = 2, 4, 600
    z = torch.randn((N * K, V), device="cuda")
    search = BeamSearch(s, N, K, 6, V)
    search.begin()
    scores = search.scores.clone()
    with pytest.raises(InvalidArgument):
        search.step(z, states=[torch.zeros((N * K + 1, 8), device="cuda")])
    assert search.steps == 0 and torch.equal(search.scores, scores)


def test_sizes_that_are_refused(s):
    import torch
    from born_b200 import InvalidArgument, SamplerError, _lib as L
    i32 = dict(dtype=torch.int32, device="cuda")
    p, z = torch.zeros(8, **i32), torch.zeros((8, 100), device="cuda")
    with pytest.raises(InvalidArgument):  # rows would be moved twice at once
        s.beam_reorder([z, torch.zeros_like(z), z], p, 4)
    t, e = torch.zeros((5, 8), **i32), torch.zeros((2, 4), **i32)
    call = s.prepare_beam_sequences(t, t, e, e, e, 4)
    call.args.steps = call.args.out_stride = 2 ** 30 + 1
    with pytest.raises(SamplerError) as err:
        call.run()
    assert err.value.code == L.ERR_UNSUPPORTED


def test_thousands_of_groups(lib):
    """More rows than 2^31 tokens hold; every row has its best tokens at places of its own."""
    import torch
    from born_b200 import Sampler
    N, K, V = 2200, 8, 131072
    R = N * K
    z = torch.zeros((R, V), dtype=torch.bfloat16, device="cuda")
    at = torch.arange(R, device="cuda") * 7919 % (V - 8)
    for j in range(K):
        z[torch.arange(R, device="cuda"), at + j] = 12.0 - j
    scores = torch.full((R,), -math.inf, device="cuda")
    scores[::K] = 0.0
    with Sampler(device=0, max_batch=R, max_vocab=V) as big:
        out = big.beam_step(z, scores, K)
        want = at[::K, None] + torch.arange(K, device="cuda")
        assert torch.equal(out["token"].view(N, K).long(), want)
        assert (out["parent"] == 0).all()
        # All beams alive and alike in score: the best token of each.  In which order is open: the rows hold the same values
        # in different places, so their normalisers are equal but for the rounding of a sum in another order.
        out = big.beam_step(z, torch.zeros(R, device="cuda"), K)
        parent = out["parent"].view(N, K).long()
        assert torch.equal(parent.sort(1).values, torch.arange(K, device="cuda").expand(N, K))
        assert torch.equal(out["token"].view(N, K).long(), at.view(N, K).gather(1, parent))
