"""Beam search over histories as texts have them: long, and with the same tokens over and over."""
import numpy as np
import pytest

from tests import np_beam as R
from tests.test_gpu_beam import bits_of, check, dev, to_bf16

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def s(lib):
    from born_b200 import Sampler
    with Sampler(device=0, max_batch=64, max_vocab=131072) as h:
        yield h


def text_like(rng, shape, V):
    """Ids by rank: the r-th most frequent one in proportion to 1/r."""
    ids = np.exp(rng.random(shape) * np.log(V)).astype(np.int64) - 1
    return ids.clip(0, V - 1).astype(np.int32)


@pytest.mark.parametrize("N,K,V,H", [(2, 16, 1000, 1024), (4, 4, 128256, 512), (1, 3, 50257, 1023), (8, 8, 300, 257), (2, 2, 40, 1024)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("masked", [False, True])
def test_repeated_tokens(s, N, K, V, H, dtype, masked):
    from born_b200 import BeamConfig
    rng = np.random.default_rng(V + H)
    z = (rng.standard_normal((N * K, V)) * 2).astype(np.float32)
    z[:, :20] += 3  # (frequent tokens are likely ones)
    if dtype == "bf16":
        z = to_bf16(z)
    scores = (-20 - 3 * rng.random(N * K)).astype(np.float32)
    history, lens = text_like(rng, (N * K, H), V), rng.integers(0, H + 1, N * K).astype(np.int32)
    allowed = rng.random((N * K, V)) < 0.3 if masked else None
    pen = dict(frequency=0.2, presence=0.3)
    stops = (3, V - 1)
    out = s.beam_step(dev(z, dtype), dev(scores), K, history=dev(history), history_len=dev(lens), mask=dev(bits_of(allowed)) if masked else None,
                      config=BeamConfig(frequency_penalty=0.2, presence_penalty=0.3, stop_tokens=stops))
    check(out, z, scores, K, stops, allowed=allowed, history=history, lens=lens, pen=pen)


@pytest.mark.parametrize("N,K,V,cap,prompt", [(2, 16, 2000, 600, 595), (3, 4, 50257, 1024, 1100), (5, 3, 900, 257, 0), (1, 1, 500, 1, 3), (2, 5, 700, 256, 256)])
@pytest.mark.parametrize("keep", [False, True])
def test_next_with_a_pool(s, N, K, V, cap, prompt, keep):
    """Histories of every length move with their beams, step after step, while ended hypotheses gather in the pool."""
    from born_b200 import BeamConfig
    rng = np.random.default_rng(cap)
    stops, alpha, steps = (2, 9), 0.7, 10
    cfg = BeamConfig(repetition_penalty=1.2, frequency_penalty=0.1, stop_tokens=stops, keep_slots=keep, length_penalty=alpha)
    pen = dict(repetition=1.2, frequency=0.1)
    prompts = text_like(rng, (N * K, prompt), V)
    s.history_create(cap)
    s.history_reset(dev(prompts) if prompt else prompts.reshape(N * K, 0))
    text = [list(p[-cap:]) for p in prompts]
    pool, refs = s.beam_pool(N, K), [R.Pool(K) for _ in range(N)]
    scores = np.full(N * K, -np.inf, np.float32)
    scores[::K] = 0
    for t in range(steps):
        z = (rng.standard_normal((N * K, V)) * 2).astype(np.float32)
        z[:, 2] += 4.0 * (rng.random(N * K) < 0.3)
        was_done = [r.done for r in refs]
        out = s.beam_next(dev(z), dev(scores), K, config=cfg, pool=pool, step=t)
        got = {k: v.cpu().numpy() for k, v in out.items()}
        for n in range(N):
            sl = slice(n * K, (n + 1) * K)
            if was_done[n]:
                assert (got["status"][sl] == R.FINISHED).all() and (got["token"][sl] == -1).all() and (got["score"][sl] == -np.inf).all()
                assert got["parent"][sl].tolist() == list(range(K)) and (got["end_token"][n] == -1).all()
                continue
            rows = [R.penalised(z[r], text[r][-cap:], **pen) for r in range(n * K, (n + 1) * K)]
            want = R.step(rows, scores[sl], stops, 0.0, keep)
            for k in ("status", "token", "parent"):
                assert got[k][sl].tolist() == want[k], (t, n, k)
            assert got["end_token"][n].tolist() == want["end_token"] and got["end_parent"][n].tolist() == want["end_parent"]
            refs[n].add(want, t, alpha, False)
        text = [text[r // K * K + got["parent"][r]] + ([int(got["token"][r])] if got["token"][r] >= 0 else []) for r in range(N * K)]
        scores = got["score"]
        ring, total, _ = s.history_read(N * K, cap)
        held = {k: getattr(pool, k).cpu().numpy() for k in ("step", "parent", "token", "done")}
        for r, x in enumerate(text):
            assert total[r] == len(x)
            for i in range(max(0, len(x) - cap), len(x)):
                assert ring[r, i % cap] == x[i], (t, r, i)
        for n in range(N):
            items = [(i[1], i[2], i[3]) for i in refs[n].items]
            assert list(zip(held["step"][n], held["parent"][n], held["token"][n]))[:len(items)] == items, (t, n)
            assert (held["step"][n][len(items):] == -1).all() and bool(held["done"][n]) == refs[n].done
    s.check_error()
