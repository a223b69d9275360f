"""Calls on streams of their own while the default stream has work pending.

Torch's streams do not wait for the default stream, so nothing that a call on one of them depends on may be left there."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

BUSY = 400_000_000  # clock cycles that the default stream is kept busy for: a fifth of a second and more


def busy(stream=None):
    """Occupies the default stream (or the given one) with a kernel that only waits; returns an event behind it."""
    import torch
    with torch.cuda.stream(stream or torch.cuda.default_stream()):
        torch.cuda._sleep(BUSY)
        done = torch.cuda.Event()
        done.record()
    return done


def test_new_handles_and_histories_are_ready(lib):
    """What a handle and its history start from is there when the calls that make them return."""
    import torch
    from born_b200 import Sampler, SamplingConfig
    B, V, cap = 8, 5000, 40
    g = torch.Generator(device="cuda").manual_seed(3)
    z = torch.randn((B, V), generator=g, device="cuda")
    prompts = torch.randint(0, V, (B, 30), generator=g, device="cuda", dtype=torch.int32)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    end = busy()
    with Sampler(device=0, max_batch=B, max_vocab=V) as s, torch.cuda.stream(side):
        s.history_create(cap)
        s.history_reset(prompts, stream=side.cuda_stream)
        out = s.sample_next(z, config=SamplingConfig(), stream=side.cuda_stream)
        beam = s.beam_step(z, torch.zeros(B, device="cuda"), 4, stream=side.cuda_stream)
        end.synchronize()
        side.synchronize()
        tokens, total, _ = s.history_read(B, cap, stream=side.cuda_stream)
        assert total.tolist() == [31] * B
        assert np.array_equal(tokens[:, :30], prompts.cpu().numpy())
        assert torch.equal(out["token"].long(), z.argmax(1)) and np.array_equal(tokens[:, 30], out["token"].cpu().numpy())
        assert (beam["status"] == 0).all() and (beam["token"] >= 0).all()
        s.check_error()


@pytest.mark.parametrize("history", [0, 24])
def test_a_search_made_while_the_default_stream_is_busy(lib, history):
    """A search that is made and run on a side stream while the default stream has work pending finds what it finds alone."""
    import torch
    from born_b200 import BeamConfig, BeamSearch, Sampler
    N, K, V, steps = 3, 4, 700, 8
    g = torch.Generator(device="cuda").manual_seed(11)
    z = torch.randn((steps, N * K, V), generator=g, device="cuda") * 2
    z[:, :, 5] += 5.0  # (hypotheses end in many steps)
    prompts = torch.randint(0, V, (N, 6), generator=g, device="cuda", dtype=torch.int32)
    cfg = BeamConfig(stop_tokens=(5,), length_penalty=0.9, presence_penalty=0.5 if history else 0.0)

    def run(s, stream):
        search = BeamSearch(s, N, K, steps, V, cfg, history=history)
        search.begin(prompts if history else None, stream=stream)
        for t in range(steps):
            search.step(z[t], stream=stream)
        return search, search.result(stream=stream)

    with Sampler(device=0, max_batch=64, max_vocab=1024) as s:
        search, alone = run(s, None)
        torch.cuda.synchronize()
        assert (search.pool.step >= 0).any()
        side = torch.cuda.Stream()
        for current in (torch.cuda.default_stream(), side):
            end = busy()
            with torch.cuda.stream(current):
                search, found = run(s, side.cuda_stream)
            end.synchronize()
            torch.cuda.synchronize()
            for k in alone:
                assert torch.equal(alone[k], found[k]), k
        s.check_error()


def test_a_search_dropped_before_its_stream_has_run(lib):
    """The memory of a search that is gone is not handed out while its calls still wait on their stream."""
    import torch
    from born_b200 import BeamSearch, Sampler
    N, K, V, steps = 2, 4, 500, 6
    z = torch.randn((steps, N * K, V), device="cuda") * 2
    side = torch.cuda.Stream()
    with Sampler(device=0, max_batch=64, max_vocab=1024) as s:
        def run(stream):
            search = BeamSearch(s, N, K, steps, V)
            search.begin(stream=stream)
            for t in range(steps):
                search.step(z[t], stream=stream)
            return search.result(stream=stream)
        alone = run(None)
        torch.cuda.synchronize()
        end = busy(side)
        found = run(side.cuda_stream)
        # what a program does next with such sizes, on the stream where the search was made
        next_ones = [torch.full((n,), 7, dtype=torch.int32, device="cuda") for n in (steps * N * K, N * K, N) for _ in range(6)]
        assert not end.query()
        torch.cuda.synchronize()
        for k in alone:
            assert torch.equal(alone[k], found[k]), k
        assert all((x == 7).all() for x in next_ones)
        s.check_error()
