"""The host side of `BeamSearch` without a device: a sampler and a `torch.cuda` that only write down what is asked of them."""
import contextlib

import pytest

torch = pytest.importorskip("torch")


class Stream:
    def __init__(self, raw):
        self.cuda_stream = raw


class Cuda:
    """`torch.cuda` as far as a search uses it."""

    def __init__(self, log, current):
        self.log, self.now, self.capturing = log, Stream(current), False
        cuda = self

        class Event:
            def record(self, stream=None):
                cuda.log.append(("record", (stream or cuda.now).cuda_stream))

            def wait(self, stream=None):
                cuda.log.append(("wait", (stream or cuda.now).cuda_stream))

        self.Event = Event

    def current_stream(self, device=None):
        return self.now

    def default_stream(self, device=None):
        return Stream(0)

    def ExternalStream(self, raw, device=None):  # noqa: N802
        return Stream(raw)

    def is_current_stream_capturing(self):
        return self.capturing

    @contextlib.contextmanager
    def stream(self, s):
        before, self.now = self.now, s
        yield
        self.now = before


class Torch:
    """torch with every tensor on the CPU."""

    def __init__(self, cuda):
        self.cuda = cuda

    def __getattr__(self, name):
        return getattr(torch, name)

    @staticmethod
    def empty(*a, device=None, **kw):
        return torch.zeros(*a, **kw)


class FakeSampler:
    device = 0

    def __init__(self, log):
        self.log = log

    def beam_pool(self, groups, beams, stream=None):
        self.log.append(("launch", stream or 0))

    def beam_pool_reset(self, pool, stream=None):
        self.log.append(("launch", stream or 0))

    def history_create(self, capacity):
        self.log.append(("history", capacity))

    def history_reset(self, tokens, lens=None, stream=None):
        self.log.append(("launch", stream or 0))
        self.loaded = (tokens, lens)


@pytest.fixture
def fakes(monkeypatch):
    from born_b200 import beam, sampler

    def make(current):
        log = []
        cuda = Cuda(log, current)
        for module in (beam, sampler):
            monkeypatch.setattr(module, "torch", Torch(cuda))
        return log, cuda, FakeSampler(log)
    return make


@pytest.mark.parametrize("history", [0, 8])
@pytest.mark.parametrize("current,used", [(0, 7), (5, 7), (5, None), (0, None), (7, 7)])
def test_a_search_starts_on_its_own_stream(fakes, history, current, used):
    """Making a search launches nothing (a launch on the default stream could come behind the steps of another one), and
    its first launch comes behind what the tables' memory was used for before."""
    from born_b200 import BeamSearch
    log, _, s = fakes(current)
    search = BeamSearch(s, 2, 4, 5, 100, history=history)
    assert [e for e in log if e[0] == "launch"] == []
    del log[:]
    search.begin(stream=used)
    at = used or 0
    assert {e[1] for e in log} == {at}
    launches = ["launch"] * (2 if history else 1)
    assert [e[0] for e in log if e[0] != "record"] == (launches if at == current else ["wait"] + launches)


def test_a_captured_start_waits_for_nothing_outside(fakes):
    from born_b200 import BeamSearch
    log, cuda, s = fakes(0)
    search = BeamSearch(s, 2, 4, 5, 100)
    del log[:]
    cuda.capturing = True
    search.begin(stream=7)
    assert log == [("launch", 7)]


@pytest.mark.parametrize("current,used", [(0, 7), (5, None)])
def test_a_search_that_goes_leaves_its_memory_behind_its_calls(fakes, current, used):
    """The tables' memory returns to the stream on which they were made: that stream waits for what was called on another."""
    from born_b200 import BeamSearch
    log, cuda, s = fakes(current)
    search = BeamSearch(s, 2, 4, 5, 100)
    search.begin(stream=used)
    assert log[-1] == ("record", used or 0)
    del search
    assert log[-1] == ("wait", current)


def test_a_search_on_one_stream_needs_no_events(fakes):
    from born_b200 import BeamSearch
    log, cuda, s = fakes(7)
    search = BeamSearch(s, 2, 4, 5, 100)
    del log[:]
    search.begin(stream=7)
    del search
    assert log == [("launch", 7)]


def test_a_search_that_goes_during_a_capture_keeps_its_memory(fakes):
    from born_b200 import BeamSearch, beam
    log, cuda, s = fakes(0)
    search = BeamSearch(s, 2, 4, 5, 100)
    search.begin(stream=7)
    table = search.token_table
    cuda.capturing = True
    del log[:]
    del search
    assert log == [] and beam._parked.pop()["token_table"] is table


def test_prompts_of_another_type_or_shape_are_refused(fakes):
    from born_b200 import BeamSearch, InvalidArgument
    log, cuda, s = fakes(0)
    search = BeamSearch(s, 3, 2, 5, 100, history=8)
    good, lens = torch.arange(12, dtype=torch.int32).view(3, 4), torch.tensor([4, 0, 2], dtype=torch.int32)
    for prompts, n in ((good.long(), None), (good.float(), None), (good[:2], None), (good.view(6, 2), None), (good[0], None),
                       (good, lens.long()), (good, lens[:2]), (good, lens[:, None])):
        with pytest.raises(InvalidArgument):
            search.begin(prompts, n)
        assert search.steps is None
    search.begin(good, lens)
    rows, n = s.loaded
    assert torch.equal(rows, good.repeat_interleave(2, 0)) and n.tolist() == [4, 4, 0, 0, 2, 2]
