"""A captured verify pass and its 8-bit cache's buffers, on the CPU: the capture is a
stand-in that runs the pass, the kernels' stand-ins are those of the cache's own
tests."""
import contextlib
import types
import weakref

import pytest
import torch

from specfit_b200.runtime import verify_graph as vg
from test_kv8_cpu import cache, feed, plain, rows_of  # noqa: F401 (plain is a fixture)


class Stream:
    def wait_stream(self, other):
        pass


class Graph:
    def __init__(self):
        self.replays = 0

    def replay(self):
        self.replays += 1


@pytest.fixture
def captured(plain, monkeypatch):  # noqa: F811
    """(cache, graph): captured over 70 rows, trees of 4."""
    cuda = types.SimpleNamespace(Stream=lambda device=None: Stream(), current_stream=lambda device=None: Stream(),
                                 stream=lambda s: contextlib.nullcontext(), synchronize=lambda device=None: None,
                                 CUDAGraph=Graph, graph=lambda g: contextlib.nullcontext())
    monkeypatch.setattr(vg.torch, "cuda", cuda)
    c = cache()
    feed(c, 70, 1)

    def forward(input_ids, past_key_values, **kw):
        for layer in range(2):
            past_key_values.update(*rows_of(input_ids.shape[1], 9), layer)
        return types.SimpleNamespace(logits=torch.zeros(1, input_ids.shape[1], 8))

    model = types.SimpleNamespace(model=types.SimpleNamespace(layers=[]))
    g = vg.VerifyGraph(model, c, q_len=4, device="cpu", forward=forward)
    g.capture(torch.zeros(1, 4, dtype=torch.long), torch.ones(1, 1, 4, 74, dtype=torch.bool),
              torch.zeros(1, 4, dtype=torch.long))
    return c, g


def test_a_graph_replays_over_the_cache_that_it_was_captured_over(captured):
    c, g = captured
    g.replay()
    feed(c, 4, 3)  # an eager pass, whose rows are written over, or taken back
    g.replay()
    c.crop(70)
    g.replay()
    assert g.graph.replays == 3


def test_a_pass_that_replaces_the_buffers_is_noticed(captured):
    c, g = captured
    feed(c, 50, 3)  # more rows than the tail holds
    c.crop(70)
    with pytest.raises(RuntimeError, match="laid out"):
        g.replay()
    assert g.graph.replays == 0


def test_a_cache_of_another_length_is_noticed(captured):
    c, g = captured
    c.crop(69)
    with pytest.raises(RuntimeError, match="laid out"):
        g.replay()
    c.crop(20)       # other rows, not sealed yet, up to the same length
    feed(c, 8, 4)
    feed(c, 8, 5)
    feed(c, 34, 6)
    assert c.get_seq_length() == 70
    with pytest.raises(RuntimeError, match="laid out"):
        g.replay()


def test_codes_that_were_replaced_are_noticed(captured):
    c, g = captured
    for n in range(8):
        feed(c, 30, n)
    c.crop(70)
    with pytest.raises(RuntimeError, match="laid out"):
        g.replay()


def test_a_graph_keeps_the_buffers_that_it_writes(captured):
    c, g = captured
    held = [weakref.ref(t) for layer in c.layers for t in (*layer._codes, layer._kt, layer._vt)]
    feed(c, 200, 3)
    feed(c, 1, 4)
    assert all(r() is not None for r in held)


def test_an_eviction_without_weights_says_so(plain):  # noqa: F811
    import warnings

    c = cache(budget=40, sinks=2, recent=8)
    feed(c, 90, 1)
    with pytest.warns(RuntimeWarning, match="weights"):
        assert c.evict() == 50
    c.reset()
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        for l in c.layers:  # as the lean forward appends
            l.begin(60)
            l.end(60)
        assert c.evict() == 20
