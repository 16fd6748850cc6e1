"""Captures and the garbage collector: conftest.py's captures_without_collections.

No GPU: what a capture does on one is replaced.
"""
import gc

import pytest
import torch

import gpipes
from test_bert_ffn_gpu import capture_error


@pytest.fixture
def recorded(monkeypatch):
    """Graphs that write down whether a capture was open when they ended."""
    seen = {"open": False, "ended": []}

    class Graph:
        def capture_begin(self, *args, **kw):
            seen["open"] = True

        def capture_end(self):
            seen["open"] = False

        def __del__(self):
            seen["ended"].append(seen["open"])

    class OnStream:
        def __enter__(self):
            return self

        def __exit__(self, *args):
            return None

    monkeypatch.setattr(torch.cuda, "CUDAGraph", Graph)
    monkeypatch.setattr(torch.cuda, "stream", lambda s: OnStream())
    monkeypatch.setattr(torch.cuda, "synchronize", lambda *args: None)
    monkeypatch.setattr(torch.cuda, "empty_cache", lambda: None)
    if hasattr(torch._C, "_host_emptyCache"):
        monkeypatch.setattr(torch._C, "_host_emptyCache", lambda: None)
    monkeypatch.setattr(torch.cuda.graph, "default_capture_stream", object())
    return seen


def refused():
    raise gpipes.GpipesError(-1, "cannot be captured")


def test_a_graph_in_a_cycle_ends_outside_of_the_next_capture(recorded):
    """An error that is kept holds the frames it came through, and one of them holds the error and the graph."""
    gc.disable()
    try:
        err = capture_error(refused)
        assert isinstance(err, gpipes.GpipesError)
        del err
        assert recorded["ended"] == []  # the cycle keeps it
    finally:
        gc.enable()
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        many = [[i] for i in range(200000)]  # enough for the collector to run over what is young, and a while ago was
    assert len(many) == 200000 and recorded["ended"][0] is False


def test_the_collector_runs_again_after_a_capture(recorded):
    for error in (None, ValueError):
        try:
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                assert not gc.isenabled()
                if error:
                    raise error
        except ValueError:
            pass
        assert gc.isenabled()
    gc.disable()
    try:
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            pass
        assert not gc.isenabled()
    finally:
        gc.enable()
