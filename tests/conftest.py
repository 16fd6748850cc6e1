import gc
import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
for p in (ROOT, os.path.join(ROOT, "gpu-pipes_amd")):
    if p not in sys.path:
        sys.path.insert(0, p)

GOLDEN = os.path.join(ROOT, "tests", "golden")


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a gfx950 GPU (runs on the MI355X box)")


@pytest.fixture(scope="session")
def cuda():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no GPU visible")
    return torch.device("cuda:0")


@pytest.fixture(scope="session", autouse=True)
def captures_without_collections():
    """torch waits for the device when a CUDAGraph object ends; while a stream is being captured that is an error,
    and one in a destructor ends the process.  A test that keeps the error of a refused capture leaves its graph in a
    cycle (error, traceback, frame), and such a graph ends when the collector runs, which can be inside the next
    capture: so garbage is collected before a capture begins, and not during it."""
    import torch
    graph = torch.cuda.graph
    enter, leave = graph.__enter__, graph.__exit__
    was = []  # of the captures that are open: whether the collector was on

    def begin(self):
        gc.collect()
        was.append(gc.isenabled())
        gc.disable()
        try:
            return enter(self)
        except BaseException:
            end()
            raise

    def end():
        if was.pop():
            gc.enable()

    def finish(self, *args):
        try:
            return leave(self, *args)
        finally:
            end()

    graph.__enter__, graph.__exit__ = begin, finish
    yield
    graph.__enter__, graph.__exit__ = enter, leave


def bf16_to_f32(bits):
    """uint16 bfloat16 bit patterns -> float32 values (exact: the upper half of the float)."""
    import numpy as np
    return (np.asarray(bits, dtype=np.uint16).astype(np.uint32) << 16).view(np.float32)


def load_golden(name):
    import numpy as np
    with np.load(os.path.join(GOLDEN, name), allow_pickle=False) as z:
        return {k: z[k] for k in z.files}
