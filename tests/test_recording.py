"""What happens around the recording of a step, with stand-ins for the GPU's part (CPU)."""
import contextlib
import gc
import types

import pytest
import torch

from pytriton_llama_amd.engine import graphs


@pytest.fixture
def no_gpu(monkeypatch):
    stream = types.SimpleNamespace(wait_stream=lambda other: None)
    monkeypatch.setattr(torch.cuda, "Stream", lambda device=None: stream)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda: stream)
    monkeypatch.setattr(torch.cuda, "stream", lambda s: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "synchronize", lambda: None)
    monkeypatch.setattr(torch.cuda, "CUDAGraph", lambda: "graph")
    monkeypatch.setattr(torch.cuda, "graph", lambda graph, pool=None: contextlib.nullcontext())
    monkeypatch.setattr(graphs.ops, "timed_library_products", lambda on: contextlib.nullcontext())


@pytest.mark.parametrize("collects", [True, False])
@pytest.mark.parametrize("fails", [True, False])
def test_no_garbage_is_collected_while_a_step_is_recorded(no_gpu, collects, fails):
    """A cycle with an engine's graphs in it, dropped before, must not be taken apart then; afterwards all is as it was."""
    seen = []

    def forward(ctx, storage):
        seen.append(gc.isenabled())
        if fails and len(seen) == 2:
            raise RuntimeError("a kernel refuses")
        return "logits"
    before = gc.isenabled()
    try:
        (gc.enable if collects else gc.disable)()
        if fails:
            with pytest.raises(RuntimeError, match="refuses"):
                graphs.capture_forward(types.SimpleNamespace(forward=forward), None, None, "cuda:0")
        else:
            assert graphs.capture_forward(types.SimpleNamespace(forward=forward), None, None, "cuda:0") == ("graph", "logits")
        assert seen == [collects, False] and gc.isenabled() == collects
    finally:
        (gc.enable if before else gc.disable)()


@pytest.mark.parametrize("inference", [True, False])
def test_a_recording_begins_and_ends_outside_of_inference_mode(no_gpu, monkeypatch, inference):
    """What torch makes for all recordings of a process is made as the first begins; the step itself runs as its caller does."""
    seen = []

    @contextlib.contextmanager
    def recording(graph, pool=None):
        seen.append(("begin", torch.is_inference_mode_enabled()))
        yield
        seen.append(("end", torch.is_inference_mode_enabled()))
    monkeypatch.setattr(torch.cuda, "graph", recording)
    model = types.SimpleNamespace(forward=lambda ctx, storage: seen.append(("forward", torch.is_inference_mode_enabled())))
    with torch.inference_mode(inference):
        graphs.capture_forward(model, None, None, "cuda:0")
        assert torch.is_inference_mode_enabled() == inference
    assert seen == [("forward", inference), ("begin", False), ("forward", inference), ("end", False)]


OWN_GRAPH = """
import sys, torch
sys.path[:0] = ["tests", "."]
from tiny_configs import tiny
from pytriton_llama_amd.config import EngineConfig
from pytriton_llama_amd.engine import Engine, SamplingParams
e = Engine(tiny("B")[0], EngineConfig(dtype="bfloat16", page_size=16, num_pages=16, max_num_seqs=2, max_model_len=64, use_graphs=True),
           random_seed=1)
want = e.generate([[1, 2, 3]], SamplingParams(temperature=0.0, max_new_tokens=4))
x, graph = torch.zeros(8, device="cuda"), torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y = x + 1
for i in range(3):
    x.fill_(i)
    graph.replay()
    assert y.tolist() == [i + 1.0] * 8
    assert e.generate([[1, 2, 3]], SamplingParams(temperature=0.0, max_new_tokens=4)) == want
print("recorded")
"""


@pytest.mark.gpu
def test_a_program_records_a_graph_of_its_own_behind_an_engine():
    import os
    import subprocess
    import sys
    run = subprocess.run([sys.executable, "-c", OWN_GRAPH], cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                         capture_output=True, text=True, timeout=110)
    assert run.returncode == 0 and "recorded" in run.stdout, run.stderr[-2000:]
