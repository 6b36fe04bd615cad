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
