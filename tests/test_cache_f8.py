"""What the faces of the 8-bit cache's kernels refuse before anything is launched (no GPU needed: a refusal comes first)."""
import os
import re

import pytest
import torch

from pytriton_llama_amd import ops
from pytriton_llama_amd.ops import cache_f8, library


@pytest.mark.parametrize("name", sorted(cache_f8._ENTRIES))
def test_entries_take_the_arguments_of_the_source(name):
    """ctypes passes what is too many as an int: the types that the faces state are those of the source."""
    lib, types = cache_f8._ENTRIES[name]
    with open(os.path.join(library.CSRC_DIR, lib + ".hip"), encoding="utf-8") as f:
        found = re.search(r'extern "C" int ' + name + r"\((.*?)\) \{", f.read(), re.S).group(1).split(",")
    kinds = ["p" if "*" in a or "hipStream_t" in a else {"long": "l", "float": "f", "int": "i"}[a.split()[0]] for a in found]
    assert "".join(kinds) == types


def test_tensors_on_the_host_are_refused():
    cache = torch.zeros(2, 1, 16, 64).to(ops.CACHE_F8)
    scale = torch.ones(2, 1)
    q = torch.zeros(1, 1, 64, dtype=torch.bfloat16)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ops.KernelError, match="GPU"):
        ops.rope_store_f8(q, q, q, i[:1], None, i[:1], cache, cache, scale, scale)
    with pytest.raises(ops.KernelError, match="GPU"):
        ops.attention_decode_f8(q, q, cache, cache, scale, scale, i, i[:1], i.view(2, 1), 1, 1.0)
    with pytest.raises(ops.KernelError, match="GPU"):
        ops.attention_generic_f8(q, q, cache, cache, scale, scale, i, i[:1], i.view(2, 1), i[:1], i[:1], 1.0)
    with pytest.raises(ops.KernelError, match="GPU"):
        ops.copy_pages([cache[None]], [0], [1])


def test_which_sizes_the_matrix_cores_take():
    fits = ops.attention_f8_fits
    for D in (32, 64, 96, 128):
        assert fits(torch.bfloat16, 32, 8, D, 16) and fits(torch.bfloat16, 40, 1, D, 64)
        assert not fits(torch.float32, 32, 8, D, 16) and not fits(torch.bfloat16, 32, 8, D, 8)
        assert not fits(torch.bfloat16, 32, 8, D, 24) and not fits(torch.bfloat16, 7, 2, D, 16)
    assert not fits(torch.bfloat16, 8, 8, 160, 16) and not fits(torch.bfloat16, 8, 8, 48, 16) and not fits(torch.bfloat16, 8, 0, 64, 16)


def test_the_plan_of_prompt_portions(monkeypatch):
    """Blocks of 128 rows where there are many, or some and many keys for each; a workgroup a block up to twice what runs at once."""
    from pytriton_llama_amd import ops
    from pytriton_llama_amd.ops import cache_f8
    monkeypatch.setattr(cache_f8, "compute_units", lambda device: 256)

    def plan(D, rows, keys, bound=False):
        return ops.attention_prefill_f8_plan("cuda", 32, D, -(-rows // 64), -(-rows // 128), keys, bound)

    assert plan(128, 2048, 2048) == (64, 32) and plan(128, 2048, 4096) == (128, 16) and plan(128, 1531, 7676) == (128, 12)
    assert plan(128, 1536, 2036) == (64, 24) and plan(128, 1531, 2531) == (128, 12)
    assert plan(128, 1024, 2024) == (64, 16) and plan(128, 1024, 5024) == (128, 8) and plan(128, 384, 100000) == (64, 6)
    assert plan(128, 8192, 8192) == (128, 16)
    assert plan(64, 2048, 5048) == (64, 32) and plan(64, 1024, 5024) == (128, 8) and plan(64, 2048, 2048) == (64, 32)
    assert plan(128, 1024, 8192, True) == (64, 16) and plan(128, 1152, 8192, True) == (128, 9) and plan(128, 1152, 4000, True) == (64, 18)
    assert plan(64, 2048, 100000, True) == (64, 32) and plan(64, 4096, 100000, True) == (128, 32)
    assert ops.attention_prefill_f8_plan("cuda", 1024, 64, 2, 1, 64) == (64, 2)


@pytest.mark.parametrize("D,need", [(64, 16), (48, 16), (12, 4), (8, 4), (10, 2), (33, 1)])
def test_a_layer_of_a_pool_begins_at_a_multiple_of_its_rows(D, need):
    """Pages of odd sizes: the layers of one pool begin where the pages before them end; what lies between rows is refused."""
    pool, scale = torch.zeros(3, 5, 1, 3, D).to(ops.CACHE_F8), torch.ones(3, 5, 1)
    for layer in range(3):
        pages, page_size, at = cache_f8._cache("a call", 1, D, pool[layer], pool[layer], scale[layer], scale[layer])
        assert (pages, page_size) == (5, 3) and at[0] == pool.data_ptr() + layer * 15 * D
    if need > 1:
        off = pool.flatten()[need // 2:need // 2 + 15 * D].view(5, 1, 3, D)
        with pytest.raises(ops.KernelError, match=f"{need}-byte"):
            cache_f8._cache("a call", 1, D, pool[0], off, scale[0], scale[0])


def test_layers_of_a_step_share_the_tickets_of_their_blocks(monkeypatch):
    """Made once, by the first layer whose blocks are cut, and as many as the call counts in; none where blocks stay whole."""
    import types

    from pytriton_llama_amd.parts import attention
    monkeypatch.setattr(cache_f8, "compute_units", lambda device: 256)
    calls = []
    monkeypatch.setattr(ops, "attention_prefill_f8", lambda *args, tickets=None, **more: calls.append((args, tickets)))

    def step(rows, pages, layers):
        calls.clear()
        lists = {w: (torch.zeros(-(-rows // w.block_rows), dtype=torch.int32),) * 2 for w in (attention.PORTIONS_64, attention.PORTIONS_128)}
        ctx = types.SimpleNamespace(num_decode_seqs=0, num_seqs=1, ctx_lens=[16 * pages], work=lists, lens_are_bounds=False, q_start=None,
                                    ctx_len=None)
        group = types.SimpleNamespace(block_table=torch.zeros(1, pages, dtype=torch.int32))
        for heads in layers:
            part = attention.PagedAttention(64, heads, 8, 64)
            codes, scales = torch.zeros(1, 8, 16, 64).to(ops.CACHE_F8), torch.zeros(1, 8)
            cache = types.SimpleNamespace(k=codes, v=codes, k_scale=scales, v_scale=scales, page_size=16)
            q = torch.zeros(rows, heads, 64, dtype=torch.bfloat16)
            part.attend(torch.empty_like(q), q, cache, ctx, group)
        return [t for _, t in calls]

    a, b, c = step(500, 200, (32, 32, 8))
    blocks = calls[0][0][9].numel()
    assert a is b is c and a.numel() == ops.TICKET * blocks * 32 and a.dtype == torch.int32 and not a.any()
    few, many = step(200, 200, (8, 64))[-2:]                 # (a later layer that needs more)
    assert few.numel() == ops.TICKET * 4 * 8 and many.numel() == ops.TICKET * 4 * 64
    assert step(500, 20, (32,)) == [None] and step(1500, 120, (32,)) == [None]


@pytest.mark.parametrize("heads", [1, 8, 32, 40])
@pytest.mark.parametrize("dim", [32, 64, 96, 128])
def test_parts_of_blocks_are_within_what_the_kernel_takes(monkeypatch, heads, dim):
    monkeypatch.setattr(cache_f8, "compute_units", lambda device: 256)
    for rows in (64, 128):
        for blocks in (1, 2, 5, 12, 13, 20, 64, 65):
            parts = cache_f8._cut_into("cuda", heads, dim, blocks, blocks, rows, 4096)
            assert 0 <= parts <= 4096 and (parts == 0 or blocks <= min(64, parts))
            assert cache_f8._cut_into("cuda", heads, dim, blocks, blocks, rows, 768) == 0
            assert cache_f8._cut_into("cuda", heads, dim, blocks, blocks + 1, rows, 4096) == 0
            n = ops.attention_prefill_f8_tickets("cuda", heads, dim, blocks, blocks, rows, 4096)
            assert n == (ops.TICKET * blocks * heads if parts else 0)


@pytest.mark.parametrize("heads,kv,dim,seqs", [(32, 8, 64, 8), (32, 8, 128, 64), (8, 1, 96, 300), (2, 2, 32, 1), (40, 2, 128, 5), (1024, 8, 64, 3)])
def test_the_workspace_of_every_call_is_within_what_is_said(monkeypatch, heads, kv, dim, seqs):
    """What the faces would make for calls of all numbers of blocks and sequences, by the sizes that they ask torch for."""
    monkeypatch.setattr(cache_f8, "compute_units", lambda device: 256)
    most = ops.attention_f8_workspace_bytes("cuda", heads, kv, dim, seqs)
    made = [0]
    real = torch.empty

    def empty(n, **more):
        made[0] = max(made[0], 4 * n)
        return real(1)
    monkeypatch.setattr(cache_f8, "_launch_stream", lambda *a: 0)
    monkeypatch.setattr(cache_f8, "_entry", lambda name: lambda *a: 0)
    monkeypatch.setattr(cache_f8.torch, "empty", empty)
    codes, scales = torch.zeros(1, kv, 16, dim).to(ops.CACHE_F8), torch.zeros(1, kv)
    i32 = lambda n: torch.zeros(n, dtype=torch.int32)   # noqa: E731
    for blocks in (1, 2, 3, 5, 8, 12, 13, 16, 20, 33, 64, 65):
        for rows in (64, 128):
            q = torch.zeros(1, heads, dim, dtype=torch.bfloat16)
            ops.attention_prefill_f8(q, q, codes, codes, scales, scales, i32(2), i32(1), i32(100).view(1, 100), i32(blocks), i32(blocks), 1.0,
                                     0, rows)
    for n in {1, seqs}:
        q = torch.zeros(n, heads, dim, dtype=torch.bfloat16)
        ops.attention_decode_f8(q, q, codes, codes, scales, scales, i32(n + 1), i32(n), i32(100 * n).view(n, 100), n, 1.0)
    assert 0 < made[0] <= most <= 2 * made[0]


def test_the_recorded_steps_pool_counts_the_parts_of_keys(monkeypatch):
    from pytriton_llama_amd.config import EngineConfig, build_model
    from pytriton_llama_amd.engine import llm
    from tiny_configs import tiny
    monkeypatch.setattr(cache_f8, "compute_units", lambda device: 256)
    model = build_model(tiny("B")[0])
    model.dtype = torch.bfloat16
    config = dict(dtype="bfloat16", device="cpu", page_size=16, max_num_seqs=4, max_model_len=4096, use_graphs=True)
    plain, eight = (llm.graph_pool_bytes(model, EngineConfig(**config, cache_dtype=c)) for c in (None, "fp8"))
    mixer = model.blocks[0].mixer
    assert eight - plain == ops.attention_f8_workspace_bytes("cpu", mixer.num_heads, mixer.num_kv_heads, mixer.head_dim, 4) > 0
    config["page_size"] = 8                                   # (the general kernel has no parts)
    assert llm.graph_pool_bytes(model, EngineConfig(**config, cache_dtype="fp8")) == llm.graph_pool_bytes(model, EngineConfig(**config))
    assert llm.graph_pool_bytes(model, EngineConfig(**{**config, "use_graphs": False}, cache_dtype="fp8")) == 0


@pytest.mark.parametrize("heads,dim,rows,keys,want", [
    (8, 64, 512, 6512, 64), (8, 64, 1024, 5024, 64), (8, 64, 2048, 8048, 64), (8, 128, 512, 6512, 64), (8, 128, 1024, 5024, 64),
    (16, 64, 512, 6512, 64), (16, 64, 1024, 5024, 64), (16, 64, 2048, 4048, 64), (16, 64, 2048, 8048, 128), (16, 128, 512, 6512, 64),
    (16, 128, 1024, 5024, 64), (16, 128, 2048, 4048, 64), (16, 128, 2048, 8048, 128), (32, 64, 512, 6512, 64), (32, 64, 2048, 8048, 128),
    (32, 128, 512, 6512, 128), (64, 64, 512, 6512, 128), (64, 64, 512, 1512, 64), (64, 128, 256, 3256, 64), (64, 128, 512, 6512, 128),
    (64, 128, 1024, 2024, 128)])
def test_the_plan_at_other_numbers_of_heads(monkeypatch, heads, dim, rows, keys, want):
    """The side that was the faster one, where they differ by more than a few parts in a hundred."""
    monkeypatch.setattr(cache_f8, "compute_units", lambda device: 256)
    assert ops.attention_prefill_f8_plan("cuda", heads, dim, -(-rows // 64), -(-rows // 128), keys)[0] == want
