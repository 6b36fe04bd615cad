"""Whole models over a cache that is held in 8 bits, and requests that branch, through the runner, the engine and the command
line. The oracle of a step reads what the cache holds after it: the plain model with those keys and values in the place of its
own, so that a step is checked without what earlier roundings did to the cache."""
import os
import subprocess
import sys

import pytest
import torch

import plain_llama
from engine_helpers import TOL, make_folder, random_sequences
from tiny_configs import tiny

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F8 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def folders(tmp_path_factory, gpu_device):
    return {n: make_folder(tmp_path_factory, n, seed=31)[0] for n in "ABC"}


def load(folder, dtype, page, pages, max_len=None, graphs=False, seqs=8, cache_dtype=F8):
    import pytriton_llama_amd  # noqa: F401
    from pytriton_llama_amd.config import build_model, read_config_json
    from pytriton_llama_amd.engine.runner import ModelRunner
    from pytriton_llama_amd.weights import load_weights
    model = build_model(read_config_json(folder))
    load_weights(model, folder, dtype, "cuda:0")
    model.make_decode_copies()
    return ModelRunner(model, page, pages, seqs, max_len, graphs, timed_library_products=False, cache_dtype=cache_dtype)


def held(runner, request, layer):
    """Keys and values [tokens, Hkv, D] that the cache holds of a request, float32 on the CPU."""
    view = runner.storage.view(layer)
    n, P = runner.manager.num_tokens[request], runner.manager.page_size
    pages = runner.manager.block_table(request, view.group)
    out = []
    for codes, scale in ((view.k, view.k_scale), (view.v, view.v_scale)):
        x = codes[pages].float() * scale[pages][:, :, None, None]
        out.append(x.transpose(1, 2).reshape(len(pages) * P, *x.shape[1::2])[:n].cpu())
    return out


def last_logits(runner, folder, request, tokens, monkeypatch, dtype):
    """The plain logits behind the last of ``tokens``, all of which are in the cache."""
    cfg, w = plain_llama.read_model_folder(folder)
    if dtype != torch.float32:
        w = {k: (v.to(dtype).float() if v.dim() == 2 else v) for k, v in w.items()}
    layers = iter(range(cfg["num_hidden_layers"]))
    real = plain_llama.causal_attention

    def attention(q, k, v, scale):
        k, v = held(runner, request, next(layers))
        return real(q, k, v, scale)
    with monkeypatch.context() as m:
        m.setattr(plain_llama, "causal_attention", attention)
        return plain_llama.forward(cfg, w, tokens)[-1]


@pytest.mark.parametrize("name,page,dtype,graphs", [
    ("A", 4, torch.float32, False), ("A", 16, torch.bfloat16, False), ("B", 16, torch.bfloat16, True), ("B", 32, torch.bfloat16, False),
    ("C", 8, torch.float32, False), ("C", 16, torch.bfloat16, True), ("C", 16, torch.float32, True)])
def test_steps(folders, monkeypatch, name, page, dtype, graphs):
    """Prompts whole and in portions, beside requests that decode, one after the other in one cache."""
    from pytriton_llama_amd.engine.batch import StepEntry
    folder = folders[name]
    runner = load(folder, dtype, page, 60, 256, graphs)
    V = tiny(name)[0]["vocab_size"]
    seqs = random_sequences(V, [37, 90, 21], seed=page)
    fed = dict.fromkeys(seqs, 0)
    steps = [[("r0", 30)], [("r0", 1), ("r1", 33)], [("r0", 1), ("r1", 50)], [("r1", 1), ("r0", 1), ("r2", 17)],
             [("r2", 1), ("r0", 1), ("r1", 1)], [("r1", 2), ("r0", 1)], [("r0", 1), ("r1", 1)]]
    for step in steps:
        entries = [StepEntry(r, seqs[r][fed[r]:fed[r] + n], [n - 1]) for r, n in step]
        logits = runner.step(entries).float().cpu()
        runner.manager.check()
        for row, (r, n) in enumerate(step):
            fed[r] += n
            want = last_logits(runner, folder, r, seqs[r][:fed[r]], monkeypatch, dtype)
            assert (logits[row] - want).abs().max() <= TOL[dtype] * want.abs().max(), (r, fed[r])
    for r in seqs:
        runner.end(r)
    runner.manager.check()


@pytest.mark.parametrize("dim", [64, 128])
def test_long_prompts_at_full_widths(tmp_path, gpu_device, monkeypatch, dim):
    """32 heads on 8, two layers: portions whose few blocks are cut along their keys, recorded and not, and decode steps with and
    without parts, one and several sequences."""
    from pytriton_llama_amd.engine.batch import StepEntry
    from pytriton_llama_amd.weights import write_random_model
    cfg = dict(tiny("A")[0], num_hidden_layers=2, hidden_size=512, num_attention_heads=32, num_key_value_heads=8, head_dim=dim,
               intermediate_size=512, max_position_embeddings=4096)
    folder = str(tmp_path)
    write_random_model(cfg, folder, seed=5, dtype=torch.float32, std=0.06)
    runner = load(folder, torch.bfloat16, 16, 420, 4096, True)
    seqs = random_sequences(256, [2813, 700, 40], seed=dim)
    fed = dict.fromkeys(seqs, 0)
    for step in [[("r0", 1400)], [("r0", 700)], [("r0", 700)], [("r0", 1)], [("r0", 1), ("r1", 600)], [("r2", 20), ("r0", 1), ("r1", 1)],
                 [("r0", 1), ("r1", 1), ("r2", 1)], [("r0", 1), ("r1", 1), ("r2", 1)], [("r0", 1)]]:
        entries = [StepEntry(r, seqs[r][fed[r]:fed[r] + n], [n - 1]) for r, n in step]
        logits = runner.step(entries).float().cpu()
        runner.manager.check()
        for r, n in step:
            fed[r] += n
        for row, (r, n) in enumerate(step):
            if r != "r0" or n > 1 or len(step) == 3:            # (the long one's plain form takes seconds)
                want = last_logits(runner, folder, r, seqs[r][:fed[r]], monkeypatch, torch.bfloat16)
                assert (logits[row] - want).abs().max() <= TOL[torch.bfloat16] * want.abs().max(), (r, fed[r])


def test_first_layer_holds_the_rounded_keys(folders):
    """The first layer's keys and values do not depend on the cache: what it holds is them, rounded."""
    from pytriton_llama_amd.engine.batch import StepEntry
    folder = folders["B"]
    runner = load(folder, torch.float32, 16, 10)
    cfg, w = plain_llama.read_model_folder(folder)
    toks = random_sequences(384, [43])["r0"]
    runner.step([StepEntry("r", toks[:40], [])])
    for t in toks[40:]:
        runner.step([StepEntry("r", [t], [])])
    h, _ = plain_llama.add_rms_norm(w["model.embed_tokens.weight"][torch.tensor(toks)], None, w["model.layers.0.input_layernorm.weight"],
                                    cfg["rms_norm_eps"])
    cos, sin = plain_llama.rope_cos_sin(plain_llama.rope_inv_freq(cfg), torch.arange(43))
    k = plain_llama.apply_rope((h @ w["model.layers.0.self_attn.k_proj.weight"].T).view(43, 1, 32), cos, sin)
    v = (h @ w["model.layers.0.self_attn.v_proj.weight"].T).view(43, 1, 32)
    for got, want in zip(held(runner, "r", 0), (k, v)):
        # half a step of e4m3, 2^-4 of the number or 2^-10 of the scale (at most 2^-17 of the block's largest number), twice where
        # a block's scale grew, and what float32 sums of 128 products differ by
        largest = want.abs().max()
        assert ((got - want).abs() <= 2.0 ** -4 * want.abs() + (2 * 2.0 ** -17 + 128 * 2.0 ** -22) * largest).all()


def test_recorded_steps_give_the_same_bits(folders):
    from pytriton_llama_amd.engine.batch import StepEntry
    runs = []
    for graphs in (False, True):
        runner = load(folders["C"], torch.bfloat16, 16, 40, 128, graphs)
        seqs = random_sequences(300, [50, 31, 9], seed=4)
        got = []
        for r, s in seqs.items():
            got.append(runner.step([StepEntry(r, s[:-6], [len(s) - 7])]).clone())
        for i in range(6, 0, -1):
            got.append(runner.step([StepEntry(r, [s[-i]], [0]) for r, s in seqs.items()]).clone())
        caches = [t.view(torch.uint8).clone() for t in runner.storage.paged_pools[0].values()]
        runs.append((got, caches))
    for a, b in zip(runs[0][1], runs[1][1]):
        assert torch.equal(a, b)
    for a, b in zip(runs[0][0][3:], runs[1][0][3:]):                 # (the decode steps)
        assert (a - b).abs().max() <= TOL[torch.bfloat16] * a.abs().max()


def engine(folder, dtype="float32", cache_dtype=None, graphs=True, seqs=8, pages=64, page=8, max_len=128, **more):
    from pytriton_llama_amd.config import EngineConfig
    from pytriton_llama_amd.engine import Engine
    return Engine(folder, EngineConfig(dtype=dtype, page_size=page, num_pages=pages, max_num_seqs=seqs, max_model_len=max_len,
                                       use_graphs=graphs, cache_dtype=cache_dtype, timed_library_products=False, **more))


@pytest.mark.parametrize("cache_dtype", [None, "float8_e4m3fn"])
@pytest.mark.parametrize("graphs", [False, True])
def test_samples_of_one_prompt(folders, cache_dtype, graphs):
    """Greedy samples are all the same; drawn ones are those of requests that draw the same numbers; the prompt is computed once."""
    from pytriton_llama_amd.engine import SamplingParams
    e = engine(folders["C"], cache_dtype=cache_dtype, graphs=graphs)
    prompts = list(random_sequences(300, [33, 8, 1, 17], seed=9).values())
    seen = []
    real = e.runner.step
    e.runner.step = lambda entries, feed=None: (seen.extend(len(x.tokens) for x in entries), real(entries, feed))[1]
    p = SamplingParams(temperature=0.0, max_new_tokens=7, ignore_eos=True, logprobs=True)
    groups = e.generate_samples(prompts, 2, p)
    assert sum(n for n in seen if n > 1) == 33 + 8 + 17          # (each prompt once)
    for prompt, group in zip(prompts, groups):
        alone = e.generate_requests([prompt], p)[0]
        for r in group:
            assert r.output == alone.output and len(r.output_logprobs) == 7 and r.finish_reason == "length"
    p = SamplingParams(temperature=0.8, top_p=0.95, max_new_tokens=9, seed=5, ignore_eos=True)
    groups = e.generate_samples(prompts, 3, p)
    for prompt, group in zip(prompts, groups):
        each = [SamplingParams(temperature=0.8, top_p=0.95, max_new_tokens=9, seed=5 + i, ignore_eos=True) for i in range(3)]
        assert [r.output for r in group] == e.generate([prompt] * 3, each)
        assert len({tuple(r.output) for r in group}) > 1
    assert [len(g) for g in e.generate_samples(prompts, 4, SamplingParams(max_new_tokens=1))] == [4] * 4
    e.runner.manager.check()
    assert not e.has_work and not e.requests and e.runner.manager.paged[0].pool.num_free == 64


@pytest.mark.parametrize("cache_dtype", [None, "float8_e4m3fn"])
@pytest.mark.parametrize("graphs", [False, True])
def test_branches_while_generating(folders, cache_dtype, graphs):
    """A request branches between steps, also a branch of a branch, with pages shared, and when there is no room."""
    from pytriton_llama_amd.engine import SamplingParams
    e = engine(folders["C"], cache_dtype=cache_dtype, graphs=graphs, seqs=4, pages=24)
    prompt = random_sequences(300, [27], seed=2)["r0"]
    greedy = SamplingParams(temperature=0.0, max_new_tokens=20, ignore_eos=True)
    want = e.generate([prompt], greedy)[0]
    rid = e.add_request(prompt, greedy)
    made = []
    for turn in range(6):
        e.step()
        e.runner.manager.check()
    made += e.fork(rid)                                          # goes on as the request does
    a = e.requests[rid]
    assert e.requests[made[0]].output == a.output
    assert e.runner.manager.block_table(made[0], 0)[:3] == e.runner.manager.block_table(rid, 0)[:3]
    made += e.fork(made[0], num_output=2)                        # two tokens back
    drawn = SamplingParams(temperature=1.0, top_p=1.0, max_new_tokens=20, seed=3, ignore_eos=True)
    made += e.fork(rid, [drawn, drawn], 2, num_output=0)         # five in all: no slot for the second
    with pytest.raises(ValueError):
        e.fork("nobody")
    with pytest.raises(ValueError):
        e.fork(rid, num_output=len(a.output) + 1)
    with pytest.raises(ValueError):
        e.fork(rid, SamplingParams(max_new_tokens=2), num_output=2)
    outs = {r: e.requests[r] for r in [rid] + made}
    while e.has_work:
        e.step()
        e.runner.manager.check()
    assert all(outs[r].output == want for r in [rid] + made[:2])
    assert outs[made[2]].output == outs[made[3]].output == e.generate([prompt], drawn)[0]
    for r in [rid] + made:
        e.requests.pop(r)
    assert e.runner.manager.paged[0].pool.num_free == 24


def test_log_probabilities_of_branches(folders):
    """One a token, those of the tokens they share as well; not where the request did not keep them."""
    import dataclasses
    from pytriton_llama_amd.engine import SamplingParams
    e = engine(folders["C"], cache_dtype="float8_e4m3fn", seqs=4, pages=40)
    prompt = random_sequences(300, [19], seed=4)["r0"]
    keeps = SamplingParams(temperature=0.0, max_new_tokens=9, ignore_eos=True, logprobs=True)
    drops = dataclasses.replace(keeps, logprobs=False)
    a, b = e.add_request(prompt, keeps), e.add_request(prompt, drops)
    for _ in range(4):
        e.step()
    n = len(e.requests[a].output)
    assert n > 2
    made = e.fork(a) + e.fork(b, keeps, num_output=0)
    with pytest.raises(ValueError):
        e.fork(b, keeps)
    reqs = {r: e.requests[r] for r in [a, b] + made}
    assert reqs[made[0]].output_logprobs == reqs[a].output_logprobs
    while e.has_work:
        e.step()
    assert [len(reqs[r].output_logprobs) for r in [a, b] + made] == [9, 0, 9, 9]
    assert reqs[made[0]].output == reqs[a].output == reqs[made[1]].output


@pytest.mark.parametrize("cache_dtype", [None, "float8_e4m3fn"])
@pytest.mark.parametrize("seed", range(3))
def test_branches_and_aborts_in_random_order(folders, cache_dtype, seed):
    """Requests come, branch and are aborted between steps, some under way, with too few pages for all: every page is held by whom it is
    counted for, and each ends with the tokens that it began with and as many as it was to have."""
    import random
    from pytriton_llama_amd.engine import SamplingParams
    rng = random.Random(seed)
    e = engine(folders["C"], cache_dtype=cache_dtype, graphs=True, seqs=5, pages=22)
    free = e.runner.manager.paged[0].pool.num_free
    live, began = {}, {}
    for turn in range(60):
        act = rng.random()
        if act < 0.25 and len(live) < 9:
            p = SamplingParams(temperature=1.0, max_new_tokens=rng.randint(1, 24), seed=rng.randint(0, 99), ignore_eos=True)
            rid = e.add_request([rng.randrange(300) for _ in range(rng.randint(1, 45))], p)
            live[rid], began[rid] = e.requests[rid], []
        elif act < 0.5 and live:
            rid = rng.choice(sorted(live))
            n = rng.randint(0, len(live[rid].output))
            if live[rid].status != "finished" and len(live) < 9 and n < live[rid].params.max_new_tokens:
                for b in e.fork(rid, count=rng.randint(1, 2), num_output=n):
                    live[b], began[b] = e.requests[b], live[rid].output[:n]
        elif act < 0.6 and live:
            rid = rng.choice(sorted(live))
            e.abort(rid)
            del live[rid]
        if e.has_work:
            e.step()
        e.runner.manager.check()
    while e.has_work:
        e.step()
        e.runner.manager.check()
    assert e.runner.manager.paged[0].pool.num_free == free
    for rid, r in live.items():
        assert r.status == "finished" and len(r.output) == r.params.max_new_tokens and r.output[:len(began[rid])] == began[rid]


def test_branches_are_preempted_like_others(folders):
    """Few pages: branches give way and are computed again; shared pages stay with who holds them."""
    from pytriton_llama_amd.engine import SamplingParams
    e = engine(folders["C"], cache_dtype="float8_e4m3fn", seqs=6, pages=13)
    prompt = random_sequences(300, [20], seed=6)["r0"]
    p = SamplingParams(temperature=0.9, max_new_tokens=25, seed=11, ignore_eos=True)
    group = e.generate_samples([prompt], 5, p)[0]
    e.runner.manager.check()
    assert e.scheduler.num_preemptions > 0 and all(len(r.output) == 25 for r in group)
    assert e.runner.manager.paged[0].pool.num_free == 13


def test_a_model_with_state_branches_at_its_end_only(tmp_path_factory, gpu_device):
    """State cannot go back: behind the whole of what is in the cache it is copied, otherwise the branch is computed anew."""
    import virusun_configs
    from pytriton_llama_amd.config import EngineConfig
    from pytriton_llama_amd.engine import Engine, SamplingParams
    cfg = next(iter(virusun_configs.VIRUSUN.values()))[0]
    e = Engine(cfg, EngineConfig(dtype="float32", page_size=8, num_pages=60, max_num_seqs=6, max_model_len=96, async_decode=False,
                                 timed_library_products=False), random_seed=3)
    assert e.runner.manager.states
    prompt = random_sequences(e.model.vocab_size, [19], seed=1)["r0"]
    p = SamplingParams(temperature=0.0, max_new_tokens=10, ignore_eos=True)
    want = e.generate([prompt], p)[0]
    rid = e.add_request(prompt, p)
    for _ in range(4):
        e.step()
    copies = []
    real = e.runner.storage.copy_slot
    e.runner.storage.copy_slot = lambda s, d: (copies.append((s, d)), real(s, d))[1]
    made = e.fork(rid) + e.fork(rid, num_output=1)
    assert len(copies) == 1 and e.requests[made[0]].status == "running" and e.requests[made[1]].status == "waiting"
    reqs = [e.requests[r] for r in [rid] + made]
    while e.has_work:
        e.step()
        e.runner.manager.check()
    assert [r.output for r in reqs] == [want] * 3


def test_samples_of_a_model_with_state(gpu_device):
    """With steps launched ahead and recorded, as by default: the prompt is computed once, its state copied for each branch; a
    request that branches while it decodes is a token further in its state than in its output, and its branches are computed anew."""
    import virusun_configs
    from pytriton_llama_amd.config import EngineConfig
    from pytriton_llama_amd.engine import Engine, SamplingParams
    cfg = next(iter(virusun_configs.VIRUSUN.values()))[0]
    e = Engine(cfg, EngineConfig(dtype="float32", page_size=8, num_pages=60, max_num_seqs=6, max_model_len=96,
                                 timed_library_products=False), random_seed=3)
    assert e.runner.manager.states
    copies, seen = [], []
    real_copy, real_step = e.runner.storage.copy_slot, e.runner.step
    e.runner.storage.copy_slot = lambda s, d: (copies.append((s, d)), real_copy(s, d))[1]
    e.runner.step = lambda entries, feed=None: (seen.extend(len(x.tokens) for x in entries), real_step(entries, feed))[1]
    prompts = list(random_sequences(e.model.vocab_size, [19, 2, 33, 1], seed=1).values())
    p = SamplingParams(temperature=0.0, max_new_tokens=8, ignore_eos=True)
    groups = e.generate_samples(prompts[:1], 4, p) + e.generate_samples(prompts[1:], 2, p)
    assert len(copies) == 3 + 2 and sum(n for n in seen if n > 1) == 18 + 32
    for prompt, group in zip(prompts, groups):
        want = e.generate([prompt], p)[0]
        assert all(r.output == want for r in group)
    want = e.generate(prompts[:1], p)[0]
    rid = e.add_request(prompts[0], p)
    for _ in range(4):
        e.step()
    reqs = [e.requests[r] for r in [rid] + e.fork(rid)]
    while e.has_work:
        e.step()
        e.runner.manager.check()
    assert [r.output for r in reqs] == [want] * 2


@pytest.mark.parametrize("cache_dtype", [None, "float8_e4m3fn"])
@pytest.mark.parametrize("graphs", [False, True])
def test_more_samples_than_places(folders, cache_dtype, graphs):
    """Branches that wait with their pages: the prompt is computed once, tokens are those of requests of their own."""
    from pytriton_llama_amd.engine import SamplingParams
    e = engine(folders["C"], cache_dtype=cache_dtype, graphs=graphs, seqs=3, pages=80)
    prompts = list(random_sequences(300, [37, 9], seed=9).values())
    seen = []
    real = e.runner.step
    e.runner.step = lambda entries, feed=None: (seen.extend(len(x.tokens) for x in entries), real(entries, feed))[1]
    for p in (SamplingParams(temperature=0.0, max_new_tokens=7, ignore_eos=True), SamplingParams(temperature=0.0, max_new_tokens=1)):
        seen.clear()
        groups = e.generate_samples(prompts, 8, p)
        assert sum(n for n in seen if n > 1) == 37 + 9
        for prompt, group in zip(prompts, groups):
            want = e.generate([prompt], p)[0]
            assert all(r.output == want for r in group) and len(group) == 8
    p = SamplingParams(temperature=0.9, max_new_tokens=9, seed=5, ignore_eos=True)
    for prompt, group in zip(prompts, e.generate_samples(prompts, 8, p)):
        each = [SamplingParams(temperature=0.9, max_new_tokens=9, seed=5 + i, ignore_eos=True) for i in range(8)]
        assert [r.output for r in group] == e.generate([prompt] * 8, each)
    e.runner.manager.check()
    assert not e.has_work and not e.requests and e.runner.manager.paged[0].pool.num_free == 80


def test_the_command_line(folders):
    prompt = random_sequences(300, [12], seed=8)["r0"]
    args = [sys.executable, os.path.join(ROOT, "cli.py"), "--checkpoints_dir", folders["C"], "--temperature", "0", "--max_gen_len", "6",
            "--max_seq_len", "64", "--max_gpu_num_blocks", "40", "--cache_dtype", "float8_e4m3fn", "--prompt_ids", ",".join(map(str, prompt))]
    one = subprocess.run(args, capture_output=True, text=True, timeout=110)
    assert one.returncode == 0, one.stderr[-2000:]
    three = subprocess.run(args + ["--samples", "3"], capture_output=True, text=True, timeout=110)
    assert three.returncode == 0, three.stderr[-2000:]
    lines = three.stdout.strip().splitlines()
    assert len(lines) == 3 and set(lines) == {one.stdout.strip()}
