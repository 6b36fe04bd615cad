"""Requests that branch: who holds which page, on the CPU. And which models hold their cache in 8 bits."""
import itertools
import random

import pytest
import torch

from pytriton_llama_amd.cache import RELEASED, CacheManager, CannotShare, OutOfPages, OutOfSlots
from pytriton_llama_amd.cache.storage import CacheStorage
from pytriton_llama_amd.config import EngineConfig, build_model
from pytriton_llama_amd.engine.llm import Engine
from pytriton_llama_amd.engine.request import Request, SamplingParams
from pytriton_llama_amd.engine.runner import ModelRunner
from pytriton_llama_amd.engine.scheduler import Scheduler
from pytriton_llama_amd.parts import StateSpec, paged_kv_spec
from tiny_configs import tiny

FULL = paged_kv_spec(2, 16)
WIN = paged_kv_spec(2, 16, window=10)
F8 = torch.float8_e4m3fn


def live(m, name, n):
    m.admit(name)
    m.append(name, n)


@pytest.mark.parametrize("n,shared,copied", [(1, 0, 1), (3, 0, 1), (4, 1, 0), (5, 1, 1), (8, 2, 0), (9, 2, 1), (None, 2, 1)])
def test_full_pages_are_shared_and_the_last_one_is_copied(n, shared, copied):
    m = CacheManager([FULL, FULL], page_size=4, num_pages=9, max_num_seqs=3)
    live(m, "a", 9)
    copies = m.fork("a", "b", n)
    a, b = m.block_table("a", 0), m.block_table("b", 0)
    assert b[:shared] == a[:shared] and len(b) == shared + copied
    assert copies == ([(0, a[shared], b[shared])] if copied else [])
    assert m.num_tokens["b"] == (9 if n is None else n) and m.slot_of["b"] != m.slot_of["a"]
    assert m.paged[0].pool.num_free == 9 - 3 - copied
    m.check()
    m.append("b", 6)                                   # into pages of its own
    assert set(m.block_table("b", 0)[shared:]).isdisjoint(a)
    m.check()
    m.free("a")
    assert all(m.paged[0].pool.is_held(p) for p in m.block_table("b", 0))
    m.check()
    m.free("b")
    assert m.paged[0].pool.num_free == 9
    m.check()


def test_a_fork_that_cannot_be_changes_nothing():
    m = CacheManager([FULL], page_size=4, num_pages=3, max_num_seqs=2)
    live(m, "a", 9)
    for n in (0, 10, -1):
        with pytest.raises(ValueError):
            m.fork("a", "b", n)
    with pytest.raises(OutOfPages):
        m.fork("a", "b")
    with pytest.raises(RuntimeError):
        m.fork("x", "b")
    with pytest.raises(RuntimeError):
        m.fork("a", "a", 4)
    m.check()
    assert not m.is_live("b") and m.num_free_slots == 1
    m.fork("a", "b", 8)
    with pytest.raises(OutOfSlots):
        m.fork("a", "c", 4)
    m.check()


def test_pages_that_a_window_has_left_behind():
    m = CacheManager([WIN], page_size=4, num_pages=12, max_num_seqs=4)
    live(m, "a", 30)
    m.release_behind_window("a")
    assert m.block_table("a", 0)[:5] == [RELEASED] * 5
    m.fork("a", "b")
    m.fork("a", "c", 29)                                # a query at 29 sees 20 .. 29: page 5 and on
    with pytest.raises(CannotShare):
        m.fork("a", "d", 28)                            # ... at 28 sees 19, on page 4
    m.check()
    for name in "abc":
        m.append(name, 9)
        m.release_behind_window(name)
        m.check()
    for name in "abc":
        m.free(name)
    assert m.paged[0].pool.num_free == 12


def test_state_is_that_of_all_tokens():
    m = CacheManager([FULL, StateSpec((3,))], page_size=4, num_pages=8, max_num_seqs=3)
    live(m, "a", 9)
    with pytest.raises(CannotShare):
        m.fork("a", "b", 8)
    m.fork("a", "b", 9)
    m.check()


@pytest.mark.parametrize("seed", range(6))
def test_random_orders(seed):
    rng = random.Random(seed)
    m = CacheManager([FULL, WIN], page_size=3, num_pages=[40, 25], max_num_seqs=7)
    names = iter(range(10 ** 6))
    for _ in range(400):
        alive = list(m.slot_of)
        what = rng.random()
        try:
            if what < 0.2 or not alive:
                n = next(names)
                m.admit(n)
                if m.can_append(n, 5):
                    m.append(n, rng.randint(1, 5))
                else:
                    m.free(n)
            elif what < 0.4 and m.num_tokens[alive[0]]:
                r = rng.choice([a for a in alive if m.num_tokens[a]])
                m.fork(r, next(names), rng.choice([None, rng.randint(1, m.num_tokens[r])]))
            elif what < 0.8:
                r, k = rng.choice(alive), rng.randint(1, 7)
                if m.can_append(r, k):
                    m.append(r, k)
                    m.release_behind_window(r)
            else:
                m.free(rng.choice(alive))
        except (OutOfSlots, OutOfPages, CannotShare):
            pass
        m.check()
    for r in list(m.slot_of):
        m.free(r)
    assert [g.pool.num_free for g in m.paged] == [40, 25]


def test_check_finds_a_page_held_without_being_shared():
    m = CacheManager([FULL], page_size=4, num_pages=8, max_num_seqs=3)
    live(m, "a", 8)
    live(m, "b", 4)
    m.paged[0].tables["b"][0] = m.paged[0].tables["a"][0]
    with pytest.raises(AssertionError):
        m.check()


def test_the_scheduler_runs_branches_and_preempts_them():
    m = CacheManager([FULL], page_size=4, num_pages=6, max_num_seqs=3)
    s = Scheduler(m, 3, 64, eos_token_ids=())
    a = Request("a", list(range(7)), SamplingParams(max_new_tokens=8))
    s.add(a)

    def step():
        plan = s.schedule()
        for e in plan.entries:
            if not m.is_live(e.request.id):
                m.admit(e.request.id)
            m.append(e.request.id, e.num_tokens)
        s.update(plan, {e.request.id: 1 for e in plan.entries if e.samples})
        m.check()
        return [(e.request.id, e.num_tokens) for e in plan.entries]
    assert step() == [("a", 7)]
    branches = [Request(n, a.prompt, a.params) for n in "bc"]
    for b in branches:
        m.fork("a", b.id, 6)
        b.num_computed = 6
    with pytest.raises(ValueError):
        s.adopt([Request("x", [1, 2], SamplingParams())])        # lives nowhere
    s.adopt(branches)
    assert m.paged[0].pool.num_free == 6 - 2 - 2
    assert step() == [("a", 1), ("b", 1), ("c", 1)]
    seen = set()
    while s.has_work:
        seen |= {r for r, _ in step()}
    assert seen == {"a", "b", "c"} and s.num_preemptions > 0
    assert all(len(r.output) == 8 for r in [a] + branches) and m.paged[0].pool.num_free == 6


# ---- which models hold their cache in 8 bits -----------------------------------------------------
def test_the_llama_cache_in_8_bits():
    cfg = EngineConfig(cache_dtype="fp8", max_num_seqs=4)
    assert cfg.cache_dtype == F8 and EngineConfig().cache_dtype is None and EngineConfig(cache_dtype=F8).cache_dtype == F8
    with pytest.raises(ValueError):
        EngineConfig(cache_dtype="int8")
    model = build_model(tiny("B")[0])
    assert model.cache_layers_in(None) == model.cache_layers
    layers = model.cache_layers_in(F8)
    assert [t.name for t in layers[0].tensors] == ["k", "v", "k_scale", "v_scale"] and len(set(layers)) == 1
    m = CacheManager(layers, 16, 5, 2)
    storage = CacheStorage(m, torch.bfloat16, "cpu")
    view = storage.view(1)
    assert view.k.shape == (5, 1, 16, 32) and view.k.dtype == F8 and view.k_scale.shape == (5, 1)
    assert view.v_scale.dtype == torch.float32
    assert CacheStorage.bytes_per_page(m, torch.bfloat16) == 3 * 2 * (16 * 32 + 4)
    plain = CacheManager(model.cache_layers, 16, 5, 2)
    assert CacheStorage.bytes_per_page(plain, torch.bfloat16) == 3 * 2 * 16 * 32 * 2


def other_models():
    import bimopel_configs
    import fogapel_configs
    import matusun_configs
    import rubasun_configs
    import senavik_configs
    import virusun_configs
    return [bimopel_configs, fogapel_configs, matusun_configs, rubasun_configs, senavik_configs, virusun_configs]


@pytest.mark.parametrize("module", other_models(), ids=lambda m: m.__name__)
def test_other_models_refuse(module):
    table = getattr(module, module.__name__.split("_")[0].upper())            # name -> (configuration, ...)
    model = build_model(next(iter(table.values()))[0])
    with pytest.raises(ValueError, match="engine's type only"):
        model.cache_layers_in(F8)


@pytest.mark.parametrize("samples", ["0", "-2"])
def test_the_command_line_refuses_no_samples(samples, capsys):
    from pytriton_llama_amd import cli
    with pytest.raises(SystemExit):
        cli.main(["--checkpoints_dir", "nowhere", "--samples", samples])
    assert "--samples" in capsys.readouterr().err


# ---- the runner's part ---------------------------------------------------------------------------
class Copies:
    """Stands for the device memory: what was asked for, or an error at the copy named ``fails``."""

    def __init__(self, fails=None):
        self.fails, self.pages, self.slots = fails, [], []

    def copy_pages(self, group, src, dst):
        if self.fails == "pages":
            raise OSError("no such kernel")
        self.pages += [(group, s, d) for s, d in zip(src, dst)]

    def copy_slot(self, src, dst):
        if self.fails == "slot":
            raise OSError("no such kernel")
        self.slots.append((src, dst))


def host_runner(manager, storage):
    r = object.__new__(ModelRunner)
    r.manager, r.storage = manager, storage
    return r


@pytest.mark.parametrize("fails", ["pages", "slot"])
def test_branches_whose_copies_fail_hold_nothing(fails):
    m = CacheManager([FULL], page_size=4, num_pages=8, max_num_seqs=4)
    live(m, "a", 6)
    with pytest.raises(OSError):
        host_runner(m, Copies(fails)).fork("a", ["b", "c"], 5)
    assert not m.is_live("b") and not m.is_live("c") and m.num_free_slots == 3 and m.paged[0].pool.num_free == 6
    m.check()


@pytest.mark.parametrize("cache_dtype", [None, F8])
def test_the_kernel_that_copies_pages_is_loaded_with_the_model(monkeypatch, cache_dtype):
    """Whatever the cache is held in: the first branch comes between two steps."""
    import types

    from pytriton_llama_amd import ops

    class Asked(Exception):
        pass

    def require(names):
        raise Asked(tuple(names))
    monkeypatch.setattr(ops.library, "require", require)
    model = types.SimpleNamespace(dtype=torch.bfloat16, device=torch.device("cuda"), kernel_libraries=lambda: ("norm",))
    with pytest.raises(Asked) as asked:
        ModelRunner(model, 16, 4, 2, cache_dtype=cache_dtype)
    assert "cache_f8" in asked.value.args[0] and ("attention_f8" in asked.value.args[0]) == (cache_dtype is not None)


# ---- the engine's part ---------------------------------------------------------------------------
class HostEngine(Engine):
    """The engine's requests, scheduler, cache manager and branches; a step is its book-keeping alone. ``computed``: how many rows
    each step computed of what request at what position; a token is a rule of what comes before it and the request's seed."""

    def __init__(self, specs=(FULL,), page=4, pages=400, seqs=8, budget=4096, eos=(), **more):
        self.scheduler = Scheduler(CacheManager(list(specs), page, pages, seqs), seqs, budget, eos_token_ids=eos, **more)
        self.manager, self.copies = self.scheduler.manager, Copies()
        self.runner = host_runner(self.manager, self.copies)
        self.requests, self._ids, self._inflight = {}, itertools.count(), None
        self.computed = []

    def add_request(self, prompt, params=None, request_id=None):
        rid = self._new_id()
        req = self.requests[rid] = Request(rid, prompt, params or SamplingParams())
        self.scheduler.add(req)
        return rid

    def step(self):
        plan, sampled = self.scheduler.schedule(), {}
        for e in plan.entries:
            r = e.request
            if not self.manager.is_live(r.id):
                self.manager.admit(r.id)
            assert self.manager.append(r.id, e.num_tokens) == e.start
            self.computed += [(r.id, p) for p in range(e.start, e.start + e.num_tokens)]
            if e.samples:
                sampled[r.id] = hash((tuple(r.tokens), r.params.seed)) % 1000
        for e in plan.entries:
            self.manager.release_behind_window(e.request.id)
        outs = self.scheduler.update(plan, sampled)
        for o in outs:
            if self.requests[o.request].params.logprobs:
                self.requests[o.request].output_logprobs.append(-1.0)
        self.manager.check()
        return outs

    def all_back(self):
        assert not self.has_work and not self.requests and self.manager.num_free_slots == self.manager.max_num_seqs
        assert all(g.pool.num_free == g.pool.num_pages for g in self.manager.paged)


def test_a_branch_without_log_probabilities_has_none_of_its_request():
    e = HostEngine()
    rid = e.add_request(range(9), SamplingParams(max_new_tokens=8, logprobs=True))
    for _ in range(3):
        e.step()
    with_them, without = e.fork(rid, [SamplingParams(max_new_tokens=6, logprobs=True), SamplingParams(max_new_tokens=6)], 2)
    reqs = [e.requests[r] for r in (rid, with_them, without)]
    while e.has_work:
        e.step()
    assert [len(r.output_logprobs) for r in reqs] == [8, 6, 0] and [len(r.output) for r in reqs] == [8, 6, 6]


def prompt_rows(e, length, but=None):
    """Rows computed at positions of the prompt that are before its last (not those of request ``but``)."""
    return sum(p < length - 1 for r, p in e.computed if r != but)


@pytest.mark.parametrize("count", [1, 6, 7, 8, 30])
def test_branches_beyond_the_places_keep_their_share(count):
    """Eight places, two of them taken: whatever the number of branches, the prompt is computed once."""
    e = HostEngine()
    other = e.add_request(range(5), SamplingParams(max_new_tokens=40))
    rid = e.add_request(range(101), SamplingParams(max_new_tokens=9))
    for _ in range(3):
        e.step()
    made = e.fork(rid, SamplingParams(max_new_tokens=9), count)
    reqs = [e.requests[r] for r in [rid] + made]
    assert sum(r.status == "running" for r in reqs[1:]) == min(count, 6)
    assert all(r.num_computed == reqs[0].num_computed for r in reqs)
    more = e.fork(made[-1], SamplingParams(max_new_tokens=5), 2, num_output=0)      # (of one that may itself be waiting)
    e.manager.check()
    e.abort(made[0])
    while e.has_work:
        e.step()
    assert prompt_rows(e, 101, but=other) == 100
    assert all(len(r.output) == 9 for r in reqs[:1] + reqs[2:]) and len(e.requests[other].output) == 40
    assert [len(e.requests[r].output) for r in more] == [5, 5]
    e.requests.clear()
    e.all_back()


def test_waiting_branches_give_way_to_whom_runs():
    """Too few pages for all that wait: running requests are not preempted for them, an earlier request that waits gets in, and
    the branches are computed from their tokens then."""
    e = HostEngine(pages=16, seqs=2)
    rid = e.add_request(range(22), SamplingParams(max_new_tokens=18))          # (6 pages, 10 at its end)
    e.step()
    made = e.fork(rid, SamplingParams(max_new_tokens=18), 6, num_output=0)     # (a page more each)
    assert [e.requests[r].status for r in made] == ["running"] + ["waiting"] * 5
    assert e.manager.paged[0].pool.num_free == 16 - 6 - 6
    late = e.add_request(range(3), SamplingParams(max_new_tokens=2))
    reqs = [e.requests[r] for r in [rid] + made + [late]]
    while reqs[0].status != "finished":
        e.step()
    assert reqs[0].num_preemptions == reqs[1].num_preemptions == 0
    while e.has_work:
        e.step()
    assert [len(r.output) for r in reqs] == [18] * 7 + [2]
    e.requests.clear()
    e.all_back()


def test_a_request_ahead_of_waiting_branches_gets_their_pages():
    e = HostEngine(pages=12, seqs=2)
    rid = e.add_request(range(10), SamplingParams(max_new_tokens=6))           # (3 pages; a page more for a branch)
    e.step()
    first = e.add_request(range(30), SamplingParams(max_new_tokens=4))         # (8 pages)
    made = e.fork(rid, SamplingParams(max_new_tokens=6), 6, num_output=0)
    for r in made[1:]:
        assert e.manager.is_parked(r)
    e.abort(made[0])
    reqs = [e.requests[r] for r in [rid, first] + made[1:]]
    e.step()
    assert reqs[1].status == "running" and not e.manager.is_parked(made[-1])
    while e.has_work:
        e.step()
    assert [len(r.output) for r in reqs] == [6, 4] + [6] * 5
    e.requests.clear()
    e.all_back()


def test_waiting_branches_keep_their_pages_where_those_would_not_do():
    e = HostEngine(pages=30, seqs=3)
    running = e.add_request(range(60), SamplingParams(max_new_tokens=20))      # (15 pages to begin with)
    rid = e.add_request(range(10), SamplingParams(max_new_tokens=20))          # (3)
    e.step()
    filler = e.add_request(range(4), SamplingParams(max_new_tokens=3))
    e.step()
    large = e.add_request(range(99), SamplingParams(max_new_tokens=2))         # (25: not while the others run)
    made = e.fork(rid, SamplingParams(max_new_tokens=20), 4, num_output=0)
    while e.requests[filler].status != "finished":
        e.step()
    for _ in range(3):
        e.step()
    assert e.requests[large].status == "waiting" and all(e.manager.is_parked(r) for r in made)
    reqs = [e.requests[r] for r in [running, rid, filler, large] + made]
    while e.has_work:
        e.step()
    assert [len(r.output) for r in reqs] == [20, 20, 3, 2] + [20] * 4
    e.requests.clear()
    e.all_back()


def test_parked_requests_of_the_manager():
    m = CacheManager([FULL], page_size=4, num_pages=9, max_num_seqs=1)
    live(m, "a", 9)
    with pytest.raises(OutOfSlots):
        m.fork("a", "b")
    m.fork("a", "b", parked=True)
    m.fork("b", "c", 8, parked=True)
    assert m.is_parked("b") and not m.is_live("b") and not m.is_parked("a") and not m.is_parked("x")
    m.check()
    with pytest.raises(OutOfSlots):
        m.admit("b")
    m.free("a")
    m.admit("b")
    assert m.is_live("b") and m.num_tokens["b"] == 9 and m.append("b", 2) == 9
    m.check()
    for name in "bc":
        m.free(name)
    assert m.paged[0].pool.num_free == 9
    with pytest.raises(RuntimeError):
        m.free("c")
    m.check()
    s = CacheManager([FULL, StateSpec((3,))], page_size=4, num_pages=8, max_num_seqs=3)
    live(s, "a", 9)
    with pytest.raises(CannotShare):
        s.fork("a", "b", parked=True)
    s.check()


@pytest.mark.parametrize("seed", range(8))
def test_branches_in_random_order(seed):
    """Requests come, branch and are aborted, with few places and too few pages for all: every page is held by whom it is counted
    for (checked after every step), all end with their tokens."""
    rng = random.Random(seed)
    e = HostEngine(page=rng.choice([1, 3, 8]), pages=60 if seed % 2 else 200, seqs=rng.randint(1, 5), budget=rng.choice([7, 64]), max_model_len=60)
    live_ones = {}
    for _ in range(300):
        act = rng.random()
        if act < 0.2 and len(live_ones) < 12:
            rid = e.add_request([rng.randrange(100) for _ in range(rng.randint(1, 30))], SamplingParams(max_new_tokens=rng.randint(1, 24)))
            live_ones[rid] = e.requests[rid]
        elif act < 0.4 and live_ones:
            r = live_ones[rng.choice(sorted(live_ones))]
            n = rng.randint(0, len(r.output))
            if r.status != "finished" and n < r.params.max_new_tokens and len(live_ones) < 20:
                for b in e.fork(r.id, count=rng.randint(1, 4), num_output=n):
                    live_ones[b] = e.requests[b]
        elif act < 0.5 and live_ones:
            rid = rng.choice(sorted(live_ones))
            e.abort(rid)
            del live_ones[rid]
        elif e.has_work:
            e.step()
        e.manager.check()
    while e.has_work:
        e.step()
    for r in live_ones.values():
        assert r.status == "finished" and len(r.output) == r.params.max_new_tokens
    e.requests.clear()
    e.all_back()


# ---- samples -------------------------------------------------------------------------------------
@pytest.mark.parametrize("new", [1, 7])
@pytest.mark.parametrize("count", [1, 2, 8, 9, 16, 40])
def test_samples_compute_a_prompt_once(count, new):
    e = HostEngine(pages=600)
    group = e.generate_samples([range(1000)], count, SamplingParams(max_new_tokens=new, seed=4))[0]
    assert prompt_rows(e, 1000) == 999
    assert [len(r.output) for r in group] == [new] * count and [r.params.seed for r in group] == [4 + i for i in range(count)]
    assert all(r.output == HostEngine(pages=600).generate([range(1000)], r.params)[0] for r in group[:3])
    e.all_back()


@pytest.mark.parametrize("prompts,count,seqs", [(64, 4, 64), (10, 3, 4), (5, 5, 1)])
def test_samples_of_many_prompts_compute_each_once(prompts, count, seqs):
    e = HostEngine(pages=4000, seqs=seqs)
    lengths = [17 + 3 * i for i in range(prompts)]
    groups = e.generate_samples([range(n) for n in lengths], count, SamplingParams(max_new_tokens=5, seed=1))
    firsts = {g[0].id: n for g, n in zip(groups, lengths)}
    owner = {r.id: g[0].id for g in groups for r in g}
    assert sum(p < firsts[owner[r]] - 1 for r, p in e.computed) == sum(n - 1 for n in lengths)
    assert all(len(g) == count and all(len(r.output) == 5 for r in g) for g in groups)
    e.all_back()


def test_samples_that_their_first_token_may_end():
    """Some prompts' first request ends with its first token, others not; too few pages for all that wait."""
    for eos in (range(0, 1000, 3), range(1000)):
        e = HostEngine(pages=14, seqs=2, eos=tuple(eos), budget=9)
        groups = e.generate_samples([range(n) for n in (1, 4, 21, 5, 30)], 4, SamplingParams(max_new_tokens=6, seed=3))
        for group in groups:
            for r in group:
                assert r.output == HostEngine(eos=tuple(eos)).generate([r.prompt], r.params)[0]
        e.all_back()


def test_samples_that_are_interrupted_hold_nothing_for_good():
    class Stop(Exception):
        pass
    for when in range(1, 6):
        e = HostEngine(pages=60, seqs=3)
        real, calls = e.step, []

        def step():
            calls.append(1)
            if len(calls) == when:
                raise Stop
            return real()
        e.step = step
        with pytest.raises(Stop):
            e.generate_samples([range(9), range(14), range(6), range(3)], 3, SamplingParams(max_new_tokens=2))
        e.step = real
        while e.has_work:
            e.step()
        assert not any(r.keeps_pages for r in e.requests.values())
        e.requests.clear()
        e.all_back()


@pytest.mark.parametrize("length", range(1, 25))
@pytest.mark.parametrize("specs", [(FULL, WIN), (FULL, StateSpec((3,))), (WIN, StateSpec((3,)))], ids=["window", "state", "both"])
def test_samples_of_models_that_only_go_on(specs, length):
    """A window may have passed by the page that holds the prompt's last token but one, and state cannot go back by a token: the
    branches are made before the prompt's last token."""
    e = HostEngine(specs=specs, seqs=5, budget=10)
    other = e.add_request(range(3), SamplingParams(max_new_tokens=30))
    group = e.generate_samples([range(length)], 4, SamplingParams(max_new_tokens=6, seed=2))[0]
    assert prompt_rows(e, length, but=other) == length - 1
    assert len(e.copies.slots) == (3 if length > 1 else 0)
    for r in group:
        assert r.output == HostEngine().generate([r.prompt], r.params)[0]
    while e.has_work:
        e.step()
    e.requests.clear()
    e.all_back()


def test_samples_with_state_beyond_the_places_compute_the_prompt_themselves():
    e = HostEngine(specs=(FULL, StateSpec((3,))), seqs=3)
    group = e.generate_samples([range(50)], 7, SamplingParams(max_new_tokens=4, seed=2))[0]
    assert prompt_rows(e, 50) == 49 * 5 and len(e.copies.slots) == 2
    for r in group:
        assert r.output == HostEngine().generate([r.prompt], r.params)[0]
    e.all_back()


def test_a_request_that_stops_is_let_alone():
    e = HostEngine(budget=4)
    a, b = e.add_request(range(7), SamplingParams(max_new_tokens=3)), e.add_request(range(5), SamplingParams(max_new_tokens=9))
    e.requests[a].stops_at = 6
    for _ in range(6):
        e.step()
    assert e.requests[a].num_computed == 6 and not e.requests[a].output and len(e.requests[b].output) > 2
    e.requests[a].stops_at = None
    reqs = [e.requests[a], e.requests[b]]
    while e.has_work:
        e.step()
    assert [len(r.output) for r in reqs] == [3, 9]


@pytest.mark.parametrize("then", ["abort", "preempt"])
def test_a_branch_whose_first_step_failed(then):
    """It was planned, the step did not run: it has its pages and no slot, and gives them back like any other."""
    e = HostEngine(pages=14, seqs=3)
    rid = e.add_request(range(10), SamplingParams(max_new_tokens=12))
    e.step()
    made = e.fork(rid, SamplingParams(max_new_tokens=12), 3, num_output=0)
    for r in made[:2]:
        e.abort(r)
    e.scheduler.schedule()                                   # (and an error in the step)
    branch = e.requests[made[2]]
    assert branch.status == "running" and e.manager.is_parked(branch.id)
    if then == "abort":
        e.abort(branch.id)
    else:
        e.manager.admit("filler")
        e.manager.append("filler", 4 * e.manager.paged[0].pool.num_free)
        while branch.num_preemptions == 0:
            e.step()
        assert not e.manager.holds(branch.id) or e.manager.num_tokens[branch.id] == branch.num_computed
        e.manager.free("filler")
    e.manager.check()
    first = e.requests[rid]
    while e.has_work:
        e.step()
    assert len(first.output) == 12 and (then == "abort" or len(branch.output) == 12)
    e.requests.clear()
    e.all_back()
