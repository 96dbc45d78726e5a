"""Several answers to one prompt on the host: forks of requests and compaction in the cache manager, draws under top-k and min-p, and
the engine and its entry points over them (plain operations on the CPU in the kernels' place)."""
from __future__ import annotations

import math
import random

import numpy as np
import pytest
import torch

from kernel_refs import PlainOps
from tiny_configs import random_ids
from tokenizer_amd.cache import CacheManager, OutOfPages
from tokenizer_amd.cli import ArgError, parse_args
from tokenizer_amd.engine import Engine, GenerateParams, Scheduler, SchedulerConfig, StepEntry, StopReason, generate, generate_answers, load_model
from tokenizer_amd.parts.spec import CacheNeed
from tokenizer_amd.sampling import Rng, SampleError, sample_filtered, sample_token, sample_with_uniform


# ------------------------------------------------------------------------------------------------ draws
def _draw(logits, temperature, top_k, top_p, min_p, uniform):
    """The definition, token by token, in whole weights."""
    order = sorted((i for i in range(len(logits)) if not math.isnan(logits[i])), key=lambda i: (-logits[i], i))
    top = logits[order[0]]
    share = [math.exp((logits[i] - top) / temperature) for i in order]
    weight = [round(s * 2 ** 44) for s in share]
    kept = min(top_k, len(order)) if top_k else len(order)
    if top_p < 1:
        total, run = sum(weight[:kept]), 0
        for at in range(kept):
            run += weight[at]
            if run >= max(1, math.ceil(top_p * float(total))):
                kept = at + 1
                break
    kept = max(1, min(kept, sum(s >= min_p for s in share)))
    total, run = sum(weight[:kept]), 0
    for at in range(kept):
        run += weight[at]
        if run > uniform * float(total):
            return order[at]
    raise AssertionError


@pytest.mark.parametrize("top_k", [0, 1, 3, 50, 10000])
@pytest.mark.parametrize("top_p", [1.0, 0.9, 0.25, 0.0])
@pytest.mark.parametrize("min_p", [0.0, 0.0625, 1.0])
def test_draws_by_the_definition(top_k, top_p, min_p):
    rng = np.random.default_rng(top_k + int(100 * top_p))
    for trial in range(6):
        logits = rng.normal(size=300).astype(np.float32) * 2
        if trial % 2:
            logits = np.round(logits * 4) / 4                   # many equal ones
        for uniform in (0.0, 0.3, 0.9990234375, float(np.float32(rng.random()))):
            temperature, p, m = (float(np.float32(v)) for v in (rng.uniform(0.3, 2), top_p, min_p))
            assert sample_filtered(logits, temperature, top_k, p, m, uniform) == _draw([float(v) for v in logits], temperature, top_k, p, m, uniform)


def test_draws_of_rows_with_nothing_to_weigh():
    inf, nan = float("inf"), float("nan")
    assert sample_filtered([nan, nan], 1.0, 3, 0.5, 0.1, 0.5) == 0
    assert sample_filtered([-inf, nan, -inf], 1.0, 3, 0.5, 0.1, 0.5) == 0
    assert sample_filtered([1.0, inf, inf, nan], 1.0, 3, 0.5, 0.1, 0.9) == 1
    assert sample_filtered([nan, -inf, 2.0, 2.0], 1.0, 0, 1.0, 0.5, 0.75) == 3
    assert sample_filtered([1.0, 5.0, 2.0], 0.0, 2, 0.5, 0.1, 0.9) == 1


def test_draws_without_filters_are_as_before():
    logits = np.random.default_rng(1).normal(size=500).astype(np.float32)
    for seed in range(20):
        a, b = Rng(seed), Rng(seed)
        assert sample_token(logits, 0.8, 0.9, a) == sample_with_uniform(logits, 0.8, 0.9, b.random_f32())


def test_bad_filters_are_refused():
    for top_k, min_p in ((-1, 0.0), (1.5, 0.0), (True, 0.0), (2 ** 31, 0.0), (0, -0.1), (0, 1.1), (0, float("nan")), (0, float("inf"))):
        with pytest.raises(SampleError):
            sample_token([1.0, 2.0], 1.0, 1.0, Rng(0), top_k, min_p)
        with pytest.raises(SampleError):
            from tokenizer_amd.engine.generate import validate
            validate(GenerateParams(top_k=top_k, min_p=min_p))


def test_command_line_flags():
    args = parse_args(["--model", "m", "--top-k", "40", "--min-p", "0.05", "--answers", "4", "hi"])
    assert (args["top_k"], args["min_p"], args["answers"]) == (40, 0.05, 4)
    for bad in (["--top-k", "-1"], ["--top-k", "x"], ["--min-p", "x"], ["--answers", "0"], ["--answers"]):
        with pytest.raises(ArgError):
            parse_args(bad)


# ------------------------------------------------------------------------------------------------ cache
FULL, WINDOW = CacheNeed(kind="full", n_kv_heads=2, head_dim=8), CacheNeed(kind="window", n_kv_heads=1, head_dim=8, window=20)


def _held(manager, rid, length):
    manager.add_request(rid)
    assert manager.reserve(rid, length + 5)
    manager.advance(rid, length)


@pytest.mark.parametrize("length", [0, 1, 15, 16, 17, 100])
def test_a_fork_shares_full_pages_and_has_its_own_last_one(length):
    manager = CacheManager([FULL, WINDOW], 40, 16, 4)
    _held(manager, "a", length)
    copies, (src, dst) = manager.fork("a", 7)
    assert (src, dst) == (manager.slot("a"), manager.slot(7)) and manager.seq_len(7) == length
    full, part = length // 16, length % 16 > 0
    assert len(copies) == 2 * part
    for g in range(2):
        mine, theirs = manager.table("a", g), manager.table(7, g)
        assert len(theirs) == full + part and theirs[:full] == mine[:full]
        if part:
            assert theirs[full] != mine[full] and (g, mine[full], theirs[full]) in copies
    manager.check_invariants()
    for rid in ("a", 7):                                        # both go on, each in pages of its own, and end in any order
        assert manager.reserve(rid, length + 40)
        manager.advance(rid, length + 40)
    manager.check_invariants()
    manager.release("a")
    manager.check_invariants()
    again, _ = manager.fork(7, "c")
    manager.release(7)
    manager.release("c")
    manager.check_invariants()
    assert all(g.allocator.free_count() == 40 for g in manager.groups)


def test_a_fork_without_room_changes_nothing():
    manager = CacheManager([FULL, WINDOW], 3, 16, 2)
    _held(manager, "a", 40)
    epoch = manager.epoch
    with pytest.raises(OutOfPages):
        manager.fork("a", "b")
    assert not manager.has_request("b") and manager.epoch == epoch
    manager.check_invariants()
    with pytest.raises(KeyError):
        manager.fork("x", "b")
    with pytest.raises(KeyError):
        manager.fork("a", "a")
    manager = CacheManager([FULL], 30, 16, 1)
    _held(manager, "a", 40)
    with pytest.raises(OutOfPages):
        manager.fork("a", "b")
    manager.check_invariants()


def test_tables_of_many_requests_at_once():
    manager = CacheManager([FULL, WINDOW], 60, 16, 6)
    for rid, length in ((3, 1), ("a", 100), (("b", 1), 55), (9, 0)):
        manager.add_request(rid)
        manager.reserve(rid, length)
        manager.advance(rid, length)
    for rids in ([3], ["a", 3, 9, ("b", 1)], [9], []):
        for group in range(2):
            got, want = manager.tables(rids, group), [manager.table(r, group) for r in rids]
            width = max([1] + [len(t) for t in want])
            assert got.dtype == np.int32 and got.shape == (len(rids), width)
            assert got.tolist() == [t + [-1] * (width - len(t)) for t in want]
    with pytest.raises(KeyError):
        manager.tables(["a", "none"], 0)


def test_the_epoch_tells_when_requests_come_go_or_take_pages():
    manager = CacheManager([FULL], 30, 16, 4, prefix_cache=True)
    seen = [manager.epoch]

    def changed(yes):
        assert (manager.epoch != seen[-1]) == yes
        seen.append(manager.epoch)

    _held(manager, "a", 40)
    changed(True)
    manager.reserve("a", 100)
    manager.advance("a", 90)
    changed(False)
    manager.fork("a", "b")
    changed(True)
    manager.publish("a", list(range(90)))
    changed(False)
    manager.add_request("c")
    changed(True)
    assert manager.attach_shared_prefix("c", list(range(90))) == 80
    changed(True)
    manager.detach("c")
    changed(True)
    manager.release("b")
    changed(True)


@pytest.mark.parametrize("seed", range(25))
def test_compaction_keeps_what_requests_hold(seed):
    rng = random.Random(seed)
    manager = CacheManager([FULL, CacheNeed(kind="full", n_kv_heads=1, head_dim=16)], 60, 16, 12, prefix_cache=True)
    # What every page holds, by group: a name each, written when a request takes the page.
    content = [dict() for _ in manager.groups]
    live, names = {}, iter(range(10 ** 6))

    def write(rid):
        for g in range(len(manager.groups)):
            table = manager.table(rid, g)
            for index, page in enumerate(table):
                if index >= len(live[rid][g]):
                    live[rid][g].append(next(names))
                    content[g][page] = live[rid][g][-1]

    def apply(moves):
        assert len({(g, d) for g, _, d in moves}) == len(moves) and not {(g, s) for g, s, _ in moves} & {(g, d) for g, _, d in moves}
        for g, src, dst in moves:
            content[g][dst] = content[g][src]

    def check():
        manager.check_invariants()
        for rid in live:
            for g in range(len(manager.groups)):
                assert [content[g][p] for p in manager.table(rid, g)] == live[rid][g]

    for turn in range(60):
        what = rng.choice(["add", "add", "end", "fork", "compact", "grow"])
        if what == "add" and len(live) < 10:
            rid, tokens = ("r", turn), [rng.choice([0, 1])] * 16 + [turn] * rng.randint(1, 90)
            manager.add_request(rid)
            live[rid] = [[] for _ in manager.groups]
            taken = manager.attach_shared_prefix(rid, tokens)
            for g in range(len(manager.groups)):
                live[rid][g] = [content[g][p] for p in manager.table(rid, g)]
            if not manager.reserve(rid, len(tokens)):
                manager.release(rid)
                del live[rid]
                continue
            write(rid)
            manager.advance(rid, len(tokens))
            manager.publish(rid, tokens)
            assert taken % 16 == 0
        elif what == "end" and live:
            rid = rng.choice(sorted(live))
            manager.release(rid)
            del live[rid]
        elif what == "fork" and live and len(live) < 10:
            rid, new = rng.choice(sorted(live)), ("f", turn)
            try:
                copies, _ = manager.fork(rid, new)
            except OutOfPages:
                continue
            apply(copies)
            live[new] = [list(held[:len(manager.table(new, g))]) for g, held in enumerate(live[rid])]
        elif what == "grow" and live:
            rid = rng.choice(sorted(live))
            length = manager.seq_len(rid) + rng.randint(1, 40)
            if manager.reserve(rid, length):
                write(rid)
                manager.advance(rid, length)
        elif what == "compact":
            apply(manager.compact())
            for g, group in enumerate(manager.groups):
                allocator = group.allocator
                used = allocator.live_count() + allocator.cached_count()
                assert all(p < used for rid in live for p in manager.table(rid, g))
            assert manager.compact() == []
        check()
    for rid in list(live):
        manager.release(rid)
    manager.check_invariants()


# ------------------------------------------------------------------------------------------------ engine
class AnswerOps(PlainOps):
    """The plain operations with those of this file's subject."""

    def copy_pages(self, pages, n_pages, widths, src, dst):
        at = 0
        for width in widths:
            plane = pages[:, at:at + n_pages * width].view(pages.shape[0], n_pages, width)
            plane[:, dst.long()] = plane[:, src.long()]
            at += n_pages * width
        return pages

    def sample_filtered(self, logits, temperature, top_k, top_p, min_p, uniform, out=None):
        got = torch.tensor([sample_filtered(row.float().numpy(), float(t), int(k), float(p), float(m), float(u))
                            for row, t, k, p, m, u in zip(logits, temperature, top_k, top_p, min_p, uniform)], dtype=torch.int32)
        return got if out is None else out.copy_(got)


def _engine(folder, **more):
    model = load_model(folder, "float32", "cpu", ops=AnswerOps())
    return Engine(model, **{**dict(num_pages=64, page_size=16, max_requests=8), **more})


def _alone(folder, prompt, params):
    return generate(_engine(folder), prompt, params)


@pytest.mark.parametrize("name", ["A", "B"])
@pytest.mark.parametrize("length", [1, 16, 37])
def test_forked_requests_go_on_as_if_each_had_run_the_prompt(model_folders, name, length):
    folder = model_folders[name]
    engine = _engine(folder)
    vocab = engine.model.vocab_size
    prompt, more = random_ids(vocab, length, 3), [random_ids(vocab, 21, 10 + i) for i in range(3)]
    engine.add_request("a")
    engine.step([StepEntry("a", prompt)])
    engine.fork_request("a", ["b", "c"])
    got = engine.step([StepEntry(r, t, list(range(21))) for r, t in zip("cab", more)])
    for at, tokens in enumerate(more):
        fresh = _engine(folder)
        fresh.add_request(0)
        fresh.step([StepEntry(0, prompt)])
        want = fresh.step([StepEntry(0, tokens, list(range(21)))])
        assert torch.allclose(got[21 * at:21 * at + 21], want, rtol=1e-5, atol=1e-5)
    for rid in "bac":
        engine.end_request(rid)
    engine.cache.check_invariants()


def test_a_request_is_no_fork_for_its_name(model_folders):
    # A fork that leaves by the cache, as a scheduler's requests do; the next request of that name is one of its own.
    engine = _engine(model_folders["A"])
    engine.add_request("a")
    engine.fork_request("a", ["b"])                       # (a request without a token, too)
    assert engine.cache.seq_len("b") == 0 and engine._family == {"a", "b"}
    engine.cache.release("b")
    engine.add_request("b")
    assert engine._family == {"a"}


def test_requests_go_on_behind_a_compaction(model_folders):
    engine, still = _engine(model_folders["A"]), _engine(model_folders["A"])
    vocab = engine.model.vocab_size
    for e in (engine, still):
        for r, length in enumerate((50, 33, 70)):
            e.add_request(r)
            e.step([StepEntry(r, random_ids(vocab, length, r))])
    engine.end_request(0)
    assert engine.compact_cache() > 0 and engine.compact_cache() == 0
    more = [StepEntry(r, random_ids(vocab, 5, 9 + r), [0, 4]) for r in (1, 2)]
    assert torch.equal(engine.step(more), still.step(more))


@pytest.mark.parametrize("params", [GenerateParams(max_tokens=12, temperature=0.9, seed=5), GenerateParams(max_tokens=9, temperature=1.2, top_k=8, seed=2),
                                    GenerateParams(max_tokens=7, temperature=0.7, top_p=0.9, min_p=0.02, seed=11), GenerateParams.greedy(6),
                                    GenerateParams(max_tokens=1, temperature=1.0, seed=3), GenerateParams(max_tokens=0)],
                         ids=["warm", "top-k", "min-p", "greedy", "one token", "none"])
def test_answers_are_those_of_single_requests(model_folders, params):
    import dataclasses
    folder = model_folders["A"]
    prompt = random_ids(_engine(folder).model.vocab_size, 23, 4)
    engine = _engine(folder)
    answers = generate_answers(engine, prompt, params, 5)
    for i, answer in enumerate(answers):
        want = _alone(folder, prompt, dataclasses.replace(params, seed=params.seed + i))
        assert (answer.tokens, answer.reason, answer.completion_tokens) == (want.tokens, want.reason, want.completion_tokens)
    assert len(engine.cache.requests) == 0
    engine.cache.check_invariants()
    one = generate_answers(engine.model, prompt, params, 1)      # a bare model gets an engine of its own
    assert one[0].tokens == answers[0].tokens


def test_answers_that_end_early_leave_the_others(model_folders):
    import dataclasses
    folder = model_folders["A"]
    vocab = _engine(folder).model.vocab_size
    prompt = random_ids(vocab, 20, 6)
    params = GenerateParams(max_tokens=25, temperature=3.0, seed=1, eos=list(range(0, vocab, 7)))
    answers = generate_answers(_engine(folder), prompt, params, 6)
    assert len({len(a.tokens) for a in answers}) > 1 and any(a.reason == StopReason.Eos for a in answers)
    for i, answer in enumerate(answers):
        want = _alone(folder, prompt, dataclasses.replace(params, seed=1 + i))
        assert (answer.tokens, answer.reason) == (want.tokens, want.reason)


def test_answers_refused_and_out_of_pages(model_folders):
    engine = _engine(model_folders["A"], num_pages=4)
    for bad in (dict(n=0), dict(prompt=[]), dict(prompt="text"), dict(params=GenerateParams(top_k=-1))):
        with pytest.raises(ValueError):
            generate_answers(engine, **{**dict(prompt=[1, 2], params=GenerateParams(max_tokens=2), n=2), **bad})
    with pytest.raises(OutOfPages):
        generate_answers(engine, random_ids(engine.model.vocab_size, 30, 1), GenerateParams(max_tokens=30, temperature=1.0), 4)
    assert len(engine.cache.requests) == 0
    engine.cache.check_invariants()


def test_scheduled_requests_draw_under_their_own_filters(model_folders):
    folder = model_folders["A"]
    engine = _engine(folder)
    vocab = engine.model.vocab_size
    scheduler = Scheduler(engine, SchedulerConfig(num_blocks=64, max_batch_size=4))
    asked = [GenerateParams(max_tokens=8, temperature=1.0, top_k=3, seed=1), GenerateParams(max_tokens=8, temperature=1.0, top_p=0.8, seed=2),
             GenerateParams.greedy(8), GenerateParams(max_tokens=8, temperature=1.5, min_p=0.1, seed=4)]
    ids = [scheduler.add_request(random_ids(vocab, 9 + i, i), p) for i, p in enumerate(asked)]
    results = scheduler.run()
    for i, (rid, p) in enumerate(zip(ids, asked)):
        assert results[rid].tokens == _alone(folder, random_ids(vocab, 9 + i, i), p).tokens


def test_graphs_of_steps_with_plans_are_bounded(model_folders, monkeypatch):
    # (Stand-ins for the graphs and for the plans: what is kept, what makes room and which steps run eagerly is decided on the host.)
    from types import SimpleNamespace
    from tokenizer_amd.engine import engine as of_engine
    monkeypatch.setattr(of_engine, "StepGraph", lambda engine, entries, bucket: SimpleNamespace(bucket=bucket, last_used=0))
    engine = _engine(model_folders["A"], shared_attention=True)
    engine.use_graphs = True
    engine.PLAN_GRAPHS, engine.PLAN_IDLE_STEPS = 3, 10
    for r in range(2):
        engine.add_request(r)
    entries = [StepEntry(r, [1], [0]) for r in range(2)]
    make = 0
    engine.sharing = lambda entries: {} if make is None else {(0, 2, 2, 16): SimpleNamespace(signature=make)}
    for make in (1, 2, 3, 2):
        assert engine._replays(entries) and engine._graph_for(entries) is not None
        engine.steps += 1
    assert engine.graphs_captured == 3 and engine.steps_replayed == 4
    make = 4                                                    # no room, and the oldest has been used three steps ago
    assert not engine._replays(entries) and engine._graph_for(entries) is None and len(engine.graphs) == 3
    for make in (None, 1, 2, 3):                                # steps without a plan are captured as ever, those that are kept are replayed
        assert engine._replays(entries) and engine._graph_for(entries) is not None
    assert len(engine.graphs) == 4 and engine.graphs_captured == 4
    engine.steps += 5
    make = 2
    assert engine._graph_for(entries) is not None
    engine.steps += 5
    make = 4                                                    # one that has idled long enough makes room: not the one used since
    assert engine._replays(entries) and engine._graph_for(entries) is not None
    kept = [key[2][0][1] for key in engine.graphs if len(key) > 2]
    assert len(kept) == 3 and 2 in kept and 4 in kept and any(len(key) == 2 for key in engine.graphs)
    make = 5
    assert engine._graph_for(entries) is not None               # (the other idle one)
    make = 6
    assert engine._graph_for(entries) is None and len(engine.graphs) == 4


@pytest.mark.parametrize("name", ["A", "B"])
@pytest.mark.parametrize("num_pages", [5, 6, 7, 9, 12])
@pytest.mark.parametrize("params", [GenerateParams(max_tokens=40, temperature=1.2, top_k=20, seed=3), GenerateParams(max_tokens=37, temperature=3.0, seed=1, eos=list(range(0, 64, 9))),
                                    GenerateParams.greedy(35)], ids=["top-k", "some end early", "greedy"])
def test_answers_wait_where_the_pool_runs_out(model_folders, name, num_pages, params):
    # Five answers hold up to sixteen pages together, one of them four: the newest wait until the others have ended, and lose nothing.
    import dataclasses
    folder = model_folders[name]
    prompt = random_ids(_engine(folder).model.vocab_size, 16, 8)
    engine = _engine(folder, num_pages=num_pages)
    forked = []
    inner = engine.fork_request
    engine.fork_request = lambda rid, new: (forked.append(len(new)), inner(rid, new))[1]
    answers = generate_answers(engine, prompt, params, 5)
    for i, answer in enumerate(answers):
        want = _alone(folder, prompt, dataclasses.replace(params, seed=params.seed + i))
        assert (answer.tokens, answer.text, answer.reason, answer.completion_tokens) == (want.tokens, want.text, want.reason, want.completion_tokens)
    assert params.eos or num_pages > 9 or len(forked) > 1
    assert len(engine.cache.requests) == 0
    engine.cache.check_invariants()
    assert all(g.allocator.free_count() == num_pages for g in engine.cache.groups)


def test_one_answer_that_the_pool_cannot_hold_is_out_of_pages(model_folders):
    engine = _engine(model_folders["A"], num_pages=3)
    with pytest.raises(OutOfPages):
        generate_answers(engine, random_ids(engine.model.vocab_size, 16, 8), GenerateParams(max_tokens=60, temperature=1.0), 3)
    assert len(engine.cache.requests) == 0
    engine.cache.check_invariants()


def test_forks_that_cannot_all_be_made_leave_everything_as_it_was(model_folders):
    # Not the requests alone: the prefixes that the pool keeps are still there too, and so are names that cannot be a request's.
    engine = _engine(model_folders["A"], num_pages=10, prefix_cache=True)
    vocab = engine.model.vocab_size
    kept = random_ids(vocab, 49, 1)
    engine.add_request("old")
    engine.step([StepEntry("old", kept)])
    engine.cache.publish("old", kept)
    engine.end_request("old")
    engine.add_request("a")
    engine.step([StepEntry("a", random_ids(vocab, 70, 2))])
    free, epoch = [g.allocator.available() for g in engine.cache.groups], engine.cache.epoch
    for bad, error in (([f"b{i}" for i in range(6)], OutOfPages), (["b", "c", "b"], KeyError), (["b", "a"], KeyError), (["b", []], TypeError),
                       (["b", "c", "d", "e", "f", "g", "h", "i"], OutOfPages)):
        with pytest.raises(error):
            engine.fork_request("a", bad)
        assert list(engine.cache.requests) == ["a"] and engine.cache.epoch == epoch
        assert [g.allocator.available() for g in engine.cache.groups] == free
        engine.cache.check_invariants()
    with pytest.raises(KeyError):
        engine.fork_request("none", ["b"])
    engine.add_request("again")
    assert engine.cache.attach_shared_prefix("again", kept) == 48
    engine.end_request("again")
    engine.fork_request("a", [f"b{i}" for i in range(5)])         # as many as there are pages for (the kept ones make room)
    assert len(engine.cache.requests) == 6
