"""Which leading pages the requests of a batch share, against a look at every pair of rows; no GPU."""
from __future__ import annotations

import itertools
import random

import numpy as np
import pytest
import torch

from tokenizer_amd.kernels.shared_prefix import SharedPrefixes, find_shared_runs


def _table(rows, width=None):
    width = width or max([1] + [len(r) for r in rows])
    return np.array([list(r) + [-1] * (width - len(r)) for r in rows], dtype=np.int32).reshape(len(rows), width)


def _checked(rows, positions, page_size, min_keys, width=None):
    table = _table(rows, width)
    order, runs, own = find_shared_runs(table, positions, page_size, min_keys)
    assert sorted(order) == list(range(len(rows)))
    place = {r: i for i, r in enumerate(order)}
    covered = {r: 0 for r in range(len(rows))}
    for run in runs:
        at = sorted(place[r] for r in run.rows)
        assert len(at) >= 2 and at == list(range(at[0], at[0] + len(at))) and [order[i] for i in at] == run.rows
        assert run.key_end - run.key_begin >= min_keys and run.key_begin % page_size == 0 and run.key_end % page_size == 0
        first = run.rows[0]
        for r in run.rows:
            assert covered[r] == run.key_begin                 # a row's runs follow each other from its first key on
            covered[r] = run.key_end
            assert run.key_end <= positions[r] + 1
            assert rows[r][:run.key_end // page_size] == rows[first][:run.key_end // page_size]
    assert [covered[r] for r in range(len(rows))] == own.tolist()
    return order, runs, own


def test_nothing_shared():
    _, runs, own = _checked([[0, 1], [2, 3], [4]], [31, 20, 3], 16, 16)
    assert runs == [] and own.tolist() == [0, 0, 0]


def test_no_rows_and_rows_without_keys():
    order, runs, own = find_shared_runs(np.zeros((0, 3), np.int32), np.zeros(0, np.int64), 16, 16)
    assert (order, runs, own.tolist()) == ([], [], [])
    _, runs, own = _checked([[3, 4], [3, 4], [3, 4]], [-1, -1, 14], 16, 16)
    assert runs == [] and own.tolist() == [0, 0, 0]


def test_all_share_and_the_last_page_is_not_full():
    _, runs, own = _checked([[5, 6, 7], [5, 6, 8], [5, 6, 7]], [40, 33, 46], 16, 16)
    assert [(sorted(r.rows), r.key_begin, r.key_end) for r in runs] == [([0, 1, 2], 0, 32)] and own.tolist() == [32, 32, 32]


def test_rows_that_are_all_alike_up_to_the_width():
    _, runs, own = _checked([[5, 6], [5, 6]], [31, 31], 16, 16)
    assert [(r.key_begin, r.key_end) for r in runs] == [(0, 32)] and own.tolist() == [32, 32]


def test_branches():
    rows = [[1, 2, 3, 10], [1, 2, 3, 11], [1, 2, 4, 12], [9, 2, 3, 13], [1, 2, 4, 14]]
    _, runs, own = _checked(rows, [63] * 5, 16, 16)
    found = {(tuple(sorted(r.rows)), r.key_begin, r.key_end) for r in runs}
    assert found == {((0, 1, 2, 4), 0, 32), ((0, 1), 32, 48), ((2, 4), 32, 48)}
    assert own.tolist() == [48, 48, 48, 0, 48]


def test_a_short_run_goes_to_the_runs_behind_it():
    rows = [[1, 2, 3, 4, 20], [1, 2, 3, 4, 21], [1, 30, 31, 32, 33]]
    _, runs, own = _checked(rows, [70, 70, 70], 16, 32)
    assert [(sorted(r.rows), r.key_begin, r.key_end) for r in runs] == [([0, 1], 0, 64)] and own.tolist() == [64, 64, 0]


def test_a_page_that_is_not_there_ends_what_is_shared():
    _, runs, own = _checked([[1, -1, 3], [1, -1, 3]], [47, 47], 16, 16)
    assert [(r.key_begin, r.key_end) for r in runs] == [(0, 16)] and own.tolist() == [16, 16]


@pytest.mark.parametrize("seed", range(30))
def test_any_batch(seed):
    rng = random.Random(seed)
    pool, rows = list(range(10 ** 4)), []
    rng.shuffle(pool)
    for _ in range(rng.randint(1, 25)):
        table = list(rng.choice(rows))[:rng.randint(0, 30)] if rows and rng.random() < 0.7 else []
        table += [pool.pop() for _ in range(rng.randint(1, 12))]
        rows.append(table)
    page = rng.choice([16, 32])
    positions = [rng.randint((len(t) - 1) * page, len(t) * page - 1) for t in rows]
    min_keys = rng.choice([16, 64, 100])
    order, runs, own = _checked(rows, positions, page, min_keys, width=max(len(t) for t in rows) + rng.randint(0, 2))
    # Whatever two rows share stands in runs of both, but for less than `min_keys` at its end.
    for a in range(len(rows)):
        for b in range(a):
            alike = 0
            while alike < min((positions[a] + 1) // page, (positions[b] + 1) // page) and rows[a][alike] == rows[b][alike]:
                alike += 1
            both = max([0] + [r.key_end for r in runs if a in r.rows and b in r.rows])
            assert both <= alike * page and alike * page - both < min_keys


@pytest.mark.parametrize("work", [-1, 10 ** 9])       # (with items of many columns, and without)
@pytest.mark.parametrize("seed", range(12))
def test_the_work_list_covers_every_query_and_key_once(seed, work, monkeypatch):
    monkeypatch.setattr(SharedPrefixes, "WIDE_WORK", work)
    rng = random.Random(100 + seed)
    group, n_kv, page = rng.choice([1, 3, 7, 40]), rng.choice([1, 2, 4]), 16
    shared = list(range(rng.randint(0, 90)))
    rows = [shared + list(range(1000 * (r + 1), 1000 * (r + 1) + rng.randint(1, 5))) for r in range(rng.randint(1, 40))]
    for r in rows[:len(rows) // 2]:
        r[len(shared):len(shared)] = list(range(500, 500 + 9))
    positions = [len(t) * page - 1 - rng.randint(0, page - 1) for t in rows]
    plan = SharedPrefixes(_table(rows), positions, page, group * n_kv, n_kv, 64, torch.bfloat16, "cpu")
    items = plan.items.reshape(-1, 8).tolist()
    order, by_row = plan.order_dev.tolist(), plan.own_of_row_dev.reshape(-1, 4).tolist()
    own, parts = [r[1] for r in by_row], [r[2] for r in by_row]
    assert [r[0] for r in by_row] == list(range(len(rows))) and plan.own_dev.reshape(-1, 4).tolist() == [by_row[r] for r in order]
    assert len(items) == plan.n_few + plan.n_many and order == plan.order and own == plan.own_begin.tolist()
    seen = {}                                               # (row, kv head, head in its group) -> {slot: (begin, end)}
    for at, (rows_at, columns, first, begin, end, slot, table_row, kv_head) in enumerate(items):
        if columns == 0:                                    # an item that only fills the list up
            continue
        assert table_row == order[rows_at]
        takes = plan.FEW_COLUMNS if at < plan.n_few else plan.WIDE_COLUMNS
        assert 0 <= first < columns and columns % group == 0 and rows_at + columns // group <= len(rows)
        assert begin < end <= plan.keys_end and begin % page == 0 and 0 <= kv_head < n_kv
        for column in range(first, min(columns, first + takes)):
            slots = seen.setdefault((order[rows_at + column // group], kv_head, column % group), {})
            assert slot not in slots
            slots[slot] = (begin, end)
    for row, head in itertools.product(range(len(rows)), range(group)):
        for kv_head in range(n_kv):
            slots = seen.get((row, kv_head, head), {})
            assert sorted(slots) == list(range(parts[row])) and parts[row] <= plan.shared_parts
            ranges = [slots[s] for s in sorted(slots)]
            assert [b for b, _ in ranges] + [own[row]] == [0] + [e for _, e in ranges] if ranges else own[row] == 0


def _own_parts(plan):
    """Per row its own keys' parts: (begin, slot, parts left), in order."""
    parts = {}
    for row, begin, slot, left in plan.own_items.reshape(-1, 4).tolist():
        if row >= 0:
            parts.setdefault(row, []).append((begin, slot, left))
    return parts


@pytest.mark.parametrize("fill", [False, True])
@pytest.mark.parametrize("growth", [0, 512, None])
@pytest.mark.parametrize("lengths,shared,n_kv,group", [([100] * 255 + [32000], 8192, 4, 7), ([300] * 63 + [32000], 4096, 2, 7), ([5], 0, 1, 1),
                                                       ([1, 700, 20, 4000], 640, 2, 40), ([40] * 300, 1024, 4, 4)])
def test_own_keys_fall_into_parts_by_each_rows_own_length(lengths, shared, n_kv, group, growth, fill):
    # A long request among many short ones is many parts, and the short ones are no more than they need.
    rows, used = [], shared // 16
    for at, length in enumerate(lengths):
        pages = -(-length // 16)
        alone = at == len(lengths) - 1
        rows.append(([] if alone else list(range(shared // 16))) + list(range(used, used + pages)))
        used += pages
    positions = [len(r) * 16 - 1 for r in rows]
    plan = SharedPrefixes(_table(rows), positions, 16, n_kv * group, n_kv, 64, torch.bfloat16, "cpu", fill, growth)
    own_keys, by_row, parts = int(plan.own_keys_dev), plan.own_of_row_dev.reshape(-1, 4).tolist(), _own_parts(plan)
    reach = [-(-(max(positions) + 1 if growth is None else p + 1 + growth) // 512) * 512 for p in positions]
    assert sorted(parts) == list(range(len(rows))) and plan.n_own % (64 if fill else 1) == 0 and len(plan.own_items) == 4 * plan.n_own
    for row, held in parts.items():
        begins, slots, left = zip(*held)
        assert by_row[row][1:] == [begins[0], slots[0], len(held)] and begins[0] == plan.own_begin[row]
        assert list(begins) == [begins[0] + i * own_keys for i in range(len(held))]
        assert list(slots) == [by_row[row][2] + i for i in range(len(held))] and slots[-1] < plan.slots
        assert list(left) == list(range(len(held), 0, -1))
        assert len(held) * own_keys >= reach[row] - begins[0] > (len(held) - 1) * own_keys or len(held) == 1
    # About as many parts as there are workgroups to be had, and none that holds the others up.
    work = sum(reach[r] - b for r, b in enumerate(plan.own_begin.tolist())) * n_kv * -(-group // 16)
    assert own_keys >= 128 and own_keys % 32 == 0 and own_keys <= max(128, 2 * work // 1024 + 32, -(-max(r - b for r, b in zip(reach, plan.own_begin.tolist())) // 64) + 31)
    if growth is not None and max(lengths) == 32000:
        assert own_keys <= 1280 and len(parts[len(rows) - 1]) >= 25


def test_parts_are_planned_for_the_growth_that_is_named():
    rows = [list(range(10)) + [100 + r] for r in range(4)]
    table, positions = _table(rows), [170] * 4
    plans = [SharedPrefixes(table, positions, 16, 14, 2, 64, torch.bfloat16, "cpu", 0, more) for more in (0, 341, 342, 3800, None)]
    assert [len(_own_parts(p)[0]) for p in plans] == [3, 3, 7, 31, 3]


def test_a_row_has_no_more_parts_than_a_wave_joins_at_a_time():
    rows = [list(range(256)) + [10000 + r] for r in range(7)] + [list(range(20000, 22000))]
    plan = SharedPrefixes(_table(rows), [4100] * 7 + [31999], 16, 14, 2, 64, torch.bfloat16, "cpu", 0, 512)
    assert [len(p) for _, p in sorted(_own_parts(plan).items())] == [2] * 7 + [64]


@pytest.mark.parametrize("n_q,n_kv,d", [(14, 2, 64), (28, 4, 128)])
def test_plans_of_many_prompts_have_few_makes(n_q, n_kv, d):
    # Captured steps are kept by a plan's make.  Eight answers to each of a hundred prompts of any length, ending one by one: there are not many
    # more makes than there are counts of requests and buckets of 512 tokens of context.
    rng = random.Random(1)
    makes, plain = set(), set()
    for _ in range(100):
        length, produced, live = rng.randint(64, 8000), 0, 8
        for end in sorted(rng.randint(1, 400) for _ in range(8)):
            while produced < end and live > 1:
                bucket = -(-(length + produced + 1) // 512) * 512
                shared = length // 16
                own = -(-(length + produced + 1) // 16) - shared
                rows = [list(range(shared)) + list(range(1000 * (r + 1), 1000 * (r + 1) + own)) for r in range(live)]
                plan = SharedPrefixes(_table(rows), [length + produced] * live, 16, n_q, n_kv, d, torch.bfloat16, "cpu", True, 512)
                makes.add((live, bucket, plan.signature if plan.runs else None))
                plain.add((live, bucket))
                produced = min(end, bucket - length)
            live -= 1
    assert len(makes) <= 1.75 * len(plain)


@pytest.mark.parametrize("rows,keys,n_q,n_kv,d,dtype,pays", [
    (2, 256, 14, 2, 64, torch.bfloat16, False), (2, 4096, 14, 2, 64, torch.bfloat16, False), (8, 1024, 14, 2, 64, torch.bfloat16, False),
    (16, 4096, 14, 2, 64, torch.bfloat16, True), (64, 2048, 14, 2, 64, torch.bfloat16, True), (128, 512, 14, 2, 64, torch.bfloat16, False),
    (4, 4096, 28, 4, 128, torch.bfloat16, True), (64, 512, 28, 4, 128, torch.bfloat16, False), (64, 1024, 28, 4, 128, torch.bfloat16, True),
    (4, 1024, 14, 2, 64, torch.float32, False), (64, 512, 14, 2, 64, torch.float32, True)])
def test_plans_say_whether_they_are_faster_than_none(rows, keys, n_q, n_kv, d, dtype, pays):
    table = _table([list(range(keys // 16)) + [10000 + 3 * r + i for i in range(3)] for r in range(rows)])
    assert SharedPrefixes(table, [keys + 40] * rows, 16, n_q, n_kv, d, dtype, "cpu").pays == pays
    assert not SharedPrefixes(np.arange(rows * 3, dtype=np.int32).reshape(rows, 3), [40] * rows, 16, n_q, n_kv, d, dtype, "cpu").pays
