"""The kernels behind several answers to one prompt, each against a plain computation in 64 bits: draws under temperature, top-k,
top-p and min-p, copied pages, attention of single tokens behind shared prefixes."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from tokenizer_amd.kernels import KernelError
from tokenizer_amd.kernels.shared_prefix import SharedPrefixes

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16]


@pytest.fixture(scope="module")
def ops():
    from tokenizer_amd.kernels import get_ops
    return get_ops()


# ------------------------------------------------------------------------------------------------ draws
UNIT = 2.0 ** 44


def draw_of(logits, temperature, top_k, top_p, min_p, uniform) -> int:
    """One row's draw, token by token, in whole weights (`logits` as 64-bit numbers)."""
    numbers = np.nonzero(logits == logits)[0]
    if numbers.size == 0 or logits[numbers].max() == -np.inf:
        return 0
    top = logits[numbers].max()
    if not temperature > 0 or top == np.inf:
        return int(numbers[np.nonzero(logits[numbers] == top)[0][0]])
    order = numbers[np.lexsort((numbers, -logits[numbers]))]
    share = np.exp((logits[order] - top) / np.float64(temperature))
    weight = [int(w) for w in np.rint(share * UNIT)]
    kept = len(order) if top_k <= 0 else min(int(top_k), len(order))
    total = sum(weight[:kept])
    if top_p < 1.0:
        run = 0
        for at in range(kept):
            run += weight[at]
            if run >= max(1, math.ceil(max(np.float64(top_p), 0.0) * np.float64(total))):
                kept = at + 1
                break
    kept = max(1, min(kept, int(np.sum(share >= np.float64(min_p)))))
    total, run = sum(weight[:kept]), 0
    for at in range(kept):
        run += weight[at]
        if run > np.float64(uniform) * np.float64(total):
            return int(order[at])
    return int(order[max(at for at in range(kept) if weight[at])])


def settings(rows, **given):
    made = dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, uniform=0.5)
    made.update(given)
    return {name: torch.tensor(np.broadcast_to(np.asarray(value), (rows,)).copy(),
                               dtype=torch.int32 if name == "top_k" else torch.float32).cuda() for name, value in made.items()}


def check_draws(ops, logits, **given):
    numbers = settings(logits.shape[0], **given)
    got = ops.sample_filtered(logits, **numbers).cpu().tolist()
    host = {name: t.cpu().numpy().astype(np.float64) for name, t in numbers.items()}
    rows = logits.double().cpu().numpy()
    want = [draw_of(rows[r], *(host[name][r] for name in ("temperature", "top_k", "top_p", "min_p", "uniform")))
            for r in range(logits.shape[0])]
    assert got == want
    return got


def hills(rows, vocab, dtype, seed, spread=2.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn((rows, vocab), generator=gen) * spread).to(dtype).cuda()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [1, 2, 63, 64, 65, 1000, 2048, 2049, 4096, 8192, 8193, 32003, 151936])
def test_draws_over_vocabularies(ops, vocab, dtype):
    rows = 24 if vocab < 100000 else 6
    rng = np.random.default_rng(vocab)
    check_draws(ops, hills(rows, vocab, dtype, vocab), temperature=rng.uniform(0.3, 2.0, rows), top_k=rng.integers(0, 60, rows),
                top_p=rng.uniform(0.5, 1.1, rows), min_p=rng.uniform(0, 0.1, rows), uniform=rng.uniform(0, 1, rows))


@pytest.mark.parametrize("name,given", [
    ("everything", {}), ("top-k 1", dict(top_k=1)), ("top-k 5", dict(top_k=5)), ("top-k past the row", dict(top_k=100000)),
    ("top-k below none", dict(top_k=-3)), ("top-p 0", dict(top_p=0.0)), ("top-p 0.1", dict(top_p=0.1)), ("top-p 0.9", dict(top_p=0.9)),
    ("top-p 0.99999", dict(top_p=0.99999)), ("top-p above 1", dict(top_p=1.5)), ("top-p below 0", dict(top_p=-1.0)),
    ("min-p 1", dict(min_p=1.0)), ("min-p above 1", dict(min_p=2.0)), ("min-p 0.05", dict(min_p=0.05)), ("min-p tiny", dict(min_p=1e-9)),
    ("cold", dict(temperature=0.01)), ("hot", dict(temperature=50.0)), ("very hot", dict(temperature=1e30)), ("greedy", dict(temperature=0.0)),
    ("below zero", dict(temperature=-1.0)), ("all of them", dict(top_k=50, top_p=0.95, min_p=0.02, temperature=0.8)),
], ids=lambda v: v if isinstance(v, str) else "")
def test_draws_over_settings(ops, name, given):
    uniform = [0.0, 1e-7, 0.1, 0.25, 0.5, 0.75, 0.9, 0.999, 1 - 2.0 ** -24, 0.3, 0.6, 0.45]
    check_draws(ops, hills(len(uniform), 5000, torch.float32, 7), uniform=uniform, **given)


@pytest.mark.parametrize("levels", [1, 2, 7, 300])
@pytest.mark.parametrize("dtype", DTYPES)
def test_draws_among_equal_logits(ops, levels, dtype):
    # Ties at every border: the lower index comes first; with one level the borders are whole numbers of equal tokens.
    gen = torch.Generator().manual_seed(levels)
    logits = (torch.randint(0, levels, (16, 20001), generator=gen).float() / 8).to(dtype).cuda()
    rng = np.random.default_rng(levels)
    for given in (dict(), dict(top_k=777), dict(top_p=0.5), dict(min_p=0.9), dict(top_k=3000, top_p=0.25, min_p=0.3)):
        check_draws(ops, logits, uniform=rng.integers(0, 1024, 16) / 1024.0, **given)


def test_zeros_of_both_signs_are_equal(ops):
    logits = torch.zeros((8, 300))
    logits[:, ::3] = -0.0
    check_draws(ops, logits.cuda(), uniform=np.arange(8) / 8.0, top_k=[0, 0, 0, 0, 10, 10, 10, 10])


def test_draws_among_what_is_no_number(ops):
    inf, nan = float("inf"), float("nan")
    rows = [[nan] * 6, [-inf] * 6, [nan, -inf, nan, -inf, -inf, -inf], [nan, 1.0, 2.0, nan, 2.0, -inf], [inf, 1.0, inf, nan, 0.0, 0.0],
            [-inf, -inf, -inf, 3.0, -inf, -inf], [3.4e38, -3.4e38, 0.0, 1.0, -inf, nan], [-3.4e38, -3.4e38, -inf, nan, -inf, -inf],
            [1e-45, -1e-45, 0.0, -0.0, 1e-40, nan]]
    logits = torch.tensor(rows).cuda()
    for uniform in (0.0, 0.3, 0.9):
        for given in (dict(), dict(top_k=2), dict(top_p=0.4), dict(min_p=0.5), dict(temperature=0.0)):
            check_draws(ops, logits, uniform=uniform, **given)
    numbers = settings(len(rows), uniform=nan, top_p=nan, min_p=nan)      # settings that are no numbers: some token of the row
    got = ops.sample_filtered(logits, **numbers).cpu().tolist()
    assert all(0 <= g < 6 for g in got)


def test_a_uniform_number_past_its_range_takes_an_end(ops):
    logits = hills(4, 500, torch.float32, 3)
    order = torch.argsort(logits, dim=1, descending=True, stable=True).cpu()
    numbers = settings(4, uniform=[1.0, 7.0, -0.5, float("-inf")], top_k=9)
    assert ops.sample_filtered(logits, **numbers).cpu().tolist() == [int(order[0, 8]), int(order[1, 8]), int(order[2, 0]), int(order[3, 0])]


@pytest.mark.parametrize("vocab", [7, 3000, 20000, 151936])
@pytest.mark.parametrize("min_p", [1.0, 1.0 + 2.0 ** -23, 2.0, float("inf")])
def test_a_share_above_one_leaves_the_first_of_equal_maxima(ops, vocab, min_p):
    # No token weighs more than the first one: nothing but that is left, whichever of the equal maxima the uniform number would point at.
    logits = hills(6, vocab, torch.float32, 13)
    logits[:, 1::2] = 9.0                                    # (a few rows of the long ones reach higher by themselves)
    first = np.argmax(logits.cpu().numpy(), axis=1).tolist()
    for given in (dict(), dict(top_k=3), dict(top_p=0.9), dict(top_k=vocab)):
        got = check_draws(ops, logits, min_p=min_p, uniform=[0.0, 0.2, 0.4, 0.6, 0.8, 0.99], **given)
        assert min_p == 1.0 or got == first


def test_a_flat_row_is_drawn_to_the_token(ops):
    # 150,000 tokens of nearly one weight: 32-bit weights' sums would be tokens away from the border.
    gen = torch.Generator().manual_seed(11)
    logits = (torch.rand((8, 150001), generator=gen) * 1e-3).cuda()
    check_draws(ops, logits, uniform=np.random.default_rng(1).uniform(0, 1, 8), top_p=[1, 1, 1, 0.5, 0.9, 1, 1, 0.7], top_k=[0, 100000, 0, 0, 0, 7, 0, 0])


def test_most_of_a_row_in_one_place(ops):
    # Thousands of different logits within a hair of each other beside far-away ones: one range holds them nearly all.
    gen = torch.Generator().manual_seed(12)
    logits = 20.0 + torch.rand((6, 60000), generator=gen) * 1e-4
    logits[:, ::1000] = -30.0
    logits[:, 17] = 24.0
    check_draws(ops, logits.cuda(), uniform=[0.2, 0.5, 0.9, 0.99, 0.4, 0.7], top_p=[1, 0.9, 0.95, 1, 1, 0.6], top_k=[0, 0, 0, 30000, 50001, 0])


@pytest.mark.parametrize("vocab", [300, 40000, 151936])
@pytest.mark.parametrize("masked", [float("-inf"), torch.finfo(torch.float32).min, -1e30, -1000.0])
def test_masked_rows(ops, vocab, masked):
    # Most of a row ruled out, by what no number is below or by a number far below: few tokens are left, and fewer than top-k asks for.
    logits = hills(12, vocab, torch.float32, 9)
    gen = torch.Generator().manual_seed(vocab)
    for row, left in enumerate([1, 2, 3, 7, 40, 41, 64, 100, 150, 250, 299, 300]):
        keep = torch.randperm(vocab, generator=gen)[:left].cuda()
        mask = torch.ones(vocab, dtype=torch.bool).cuda()
        mask[keep] = False
        logits[row, mask] = masked
    uniform = np.random.default_rng(3).uniform(0, 1, 12)
    for given in (dict(), dict(top_k=40), dict(top_k=200), dict(top_k=40, top_p=0.9), dict(min_p=0.02), dict(top_k=20, min_p=0.3), dict(top_p=0.8),
                  dict(top_k=60, temperature=30.0)):
        check_draws(ops, logits, uniform=uniform, **given)


@pytest.mark.parametrize("vocab", [8193, 20481, 30000, 151936])
def test_draws_under_counts_around_those_of_the_waves(ops, vocab):
    # (A row in pieces of 4,096 logits has four waves a piece.)
    waves = 4 * -(-vocab // 4096)
    counts = [1, 2, waves // 2, waves // 2 + 1, 8 * (vocab // 4096), 8 * (vocab // 4096) + 1, 1000, 8191, 8192, 8193, vocab - 1, vocab, vocab + 1]
    logits = hills(len(counts), vocab, torch.float32, 10)
    logits[3] = logits[3].sort().values                       # the largest side by side, at the end and at the start
    logits[4] = logits[4].sort(descending=True).values
    logits[1, :] = 1.0
    logits[1, 5] = 2.0
    for given in (dict(), dict(top_p=0.9), dict(min_p=0.05), dict(top_p=0.95, min_p=0.01)):
        check_draws(ops, logits, top_k=counts, uniform=np.linspace(0, 0.9999, len(counts)), **given)


@pytest.mark.parametrize("rows", [1, 9, 40])
@pytest.mark.parametrize("vocab", [8193, 60000, 151936])
def test_draws_where_a_floor_keeps_few_or_thousands(ops, rows, vocab):
    # Under min-p alone (and under a top-k that fewer parts of the row reach than it asks for) a row is listed only where the list is short.
    logits = hills(rows, vocab, torch.float32, rows, 2.2)
    logits[::3, vocab // 7:] = float("-inf")                 # neighbours alone are allowed
    logits[1::3, ::64] += 7.0                                # some stand out
    rng = np.random.default_rng(rows)
    for given in (dict(min_p=1e-9), dict(min_p=1e-3), dict(min_p=0.01, temperature=1.5), dict(min_p=0.05), dict(top_k=40), dict(top_k=200),
                  dict(top_k=150, min_p=1e-6), dict(min_p=10.0 ** rng.uniform(-8, 0, rows), top_k=rng.integers(0, 2, rows) * 30),
                  dict(min_p=1e-30, temperature=1e30), dict(min_p=0.5, temperature=1e-3)):
        check_draws(ops, logits, uniform=rng.uniform(0, 1, rows), **given)


@pytest.mark.parametrize("rows", [3, 40])
@pytest.mark.parametrize("vocab", [9000, 60000, 151936])
def test_draws_where_fewer_tokens_weigh_anything_than_top_k_asks_for(ops, rows, vocab):
    # A cold row, or one with a token far above the rest: a few dozen tokens, here and there or side by side, are all there is to list.
    logits = hills(rows, vocab, torch.float32, rows + 1, 2.2)
    logits[::3, 100:160] += 15.0
    logits[1::3, 5] += 18.0
    rng = np.random.default_rng(rows)
    for given in (dict(top_k=100), dict(top_k=15, top_p=0.9), dict(top_k=200, min_p=1e-4)):
        for temperature in (0.05, 0.2, 0.4, 1.0):
            check_draws(ops, logits, uniform=rng.uniform(0, 1, rows), temperature=temperature, **given)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [196609, 256000, 1 << 19])
def test_draws_from_the_largest_vocabularies(ops, vocab, dtype):
    logits = hills(5, vocab, dtype, 14, 2.5)
    logits[3, vocab // 9:] = float("-inf")
    for given in (dict(top_k=[1, 40, 300, 50, 1000]), dict(top_k=[255, 256, 257, 1023, 1024], top_p=0.9), dict(min_p=[0.1, 0.02, 1e-3, 0.01, 1e-6]),
                  dict(top_p=0.7), dict(top_k=[0, 60, 0, 500, 512], min_p=0.03, top_p=[1.0, 0.95, 0.9, 1.0, 1.0])):
        check_draws(ops, logits, uniform=[0.1, 0.9, 0.5, 0.7, 0.3], **given)


@pytest.mark.parametrize("name,logits,given", [("a low floor", "flat", dict(min_p=1e-6)), ("a floor that keeps thousands", "flat", dict(min_p=0.01, temperature=1.5)),
                                               ("neighbours alone", "neighbours", dict(top_k=40))], ids=lambda v: v if isinstance(v, str) else "")
def test_a_filter_of_many_tokens_costs_about_what_all_tokens_cost(ops, name, logits, given):
    # (Rows that one workgroup went through again and again took three to thirteen times as long as the same rows without the filter.)
    rows = hills(8, 151936, torch.float32, 15, 2.2)
    if logits == "neighbours":
        rows[:, 20000:] = float("-inf")

    def time_of(numbers):
        run = lambda: ops.sample_filtered(rows, **numbers)
        run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run()
        best = float("inf")
        for _ in range(5):
            start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            start.record()
            for _ in range(10):
                graph.replay()
            end.record()
            torch.cuda.synchronize()
            best = min(best, start.elapsed_time(end))
        return best

    numbers = settings(8, uniform=np.arange(8) / 8.0, **given)
    check_draws(ops, rows, uniform=np.arange(8) / 8.0, **given)
    assert time_of(numbers) < 2.5 * time_of(settings(8, uniform=np.arange(8) / 8.0))


def test_draws_from_rows_that_lie_apart_and_into_a_given_place(ops):
    wide = hills(9, 3001, torch.float32, 4)
    numbers = settings(9, uniform=np.arange(9) / 9.0, top_k=30)
    want = ops.sample_filtered(wide[:, 5:2905].contiguous(), **numbers)
    out = torch.full((9,), -1, dtype=torch.int32).cuda()
    assert ops.sample_filtered(wide[:, 5:2905], out=out, **numbers) is out and torch.equal(out, want)
    same = wide[:1].expand(9, -1)                            # one row of logits for nine answers
    assert torch.equal(ops.sample_filtered(same, **numbers), ops.sample_filtered(same.contiguous(), **numbers))
    assert ops.sample_filtered(wide[:0], **settings(0)).numel() == 0


def test_a_draw_does_not_depend_on_the_batch(ops):
    logits = hills(70, 33333, torch.float32, 5)
    rng = np.random.default_rng(2)
    numbers = settings(70, uniform=rng.uniform(0, 1, 70), top_k=rng.integers(0, 100, 70), top_p=rng.uniform(0.5, 1.0, 70))
    whole = ops.sample_filtered(logits, **numbers)
    for part in (slice(0, 1), slice(3, 10), slice(30, 70)):
        assert torch.equal(whole[part], ops.sample_filtered(logits[part], **{n: t[part].contiguous() for n, t in numbers.items()}))


@pytest.mark.parametrize("rows", [1, 8, 9, 19, 20, 40])
def test_draws_of_few_and_many_long_rows(ops, rows):
    # (Rows of up to 256 pieces of 4,096 logits together are gathered and drawn in one launch.)
    logits = hills(rows, 50001, torch.float32, rows, 3.0)
    rng = np.random.default_rng(rows)
    for given in (dict(), dict(top_p=0.9), dict(top_k=30), dict(top_k=rng.integers(0, 2, rows) * 40, top_p=rng.uniform(0.5, 1.1, rows)),
                  dict(temperature=rng.integers(0, 2, rows) * 1.0, top_p=0.8)):
        check_draws(ops, logits, uniform=rng.uniform(0, 1, rows), **given)


@pytest.mark.parametrize("rows,spread", [(1, 2.2), (2, 0.5), (5, 3.0)])
def test_the_workgroup_that_comes_last_finds_every_token(ops, rows, spread):
    # Few rows: the workgroups of a row's pieces leave their tokens, and the last one to come draws.  Hundreds of draws of other logits each time, a
    # list of up to some thousands from all pieces, in memory that the draw before has left full of its own.
    first, second = hills(rows, 151936, torch.float32, rows, spread), hills(rows, 151936, torch.float32, 100 + rows, spread)
    uniform = np.random.default_rng(rows).uniform(0, 1, rows)
    given = dict(top_p=0.9, uniform=uniform)
    want = [check_draws(ops, x, **given) for x in (first, second)]
    numbers, held = settings(rows, **given), first.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.sample_filtered(held, **numbers)
    seen = torch.empty((300, rows), dtype=torch.int32).cuda()
    for turn in range(300):
        held.copy_((first, second)[turn % 2])
        graph.replay()
        seen[turn] = out
    assert seen[0::2].tolist() == [want[0]] * 150 and seen[1::2].tolist() == [want[1]] * 150


@pytest.mark.parametrize("rows,vocab,dtype", [(216, 151936, torch.bfloat16), (830, 40001, torch.float32)])
def test_draws_of_very_many_long_rows(ops, rows, vocab, dtype):
    # (A workgroup sees to several pieces of a row then.)  Each row's draw is what it is among eight, and of some by the definition.
    logits = hills(rows, vocab, dtype, rows, 3.0)
    logits[::7, 5:] = float("-inf")
    logits[3::11, 9000:] = float("nan")
    rng = np.random.default_rng(rows)
    given = dict(temperature=rng.integers(0, 5, rows) * 0.4, top_k=rng.integers(-1, 3, rows) * 45, top_p=rng.uniform(0.6, 1.3, rows),
                 min_p=rng.integers(0, 2, rows) * 0.03, uniform=rng.uniform(0, 1, rows))
    got = ops.sample_filtered(logits, **settings(rows, **given)).tolist()
    for at in range(0, rows, 8):
        part = {name: value[at:at + 8] for name, value in given.items()}
        some = logits[at:at + 8]
        assert ops.sample_filtered(some, **settings(len(some), **part)).tolist() == got[at:at + 8]
    some = list(range(0, rows, rows // 9))
    assert check_draws(ops, logits[some], **{name: value[some] for name, value in given.items()}) == [got[r] for r in some]


def test_the_largest_counts(ops):
    logits = hills(4, 50001, torch.float32, 2)
    check_draws(ops, logits, top_k=[2 ** 30, 2 ** 30 + 1, 2 ** 31 - 1, -2 ** 31], uniform=[0.1, 0.5, 0.7, 0.9])


def test_draws_on_another_stream_and_replayed(ops):
    first, second = hills(5, 20000, torch.float32, 6), hills(5, 20000, torch.float32, 8)
    numbers = settings(5, uniform=[0.1, 0.4, 0.6, 0.8, 0.95], top_k=40, top_p=0.9)
    want = [ops.sample_filtered(x, **numbers).tolist() for x in (first, second)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        beside = ops.sample_filtered(first, **numbers)
    other = ops.sample_filtered(second, **numbers)
    torch.cuda.synchronize()
    assert beside.tolist() == want[0] and other.tolist() == want[1]
    held = first.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.sample_filtered(held, **numbers)
    for turn in range(4):
        held.copy_((first, second)[turn % 2])
        graph.replay()
        assert out.tolist() == want[turn % 2]
        assert ops.sample_filtered(second, **numbers).tolist() == want[1]


def test_draws_refused(ops):
    logits, numbers = hills(3, 100, torch.float32, 1), settings(3)
    for bad in (dict(top_k=settings(3)["top_p"]), dict(top_p=settings(2)["top_p"]), dict(uniform=numbers["uniform"].cpu()),
                dict(out=torch.empty(3, dtype=torch.int64).cuda()), dict(temperature=numbers["temperature"].double())):
        with pytest.raises(KernelError):
            ops.sample_filtered(logits, **{**numbers, **bad})
    for bad in (logits.half(), logits[0], logits.t()[:3], logits.cpu(), logits[:, :0]):
        with pytest.raises(KernelError):
            ops.sample_filtered(bad, **numbers)
    with pytest.raises(KernelError):
        ops.sample_filtered(torch.zeros((1, 1)).cuda().expand(1, (1 << 19) + 1), **settings(1))


# ------------------------------------------------------------------------------------------------ pages
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layers,n_pages,widths,pairs", [
    (1, 2, (1,), 1), (3, 10, (16, 16), 4), (24, 40, (2048, 2048), 3), (2, 9, (7, 13, 1, 5), 4), (1, 70, (2048, 1024), 33),
    (5, 6, (20000,), 2), (2, 5, (6, 2), 2), (4, 7, (100001, 3), 3)])
def test_copied_pages(ops, dtype, layers, n_pages, widths, pairs):
    gen = torch.Generator().manual_seed(n_pages)
    pool = torch.randn((layers, n_pages * sum(widths)), generator=gen).to(dtype).cuda()
    order = torch.randperm(n_pages, generator=gen)
    dst = order[:pairs]
    src = order[pairs:][torch.randint(0, n_pages - pairs, (pairs,), generator=gen)]          # (a page may go to several)
    want, at = pool.clone(), 0
    for width in widths:
        plane = want[:, at:at + n_pages * width].view(layers, n_pages, width)
        plane[:, dst.cuda()] = plane[:, src.cuda()]
        at += n_pages * width
    got = ops.copy_pages(pool, n_pages, widths, src.int().cuda(), dst.int().cuda())
    assert got is pool and torch.equal(pool, want)


def test_pages_at_any_alignment(ops):
    base = torch.randn(2 * 9 * 24 + 3).to(torch.bfloat16).cuda()
    for offset in (0, 1, 2, 3):
        whole = base.clone()
        pool = whole[offset:offset + 2 * 9 * 24].view(2, 9 * 24)
        want = whole.clone()
        view = want[offset:offset + 2 * 9 * 24].view(2, 9 * 24)
        for start, width in ((0, 16), (9 * 16, 8)):
            plane = view[:, start:start + 9 * width].view(2, 9, width)
            plane[:, 4] = plane[:, 1].clone()
        ops.copy_pages(pool, 9, (16, 8), torch.tensor([1], dtype=torch.int32).cuda(), torch.tensor([4], dtype=torch.int32).cuda())
        assert torch.equal(whole, want)                      # what lies before and behind the pool stays too


def test_pages_outside_the_pool_are_passed_over(ops):
    whole = torch.arange(3 * 8 * 6, dtype=torch.float32).cuda()
    pool = whole[48:96].view(1, 48)
    want = whole.clone()
    want[48 + 12:48 + 18] = want[48:54]
    src = torch.tensor([-1, 8, 0, 2 ** 31 - 1, 1, -2 ** 31, 5], dtype=torch.int32).cuda()
    dst = torch.tensor([3, 4, 2, 5, 8, 6, -1], dtype=torch.int32).cuda()
    ops.copy_pages(pool, 8, (6,), src, dst)
    assert torch.equal(whole, want)


def test_no_pages_and_the_same_page(ops):
    pool = torch.randn((2, 40)).cuda()
    kept, none = pool.clone(), torch.empty(0, dtype=torch.int32).cuda()
    ops.copy_pages(pool, 10, (4,), none, none)
    same = torch.tensor([3, 3], dtype=torch.int32).cuda()
    ops.copy_pages(pool, 10, (4,), same, same)
    assert torch.equal(pool, kept)


def test_copied_pages_replayed(ops):
    pool = torch.randn((4, 300 * 512)).to(torch.bfloat16).cuda()
    src, dst = torch.tensor([1, 2, 3], dtype=torch.int32).cuda(), torch.tensor([101, 102, 103], dtype=torch.int32).cuda()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.copy_pages(pool, 300, (256, 256), src, dst)
    for turn in range(3):
        src.copy_(torch.tensor([4 + turn, 9, 20 + turn], dtype=torch.int32))
        want = pool.clone()
        for start in (0, 300 * 256):
            plane = want[:, start:start + 300 * 256].view(4, 300, 256)
            plane[:, [101, 102, 103]] = plane[:, [4 + turn, 9, 20 + turn]]
        graph.replay()
        assert torch.equal(pool, want)


def test_copies_refused(ops):
    pool, one = torch.randn((2, 40)).cuda(), torch.tensor([1], dtype=torch.int32).cuda()
    for args in ((pool, 10, (5,), one, one), (pool, 10, (), one, one), (pool, 10, (1, 1, 1, 0, 2), one, one), (pool, 0, (4,), one, one),
                 (pool.half(), 10, (4,), one, one), (pool, 10, (4,), one.long(), one.long()), (pool, 10, (4,), one, one.repeat(2)),
                 (pool, 10, (4,), one.cpu(), one.cpu()), (pool.t(), 10, (4,), one, one), (pool.view(80), 10, (4,), one, one)):
        with pytest.raises(KernelError):
            ops.copy_pages(*args)


# ------------------------------------------------------------------------------------------------ attention
class Batch:
    """Requests over pages in any order; `tables[r]`: request r's pages, `positions[r]`: its newest token."""

    def __init__(self, tables, positions, n_q, n_kv, d, page, dtype, seed, sharp=2.0, spare=3):
        gen = torch.Generator().manual_seed(seed)
        used = 1 + max([-1] + [p for t in tables for p in t])
        where = torch.randperm(used + spare, generator=gen)
        width = max([1] + [len(t) for t in tables])
        self.tables = [[int(where[p]) for p in t] for t in tables]
        table = torch.full((len(tables), width), -1, dtype=torch.int32)
        for r, t in enumerate(self.tables):
            table[r, :len(t)] = torch.tensor(t, dtype=torch.int32)
        normal = lambda *shape: torch.randn(shape, generator=gen)
        self.k, self.v = normal(used + spare, n_kv, page, d).to(dtype), normal(used + spare, n_kv, d, page).to(dtype)
        self.qkv = normal(len(tables), (n_q + 2 * n_kv) * d)
        self.qkv[:, :n_q * d] *= sharp
        self.qkv = self.qkv.to(dtype)
        self.positions, self.table = positions, table
        self.n_q, self.n_kv, self.d, self.page, self.dtype = n_q, n_kv, d, page, dtype
        # Slots that no request has written hold what is no number: whatever reads them shows.
        written = torch.zeros((used + spare, page), dtype=torch.bool)
        for t, p in zip(self.tables, positions):
            for at, name in enumerate(t):
                written[name, :max(0, min(page, p + 1 - at * page))] = True
        self.k.transpose(1, 2)[~written] = float("nan")
        self.v.permute(0, 3, 1, 2)[~written] = float("nan")

    def run(self, ops, plan=None, **more):
        on = lambda t: t.cuda()
        if plan is None:
            plan = ops.plan_shared_prefixes(self.table.numpy(), self.positions, self.page, self.n_q, self.n_kv, self.d, self.dtype, "cuda:0")
        out = torch.full((len(self.positions), self.n_q * self.d), float("nan"), dtype=self.dtype).cuda()
        ops.shared_prefix_attention(on(self.qkv), out, on(self.k), on(self.v), on(torch.tensor(self.positions, dtype=torch.int32)),
                                    on(self.table), plan, self.n_q, self.n_kv, self.d, 1.0 / math.sqrt(self.d), **more)
        return out.cpu(), plan

    def check(self, got, sinks=None, softcap=None):
        """Against the formula in 64 bits.  A result is off by the rounding of the weights to the values' type (bfloat16: 2^-8 of
        each weight's share of sum |w v| / sum w), that of the result, and, twice over, by what 32-bit sums and exponentials leave: a score
        is a sum of d products (d + 4 roundings of sum |q k|), a cap turns it by as many, the exponential adds some 4 (1 + its
        range) roundings of itself, and the sums over n keys, joined in parts, at most log2(n) + 32."""
        group, d = self.n_q // self.n_kv, self.d
        u = 2.0 ** -24
        for r, p in enumerate(self.positions):
            if p < 0:
                assert (got[r] == 0).all()
                continue
            at = torch.arange(p + 1)
            pages = torch.tensor(self.tables[r])[at // self.page]
            for g in range(self.n_kv):
                keys, values = self.k[pages, g, at % self.page].double(), self.v[pages, g, :, at % self.page].double()
                query = self.qkv[r, g * group * d:(g + 1) * group * d].view(group, d).double()
                scores = query @ keys.T / math.sqrt(d)
                size = (query.abs() @ keys.abs().T / math.sqrt(d)).amax()
                if softcap:
                    scores = softcap * torch.tanh(scores / softcap)
                mass = torch.logsumexp(scores, 1)
                if sinks is not None:
                    mass = torch.logaddexp(mass, sinks.double()[g * group:(g + 1) * group])
                weight = torch.exp(scores - mass[:, None])
                want, spread = weight @ values, weight @ values.abs()
                reach = (scores.amax() - scores.amin()).abs() + 1
                less = 2 * u * ((d + 4) * size + 4 * reach + math.log2(p + 2) + 32 + (softcap or 0) * 4)
                half = 2.0 ** -8 if self.dtype == torch.bfloat16 else 0.0
                bound = spread * (half + less) + want.abs() * (half + 2 * u) + 1e-30
                mine = got[r, g * group * d:(g + 1) * group * d].view(group, d).double()
                off = ((mine - want).abs() / bound).max().item()
                assert off <= 1.0, f"request {r} at {p}, kv head {g}: {off} of the bound"


@pytest.fixture(params=["as planned", "many columns"])
def any_work(request, monkeypatch):
    """As the plan's rule says for the (small) batches of these tests, and with the items of many columns that larger ones get."""
    if request.param == "many columns":
        monkeypatch.setattr(SharedPrefixes, "WIDE_WORK", -1)
        monkeypatch.setattr(SharedPrefixes, "MANY_WORK", -1)


def shared_tables(rows, prefix_pages, page, own, branch=None):
    """`rows` requests behind `prefix_pages` common pages, request r with own[r] keys of its own; branch: (every, pages)."""
    used, tables, positions = prefix_pages, [], []
    branches = {}
    for r in range(rows):
        table = list(range(prefix_pages))
        if branch:
            key = r // branch[0]
            if key not in branches:
                branches[key] = list(range(used, used + branch[1]))
                used += branch[1]
            table += branches[key]
        pages = -(-own[r] // page)
        table += list(range(used, used + pages))
        used += pages
        tables.append(table)
        positions.append((len(table) - pages) * page + own[r] - 1)
    return tables, positions


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [16, 32, 48, 64, 80, 96, 112, 128, 160, 192, 224, 256])
def test_attention_over_head_sizes(ops, any_work, d, dtype):
    tables, positions = shared_tables(6, 11, 16, [1, 5, 16, 17, 40, 70])
    batch = Batch(tables, positions, 6, 2, d, 16, dtype, d)
    got, plan = batch.run(ops)
    assert [(len(r.rows), r.key_begin, r.key_end) for r in plan.runs] == [(6, 0, 176)]
    batch.check(got)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n_q,n_kv", [(1, 1), (14, 2), (4, 4), (7, 1), (33, 1), (64, 2), (70, 1)])
def test_attention_over_heads(ops, any_work, n_q, n_kv, dtype):
    tables, positions = shared_tables(11, 9, 16, [3 * r + 1 for r in range(11)])
    batch = Batch(tables, positions, n_q, n_kv, 64, 16, dtype, n_q)
    batch.check(batch.run(ops)[0])


@pytest.mark.parametrize("page", [16, 32, 48, 64])
@pytest.mark.parametrize("prefix_keys", [0, 48, 64, 192, 960, 2880])
@pytest.mark.parametrize("rows", [2, 5, 40])
def test_attention_over_lengths(ops, any_work, rows, prefix_keys, page):
    prefix = prefix_keys // page
    tables, positions = shared_tables(rows, prefix, page, [1 + (37 * r) % 150 for r in range(rows)])
    batch = Batch(tables, positions, 14, 2, 64, page, torch.bfloat16, rows + prefix)
    batch.check(batch.run(ops)[0])


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rows,n_q,n_kv", [(33, 2, 1), (13, 14, 2), (19, 28, 4), (60, 12, 2), (129, 1, 1), (40, 40, 1)])
@pytest.mark.parametrize("keys,page", [(64, 16), (80, 16), (1008, 16), (96, 32), (1056, 48), (1600, 64)])
def test_attention_of_many_columns(ops, monkeypatch, keys, page, rows, n_q, n_kv, d):
    monkeypatch.setattr(SharedPrefixes, "WIDE_WORK", -1)
    # (More than 64 query columns of a kv head go through the shared keys together; parts and blocks of them end anywhere.)
    tables, positions = shared_tables(rows, keys // page, page, [1 + (13 * r) % 40 for r in range(rows)])
    batch = Batch(tables, positions, n_q, n_kv, d, page, torch.bfloat16, rows + keys)
    got, plan = batch.run(ops)
    assert plan.n_many > 0
    batch.check(got)


@pytest.mark.parametrize("n_q,n_kv,d,dtype,rows,keys", [(14, 2, 64, torch.bfloat16, 40, 12048), (14, 2, 64, torch.float32, 64, 24000),
                                                        (14, 2, 64, torch.float32, 104, 24000),
                                                        (14, 2, 96, torch.bfloat16, 100, 16000)])
def test_attention_with_work_for_many_columns(ops, n_q, n_kv, d, dtype, rows, keys):
    tables, positions = shared_tables(rows, keys // 16, 16, [1 + (13 * r) % 40 for r in range(rows)])
    batch = Batch(tables, positions, n_q, n_kv, d, 16, dtype, keys)
    got, plan = batch.run(ops)
    wide = dtype == torch.bfloat16 and d in SharedPrefixes.WIDE_HEADS
    assert (plan.n_many > 0) == (rows * keys * n_q > (SharedPrefixes.WIDE_WORK if wide else SharedPrefixes.MANY_WORK))
    batch.check(got)


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_behind_branches(ops, any_work, dtype):
    tables, positions = shared_tables(23, 13, 16, [1 + (29 * r) % 200 for r in range(23)], branch=(4, 7))
    tables += [[900 + i for i in range(12)], [950]]           # two that share nothing, one of them short
    positions += [12 * 16 - 4, 0]
    batch = Batch(tables, positions, 12, 2, 128, 16, dtype, 3)
    got, plan = batch.run(ops)
    assert len(plan.runs) >= 6
    batch.check(got)


def test_attention_with_sinks_and_capped_scores(ops, any_work):
    tables, positions = shared_tables(9, 20, 16, [1 + 11 * r for r in range(9)])
    for dtype in DTYPES:
        batch = Batch(tables, positions, 10, 2, 64, 16, dtype, 5, sharp=6.0)
        sinks = torch.linspace(-4, 9, 10)
        sinks[3] = float("-inf")
        batch.check(batch.run(ops, sinks=sinks.cuda(), softcap=15.0)[0], sinks, 15.0)
        batch.check(batch.run(ops, softcap=3.0)[0], None, 3.0)
        batch.check(batch.run(ops, sinks=sinks.cuda())[0], sinks)


def test_one_row_and_rows_without_keys(ops, any_work):
    batch = Batch([[4, 2, 0]], [40], 14, 2, 64, 16, torch.bfloat16, 1)
    batch.check(batch.run(ops)[0])
    batch = Batch([[0], [0, 1], [2, 3]], [-1, 20, 31], 6, 3, 32, 16, torch.float32, 1)
    batch.check(batch.run(ops)[0])
    batch.check(batch.run(ops, sinks=torch.zeros(6).cuda())[0], torch.zeros(6))


def test_scores_far_apart_and_equal(ops, any_work):
    # Keys whose scores leave all others behind, in the shared run and in a request's own; then scores that are all zero.
    tables, positions = shared_tables(4, 40, 16, [100, 3, 50, 17])
    batch = Batch(tables, positions, 4, 2, 64, 16, torch.bfloat16, 9, sharp=40.0)
    batch.check(batch.run(ops)[0])
    batch.qkv.zero_()
    batch.check(batch.run(ops)[0])


def test_a_plan_holds_while_requests_grow(ops, any_work):
    tables, positions = shared_tables(7, 12, 16, [16 * 12] * 7)
    batch = Batch(tables, [12 * 16] * 7, 14, 2, 64, 16, torch.bfloat16, 2)
    plan = batch.run(ops)[1]
    for grown in (1, 15, 16, 17, 100, 191):
        later = Batch(tables, [12 * 16 + (grown * (r + 1)) // 7 for r in range(7)], 14, 2, 64, 16, torch.bfloat16, 2)
        later.check(later.run(ops, plan)[0])
        narrow = Batch(tables, later.positions, 14, 2, 64, 16, torch.bfloat16, 2)
        assert torch.equal(later.run(ops, plan, max_position=max(later.positions))[0], narrow.run(ops, plan, max_position=max(later.positions))[0])


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_of_a_long_request_among_short_ones(ops, any_work, dtype):
    # One that shares nothing and has many parts of its own among ones that have one; parts end inside blocks and pages.
    tables, positions = shared_tables(30, 20, 16, [1 + (5 * r) % 33 for r in range(30)])
    tables.insert(7, [5000 + i for i in range(301)])
    positions.insert(7, 300 * 16 + 4)
    batch = Batch(tables, positions, 14, 2, 64, 16, dtype, 21)
    for growth in (0, 512, None):
        plan = ops.plan_shared_prefixes(batch.table.numpy(), positions, 16, 14, 2, 64, dtype, "cuda:0", growth=growth)
        by_row = plan.own_of_row_dev.reshape(-1, 4).tolist()
        assert growth is None or (by_row[7][3] > 20 and by_row[6][3] < 10)
        batch.check(batch.run(ops, plan)[0])


@pytest.mark.parametrize("dtype", DTYPES)
def test_requests_may_grow_past_what_was_planned_for(ops, any_work, dtype):
    # The last part of a row takes whatever comes; a plan for no growth at all and one for the whole table give the same keys.
    tables, _ = shared_tables(5, 9, 16, [900] * 5)
    start = [9 * 16 + 3 * r for r in range(5)]
    for growth in (0, 500, None):
        first = Batch(tables, start, 14, 2, 64, 16, dtype, 22)
        plan = ops.plan_shared_prefixes(first.table.numpy(), start, 16, 14, 2, 64, dtype, "cuda:0", growth=growth)
        for grown in (0, 200, 511, 512, 890):
            later = Batch(tables, [p + grown for p in start[:-1]] + [9 * 16], 14, 2, 64, 16, dtype, 22)
            later.check(later.run(ops, plan)[0])


def test_a_table_cut_to_the_pages_in_use_and_a_named_end_change_nothing(ops, any_work):
    tables, _ = shared_tables(7, 12, 16, [16 * 12] * 7)
    for grown in (1, 16, 100, 190):
        positions = [12 * 16 + (grown * (r + 1)) // 7 for r in range(7)]
        batch = Batch(tables, positions, 14, 2, 64, 16, torch.bfloat16, 2)
        got, plan = batch.run(ops)
        batch.check(got)
        assert torch.equal(batch.run(ops, plan, max_position=max(positions))[0], got)
        batch.table = batch.table[:, :max(positions) // 16 + 1].contiguous()
        assert batch.table.shape[1] == (13, 14, 19, 24)[(1, 16, 100, 190).index(grown)] and torch.equal(batch.run(ops, plan)[0], got)


def test_attention_replayed_on_new_data_and_beside_another_stream(ops, any_work):
    tables, positions = shared_tables(16, 30, 16, [1 + 7 * r for r in range(16)])
    first, second = (Batch(tables, positions, 14, 2, 64, 16, torch.bfloat16, s) for s in (1, 2))
    plan = first.run(ops)[1]
    place = second.table                                    # (the two batches lie in different pages: one plan each)
    plans = [plan, second.run(ops)[1]]
    want = [b.run(ops, p)[0] for b, p in zip((first, second), plans)]
    moved = [t.cuda() for t in (first.qkv, first.k, first.v, first.table)]
    where = torch.tensor(positions, dtype=torch.int32).cuda()
    out = torch.zeros((16, 14 * 64), dtype=torch.bfloat16).cuda()
    run = lambda: ops.shared_prefix_attention(moved[0], out, moved[1], moved[2], where, moved[3], plan, 14, 2, 64, 0.125)
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for turn in range(4):
        for held, new in zip(moved, (b := (first, second)[turn % 2]) and (b.qkv, b.k, b.v, b.table)):
            held.copy_(new)
        out.fill_(7.0)
        graph.replay()
        assert torch.equal(out.cpu(), want[turn % 2])
        assert torch.equal(second.run(ops, plans[1])[0], want[1])
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        beside = first.run(ops, plan)[0]
    assert torch.equal(beside, want[0]) and place is second.table


def test_attention_refused(ops):
    tables, positions = shared_tables(3, 6, 16, [5, 9, 20])
    batch = Batch(tables, positions, 4, 2, 64, 16, torch.bfloat16, 1)
    _, plan = batch.run(ops)
    args = dict(qkv=batch.qkv.cuda(), out=torch.empty((3, 256), dtype=torch.bfloat16).cuda(), k_pages=batch.k.cuda(), v_pages=batch.v.cuda(),
                positions=torch.tensor(positions, dtype=torch.int32).cuda(), block_table=batch.table.cuda(), plan=plan, n_q=4, n_kv=2,
                head_dim=64, scale=0.125)
    ops.shared_prefix_attention(**args)
    for bad in (dict(qkv=args["qkv"][:2].contiguous()), dict(qkv=args["qkv"][None]), dict(v_pages=args["v_pages"][1:].contiguous()),
                dict(k_pages=args["k_pages"][1:].contiguous()), dict(block_table=args["block_table"][0]), dict(qkv=args["qkv"].float()), dict(out=args["out"][:, :128].contiguous()), dict(n_q=2),
                dict(head_dim=32), dict(block_table=args["block_table"][:, :4].contiguous()), dict(block_table=args["block_table"].long()),
                dict(positions=args["positions"][:2]), dict(k_pages=args["k_pages"].transpose(2, 3)), dict(v_pages=args["k_pages"]),
                dict(max_position=16 * batch.table.shape[1]), dict(sinks=torch.zeros(3).cuda()), dict(softcap=-1.0),
                dict(positions=args["positions"].cpu()), dict(k_pages=args["k_pages"].repeat(1, 1, 2, 1), v_pages=args["v_pages"].repeat(1, 1, 1, 2))):
        with pytest.raises(KernelError):
            ops.shared_prefix_attention(**{**args, **bad})
    for bad in (dict(page_size=8), dict(head_dim=72), dict(n_kv=3), dict(dtype=torch.float16), dict(positions=[1, 2])):
        with pytest.raises(KernelError):
            ops.plan_shared_prefixes(**{**dict(block_table=batch.table.numpy(), positions=positions, page_size=16, n_q=4, n_kv=2, head_dim=64,
                                               dtype=torch.bfloat16, device="cuda:0"), **bad})
