"""The operators behind several answers to one prompt, as a program that serves them calls them: draws under temperature,
top-k, top-p and min-p, pages of the cache copied for a fork or moved to its low end, and attention of single tokens whose
requests share leading pages.

    own                 whether `run` calls the framework's kernels (else plain torch)
    listed()            the cases
    draw(rng)           one more case of the same ranges
    prepare(case, seed) inputs on the GPU, and the plan that a program keeps while its requests stay the same
    run(state)          one pass through an operator
    work(case)          the bytes and operations a pass cannot do without
    exact(case, seed)   the results in 64 bits
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEVICE = "cuda:0"
_TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}

# Layer sizes of the Qwen2.5 models that the benchmark runs at.
SIZES = {"0.5b": dict(heads=14, kv=2, dim=64, layers=24, vocab=151936),
         "1.5b": dict(heads=12, kv=2, dim=128, layers=28, vocab=151936),
         "7b": dict(heads=28, kv=4, dim=128, layers=28, vocab=152064)}


def _sampling(name, rows, vocab, top_k, top_p, min_p, temperature, greedy=0, dtype="float32", banned=0.0):
    """`top_k`, `top_p`, `min_p`, `temperature`: (lowest, highest) of the rows' values; top_k 0, top_p 1 and min_p 0 keep
    everything.  `greedy`: every so many-th row has temperature 0.  `banned`: the share of a row's logits at -inf."""
    case = {"op": "sampling", "rows": rows, "vocab": vocab, "top_k_low": top_k[0], "top_k_high": top_k[1],
            "top_p_low": top_p[0], "top_p_high": top_p[1], "min_p_low": min_p[0], "min_p_high": min_p[1],
            "temperature_low": temperature[0], "temperature_high": temperature[1], "greedy": greedy, "dtype": dtype,
            "banned": banned}
    return dict(case, name=name) if name else case


def _copying(name, layers, heads, dim, page, pages, copied, dtype="bfloat16", tied=False):
    """`pages`: pages of the pool; `copied`: how many of them a pass copies, in all layers."""
    case = {"op": "copying", "layers": layers, "heads": heads, "dim": dim, "page": page, "pages": pages,
            "copied": copied, "dtype": dtype, "tied": tied}
    return dict(case, name=name) if name else case


def _attention(name, rows, heads, kv, dim, prefix, branches, branch, own_low, own_high, page=16, dtype="bfloat16", loners=0,
               softcap=0.0, sink=False):
    """`rows` requests share `prefix` keys; they fall into `branches` equal runs that share `branch` more each (0: none);
    every request has between `own_low` and `own_high` keys of its own behind; the last `loners` share nothing."""
    case = {"op": "attention", "rows": rows, "heads": heads, "kv": kv, "dim": dim, "prefix": prefix, "branches": branches,
            "branch": branch, "own_low": own_low, "own_high": own_high, "page": page, "dtype": dtype, "loners": loners,
            "softcap": softcap, "sink": sink}
    return dict(case, name=name) if name else case


def listed() -> list[dict]:
    small, middle, large = SIZES["0.5b"], SIZES["1.5b"], SIZES["7b"]
    return [
        # One conversation's next token under the usual settings: the latency of a draw.
        _sampling("a draw for one request", 1, small["vocab"], (40, 40), (0.95, 0.95), (0.0, 0.0), (0.7, 0.7)),
        # A busy server's batch: every request brings settings of its own, some are greedy.
        _sampling("draws for 64 requests", 64, small["vocab"], (0, 200), (0.8, 1.0), (0.0, 0.1), (0.4, 1.3), greedy=5),
        # Many answers to one prompt at the largest vocabulary, cut by min-p alone.
        _sampling("256 answers under min-p", 256, large["vocab"], (0, 0), (1.0, 1.0), (0.02, 0.1), (1.0, 1.5)),
        # Logits kept in 16 bits (many equal ones), an odd vocabulary, half of it ruled out by a grammar.
        _sampling("16-bit logits with a grammar", 7, 32003, (0, 50), (0.7, 1.0), (0.0, 0.05), (0.6, 1.0),
                  dtype="bfloat16", banned=0.5),
        # Three forks of a request: each takes a copy of the last, partly filled page.
        _copying("the last page for three forks", small["layers"], small["kv"], small["dim"], 16, 512, 3),
        # Forks of a batch in 32 bits with larger pages.
        _copying("31 pages in 32 bits", middle["layers"], middle["kv"], middle["dim"], 48, 160, 31, dtype="float32"),
        # A cache of the largest sizes brought together after long requests have gone.
        _copying("a compaction of 1,600 pages", large["layers"], large["kv"], large["dim"], 16, 3600, 1600),
        # Four answers to a short prompt.
        _attention("four answers to a short prompt", 4, small["heads"], small["kv"], small["dim"], 512, 0, 0, 1, 60),
        # A server whose requests share a system prompt, with tools or documents shared by some and a history of their own.
        _attention("64 requests behind a system prompt", 64, large["heads"], large["kv"], large["dim"], 4096, 8, 512, 20, 700),
        # The 32-bit path: ragged requests, some of which share nothing.
        _attention("21 ragged requests in 32 bits", 21, small["heads"], small["kv"], small["dim"], 1040, 0, 0, 1, 333,
                   dtype="float32", loners=2),
        # As many answers as a batch holds, behind the longest prompt.
        _attention("256 answers to a prompt of 32,000", 256, large["heads"], large["kv"], large["dim"], 32000, 0, 0, 1, 500),
    ]


def _between(rng, low, high):
    """A whole number, spread over the logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def draw(rng) -> dict:
    op = rng.choice(["sampling", "copying", "attention"])
    if op == "sampling":
        rows, vocab = _between(rng, 1, 256), _between(rng, 1000, 152064)
        top_k = rng.choice([(0, 0), (1, 1), (20, 20), (40, 40), (0, 200), (1, 1000)])
        top_p = rng.choice([(1.0, 1.0), (0.9, 0.9), (0.95, 0.95), (0.3, 1.0)])
        min_p = rng.choice([(0.0, 0.0), (0.05, 0.05), (0.0, 0.2)])
        temperature = rng.choice([(0.7, 0.7), (1.0, 1.0), (0.2, 1.5)])
        return _sampling(None, rows, vocab, top_k, top_p, min_p, temperature, greedy=rng.choice([0, 0, 3]),
                         dtype=rng.choice(["float32", "float32", "float32", "bfloat16"]), banned=rng.choice([0.0, 0.0, 0.5, 0.999]))
    if op == "copying":
        size = SIZES[rng.choice(sorted(SIZES))]
        dtype, page = rng.choice(["bfloat16", "bfloat16", "float32"]), rng.choice([8, 16, 16, 24, 32])
        layers, heads, dim = rng.choice([1, 4, size["layers"]]), rng.choice([1, size["kv"], 7]), rng.choice([40, size["dim"], 112])
        page_bytes = layers * heads * dim * page * 2 * (2 if dtype == "bfloat16" else 4)
        copied = _between(rng, 1, max(1, min(1600, (1 << 30) // page_bytes)))
        return _copying(None, layers, heads, dim, page, 2 * copied + rng.randint(1, 60), copied, dtype, tied=rng.random() < 0.2)
    heads, kv, dim = rng.choice([(14, 2, 64), (12, 2, 128), (28, 4, 128), (8, 8, 96), (15, 5, 48), (16, 1, 256), (20, 2, 80)])
    dtype = rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"])
    rows, prefix = _between(rng, 2, 256), _between(rng, 17, 32000)
    while rows * prefix * heads * dim > (1 if dtype == "bfloat16" else 0.25) * 6e9:
        rows, prefix = max(2, rows // 2), max(17, prefix * 2 // 3)
    branches = rng.choice([0, 0, 0, 2, 5]) if rows >= 10 else 0
    return _attention(None, rows, heads, kv, dim, prefix, branches, rng.randint(100, 900) if branches else 0,
                      1, _between(rng, 1, 800), page=rng.choice([16, 16, 32]), dtype=dtype, loners=rng.choice([0, 0, 1]) if rows > 3 else 0,
                      softcap=rng.choice([0.0, 0.0, 30.0]), sink=rng.random() < 0.2)


# ------------------------------------------------------------------------------------------------ inputs
def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(int(seed) % (1 << 62))


def _lengths(case, rng):
    """Keys of every request's own behind what it shares."""
    return [int(round(math.exp(v))) for v in
            rng.uniform(math.log(case["own_low"]), math.log(case["own_high"]), case["rows"])]


def prepare(case, seed):
    state = _inputs(case, seed)
    if own and case["op"] == "attention":
        from tokenizer_amd.kernels import get_ops
        # The batch's sharing is looked up when its requests change, not at every layer and token.
        state["plan"] = get_ops().plan_shared_prefixes(state["table_host"], state["positions_host"], case["page"], case["heads"],
                                                       case["kv"], case["dim"], _TYPES[case["dtype"]], DEVICE)
    return state


def _inputs(case, seed):
    gen, rng = _generator(seed), np.random.default_rng(int(seed) % (1 << 62))
    dtype = _TYPES[case["dtype"]]
    state = dict(case=case)
    if case["op"] == "sampling":
        rows, vocab = case["rows"], case["vocab"]
        # A trained model's logits: a wide hill, and a handful of likely tokens that stand out of it.
        logits = torch.randn((rows, vocab), generator=gen, device=DEVICE) * 2.2
        likely = torch.randint(0, vocab, (rows, 24), generator=gen, device=DEVICE)
        lift = torch.rand((rows, 24), generator=gen, device=DEVICE) * 9.0 + 4.0
        logits.scatter_add_(1, likely, lift)
        if case["banned"]:
            banned = torch.rand((rows, vocab), generator=gen, device=DEVICE) < case["banned"]
            logits.masked_fill_(banned.scatter_(1, likely[:, :3], False), float("-inf"))      # (a grammar leaves something)
        numbers = lambda low, high: torch.tensor(rng.uniform(low, high, rows), dtype=torch.float32, device=DEVICE)
        temperature = numbers(case["temperature_low"], case["temperature_high"])
        if case["greedy"]:
            temperature[::case["greedy"]] = 0.0
        state.update(logits=logits.to(dtype), temperature=temperature,
                     top_k=torch.tensor(rng.integers(case["top_k_low"], case["top_k_high"] + 1, rows), dtype=torch.int32, device=DEVICE),
                     top_p=numbers(case["top_p_low"], case["top_p_high"]), min_p=numbers(case["min_p_low"], case["min_p_high"]),
                     uniform=torch.rand(rows, generator=gen, device=DEVICE))
    elif case["op"] == "copying":
        plane = case["heads"] * case["dim"] * case["page"]
        widths = (plane,) if case["tied"] else (plane, plane)
        pool = torch.empty((case["layers"], case["pages"] * sum(widths)), dtype=dtype, device=DEVICE)
        for layer in pool:
            layer.copy_(torch.randn(layer.shape, generator=gen, device=DEVICE))
        order = rng.permutation(case["pages"])[:2 * case["copied"]].astype(np.int32)
        state.update(pool=pool, widths=widths, src=torch.tensor(order[:case["copied"]], device=DEVICE),
                     dst=torch.tensor(order[case["copied"]:], device=DEVICE))
    else:
        heads, kv, dim, page, rows = case["heads"], case["kv"], case["dim"], case["page"], case["rows"]
        whole = lambda keys: -(-keys // page)
        # (What is shared is whole pages; a prefix that ends inside a page is shared up to there.)
        shared, branch, together = case["prefix"] // page, case["branch"] // page, rows - case["loners"]
        lengths, tables, used = _lengths(case, rng), [], 0

        def fresh(count):
            nonlocal used
            used += count
            return list(range(used - count, used))

        prefix = fresh(shared)
        runs = [fresh(branch) for _ in range(case["branches"])]
        positions = []
        for row in range(rows):
            if row < together:
                table = prefix + (runs[row * len(runs) // together] if runs else [])
            else:
                table = fresh(shared)
            keys = len(table) * page + lengths[row]
            positions.append(keys - 1)
            tables.append(table + fresh(whole(lengths[row])))
        n_pages, width = used + 3, max(len(t) for t in tables) + 2
        where = rng.permutation(n_pages).astype(np.int32)
        block_table = np.full((rows, width), -1, dtype=np.int32)
        for row, table in enumerate(tables):
            block_table[row, :len(table)] = where[table]
        mixed = rng.permutation(rows)                 # requests come in no order
        block_table, positions = block_table[mixed], [positions[r] for r in mixed]
        normal = lambda *shape: torch.randn(shape, generator=gen, device=DEVICE)
        qkv = normal(rows, (heads + 2 * kv) * dim)
        qkv[:, :heads * dim] *= 2.0                   # scores spread as a trained model's
        state.update(qkv=qkv.to(dtype), k_pages=normal(n_pages, kv, page, dim).to(dtype), v_pages=normal(n_pages, kv, dim, page).to(dtype),
                     positions_host=positions, table_host=block_table, positions=torch.tensor(positions, dtype=torch.int32, device=DEVICE),
                     block_table=torch.tensor(block_table, device=DEVICE), scale=1.0 / math.sqrt(dim),
                     softcap=case["softcap"] or None, sinks=normal(heads) if case["sink"] else None, plan=None)
    return state


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    return _PASSES[state["case"]["op"]][1 if own else 0](state)


def _plain_sampling(s):
    ordered, index = torch.sort(s["logits"].to(torch.float64), dim=1, descending=True, stable=True)
    temperature = s["temperature"].to(torch.float64)[:, None]
    # (In 64 bits: long sums, and numbers next to the border of a token.)
    weight = torch.exp((ordered - ordered[:, :1]) / torch.where(temperature > 0, temperature, 1.0))
    place = torch.arange(ordered.shape[1], device=ordered.device)[None]
    top_k, top_p = s["top_k"][:, None], s["top_p"].to(torch.float64)[:, None]
    weight = torch.where((top_k > 0) & (place >= top_k), 0.0, weight)
    running = torch.cumsum(weight, dim=1)
    # A token goes once what stands before it has reached the share.
    reached = torch.cat([torch.zeros_like(running[:, :1], dtype=torch.bool), running[:, :-1] >= top_p * running[:, -1:]], dim=1)
    weight = torch.where((top_p < 1.0) & reached, 0.0, weight)
    weight = torch.where(weight >= s["min_p"].to(torch.float64)[:, None], weight, 0.0)
    running = torch.cumsum(weight, dim=1)
    past = running > s["uniform"].to(torch.float64)[:, None] * running[:, -1:]
    pick = torch.where(past, place, ordered.shape[1]).amin(dim=1)
    last = torch.where(weight > 0, place, 0).amax(dim=1)
    pick = torch.where(s["temperature"] > 0, torch.minimum(pick, last), 0)
    return index.gather(1, pick[:, None])[:, 0].to(torch.int32)


def _own_sampling(s):
    from tokenizer_amd.kernels import get_ops
    return get_ops().sample_filtered(s["logits"], s["temperature"], s["top_k"], s["top_p"], s["min_p"], s["uniform"])


def _plain_copying(s):
    n_pages = s["case"]["pages"]
    src, dst = s["src"].long(), s["dst"].long()
    for layer in s["pool"]:
        at = 0
        for width in s["widths"]:
            plane = layer[at:at + n_pages * width].view(n_pages, width)
            plane[dst] = plane[src]
            at += n_pages * width
    return s["pool"]


def _own_copying(s):
    from tokenizer_amd.kernels import get_ops
    return get_ops().copy_pages(s["pool"], s["case"]["pages"], s["widths"], s["src"], s["dst"])


def _plain_attention(s):
    case = s["case"]
    heads, kv, dim, page = case["heads"], case["kv"], case["dim"], case["page"]
    group = heads // kv
    out = torch.empty((case["rows"], heads * dim), dtype=s["qkv"].dtype, device=s["qkv"].device)
    for row, position in enumerate(s["positions_host"]):
        pages = s["block_table"][row, :position // page + 1].long()
        keys = s["k_pages"][pages].to(torch.float32).transpose(0, 1).reshape(kv, -1, dim)[:, :position + 1]
        values = s["v_pages"][pages].to(torch.float32).permute(1, 0, 3, 2).reshape(kv, -1, dim)[:, :position + 1]
        query = s["qkv"][row, :heads * dim].to(torch.float32).view(kv, group, dim)
        scores = torch.matmul(query, keys.transpose(1, 2).contiguous()) * s["scale"]
        if s["softcap"]:
            scores = s["softcap"] * torch.tanh(scores / s["softcap"])
        high = scores.amax(dim=2, keepdim=True)
        if s["sinks"] is not None:
            sink = s["sinks"].view(kv, group, 1)
            high = torch.maximum(high, sink)
        weight = torch.exp(scores - high)
        below = weight.sum(dim=2, keepdim=True)
        if s["sinks"] is not None:
            below = below + torch.exp(sink - high)
        out[row] = (torch.matmul(weight, values) / below).reshape(-1).to(out.dtype)
    return out


def _own_attention(s):
    from tokenizer_amd.kernels import get_ops
    case = s["case"]
    out = torch.empty((case["rows"], case["heads"] * case["dim"]), dtype=s["qkv"].dtype, device=s["qkv"].device)
    return get_ops().shared_prefix_attention(s["qkv"], out, s["k_pages"], s["v_pages"], s["positions"], s["block_table"], s["plan"],
                                             case["heads"], case["kv"], case["dim"], s["scale"], sinks=s["sinks"], softcap=s["softcap"])


_PASSES = {"sampling": (_plain_sampling, _own_sampling), "copying": (_plain_copying, _own_copying),
           "attention": (_plain_attention, _own_attention)}


# ------------------------------------------------------------------------------------------------ work
def work(case):
    size = 2 if case["dtype"] == "bfloat16" else 4
    if case["op"] == "sampling":
        # Every logit once; an exponential, a product and two sums for each.
        return {"bytes": case["rows"] * (case["vocab"] * size + 24), "flops": 4 * case["rows"] * case["vocab"]}
    if case["op"] == "copying":
        page = case["heads"] * case["dim"] * case["page"] * size * (1 if case["tied"] else 2)
        return {"bytes": case["copied"] * (2 * case["layers"] * page + 8), "flops": 0}
    page, rows, together = case["page"], case["rows"], case["rows"] - case["loners"]
    shared = case["prefix"] // page * page
    branch = case["branch"] // page * page
    low, high = case["own_low"], case["own_high"]
    own_keys = rows * ((high - low) / math.log(high / low) if high > low else low)      # as spread over the logarithm
    distinct = shared * (1 + case["loners"]) + branch * case["branches"] + own_keys
    seen = rows * shared + together * (branch if case["branches"] else 0) + own_keys
    return {"bytes": int(distinct * 2 * case["kv"] * case["dim"] * size + 2 * rows * case["heads"] * case["dim"] * size),
            "flops": int(4 * seen * case["heads"] * case["dim"])}


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    if case["op"] == "copying":
        return None                                  # bits are copied, nothing is computed
    state = _inputs(case, seed)
    if case["op"] == "sampling":
        columns = ("temperature", "top_k", "top_p", "min_p", "uniform")
        settings = zip(*(state[name].cpu().numpy().astype(np.float64) for name in columns))
        picked = [_draw_of(row, *numbers) for row, numbers in zip(state["logits"].to(torch.float64).cpu().numpy(), settings)]
        return torch.tensor(picked, dtype=torch.int64)
    heads, kv, dim, page = case["heads"], case["kv"], case["dim"], case["page"]
    answers = []
    for row, position in enumerate(state["positions_host"]):
        at = torch.arange(position + 1, device=DEVICE)
        pages, slot = state["block_table"][row].long()[at // page], at % page
        rows = []
        for g in range(kv):
            query = state["qkv"][row, :heads * dim].view(heads, dim)[g * heads // kv:(g + 1) * heads // kv].double()
            scores = query @ state["k_pages"][pages, g, slot].double().T.contiguous() * state["scale"]
            if case["softcap"]:
                scores = torch.tanh(scores / case["softcap"]) * case["softcap"]
            mass = torch.logsumexp(scores, dim=1)
            if case["sink"]:
                mass = torch.logaddexp(mass, state["sinks"].double()[g * heads // kv:(g + 1) * heads // kv])
            rows.append(torch.exp(scores - mass[:, None]) @ state["v_pages"][pages, g, :, slot].double())
        answers.append(torch.cat(rows).reshape(-1))
    return torch.stack(answers)


def _draw_of(logits, temperature, top_k, top_p, min_p, uniform):
    """One row's draw, token by token as it is defined (NumPy, 64 bits)."""
    order = np.lexsort((np.arange(logits.size), -logits))
    if temperature == 0.0:
        return int(order[0])
    kept = order[:int(top_k)] if top_k > 0 else order
    weight = np.exp((logits[kept] - logits[order[0]]) / temperature)
    if top_p < 1.0:
        reached = np.nonzero(np.cumsum(weight) >= top_p * weight.sum())[0]
        weight = weight[:reached[0] + 1 if reached.size else weight.size]
    weight = weight[weight >= min_p]
    past = np.nonzero(np.cumsum(weight) > uniform * weight.sum())[0]
    return int(kept[past[0] if past.size else weight.size - 1])
