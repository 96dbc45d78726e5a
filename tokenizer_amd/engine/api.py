"""Entry points in the manner of qwen-infer's library (qwen-infer/src/lib.rs:14-24, 116-130):
`generate`, `generate_with`, `greedy_tokens`."""
from __future__ import annotations

import dataclasses
import time

from ..cache import OutOfPages
from .batch import StepEntry
from .generate import (Control, GenerateParams, Generated, SampleCursor, Sampled, StopReason, _go_on, _no_bytes,
                       filters_of)


def _next(engine, cursor: SampleCursor, logits, token_bytes, on_chunk):
    """Pick the next id on the device (greedy, or a warm draw with the cursor's next uniform number) and hand
    it to the cursor; an engine without a device sampler gets the logits row drawn on the host."""
    if cursor.exhausted:
        return cursor.push_token(0, token_bytes, on_chunk)        # finishes, nothing is drawn
    if cursor.is_greedy:
        token = engine.argmax(logits, [0])[0]
    elif hasattr(engine, "sample"):
        token = engine.sample(logits, [0], [cursor.params.temperature], [cursor.params.top_p],
                              [cursor.next_uniform()], *filters_of([cursor]))[0]
    else:
        return cursor.push_logits(engine.rows_to_host(logits, [0])[0], token_bytes, on_chunk)
    return cursor.push_token(token, token_bytes, on_chunk)


def _engine_for(model_or_engine, prompt, params):
    """`generate(model, ...)` as in the reference: a bare model gets an engine sized for this one request."""
    if hasattr(model_or_engine, "step"):
        return model_or_engine
    from .engine import Engine
    return Engine(model_or_engine, max_tokens=len(prompt) + params.max_tokens + 1, max_requests=1)


def generate_with(engine, prompt: list[int], params: GenerateParams, token_bytes=_no_bytes,
                  on_chunk=_go_on) -> Generated:
    """Prefill `prompt`, then sample up to `params.max_tokens` ids, one cached forward per id.

    The forward after the last allowed sample is not run; `max_tokens == 0` still runs the prompt;
    the chunk callback is probed once with "" after the prompt so that a caller who is gone
    cancels before the first draw (qwen-infer/src/generate.rs:340-394).
    """
    if not prompt:
        raise ValueError("prompt encoded to no tokens")
    engine = _engine_for(engine, prompt, params)
    cursor = SampleCursor(params)
    rid = ("generate", id(cursor))
    engine.add_request(rid)
    try:
        started = time.perf_counter()
        logits = engine.step([StepEntry(rid, list(prompt), [len(prompt) - 1] if params.max_tokens > 0 else [])])
        if params.max_tokens > 0:
            engine.argmax(logits, [0])                 # waits for the prompt's forward, so the clock is honest
        prefill = time.perf_counter() - started
        started = time.perf_counter()
        if params.max_tokens == 0:
            done = cursor.finish_without_sample(on_chunk)
        elif on_chunk("") == Control.Stop:
            done = Sampled([], "", [], StopReason.Cancelled, 0)
        else:
            outcome = _next(engine, cursor, logits, token_bytes, on_chunk)
            on_device = hasattr(engine, "decode_greedy") and (
                cursor.is_greedy or (hasattr(engine, "decode_sampled") and hasattr(engine, "sample")))
            if not isinstance(outcome, Sampled) and on_device:
                # The remaining steps run back to back on the device, greedy picks or draws (the cursor gives a
                # step's uniform number when it is launched); the cursor sees each id one step late and ends the
                # run when it stops (at most one forward is then run for nothing).
                ended = []

                def on_step(_k, ids):
                    result = cursor.push_token(ids[0], token_bytes, on_chunk)
                    if isinstance(result, Sampled):
                        ended.append(result)
                        return False
                    return True

                if cursor.is_greedy:
                    engine.decode_greedy([rid], [int(outcome)], params.max_tokens - cursor.produced, on_step)
                else:
                    draw = lambda _k: ([params.temperature], [params.top_p], [cursor.next_uniform()], *filters_of([cursor]))
                    engine.decode_sampled([rid], [int(outcome)], params.max_tokens - cursor.produced, draw, on_step)
                outcome = ended[0]
            while not isinstance(outcome, Sampled):
                logits = engine.step([StepEntry(rid, [int(outcome)], [0])])
                outcome = _next(engine, cursor, logits, token_bytes, on_chunk)
            done = outcome
        decode = time.perf_counter() - started
    finally:
        engine.end_request(rid)
    return Generated(done.tokens, done.text, done.chunks, done.reason, done.completion_tokens, prefill, decode)


def generate(engine, prompt, params: GenerateParams, token_bytes=_no_bytes, tokenizer=None) -> Generated:
    """Generate from token ids, or from text when a `tokenizer` (tokenizer_amd.Tokenizer) is given: the text is
    encoded with it and the sampled ids are decoded with it.  `engine`: an `Engine` or a bare model."""
    if isinstance(prompt, str):
        if tokenizer is None:
            raise ValueError("a text prompt needs a tokenizer")
        prompt = tokenizer.encode(prompt)
    if tokenizer is not None and token_bytes is _no_bytes:
        token_bytes = lambda token: tokenizer.decode_bytes([token])
    return generate_with(engine, prompt, params, token_bytes, _go_on)


def generate_answers(engine, prompt, params: GenerateParams, n: int, token_bytes=_no_bytes, tokenizer=None) -> list[Generated]:
    """`n` answers to one prompt, decoded together: the prompt is run once, its request forked (the answers share its pages of the
    cache, which every decode step goes through once for all of them), and answer i is drawn with the seed `params.seed` + i.
    `engine`: an `Engine` with room for `n` requests, or a bare model; `prompt`, `token_bytes`, `tokenizer` as for `generate`.
    The times of an answer are those of all.  Where the pool runs out of pages while they decode, the newest answers' requests go, and come
    back, the prompt and what they had drawn run again, when the others have ended; `OutOfPages` where there is no room for the
    forks to begin with, or for a single answer."""
    if n < 1:
        raise ValueError("at least one answer")
    if isinstance(prompt, str):
        if tokenizer is None:
            raise ValueError("a text prompt needs a tokenizer")
        prompt = tokenizer.encode(prompt)
    if not prompt:
        raise ValueError("prompt encoded to no tokens")
    if tokenizer is not None and token_bytes is _no_bytes:
        token_bytes = lambda token: tokenizer.decode_bytes([token])
    cursors = [SampleCursor(dataclasses.replace(params, seed=params.seed + i)) for i in range(n)]
    if not hasattr(engine, "step"):
        from .engine import Engine
        page = 16
        engine = Engine(engine, num_pages=-(-len(prompt) // page) + n * (params.max_tokens // page + 2), page_size=page, max_requests=n)
    rids = [("answer", id(cursors[0]), i) for i in range(n)]
    done: list[Sampled | None] = [None] * n
    started = time.perf_counter()
    engine.add_request(rids[0])
    live = [rids[0]]
    try:
        logits = engine.step([StepEntry(rids[0], list(prompt), [len(prompt) - 1] if params.max_tokens > 0 else [])])
        if params.max_tokens == 0:
            first = []
            done = [cursor.finish_without_sample() for cursor in cursors]
        elif cursors[0].is_greedy:
            first = engine.argmax(logits, [0]) * n
        else:
            first = engine.sample(logits, [0] * n, [params.temperature] * n, [params.top_p] * n, [c.next_uniform() for c in cursors],
                                  *filters_of(cursors))
        prefill = time.perf_counter() - started
        started = time.perf_counter()
        tokens: dict[int, int] = {}                       # the answers that go on, and their next tokens

        def take(answers, ids) -> bool:
            """Hands every answer that goes on its new token; False if one ended."""
            before = len(tokens)
            for i, token in zip(answers, ids):
                if done[i] is None:
                    outcome = cursors[i].push_token(int(token), token_bytes)
                    if isinstance(outcome, Sampled):
                        done[i] = outcome
                        tokens.pop(i, None)
                    else:
                        tokens[i] = int(outcome)
            return len(tokens) >= before

        take(range(n), first)
        going_on = sorted(tokens)
        if going_on:
            # (The prompt's own request is the first answer that goes on.)
            names = {i: rids[i] if at else rids[0] for at, i in enumerate(going_on)}
            others = [names[i] for i in going_on[1:]]
            if others:
                engine.fork_request(rids[0], others)
                live += others
        waiting: list[int] = []                           # answers whose requests had to go, the oldest first
        while tokens or waiting:
            if not tokens:
                back = _come_back(engine, prompt, [(names[i], cursors[i].tokens) for i in waiting], live)
                tokens.update((i, cursors[i].tokens[-1]) for i in waiting[:back])
                waiting = waiting[back:]
            answers = sorted(tokens)
            steps = min(min(params.max_tokens - cursors[i].produced for i in answers), ANSWER_BURST)
            steps = engine.steps_with_pages([names[i] for i in answers], steps)
            if steps == 0 and len(answers) > 1:
                waiting.insert(0, answers[-1])
                engine.end_request(names[answers[-1]])
                live.remove(names[answers[-1]])
                tokens.pop(answers[-1])
                continue
            steps, handled = max(1, steps), 0             # (no page for a single answer: its step says so)

            def on_step(_k, ids):
                nonlocal handled
                handled += 1
                return take(answers, ids)

            given = [cursors[i] for i in answers]
            rows, ids = [names[i] for i in answers], [tokens[i] for i in answers]
            if cursors[0].is_greedy:
                picked = engine.decode_greedy(rows, ids, steps, on_step)
            else:
                draw = lambda _k: ([params.temperature] * len(given), [params.top_p] * len(given), [c.next_uniform() for c in given],
                                   *filters_of(given))
                picked = engine.decode_sampled(rows, ids, steps, draw, on_step)
            for ids in picked[handled:]:                  # the step that was under way when an answer ended
                take(answers, ids)
            for i in answers:
                if done[i] is not None:
                    engine.end_request(names[i])
                    live.remove(names[i])
    finally:
        for rid in live:
            engine.end_request(rid)
    decode = time.perf_counter() - started
    return [Generated(d.tokens, d.text, d.chunks, d.reason, d.completion_tokens, prefill, decode) for d in done]


def _come_back(engine, prompt, answers, live) -> int:
    """Makes requests for answers, (name, tokens drawn) each, that hold the prompt and all but the last of those tokens: the prompt is run
    once, for the first of them, and as many others are its forks as there are pages for.  Returns how many answers are back."""
    names = []

    def fits() -> bool:
        missing = [0] * len(engine.cache.groups)
        for name, drawn in answers[:len(names)]:
            for group, pages in enumerate(engine.cache.pages_missing(name, len(prompt) + len(drawn))):
                missing[group] += pages
        return all(pages <= group.allocator.available() for pages, group in zip(missing, engine.cache.groups))

    for name, _ in answers:
        if not names:
            engine.add_request(name)
            live.append(name)
            engine.step([StepEntry(name, list(prompt), [])])
        else:
            try:
                engine.fork_request(names[0], [name])
            except OutOfPages:
                break
            live.append(name)
        names.append(name)
        if len(names) > 1 and not fits():
            names.pop()
            engine.end_request(name)
            live.remove(name)
            break
    entries = [StepEntry(name, list(drawn[:-1]), []) for name, drawn in answers[:len(names)] if len(drawn) > 1]
    if entries:
        engine.step(entries)
    return len(names)


ANSWER_BURST = 16       # decode steps of answers that run back to back before finished ones leave


def greedy_tokens(engine, prompt: list[int], new_tokens: int) -> list[int]:
    """Greedy ids through the cache (the reference's `greedy_tokens` recomputes everything each step;
    the ids are the same)."""
    return generate(engine, prompt, GenerateParams.greedy(new_tokens)).tokens
