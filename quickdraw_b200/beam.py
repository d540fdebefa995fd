"""Beam search over ``BatchDecode`` (the reference generates greedily, quickdraw/engine/engine.py:129-148): the choice of the
best continuations, the beams' states in the order of their parents, and the search itself.
"""

from __future__ import annotations

import torch

from ._lib import ptr
from .paged import PagedBatchState, _is_ids, device_status, launch, scratch_size
from .state import DecodeState

BF16 = torch.bfloat16
MOST_BEAMS = 32
MOST_ROWS = 7000            # that reorder_states puts in order at once


def beam_select(logits: torch.Tensor, scores: torch.Tensor, *, finished: torch.Tensor | None = None, eos: int | None = None,
                candidates: int | None = None):
    """The best continuations of every group of beams by ``scores[b, i] + log_softmax(logits[b, i])[v]``, the lowest (i, v) among equals:
    (fp32 scores, int32 parents ``b * beams + i``, int64 tokens).

    logits    [batch, beams, vocab], bf16 or fp32, rows any distance apart
    scores    fp32 [batch, beams]; a beam whose score is not finite, or whose logits have no finite log-sum-exp (NaN, +inf, nothing but
              -inf), has no continuation, and what is none counts -inf
    finished  bool [batch, beams]: such a beam has one continuation, ``eos``, at no cost
    candidates  None: as many as beams, [batch, beams], a beam's best continuation in the beam's own place (whose state then need not
              move), the others in the places left, best first.  A number: that many, best first.  At most 32 of beams and candidates."""
    assert logits.is_cuda and logits.ndim == 3 and logits.dtype in (BF16, torch.float32), "bf16 or fp32 logits [batch, beams, vocab] on a CUDA device"
    batch, beams, vocab = logits.shape
    device = logits.get_device()
    assert batch > 0 and 0 < beams <= MOST_BEAMS and vocab > 0 and batch * beams <= 65535, "1 to 32 beams"
    apart = logits.stride(1) if beams > 1 else logits.stride(0)            # (of one beam or one group the stride says nothing)
    assert logits.stride(2) == 1 and (batch == 1 or beams == 1 or logits.stride(0) == beams * apart), "rows of contiguous logits, evenly apart"
    assert scores.dtype is torch.float32 and scores.shape == (batch, beams) and scores.is_contiguous() and scores.get_device() == device
    if finished is not None:
        assert finished.dtype is torch.bool and finished.shape == (batch, beams) and finished.is_contiguous() and finished.get_device() == device
        assert eos is not None and 0 <= eos < vocab, "finished beams go on with eos"
    placed = candidates is None
    count = beams if placed else candidates
    assert 0 < count <= MOST_BEAMS and count <= beams * vocab, "1 to 32 candidates, no more than there are continuations"
    scores_out = torch.empty_like(scores) if placed else scores.new_empty((batch, count))
    parents, tokens = torch.empty_like(scores_out, dtype=torch.int32), torch.empty_like(scores_out, dtype=torch.long)
    size = scratch_size(device, "qd_beam_scratch_bytes", batch, beams, vocab, count)
    scratch = scores.new_empty(size // 4) if size else None
    launch(logits, "qd_beam_select", ptr(logits), apart, int(logits.dtype is torch.float32), ptr(scores),
           ptr(finished), 0 if finished is None else eos, ptr(scores_out), ptr(parents), ptr(tokens), ptr(scratch), batch, beams, vocab, count, int(placed))
    return scores_out, parents, tokens


def reorder_states(states, parents: torch.Tensor, *, status: torch.Tensor | None = None) -> None:
    """``state[b] = old state[parents[b]]`` in place, for tensors [sequences, ...] that do not overlap (rows contiguous, any distance apart): -1 is
    a row of zeros, a row that is its own parent is not touched, one whose parent is no row neither (a bit of ``status``).  At most 7000 rows."""
    states = [states] if isinstance(states, torch.Tensor) else list(states)
    assert parents.is_cuda and parents.ndim == 1 and _is_ids(parents, parents.get_device(), *parents.shape) and parents.numel() > 0
    device, count = parents.get_device(), parents.numel()
    assert count <= MOST_ROWS, "1 to 7000 rows"
    status = device_status(parents.device) if status is None else status
    assert _is_ids(status, device, 1)
    rows = []
    for t in states:
        shape, strides = t.shape, t.stride()
        row = t.numel() // count
        assert t.get_device() == device and len(shape) >= 1 and shape[0] == count, "tensors [sequences, ...] on one device"
        assert (t.is_contiguous() or t[0].is_contiguous()) and (count == 1 or strides[0] >= row), "contiguous rows that do not overlap"
        size = t.element_size()
        if row:
            rows += (ptr(t), row * size, strides[0] * size)
    assert 3 * len(set(rows[::3])) == len(rows), "each tensor once"
    for first in range(0, len(rows), 12):
        some = rows[first:first + 12]
        launch(parents, "qd_reorder_states", *some, *(None, 0, 0) * (4 - len(some) // 3), ptr(parents), ptr(status), count)


@torch.inference_mode()
def beam_search(decoder, prompts: list[list[int]], beams: int, max_tokens: int, *, eos: int | None = None, length_penalty: float = 0.0,
                page: int = 64, graph: bool = False) -> list[list[tuple[list[int], float]]]:
    """The ``beams`` best answers to every prompt, each (token ids, EOS included; log-probability / length ** length_penalty), best first.

    ``decoder`` is a ``BatchDecode``; all beams of all prompts are one batch.  The beams of a prompt share the pages of what they have in
    common; a step appends a token to every beam, chooses, and forks the state by the parents.  The host waits for the device only
    where ``eos`` is given, every sixteenth step, to see whether all have ended.  The choice goes by the log-probability alone, of
    beams that have ended as of the others: ``length_penalty`` orders the answers that are left at the end.  ``graph``: the step
    replayed from a CUDA graph (``BatchDecode.graph_step``)."""
    config = decoder.ckpt.config
    assert prompts and all(len(p) > 0 for p in prompts), "at least one prompt of at least one token"
    assert 1 <= beams <= MOST_BEAMS and max_tokens >= 0, "1 to 32 beams"
    assert all(0 <= t < config.vocab_size for p in prompts for t in p), "token id outside the vocabulary"
    assert eos is None or 0 <= eos < config.vocab_size
    groups, longest = len(prompts), max(len(p) for p in prompts)
    if max_tokens == 0:
        return [[([], 0.0)] for _ in prompts]
    device = decoder.device
    count = groups * beams
    # what the beams of a prompt share, its full pages and what each adds
    pages = sum(-(-len(p) // page) for p in prompts) + count * (-(-(max_tokens + page) // page) + 1)
    state = PagedBatchState(config, count, longest + max_tokens, device, pages, page)
    for g, prompt in enumerate(prompts):
        if len(prompt) > 1:
            one = DecodeState.allocate(config, len(prompt), device)
            tokens = torch.tensor(prompt[:-1], dtype=torch.long).to(device, non_blocking=True)
            for first in range(0, len(prompt) - 1, 2048):
                decoder.run(tokens[first:first + 2048], first, one)
            one.position = len(prompt) - 1
            state.admit(g * beams, one)
    first = torch.arange(groups, dtype=torch.int32, device=device).repeat_interleave(beams) * beams
    state.fork(first)
    tokens = torch.tensor([p[-1] for p in prompts], dtype=torch.long).to(device, non_blocking=True).repeat_interleave(beams)
    scores = torch.full((groups, beams), -torch.inf, device=device)
    scores[:, 0] = 0.0                                     # all beams of a prompt are alike so far: one of them counts
    finished = torch.zeros((groups, beams), dtype=torch.bool, device=device)
    history = []
    try:
        for step in range(max_tokens):
            if graph:
                _, logits = decoder.graph_step(tokens, state)
            else:
                _, logits = decoder.step(tokens, state, positions_checked=True)
            scores, parents, chosen = beam_select(logits.view(groups, beams, -1), scores, finished=None if eos is None else finished, eos=eos)
            tokens = chosen.view(-1)
            history.append((parents.view(-1), tokens))
            if eos is not None:
                finished = finished.view(-1)[parents.view(-1).long()].view(groups, beams) | (chosen == eos)
                if step % 16 == 15 and bool(finished.all()):
                    break
            if step + 1 < max_tokens:
                state.fork(parents.view(-1))
    finally:
        decoder.forget(state)                              # a captured step holds the pages; nobody else can drop it
    word = state.cache.check()
    assert word == 0, f"the search ran out of pages (status {word})"
    back, ids = torch.stack([p for p, _ in history]).tolist(), torch.stack([t for _, t in history]).tolist()
    total = scores.view(-1).tolist()
    results: list[list[tuple[list[int], float]]] = []
    for g in range(groups):
        answers = []
        for b in range(g * beams, (g + 1) * beams):
            if total[b] == -float("inf"):
                continue
            at, answer = b, []
            for s in reversed(range(len(ids))):
                answer.append(ids[s][at])
                at = back[s][at]
            answer.reverse()
            if eos is not None and eos in answer:
                answer = answer[:answer.index(eos) + 1]
            answers.append((answer, total[b] / len(answer) ** length_penalty))
        results.append(sorted(answers, key=lambda a: -a[1]))
    return results
