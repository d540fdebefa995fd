"""Refusals of the paged cache's and the beams' entry points, and what their drivers pass on, without a GPU."""

import contextlib
import math

import pytest
import torch

from quickdraw_b200 import _lib, beam, paged, synthetic
from tests import paged_plain as plain

BF16, F32, I32 = torch.bfloat16, torch.float32, torch.int32


class AsIfOnGpu(torch.Tensor):
    is_cuda = property(lambda self: True)


def on_gpu(t):
    return t.as_subclass(AsIfOnGpu)


@pytest.fixture
def calls(monkeypatch):
    """The library replaced by a recorder that knows how many arguments each entry point takes."""
    seen = []

    def record(name, *args):
        assert len(args) == len(_lib.SIGNATURES[name]), (name, len(args), len(_lib.SIGNATURES[name]))
        seen.append((name, args))

    monkeypatch.setattr(paged, "call", record)
    monkeypatch.setattr(paged, "stream_of", lambda t: None)
    return seen


def attention_arguments(**changes):
    given = dict(q=torch.zeros(2, 16, 256, dtype=BF16), k_pages=torch.zeros(9, 16, 2, 256, dtype=BF16), v_pages=torch.zeros(9, 16, 2, 256, dtype=BF16),
                 table=torch.zeros(2, 5, dtype=I32), lengths=torch.zeros(2, dtype=I32)) | changes
    return {name: on_gpu(t) if isinstance(t, torch.Tensor) else t for name, t in given.items()}


def test_attention_passes_its_arguments(calls):
    out = paged.paged_attention(**attention_arguments())
    assert out.shape == (2, 16, 256) and out.dtype is BF16 and [name for name, _ in calls] == ["qd_paged_attention"]
    args = calls[0][1]
    assert args[1:3] == (16 * 256, 256) and args[5:8] == (16 * 2 * 256, 2 * 256, 256) and args[16:25] == (2, 16, 2, 256, 9, 16, 5, 0, 0)
    assert args[25] == 1 / 16 and args[26] == 0


@pytest.mark.parametrize("changes", [
    dict(q=torch.zeros(2, 16, 256, dtype=torch.float16)), dict(q=torch.zeros(16, 256, dtype=BF16)), dict(q=torch.zeros(2, 15, 256, dtype=BF16)),
    dict(q=torch.zeros(2, 16, 256)), dict(q=torch.zeros(3, 16, 256, dtype=BF16)), dict(q=torch.zeros(2, 256, 16, dtype=BF16).transpose(1, 2)),
    dict(q=torch.zeros(0, 16, 256, dtype=BF16), table=torch.zeros(0, 5, dtype=I32), lengths=torch.zeros(0, dtype=I32)),
    dict(q=torch.zeros(2, 16, 264, dtype=BF16), k_pages=torch.zeros(9, 16, 2, 264, dtype=BF16), v_pages=torch.zeros(9, 16, 2, 264, dtype=BF16)),
    dict(q=torch.zeros(2, 16, 12, dtype=BF16), k_pages=torch.zeros(9, 16, 2, 12, dtype=BF16), v_pages=torch.zeros(9, 16, 2, 12, dtype=BF16)),
    dict(k_pages=torch.zeros(9, 16, 2, 256)), dict(v_pages=torch.zeros(8, 16, 2, 256, dtype=BF16)), dict(k_pages=torch.zeros(9, 2, 256, dtype=BF16)),
    dict(k_pages=torch.zeros(9, 2, 16, 256, dtype=BF16).transpose(1, 2)), dict(k_pages=torch.zeros(0, 16, 2, 256, dtype=BF16), v_pages=torch.zeros(0, 16, 2, 256, dtype=BF16)),
    dict(k_pages=torch.zeros(9 * 16 * 2 * 256 + 1, dtype=BF16)[1:].view(9, 16, 2, 256)),
    dict(table=torch.zeros(2, 5, dtype=torch.long)), dict(table=torch.zeros(3, 5, dtype=I32)), dict(table=torch.zeros(2, 0, dtype=I32)),
    dict(table=torch.zeros(5, 2, dtype=I32).T), dict(lengths=torch.zeros(3, dtype=I32)), dict(lengths=torch.zeros(2)), dict(window=-1), dict(sinks=3),
    dict(window=3, sinks=-1), dict(gate=torch.zeros(2, 16, 256)), dict(gate=torch.zeros(2, 16, 128, dtype=BF16))])
def test_attention_refuses(calls, changes):
    with pytest.raises(AssertionError):
        paged.paged_attention(**attention_arguments(**changes))
    assert not calls


def test_attention_refuses_the_cpu(calls):
    given = attention_arguments()
    with pytest.raises(AssertionError, match="CUDA"):
        paged.paged_attention(**{name: t.as_subclass(torch.Tensor) for name, t in given.items()})


def page_arguments(**changes):
    given = dict(k_pages=torch.zeros(9, 3, 16, 2, 64, dtype=BF16), v_pages=torch.zeros(9, 3, 16, 2, 64, dtype=BF16), table=torch.zeros(4, 5, dtype=I32),
                 lengths=torch.zeros(4, dtype=I32), refs=torch.zeros(9, dtype=I32), parents=torch.zeros(4, dtype=I32), status=torch.zeros(1, dtype=I32)) | changes
    return {name: on_gpu(t) for name, t in given.items()}


def test_forks_and_compactions_pass_their_arguments(calls):
    given = page_arguments()
    out = paged.fork_pages(**given)
    assert [t.shape for t in out] == [(4, 5), (4,), (9,)]
    assert calls[-1][0] == "qd_pages_fork" and calls[-1][1][2:6] == (3 * 16 * 256, 16 * 256, 256, 3) and calls[-1][1][15:19] == (4, 5, 9, 16)
    out = paged.compact_pages(*(given[name] for name in ("k_pages", "v_pages", "table", "refs")))
    assert [t.shape for t in out] == [(4, 5), (9,), ()] and calls[-1][0] == "qd_pages_compact"
    paged.reserve_pages(given["table"], given["lengths"], given["refs"], 16, 3, status=given["status"])
    assert calls[-1][0] == "qd_pages_reserve" and calls[-1][1][3:5] == (None, 3)
    paged.reserve_pages(given["table"], given["lengths"], given["refs"], 16, given["lengths"], status=given["status"])
    assert calls[-1][1][4] == 0


@pytest.mark.parametrize("changes", [
    dict(k_pages=torch.zeros(9, 16, 2, 64, dtype=BF16)), dict(k_pages=torch.zeros(9, 3, 16, 2, 64)), dict(k_pages=torch.zeros(9, 2, 16, 2, 64, dtype=BF16)),
    dict(k_pages=torch.zeros(9, 16, 3, 2, 64, dtype=BF16).transpose(1, 2)),
    dict(k_pages=torch.zeros(9, 3, 16, 1, 4, dtype=BF16), v_pages=torch.zeros(9, 3, 16, 1, 4, dtype=BF16)), dict(refs=torch.zeros(8, dtype=I32)),
    dict(refs=torch.zeros(9)), dict(table=torch.zeros(4, 5)), dict(table=torch.zeros(4, 10, dtype=I32)[:, ::2]), dict(lengths=torch.zeros(5, dtype=I32)),
    dict(parents=torch.zeros(4, dtype=torch.long)), dict(parents=torch.zeros(3, dtype=I32)), dict(status=torch.zeros(2, dtype=I32))])
def test_forks_refuse(calls, changes):
    with pytest.raises(AssertionError):
        paged.fork_pages(**page_arguments(**changes))
    assert not calls


def test_reserves_refuse(calls):
    table, lengths, refs, status = (on_gpu(torch.zeros(*shape, dtype=I32)) for shape in ((4, 5), (4,), (9,), (1,)))
    for page, counts in ((0, 1), (16, -1), (16, torch.zeros(4)), (16, torch.zeros(3, dtype=I32)), (2 ** 30, 1)):
        with pytest.raises(AssertionError):
            paged.reserve_pages(table, lengths, refs, page, counts, status=status)
    assert not calls


@pytest.mark.parametrize("several", [list, iter, set, range])
def test_sequences_end_by_any_row_of_numbers(monkeypatch, several):
    cache = paged.PagedCache(1, 1, 8, 4, 4, 3, 8, "cpu")
    seen = []
    monkeypatch.setattr(cache, "fork", lambda parents: seen.append(parents.tolist()))
    cache.free(range(1, 3) if several is range else several([1, 2]))
    assert seen == [[0, -1, -1]]
    with pytest.raises(AssertionError):
        cache.free(iter([0, 3]))


def test_cache_of_no_size_is_refused():
    for sizes in ((0, 2, 64, 4, 16, 2, 100), (1, 2, 64, 0, 16, 2, 100), (1, 2, 64, 4, 0, 2, 100), (1, 2, 64, 4, 16, 0, 100), (1, 2, 64, 4, 16, 2, 0)):
        with pytest.raises(AssertionError):
            paged.PagedCache(*sizes, "cpu")
    cache = paged.PagedCache(2, 2, 64, 4, 16, 3, 100, "cpu")
    assert cache.table.shape == (3, 7) and bool((cache.table == -1).all()) and cache.pages == 4 and cache.check() == 0
    with pytest.raises(AssertionError):
        cache.free([3])
    config = synthetic.model_config(num_layers=4, vocab_size=64)
    with pytest.raises(AssertionError):
        paged.PagedBatchState(config, 2, 64, "cpu", pages=0)
    state = paged.PagedBatchState(config, 2, 65, "cpu", page=16)
    assert state.cache.pages == 10 and state.cache.k.shape == (10, 1, 16, 2, 256) and state.positions is state.cache.lengths


def test_select_passes_its_arguments(calls):
    logits, scores = on_gpu(torch.zeros(2, 3, 50)), on_gpu(torch.zeros(2, 3))
    out = beam.beam_select(logits, scores)
    assert [(t.shape, t.dtype) for t in out] == [((2, 3), F32), ((2, 3), I32), ((2, 3), torch.long)]
    assert calls[-1][0] == "qd_beam_select" and calls[-1][1][1:3] == (50, 1) and calls[-1][1][10:15] == (2, 3, 50, 3, 1)
    out = beam.beam_select(logits, scores, candidates=6, finished=on_gpu(torch.zeros(2, 3, dtype=torch.bool)), eos=49)
    assert out[0].shape == (2, 6) and calls[-1][1][5] == 49 and calls[-1][1][13:15] == (6, 0)


@pytest.mark.parametrize("logits,scores,kwargs", [
    (torch.zeros(2, 3, 50, dtype=torch.float16), torch.zeros(2, 3), {}), (torch.zeros(6, 50), torch.zeros(2, 3), {}), (torch.zeros(2, 33, 50), torch.zeros(2, 33), {}),
    (torch.zeros(2, 3, 50), torch.zeros(3, 2), {}), (torch.zeros(2, 3, 50), torch.zeros(2, 3, dtype=BF16), {}), (torch.zeros(2, 50, 3).transpose(1, 2), torch.zeros(2, 3), {}),
    (torch.zeros(3, 2, 50).transpose(0, 1), torch.zeros(2, 3), {}), (torch.zeros(2, 3, 50), torch.zeros(2, 3), dict(candidates=0)),
    (torch.zeros(2, 3, 50), torch.zeros(2, 3), dict(candidates=33)), (torch.zeros(2, 3, 5), torch.zeros(2, 3), dict(candidates=16)),
    (torch.zeros(2, 3, 50), torch.zeros(2, 3), dict(finished=torch.zeros(2, 3, dtype=torch.bool))),
    (torch.zeros(2, 3, 50), torch.zeros(2, 3), dict(finished=torch.zeros(2, 3, dtype=torch.bool), eos=50)),
    (torch.zeros(2, 3, 50), torch.zeros(2, 3), dict(finished=torch.zeros(2, 3), eos=5)), (torch.zeros(0, 3, 50), torch.zeros(0, 3), {}),
    (torch.zeros(2, 3, 0), torch.zeros(2, 3), {})])
def test_select_refuses(calls, logits, scores, kwargs):
    with pytest.raises(AssertionError):
        beam.beam_select(on_gpu(logits), on_gpu(scores), **{name: on_gpu(t) if isinstance(t, torch.Tensor) else t for name, t in kwargs.items()})
    assert not calls


def test_reorder_passes_its_arguments_and_refuses(calls):
    parents, status = on_gpu(torch.zeros(3, dtype=I32)), on_gpu(torch.zeros(1, dtype=I32))
    beam.reorder_states([on_gpu(torch.zeros(3, 4)) for _ in range(6)], parents, status=status)
    assert [len(args) for _, args in calls] == [16, 16] and calls[1][1][6] is None and calls[0][1][1:3] == (16, 16)
    calls.clear()
    for state in (torch.zeros(4, 4), torch.zeros(3, 4, 4).transpose(1, 2), torch.zeros(1, 4).expand(3, 4), torch.zeros(())):
        with pytest.raises(AssertionError):
            beam.reorder_states(on_gpu(state), parents, status=status)
    twice = torch.zeros(3, 4)
    with pytest.raises(AssertionError):
        beam.reorder_states([on_gpu(twice), on_gpu(twice)], parents, status=status)
    with pytest.raises(AssertionError):
        beam.reorder_states(on_gpu(torch.zeros(3, 4)), on_gpu(torch.zeros(3, dtype=torch.long)), status=status)
    assert not calls


def test_a_device_s_status_is_not_made_in_a_capture(monkeypatch):
    monkeypatch.setattr(paged, "_status", {})
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(AssertionError):
        paged.device_status(torch.device("cuda", 0))
    word = paged.device_status(torch.device("cpu"))
    assert int(word) == 0 and paged.device_status(torch.device("cpu")) is word


def test_search_refuses():
    class Decoder:
        class ckpt:
            config = synthetic.model_config(num_layers=4, vocab_size=64)
        device = "cpu"
    for prompts, beams, tokens, kwargs in (([], 2, 3, {}), ([[]], 2, 3, {}), ([[1]], 0, 3, {}), ([[1]], 33, 3, {}), ([[64]], 2, 3, {}), ([[1]], 2, -1, {}),
                                           ([[1]], 2, 3, dict(eos=64))):
        with pytest.raises(AssertionError):
            beam.beam_search(Decoder, prompts, beams, tokens, **kwargs)
    assert beam.beam_search(Decoder, [[1], [2]], 2, 0) == [[([], 0.0)], [([], 0.0)]]


def test_plain_forms_agree_with_themselves():
    """The oracle's fork keeps every sequence's rows and counts every entry; its attention of a forked sequence is its parent's."""
    k, v, table, lengths, refs = plain.cache([37, 5, 0, 16], 16, 1, 2, 8, F32, seed=1, spare=6, device="cpu")
    new = plain.fork(k, v, table, lengths, refs, [0, 0, 1, 0], 16)
    assert new[5] == 0 and new[3].tolist() == [37, 37, 5, 37] and int(new[4].sum()) == int((new[2] >= 0).sum())
    q = torch.randn(4, 2, 8, generator=torch.Generator().manual_seed(1))[:1].expand(4, 2, 8)
    out, bound = plain.attention(q, new[0][:, 0], new[1][:, 0], new[2], new[3])
    assert torch.equal(out[0], out[1]) and torch.equal(out[0], out[3]) and not math.isnan(float(out.sum())) and float(bound.max()) < 1e-2


def test_a_captured_step_is_not_replayed_after_a_resize(monkeypatch):
    """Its kernels have the addresses of pools whose memory was given back."""
    from types import SimpleNamespace

    from quickdraw_b200 import batch
    done = []
    monkeypatch.setattr(torch.cuda, "CUDAGraph", lambda: SimpleNamespace(replay=lambda: done.append("replay")))
    monkeypatch.setattr(torch.cuda, "graph", lambda graph: contextlib.nullcontext())
    monkeypatch.setattr(batch, "lib", lambda: SimpleNamespace(qd_set_chained_launches=lambda on: 1))
    monkeypatch.setattr(paged, "compact_pages", lambda k, v, table, refs: (table.clone(), refs.clone(), torch.zeros((), dtype=I32)))
    decoder = batch.BatchDecode.__new__(batch.BatchDecode)
    decoder._graphs = {}
    monkeypatch.setattr(decoder, "step", lambda tokens, state, positions_checked=False: done.append("capture" if positions_checked else "eager"), raising=False)
    state, tokens = paged.PagedBatchState(synthetic.model_config(num_layers=4, vocab_size=64), 2, 64, "cpu", page=16), torch.zeros(2, dtype=torch.long)
    for _ in range(3):
        decoder.graph_step(tokens, state)
    assert done == ["eager", "capture", "replay", "replay"]
    for pages in (5, 5, 9):
        done.clear()
        state.cache.resize(pages)
        for _ in range(3):
            decoder.graph_step(tokens, state)
        assert done == ["eager", "capture", "replay", "replay"], pages


def test_reorder_refuses_more_rows_than_it_holds(calls):
    status = on_gpu(torch.zeros(1, dtype=I32))
    beam.reorder_states(on_gpu(torch.zeros(7000, 1)), on_gpu(torch.zeros(7000, dtype=I32)), status=status)
    assert calls.pop()[1][14] == 7000
    with pytest.raises(AssertionError, match="7000"):
        beam.reorder_states(on_gpu(torch.zeros(7001, 1)), on_gpu(torch.zeros(7001, dtype=I32)), status=status)
    assert not calls


def test_forks_refuse_more_sequences_than_they_hold(calls):
    many = lambda count: dict(table=torch.zeros(count, 1, dtype=I32), lengths=torch.zeros(count, dtype=I32), parents=torch.zeros(count, dtype=I32))  # noqa: E731
    paged.fork_pages(**page_arguments(**many(12800)))
    assert calls.pop()[1][15] == 12800
    with pytest.raises(AssertionError, match="12800"):
        paged.fork_pages(**page_arguments(**many(12801)))
    assert not calls


def test_select_takes_single_beams_in_rows_any_distance_apart(calls):
    wide, scores = torch.zeros(5, 64), on_gpu(torch.zeros(5, 1))
    for logits in (wide[:, :50].unsqueeze(1), wide[:, None, :50], wide.as_strided((5, 1, 50), (64, 7, 1))):
        beam.beam_select(on_gpu(logits), scores)
        assert calls.pop()[1][1] == 64
    beam.beam_select(on_gpu(wide[:1, :50].unsqueeze(0).expand(1, 1, 50)), on_gpu(torch.zeros(1, 1)))
    assert len(calls) == 1


@pytest.mark.parametrize("several", [torch.tensor, lambda b: torch.tensor(b, dtype=I32).unbind(), lambda b: torch.tensor(b).numpy(), lambda b: (b[0], torch.tensor(b[1]))])
def test_sequences_end_by_numbers_of_tensors(monkeypatch, several):
    """A tensor's elements are not found in a set of whole numbers: nothing ended, without a word."""
    cache, state = paged.PagedCache(1, 1, 8, 4, 4, 3, 8, "cpu"), paged.PagedBatchState(synthetic.model_config(num_layers=4, vocab_size=64), 3, 8, "cpu")
    for of in (cache, state):
        seen = []
        monkeypatch.setattr(of, "fork", lambda parents, seen=seen: seen.append(parents.tolist()))
        of.free(several([0, 2]))
        assert seen == [[-1, 1, -1]]
        with pytest.raises(AssertionError):
            of.free(several([0, 3]))
        with pytest.raises(TypeError):
            of.free([0.5])
        assert len(seen) == 1


def test_a_device_has_one_status_however_it_is_named(monkeypatch):
    zeros = torch.zeros
    monkeypatch.setattr(paged, "_status", {})
    monkeypatch.setattr(paged, "_current_device", lambda: 1)
    monkeypatch.setattr(torch, "zeros", lambda *shape, device=None, **kwargs: zeros(*shape, **kwargs))
    monkeypatch.setattr(torch.cuda, "device", lambda device: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device: type("Stream", (), {"synchronize": lambda self: None})())
    word = paged.device_status(torch.device("cuda", 1))
    assert all(paged.device_status(device) is word for device in (torch.device("cuda"), "cuda", "cuda:1", torch.device("cuda:1")))
    assert paged.device_status("cuda:0") is not word and paged.device_status("cpu") is paged.device_status(torch.device("cpu"))


@pytest.mark.parametrize("graph", [False, True])
def test_a_search_that_fails_leaves_no_captured_step(monkeypatch, graph):
    class Decoder:
        class ckpt:
            config = synthetic.model_config(num_layers=4, vocab_size=64)
        device = "cpu"
        held: list = []

        def graph_step(self, tokens, state, **kwargs):
            self.held.append(state)
            if len(self.held) == 3:
                raise KeyboardInterrupt
            return None, torch.zeros(4, 64)
        step = graph_step

        def forget(self, state):
            self.held = [kept for kept in self.held if kept is not state]

    decoder = Decoder()
    monkeypatch.setattr(paged.PagedBatchState, "fork", lambda self, parents: None)
    monkeypatch.setattr(beam, "beam_select", lambda logits, scores, **kwargs: (scores, torch.zeros(2, 2, dtype=I32), torch.zeros(2, 2, dtype=torch.long)))
    with pytest.raises(KeyboardInterrupt):
        beam.beam_search(decoder, [[1], [2]], 2, 9, graph=graph)
    assert decoder.held == []


@pytest.mark.parametrize("mask", [[True, False, True], torch.tensor([True, False, True]), torch.tensor([True, False, True]).numpy()])
def test_sequences_do_not_end_by_a_mask(monkeypatch, mask):
    """True and False are 1 and 0 as numbers: other sequences than meant would end."""
    cache = paged.PagedCache(1, 1, 8, 4, 4, 3, 8, "cpu")
    monkeypatch.setattr(cache, "fork", lambda parents: pytest.fail("ended"))
    with pytest.raises((AssertionError, TypeError)):
        cache.free(mask)
