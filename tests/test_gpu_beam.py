"""Selection of beams against a sort in 64 bits, the order of states, and the whole search against one without pages."""

import math

import pytest
import torch

from quickdraw_b200 import beam, paged, synthetic
from tests import paged_plain as plain

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def same(got, logits, scores, **kwargs):
    """Whole numbers equal; the score is one sum in 64 bits, rounded once, of a log-sum-exp from 32-bit terms (each off by 2^-22, at arguments
    of at most 64 by 64 * 2^-24 more)."""
    want = plain.select(logits, scores, **kwargs)
    assert torch.equal(got[1].cpu(), want[1]) and torch.equal(got[2].cpu(), want[2]), (got, want)
    finite = torch.isfinite(want[0])
    assert torch.equal(torch.isfinite(got[0].cpu()), finite) and bool((got[0].cpu()[~finite] == -math.inf).all())
    error = (got[0].cpu().double() - want[0])[finite].abs()
    assert bool((error <= 2 ** -17 + 2 ** -24 * want[0][finite].abs()).all()), float(error.max())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("batch,beams,vocab", [(1, 1, 1), (1, 1, 40), (2, 4, 5), (3, 5, 1000), (1, 4, 151936), (2, 16, 4097), (1, 32, 33), (7, 3, 20000), (40, 8, 515), (3, 32, 2048), (3, 12, 2049)])
def test_select(cuda_device, batch, beams, vocab, dtype):
    g = torch.Generator().manual_seed(vocab)
    logits = (torch.randn((batch, beams, vocab), generator=g) * 3).to(dtype).cuda()
    scores = (torch.randn((batch, beams), generator=g) - 10).cuda()
    same(beam.beam_select(logits, scores), logits, scores)
    for count in {1, min(2 * beams, 32, beams * vocab), min(32, beams * vocab)}:
        same(beam.beam_select(logits, scores, candidates=count), logits, scores, candidates=count)
    finished = torch.rand((batch, beams), generator=g).cuda() < 0.4
    for eos in {0, vocab // 2, vocab - 1}:
        same(beam.beam_select(logits, scores, finished=finished, eos=eos), logits, scores, finished=finished, eos=eos)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("vocab", [16, 300, 9000, 60001])
def test_ties_go_to_the_lowest(cuda_device, vocab, dtype):
    logits = torch.zeros((2, 4, vocab), dtype=dtype, device="cuda")
    scores = torch.tensor([[0.0, 0.0, 0.0, 0.0], [-1.0, 0.0, 0.0, -1.0]], device="cuda")
    same(beam.beam_select(logits, scores), logits, scores)
    same(beam.beam_select(logits, scores, candidates=11), logits, scores, candidates=11)
    logits[:, :, vocab // 2:] = 1.0
    logits[1, 2, -1] = 2.0
    same(beam.beam_select(logits, scores), logits, scores)
    ascending = torch.arange(vocab, device="cuda").to(dtype).expand(2, 4, vocab).contiguous() / 64
    same(beam.beam_select(ascending, scores), ascending, scores)
    same(beam.beam_select(ascending.flip(2).contiguous(), scores, candidates=9), ascending.flip(2), scores, candidates=9)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("vocab", [100, 5000, 70001])
def test_neighbours_that_32_bits_do_not_tell_apart(cuda_device, vocab, dtype):
    """Beams with the same logits in another order, whose sums differ by rounding alone, and scores one step apart: the step decides."""
    for seed in range(12):
        g = torch.Generator().manual_seed(seed)
        row = (torch.randn(vocab, generator=g) * 3).to(dtype)
        logits = torch.stack([row[torch.randperm(vocab, generator=g)] for _ in range(6)])[None].cuda()
        scores = torch.full((1, 6), -10.0)
        for i in torch.randperm(6, generator=g).tolist()[:3]:
            scores[0, i] = torch.nextafter(scores[0, i], torch.tensor(0.0 if seed % 2 else -20.0))
        got = beam.beam_select(logits, scores.cuda(), candidates=12)
        # beams of equal scores are told apart by the last bits of 64-bit sums alone: only the scores' order, and the tokens of each beam's best, are fixed
        chosen = scores[0][got[1][0].cpu().long()]
        value = row.double()[:, None].new_tensor([float(logits[0, p, t]) for p, t in zip(got[1][0].tolist(), got[2][0].tolist())]) + chosen.double()
        assert bool((value[1:] <= value[:-1]).all()), seed
        best = torch.sort((torch.stack([logits[0, i].cpu().double() + scores[0, i].double() for i in range(6)])).view(-1), descending=True).values[:12]
        assert torch.equal(value, best), seed


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_what_is_no_continuation(cuda_device, dtype):
    g = torch.Generator().manual_seed(2)
    for vocab in (50, 5000):
        logits = torch.randn((7, 3, vocab), generator=g).to(dtype).cuda()
        scores = torch.zeros((7, 3), device="cuda")
        logits[0, 0, 7], logits[0, 1, 9] = math.nan, math.inf           # only the third beam goes on
        logits[1] = -math.inf                                           # nobody does
        logits[2, :, 2:] = -math.inf                                    # two tokens each
        logits[2, 1:, :] = -math.inf
        scores[3, :2], scores[4] = -math.inf, -math.inf
        logits[5, 1] = torch.finfo(dtype).min
        logits[6, 0, ::2] = torch.finfo(dtype).min
        scores[6, 1:] = -math.inf
        same(beam.beam_select(logits, scores), logits, scores)
        same(beam.beam_select(logits, scores, candidates=7), logits, scores, candidates=7)
        finished = torch.zeros((7, 3), dtype=torch.bool, device="cuda")
        finished[3, 2] = finished[1, 1] = finished[4, 0] = finished[0, 0] = finished[6, 0] = True
        same(beam.beam_select(logits, scores, finished=finished, eos=1), logits, scores, finished=finished, eos=1)


def test_rows_of_a_larger_matrix_and_a_graph(cuda_device):
    g = torch.Generator().manual_seed(3)
    whole = torch.randn((6, 2000), generator=g).to(BF16).cuda()
    scores = torch.zeros((2, 3), device="cuda")
    for first, vocab in ((0, 1999), (1, 1000), (8, 1992), (3, 1001)):
        logits = whole[:, first:first + vocab].view(2, 3, vocab) if first + vocab == 2000 else whole[:, first:first + vocab].unflatten(0, (2, 3))
        same(beam.beam_select(logits, scores), logits, scores)
    logits = whole.view(2, 3, 2000)
    want = beam.beam_select(logits, scores)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = beam.beam_select(logits, scores)
    for t in got:
        t.zero_()
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("vocab", [1, 7, 2041, 2047, 2048, 2049, 4100, 6151])
def test_rows_that_begin_anywhere(cuda_device, vocab, dtype):
    """Between the rows lies what would spoil them."""
    g = torch.Generator().manual_seed(vocab)
    for first in range(9):
        whole = torch.full((6, vocab + 17 - first), math.nan, dtype=dtype, device="cuda")
        whole[:, first:first + vocab] = (torch.randn((6, vocab), generator=g) * 3).to(dtype).cuda()
        logits = whole[:, first:first + vocab].unflatten(0, (2, 3))
        scores = torch.randn((2, 3), generator=g).cuda()
        same(beam.beam_select(logits, scores), logits, scores)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("batch,beams,vocab", [(2, 32, 2049), (1, 32, 70001), (3, 31, 6151), (2, 17, 66000)])
def test_many_beams_of_long_rows(cuda_device, batch, beams, vocab, dtype):
    """The most lists that a group's blocks join, from two pieces a row to thirty-two; scores near one another, so that many beams count."""
    g = torch.Generator().manual_seed(vocab)
    logits = (torch.randn((batch, beams, vocab), generator=g) * 3).to(dtype).cuda()
    scores = (torch.randn((batch, beams), generator=g) * 0.5 - 10).cuda()
    finished = torch.rand((batch, beams), generator=g).cuda() < 0.2
    for kwargs in (dict(), dict(candidates=32), dict(finished=finished, eos=vocab - 1), dict(finished=finished, eos=0, candidates=32)):
        same(beam.beam_select(logits, scores, **kwargs), logits, scores, **kwargs)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("vocab", [50, 5000])
def test_single_beams_in_rows_apart(cuda_device, vocab, dtype):
    whole = torch.full((6, vocab + 13), math.nan, dtype=dtype, device="cuda")
    whole[:, :vocab] = (torch.randn((6, vocab), generator=torch.Generator().manual_seed(3)) * 3).to(dtype).cuda()
    logits, scores = whole[:, :vocab].unsqueeze(1), torch.zeros((6, 1), device="cuda")
    same(beam.beam_select(logits, scores), logits, scores)
    same(beam.beam_select(logits, scores, candidates=5), logits, scores, candidates=5)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("candidates", [1, 8, 32])
@pytest.mark.parametrize("order", ["up", "down", "steps", "one in front"])
def test_rows_in_order(cuda_device, order, candidates, dtype):
    """Every chunk above those before it, below them, of equal logits, or below one."""
    vocab = 30011
    row = {"up": torch.linspace(-9, 9, vocab), "down": torch.linspace(9, -9, vocab), "steps": torch.arange(vocab).div(2048, rounding_mode="floor") * 0.5,
           "one in front": torch.cat((torch.tensor([5.0]), torch.zeros(vocab - 1)))}[order]
    logits = torch.stack((row, row.roll(77), row.flip(0))).view(1, 3, vocab).to(dtype).cuda()
    scores = torch.tensor([[0.0, -0.3, -0.7]], device="cuda")
    same(beam.beam_select(logits, scores, candidates=candidates), logits, scores, candidates=candidates)


@pytest.mark.parametrize("count,parents", [(1, [0]), (2, [1, 0]), (5, [4, 4, 4, 4, 4]), (4, [1, 2, 3, 0]), (6, [-1, 0, 0, 3, -1, 4]), (3, [0, 1, 2]), (3, [-1, -1, -1])])
def test_reorder(cuda_device, count, parents):
    shapes = [((3, 8, 16), F32), ((5,), BF16), ((700, 33), BF16), ((7,), torch.uint8), ((1, 1), F32), ((0,), F32)]
    g = torch.Generator().manual_seed(1)
    for chosen in (shapes[:1], shapes[1:2], shapes[2:3], shapes[3:4], shapes):
        states = [torch.randint(0, 100, (count, *shape), generator=g).to(dtype).cuda() for shape, dtype in chosen]
        want = [torch.stack([t[p] if p >= 0 else torch.zeros_like(t[0]) for p in parents]) for t in states]
        beam.reorder_states(states, torch.tensor(parents, dtype=torch.int32, device="cuda"))
        assert all(torch.equal(a, b) for a, b in zip(states, want))


def test_reorder_of_many_rows_apart(cuda_device):
    g = torch.Generator().manual_seed(1)
    for count in (300, 3000):
        wide = torch.randn((count, 3, 40), generator=g).cuda()
        parents = torch.randint(-1, count, (count,), generator=g).int()
        middle, before = wide[:, 1], wide.clone()
        beam.reorder_states(middle, parents.cuda())
        want = before.clone()
        want[:, 1] = torch.where((parents >= 0).cuda()[:, None], before[parents.clamp(min=0).long().cuda(), 1], 0.0)
        assert torch.equal(wide, want)


@pytest.mark.parametrize("count", [1753, 1754, 1755, 1756, 7000])
@pytest.mark.parametrize("dtype,row", [(F32, 4), (F32, 3), (BF16, 3), (torch.uint8, 5)])
def test_reorder_of_as_many_rows_as_shared_memory_takes(cuda_device, count, dtype, row):
    """Around the size from which a launch has to ask for more than it gets without asking, with units of 16, 4, 2 and 1 bytes; and the most."""
    g = torch.Generator().manual_seed(1)
    state = torch.randint(0, 100, (count, row), generator=g).to(dtype)
    parents = torch.randint(-1, count, (count,), generator=g).int()
    want = torch.where((parents >= 0)[:, None], state[parents.clamp(min=0).long()], 0)
    got = state.cuda()
    beam.reorder_states(got, parents.cuda())
    assert torch.equal(got.cpu(), want.to(dtype))


def test_reorder_with_parents_that_are_none(cuda_device):
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    state = torch.arange(12.0, device="cuda").view(3, 4).clone()
    beam.reorder_states(state, torch.tensor([3, -2, 0], dtype=torch.int32, device="cuda"), status=status)
    assert int(status) == paged.BAD_ARGUMENT and state.tolist() == [[0, 1, 2, 3], [4, 5, 6, 7], [0, 1, 2, 3]]


# ----------------------------------------------------------------------------------- the whole search
class Remembering:
    """A decoder whose logits go by the token, by the one before it, which the recurrent state carries, and by the one two before it, which
    lies in the pages: a beam with another's state or pages goes another way."""

    class ckpt:
        config = synthetic.model_config(num_layers=4, vocab_size=40)
    device = "cuda"

    def __init__(self):
        self.table = (torch.randn((40, 40, 40, 40), generator=torch.Generator().manual_seed(9)) * 2).cuda()

    def run(self, tokens, first, one):
        for i, t in enumerate(tokens.tolist()):
            one.kv_k[0, first + i, 0, 0] = t
            one.rec_state[0, 0, 0, 0] = t

    def step(self, tokens, state, *, positions_checked=False):
        cache, at, rows = state.cache, state.positions.long(), torch.arange(state.batch, device="cuda")
        cache.reserve()
        place = lambda p: (cache.table[rows, p // cache.page].long(), 0, p % cache.page, 0, 0)  # noqa: E731
        cache.k[place(at)] = tokens.to(BF16)
        earlier = torch.where(at >= 2, cache.k[place((at - 2).clamp(min=0))].float(), 0.0).long()
        logits = self.table[earlier, state.rec_state[:, 0, 0, 0, 0].long(), tokens]
        state.rec_state[:, 0, 0, 0, 0] = tokens.float()
        state.positions += 1
        return logits.argmax(-1), logits

    def forget(self, state):
        pass


def remembered_search(table, prompt, beams, steps, eos):
    """The same search over lists of tokens."""
    table = table.cpu().double()
    kept = [(0.0, [], False)] + [(-math.inf, [], False)] * (beams - 1)
    for _ in range(steps):
        found = []
        for i, (score, answer, done) in enumerate(kept):
            seen = [0, 0] + prompt + answer
            each = torch.log_softmax(table[seen[-3], seen[-2], seen[-1]], 0).tolist()
            found += [(score + (each[t] if not done else 0.0 if t == eos else -math.inf), -i, -t) for t in range(len(each))]
        best = sorted(found, reverse=True)[:beams]
        places, left = [None] * beams, [i for i in range(beams) if i not in {-b[1] for b in best}]
        for score, i, t in best:
            entry = (score, kept[-i][1] + [-t], kept[-i][2] or -t == eos)
            places[-i if places[-i] is None and -i not in left else left.pop(0)] = entry
        kept = places
    cut = [(a[:a.index(eos) + 1] if eos in a else a, score) for score, a, _ in kept if score > -math.inf]
    return sorted(cut, key=lambda a: -a[1])


@pytest.mark.parametrize("beams,page,steps", [(1, 4, 9), (4, 4, 30), (5, 16, 21), (16, 3, 12), (32, 1, 5)])
def test_search_carries_states_and_pages(cuda_device, beams, page, steps):
    decoder = Remembering()
    prompts = [[3, 7, 20, 11, 5], [9], [1, 2], [(11 * i) % 40 for i in range(35)]]
    found = beam.beam_search(decoder, prompts, beams, steps, eos=7, page=page)
    for prompt, answers in zip(prompts, found):
        want = remembered_search(decoder.table, prompt, beams, steps, 7)
        assert [a for a, _ in answers] == [a for a, _ in want]
        assert all(abs(a[1] - b[1]) < 1e-3 for a, b in zip(answers, want))
    no_end = beam.beam_search(decoder, prompts[:1], beams, 3, page=page, length_penalty=1.0)[0]
    assert all(len(a) == 3 for a, _ in no_end)


@pytest.mark.parametrize("graph", [False, True])
def test_search_over_the_model(cuda_device, graph):
    """Every answer's score is the sum of its tokens' log-probabilities in a run of that answer alone over contiguous caches.  (Which answers
    survive is decided by near ties of bf16 logits, and these by the order of the attention's sums.)"""
    from quickdraw_b200.batch import BatchDecode, BatchState
    cfg = synthetic.model_config(num_layers=4, vocab_size=512, experts=16, topk=8)
    ckpt = synthetic.make_checkpoint(cfg, seed=5, device="cuda")
    decoder = BatchDecode(ckpt)
    prompts, beams, steps = [[3, 77, 200, 11, 5], [9], list(range(40, 75))], 4, 12
    found = beam.beam_search(decoder, prompts, beams, steps, eos=7, page=8, graph=graph)
    assert len(found) == 3
    for prompt, answers in zip(prompts, found):
        assert len(answers) == beams and all(a[1] >= b[1] for a, b in zip(answers, answers[1:]))
        assert len({tuple(a) for a, _ in answers}) == beams
        for answer, score in answers:
            state = BatchState(cfg, 1, 64, "cuda")
            if len(prompt) > 1:
                decoder.run(torch.tensor(prompt[:-1], device="cuda"), 0, state.sequence(0))
            state.positions[0] = len(prompt) - 1
            token, total = torch.tensor([prompt[-1]], device="cuda"), 0.0
            for t in answer:
                _, logits = decoder.step(token, state)
                total += float(torch.log_softmax(logits[0].double(), 0)[t])
                token = torch.tensor([t], device="cuda")
            # logits of bf16 below 4 in magnitude: half a step is 2^-7, of the token's and of the log-sum-exp, and as much again for what rounds before them
            assert abs(total - score) <= len(answer) * 4 * 2 ** -7, (answer, score, total)
    assert beam.beam_search(decoder, prompts[:1], 2, 0) == [[([], 0.0)]]
