"""Paged caches on the GPU: attention of one token against 64 bits, and pages forked, set aside, compacted against a plain account."""

import itertools
import math

import pytest
import torch

from oracle import decode_oracle as O
from quickdraw_b200 import beam, paged, synthetic
from tests import paged_plain as plain

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def problem(lengths, heads, kv_heads, dim, page, dtype, seed=0, gate=False, std=2.0, **kwargs):
    g = torch.Generator().manual_seed(seed + 1000)
    k, v, table, n, _ = plain.cache(lengths, page, 1, kv_heads, dim, dtype, seed, **kwargs)
    q = (torch.randn((len(lengths), heads, dim), generator=g) * std).to(dtype).cuda()
    gates = torch.randn((len(lengths), heads, dim), generator=g).to(dtype).cuda() if gate else None
    return q, k[:, 0], v[:, 0], table, n, gates


def check(got, q, k, v, table, n, gate=None, **kwargs):
    want, bound = plain.attention(q, k, v, table, n, gate=gate, **kwargs)
    error = (got.cpu().double() - want).abs()
    assert bool(torch.isfinite(got).all())
    assert bool((error <= bound).all()), (float((error - bound).max()), float(error.max()))


LENGTHS = [[1], [0], [17], [16], [100, 0, 1, 33], [255, 256, 257, 7], [1030, 64, 63, 65, 513], [3001]]
SHAPES = [(16, 2, 256), (32, 8, 128), (16, 4, 64), (8, 8, 128), (12, 4, 96), (7, 1, 80), (5, 5, 40), (24, 2, 128), (17, 1, 64), (64, 1, 192), (40, 1, 256), (2, 1, 8)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads,kv_heads,dim", SHAPES)
def test_attention_of_every_shape(cuda_device, heads, kv_heads, dim, dtype):
    for number, (lengths, page) in enumerate(itertools.product(LENGTHS[4:7], [1, 16, 24, 100])):
        args = problem(lengths, heads, kv_heads, dim, page, dtype, seed=number, gate=number % 2 == 1)
        *args, gate = args
        check(paged.paged_attention(*args, gate=gate), *args, gate=gate)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("lengths", LENGTHS)
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (5, 1), (64, 4), (300, 17), (4000, 3)])
def test_lengths_windows_and_first_rows(cuda_device, lengths, window, sinks, dtype):
    for heads, kv_heads, dim, page in ((16, 2, 256, 16), (4, 2, 64, 7)):
        *args, _ = problem(lengths, heads, kv_heads, dim, page, dtype, seed=len(lengths))
        check(paged.paged_attention(*args, window=window, sinks=sinks), *args, window=window, sinks=sinks)


def test_a_scale_of_ones_own(cuda_device):
    *args, _ = problem([50, 90], 16, 2, 256, 16, BF16, std=0.1)
    check(paged.paged_attention(*args, scale=0.5), *args, scale=0.5)
    check(paged.paged_attention(*args, scale=-0.25), *args, scale=-0.25)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_entries_that_are_no_page_are_not_seen(cuda_device, dtype):
    q, k, v, table, n, _ = problem([200, 64, 48, 30], 16, 2, 256, 16, dtype, width=15)
    table[0, 3], table[0, 7], table[1, :] = -1, k.shape[0], -7
    table[3, 0] = 2 ** 31 - 1
    n[2] = 100000                                       # more than the table holds: what it holds
    check(paged.paged_attention(q, k, v, table, n), q, k, v, table, n)
    n[0] = -5
    check(paged.paged_attention(q, k, v, table, n), q, k, v, table, n)
    # pages that a window does not reach need not exist
    q, k, v, table, n, _ = problem([500], 16, 2, 256, 16, dtype)
    want = paged.paged_attention(q, k, v, table, n, window=100, sinks=4)
    table[0, 1:500 // 16 - 7] = -1
    assert torch.equal(paged.paged_attention(q, k, v, table, n, window=100, sinks=4), want)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_scores_far_apart_and_infinite(cuda_device, dtype):
    q, k, v, table, n, _ = problem([300, 300, 40], 4, 2, 64, 16, dtype, std=60.0)
    check(paged.paged_attention(q, k, v, table, n), q, k, v, table, n)
    # scores of -inf weigh nothing; nothing but -inf gives zeros; +inf and NaN give NaN, in their rows alone
    q.fill_(1.0)
    k[table[0, :19].long()] = torch.where(torch.isnan(k[table[0, :19].long()]), math.nan, 0.0).to(dtype)
    k[table[0, 2].long(), 3] = -math.inf
    k[table[1, :19].long()] = torch.where(torch.isnan(k[table[1, :19].long()]), math.nan, -math.inf).to(dtype)
    k[table[2, 0].long(), 1, 0] = math.inf
    out = paged.paged_attention(q, k, v, table, n)
    assert bool(torch.isfinite(out[0]).all()) and bool((out[1] == 0).all())
    assert bool(torch.isnan(out[2, :2]).all()) and bool(torch.isfinite(out[2, 2:]).all())
    k[table[2, 0].long(), 1, 0] = math.nan
    out = paged.paged_attention(q, k, v, table, n)
    assert bool(torch.isnan(out[2, :2]).all()) and bool(torch.isfinite(out[2, 2:]).all())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads,kv_heads,dim", SHAPES)
def test_infinite_and_largest_values(cuda_device, heads, kv_heads, dim, dtype):
    """An infinity among the values is the mean of its column, those of both signs and NaN give NaN there, and means of the largest numbers stay below
    them; the other columns do not notice.  One launch and two, one row and many, pages that are missing between them."""
    largest = 3.3e38
    for lengths, page, width in (([1, 2, 40, 0], 16, 4), ([700, 1, 333, 64], 16, None)):
        q, k, v, table, n, _ = problem(lengths, heads, kv_heads, dim, page, dtype, seed=dim, width=width)
        inside, last = table.cpu(), [n - 1 for n in lengths]
        at = lambda b, p: (int(inside[b, p // page]), p % page)  # noqa: E731
        clean = v.clone()
        for t in (v, clean):
            for b in (0, 2):
                for p in range(lengths[b]):
                    t[at(b, p)][:, 1] = largest if p % 7 else largest / 2           # a column of them
                    t[at(b, p)][:, 4] = largest if p % 2 else -largest
        for b in (0, 2):
            v[at(b, last[b])][:, 2], clean[at(b, last[b])][:, 2] = math.inf, 0.0
            v[at(b, 0)][:, 3], clean[at(b, 0)][:, 3] = -math.inf, 0.0
            v[at(b, last[b])][:, 5], clean[at(b, last[b])][:, 5] = math.nan, 0.0
            v[at(b, last[b] // 2)][0, 6], clean[at(b, last[b] // 2)][0, 6] = math.inf, 0.0
            v[at(b, last[b])][:, 7], clean[at(b, last[b])][:, 7] = math.inf, 0.0
            if last[b]:
                v[at(b, 0)][:, 7], clean[at(b, 0)][:, 7] = -math.inf, 0.0
        for seen in (dict(), dict(window=30, sinks=2)):
            got = paged.paged_attention(q, k, v, table, n, **seen)
            want, bound = plain.attention(q, k, clean, table, n, **seen)
            for b in (0, 2):
                want[b, :, 2], want[b, :, 3], want[b, :, 5] = math.inf, -math.inf, math.nan
                if not seen or last[b] // 2 < 2 or last[b] - last[b] // 2 < 30:
                    want[b, :heads // kv_heads, 6] = math.inf
                want[b, :, 7] = math.nan if last[b] else math.inf
            got, fine = got.cpu().double(), torch.isfinite(want)
            assert torch.equal(torch.nan_to_num(got[~fine], nan=5.0), torch.nan_to_num(want[~fine], nan=5.0)), (lengths, seen)
            assert bool(torch.isfinite(got[fine]).all()) and bool(((got - want).abs() <= bound)[fine].all()), (lengths, seen)
            # the bound of a column of such values says nothing of the others
            small = clean.clone()
            small[..., 1], small[..., 4] = 0.0, 0.0
            want, bound = plain.attention(q, k, small, table, n, **seen)
            columns = [0, *range(8, dim)]
            assert bool(((got - want).abs() <= bound)[:, :, columns].all()), (lengths, seen)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads,kv_heads,dim", [(16, 2, 256), (4, 2, 64), (24, 2, 128)])
def test_attention_over_pages_that_sequences_share(cuda_device, heads, kv_heads, dim, dtype):
    """Beams behind a common beginning, as forks leave them: 700 rows of the first sequence in all tables, then rows of their own."""
    *args, gate = problem([777, 777, 703, 720, 300, 777], heads, kv_heads, dim, 20, dtype, seed=4, gate=True, shared=35)
    assert int((args[3] == args[3][:1]).sum(0)[:15].min()) == 6                  # one page in six tables
    check(paged.paged_attention(*args, gate=gate), *args, gate=gate)
    check(paged.paged_attention(*args, gate=gate, window=100, sinks=30), *args, gate=gate, window=100, sinks=30)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_largest_values_under_scores_that_rise(cuda_device, dtype):
    """A softmax's reference may lie 2^8 below its scores: weights of 256, and many of them, times the largest numbers."""
    largest = 3.3e38
    for heads, kv_heads, dim in ((16, 2, 256), (32, 1, 128), (4, 2, 64)):
        q, k, v, table, n, _ = problem([5000, 200, 60], heads, kv_heads, dim, 16, dtype)
        q.fill_(1.0)
        for b, count in enumerate((5000, 200, 60)):
            p = torch.arange(count, device="cuda")
            k[table[b, p // 16].long(), p % 16] = (torch.clamp(p / 40, max=5.25) / dim).to(dtype)[:, None, None]
            v[table[b, p // 16].long(), p % 16] = largest
            v[table[b, p // 16].long(), p % 16, :, dim // 2:] = -largest
        check(paged.paged_attention(q, k, v, table, n, scale=1.0), q, k, v, table, n, scale=1.0)


def test_views_with_other_strides(cuda_device):
    """Layers of one pool, pools with the heads outside of the rows, queries and gates inside a projection, a table inside a larger one."""
    lengths, page = [120, 77, 300], 16
    *args, _ = problem(lengths, 16, 2, 256, page, BF16)
    q, k, v, table, n = args
    gate = torch.randn_like(q)
    want = paged.paged_attention(*args, gate=gate)
    both = torch.cat([q, gate], dim=2)
    wide = torch.cat([table, table], dim=1)[:, :table.shape[1]]
    assert torch.equal(paged.paged_attention(both[:, :, :256], k, v, wide, n, gate=both[:, :, 256:]), want)
    layers = [torch.stack([torch.full_like(t, math.nan), t, torch.zeros_like(t)], dim=1)[:, 1] for t in (k, v)]
    assert torch.equal(paged.paged_attention(q, *layers, table, n, gate=gate), want)
    outside = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v)]
    assert torch.equal(paged.paged_attention(q, *outside, table, n, gate=gate), want)
    heads_first = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(paged.paged_attention(heads_first, k, v, table, n, gate=gate), want)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads,kv_heads,dim", [(16, 2, 256), (24, 2, 128), (4, 2, 64), (7, 1, 80)])
def test_queries_and_gates_anywhere(cuda_device, heads, kv_heads, dim, dtype):
    """Rows that start off every boundary but their elements' own."""
    q, k, v, table, n, _ = problem([90, 0, 333], heads, kv_heads, dim, 16, dtype)
    gate = torch.randn((3, heads, dim), generator=torch.Generator().manual_seed(7)).to(dtype).cuda()
    want = paged.paged_attention(q, k, v, table, n, gate=gate)
    for shift in (1, 3):
        off = [torch.zeros((3, heads, dim + 5), dtype=dtype, device="cuda")[:, :, shift:shift + dim] for _ in range(2)]
        off[0].copy_(q), off[1].copy_(gate)
        assert torch.equal(paged.paged_attention(off[0], k, v, table, n, gate=off[1]), want)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("width", [1, 16, 17, 64, 900])
def test_short_sequences_of_short_and_long_tables(cuda_device, width, dtype):
    """One launch or two, by what the table could hold."""
    for heads, kv_heads, dim in ((16, 2, 256), (32, 1, 128), (4, 4, 64)):
        *args, gate = problem([0, 1, 16, 9, 0], heads, kv_heads, dim, 16, dtype, width=width, gate=True)
        check(paged.paged_attention(*args, gate=gate), *args, gate=gate)


def test_a_sequence_does_not_depend_on_its_neighbours(cuda_device):
    q, k, v, table, n, _ = problem([700, 3, 1500, 64], 16, 2, 256, 64, BF16)
    first = paged.paged_attention(q, k, v, table, n)
    assert torch.equal(paged.paged_attention(q, k, v, table, n), first)
    n[1], n[3] = 0, 1
    assert torch.equal(paged.paged_attention(q, k, v, table, n)[[0, 2]], first[[0, 2]])


@pytest.mark.parametrize("count,heads,kv_heads,dim,dtype,width", [(1500, 2, 1, 64, BF16, None), (1100, 2, 1, 64, BF16, 40), (300, 2, 1, 64, F32, 40),
                                                                 (200, 16, 1, 256, BF16, 40), (300, 3, 1, 40, F32, None)])
def test_more_sequences_than_a_launch_takes(cuda_device, count, heads, kv_heads, dim, dtype, width):
    lengths = [(37 * b) % 50 for b in range(count)]
    *args, _ = problem(lengths, heads, kv_heads, dim, 16, dtype, width=width)
    check(paged.paged_attention(*args), *args)


def test_offsets_past_32_bits(cuda_device):
    """A pool of 5 GB whose pages in use lie at its end."""
    small_k, small_v = (torch.randn((4, 64, 2, 256), generator=torch.Generator().manual_seed(s)).to(BF16).cuda() for s in (1, 2))
    pages = 80000
    k, v = (torch.zeros((pages, 64, 2, 256), dtype=BF16, device="cuda") for _ in range(2))
    k[-4:], v[-4:] = small_k, small_v
    table = torch.tensor([[3, 0, 2, 1]], dtype=torch.int32, device="cuda")
    n = torch.tensor([250], dtype=torch.int32, device="cuda")
    q = torch.randn((1, 16, 256), generator=torch.Generator().manual_seed(3)).to(BF16).cuda()
    assert torch.equal(paged.paged_attention(q, k, v, table + pages - 4, n), paged.paged_attention(q, small_k, small_v, table, n))


def test_another_stream_and_two_graphs(cuda_device):
    """Two captured calls replayed at the same time, and eager calls between them, do not share scratch."""
    problems = [problem([2000, 900 + 40 * s, 5], 16, 2, 256, 64, BF16, seed=s)[:5] for s in range(2)]
    want = [paged.paged_attention(*args) for args in problems]
    torch.cuda.synchronize()
    streams, graphs, outs = [torch.cuda.Stream() for _ in problems], [], []
    for stream, args in zip(streams, problems):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            outs.append(paged.paged_attention(*args))
        graphs.append(graph)
    for _ in range(20):
        for stream, graph in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
        eager = paged.paged_attention(*problems[0])
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1]) and torch.equal(eager, want[0])


# ----------------------------------------------------------------------------------- pages
FORKS = {
    "swap": ([37, 52], [1, 0], 0),
    "all from one": ([37, 5, 0, 16], [0, 0, 0, 0], 0),
    "all from another": ([37, 5, 0, 16], [1, 1, 1, 1], 0),
    "from an empty one": ([37, 5, 0, 16], [2, 1, 2, 2], 0),
    "full pages only": ([32, 48, 16, 64], [1, 1, 3, 3], 1),
    "some end": ([33, 33, 33, 33, 40], [-1, 0, 0, -1, 2], 2),
    "all end": ([33, 33], [-1, -1], 1),
    "nothing moves": ([33, 7, 1], [0, 1, 2], 1),
    "a cycle": ([50, 60, 70], [1, 2, 0], 3),
}


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("name", FORKS)
def test_fork(cuda_device, name, dtype):
    lengths, parents, shared = FORKS[name]
    for page, layers, heads, dim in ((16, 2, 2, 64), (1, 1, 1, 8), (7, 3, 2, 256)):
        k, v, table, n, refs = plain.cache(lengths, page, layers, heads, dim, dtype, seed=3, spare=10, shared=shared)
        want = plain.fork(k, v, table, n, refs, parents, page)
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        before = [t.clone() for t in (table, n, refs)]
        got = paged.fork_pages(k, v, table, n, refs, torch.tensor(parents, dtype=torch.int32, device="cuda"), status=status)
        for a, b in zip((k, v, *got, status), (*want[:5], torch.tensor([want[5]]))):
            assert torch.equal(torch.nan_to_num(a.cpu().float(), nan=7e7), torch.nan_to_num(b.float(), nan=7e7)), (name, page)
        assert all(torch.equal(a, b) for a, b in zip((table, n, refs), before))


def test_fork_of_many(cuda_device):
    """More sequences than a block has threads, more pages than a warp looks at, parents at random."""
    g = torch.Generator().manual_seed(5)
    lengths = torch.randint(0, 90, (1300,), generator=g).tolist()
    parents = torch.randint(-1, 1300, (1300,), generator=g).tolist()
    k, v, table, n, refs = plain.cache(lengths, 16, 1, 1, 8, BF16, seed=6, spare=2000)
    want = plain.fork(k, v, table, n, refs, parents, 16)
    got = paged.fork_pages(k, v, table, n, refs, torch.tensor(parents, dtype=torch.int32, device="cuda"))
    for a, b in zip((k, v, *got), want):
        assert torch.equal(torch.nan_to_num(a.cpu().float(), nan=7e7), torch.nan_to_num(b.float(), nan=7e7))


def test_fork_compaction_and_reservation_of_large_tables(cuda_device):
    """More entries and pages than one block goes through."""
    g = torch.Generator().manual_seed(8)
    lengths = torch.randint(0, 1600, (60,), generator=g).tolist()
    parents = torch.randint(-1, 60, (60,), generator=g).tolist()
    k, v, table, n, refs = plain.cache(lengths, 8, 1, 1, 8, BF16, seed=6, spare=30000, width=210)
    want = plain.fork(k, v, table, n, refs, parents, 8)
    got = paged.fork_pages(k, v, table, n, refs, torch.tensor(parents, dtype=torch.int32, device="cuda"))
    for a, b in zip((k, v, *got), want):
        assert torch.equal(torch.nan_to_num(a.cpu().float(), nan=7e7), torch.nan_to_num(b.float(), nan=7e7))
    table, n, refs = got
    held = int((table >= 0).sum())
    free = (refs.cpu() <= 0).nonzero()[:, 0].tolist()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    before = table.clone()
    paged.reserve_pages(table, n, refs, 8, 33, status=status)
    fresh = table[before < 0]
    assert int(status) == 0 and fresh[fresh >= 0].tolist() == free[:int((table >= 0).sum()) - held]
    want = plain.compact(k, v, table, refs)
    got = paged.compact_pages(k, v, table, refs)
    for a, b in zip((k, v, *got[:2]), want):
        assert torch.equal(torch.nan_to_num(a.cpu().float(), nan=7e7), torch.nan_to_num(b.float(), nan=7e7))
    assert int(got[2]) == want[4]


@pytest.mark.parametrize("width", [1, 4])
@pytest.mark.parametrize("count", [3064, 3065, 3069, 12800])
def test_fork_of_as_many_as_shared_memory_takes(cuda_device, count, width):
    """Around the size from which a launch has to ask for more than it gets without asking, by one block and by a cluster; and the most."""
    g = torch.Generator().manual_seed(count)
    lengths = torch.randint(0, 4 * width + 1, (count,), generator=g).tolist()
    parents = torch.randint(-1, count, (count,), generator=g).tolist()
    k, v, table, n, refs = plain.cache(lengths, 4, 1, 1, 8, BF16, seed=6, spare=count, width=width)
    want = plain.fork(k, v, table, n, refs, parents, 4)
    got = paged.fork_pages(k, v, table, n, refs, torch.tensor(parents, dtype=torch.int32, device="cuda"))
    for a, b in zip((k, v, *got), want):
        assert torch.equal(torch.nan_to_num(a.cpu().float(), nan=7e7), torch.nan_to_num(b.float(), nan=7e7))


def test_fork_without_room_and_with_parents_that_are_none(cuda_device):
    lengths, page = [37, 20, 40], 16
    for parents, spare, bits in (([0, 0, 0], 0, 0), ([1, 1, 2], 0, 0), ([0, 0, 5], 1, 4), ([-2, 1, 1], 0, 12), ([2, 2, 2], 0, 0)):
        k, v, table, n, refs = plain.cache(lengths, page, 1, 1, 64, BF16, seed=3, spare=spare, shared=2)
        want = plain.fork(k, v, table, n, refs, parents, page)
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        got = paged.fork_pages(k, v, table, n, refs, torch.tensor(parents, dtype=torch.int32, device="cuda"), status=status)
        assert int(status) == want[5]
        for a, b in zip((k, v, *got), want):
            assert torch.equal(torch.nan_to_num(a.cpu().float(), nan=7e7), torch.nan_to_num(b.float(), nan=7e7)), parents


@pytest.mark.parametrize("hole", [-1, -9, 2 ** 31 - 1])
@pytest.mark.parametrize("parents", [[0, 0, 0, 3], [1, 0, 0, 0], [3, 3, 0, -1], [0, 1, 2, 3]])
def test_fork_of_a_sequence_without_its_last_page(cuda_device, parents, hole):
    """Rows that the parent does not see, its copies do not see either: no page with what its last owner left there (NaN here)."""
    page, lengths = 16, [37, 20, 16, 50]
    k, v, table, n, refs = plain.cache(lengths, page, 1, 1, 64, BF16, seed=3, spare=10)
    refs[table[0, 2].long()] -= 1
    table[0, 2] = hole
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    before = [t.clone() for t in (k, v, table, n)]
    new = paged.fork_pages(k, v, table, n, refs, torch.tensor(parents, dtype=torch.int32, device="cuda"), status=status)
    assert int(status) == 0 and new[1].tolist() == [lengths[p] if p >= 0 else 0 for p in parents]
    held = new[0][(new[0] >= 0) & (new[0] < refs.numel())].long()
    assert torch.equal(torch.bincount(held, minlength=refs.numel()).int(), new[2])
    for b, p in enumerate(parents):
        if p == 0:
            assert torch.equal(new[0][b, :2], table[0, :2]) and not 0 <= int(new[0][b, 2]) < refs.numel()
    q = torch.randn((1, 2, 64), generator=torch.Generator().manual_seed(3)).to(BF16).cuda().expand(4, 2, 64)
    was = paged.paged_attention(q, before[0][:, 0], before[1][:, 0], *before[2:])
    now = paged.paged_attention(q, k[:, 0], v[:, 0], *new[:2])
    for b, p in enumerate(parents):
        assert torch.equal(now[b], was[p] if p >= 0 else torch.zeros_like(now[b])), (b, p)


@pytest.mark.parametrize("lengths,spare", [([5, 700, 0, 64], 60), ([16], 0), ([1], 5000), ([0, 0], 7), ([100] * 40, 130)])
def test_compact(cuda_device, lengths, spare):
    for page, layers, heads, dim, dtype in ((16, 2, 2, 64, BF16), (1, 1, 1, 8, F32), (24, 1, 5, 40, BF16)):
        k, v, table, _, refs = plain.cache(lengths, page, layers, heads, dim, dtype, seed=4, spare=spare, shared=1)
        want = plain.compact(k, v, table, refs)
        got = paged.compact_pages(k, v, table, refs)
        for a, b in zip((k, v, *got[:2]), want):
            assert torch.equal(torch.nan_to_num(a.cpu().float(), nan=7e7), torch.nan_to_num(b.float(), nan=7e7))
        assert int(got[2]) == want[4]


def test_reserve(cuda_device):
    k, v, table, n, refs = plain.cache([33, 16, 0, 48], 16, 1, 1, 8, BF16, seed=1, spare=6, width=6)
    first = (refs.cpu() == 0).nonzero()[:, 0].tolist()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    before = table.clone()
    paged.reserve_pages(table, n, refs, 16, status=status)
    assert table[:, :].tolist()[1][1] == first[0] and int(table[2, 0]) == first[1] and int(table[3, 3]) == first[2] and torch.equal(table[0], before[0])
    again = table.clone()
    paged.reserve_pages(table, n, refs, 16, status=status)              # set aside already
    assert torch.equal(table, again) and int(status) == 0 and int(refs.sum()) == int((table >= 0).sum())
    counts = torch.tensor([0, 33, 0, 100], dtype=torch.int32, device="cuda")
    paged.reserve_pages(table, n, refs, 16, counts, status=status)     # two more for the second; the fourth has no such rows
    assert int(status) == 4 and (table >= 0).sum(1).tolist() == [3, 4, 1, 4]
    paged.reserve_pages(table, n, refs, 16, 40, status=status)         # one page is left, for the first
    assert int(status) == 12 and (table >= 0).sum(1).tolist() == [4, 4, 1, 4] and bool((refs == 1).all())


def test_reserve_of_pages_as_long_as_numbers_go(cuda_device):
    table, refs = torch.full((2, 1), -1, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    lengths, status = torch.tensor([0, 2 ** 31 - 4], dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    paged.reserve_pages(table, lengths, refs, 2 ** 31 - 1, 3, status=status)            # the second's page began long ago
    assert table.tolist() == [[0], [-1]] and refs.tolist() == [1, 0, 0] and int(status) == 0
    paged.reserve_pages(table, lengths, refs, 2 ** 31 - 1, 4, status=status)
    assert table.tolist() == [[0], [-1]] and int(status) == paged.BAD_ARGUMENT


@pytest.mark.parametrize("sequences", [2, 1100, 9000])
def test_every_row_without_a_page_is_said(cuda_device, sequences):
    """A pool that was empty at a page's first row: each of the page's other rows is lost too, and each time the status says so."""
    page = 4
    cache = paged.PagedCache(1, 1, 8, sequences - 1, page, sequences, 16, "cuda")
    words = []
    for step in range(3 * page):
        if step == page + 1:
            cache.free([0])                                            # its place takes the page again; the last one is in the middle of one
        cache.reserve()
        words.append(cache.check())
        cache.lengths += 1
    assert words[:page] == [paged.NO_PAGE] * page and cache.table[-1, 0] == -1
    assert words[page] == paged.NO_PAGE and words[page + 1:2 * page] == [paged.NO_PAGE] * (page - 1)
    last = cache.lengths[-1:].clone()
    # nothing is said of a sequence that asks for no row, of a full page, and by the tables' own form without `begun`
    only = torch.zeros(sequences, dtype=torch.int32, device="cuda")
    cache.lengths.fill_(page), cache.table.fill_(-1), cache.refs.zero_()
    cache.reserve(only)
    assert cache.check() == 0
    only[0] = 1
    cache.reserve(only)
    assert cache.check() == 0 and cache.table[0].tolist() == [-1, 0, -1, -1] and int(last) == 3 * page
    cache.lengths.fill_(page + 1)
    paged.reserve_pages(cache.table, cache.lengths, cache.refs, page, only, status=cache.status)
    assert cache.check() == 0
    cache.reserve(only)
    assert cache.check() == 0
    only[1] = 1
    cache.reserve(only)
    assert cache.check() == paged.NO_PAGE and cache.table[1].tolist() == [-1] * 4


def test_forks_and_reservations_from_a_graph(cuda_device):
    def life(cache, state, parents, fork):
        fork()
        for _ in range(5):
            parents.copy_(torch.roll(parents, 1))
            fork()
        return [cache.table.clone(), cache.lengths.clone(), cache.refs.clone(), state.clone(), cache.k.clone()]

    results = []
    for captured in (False, True):
        cache = paged.PagedCache(2, 1, 64, 40, 8, 4, 64, "cuda")
        cache.lengths.copy_(torch.tensor([13, 8, 0, 21], dtype=torch.int32))
        counts = cache.lengths.clone()
        cache.lengths.zero_()
        cache.reserve(counts)
        cache.lengths.copy_(counts)
        cache.k.copy_(torch.arange(cache.k.numel(), device="cuda").view_as(cache.k) % 251)
        state = torch.arange(4 * 48.0, device="cuda").view(4, 48).clone()
        parents = torch.tensor([0, 0, 3, 1], dtype=torch.int32, device="cuda")

        def step():
            cache.reserve(3)
            cache.lengths += 1
            cache.fork(parents)
            beam.reorder_states(state, parents, status=cache.status)

        fork = step
        if captured:
            graph, other = torch.cuda.CUDAGraph(), torch.cuda.Stream()
            with torch.cuda.graph(graph, stream=other):
                step()
            fork = graph.replay
        results.append(life(cache, state, parents, fork))
        assert cache.check() == 0
    assert all(torch.equal(a, b) for a, b in zip(*results))


def test_the_status_of_a_device_by_any_name(cuda_device):
    table, lengths, refs = (torch.full(shape, fill, dtype=torch.int32, device="cuda") for shape, fill in (((1, 1), -1), ((1,), 0), ((1,), 1)))
    word = paged.device_status(torch.device("cuda"))
    word.zero_()
    paged.reserve_pages(table, lengths, refs, 16)
    assert int(paged.device_status("cuda")) == int(paged.device_status("cuda:0")) == int(word) == paged.NO_PAGE
    word.zero_()


def test_cache_through_its_life(cuda_device):
    """Rows written, sequences forked, ended, the pool compacted and resized: what every sequence sees stays the same."""
    page, layers, heads, dim = 16, 2, 2, 64
    cache = paged.PagedCache(layers, heads, dim, 40, page, 5, 200, "cuda")
    rows = {}
    for b, n in ((0, 50), (3, 33)):
        counts = torch.zeros(5, dtype=torch.int32, device="cuda")
        counts[b] = n
        cache.reserve(counts)
        k, v = (torch.randn((layers, n + 3, heads, dim), generator=torch.Generator().manual_seed(10 * b + s)).to(BF16).cuda() for s in (0, 1))
        cache.write(b, k, v, 0, n)
        cache.lengths[b] = n
        rows[b] = (k[:, :n], v[:, :n])

    def same(b, of, n):
        k, v = (torch.zeros((layers, n, heads, dim), dtype=BF16, device="cuda") for _ in range(2))
        cache.read(b, k, v, 0, n)
        assert torch.equal(k, rows[of][0][:, :n]) and torch.equal(v, rows[of][1][:, :n])

    cache.fork(torch.tensor([0, 0, 3, 3, 0], dtype=torch.int32, device="cuda"))
    for b, of in ((0, 0), (1, 0), (2, 3), (3, 3), (4, 0)):
        same(b, of, 50 if of == 0 else 33)
    assert cache.refs.sum() == (cache.table >= 0).sum() and int((cache.refs > 0).sum()) == 3 + 3 + 2 + 2
    cache.free([0, 3])
    same(1, 0, 50), same(4, 0, 50), same(2, 3, 33)
    cache.resize(3 + 2 + 3)
    same(1, 0, 50), same(4, 0, 50), same(2, 3, 33)
    assert cache.pages == 8 and bool((cache.refs > 0).all())
    with pytest.raises(AssertionError, match="in use"):
        cache.resize(7)
    cache.reserve(17)                                                   # nothing is left
    assert cache.check() == paged.NO_PAGE and cache.check() == 0
    cache.resize(30)
    cache.reserve(17)
    assert cache.check() == 0
    same(1, 0, 50), same(2, 3, 33)
    with pytest.raises(AssertionError):
        cache.free([5])


def test_a_copy_goes_on_by_itself(cuda_device):
    """The page that is not full is not shared: rows that a copy appends are its own."""
    cache = paged.PagedCache(1, 1, 64, 10, 16, 2, 100, "cuda")
    k, v = (torch.randn((1, 30, 1, 64), generator=torch.Generator().manual_seed(s)).to(BF16).cuda() for s in (0, 1))
    cache.reserve(torch.tensor([20, 0], dtype=torch.int32, device="cuda"))
    cache.write(0, k, v, 0, 20)
    cache.lengths[0] = 20
    cache.fork(torch.tensor([0, 0], dtype=torch.int32, device="cuda"))
    cache.reserve()
    cache.write(1, k[:, 25:], v[:, 25:], 20, 1)
    cache.write(0, k[:, 20:], v[:, 20:], 20, 1)
    got = [torch.zeros_like(k), torch.zeros_like(v)]
    cache.read(1, *got, 0, 21)
    assert torch.equal(got[0][:, :20], k[:, :20]) and torch.equal(got[0][:, 20], k[:, 25]) and torch.equal(got[1][:, 20], v[:, 25])
    cache.read(0, *got, 0, 21)
    assert torch.equal(got[0][:, :21], k[:, :21])


# ----------------------------------------------------------------------------------- the batched step
def small_model(vocab=512):
    cfg = synthetic.model_config(num_layers=4, vocab_size=vocab, experts=16, topk=8)
    return cfg, synthetic.make_checkpoint(cfg, seed=5, device="cuda")


def test_batched_step_over_pages_follows_the_one_over_caches(cuda_device):
    """Prompts of different lengths admitted, then steps of both kinds of state with the same tokens; then a fork, whose copies give the
    same logits as their parent."""
    from quickdraw_b200.batch import BatchDecode, BatchState
    from quickdraw_b200.state import DecodeState
    cfg, ckpt = small_model()
    decoder = BatchDecode(ckpt)
    lengths, context = (5, 31, 20), 64
    g = torch.Generator().manual_seed(4)
    prompts = [torch.randint(0, cfg.vocab_size, (n,), generator=g).to("cuda") for n in lengths]
    flat, pages = BatchState(cfg, 3, context, "cuda"), paged.PagedBatchState(cfg, 3, context, "cuda", page=16)
    for b, prompt in enumerate(prompts):
        one = DecodeState.allocate(cfg, context, "cuda")
        decoder.run(prompt[:-1], 0, one)
        one.position = len(prompt) - 1
        pages.admit(b, one)
        decoder.run(prompt[:-1], 0, flat.sequence(b))
        flat.positions[b] = len(prompt) - 1
    tokens = torch.stack([p[-1] for p in prompts])
    for _ in range(6):
        _, want = decoder.step(tokens, flat)
        picked, got = decoder.step(tokens, pages)
        assert O.rel_l2(got.float().cpu(), want.float().cpu()) < 2e-2 and torch.equal(pages.positions, flat.positions)
        tokens = want.float().argmax(-1)
    parents = torch.tensor([1, 1, 1], dtype=torch.int32, device="cuda")
    pages.fork(parents)
    tokens = tokens[[1, 1, 1]]
    for _ in range(20):
        picked, got = decoder.step(tokens, pages)
        assert torch.equal(got[0], got[1]) and torch.equal(got[2], got[1])
        tokens = picked
    assert pages.cache.check() == 0
    back = DecodeState.allocate(cfg, context, "cuda")
    pages.extract(2, back)
    assert back.position == lengths[1] - 1 + 26 and torch.equal(back.rec_state, pages.rec_state[0])


def test_batched_step_over_pages_from_a_graph(cuda_device):
    from quickdraw_b200.batch import BatchDecode
    cfg, ckpt = small_model()
    decoder = BatchDecode(ckpt)
    runs = []
    for method in (decoder.step, decoder.graph_step):
        state = paged.PagedBatchState(cfg, 3, 60, "cuda", page=8)
        tokens, seen = torch.tensor([3, 5, 8], device="cuda"), []
        for step in range(30):
            picked, logits = method(tokens, state)
            seen.append((picked.clone(), logits.clone()))
            tokens = picked.clone()
            if step % 7 == 6:
                state.fork(torch.tensor([2, 1, 2], dtype=torch.int32, device="cuda"))
                tokens = tokens[[2, 1, 2]]
        assert state.cache.check() == 0
        runs.append(seen)
    for (a, x), (b, y) in zip(*runs):
        assert torch.equal(a, b) and torch.equal(x, y)


def test_a_pool_that_is_too_small_is_said(cuda_device):
    from quickdraw_b200.batch import BatchDecode
    cfg, ckpt = small_model()
    decoder = BatchDecode(ckpt)
    state = paged.PagedBatchState(cfg, 2, 64, "cuda", pages=1, page=16)
    with pytest.raises(AssertionError, match="no free page"):
        decoder.step(torch.tensor([3, 5], device="cuda"), state)


def test_a_captured_step_says_each_row_that_is_lost(cuda_device):
    from quickdraw_b200.batch import BatchDecode
    cfg, ckpt = small_model()
    decoder = BatchDecode(ckpt)
    state, words = paged.PagedBatchState(cfg, 2, 32, "cuda", pages=3, page=4), []
    tokens = torch.tensor([3, 5], device="cuda")
    for step in range(14):
        if step == 10:
            state.free([0])                                     # two pages: for its place's row 0 and for the second's row 12
        decoder.graph_step(tokens, state)
        words.append(state.cache.check())
    # rows 4 to 11 of the second have no page
    assert words == [0] * 4 + [paged.NO_PAGE] * 8 + [0] * 2


def test_a_captured_step_goes_on_after_a_resize(cuda_device):
    """Pools that get smaller, and larger, between replayed steps; what the old ones' memory holds now stays as it is."""
    from quickdraw_b200.batch import BatchDecode
    cfg, ckpt = small_model()
    decoder = BatchDecode(ckpt)
    runs, others = [], []
    for method in (decoder.step, decoder.graph_step):
        state = paged.PagedBatchState(cfg, 3, 60, "cuda", pages=24, page=8)
        tokens, seen = torch.tensor([3, 5, 8], device="cuda"), []
        for step in range(24):
            picked, logits = method(tokens, state)
            seen.append((picked.clone(), logits.clone()))
            tokens = picked.clone()
            if step in (7, 15):
                was = state.cache.k.numel()
                state.cache.resize(12 if step == 7 else 20)
                others.append(torch.full((was,), 7.0, dtype=BF16, device="cuda"))
        assert state.cache.check() == 0 and int(state.cache.refs.sum()) == int((state.cache.table >= 0).sum()) == 9
        runs.append(seen)
    for (a, x), (b, y) in zip(*runs):
        assert torch.equal(a, b) and torch.equal(x, y)
    assert all(bool((t == 7.0).all()) for t in others)
