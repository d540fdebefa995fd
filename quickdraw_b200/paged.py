"""Key-value caches of many sequences in pages of one pool, shared by reference counts (the reference has one contiguous
cache for one request, quickdraw/kvcache/state.py:8-20; its decode attention is quickdraw/kernel/triton/attention.py:10-100).

Row p of sequence b is row ``p % page`` of page ``table[b][p // page]`` of the pool; an entry -1 names no page.  ``refs[i]``
counts the sequences that hold page i.  Pages are given out lowest first, in the order of the requests, so that tables are
the same from run to run.  A page that is not full belongs to one sequence.

The functions take the tensors as they are: ``paged_attention`` (one new token of every sequence), ``reserve_pages`` (rows for
the next tokens), ``fork_pages`` (sequences that go on as copies of others, or end) and ``compact_pages`` (the pages in use to
the front).  ``PagedCache`` holds the tensors of several layers; ``PagedBatchState`` is the state of a batch of sequences
for ``BatchDecode`` that can be forked (beam search, several answers to one prompt), whose pages need no more memory than
the tokens in it.

The functions stay on the device and can be captured, and so do ``reserve``, ``fork``, ``compact``, ``write`` and ``read``; ``free`` and
``admit`` take their numbers from the host (not in a capture), ``resize``, ``extract`` and ``check`` wait for it.  Calls go to the
current stream of the tensors' device.  What only the device
knows (a pool without a free page, a parent that is no sequence) sets bits of a status word, ``PagedCache.check``; nothing
outside the tensors is touched.
"""

from __future__ import annotations

import functools
import operator

import torch

from ._lib import call, lib, ptr, stream_of
from .state import DecodeState

BF16 = torch.bfloat16
BAD_ARGUMENT, NO_PAGE = 4, 8            # bits of the status word
MOST_FORKED = 12800                     # sequences that fork_pages takes at once

_status: dict = {}
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_IN_CAPTURE = "a graph's memory is not shared: call device_status(device) before the capture, or give a status"


def device_status(device) -> torch.Tensor:
    """The status word of a device (without a number: of the current one) that calls without a word of their own share."""
    word = _status.get(device)
    if word is None:
        device = torch.device(device)
        if device.type == "cuda":
            if device.index is None:
                return device_status(torch.device("cuda", _current_device()))
            assert not torch.cuda.is_current_stream_capturing(), _IN_CAPTURE
            with torch.cuda.device(device):
                assert not torch.cuda.is_current_stream_capturing(), _IN_CAPTURE
        word = _status.setdefault(device, torch.zeros(1, dtype=torch.int32, device=device))
        if device.type == "cuda":
            torch.cuda.current_stream(device).synchronize()         # any stream may use it from now on
    return word


def launch(tensor: torch.Tensor, name: str, *args) -> None:
    """A library call on the device of ``tensor``, whichever is current."""
    index = tensor.get_device()
    if index < 0 or index == _current_device():
        call(name, *args, stream_of(tensor))
    else:
        with torch.cuda.device(index):
            call(name, *args, stream_of(tensor))


@functools.lru_cache(maxsize=4096)
def scratch_size(device: int, name: str, *sizes: int) -> int:
    """What an entry point that computes a size says (these go by the device's number of SMs); a short call is as long as its host side."""
    if device < 0 or device == _current_device():
        return int(getattr(lib(), name)(*sizes))
    with torch.cuda.device(device):
        return int(getattr(lib(), name)(*sizes))


def _is_ids(t, device, *shape) -> bool:
    return t.dtype is torch.int32 and t.shape == shape and t.get_device() == device and t.is_contiguous()


def _endings(sequences, count: int, device) -> torch.Tensor:
    """The parents of a fork in which the sequences of these numbers end and all others stay."""
    sequences = list(sequences)
    assert not any(isinstance(b, bool) or getattr(b, "dtype", None) is torch.bool for b in sequences), "numbers of sequences, not a mask"
    ends = {operator.index(b) for b in sequences}            # (numbers of numpy and torch too, which need not be equal to their values in a set)
    assert all(0 <= b < count for b in ends), "no such sequence"
    return torch.tensor([-1 if b in ends else b for b in range(count)], dtype=torch.int32).to(device, non_blocking=True)


def _check_pools(k, v):
    """Pools [pages, layers, page, kv_heads, dim] whose pages are contiguous; the sizes in bytes that the kernels walk them by."""
    shape, strides = k.shape, k.stride()
    assert k.is_cuda and len(shape) == 5 and shape == v.shape and k.dtype is v.dtype and k.get_device() == v.get_device(), "two pools of one shape, type and device"
    pages, layers, page, heads, dim = shape
    size, row, at = k.element_size(), heads * dim, ptr(k) | ptr(v)
    assert pages * layers * page * row > 0 and strides[1:] == (page * row, row, dim, 1) and strides[0] >= layers * page * row, "the layers of a page are contiguous"
    assert v.stride() == strides, "the pools' pages lie alike"
    assert (at | row * size | strides[0] * size) % 16 == 0, "rows of whole 16-byte pieces"
    return strides[0] * size, page * row * size, row * size, layers


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, *,
                    scale: float | None = None, gate: torch.Tensor | None = None, window: int = 0, sinks: int = 0) -> torch.Tensor:
    """softmax(scale q k) v of one token of every sequence over its first ``lengths[b]`` cached rows, times sigmoid(gate) where
    given: [batch, heads, dim] of the type of ``q``.  A sequence that sees nothing gets zeros.

    q, gate  [batch, heads, dim], bf16 or fp32, any strides with contiguous elements; query head h uses key/value head
             h // (heads // kv_heads)
    k_pages, v_pages  [pages, page, kv_heads, dim] of the same type, any strides (alike) of whole 16-byte pieces
    table    int32 [batch, width], lengths int32 [batch], on the device; rows of entries that are no page are not seen
    scale    1 / sqrt(dim) unless given
    window   > 0: only the last ``window`` rows and the first ``sinks`` are seen (pages between them need not exist)"""
    kind = q.dtype
    assert q.is_cuda and q.ndim == 3 and kind in (BF16, torch.float32), "bf16 or fp32 queries [batch, heads, dim] on a CUDA device"
    batch, heads, dim = shape = q.shape
    device = q.get_device()
    assert k_pages.ndim == 4 and k_pages.shape == v_pages.shape and k_pages.shape[3] == dim, "pools [pages, page, kv_heads, dim]"
    assert k_pages.dtype is kind and v_pages.dtype is kind and k_pages.get_device() == device and v_pages.get_device() == device
    pages, page, kv_heads, _ = k_pages.shape
    assert batch > 0 and heads > 0 and kv_heads > 0 and heads % kv_heads == 0 and pages > 0 and page > 0
    assert 0 < dim <= 256 and dim % 8 == 0, "a head dimension of at most 256, a multiple of 8"
    assert table.ndim == 2, "a table [batch, width]"
    rows, width = table.shape
    assert table.dtype is torch.int32 and rows == batch and width > 0 and table.stride(1) == 1 and table.get_device() == device
    assert _is_ids(lengths, device, batch)
    assert width * page < 2 ** 31 - 4096, "positions of 32 bits"
    assert window >= 0 and sinks >= 0 and (window > 0 or sinks == 0), "first rows stay visible beside a window"
    page_stride, row_stride, head_stride, one = strides = k_pages.stride()
    q_row, q_head, q_one = q.stride()
    fp32 = kind is torch.float32
    at_k, at_v = ptr(k_pages), ptr(v_pages)
    assert one == 1 and v_pages.stride() == strides and q_one == 1, "contiguous elements, pools with the same strides"
    assert (at_k | at_v | (page_stride | row_stride | head_stride) * (4 if fp32 else 2)) % 16 == 0, "whole 16-byte pieces"
    gate_row = gate_head = 0
    if gate is not None:
        gate_row, gate_head, gate_one = gate.stride()
        assert gate.shape == shape and gate.dtype is kind and gate.get_device() == device and gate_one == 1
    out = torch.empty_like(q) if q.is_contiguous() else q.new_empty(shape)
    floats = scratch_size(device, "qd_paged_attention_floats", batch, heads, kv_heads, dim,
                          min(width * page, window + sinks) if window else width * page)
    partial = q.new_empty(floats if fp32 else 2 * floats) if floats else None
    launch(q, "qd_paged_attention", ptr(q), q_row, q_head, at_k, at_v, page_stride, row_stride, head_stride, ptr(table), table.stride(0), ptr(lengths),
           ptr(gate), gate_row, gate_head, ptr(out), ptr(partial), batch, heads, kv_heads, dim, pages, page, width,
           window if window < 2 ** 31 else 2 ** 31 - 1, sinks if sinks < 2 ** 31 else 2 ** 31 - 1, dim ** -0.5 if scale is None else scale, int(fp32))
    return out


def _check_tables(table, refs, device):
    """A table [sequences, width] and counts [pages] on `device`; their sizes, and scratch for them."""
    assert table.dtype is torch.int32 and refs.dtype is torch.int32 and table.get_device() == device and refs.get_device() == device
    assert table.ndim == 2 and refs.ndim == 1 and table.is_contiguous() and refs.is_contiguous()
    (count, width), (pages,) = table.shape, refs.shape
    assert 0 < count * width < 2 ** 31 - 8192 and pages > 0
    return count, width, pages, table.new_empty(scratch_size(device, "qd_pages_scratch_words", count, width, pages))


def fork_pages(k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, refs: torch.Tensor, parents: torch.Tensor, *,
               status: torch.Tensor | None = None):
    """Sequence b goes on as a copy of sequence ``parents[b]``, all at once: the new (table, lengths, refs).  -1: the sequence ends
    and gives up its pages; its own number: it stays as it is.  Full pages are shared.  A page that is not full goes to the parent
    itself where that stays, or else to the lowest child; every other child gets the lowest free page and a copy of its rows, in
    the order of the children.  Only those rows are written, in ``k_pages`` and ``v_pages`` [pages, layers, page, kv_heads, dim].  Rows that
    the parent has no page for (they are not seen) no child has a page for either.

    A parent that is no sequence leaves its child as it is, and a child for which no page is left ends where its full pages do; both
    set bits of ``status`` (int32 [1]; a word shared by the device, ``device_status``, if not given)."""
    page_bytes, layer_bytes, row_bytes, layers = _check_pools(k_pages, v_pages)
    device, (in_pool, _, page, _, _) = k_pages.get_device(), k_pages.shape
    count, width, pages, scratch = _check_tables(table, refs, device)
    assert _is_ids(lengths, device, count) and _is_ids(parents, device, count) and pages == in_pool and width * page < 2 ** 31
    assert count <= MOST_FORKED, "1 to 12800 sequences"
    status = device_status(k_pages.device) if status is None else status
    assert _is_ids(status, device, 1)
    table_out, lengths_out, refs_out = torch.empty_like(table), torch.empty_like(lengths), torch.empty_like(refs)
    launch(k_pages, "qd_pages_fork", ptr(k_pages), ptr(v_pages), page_bytes, layer_bytes, row_bytes, layers, ptr(table), ptr(lengths), ptr(refs),
           ptr(parents), ptr(table_out), ptr(lengths_out), ptr(refs_out), ptr(scratch), ptr(status), count, width, pages, page)
    return table_out, lengths_out, refs_out


def compact_pages(k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor, refs: torch.Tensor):
    """The pages in use (``refs > 0``) become the first ones of the pool: those behind move, in order, to the free ones in front.  The
    new (table, refs) and the number of pages in use (0-d int32, on the device).  Pages that are not used any more keep what they
    hold."""
    page_bytes, layer_bytes, row_bytes, layers = _check_pools(k_pages, v_pages)
    in_pool, _, page, _, _ = k_pages.shape
    count, width, pages, scratch = _check_tables(table, refs, k_pages.get_device())
    assert pages == in_pool
    table_out, refs_out, used = torch.empty_like(table), torch.empty_like(refs), table.new_empty(())
    launch(k_pages, "qd_pages_compact", ptr(k_pages), ptr(v_pages), page_bytes, layer_bytes, row_bytes, layers, ptr(table), ptr(refs), ptr(table_out),
           ptr(refs_out), ptr(used), ptr(scratch), count, width, pages, page)
    return table_out, refs_out, used


def reserve_pages(table: torch.Tensor, lengths: torch.Tensor, refs: torch.Tensor, page: int, counts=1, *, begun: bool = False,
                  status: torch.Tensor | None = None) -> None:
    """Pages for the next ``counts`` rows (a number, or int32 [sequences] on the device) of every sequence, in place in ``table`` and
    ``refs``: the lowest free ones, in the order of the sequences.  Rows past the table and an empty pool set bits of ``status``.

    A page is given for its first row: where the pool had none then, the sequence has none for the page's other rows, which are lost like
    the first.  ``begun``: that sets the bit of an empty pool too, as long as such rows are asked for."""
    assert table.is_cuda
    device = table.get_device()
    count, width, pages, scratch = _check_tables(table, refs, device)
    each = isinstance(counts, torch.Tensor)
    assert _is_ids(lengths, device, count) and page > 0 and width * page < 2 ** 31
    assert _is_ids(counts, device, count) if each else 0 <= counts < 2 ** 31, "rows to come: a number, or int32 for every sequence"
    status = device_status(table.device) if status is None else status
    assert _is_ids(status, device, 1)
    launch(table, "qd_pages_reserve", ptr(table), ptr(lengths), ptr(refs), ptr(counts) if each else None, 0 if each else int(counts),
           ptr(scratch), ptr(status), count, width, pages, page, int(begun))


class PagedCache:
    """Pools of ``pages`` pages for ``layers`` attention layers, tables of ``sequences`` sequences of at most ``max_context`` rows.

    ``k``, ``v`` [pages, layers, page, kv_heads, head_dim]; ``table``, ``lengths``, ``refs``, ``status`` int32 on the device.  The methods
    write into these tensors, which a captured graph may therefore hold; ``resize`` alone replaces ``k``, ``v`` and ``refs``."""

    def __init__(self, layers: int, kv_heads: int, head_dim: int, pages: int, page: int, sequences: int, max_context: int, device,
                 dtype: torch.dtype = BF16):
        assert min(layers, kv_heads, head_dim, pages, page, sequences, max_context) > 0 and dtype in (BF16, torch.float32)
        self.page, self.sequences, self.max_context = page, sequences, max_context
        self.k = torch.zeros((pages, layers, page, kv_heads, head_dim), dtype=dtype, device=device)
        self.v = torch.zeros_like(self.k)
        self.table = torch.full((sequences, -(-max_context // page)), -1, dtype=torch.int32, device=device)
        self.lengths = torch.zeros(sequences, dtype=torch.int32, device=device)
        self.refs = torch.zeros(pages, dtype=torch.int32, device=device)
        self.status = torch.zeros(1, dtype=torch.int32, device=device)
        self.resized = 0                    # how often: a graph that was captured before the last time must not run any more

    @property
    def pages(self) -> int:
        return self.refs.numel()

    def reserve(self, counts=1) -> None:
        """Room for the next ``counts`` rows of every sequence (``reserve_pages``); each call that leaves some without a page says so in
        ``status``."""
        reserve_pages(self.table, self.lengths, self.refs, self.page, counts, begun=True, status=self.status)

    def fork(self, parents: torch.Tensor) -> None:
        """Sequence b goes on as a copy of sequence ``parents[b]`` (``fork_pages``)."""
        table, lengths, refs = fork_pages(self.k, self.v, self.table, self.lengths, self.refs, parents, status=self.status)
        self.table.copy_(table)
        self.lengths.copy_(lengths)
        self.refs.copy_(refs)

    def free(self, sequences) -> None:
        """The sequences of these numbers end."""
        self.fork(_endings(sequences, self.sequences, self.table.device))

    def compact(self) -> torch.Tensor:
        """The pages in use to the front (``compact_pages``); their number, on the device."""
        table, refs, used = compact_pages(self.k, self.v, self.table, self.refs)
        self.table.copy_(table)
        self.refs.copy_(refs)
        return used

    def resize(self, pages: int) -> None:
        """Pools of ``pages`` pages, at least as many as are in use: what is not used is given back, or there is more of it.  Waits for
        the device.  A graph captured before has the addresses of the old pools, whose memory is given back, and must not be replayed:
        ``BatchDecode.graph_step`` sees to its own; ``resized`` counts."""
        assert pages > 0
        used = int(self.compact().item())
        assert pages >= used, f"{used} pages are in use"
        kept = min(pages, self.pages)
        for name in ("k", "v", "refs"):
            old = getattr(self, name)
            new = torch.zeros((pages, *old.shape[1:]), dtype=old.dtype, device=old.device)
            new[:kept] = old[:kept]
            setattr(self, name, new)
        self.resized += 1

    def _rows(self, b: int, k: torch.Tensor, v: torch.Tensor, first: int, count: int, out: bool) -> None:
        pages, layers, page, heads, dim = self.k.shape
        size, row = self.k.element_size(), heads * dim
        assert 0 <= b < self.sequences and 0 <= first and count >= 0 and first + count <= self.table.shape[1] * page
        for t in (k, v):
            assert t.dtype is self.k.dtype and t.device == self.k.device and t.ndim == 4 and t.shape[0] == layers and t.shape[2:] == (heads, dim)
            assert t.shape[1] >= count and t.stride()[1:] == (row, dim, 1) and t.stride(0) == k.stride(0), "rows [layers, count, kv_heads, head_dim], contiguous in a layer"
        launch(self.k, "qd_pages_rows", ptr(self.k), ptr(self.v), self.k.stride(0) * size, page * row * size, row * size, ptr(k), ptr(v), k.stride(0) * size,
               ptr(self.table[b]), ptr(self.status), layers, self.table.shape[1], pages, page, first, count, int(out))

    def write(self, b: int, k: torch.Tensor, v: torch.Tensor, first: int, count: int) -> None:
        """Rows first .. first + count - 1 of sequence b, whose pages are set aside, from k, v [layers, >= count, kv_heads, head_dim].  Rows of
        pages that it shares are theirs too who share them."""
        self._rows(b, k, v, first, count, False)

    def read(self, b: int, k: torch.Tensor, v: torch.Tensor, first: int, count: int) -> None:
        """The same rows from the pages into k, v."""
        self._rows(b, k, v, first, count, True)

    def check(self) -> int:
        """The status word (0: nothing went wrong), which is cleared; waits for the device."""
        word = int(self.status.item())
        if word:
            self.status.zero_()
        return word

    def memory_bytes(self) -> int:
        return sum(t.nbytes for t in (self.k, self.v, self.table, self.lengths, self.refs))


class PagedBatchState:
    """The state of ``batch`` sequences for ``BatchDecode``, like ``BatchState``, with the attention layers' rows in a pool of ``pages``
    pages of ``page`` rows (default: enough for ``max_context`` rows of every sequence).  ``admit`` takes a prefilled prompt in, ``fork``
    lets sequences go on as copies of others, ``free`` ends them.

    A step appends a token to every place, to an empty one as well, which takes pages as any other does until it is freed again; where
    a pool runs out of them ``cache.check`` says so.  ``admit`` may move a position past what a captured step (``graph_step``) has
    counted to: ``BatchDecode.forget`` the state then."""

    def __init__(self, config, batch: int, max_context: int, device, pages: int | None = None, page: int = 64):
        one = DecodeState.allocate(config, 1, "meta")
        enough = batch * -(-max_context // page)
        self.cache = PagedCache(one.kv_k.shape[0], config.num_key_value_heads, config.head_dim, enough if pages is None else pages, page, batch, max_context,
                                device)
        self.rec_state = torch.zeros((batch, *one.rec_state.shape), dtype=torch.float32, device=device)
        self.conv_state = torch.zeros((batch, *one.conv_state.shape), dtype=BF16, device=device)
        self.positions = self.cache.lengths
        self.seen = torch.zeros(batch, dtype=torch.int32, device=device)        # rows that the step's attention sees
        self.batch, self.max_context = batch, max_context

    def admit(self, b: int, state: DecodeState) -> None:
        """Sequence b becomes a copy of a single sequence that was run elsewhere (a prefilled prompt)."""
        n = state.position
        assert 0 <= b < self.batch and 0 <= n <= min(self.max_context, state.kv_k.shape[1]), "the sequence does not fit"
        self.cache.free([b])
        counts = torch.zeros(self.batch, dtype=torch.int32)
        counts[b] = n
        self.cache.reserve(counts.to(self.cache.table.device, non_blocking=True))
        self.cache.write(b, state.kv_k, state.kv_v, 0, n)
        self.cache.lengths[b] = n
        self.rec_state[b].copy_(state.rec_state)
        self.conv_state[b].copy_(state.conv_state)

    def extract(self, b: int, state: DecodeState) -> None:
        """The other way: sequence b into a single sequence's buffers.  Waits for the device (its length is there)."""
        n = int(self.cache.lengths[b].item())
        assert n <= state.kv_k.shape[1], "the sequence does not fit"
        self.cache.read(b, state.kv_k, state.kv_v, 0, n)
        state.rec_state.copy_(self.rec_state[b])
        state.conv_state.copy_(self.conv_state[b])
        state.position = n

    def fork(self, parents: torch.Tensor) -> None:
        """Sequence b goes on as a copy of sequence ``parents[b]`` (int32 [batch], on the device; -1: it ends, with an empty history)."""
        from .beam import reorder_states
        self.cache.fork(parents)
        reorder_states([self.rec_state, self.conv_state], parents, status=self.cache.status)

    def free(self, sequences) -> None:
        """The sequences of these numbers end; their places are empty."""
        self.fork(_endings(sequences, self.batch, self.cache.table.device))

    def memory_bytes(self) -> int:
        return self.cache.memory_bytes() + self.rec_state.nbytes + self.conv_state.nbytes
