"""A paged cache of routed keys and dense values, and the outer routed attention over it.

A served model keeps what the outer attention reads of earlier tokens: the routed keys of every branch and the dense
value, per layer.  They lie in pages of a fixed number of positions, so that sequences of any lengths share one pool:
position j of sequence b is slot ``j % page`` of page ``table[b, j // page]``.  A step brings new tokens of some or all
sequences, packed one sequence after another (:class:`PagedBatch`); :func:`append_paged` puts their keys and values
into the pages, :func:`routed_attention_paged` lets each new token attend over its sequence up to itself, from single
tokens to long chunks.  :class:`RoutedCache` holds the pages of all layers of a model and hands them out.

The sizes that vary from step to step are read by the kernels on the device: neither operator waits for the GPU, and a captured
graph follows them.  A page number outside the cache, or a length that the table has no room for, is never followed:
those positions are not written, the tokens that would need them (and others of their tile of 128 new tokens) get NaN, and
``ops.device_status`` reports bit 8, on the stream that the call ran on or was captured on.

Inference only: the operators raise on tensors that require a gradient.
"""

from __future__ import annotations

from typing import NamedTuple, Sequence

import torch
from torch import Tensor

from . import _lib, ops
from ._lib import ptr
from .eight_bit import _CODES, _HALF, _device_of, _host, _inference_only, _launch

BAD_PAGE = 8  # bit of ops.device_status


class PagedBatch(NamedTuple):
    """The sequences of one step.

    table: int32 [B, pages a sequence], unit column stride; entries that no position needs may hold anything.
    lengths: int32 [B], tokens that each sequence had before the step.
    starts: int32 [B + 1], where each sequence's new tokens begin among the packed rows (``starts[0]`` is 0, ``starts[B]``
        their number; rows behind it belong to no sequence, and sequences may have none).
    max_new: the largest number of new tokens of one sequence, if known: chooses the kernel, changes no result's meaning.
    """

    table: Tensor
    lengths: Tensor
    starts: Tensor
    max_new: int | None = None


def _check_batch(name: str, batch: PagedBatch) -> int:
    table, lengths, starts, _max_new = batch
    for what, t in (("table", table), ("lengths", lengths), ("starts", starts)):
        if t.dtype != torch.int32:
            raise ValueError(f"{name} takes its {what} in int32, got {t.dtype}")
    b = lengths.shape[0] if lengths.ndim == 1 else -1
    if table.ndim == 2 and not table.shape[1]:
        raise ValueError(f"{name} takes a table of at least one page a sequence")
    if table.ndim != 2 or table.shape[0] != b or starts.shape != (b + 1,):
        raise ValueError(f"{name} takes a table [B, pages], lengths [B] and starts [B + 1], got {tuple(table.shape)}, "
                         f"{tuple(lengths.shape)} and {tuple(starts.shape)}")
    return b


def _table_args(batch: PagedBatch) -> tuple[Tensor, Tensor, Tensor]:
    table = batch.table
    if table.shape[1] > 1 and table.stride(1) != 1 or table.shape[0] > 1 and table.stride(0) < table.shape[1]:
        table = table.contiguous()
    return table, batch.lengths.contiguous(), batch.starts.contiguous()


def _check_pages(name: str, key_pages: Tensor, value_pages: Tensor) -> tuple[int, int, int, int, int]:
    if key_pages.ndim != 4 or value_pages.ndim != 3 or value_pages.shape[:2] != key_pages.shape[:2]:
        raise ValueError(f"{name} takes key pages [pages, page, H, R] and value pages [pages, page, D], got "
                         f"{tuple(key_pages.shape)} and {tuple(value_pages.shape)}")
    if key_pages.dtype not in _HALF or value_pages.dtype != key_pages.dtype:
        raise ValueError(f"{name} takes pages of one type, bfloat16 or float16, got {key_pages.dtype} and {value_pages.dtype}")
    if not key_pages.is_contiguous() or not value_pages.is_contiguous():
        raise ValueError(f"{name} takes contiguous pages")
    pages, page, h, r = key_pages.shape
    if page < 16 or page > 65536 or page & (page - 1):
        raise ValueError(f"{name} takes pages of 16 to 65536 positions, a power of two, got {page}")
    if not pages:
        raise ValueError(f"{name} takes at least one page")
    return pages, page, h, r, value_pages.shape[2]


def append_paged(keys: Tensor, values: Tensor, key_pages: Tensor, value_pages: Tensor, batch: PagedBatch) -> None:
    """Writes the packed new tokens' keys [H, N, R] and values [N, D] behind what their sequences have, in place.

    Token i of sequence b goes to position ``batch.lengths[b] + i``, in a page that no other sequence writes; the lengths stay as
    they are.  Keys and values in
    fp32, bf16 or fp16 with unit column stride or any other (copied first then), rounded once to the pages' type.  Nothing
    but the new positions is written."""
    name = "append_paged"
    if key_pages.is_cuda and _host().append_paged(keys, values, key_pages, value_pages, batch[0], batch[1], batch[2],
                                                  ops.workspace(key_pages.device).status):
        return
    b = _check_batch(name, batch)
    pages, page, h, r, d = _check_pages(name, key_pages, value_pages)
    if keys.ndim != 3 or keys.shape[0] != h or keys.shape[2] != r or values.shape != (keys.shape[1], d):
        raise ValueError(f"{name} takes keys [{h}, N, {r}] and values [N, {d}], got {tuple(keys.shape)} and {tuple(values.shape)}")
    if r % 8 or d % 8:
        raise NotImplementedError(f"{name} covers routing and value widths divisible by 8, got {r} and {d}")
    k_code, v_code = _CODES.get(keys.dtype), _CODES.get(values.dtype)
    if k_code is None or v_code is None:
        raise ValueError(f"{name} takes keys and values in float32, bfloat16 or float16, got {keys.dtype} and {values.dtype}")
    device = _device_of(name, key_pages, value_pages, keys, values, *batch[:3])
    _inference_only(name, keys, values, key_pages, value_pages)
    n = keys.shape[1]
    if not n or not b:
        return
    keys = keys if keys.stride(2) == 1 else keys.contiguous()
    values = values if values.stride(1) == 1 else values.contiguous()
    table, lengths, starts = _table_args(batch)
    _launch(device, "da_paged_append", keys.data_ptr(), k_code, keys.stride(0), keys.stride(1), values.data_ptr(), v_code,
            values.stride(0), n, key_pages.data_ptr(), value_pages.data_ptr(), _CODES[key_pages.dtype], pages, page, h, r, d,
            table.data_ptr(), table.stride(0) if b > 1 else table.shape[1], table.shape[1], lengths.data_ptr(),
            starts.data_ptr(), b, ops.workspace(key_pages.device).status.data_ptr())


def _aligned_query(q: Tensor) -> Tensor:
    """``q`` [H, N, R] with branches and rows on 16 bytes: as it lies, or a copy."""
    h, n, r = q.shape
    if q.stride(2) != 1 or q.data_ptr() % 16 or n > 1 and (q.stride(1) % 8 or q.stride(1) < r) \
            or h > 1 and (q.stride(0) % 8 or q.stride(0) < r):
        q = q.contiguous()
        if q.data_ptr() % 16:
            q = q.clone()
    return q


def _extent(t: Tensor) -> tuple[int, int]:
    """First byte of ``t``, and the one behind its last."""
    last = sum((n - 1) * step for n, step in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size() if t.numel() else t.data_ptr()


def _check_apart(name: str, out: Tensor, *inputs: Tensor) -> None:
    first, end = _extent(out)
    for t in inputs:
        a, b = _extent(t)
        if t.device == out.device and first < b and a < end:
            raise ValueError(f"{name} cannot write over what it reads: out shares memory with an input")


def routed_attention_paged(query: Tensor, key_pages: Tensor, value_pages: Tensor, batch: PagedBatch, scales: Tensor,
                           map_weights: Tensor | None = None, *, out: Tensor | None = None) -> Tensor:
    """Outer routed attention of the packed new tokens over the pages, after :func:`append_paged` put them there.

    query [H, N, R] of the pages' type; ``scales`` [S] the maps' temperatures, S of H branches as in
    :func:`assemble_score_maps`.  Token i of sequence b sees positions 0 to ``batch.lengths[b] + i``.  With
    ``map_weights`` [S], or one map, returns the maps' mixture [N, D]; without, several maps' outputs [N, S, D].  The
    keys may be of any length: the softmax takes off each row's own maximum.  What a token does not see may hold anything;
    where a key or a value that it sees is not finite, its outputs (of any map) are not.  Rows of no sequence are zero,
    or left as they are in ``out``, which shares no memory with the inputs.

    Supported: R a multiple of 64, D 128, 256 or 512, up to 4 maps and ``max(H, S) * R`` up to 512."""
    name = "routed_attention_paged"
    if out is None and query.is_cuda:
        y = _host().attend_paged(query, key_pages, value_pages, *batch, scales, map_weights, ops.workspace(query.device).status)
        if y is not None:
            return y
    b = _check_batch(name, batch)
    pages, page, h, r, d = _check_pages(name, key_pages, value_pages)
    if query.ndim != 3 or query.shape[0] != h or query.shape[2] != r:
        raise ValueError(f"{name} takes a query [{h}, N, {r}], got {tuple(query.shape)}")
    if query.dtype != key_pages.dtype:
        raise ValueError(f"{name} takes a query of the pages' type {key_pages.dtype}, got {query.dtype}")
    maps = scales.shape[0] if scales.ndim == 1 else 0
    if not maps or (h % maps and maps % h):
        raise ValueError(f"{name} takes one scale a map, their number dividing the {h} branches or divided by it, "
                         f"got {tuple(scales.shape)}")
    if map_weights is not None and map_weights.shape != (maps,):
        raise ValueError(f"{name} takes {maps} map weights, got {tuple(map_weights.shape)}")
    ops._attention_supported(r, d, maps, max(h // maps, 1))
    n = query.shape[1]
    per_map = maps > 1 and map_weights is None
    shape = (n, maps, d) if per_map else (n, d)
    if out is not None and (out.shape != shape or out.dtype != query.dtype or not out.is_contiguous()
                            or out.data_ptr() % 16):
        raise ValueError(f"{name} writes a contiguous, 16-byte aligned {query.dtype} tensor {shape}, got {out.dtype} {tuple(out.shape)}")
    if out is not None:
        _check_apart(name, out, query, key_pages, value_pages)
    device = _device_of(name, key_pages, value_pages, query, scales, map_weights, out, *batch[:3])
    _inference_only(name, query, key_pages, value_pages, scales, map_weights, out)
    y = torch.empty(shape, dtype=query.dtype, device=query.device) if out is None else out
    if not n:
        return y
    if not b:
        return y.zero_() if out is None else y
    query = _aligned_query(query)
    scales = scales.float().contiguous()
    weights = None if per_map or map_weights is None else map_weights.float().contiguous()
    table, lengths, starts = _table_args(batch)
    most = n if batch.max_new is None else batch.max_new
    with torch.cuda.device(device):
        need = _lib.lib().da_paged_attn_workspace_size(n, b, table.shape[1], page, most, h, r, d, maps, int(per_map))
    work = torch.empty(need, dtype=torch.uint8, device=query.device) if need > 0 else None
    _launch(device, "da_paged_attn", query.data_ptr(), query.stride(0), query.stride(1) if n > 1 else r, n, key_pages.data_ptr(),
            value_pages.data_ptr(), _CODES[query.dtype], pages, page, h, r, d, maps, table.data_ptr(),
            table.stride(0) if b > 1 else table.shape[1], table.shape[1], lengths.data_ptr(), starts.data_ptr(), b, most,
            scales.data_ptr(), ptr(weights), int(per_map), int(out is None), y.data_ptr(), ptr(work), max(need, 0),
            ops.workspace(query.device).status.data_ptr())
    return y


def extend(routed: Tensor, value: Tensor, cache: tuple[Tensor, Tensor, PagedBatch], scales: Tensor,
           map_weights: Tensor | None) -> Tensor:
    """Module path: routed [2, H, 1, N, R] and value [1, N, D] of packed new tokens into the pages, and their attention over
    them."""
    key_pages, value_pages, batch = cache
    if routed.dtype != key_pages.dtype:
        raise ValueError(f"the attention computes in {routed.dtype}, the cache holds {key_pages.dtype}")
    append_paged(routed[1, :, 0], value[0], key_pages, value_pages, batch)
    return routed_attention_paged(routed[0, :, 0], key_pages, value_pages, batch, scales, map_weights)


class RoutedCache:
    """The pages of all layers of a model for ``sequences`` sequences, and who has which.

    ``max_length`` positions a sequence.  Without ``pages`` every sequence owns its pages from the start, and a step
    (``DoubleAttentionLM.extend``, ``Int8DoubleAttentionLM.extend``) of as many new tokens of every sequence can be captured into
    a CUDA graph: the device's ``lengths`` advance with every replay.  With fewer ``pages`` sequences share a pool: a step takes
    what its new tokens need and raises if there is none left; ``release`` gives a sequence's pages back.  A pool's steps cannot
    be captured, as no replay would reserve pages.  Once a step has been captured, every other one reads the lengths back from
    the device first, and waits for it: replays have moved them.  A replay that runs past ``max_length``, or the positions that
    the model has, writes nothing of such a sequence, gives it NaN and sets ``ops.device_status`` bit 8.  Not for several
    threads at once."""

    def __init__(self, config, layers: int, sequences: int, max_length: int, *, page_size: int = 64, pages: int | None = None,
                 dtype: torch.dtype = torch.bfloat16, device: torch.device | str = "cuda") -> None:
        if not config.causal:
            raise ValueError("a cache serves causal attention: later tokens change nothing of earlier ones")
        if dtype not in _HALF:
            raise ValueError(f"a cache holds bfloat16 or float16, got {dtype}")
        if layers < 1 or sequences < 1 or max_length < 1:
            raise ValueError(f"a cache has at least one layer, sequence and position, got {layers}, {sequences} and {max_length}")
        if page_size < 16 or page_size > 65536 or page_size & (page_size - 1):
            raise ValueError(f"pages have 16 to 65536 positions, a power of two, got {page_size}")
        columns = -(-max_length // page_size)
        own = pages is None
        pages = sequences * columns if own else pages
        if pages < 1:
            raise ValueError(f"a cache has at least one page, got {pages}")
        self.page_size, self.max_length, self.sequences, self.layers, self.dtype = page_size, max_length, sequences, layers, dtype
        shape = (config.qk_branches, config.routing_dim)
        # (zeros: a chunk over slots that hold NaN is computed twice)
        self.key_pages = torch.zeros(layers, pages, page_size, *shape, dtype=dtype, device=device)
        self.value_pages = torch.zeros(layers, pages, page_size, config.model_dim, dtype=dtype, device=device)
        self.lengths = torch.zeros(sequences, dtype=torch.int32, device=device)
        # (-1 where a sequence has no page: a step that was not reserved is reported, and writes nothing)
        self.table = torch.full((sequences, columns), -1, dtype=torch.int32, device=device)
        self._owned: list[list[int]] = [[] for _ in range(sequences)]
        self._free = list(range(pages - 1, -1, -1))
        self._held = [0] * sequences  # the lengths as the host knows them
        self._captured = False        # whether it may not, as replays move them
        if own:
            self.table.copy_(torch.arange(pages, dtype=torch.int32).view(sequences, columns))
            self._owned = [list(range(b * columns, (b + 1) * columns)) for b in range(sequences)]
            self._free = []
        self._fixed = own

    def layer(self, index: int) -> tuple[Tensor, Tensor]:
        """Key and value pages of one layer."""
        return self.key_pages[index], self.value_pages[index]

    def _capturing(self) -> bool:
        return self.table.is_cuda and torch.cuda.is_current_stream_capturing()

    def _known_lengths(self) -> list[int]:
        """The lengths that a step is checked against (none in a capture: its replays bring their own)."""
        if self._capturing():
            self._captured |= self._fixed
            return [0] * self.sequences
        if self._captured:
            self._held = self.lengths.tolist()
        return self._held

    def step(self, counts: Sequence[int], positions: int | None = None) -> PagedBatch:
        """The batch of a step that brings ``counts[b]`` new tokens of sequence b, its pages reserved.  ``positions``: the most
        that the model has, which replays of a captured step are held to."""
        if len(counts) != self.sequences or any(n < 0 for n in counts):
            raise ValueError(f"a step takes a number of new tokens for each of the {self.sequences} sequences, got {list(counts)}")
        if self._capturing():
            if not self._fixed:
                raise RuntimeError("a step of a cache whose sequences share a pool cannot be captured: replays reserve no pages")
            if any(n != counts[0] for n in counts):
                raise RuntimeError(f"a captured step brings as many new tokens of every sequence, got {list(counts)}")
        lengths = self._known_lengths()
        for b, n in enumerate(counts):
            if lengths[b] + n > self.max_length:
                raise ValueError(f"sequence {b} has {lengths[b]} tokens: {n} more exceed the cache's {self.max_length}")
        if not self._fixed:
            want = [max(0, -(-(held + n) // self.page_size) - len(owned))
                    for held, n, owned in zip(self._held, counts, self._owned)]
            if sum(want) > len(self._free):
                raise RuntimeError(f"the step needs {sum(want)} more pages, the cache has {len(self._free)} left")
            for b, n in enumerate(want):
                if n:
                    have = len(self._owned[b])
                    taken = [self._free.pop() for _ in range(n)]
                    self._owned[b] += taken
                    self.table[b, have:have + n] = torch.tensor(taken, dtype=torch.int32).to(self.table.device)
        n = counts[0]
        if all(c == n for c in counts):
            starts = torch.arange(self.sequences + 1, dtype=torch.int32, device=self.table.device) * n
        else:
            ends = [0]
            for c in counts:
                ends.append(ends[-1] + c)
            starts = torch.tensor(ends, dtype=torch.int32).to(self.table.device)
        held = self.lengths
        if self._capturing():
            # (the table's last page may have room behind max_length: a length that no table has room for, instead)
            most = self.max_length if positions is None else min(self.max_length, positions)
            held = held.masked_fill(held > most - n, torch.iinfo(torch.int32).max)
        return PagedBatch(self.table, held, starts, max(counts))

    def advance(self, counts: Sequence[int], batch: PagedBatch) -> None:
        """Counts a step's tokens in, after its last layer."""
        self.lengths.add_(batch.starts[1:] - batch.starts[:-1])
        if self._capturing():  # (nothing has come yet; replays bring them)
            self._captured = True
        else:
            self._held = [held + n for held, n in zip(self._held, counts)]

    def release(self, sequence: int | None = None) -> None:
        """Forgets a sequence's tokens, or all: its next step starts at position 0."""
        if self._capturing():
            if not self._fixed:
                raise RuntimeError("pages given back to a pool cannot be captured: replays would give back others' pages")
            self._captured = True
        for b in range(self.sequences) if sequence is None else (sequence,):
            self._held[b] = 0
            self.lengths[b] = 0
            if not self._fixed:
                self._free += reversed(self._owned[b])
                self._owned[b] = []
                self.table[b] = -1

    def rows(self, token_ids: Tensor, counts: Sequence[int] | None, positions: int) -> tuple[Tensor, list[int]]:
        """The packed ids of a step and its counts, checked against a model of ``positions`` positions: ids [B, T], or [N]
        with ``counts``."""
        if counts is None:
            if token_ids.ndim != 2 or token_ids.shape[0] != self.sequences:
                raise ValueError(f"token_ids must have shape [{self.sequences}, T], or [N] with counts, got {tuple(token_ids.shape)}")
            numbers = [token_ids.shape[1]] * self.sequences
        else:
            numbers = [int(n) for n in counts]
            if token_ids.ndim != 1 or token_ids.shape[0] != sum(numbers):
                raise ValueError(f"token_ids must have shape [{sum(numbers)}], one sequence after another, got {tuple(token_ids.shape)}")
        for held, n in zip(self._known_lengths(), numbers):
            if held + n > positions:
                raise ValueError(f"sequence length {held + n} exceeds configured maximum {positions}")
        return token_ids.reshape(-1), numbers

    def positions(self, batch: PagedBatch, numbers: Sequence[int], most: int) -> Tensor:
        """Each packed row's position in its sequence (at most ``most - 1``, where a replayed graph runs over it and its rows
        become NaN)."""
        n, first = sum(numbers), numbers[0]
        row = torch.arange(n, device=self.lengths.device)
        if all(c == first for c in numbers):
            sequence = row // max(first, 1)
        else:
            sequence = torch.repeat_interleave(torch.arange(self.sequences), torch.tensor(numbers)).to(self.lengths.device)
        return (self.lengths[sequence] + row - batch.starts[sequence]).clamp(max=most - 1)
