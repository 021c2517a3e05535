"""Sequences of different lengths packed into one run of rows.

    pack = SequencePack(q_lengths, k_lengths)      # once per batch
    out = kernels.causal_attention(q, k, v, pack)  # every layer

The counterpart, for packed sequences, of the tile layout of a clip: the row
offsets on the device and, per number of query heads that share a key head,
the work tables that the attention kernels walk. All of it comes from the
lengths on the host, so a pack that exists is consistent, and no call that
uses it reads the device. Making it is not free: the offsets, and the tables at
the first call for a number of heads (those of the backward with them), are
copied to the device by copies that wait for what the stream has queued, and
the host takes 0.05 ms for the first and 0.2 to 0.7 ms for the second. Keep a
pack for all layers of a batch.
"""

from __future__ import annotations

import dataclasses
from typing import Sequence

import numpy as np
import torch

# Rows of a query tile and keys of a key tile of the attention kernels.
TILE = 128
# Fields of a work item (one int32 each; csrc/causal.cuh).
ITEM_FIELDS = 8


@dataclasses.dataclass(frozen=True)
class WorkTables:
    """Work items of one group size and number of key heads: forward (pairs
    of query tiles, or parts of them), joins (of the parts), query gradient
    (query tiles) and key gradient (key tiles), each [n, 8] int32 on the
    device, longest first; `order`, which deals the last to the processors
    (may be empty); `n_tiles` query tiles and `n_parts` parts in all."""

    forward: torch.Tensor
    joins: torch.Tensor
    query: torch.Tensor
    key: torch.Tensor
    order: torch.Tensor
    n_tiles: int
    n_parts: int
    # Address and items of each table, as a launch passes them.
    forward_args: tuple[int, int, int, int, int]
    gradient_args: tuple[int, int, int, int, int, int, int, int]
    stream: int


class SequencePack:
    """Row ranges of packed sequences.

    Sequence b owns `q_lengths[b]` consecutive query rows and `k_lengths[b]`
    consecutive key rows (the same rows by default). Its queries are the last
    tokens of its keys: query i sees keys j <= i + k_length - q_length. With
    fewer keys than queries the first rows see none. Any length may be zero.

    A captured CUDA graph reads the pack's tensors: keep the pack for as long
    as the graph is replayed.

    Args:
        q_lengths: Query rows of each sequence (host integers).
        k_lengths: Key rows of each sequence; None for q_lengths.
        device: CUDA device of the offsets and tables.
    """

    def __init__(self, q_lengths: Sequence[int],
                 k_lengths: Sequence[int] | None = None,
                 device: torch.device | str = 'cuda'):
        self.q_lengths = _lengths(q_lengths, 'q_lengths')
        self.k_lengths = (self.q_lengths if k_lengths is None
                          else _lengths(k_lengths, 'k_lengths'))
        if self.q_lengths.size != self.k_lengths.size:
            raise ValueError('q_lengths and k_lengths must name the same '
                             f'sequences: {self.q_lengths.size} and '
                             f'{self.k_lengths.size}')
        self.device = torch.device(device)
        if self.device.type == 'cuda' and self.device.index is None:
            self.device = torch.device('cuda', torch.cuda.current_device())
        self.total_q = int(self.q_lengths.sum())
        self.total_k = int(self.k_lengths.sum())
        if max(self.total_q, self.total_k) >= 2 ** 31 - 2 * TILE:
            raise ValueError('a pack holds fewer than 2^31 - 256 rows')
        self._q0 = np.concatenate([[0], np.cumsum(self.q_lengths)])
        self._k0 = np.concatenate([[0], np.cumsum(self.k_lengths)])
        both = _to_device(np.stack([self._q0, self._k0]), self.device)
        self.q_offsets, self.k_offsets = both[0], both[1]
        self._stream = _stream(self.device)
        self.n_sequences = self.q_lengths.size
        # Every sequence has exactly one query.
        self.single_tokens = bool((self.q_lengths == 1).all())
        # No sequence has keys before (or without) its queries.
        self.whole = bool((self.q_lengths == self.k_lengths).all())
        self._tables: dict[tuple[int, int], WorkTables] = {}

    def offsets(self) -> tuple[torch.Tensor, torch.Tensor]:
        """(q_offsets, k_offsets) for a launch on the current stream."""
        _keep(self._stream, self.q_offsets)
        return self.q_offsets, self.k_offsets

    def tables(self, group: int, kv_heads: int) -> WorkTables:
        """The work tables for `kv_heads` key heads of `group` query heads
        each, built (and copied to the device) on first use; build them
        before capturing a CUDA graph."""
        tables = self._tables.get((group, kv_heads))
        if tables is None:
            sms = 148
            if self.device.type == 'cuda':
                if torch.cuda.is_current_stream_capturing():
                    raise RuntimeError(
                        'the work tables of this pack do not exist yet: call '
                        f'tables({group}, {kv_heads}) or run once before the '
                        'capture')
                sms = torch.cuda.get_device_properties(
                    self.device).multi_processor_count
            whole, query, key, n = work_items(self.q_lengths, self.k_lengths,
                                              group)
            forward, joins, n_parts = split_items(whole, kv_heads, sms)
            turns = deal_items(key[:, 6], kv_heads, sms)
            order = np.full((-(-turns.size // ITEM_FIELDS), ITEM_FIELDS), -1)
            order.flat[:turns.size] = turns.flat
            parts = forward, joins, query, key, order
            flat = _to_device(np.concatenate(parts), self.device)
            parts = flat.split([len(t) for t in parts])
            at = [t.data_ptr() if len(t) else 0 for t in parts]
            tables = WorkTables(
                *parts, n, n_parts,
                (at[0], len(forward), at[1], len(joins), n_parts),
                (at[2], len(query), at[3], len(key), at[4], sms, len(turns),
                 n),
                _stream(self.device))
            self._tables[group, kv_heads] = tables
        else:
            _keep(tables.stream, tables.forward)
        return tables


def _stream(device: torch.device) -> int:
    return (torch.cuda.current_stream(device).cuda_stream
            if device.type == 'cuda' else 0)


def _keep(stream: int, t: torch.Tensor) -> None:
    """Keeps the memory of a tensor made on `stream` until the work queued on
    the current stream is done, should its owner drop it before."""
    if not t.is_cuda or torch._C._cuda_getCurrentRawStream(
            t.device.index) == stream:
        return
    if not torch.cuda.is_current_stream_capturing():
        t.record_stream(torch.cuda.current_stream(t.device))


def _lengths(values: Sequence[int], name: str) -> np.ndarray:
    if isinstance(values, torch.Tensor):
        if values.is_cuda:
            raise ValueError(f'{name} must be host integers (a CUDA tensor '
                             'would have to be read back)')
        values = values.numpy()
    out = np.asarray(values)
    if out.ndim != 1 or out.size == 0 or out.dtype.kind not in 'iu':
        raise ValueError(f'{name} must be a non-empty list of integers')
    out = out.astype(np.int64)
    if (out < 0).any():
        raise ValueError(f'{name} must not be negative')
    if (out >= 2 ** 31).any():
        raise ValueError(f'{name} must be below 2^31')
    out.setflags(write=False)  # offsets and tables are made from them
    return out


def _to_device(values: np.ndarray, device: torch.device) -> torch.Tensor:
    host = torch.from_numpy(np.ascontiguousarray(values, dtype=np.int32))
    return host.to(device)


def _expand(counts: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """(sequence, index inside it) of each of counts.sum() elements."""
    seq = np.repeat(np.arange(counts.size), counts)
    first = np.cumsum(counts) - counts
    return seq, np.arange(seq.size) - first[seq]


def work_items(q_lengths: np.ndarray, k_lengths: np.ndarray, group: int
               ) -> tuple[np.ndarray, np.ndarray, np.ndarray, int]:
    """Work items of the attention kernels (int64 [n, 8] arrays; see
    csrc/causal.cuh for the fields), longest first, and the number of query
    tiles. A query tile is `128 // group` tokens of one sequence with the
    `group` heads of one key head."""
    if not 1 <= group <= TILE:
        raise ValueError('1 to 128 query heads may share a key head: '
                         f'{group}')
    tokens = TILE // group
    q0 = np.cumsum(q_lengths) - q_lengths
    k0 = np.cumsum(k_lengths) - k_lengths
    before = k_lengths - q_lengths  # keys before the first query
    tiles = -(-q_lengths // tokens)
    tile_base = np.cumsum(tiles) - tiles

    def query_items(per_item: int) -> np.ndarray:
        span = per_item * tokens
        seq, i = _expand(-(-q_lengths // span))
        t0 = i * span
        n = np.minimum(span, q_lengths[seq] - t0)
        kpos = before[seq] + t0
        blocks = -(-np.clip(kpos + n, 0, k_lengths[seq]) // TILE)
        items = np.stack([q0[seq] + t0, n, k0[seq], kpos, k_lengths[seq],
                          blocks, tile_base[seq] + i * per_item,
                          np.zeros_like(n)], axis=1)
        return items[np.argsort(-blocks, kind='stable')]

    seq, i = _expand(-(-k_lengths // TILE))
    j0 = i * TILE
    # Token t of the sequence sees key j0 + r if t >= shift + r.
    shift = j0 - before[seq]
    first = np.maximum(shift, 0) // tokens
    blocks = np.maximum(tiles[seq] - first, 0)
    key = np.stack([k0[seq] + j0, np.minimum(TILE, k_lengths[seq] - j0),
                    q0[seq], q_lengths[seq], shift, first, blocks,
                    tile_base[seq]], axis=1)
    key = key[np.argsort(-blocks, kind='stable')]
    return query_items(2), query_items(1), key, int(tiles.sum())


# With more turns than this dealing back and forth is even enough.
MOST_TURNS = 16


def deal_items(blocks: np.ndarray, kv_heads: int, sms: int) -> np.ndarray:
    """Which key gradient item each processor takes at its n-th turn: int64
    [turns, sms], -1 behind its last; no turns where back and forth, as the
    kernel deals by itself, does as well. Items cannot be cut (a key tile's
    sums stay in one processor), so that a few turns leave some processors an
    item more than others: the items, longest first and half as many as
    processors at a time, go to those that have least. Four samples of 1,000
    to 8,192 tokens, 4 key heads: 348 tiles for the busiest of 148 in place of
    390, of 341 on average, and 725 us in place of 815; from 16 turns on it is
    under 2 %. (0.06 to 0.2 ms on the host: one sequence of 35,840 tokens, 6
    key heads.) The other kernels' items are short enough
    back and forth (query gradients the same, the forward up to 6 % faster if
    dealt, for twice the time on the host)."""
    items = len(blocks) * kv_heads
    if not sms < items <= MOST_TURNS * sms:
        return np.zeros((0, sms), np.int64)
    cost = np.repeat(blocks + ITEM_COST, kv_heads)
    load = np.zeros(sms)
    taken = np.zeros(sms, np.int64)
    out = np.full((items, sms), -1, np.int64)
    order = np.argsort(-cost, kind='stable')
    step = max(1, sms // 2)
    for at in range(0, items, step):
        some = order[at:at + step]
        least = np.argsort(load, kind='stable')[:some.size]
        out[taken[least], least] = some
        load[least] += cost[some]
        taken[least] += 1
    return out[:taken.max()]


# What an item costs beside its key tiles, in key tiles: its loads and its
# epilogue; for a part, which leaves fp32 rows for a second kernel; and that
# kernel.
ITEM_COST, PART_COST, JOIN_COST = 2.0, 3.0, 3.0
# No part is shorter (a row of it is written and read again in fp32).
SHORTEST_PART = 4


def split_items(whole: np.ndarray, kv_heads: int, sms: int
                ) -> tuple[np.ndarray, np.ndarray, int]:
    """Forward items, possibly cut along the keys: (items, joins, parts).

    With few items (a chunk behind a long context) whole ones leave
    processors idle or give some of them one item more than others. Items
    longer than a limit are cut into equal parts, and the limit is the one (or
    none) for which the busiest processor's estimated cost is least, dealt
    back and forth as the kernel does. With many items nothing is gained and
    nothing tried."""
    items = whole.copy()
    items[:, 6], items[:, 7] = 0, -1  # first key tile, part
    none = np.zeros((0, ITEM_FIELDS), np.int64)
    blocks = whole[:, 5]
    total = int(blocks.sum()) * kv_heads
    longest = int(blocks.max(initial=0))
    if (longest < 2 * SHORTEST_PART
            or (len(whole) * kv_heads >= 8 * sms
                and 2 * longest * sms <= total)):
        return items, none, 0

    def pieces(limit: int) -> np.ndarray:
        return np.maximum(1, -(-blocks // limit))

    def busiest(count: np.ndarray) -> float:
        cost = np.where(count > 1, blocks / count + PART_COST,
                        blocks + ITEM_COST)
        cost = np.sort(np.repeat(cost, count * kv_heads))[::-1]
        rounds = -(-cost.size // sms)
        dealt = np.zeros(rounds * sms)
        dealt[:cost.size] = cost
        dealt = dealt.reshape(rounds, sms)
        dealt[1::2] = dealt[1::2, ::-1]
        return dealt.sum(0).max() + (JOIN_COST if (count > 1).any() else 0)

    best, best_cost = None, busiest(np.ones_like(blocks))
    for ways in (2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64, 96, 148):
        limit = -(-longest // ways)
        if limit < SHORTEST_PART:
            break
        count = pieces(limit)
        cost = busiest(count)
        if cost < best_cost:
            best, best_cost = count, cost
    if best is None:
        return items, none, 0
    src, i = _expand(best)
    out = items[src]
    n = best[src]
    first = blocks[src] * i // n
    out[:, 5] = blocks[src] * (i + 1) // n - first
    out[:, 6] = first
    cut = n > 1
    out[cut, 7] = np.arange(int(cut.sum()))
    owners = np.nonzero(best > 1)[0]
    joins = np.zeros((owners.size, ITEM_FIELDS), np.int64)
    joins[:, 0], joins[:, 1] = whole[owners, 0], whole[owners, 1]
    joins[:, 2] = np.cumsum(best[owners]) - best[owners]
    joins[:, 3] = best[owners]
    return out[np.argsort(-out[:, 5], kind='stable')], joins, int(cut.sum())
