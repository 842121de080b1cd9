"""Device-resident block pool with the reference BlockManager's interface.

The reference keeps the free list and every sequence's block list in Python
(core/block_manager.py:19-68) and rebuilds a padded int32 block table from
that dict on every step with host loops and ``.item()`` calls
(transformer/model.py:126-152), next to host-built step metadata
(core/model_runner.py:66-107).  Here the free list, the per-sequence lists and
the padded table live in device memory:

* ``DeviceBlockManager.allocate`` / ``release_blocks`` / ``num_free_blocks`` /
  ``can_allocate`` keep the reference's names, arguments and statuses.  The
  statuses are decided on the host, which tracks how many blocks are free and
  which sequences hold blocks (the decisions the reference makes,
  core/block_manager.py:32-33,49-50); the block ids themselves exist only on
  the device.  Calls are queued and applied in order by one launch at
  ``flush()`` (``block_pool_apply_sole``, or ``_shared`` where a call meets
  shared blocks), so a scheduler step costs one launch and
  one small host-to-device copy, whatever the number of calls.
* ``step_inputs(...)`` builds a step's attention inputs on the device
  (``block_pool_step``): the zero-padded block table and ``num_blocks_per_seq``
  of the scheduled sequences, and each query token's position and row.

``AllocResult.block_ids`` is a device tensor (the ids the call appended, valid
once the queued operations have been flushed) rather than a host list.

Sequences may share blocks (the reference's never do).  Every block counts its
holders (``ref_count``); a block is written only while one sequence holds it:

* ``fork(parent, child, num_tokens)`` gives the child the parent's first tokens:
  the full blocks are shared, a partly filled last one is copied in every layer
  of the caches named by ``attach_caches``;
* ``fork_beams`` / ``allocate_beams`` / ``reorder_beams`` / ``release_beams``
  keep the beams of a beam search, whose parents only the device knows, and
  ``recount`` learns which blocks its reorderings have freed;
* ``compact`` moves the blocks in use to the lowest ids.
"""
from __future__ import annotations

import ctypes
import enum
from dataclasses import dataclass
from typing import Optional, Sequence

import torch

from . import _lib, ops


class AllocStatus(enum.Enum):
    """core/block_manager.py:9-12."""

    SUCCESS = 0
    INSUFFICIENT_SPACE = 1
    FAILURE = 2


@dataclass
class AllocResult:
    status: AllocStatus
    block_ids: Optional[torch.Tensor]


class PaBlockPool(ctypes.Structure):
    """Mirror of pa_block_pool_t."""

    _fields_ = [("free_stack", ctypes.c_void_p), ("free_top", ctypes.c_void_p), ("table", ctypes.c_void_p),
                ("count", ctypes.c_void_p), ("table_stride", ctypes.c_int64), ("num_blocks", ctypes.c_int32),
                ("max_seqs", ctypes.c_int32), ("max_blocks_per_seq", ctypes.c_int32), ("_reserved", ctypes.c_int32)]


POOL_ALLOCATE, POOL_RELEASE, POOL_FORK = 0, 1, 2


class _Prefix:
    """Columns of a block table that sequences share: ``n`` blocks after those of ``up``, held by ``holders``."""

    __slots__ = ("n", "holders", "up")

    def __init__(self, n: int, holders: int, up: Optional["_Prefix"]):
        self.n, self.holders, self.up = n, holders, up


def _best_cuts(widths: Sequence[int]) -> list[int]:
    """Where the runs begin into which ``len(widths) + 1`` neighbours are cut, ``widths[i]`` columns common to i and i + 1.

    A run's columns are the fewest between its neighbours, and it saves them for all members but one.  With best[j] the most that the
    first j save, best[j] = max(best[j - 1], best[i] + (j - 1 - i) w over the runs i..j-1 whose neighbours all share w or
    more): for each w the largest best[i] - i w of the places i where such a run may have begun.
    """
    levels = sorted(set(widths))
    if len(levels) > 16:  # some of them: still runs of what their members share, perhaps not the best
        levels = [levels[i * (len(levels) - 1) // 15] for i in range(16)]
    lead = [(0, 0)] * len(levels)  # of each level: best[i] - i w, i
    best, begin = [0, 0], [0, 0]   # of the first j: what they save, where their last run begins
    for j in range(2, len(widths) + 2):
        most, first = best[j - 1], j - 1
        for k, w in enumerate(levels):
            if widths[j - 2] < w:  # a run over these two ends
                lead[k] = (best[j - 1] - (j - 1) * w, j - 1)
                continue
            value = lead[k][0] + (j - 1) * w
            if value > most:
                most, first = value, lead[k][1]
            if best[j - 1] - (j - 1) * w > lead[k][0]:
                lead[k] = (best[j - 1] - (j - 1) * w, j - 1)
        best.append(most)
        begin.append(first)
    cuts, j = [], len(widths) + 1
    while j > 0:
        cuts.append(begin[j])
        j = begin[j]
    return cuts[::-1]


class BlockLedger:
    """Host half of the pool: the decisions the reference's BlockManager makes, without the ids.

    Tracks how many blocks are free, how many each sequence holds and which
    table row (slot) it uses, decides every call's status exactly as
    core/block_manager.py:29-57 does, and queues the (kind, slot, n)
    operations the device applies in the same order.
    """

    def __init__(self, num_blocks: int, max_seqs: int, max_blocks_per_seq: int):
        self.num_blocks = int(num_blocks)
        self.max_seqs = int(max_seqs)
        self.max_blocks_per_seq = int(max_blocks_per_seq)
        self.free = self.num_blocks
        self.blocks: dict[int, int] = {}      # seq_id -> blocks held
        self.slot: dict[int, int] = {}        # seq_id -> table row
        self.free_slots = list(range(self.max_seqs - 1, -1, -1))
        self.ops: list[tuple[int, ...]] = []
        self.counted = False                  # a queued operation meets blocks that several sequences hold or held
        self.prefix: dict[int, _Prefix] = {}  # seq_id -> its last shared columns
        self.beams: dict[int, tuple[int, ...]] = {}  # first beam -> all beams of a search
        self.member: dict[int, int] = {}      # beam -> first beam
        self.regained: dict[int, int] = {}    # first beam -> blocks that reorderings freed, as last counted
        self.moved: set = set()               # first beams of searches whose rows the device has permuted

    def row(self, seq_id: int) -> int:
        """The table row of ``seq_id``.  A reordering permutes a search's rows on the device: its beams have none here."""
        if self.moved and self.member.get(seq_id, seq_id) in self.moved:
            raise ValueError(f"sequence {seq_id} is a beam of {self.member[seq_id]}, whose beams were reordered: only the "
                             "device knows their rows (reorder_beams returned them)")
        return self.slot[seq_id]

    def beams_moved(self, seq_ids: Optional[Sequence[int]] = None) -> None:
        """The beams of these searches were reordered (None: of which ones only the device knows)."""
        self.moved.update(self.beams if seq_ids is None else [s for s in seq_ids if s in self.beams])

    def _alone(self, seq_id: int) -> None:
        if seq_id in self.member:
            raise ValueError(f"sequence {seq_id} is a beam of {self.member[seq_id]}: beams are extended and released together")

    def none_is_a_beam(self, seq_ids: Sequence[int]) -> None:
        if self.member:
            for s in seq_ids:
                self._alone(s if s in self.slot else int(s))

    def allocate(self, seq_id: int, num_blocks: int) -> tuple[AllocStatus, int, int]:
        """Returns (status, slot, first new column); queues the operation on success."""
        if self.member:
            self._alone(seq_id)
        return self._allocate(seq_id, num_blocks)

    def _allocate(self, seq_id: int, num_blocks: int) -> tuple[AllocStatus, int, int]:
        num_blocks = int(num_blocks)
        if num_blocks < 0:
            raise ValueError("num_blocks must be >= 0")
        if self.free < num_blocks:
            return AllocStatus.INSUFFICIENT_SPACE, -1, 0
        held = self.blocks.get(seq_id)
        base = held or 0
        if base + num_blocks > self.max_blocks_per_seq:
            raise ValueError(f"sequence {seq_id} would hold {base + num_blocks} blocks, more than "
                             f"max_blocks_per_seq={self.max_blocks_per_seq}")
        if held is None:
            if not self.free_slots:
                raise RuntimeError(f"more than max_seqs={self.max_seqs} sequences hold blocks")
            self.slot[seq_id] = self.free_slots.pop()
        slot = self.slot[seq_id]
        self.ops.append((POOL_ALLOCATE, slot, num_blocks))
        self.blocks[seq_id] = base + num_blocks
        self.free -= num_blocks
        return AllocStatus.SUCCESS, slot, base

    def release(self, seq_id: int) -> AllocStatus:
        if self.member:
            self._alone(seq_id)
        return self._release(seq_id)

    def _release(self, seq_id: int) -> AllocStatus:
        if seq_id not in self.blocks:
            return AllocStatus.FAILURE
        slot = self.slot.pop(seq_id)
        self.ops.append((POOL_RELEASE, slot, 0))
        self.free += self.blocks.pop(seq_id)
        node = self.prefix.pop(seq_id, None) if self.prefix else None
        while node is not None:  # columns that others hold are not free
            node.holders -= 1
            if node.holders:
                self.free -= node.n
                self.counted = True
            node = node.up
        self.free_slots.append(slot)
        return AllocStatus.SUCCESS

    def _shared(self, seq_id: int, columns: int) -> Optional[_Prefix]:
        """The node that ends at ``columns`` columns of ``seq_id``, split off where there is none."""
        if columns == 0:
            return None
        node = self.prefix.get(seq_id)
        end, n = 0, node
        while n is not None:
            end += n.n
            n = n.up
        if columns > end:  # private columns become shareable
            node = self.prefix[seq_id] = _Prefix(columns - end, 1, node)
            return node
        while end - node.n >= columns:
            end -= node.n
            node = node.up
        if end > columns:
            node.up = _Prefix(columns - (end - node.n), node.holders, node.up)
            node.n = end - columns
            node = node.up
        return node

    def shared_columns(self, seq_id: int) -> int:
        """The first columns of ``seq_id`` that other sequences hold too."""
        n, node = 0, self.prefix.get(seq_id)
        while node is not None:
            if node.holders > 1:
                n += node.n
            node = node.up
        return n

    def shared_runs(self, seq_ids: Sequence[int]) -> tuple[list[int], list[int]]:
        """Neighbours in ``seq_ids`` whose first columns are the same: (where each run begins, and the end; its columns).

        A run's columns are read once instead of once per member; the order is cut so that this saves the most columns
        (``_best_cuts``; exactly so for up to 16 different widths between neighbours that share anything).
        """
        starts: list[int] = []
        columns: list[int] = []
        begin = 0                 # of the neighbours that share something
        widths: list[int] = []    # shared by each of them and the one before
        last: list[_Prefix] = []

        def close(end: int) -> None:
            if not widths:
                starts.append(begin)
                columns.append(0)
                return
            cuts = [0] if min(widths) == max(widths) else _best_cuts(widths)
            for i, j in zip(cuts, [*cuts[1:], end - begin]):
                starts.append(begin + i)
                columns.append(min(widths[i:j - 1], default=0))

        for i, s in enumerate(seq_ids):
            path, node = [], self.prefix.get(s)
            while node is not None:
                path.append(node)
                node = node.up
            path.reverse()
            if i:
                width = 0
                for x, y in zip(last, path):
                    if x is not y:
                        break
                    width += x.n
                if width:
                    widths.append(width)
                else:
                    close(i)
                    begin, widths = i, []
            last = path
        if seq_ids:
            close(len(seq_ids))
        return [*starts, len(seq_ids)], columns

    def fork(self, parent_id: int, child_id: int, num_tokens: int, block_size: int) -> tuple[AllocStatus, int]:
        """The child gets the parent's first tokens: (status, the child's slot); queues the operation on success."""
        self._alone(parent_id)
        return self._fork(parent_id, child_id, num_tokens, block_size)

    def _fork(self, parent_id: int, child_id: int, num_tokens: int, block_size: int) -> tuple[AllocStatus, int]:
        num_tokens = int(num_tokens)
        if num_tokens < 0:
            raise ValueError("num_tokens must be >= 0")
        if parent_id not in self.blocks or child_id in self.blocks:
            return AllocStatus.FAILURE, -1
        full, tail = divmod(num_tokens, block_size)
        if full + (tail > 0) > self.blocks[parent_id]:
            raise ValueError(f"sequence {parent_id} holds {self.blocks[parent_id]} blocks, fewer than {num_tokens} tokens")
        if tail and self.free < 1:
            return AllocStatus.INSUFFICIENT_SPACE, -1
        if not self.free_slots:
            raise RuntimeError(f"more than max_seqs={self.max_seqs} sequences hold blocks")
        slot = self.slot[child_id] = self.free_slots.pop()
        self.ops.append((POOL_FORK, slot, num_tokens, self.slot[parent_id]))
        self.counted = True
        self.blocks[child_id] = full + (tail > 0)
        self.free -= tail > 0
        node = self._shared(parent_id, full)
        if node is not None:
            self.prefix[child_id] = node
        while node is not None:
            node.holders += 1
            node = node.up
        return AllocStatus.SUCCESS, slot

    def fork_beams(self, seq_id: int, beam_ids: Sequence[int], num_tokens: int, block_size: int) -> AllocStatus:
        """``seq_id`` and its new forks ``beam_ids`` become the beams of one search; all or none are made."""
        self._alone(seq_id)
        beams = (seq_id, *beam_ids)
        if len(set(beams)) < len(beams):
            raise ValueError("beam ids must differ")
        if seq_id not in self.blocks or any(b in self.blocks for b in beam_ids):
            return AllocStatus.FAILURE
        num_tokens = int(num_tokens)
        if self.blocks[seq_id] != -(-num_tokens // block_size):
            raise ValueError(f"sequence {seq_id} holds {self.blocks[seq_id]} blocks: beams start with the "
                             f"{-(-num_tokens // block_size)} that {num_tokens} tokens fill")
        if num_tokens % block_size and self.shared_columns(seq_id) > num_tokens // block_size:
            raise ValueError(f"sequence {seq_id} ends inside a block that another sequence holds: its next token cannot be "
                             f"written there (fork it at {num_tokens} tokens first)")
        if len(self.free_slots) < len(beam_ids):
            raise RuntimeError(f"more than max_seqs={self.max_seqs} sequences hold blocks")
        if self.free < (len(beam_ids) if num_tokens % block_size else 0):
            return AllocStatus.INSUFFICIENT_SPACE
        for b in beam_ids:
            self._fork(seq_id, b, num_tokens, block_size)
        self.beams[seq_id] = beams
        self.member.update((b, seq_id) for b in beams)
        return AllocStatus.SUCCESS

    def dissolve_beams(self, seq_id: int) -> None:
        """Undo fork_beams before any reordering: the forks are released, ``seq_id`` keeps its blocks."""
        beams = self.beams.pop(seq_id)
        self.moved.discard(seq_id)
        for b in beams:
            del self.member[b]
        self.counted = True
        self.free -= self.regained.pop(seq_id, 0)
        for b in beams[1:]:
            self._release(b)

    def allocate_beams(self, seq_id: int, num_blocks: int) -> AllocStatus:
        beams = self.beams[seq_id]
        if self.free < num_blocks * len(beams):
            return AllocStatus.INSUFFICIENT_SPACE
        for b in beams:
            self._allocate(b, num_blocks)
        return AllocStatus.SUCCESS

    def private_columns(self, seq_id: int) -> tuple[int, int]:
        """The columns [first, last) in which each beam of the search began with blocks of its own."""
        first, node = 0, self.prefix.get(self.beams[seq_id][-1])
        while node is not None:
            first, node = first + node.n, node.up
        return first, self.blocks[seq_id]

    def count_beams(self, seq_id: int, held: int) -> None:
        """The search's beams hold ``held`` different blocks in their private columns: the others count as free.

        Later reorderings only free more of them, and an allocation adds as many blocks here as on the device.
        """
        first, last = self.private_columns(seq_id)
        freed = len(self.beams[seq_id]) * (last - first) - held
        self.free += freed - self.regained.get(seq_id, 0)
        self.regained[seq_id] = freed

    def release_beams(self, seq_id: int) -> AllocStatus:
        # Reordering keeps each column's blocks within those that the beams
        # held before, so the device never uses more than is counted here, and
        # the counts agree again when all beams are gone.
        if seq_id not in self.beams:
            return AllocStatus.FAILURE
        self.moved.discard(seq_id)
        self.counted = True  # a reordering may have given one block to several
        self.free -= self.regained.pop(seq_id, 0)
        for b in self.beams.pop(seq_id):
            del self.member[b]
            self._release(b)
        return AllocStatus.SUCCESS

    def take_ops(self) -> list[tuple[int, ...]]:
        ops, self.ops, self.counted = self.ops, [], False
        return ops


class DeviceBlockManager:
    """The paged pool's bookkeeping in device memory (see the module docstring).

    ``max_seqs`` sequences may hold blocks at once, each at most
    ``max_blocks_per_seq``; both size the device table
    ``[max_seqs, max_blocks_per_seq]`` (int32).
    """

    def __init__(self, num_blocks: int, block_size: int, max_seqs: int, max_blocks_per_seq: int,
                 device: torch.device | str = "cuda"):
        self.num_blocks = int(num_blocks)
        self.block_size = int(block_size)
        self.max_seqs = int(max_seqs)
        self.max_blocks_per_seq = int(max_blocks_per_seq)
        self.device = torch.device(device)
        i32 = dict(dtype=torch.int32, device=self.device)
        self.free_stack = torch.empty(max(1, self.num_blocks), **i32)
        self.free_top = torch.empty(1, **i32)
        self.table = torch.empty(max(1, self.max_seqs), max(1, self.max_blocks_per_seq), **i32)
        self.count = torch.empty(max(1, self.max_seqs), **i32)
        self.ref_count = torch.empty(max(1, self.num_blocks), **i32)
        self.scratch = torch.empty(ops.pool_scratch_words(max(1, self.num_blocks)), **i32)
        self.status = torch.zeros(1, **i32)
        self._desc = PaBlockPool(self.free_stack.data_ptr(), self.free_top.data_ptr(), self.table.data_ptr(),
                                 self.count.data_ptr(), self.table.stride(0), self.num_blocks, self.max_seqs,
                                 self.max_blocks_per_seq, 0)
        self._share = _lib.PaBlockShare(self.ref_count.data_ptr(), self.scratch.data_ptr(), self.scratch.numel())
        self.ledger = BlockLedger(self.num_blocks, self.max_seqs, self.max_blocks_per_seq)
        self.caches: Optional[tuple] = None  # (K, V, K scales, V scales) of every layer
        self._cache_descs = None             # and their descriptors
        self._copies: set = set()            # sequences whose queued forks copy a page
        self._results: Optional[torch.Tensor] = None
        lib = _lib.load()
        with torch.cuda.device(self.device):
            _lib.check("block_pool_init_shared", lib.block_pool_init_shared(
                ctypes.byref(self._desc), ctypes.byref(self._share), self._stream()))

    def _stream(self) -> int:
        return torch.cuda.current_stream(self.device).cuda_stream

    # ---- the reference interface (core/block_manager.py) --------------------
    def allocate(self, seq_id: int, num_blocks: int) -> AllocResult:
        """core/block_manager.py:29-44: take ``num_blocks`` ids off the free list for ``seq_id``."""
        st, slot, base = self.ledger.allocate(seq_id, num_blocks)
        if st is not AllocStatus.SUCCESS:
            return AllocResult(st, None)
        return AllocResult(st, self.table[slot, base:base + int(num_blocks)])

    def release_blocks(self, seq_id: int) -> AllocStatus:
        """core/block_manager.py:47-57: return ``seq_id``'s blocks (that no other sequence holds) to the free list."""
        if self._copies:
            self._copies_first()
        return self.ledger.release(seq_id)

    def num_free_blocks(self) -> int:
        return self.ledger.free

    def can_allocate(self, num_blocks: int) -> bool:
        return self.ledger.free >= num_blocks

    def recount(self) -> int:
        """Count as free what reorderings of beams have freed so far; returns ``num_free_blocks()``.

        Reads the beams' rows (synchronises).  Without it a search's blocks count as its beams held them at their
        widest, until they are released.
        """
        searches = list(self.ledger.beams)
        if searches:
            self.flush()
            rows = [self.ledger.slot[b] for s in searches for b in self.ledger.beams[s]]
            table = self.table[torch.tensor(rows).to(self.device)].cpu()
            for s in searches:
                mine, table = table.split([len(self.ledger.beams[s]), len(table) - len(self.ledger.beams[s])])
                first, last = self.ledger.private_columns(s)
                self.ledger.count_beams(s, mine[:, first:last].unique().numel())
        return self.ledger.free

    # ---- shared blocks ------------------------------------------------------
    def attach_caches(self, k_cache: ops.Caches, v_cache: ops.Caches, k_scale: Optional[ops.Caches] = None,
                      v_scale: Optional[ops.Caches] = None) -> None:
        """Name the pools whose pages this manager hands out: one layer's tensors or lists of every layer's.

        Forks, beams and compaction move pages in all of them.
        """
        descs = ops.layer_descs(k_cache, v_cache, k_scale, v_scale)
        if descs[0].block_size != self.block_size or descs[0].num_blocks < self.num_blocks:
            raise ValueError(f"the caches hold {descs[0].num_blocks} blocks of {descs[0].block_size} tokens, "
                             f"the manager hands out {self.num_blocks} of {self.block_size}")
        # what the page copies cannot move is refused here, not by the flush that has already applied a fork
        _lib.check("attach_caches", _lib.load().kv_copy_blocks(descs, len(descs), None, None, None, 0, None, None))
        lists = [list(ops._layers(c)) for c in (k_cache, v_cache, k_scale, v_scale)]
        if lists[0][0].device.type != "cuda" or lists[0][0].device != self.free_top.device:
            raise ValueError(f"the caches are on {lists[0][0].device}, the pool on {self.free_top.device}")
        self.caches, self._cache_descs = tuple(lists), descs

    @property
    def state(self) -> ops.PoolState:
        """The pool's device arrays, for ``ops.reorder_beams`` and ``ops.compact_blocks``.

        The manager does not see what those do: use its own methods where it goes on handing out blocks.
        """
        return ops.PoolState(self.free_stack, self.free_top, self.table[:self.max_seqs, :self.max_blocks_per_seq],
                             self.count[:self.max_seqs], self.ref_count[:self.num_blocks], self.scratch)

    def _need_caches(self):
        if self._cache_descs is None:
            raise ValueError("attach_caches() names the pools whose pages are to be moved")
        return self._cache_descs

    def _checked(self, fn: str, status: Optional[torch.Tensor] = None) -> None:
        if ops._CHECK:
            ops._raise_status(fn, self.status if status is None else status)

    def _copies_first(self) -> None:
        """A released block may be handed out again: the copies queued so far read their pages before that."""
        if self._copies:
            self.flush()

    def _before_fork(self, parent_id: int, num_tokens: int) -> None:
        """A fork that copies needs the caches, and its parent's own copy to be made: one launch's copies act at once."""
        if num_tokens % self.block_size:
            self._need_caches()
            if parent_id in self._copies:
                self.flush()

    def fork(self, parent_id: int, child_id: int, num_tokens: int) -> AllocResult:
        """Let ``child_id`` start with the first ``num_tokens`` tokens of ``parent_id``, sharing its full blocks.

        A partly filled last block is copied when the queued calls are flushed, so the parent's tokens must be
        written by work on the same stream before that.
        """
        self._before_fork(parent_id, num_tokens)
        st, slot = self.ledger.fork(parent_id, child_id, num_tokens, self.block_size)
        if st is not AllocStatus.SUCCESS:
            return AllocResult(st, None)
        if num_tokens % self.block_size:
            self._copies.add(child_id)
        return AllocResult(st, self.table[slot, :self.ledger.blocks[child_id]])

    def fork_beams(self, seq_id: int, beam_ids: Sequence[int], num_tokens: int) -> AllocStatus:
        """Make ``seq_id`` and new forks of it, ``beam_ids``, the beams of one search over ``num_tokens`` tokens."""
        self._before_fork(seq_id, num_tokens)
        st = self.ledger.fork_beams(seq_id, beam_ids, num_tokens, self.block_size)
        if st is AllocStatus.SUCCESS and num_tokens % self.block_size:
            self._copies.update(beam_ids)
        return st

    def allocate_beams(self, seq_id: int, num_blocks: int) -> AllocStatus:
        """``num_blocks`` new blocks for every beam of ``seq_id``'s search, or none."""
        return self.ledger.allocate_beams(seq_id, num_blocks)

    def dissolve_beams(self, seq_id: int) -> None:
        """Undo ``fork_beams`` before any reordering: the forks are released, ``seq_id`` is a plain sequence again."""
        self._copies_first()
        self.ledger.dissolve_beams(seq_id)

    def beam_slots(self, seq_ids: Sequence[int]) -> torch.Tensor:
        """The rows of the beams as ``fork_beams`` made them, int32 [len(seq_ids), num_beams] on the device."""
        rows = [[self.ledger.row(b) for b in self.ledger.beams[s]] for s in seq_ids]
        return torch.tensor(rows, dtype=torch.int32).to(self.device)

    def reorder_beams(self, slots: torch.Tensor, parents: torch.Tensor, num_tokens: torch.Tensor,
                      status: Optional[torch.Tensor] = None, seq_ids: Optional[Sequence[int]] = None) -> torch.Tensor:
        """Beam j of group g continues beam ``parents[g, j]``: returns the beams' rows afterwards (``ops.reorder_beams``).

        What does not fit is left as it is and reported in ``status`` (int32 [1] on the device; the manager's by default).

        Which blocks became free only the device knows; ``num_free_blocks`` counts them at ``recount`` or when the beams
        are released.  From now on only the returned rows name the beams: their ids are refused by ``slot_of``,
        ``beam_slots``, ``step_inputs`` and ``block_table`` until the search is released.  ``seq_ids`` names the searches
        whose rows ``slots`` holds; without it that counts for every search of the pool.  No host synchronisation: the call can be
        captured (with no queued calls).
        """
        descs = self._need_caches()
        self.flush()
        self.ledger.beams_moved(seq_ids)
        out = ops._reorder_call(self._desc, self._share, descs, self.free_top.device, ops._i32(slots), ops._i32(parents),
                                ops._i32(num_tokens), self.status if status is None else status)
        self._checked("reorder_beams", status)
        return out

    def release_beams(self, seq_id: int) -> AllocStatus:
        """Return the blocks of all beams of ``seq_id``'s search to the free list."""
        self._copies_first()
        return self.ledger.release_beams(seq_id)

    def compact(self, num_blocks: Optional[int] = None) -> torch.Tensor:
        """Move the blocks in use to the lowest ids; returns their number, int32 [1] on the device.

        With ``num_blocks`` the pool shrinks: ids at or above it are neither in use nor handed out any more, and
        their memory can be given up (``attach_caches`` with smaller pools).  Raises ValueError when more blocks
        are in use.
        """
        descs = self._need_caches()
        n = self.num_blocks if num_blocks is None else int(num_blocks)
        if n < self.num_blocks - self.ledger.free:
            self.recount()
        used = self.num_blocks - self.ledger.free
        if not used <= n <= self.num_blocks:
            raise ValueError(f"{used} of {self.num_blocks} blocks are in use: the pool cannot have {n}")
        self.flush()
        live = ops._compact_call(self._desc, self._share, descs, self.free_top.device, n, self.status)
        self._checked("compact")
        self.ledger.free -= self.num_blocks - n
        self.num_blocks = self.ledger.num_blocks = self._desc.num_blocks = n
        return live

    # ---- device side --------------------------------------------------------
    def flush(self, keep_results: bool = False) -> None:
        """Apply the queued allocate / release calls on the device, in order, in one launch.

        ``keep_results``: keep the per-call device statuses (``last_results``)
        for checking against the host's decisions.
        """
        sole = not self.ledger.counted
        ops_list = self.ledger.take_ops()
        if not ops_list:
            return
        n = len(ops_list)
        host = torch.tensor(ops_list if sole else [(*o, 0)[:4] for o in ops_list], dtype=torch.int32).pin_memory()
        dev_ops = host.to(self.device, non_blocking=True)
        res = torch.empty(n, dtype=torch.int32, device=self.device) if keep_results else None
        lib = _lib.load()
        if sole:
            with torch.cuda.device(self.device):
                _lib.check("block_pool_apply_sole", lib.block_pool_apply_sole(
                    ctypes.byref(self._desc), ctypes.byref(self._share), dev_ops.data_ptr(), n, ops._ptr(res), self._stream()))
            self._results = res
            return
        copies = torch.empty(3, n, dtype=torch.int32, device=self.device) if self._copies else None
        src, dst, slots = (None, None, None) if copies is None else copies
        with torch.cuda.device(self.device):
            _lib.check("block_pool_apply_shared", lib.block_pool_apply_shared(
                ctypes.byref(self._desc), ctypes.byref(self._share), dev_ops.data_ptr(), n, self.block_size,
                ops._ptr(res), ops._ptr(src), ops._ptr(dst), ops._ptr(slots), self._stream()))
        if copies is not None:
            ops._copy_call(self._need_caches(), self.free_top.device, src, dst, slots, self.status)
            self._copies.clear()
            self._checked("fork")
        self._results = res

    @property
    def last_results(self) -> Optional[torch.Tensor]:
        """Device statuses of the last ``flush(keep_results=True)``, one per queued call."""
        return self._results

    def slot_of(self, seq_id: int) -> int:
        """The table row of ``seq_id``; ValueError for a beam once ``reorder_beams`` has permuted the beams' rows."""
        return self.ledger.row(seq_id)

    def blocks_of(self, seq_id: int) -> int:
        return self.ledger.blocks.get(seq_id, 0)

    def step_inputs(self, sequence_ids: Sequence[int], q_lens: Sequence[int], kv_lens: Sequence[int],
                    bt_cols: Optional[int] = None) -> dict:
        """A step's attention inputs for ``sequence_ids`` (in the step's order), built on the device.

        Returns device int32 tensors: ``block_table`` [S, bt_cols] (zero
        padded; bt_cols defaults to the most blocks any of them holds, as
        transformer/model.py:145 sizes it), ``num_blocks_per_seq`` [S],
        ``q_len`` / ``kv_len`` [S], ``cu_seqlens`` [S + 1], and per query token
        ``positions`` [T] (``kv_len - q_len + i``) and ``token_seq`` [T] (its
        row of ``block_table``).  Queued allocate / release calls are flushed
        first.  One pinned host-to-device copy of the per-sequence values and
        one launch; no host synchronisation.
        """
        ids = [s if s in self.ledger.slot else int(s) for s in sequence_ids]
        slots = [self.ledger.row(s) for s in ids]
        self.flush()
        S = len(ids)
        if bt_cols is None:
            bt_cols = max((self.ledger.blocks[s] for s in ids), default=0)
        cu = [0]
        for q in q_lens:
            cu.append(cu[-1] + int(q))
        T = cu[-1]
        host = torch.tensor(slots + [int(q) for q in q_lens] + [int(k) for k in kv_lens] + cu,
                            dtype=torch.int32).pin_memory()
        dev = host.to(self.device, non_blocking=True)
        seq_slot, ql, kl, cus = dev[:S], dev[S:2 * S], dev[2 * S:3 * S], dev[3 * S:]
        i32 = dict(dtype=torch.int32, device=self.device)
        bt = torch.empty(S, bt_cols, **i32)
        nb = torch.empty(S, **i32)
        pos = torch.empty(T, **i32)
        tseq = torch.empty(T, **i32)
        lib = _lib.load()
        with torch.cuda.device(self.device):
            _lib.check("block_pool_step", lib.block_pool_step(
                ctypes.byref(self._desc), seq_slot.data_ptr(), ql.data_ptr(), kl.data_ptr(), cus.data_ptr(), S,
                bt.data_ptr() if bt.numel() else None, max(bt_cols, 1), bt_cols, nb.data_ptr(),
                pos.data_ptr() if T else None, tseq.data_ptr() if T else None, T, self.status.data_ptr(),
                self._stream()))
        return dict(block_table=bt, num_blocks_per_seq=nb, q_len=ql, kv_len=kl, cu_seqlens=cus, positions=pos,
                    token_seq=tseq)

    def shared_prefixes(self, sequence_ids: Sequence[int]) -> dict:
        """Which neighbours of ``sequence_ids`` share their first blocks, for ``ops.shared_prefix_attention``.

        Returns ``group_start`` [G + 1] and ``prefix_len`` [G] (tokens in whole blocks; 0 for a sequence that shares none
        with its neighbours), int32 on the device.  Forks of one sequence should stand side by side in the step's order.
        From the host's ledger: one host-to-device copy, nothing is read back.
        """
        starts, columns = self.shared_runs(sequence_ids)
        host = torch.tensor(starts + [c * self.block_size for c in columns], dtype=torch.int32).pin_memory()
        dev = host.to(self.device, non_blocking=True)
        return dict(group_start=dev[:len(starts)], prefix_len=dev[len(starts):])

    def shared_runs(self, sequence_ids: Sequence[int]) -> tuple[list[int], list[int]]:
        """``shared_prefixes`` as host lists: where each group begins (and the end), and the blocks that it shares."""
        ids = [s if s in self.ledger.slot else int(s) for s in sequence_ids]
        for s in ids:
            self.ledger.row(s)
        return self.ledger.shared_runs(ids)

    def step_rows(self, seq_slot: torch.Tensor, q_len: torch.Tensor, kv_len: torch.Tensor, cu_seqlens: torch.Tensor,
                  total_tokens: int, block_table: torch.Tensor, num_blocks: torch.Tensor, positions: torch.Tensor,
                  token_seq: torch.Tensor, status: Optional[torch.Tensor] = None) -> None:
        """``block_pool_step`` on caller-owned device tensors (no host copy, no allocation: capturable).

        ``seq_slot`` / ``q_len`` / ``kv_len`` int32 [S], ``cu_seqlens`` [S + 1]; writes ``block_table``
        [S, bt_cols] (row stride honoured), ``num_blocks`` [S], ``positions`` / ``token_seq`` [total_tokens].
        """
        S = seq_slot.numel()
        lib = _lib.load()
        with torch.cuda.device(self.device):
            _lib.check("block_pool_step", lib.block_pool_step(
                ctypes.byref(self._desc), seq_slot.data_ptr(), q_len.data_ptr(), kv_len.data_ptr(),
                cu_seqlens.data_ptr(), S, block_table.data_ptr(), block_table.stride(0), block_table.shape[1],
                num_blocks.data_ptr(), positions.data_ptr(), token_seq.data_ptr(), int(total_tokens),
                None if status is None else status.data_ptr(), self._stream()))

    @property
    def block_table(self) -> dict:
        """The per-sequence block lists as a host dict (reads the device: synchronises; for checks).

        ValueError while a search whose beams were reordered holds blocks: its rows have no names here.
        """
        rows = {sid: self.ledger.row(sid) for sid in self.ledger.slot}
        self.flush()
        tab = self.table.cpu()
        return {sid: tab[slot, :self.ledger.blocks[sid]].tolist() for sid, slot in rows.items()}

    def free_list(self) -> list[int]:
        """The free list bottom to top, as the reference's ``st`` (reads the device: synchronises)."""
        self.flush()
        top = int(self.free_top.item())
        return self.free_stack[:top].tolist()
