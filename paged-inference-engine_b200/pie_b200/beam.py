"""Beam search over the paged cache, with all decisions on the device.

``BeamSearch`` keeps K beams of each of B sequences as rows of a
``DeviceBlockManager``.  A step is: ``step_inputs()`` (a new block for beams
whose last one is full, the beams' block tables, positions and lengths), the
caller's model over them (``write_kv`` and ``paged_attention`` as in any
decode step), and ``advance(logits)``: ``ops.beam_select`` picks the best
continuations (of logits that ``ops.adjust_logits`` has been over, where the
search has penalties, a bias or a mask) and ``reorder_beams`` makes the cache follow them: beams share
their parents' full blocks, partly filled ones are copied.  ``step_inputs()`` also says
which blocks of the prompt a sequence's beams share, for
``shared_prefix_attention``.  Nothing is read
back before ``finish()``, unless the pool seems to have no block left for a
step.

The reference decodes one sampled continuation per sequence
(core/model_runner.py:28-159) and has no beams.
"""
from __future__ import annotations

from typing import Optional, Sequence

import torch

from . import ops
from .block_pool import AllocStatus, DeviceBlockManager

MAX_BEAMS = 32  # of ops.beam_select and ops.reorder_beams


class BeamSearch:
    """``num_beams`` beams of each of ``seq_ids``, which hold ``num_tokens[i]`` prompt tokens in the cache.

    ``logits`` [B, V] are those of each prompt's last token.  The pool knows the search as the sequences ``beam_id(seq_id,
    k)``, but which row beam k has only the device knows (``slots``, in the order of ``tokens``): the pool refuses these
    ids until ``finish``.  The sequences must hold exactly the blocks that their tokens fill.  A beam that emits ``eos_id`` is finished: it keeps
    its score and competes with the others until ``finish``.

    ``repetition_penalty``, ``presence_penalty`` and ``frequency_penalty`` (numbers) and ``bias`` ([V] or [B, V], float32)
    act on every step's logits as in ``ops.adjust_logits``, each beam with its own line of tokens behind
    ``prompt_tokens[i]`` (the prompts' token ids, ``num_tokens[i]`` of them; needed for penalties).  ``mask`` is that of the
    first token, one per sequence or one for all; ``advance`` takes the later ones.
    """

    def __init__(self, pool: DeviceBlockManager, seq_ids: Sequence[int], num_tokens: Sequence[int], logits: torch.Tensor,
                 num_beams: int, eos_id: int, max_new_tokens: int, *,
                 prompt_tokens: Optional[Sequence[Sequence[int]]] = None, repetition_penalty: float = 1.0,
                 presence_penalty: float = 0.0, frequency_penalty: float = 0.0, bias: Optional[torch.Tensor] = None,
                 mask: Optional[torch.Tensor] = None):
        B, K = len(seq_ids), int(num_beams)
        if logits.dim() != 2 or logits.shape[0] != B or len(num_tokens) != B:
            raise ValueError(f"logits must be [{B}, vocab] and num_tokens hold {B} lengths")
        V = logits.shape[1]
        if not 1 <= K <= min(V, MAX_BEAMS):
            raise ValueError(f"num_beams {K} is outside 1..min(vocab, {MAX_BEAMS})")
        if not 0 <= eos_id < V:
            raise ValueError(f"eos_id {eos_id} is outside the vocabulary of {V}")
        if max_new_tokens < 1 or B < 1:
            raise ValueError("at least one sequence and one new token are needed")
        self.penalties = dict(repetition_penalty=float(repetition_penalty), presence_penalty=float(presence_penalty),
                              frequency_penalty=float(frequency_penalty))
        penalised = (repetition_penalty, presence_penalty, frequency_penalty) != (1, 0, 0)
        if penalised and prompt_tokens is None:
            raise ValueError("penalties need prompt_tokens")
        if prompt_tokens is not None and [len(t) for t in prompt_tokens] != [int(n) for n in num_tokens]:
            raise ValueError("prompt_tokens must hold num_tokens[i] token ids for each sequence")
        if bias is not None and tuple(bias.shape) not in ((V,), (1, V), (B, V)):
            raise ValueError(f"bias must be [{V}] or [{B}, {V}]")
        pool._need_caches()  # not only when the first partly filled block is copied
        self.pool, self.B, self.K, self.eos = pool, B, K, int(eos_id)
        self.seq_ids = [int(s) for s in seq_ids]
        self.host_tokens = [int(n) for n in num_tokens]
        dev = pool.free_top.device
        i32 = dict(dtype=torch.int32, device=dev)
        self.num_tokens = torch.tensor(self.host_tokens, dtype=torch.int32).to(dev)
        self.status = torch.zeros(1, **i32)  # of the search's own launches, read by finish
        self.max_new = int(max_new_tokens)
        self.history = torch.empty(2, self.max_new, B, K, **i32)  # tokens and parents of every step
        self.q_len = torch.ones(B * K, **i32)
        self.cu = torch.arange(B * K + 1, **i32)
        self.scores = torch.zeros(B, 1, device=dev)
        self.finished = torch.zeros(B, 1, dtype=torch.bool, device=dev)
        self.group_start = torch.arange(B + 1, **i32) * K
        self.prefix_len = self.num_tokens // pool.block_size * pool.block_size  # the beams' common blocks, for good
        self.bias = None if bias is None else bias.to(device=dev, dtype=torch.float32).reshape(-1, V)
        self.seen = self.prompt_len = None
        if penalised:  # the beams' lines: the prompt, then what was generated
            rows = torch.full((B, max(self.host_tokens) + self.max_new), -1, dtype=torch.int32)
            for i, t in enumerate(prompt_tokens):
                rows[i, :len(t)] = torch.as_tensor(t, dtype=torch.int32)
            self.seen, self.prompt_len = rows.to(dev).unsqueeze(1), self.num_tokens.clone()
        self.steps = 0
        self._room = self._ended = False
        self._choose(logits.unsqueeze(1), mask)  # before the forks: a refused call leaves the pool as it was
        made = []
        try:
            for s, n in zip(self.seq_ids, self.host_tokens):
                st = pool.fork_beams(s, [self.beam_id(s, k) for k in range(1, K)], n)
                if st is not AllocStatus.SUCCESS:
                    raise RuntimeError(f"no beams for sequence {s}: {st.name}")
                made.append(s)
        except Exception:
            for s in made:  # the prompts stay as they were
                pool.dissolve_beams(s)
            raise
        pool.flush()
        self.slots = pool.beam_slots(self.seq_ids)

    @staticmethod
    def beam_id(seq_id: int, k: int) -> object:
        """The id under which the pool counts the blocks of the search's k-th row: the sequence itself, or (sequence, k)."""
        return seq_id if k == 0 else (seq_id, k)

    @property
    def tokens(self) -> torch.Tensor:
        """The beams' newest tokens, int32 [B, K]: the next step's inputs."""
        return self.history[0, self.steps - 1]

    def _adjust(self, logits: torch.Tensor, mask: Optional[torch.Tensor]) -> torch.Tensor:
        if self.seen is None and self.bias is None and mask is None:
            return logits
        B, K, V = logits.shape
        rule: dict = {}
        if self.seen is not None:
            rule = dict(tokens=self.seen.view(B * K, -1), prompt_len=self.prompt_len.repeat_interleave(K),
                        num_tokens=(self.prompt_len + self.steps).repeat_interleave(K), **self.penalties)
        rows = torch.arange(B, dtype=torch.int32, device=logits.device).repeat_interleave(K)
        if self.bias is not None:
            rule.update(bias=self.bias, bias_row=rows if self.bias.shape[0] > 1 else None)
        if mask is not None:
            if mask.dim() == 3:
                if tuple(mask.shape[:2]) not in ((B, K), (B, 1), (1, 1)):
                    raise ValueError(f"mask must be [{B}, {K}, words], [{B}, words] or [words], got {tuple(mask.shape)}")
                mask = mask.reshape(-1, mask.shape[-1])
            rule.update(mask=mask, mask_row=rows if mask.dim() == 2 and mask.shape[0] == B > 1 and K > 1 else None)
        out = torch.empty(B * K, V, dtype=torch.float32, device=logits.device)
        return ops.adjust_logits(logits.reshape(B * K, V), out=out, **rule).view(B, K, V)

    def _choose(self, logits: torch.Tensor, mask: Optional[torch.Tensor] = None) -> torch.Tensor:
        logits = self._adjust(logits, mask)
        self.scores, tokens, parents = ops.beam_select(logits, self.scores, self.K, finished=self.finished, eos_id=self.eos)
        self.finished = self.finished.gather(1, parents.long()) | (tokens == self.eos)
        self.history[0, self.steps] = tokens
        self.history[1, self.steps] = parents
        if self.seen is not None:
            self.seen = self.seen.gather(1, parents.long().unsqueeze(2).expand(-1, -1, self.seen.shape[2]))
            at = (self.prompt_len + self.steps).long().view(-1, 1, 1).expand(-1, self.K, 1)
            self.seen.scatter_(2, at, tokens.unsqueeze(2))
        self.steps += 1
        return parents

    def step_inputs(self) -> dict:
        """Attention inputs of the next token of every beam (row ``b * K + k``), as ``DeviceBlockManager.step_inputs``.

        ``group_start`` and ``prefix_len`` beside them name the prompt's full blocks, which a sequence's beams share, for
        ``ops.shared_prefix_attention``.  The new token of a beam of sequence b goes to position ``num_tokens[b]`` and attends to one more key.  Reads
        nothing back, unless the pool counts too few free blocks: then it looks what the reorderings have freed.
        """
        if self._ended or self.steps >= self.max_new:
            raise RuntimeError(f"the search has ended or was made for {self.max_new} new tokens")
        pool, S = self.pool, self.B * self.K
        if not self._room:
            need = [s for s, n in zip(self.seq_ids, self.host_tokens) if pool.blocks_of(s) * pool.block_size <= n]
            if pool.num_free_blocks() < len(need) * self.K and pool.recount() < len(need) * self.K:
                raise RuntimeError(f"{len(need) * self.K} blocks are needed, {pool.num_free_blocks()} are free")
            if any(pool.blocks_of(s) >= pool.max_blocks_per_seq for s in need):
                raise RuntimeError(f"a beam would hold more than max_blocks_per_seq={pool.max_blocks_per_seq} blocks")
            for s in need:
                pool.allocate_beams(s, 1)
            self._room = True
        pool.flush()
        cols = max(-(-(n + 1) // pool.block_size) for n in self.host_tokens)
        i32 = dict(dtype=torch.int32, device=self.slots.device)
        out = dict(block_table=torch.empty(S, cols, **i32), num_blocks_per_seq=torch.empty(S, **i32), q_len=self.q_len,
                   kv_len=(self.num_tokens + 1).repeat_interleave(self.K), cu_seqlens=self.cu,
                   positions=torch.empty(S, **i32), token_seq=torch.empty(S, **i32), group_start=self.group_start,
                   prefix_len=self.prefix_len)
        pool.step_rows(self.slots.view(-1), self.q_len, out["kv_len"], self.cu, S, out["block_table"],
                       out["num_blocks_per_seq"], out["positions"], out["token_seq"], self.status)
        return out

    def advance(self, logits: torch.Tensor, mask: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Take the next tokens from ``logits`` [B, K, V], after the step's K/V rows were written; returns ``tokens``.

        ``mask`` (int32 words of bits as in ``ops.adjust_logits``): [B, K, ceil(V / 32)] the tokens that each beam may take,
        [B, ...] those of each sequence's beams, or one row for all.
        """
        if not self._room:
            raise RuntimeError("the search has ended" if self._ended else "step_inputs() comes before advance()")
        if tuple(logits.shape[:2]) != (self.B, self.K):
            raise ValueError(f"logits must be [{self.B}, {self.K}, vocab]")
        parents = self._choose(logits, mask)
        self.num_tokens += 1
        self.host_tokens = [n + 1 for n in self.host_tokens]
        self.slots = self.pool.reorder_beams(self.slots, parents, self.num_tokens, self.status, self.seq_ids)
        self._room = False
        return self.tokens

    def all_finished(self) -> bool:
        """Whether every beam has ended (reads the device: synchronises)."""
        return bool(self.finished.all().item())

    def finish(self) -> list[list[tuple[float, list[int]]]]:
        """End the search and free its blocks: each sequence's (score, new tokens), best first, without what follows eos.

        IndexError if a step did not fit the pool (a reordering that left a group as it was, a row without an entry): the
        beams' cache and their tokens were out of step from there on, so there are no lines to return.
        """
        tokens, parents = self.history[:, :self.steps].cpu().tolist()
        scores = self.scores.cpu().tolist()
        if not self._ended:
            for s in self.seq_ids:
                self.pool.release_beams(s)
            self.pool.flush()
            self._ended, self._room = True, False
        ops._raise_status_value("beam search", int(self.status.item()))
        found = []
        for b in range(self.B):
            beams = []
            for k in range(self.K):
                line, j = [], k
                for t in range(self.steps - 1, -1, -1):
                    line.append(tokens[t][b][j])
                    j = parents[t][b][j]
                line.reverse()
                if self.eos in line:
                    line = line[:line.index(self.eos) + 1]
                beams.append((scores[b][k], line))
            found.append(beams)
        return found
