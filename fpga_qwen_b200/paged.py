"""Sequences over the paged KV cache: page accounting, prompts, decode steps and eviction.

:class:`PageTable` is the host's bookkeeping (which pages a sequence holds, its cached rows and
its RoPE position); :class:`PagedSequences` owns the device side: the page pool, the table, the
lengths and the calls ``qa_paged_append``, ``qa_paged_attn`` and ``qa_paged_evict``. The reference
holds one contiguous history per process (tampajohn/fpga-qwen engine/core.cpp:223, :277) and has
no counterpart; the row arithmetic and the order of the calls are those of its model
(core.cpp:395-406, :606-624), as in :class:`~fpga_qwen_b200.engine.AttentionModel`, and like it
the tensors are the attention inputs: pre-norm ``q [L][n][hq][128]``, ``k, v [L][n][hkv][128]``.

A batch row is a sequence's place in the table: rows without a sequence have length 0, so a step
always runs over all ``max_seqs`` rows with device-side lengths, and a captured step stays valid
while sequences come, go, grow and are evicted.
"""
from __future__ import annotations

import torch

from .qattn import Context, Pages, PREFIX_CHUNK, QAttnError, QA_ERR_CAPACITY, QA_ERR_INVALID, QA_ERR_STATE


class PageTable:
    """Host bookkeeping of a pool: free pages, and each open sequence's pages, rows and position."""

    def __init__(self, n_pages: int, page_rows: int, max_seqs: int, max_rows: int):
        if min(n_pages, page_rows, max_seqs, max_rows) < 1:
            raise QAttnError(QA_ERR_INVALID, "empty page pool")
        self.page_rows, self.cols = page_rows, -(-max_rows // page_rows)
        self.max_rows = max_rows
        self.free = list(range(n_pages - 1, -1, -1))
        self.pages: list[list[int] | None] = [None] * max_seqs        # None: no sequence
        self.rows, self.position = [0] * max_seqs, [0] * max_seqs

    def open(self) -> int:
        for seq, held in enumerate(self.pages):
            if held is None:
                self.pages[seq], self.rows[seq], self.position[seq] = [], 0, 0
                return seq
        raise QAttnError(QA_ERR_CAPACITY, "all sequences are in use")

    def _check(self, seq: int):
        if not 0 <= seq < len(self.pages) or self.pages[seq] is None:
            raise QAttnError(QA_ERR_STATE, f"no sequence {seq}")

    def close(self, seq: int):
        self._check(seq)
        self.free += reversed(self.pages[seq])
        self.pages[seq], self.rows[seq], self.position[seq] = None, 0, 0

    def live(self) -> list[int]:
        return [seq for seq, held in enumerate(self.pages) if held is not None]

    def grow(self, counts: dict[int, int]) -> list[tuple[int, int, int]]:
        """Adds counts[seq] rows to each listed sequence; returns the new table entries (seq, column,
        page). Nothing changes where a sequence or the pool cannot hold them."""
        need = {}
        for seq, n in counts.items():
            self._check(seq)
            if n < 1:
                raise QAttnError(QA_ERR_INVALID, "Empty token input")
            if self.rows[seq] + n > self.max_rows:
                raise QAttnError(QA_ERR_CAPACITY, f"sequence {seq}: {self.rows[seq]} + {n} rows exceed {self.max_rows}")
            need[seq] = -(-(self.rows[seq] + n) // self.page_rows) - len(self.pages[seq])
        if sum(need.values()) > len(self.free):
            raise QAttnError(QA_ERR_CAPACITY, f"{sum(need.values())} pages wanted, {len(self.free)} free")
        entries = []
        for seq, n in counts.items():
            for _ in range(need[seq]):
                page = self.free.pop()
                entries.append((seq, len(self.pages[seq]), page))
                self.pages[seq].append(page)
            self.rows[seq] += n
            self.position[seq] += n
        return entries

    def shrink(self, seq: int, rows: int):
        """The sequence now holds `rows` cached rows (its position stays); returns pages to the pool."""
        self._check(seq)
        if not 0 <= rows <= self.rows[seq]:
            raise QAttnError(QA_ERR_STATE, f"sequence {seq} holds {self.rows[seq]} rows, not {rows}")
        keep = -(-rows // self.page_rows)
        self.free += reversed(self.pages[seq][keep:])
        del self.pages[seq][keep:]
        self.rows[seq] = rows


class StepOrder:
    """Which layers of the step under way have their new rows. From begin_step, which counts the rows, to the append of
    the last layer they are not all written: an eviction would take whatever their page held before, and another
    begin_step would leave it behind for attention to read."""

    def __init__(self, layers: int):
        self.layers, self.unwritten, self.seqs, self.replays = layers, set(), set(), False

    def begin(self, seqs):
        self.seqs = set(seqs)
        self.unwritten = set() if self.replays else set(range(self.layers))

    def wrote(self, layer: int, n: int):
        self.unwritten -= set(range(layer, layer + n))

    def captured(self):
        """An append was captured and not run: steps are made by replays from now on, which nothing here sees."""
        self.replays = True
        self.unwritten = set()

    def close(self, seq: int):
        self.seqs.discard(seq)
        if not self.seqs:
            self.unwritten = set()

    def check_complete(self, what: str):
        if self.unwritten:
            raise QAttnError(QA_ERR_STATE, f"{what} before the step's rows are appended (layers {sorted(self.unwritten)})")

    def check_written(self, layer: int, n: int):
        missing = sorted(self.unwritten & set(range(layer, layer + n)))
        if missing:
            raise QAttnError(QA_ERR_STATE, f"attend before the step's rows of layers {missing} are appended")


class PagedSequences:
    """Up to max_seqs sequences of a context over a pool of n_pages pages.

    ``prefill`` runs a prompt in sequence slot `slot` of the context (the prefill kernels read
    contiguous rows; what the slot held before is gone) and leaves its rows in pages; ``begin_step``,
    then ``append`` and ``attend`` per layer (or for all layers), make one decode step of every open
    sequence; ``evict`` brings them under a budget by accumulated attention weight. ``max_position``
    bounds RoPE positions, which go on past the cached rows once rows are evicted; ``step_layers`` is the
    most layers of one ``attend`` call (it sizes the workspace, which is made once, so that captured steps
    stay valid: 8 bytes for every sequence, layer, KV head and row; 1 is enough for a loop over layers).
    The constructor extends the context's RoPE tables where ``max_position`` is past them, after which
    graphs captured on the context before have to be captured again (``qa_rope_positions``).
    One caller, and one stream, at a time, as for the context.

    A step's rows count from ``begin_step`` on, so until ``append`` has written them in every layer ``evict``, another
    ``begin_step`` and ``attend`` of a layer without them are refused (``QA_ERR_STATE``; closing the step's
    sequences ends it). Once an ``append`` has been captured into a graph the replays, which nothing here sees,
    are taken to follow their ``begin_step`` at once: that order is then the caller's to keep. Only ``append``
    and ``attend`` can be captured; the calls that also keep the host's books are refused under capture.
    """

    def __init__(self, ctx: Context, n_pages: int, page_rows: int = 16, max_seqs: int = 1, max_rows: int = 4096,
                 max_position: int | None = None, slot: int = 0, step_layers: int | None = None):
        if ctx.config.io_host:
            raise QAttnError(QA_ERR_INVALID, "a device-pointer context (io_host = 0) is wanted")
        self.host = PageTable(n_pages, page_rows, max_seqs, max_rows)
        self.ctx, self.slot, self.layers = ctx, slot, ctx.config.n_layers
        self.max_position = max_position or max(max_rows, ctx.config.context)
        self.step_layers = self.layers if step_layers is None else step_layers
        self.step = StepOrder(self.layers)
        ctx.rope_positions(self.max_position)
        dev = torch.device("cuda", ctx.config.device)
        self.kv = torch.zeros(n_pages, self.layers, 2, ctx.hkv, page_rows, 128, dtype=torch.float16, device=dev)
        self.weights = torch.zeros(n_pages, self.layers, ctx.hkv, page_rows, device=dev)
        self.pages = Pages(self.kv.data_ptr(), self.weights.data_ptr(), n_pages, page_rows)
        self.table = torch.zeros(max_seqs, self.host.cols, dtype=torch.int32, device=dev)
        self.lengths = torch.zeros(max_seqs, dtype=torch.int32, device=dev)      # with the step's new row
        self.positions = torch.zeros(max_seqs, dtype=torch.int32, device=dev)    # of the step's new row
        self.workspace = torch.empty(ctx.paged_workspace(max_seqs, self.step_layers, self.host.cols * page_rows, True),
                                     dtype=torch.uint8, device=dev)

    # -- sequences ---------------------------------------------------------------------------
    def open(self) -> int:
        return self.host.open()

    def close(self, seq: int):
        self._check_uncaptured("close")
        self.host.close(seq)
        self.step.close(seq)
        self.lengths[seq] = 0

    def rows(self, seq: int) -> int:
        return self.host.rows[seq]

    def position(self, seq: int) -> int:
        return self.host.position[seq]

    def _grow(self, counts: dict[int, int]):
        for seq, n in counts.items():
            if 0 <= seq < len(self.host.pages) and self.host.position[seq] + n > self.max_position:
                raise QAttnError(QA_ERR_CAPACITY, f"sequence {seq}: position {self.host.position[seq]} + {n} exceeds {self.max_position}")
        entries = self.host.grow(counts)
        if entries:
            seq, col, page = torch.tensor(entries, dtype=torch.int64).T.to(self.table.device)
            self.table[seq, col] = page.to(torch.int32)

    def _int32(self, values) -> torch.Tensor:
        return torch.tensor(values, dtype=torch.int32).to(self.table.device)

    def _stream(self):
        self.ctx.set_stream(torch.cuda.current_stream(self.table.device).cuda_stream)

    def _capturing(self) -> bool:
        with torch.cuda.device(self.table.device):
            return torch.cuda.is_current_stream_capturing()

    def _check_uncaptured(self, what: str):
        """A replay would repeat the device's part of these calls and not the host's books."""
        if self._capturing():
            raise QAttnError(QA_ERR_STATE, f"{what} while the stream is capturing")

    def _check_inputs(self, n, layers, **tensors):
        heads = {"q": self.ctx.hq, "k": self.ctx.hkv, "v": self.ctx.hkv}
        for name, t in tensors.items():
            if not (isinstance(t, torch.Tensor) and t.device == self.table.device and t.dtype == torch.float32 and t.is_contiguous()):
                raise QAttnError(QA_ERR_INVALID, f"{name} must be a contiguous float32 tensor on {self.table.device}")
            if tuple(t.shape) != (layers, n, heads[name], 128):
                raise QAttnError(QA_ERR_INVALID, f"{name} has shape {tuple(t.shape)}")

    # -- prompts -------------------------------------------------------------------------------
    def prefill(self, seq: int, q, k, v):
        """A prompt of n rows for a new sequence; returns its attention outputs [L][n][hq][128]. The
        sequence takes part in steps from the next begin_step on."""
        n = q.shape[1] if isinstance(q, torch.Tensor) and q.dim() == 4 else 0
        self.host._check(seq)
        if self.host.rows[seq] or self.host.position[seq]:
            raise QAttnError(QA_ERR_STATE, "the sequence already holds rows")
        if n < 1:
            raise QAttnError(QA_ERR_INVALID, "Empty token input")
        if n > self.ctx.config.context:
            raise QAttnError(QA_ERR_CAPACITY, "Context capacity exceeded")
        self._check_inputs(n, self.layers, q=q, k=k, v=v)
        self._check_uncaptured("prefill")
        self._grow({seq: n})
        try:
            self._stream()
            qn, out = torch.empty_like(q), torch.empty_like(q)
            self._run_prompt(seq, n, q, k, v, qn, out)
        except Exception:
            self.host.shrink(seq, 0)                     # as an execution failure resets a slot's sequence
            self.host.position[seq] = 0
            raise
        return out

    def _run_prompt(self, seq, n, q, k, v, qn, out):
        ctx, layers = self.ctx, self.layers
        held = torch.arange(1, n + 1, dtype=torch.int32, device=q.device)
        pos, row_seq = held - 1, torch.full_like(held, seq)
        ctx.paged_append(self.pages, self.table.data_ptr(), self.table.shape[0], self.host.cols, row_seq.data_ptr(),
                         held.data_ptr(), pos.data_ptr(), n, 0, layers, q.data_ptr(), k.data_ptr(), v.data_ptr(),
                         qn.data_ptr())
        ctx.reset(self.slot)
        for b0 in range(0, n, PREFIX_CHUNK):
            b1 = min(n, b0 + PREFIX_CHUNK)
            for layer in range(layers):
                chunk = [t[layer, b0:b1].data_ptr() for t in (q, k, v, qn)]
                ctx.append(self.slot, layer, 1, b0, b1 - b0, *chunk)
                ctx.attn_prefill(self.slot, layer, 1, b0, b1 - b0, chunk[3], out[layer, b0:b1].data_ptr())
            ctx.commit(self.slot, b1 - b0)

    # -- decode --------------------------------------------------------------------------------
    def begin_step(self):
        """Makes room for one new row of every open sequence and counts it in lengths and positions."""
        live = self.host.live()
        if not live:
            raise QAttnError(QA_ERR_STATE, "no open sequence")
        self.step.check_complete("begin_step")
        self._check_uncaptured("begin_step")
        self._grow({seq: 1 for seq in live})
        self.step.begin(live)
        held = [self.host.rows[seq] for seq in range(len(self.host.pages))]
        self.lengths.copy_(self._int32(held))
        self.positions.copy_(self._int32([max(p - 1, 0) for p in self.host.position]))

    def append(self, q, k, v, layer: int = 0, q_out=None):
        """New rows [layers][max_seqs][heads][128] of layers [layer, layer + layers); returns the queries."""
        layers, n = (q.shape[0], self.table.shape[0]) if isinstance(q, torch.Tensor) and q.dim() else (0, 0)
        self._check_inputs(n, layers, q=q, k=k, v=v)
        qn = torch.empty_like(q) if q_out is None else q_out
        self._check_inputs(n, layers, q=qn)
        self._stream()
        self.ctx.paged_append(self.pages, self.table.data_ptr(), n, self.host.cols, 0, self.lengths.data_ptr(),
                              self.positions.data_ptr(), n, layer, layers, q.data_ptr(), k.data_ptr(), v.data_ptr(),
                              qn.data_ptr())
        if not self.step.replays and self._capturing():
            self.step.captured()
        self.step.wrote(layer, layers)
        return qn

    def attend(self, qn, layer: int = 0, add_weights: bool = True, out=None):
        """Attention of the rows just appended; adds their weights for a later eviction."""
        layers, n = (qn.shape[0], self.table.shape[0]) if isinstance(qn, torch.Tensor) and qn.dim() else (0, 0)
        self._check_inputs(n, layers, q=qn)
        self.step.check_written(layer, layers)
        out = torch.empty_like(qn) if out is None else out
        self._check_inputs(n, layers, q=out)
        self._stream()
        self.ctx.paged_attn(self.pages, self.table.data_ptr(), self.host.cols, self.lengths.data_ptr(), n, layer, layers,
                            qn.data_ptr(), out.data_ptr(), add_weights, self.workspace.data_ptr(), self.workspace.numel())
        return out

    def evict(self, keep: int, recent: int = 0):
        """Every sequence of more than `keep` cached rows keeps its last `recent` rows and the heaviest
        others, in each layer and head; their pages past that return to the pool. A row's weight is what
        ``attend`` calls since its append gave it: rows of a prompt weigh nothing until then, and of rows that
        weigh the same the older stay. Returns the old indices of the kept rows,
        [max_seqs][L][hkv][keep] (-1: none)."""
        n = self.table.shape[0]
        if keep < 1 or not 0 <= recent <= keep:
            raise QAttnError(QA_ERR_INVALID, f"keep {keep}, recent {recent}")
        self.step.check_complete("evict")
        self._check_uncaptured("evict")
        keep = min(keep, self.host.cols * self.host.page_rows)
        recent = min(recent, keep)
        kept = torch.empty(n, self.layers, self.ctx.hkv, keep, dtype=torch.int32, device=self.table.device)
        rows = self._int32(self.host.rows)               # (lengths leaves out prompts since the last begin_step)
        self._stream()
        self.ctx.paged_evict(self.pages, self.table.data_ptr(), self.host.cols, self.table.data_ptr(), self.host.cols,
                             rows.data_ptr(), rows.data_ptr(), n, keep, recent, kept.data_ptr())
        self.lengths.copy_(torch.minimum(self.lengths, rows))
        for seq in self.host.live():
            self.host.shrink(seq, min(self.host.rows[seq], keep))
        return kept
