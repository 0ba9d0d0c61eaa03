"""Low-rank adapters of many requests at once beside a shared projection, on
MI355X: row i of a batch, with adapter a of S (or none), gets

    y_i + scale_a * (x_i A_a^T) B_a^T

on top of the projection's y_i, whatever the projection's scheme.

* :class:`LowRankAdapters` -- the adapters of one projection, or of several that
  share their input (a stacked one's column blocks), laid out once
* :class:`AdapterRows`     -- which adapter each row of a batch has: made once a
  step and passed to every projection of every layer
* :func:`add_low_rank`     -- the addition, in place

The reference serves one model without adapters; none of this has a counterpart
there. No gradient: tensors that need one raise ``RuntimeError``.
"""

from __future__ import annotations

import ctypes

import numpy as np
import torch
from torch.autograd.graph import increment_version

from . import _lib
from .gated_delta import _FLOATS, _require_device, _stream
from .quant import QuantizedRows, _followed, _kept_rows, rows_overlap

_MAX_BLOCKS = 8
_MAX_RANKS = 1 << 16
_MAX_HIDDEN = 1 << 24
_MAX_WIDTH = 1 << 30
# Rows a tile: about as many as adapters have on average, a power of two between these
# (the kernels cut tiles as they need; places that stay empty cost workgroups).
_LEAST_ROWS, _MOST_ROWS = 16, 256
_TABLE = np.dtype([("b", "<i8"), ("a_row", "<i4"), ("rank", "<i4"), ("scale", "<f4"), ("t_col", "<i4")])


class LowRankAdapters:
    """The adapters of the projections that share one input, in the layout that
    :func:`add_low_rank` reads.

    ``projections`` holds, for each projection (column block of a stacked one), its
    S adapters in order: ``(A (r, K), B (N, r), scale)``, or None where that adapter
    leaves the projection alone. Ranks may differ. A whole projection without
    adapters is None. All tensors are of one float dtype, which is that of the rows,
    on one device. The adapters' values are copied, on the current stream: changing
    the tensors later changes nothing here, and a call on another stream has to wait
    for that copy."""

    def __init__(self, projections) -> None:
        projections = list(projections)
        if not 1 <= len(projections) <= _MAX_BLOCKS:
            raise ValueError(f"1 to {_MAX_BLOCKS} projections share their adapters' input, got {len(projections)}")
        given = [t for block in projections if block is not None for pair in block if pair is not None for t in pair[:2]]
        if not given:
            raise ValueError("no projection has an adapter")
        counts = {len(block) for block in projections if block is not None}
        if len(counts) != 1:
            raise ValueError(f"every projection lists the same adapters, got {sorted(counts)} of them")
        if _followed(*given):
            raise RuntimeError("adapters have no gradient; detach them")
        self.count = counts.pop()
        self.device = _require_device(*given)
        self.dtype = given[0].dtype
        self.hidden = given[0].shape[-1]
        widths: list[int] = []
        for j, block in enumerate(projections):
            width = 0
            for pair in block or ():
                if pair is None:
                    continue
                A, B, _ = pair
                if A.dtype != self.dtype or B.dtype != self.dtype:
                    raise ValueError(f"adapters share one dtype, got {A.dtype} and {B.dtype} beside {self.dtype}")
                if A.ndim != 2 or B.ndim != 2 or A.shape[1] != self.hidden or B.shape[1] != A.shape[0] or 0 in B.shape:
                    raise ValueError(f"an adapter is A (r, {self.hidden}) and B (N, r), got {tuple(A.shape)} and "
                                     f"{tuple(B.shape)}")
                if width not in (0, B.shape[0]):
                    raise ValueError(f"projection {j} has {width} outputs, an adapter {B.shape[0]}")
                width = B.shape[0]
            widths.append(width)
        if not 0 < self.hidden <= _MAX_HIDDEN:
            raise ValueError(f"adapters take rows of 1 to {_MAX_HIDDEN} values, got {self.hidden}")
        if max(widths) > _MAX_WIDTH:
            raise ValueError(f"adapters take projections of at most {_MAX_WIDTH} outputs, got {max(widths)}")
        self.widths = tuple(widths)
        table = np.zeros((self.count, len(projections)), dtype=_TABLE)
        a_rows, b_size = 0, 0
        for j, block in enumerate(projections):
            for a, pair in enumerate(block or ()):
                if pair is not None:
                    table[a, j]["rank"], table[a, j]["scale"] = pair[0].shape[0], float(pair[2])
        padded = -(-table["rank"] // 16) * 16
        table["t_col"] = np.cumsum(padded, axis=1) - padded
        table["a_row"] = (np.cumsum(padded) - padded.reshape(-1)).reshape(padded.shape)
        columns = [-(-n // 64) * 64 for n in widths]
        for j, n in enumerate(columns):  # B block by block
            table["b"][:, j] = b_size + (np.cumsum(padded[:, j], dtype=np.int64) - padded[:, j]) * n
            b_size += int(padded[:, j].sum()) * n
        self.rank_total, self.rank_block = int(padded.sum(axis=1).max()), int(padded.max())
        if self.rank_total > _MAX_RANKS or int(padded.sum()) >= 2 ** 31:
            raise ValueError(f"an adapter's ranks add up to at most {_MAX_RANKS}, got {self.rank_total}")
        self._A, self._B = self._laid_out(projections, padded, columns)
        self._index = self._A.get_device()
        n = len(widths)
        self._c_widths, self._c_pointers, self._c_strides = (ctypes.c_int * n)(*widths), ctypes.c_void_p * n, ctypes.c_int64 * n
        self._code = _lib.dtype_code(self.dtype)
        self._workspaces: dict[tuple[int, int], int] = {}
        self._table = torch.from_numpy(table.reshape(-1).view(np.uint8)).to(self.device)

    def _laid_out(self, projections, padded, columns) -> tuple[torch.Tensor, torch.Tensor]:
        """A of all adapters and B of all, in the order in which a wave's lanes take them
        (include/gdn.h), from a few operations whatever the number of adapters."""

        per = 16 // self.dtype.itemsize
        steps = -(-self.hidden // (8 * per))
        no_ranks = torch.zeros((15, self.hidden), dtype=self.dtype, device=self.device)
        no_columns = torch.zeros((max(self.widths), 15), dtype=self.dtype, device=self.device)
        parts = []
        for a in range(self.count):
            for j, block in enumerate(projections):
                if block is not None and block[a] is not None:
                    A = block[a][0]
                    parts.append(A)
                    if padded[a, j] > A.shape[0]:
                        parts.append(no_ranks[:padded[a, j] - A.shape[0]])
        wide = torch.nn.functional.pad(torch.cat(parts), (0, steps * 8 * per - self.hidden))
        laid_a = wide.view(-1, 16, steps, 2, 4, per).permute(0, 2, 3, 4, 1, 5).contiguous()
        laid_b = []
        for j, block in enumerate(projections):
            if not self.widths[j]:
                continue
            parts = []
            for a, pair in enumerate(block):
                if pair is not None:
                    parts.append(pair[1])
                    if padded[a, j] > pair[1].shape[1]:
                        parts.append(no_columns[:self.widths[j], :padded[a, j] - pair[1].shape[1]])
            wide = torch.nn.functional.pad(torch.cat(parts, dim=1), (0, 0, 0, columns[j] - self.widths[j]))
            if per == 8:
                wide = wide.view(columns[j] // 64, 2, 4, 2, 4, -1, 2, 8).permute(5, 0, 1, 3, 6, 2, 4, 7)
            else:
                wide = wide.view(columns[j] // 64, 4, 4, 4, -1, 4, 4).permute(4, 0, 1, 5, 2, 3, 6)
            laid_b.append(wide.reshape(-1))
        return laid_a, laid_b[0] if len(laid_b) == 1 else torch.cat(laid_b)

    def _workspace(self, tiles: int, tile_rows: int) -> int:
        nbytes = self._workspaces.get((tiles, tile_rows))
        if nbytes is None:
            if len(self._workspaces) >= 1024:
                self._workspaces.clear()
            nbytes = self._workspaces[tiles, tile_rows] = int(_lib.load().gdn_add_low_rank_workspace_size(
                self._code, len(self.widths), self.rank_total, self.rank_block, self._c_widths, tiles,
                tile_rows, self.hidden))
        return nbytes


class AdapterRows:
    """Which of ``count`` adapters each row of a batch has, -1 for none: checked,
    sorted and copied to ``device`` once, for every projection of every layer.
    ``index`` is a host sequence or a tensor of whole numbers (read back to the host
    if it is on the GPU). ``distinct``: room for batches of that many different
    adapters, for :meth:`assign`; without it there is room for as many tiles as
    ``index`` takes. Made outside of a graph's capture; its copy on the device
    belongs to the stream it was made on until that is done. Host work of 42 us for one
    row, 45 for 64, 73 for 4096 (of an array; a list of 4096 takes 200 more)."""

    def __init__(self, index, count: int, device: torch.device | str = "cuda", *, distinct: int | None = None) -> None:
        if count < 1:
            raise ValueError(f"AdapterRows needs at least one adapter, got {count}")
        self.count = int(count)
        index = self._checked(index)
        self.rows = len(index)
        used, with_one = len(np.unique(index[index >= 0])), int((index >= 0).sum())
        mean = -(-with_one // max(used, 1))
        self.tile_rows = min(_MOST_ROWS, max(_LEAST_ROWS, 1 << max(mean - 1, 0).bit_length()))
        self.tiles = int((-(-np.unique(index[index >= 0], return_counts=True)[1] // self.tile_rows)).sum())
        if distinct is not None:  # one tile that is not full an adapter
            self.tiles = max(self.tiles, min(self.rows, -(-self.rows // self.tile_rows) + distinct))
        self._plan = torch.from_numpy(self._planned(index)).to(device)
        self.device, self._index = self._plan.device, self._plan.get_device()

    @classmethod
    def of_runs(cls, runs, index, count: int) -> "AdapterRows":
        """The rows of packed prompts (:class:`PackedRuns`), run r's all with
        ``index[r]``."""

        index = cls._host(index)
        if len(index) != len(runs):
            raise ValueError(f"{len(runs)} runs, {len(index)} adapters")
        return cls(np.repeat(index, np.diff(runs.offsets)), count, runs.on_device.device)

    def assign(self, index) -> None:
        """Other adapters for the same number of rows, in the same device memory: what
        a captured graph's next replay uses. The copy goes to the current stream, and
        the host waits for it and for what that stream still has to do (31 us for one row,
        44 for 4096, of an idle one). ``ValueError`` if there is no room for them
        (``distinct``)."""

        index = self._checked(index)
        if len(index) != self.rows:
            raise ValueError(f"{self.rows} rows, {len(index)} adapters")
        self._plan.copy_(torch.from_numpy(self._planned(index)))

    @staticmethod
    def _host(index) -> np.ndarray:
        index = torch.as_tensor(index)
        if index.numel() and (index.is_floating_point() or index.is_complex() or index.dtype == torch.bool):
            raise ValueError(f"adapters are numbered by whole numbers, got {index.dtype}")
        if index.ndim != 1:
            raise ValueError("adapters are listed one a row")
        return index.to("cpu", torch.int64).numpy()

    def _checked(self, index) -> np.ndarray:
        index = self._host(index)
        if len(index) and (index.min() < -1 or index.max() >= self.count):
            raise ValueError(f"adapters must lie in [0, {self.count}), or be -1")
        if len(index) >= 2 ** 31 - 256:
            raise ValueError("the row count must fit int32")
        return index

    def _planned(self, index: np.ndarray) -> np.ndarray:
        """The rows that have an adapter, sorted by it (the rest of the array unused),
        then {adapter, first place, rows} for each tile."""

        plan = np.zeros(self.rows + 3 * self.tiles, dtype=np.int32)
        order = np.argsort(index, kind="stable")
        order = order[np.searchsorted(index[order], 0):]
        plan[:len(order)] = order
        adapters, first, rows = np.unique(index[order], return_index=True, return_counts=True)
        pieces = -(-rows // self.tile_rows)
        if pieces.sum() > self.tiles:
            raise ValueError(f"{len(adapters)} adapters over these rows take {pieces.sum()} tiles, there is room for "
                             f"{self.tiles}; reserve it (distinct=)")
        which = np.repeat(np.arange(len(adapters)), pieces)
        piece = np.arange(len(which)) - np.repeat(np.cumsum(pieces) - pieces, pieces)
        tiles = plan[self.rows:].reshape(-1, 3)
        tiles[:len(which), 0] = adapters[which]
        tiles[:len(which), 1] = first[which] + piece * self.tile_rows
        tiles[:len(which), 2] = np.minimum(rows[which] - piece * self.tile_rows, self.tile_rows)
        return plan


def add_low_rank(outs, x: torch.Tensor, adapters: LowRankAdapters, rows: AdapterRows):
    """Adds to each row of ``outs`` what its adapter makes of the row of ``x``, in
    place, and returns ``outs``.

    ``x (M, hidden)`` is the projections' input (any row stride; of
    :class:`QuantizedRows` the kept rows), ``outs`` their outputs: for one projection
    a tensor ``(M, N)``, else a list with one for each projection of ``adapters``
    (None where it has no adapters), in x's dtype at any row stride, e.g. column
    slices of a stacked output. Sums are float32; a result is rounded once more to
    its dtype. ``scale x A^T`` is kept to float32's 24 bits, 22 for float16. Rows
    without an adapter are left as they are, and a row's result does not depend on the
    rows beside it. Values that are not finite stay in their row, which may then be NaN
    where float32 sums would be infinite."""

    # decode steps are host-bound, hence the integer comparisons and the quick look
    # at the arrays' ends in front of _overlap
    blocks = [outs] if isinstance(outs, torch.Tensor) else outs
    if isinstance(x, QuantizedRows):
        x = _kept_rows(x)
    K, dtype, index = adapters.hidden, adapters.dtype, adapters._index
    if x.ndim != 2 or x.shape[1] != K:
        raise ValueError(f"x must be (rows, {K}), got {tuple(x.shape)}")
    M = x.shape[0]
    if x.dtype is not dtype:
        raise ValueError(f"the adapters are {dtype}, x {x.dtype}")
    if rows.rows != M or rows.count != adapters.count:
        raise ValueError(f"rows of {rows.rows} with {rows.count} adapters, x has {M} and there are {adapters.count}")
    if len(blocks) != len(adapters.widths):
        raise ValueError(f"{len(adapters.widths)} projections, {len(blocks)} outputs")
    if x.get_device() != index or rows._index != index:
        raise ValueError(f"the adapters are on {adapters.device}, x on {x.device}, its adapters' numbers on {rows.device}")
    x_stride, step = x.stride()
    if step != 1 or (M > 1 and x_stride < K):
        x = x.contiguous()
        x_stride = K
    n, size = len(blocks), dtype.itemsize
    pointers, strides, written = [None] * n, [0] * n, []
    at = x.data_ptr()
    ends = [(at, at + ((M - 1) * x_stride + K) * size, x)]
    for j, (out, width) in enumerate(zip(blocks, adapters.widths)):
        if not width:
            continue
        if out is None or out.ndim != 2 or out.shape[0] != M or out.shape[1] != width or out.dtype is not dtype \
                or out.get_device() != index:
            raise ValueError(f"output {j} must be {(M, width)} {dtype} on {adapters.device}")
        stride, step = out.stride()
        if (step != 1 and width > 1) or (M > 1 and stride < width):
            raise ValueError(f"output {j} must consist of packed rows")
        begin = out.data_ptr()
        end = begin + ((M - 1) * stride + width) * size
        for b, e, other in ends:
            if begin < e and b < end and M and _overlap(out, other):
                raise ValueError(f"output {j} overlaps {'x' if other is x else 'another output'}")
        ends.append((begin, end, out))
        written.append(out)
        pointers[j], strides[j] = begin, stride
    if _followed(x, *written):
        raise RuntimeError("adapters have no gradient and no forward mode; call add_low_rank under torch.no_grad()")
    increment_version(written)  # (a graph that saved an output has to see this)
    device = x.device
    nbytes = adapters._workspace(rows.tiles, rows.tile_rows)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
    plan = rows._plan.data_ptr()
    _lib.call_on(device, "gdn_add_low_rank", at, x_stride, adapters._code, adapters._A.data_ptr(),
                 adapters._B.data_ptr(), adapters._table.data_ptr(), adapters.count, n, adapters.rank_total,
                 adapters.rank_block, adapters._c_pointers(*pointers), adapters._c_strides(*strides), adapters._c_widths,
                 plan, plan + 4 * M, rows.tiles, rows.tile_rows, M, K, _lib.ptr(ws), nbytes, _stream(device))
    return outs


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two arrays of packed rows, whose ends lie in each other, share an
    element."""

    stride = a.stride(0)
    return stride != b.stride(0) or rows_overlap(a.data_ptr(), b.data_ptr(), stride, a.shape[1], b.shape[1], a.shape[0],
                                                 a.element_size())
