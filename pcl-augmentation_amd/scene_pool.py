"""Augmented scenes that stay in HBM: a pool of pages, block tables made on the GPU from the lengths a finished batch holds, slot
maps, and the points of the scenes a training step asks for, packed (include/real3daug_hip.h: r3d_block_tables, r3d_slot_map,
r3d_move_rows).  288 GB take every augmented frame of a training split (20 bytes a point); a culled or grown scene takes
the pages it needs.  Tensors on the GPU in and out, on the current stream, no host round trip; no CPU fallback.
"""
from __future__ import annotations

import math
from typing import NamedTuple

from . import _lib
from .point_ops import forward_mode, not_as_read, on_device_of


class BlockTables(NamedTuple):
    tables: object       # int32 [rows, max_blocks]: the blocks of every row, -1 behind them
    held: object         # int32 [rows]: points every row is for
    free_blocks: object  # int32 [blocks]: the stack of blocks that belong to no row, -1 behind them
    n_free: object       # int32 [1]
    status: object       # int32 [1]: 0, or _lib.S_CAPACITY where a row was not served


class SlotMap(NamedTuple):
    offsets: object   # int64 [sequences + 1]: first token of every sequence
    slots: object     # int64 [capacity]: where the token's point stands, -1 behind the last one
    sequence: object  # int32 [capacity]: which sequence it is of, -1 behind the last one


def _whole(what, name, t, dtype, dims):
    if t.dtype is not dtype or t.dim() != dims or not t.is_contiguous():
        raise ValueError(f"{what}: {name} must be a contiguous {dtype} tensor of {dims} axes, got {t.dtype} {tuple(t.shape)}")


def block_tables(lengths, block_size, tables, held, free_blocks, n_free):
    """Block tables for new lengths: row i made ready for ``lengths[i]`` points from the blocks it has (``tables[i]``, for
    ``held[i]`` points) and the stack of free ones.

    As if row after row: rows with more blocks than ``ceil(lengths[i] / block_size)`` give back the ones behind (pushed in order),
    then rows with fewer pop the rest from the end of the stack.  The first row whose blocks are not there and every later growing
    row keep what they had, and so does a row with a negative length or one beyond its table: ``held`` tells, and
    ``status`` is not 0.  All int32: lengths, held [rows], tables [rows, max_blocks], free_blocks [blocks], n_free [1].
    Returns new tensors (``BlockTables``); the inputs stay as they are."""
    import torch
    what = "block_tables"
    for name, t, dims in (("lengths", lengths, 1), ("tables", tables, 2), ("held", held, 1), ("free_blocks", free_blocks, 1), ("n_free", n_free, 1)):
        _whole(what, name, t, torch.int32, dims)
    (rows, most), blocks = tables.shape, free_blocks.shape[0]
    if lengths.shape[0] != rows or held.shape[0] != rows or n_free.shape[0] != 1:
        raise ValueError(f"{what}: lengths and held must be [{rows}], n_free [1]")
    if not 1 <= rows <= _lib.MAX_SCENES or most < 1 or blocks < 1:
        raise ValueError(f"{what}: no rows or no blocks (or more than 2^24 rows)")
    block_size = int(block_size)
    if block_size < 1 or block_size * most >= 2 ** 31:
        raise ValueError(f"{what}: block_size must be positive and block_size * max_blocks below 2^31")
    with on_device_of(what, lengths, tables, held, free_blocks, n_free):
        lib = _lib.load()
        new = torch.empty_like      # (all dense)
        out = BlockTables(new(tables), new(held), new(free_blocks), new(n_free), new(n_free))
        ws = torch.empty(lib.r3d_block_tables_workspace_bytes(rows), dtype=torch.uint8, device=lengths.device)
        _lib.check(lib.r3d_block_tables(lengths.data_ptr(), rows, block_size, most, tables.data_ptr(), held.data_ptr(), free_blocks.data_ptr(),
                                        blocks, n_free.data_ptr(), out[0].data_ptr(), out[1].data_ptr(), out[2].data_ptr(), out[3].data_ptr(),
                                        out[4].data_ptr(), ws.data_ptr(), ws.numel(), _lib.raw_stream(lengths.get_device())), "r3d_block_tables")
    return out


def slot_map(lengths, block_size, tables=None, rows=None, capacity=None):
    """Where the points of some scenes stand, one after the other (``SlotMap``): sequence i is row ``rows[i]`` (int32; None: every
    row in order) with ``lengths[row]`` points (int32), point p of it stands at ``tables[row, p // block_size] * block_size +
    p % block_size``.  tables None: one block a row, e.g. the slabs of a batch with ``block_size = batch.cap``.  ``capacity``: tokens
    there is room for (None: read from the device, which waits for it); tokens beyond it are left out, ``offsets`` tell."""
    import torch
    what = "slot_map"
    _whole(what, "lengths", lengths, torch.int32, 1)
    if tables is not None:
        _whole(what, "tables", tables, torch.int32, 2)
        if tables.shape[0] != lengths.shape[0] or tables.shape[1] < 1:
            raise ValueError(f"{what}: tables must have a row for each of the {lengths.shape[0]} lengths, and a column")
    if rows is not None:
        _whole(what, "rows", rows, torch.int32, 1)
    block_size, most = int(block_size), 1 if tables is None else tables.shape[1]
    if lengths.shape[0] < 1 or block_size < 1 or block_size * most >= 2 ** 31:
        raise ValueError(f"{what}: no rows, or block_size not positive, or block_size * max_blocks not below 2^31")
    if capacity is not None and int(capacity) < 0:
        raise ValueError(f"{what}: capacity must not be negative")
    if (lengths if rows is None else rows).shape[0] > _lib.MAX_SCENES:
        raise ValueError(f"{what}: more than 2^24 scenes")
    with on_device_of(what, lengths, *[t for t in (tables, rows) if t is not None]):
        lib = _lib.load()
        if capacity is None:
            each = lengths.clamp(0, block_size * most)
            if rows is not None:
                there = (rows >= 0) & (rows < lengths.shape[0])
                each = torch.where(there, each[rows.clamp(0, lengths.shape[0] - 1).long()], 0)
            capacity = int(each.sum(dtype=torch.int64))
        n, capacity = lengths.shape[0] if rows is None else rows.shape[0], int(capacity)
        device, empty = lengths.device, torch.empty
        out = SlotMap(empty(n + 1, dtype=torch.int64, device=device), empty(capacity, dtype=torch.int64, device=device), lengths.new_empty(capacity))
        # (an empty tensor has no address; nothing is written where capacity is 0)
        slots, sequence = (t.data_ptr() if capacity else out.offsets.data_ptr() for t in out[1:])
        _lib.check(lib.r3d_slot_map(lengths.data_ptr(), lengths.shape[0], 0 if tables is None else tables.data_ptr(), block_size, most,
                                    0 if rows is None else rows.data_ptr(), n, capacity, out.offsets.data_ptr(), slots, sequence,
                                    _lib.raw_stream(lengths.get_device())), "r3d_slot_map")
    return out


def _slots(what, name, slots):
    import torch
    _whole(what, name, slots, torch.int64, 1)


_ROWS = [_lib.Rows * n for n in range(_lib.MAX_ROW_ARRAYS + 1)]


def _move(what, sources, dests, src_slots, dst_slots, n):
    rows = []
    for s, t in zip(sources, dests):
        size, shape = s.element_size(), s.shape
        width = size * (1 if len(shape) == 1 else shape[1] if len(shape) == 2 else math.prod(shape[1:]))
        rows.append((s.data_ptr(), t.data_ptr(), s.stride(0) * size if shape[0] > 1 else width, t.stride(0) * size if t.shape[0] > 1 else width, width))
    _lib.check(_lib.load().r3d_move_rows(_ROWS[len(rows)](*rows), len(rows), 0 if src_slots is None else src_slots.data_ptr(),
                                         0 if dst_slots is None else dst_slots.data_ptr(), n, sources[0].shape[0], dests[0].shape[0],
                                         _lib.raw_stream(sources[0].get_device())), "r3d_move_rows")


def _rows_of(what, name, tensors, like=None):
    """Tensors [rows, ...] with a row in one piece, the same number of rows each."""
    import torch
    if isinstance(tensors, torch.Tensor):      # (it would be taken for its rows)
        raise ValueError(f"{what}: {name} are a tuple of tensors")
    tensors, forward = tuple(tensors), forward_mode()
    if not 1 <= len(tensors) <= _lib.MAX_ROW_ARRAYS:
        raise ValueError(f"{what}: 1 to {_lib.MAX_ROW_ARRAYS} {name}")
    n = tensors[0].shape[:1]
    for t in tensors:
        if not n or t.shape[:1] != n:
            raise ValueError(f"{what}: {name} must have the same number of rows")
        if t.requires_grad or (forward and torch.autograd.forward_ad.unpack_dual(t).tangent is not None):
            raise ValueError(f"{what}: no gradient passes through moved rows (detach them)")
        if t.is_neg() or t.is_conj():
            raise not_as_read(what)
        if t.is_contiguous() and t.numel():
            continue
        width = 1
        for e, s in zip(reversed(t.shape[1:]), reversed(t.stride()[1:])):
            if e != 1 and s != width:
                raise ValueError(f"{what}: a row of {name} must lie in one piece")
            width *= e
        if width == 0:
            raise ValueError(f"{what}: empty rows")
    return tensors


def take_rows(slots, sources):
    """Rows of up to four tensors by their slots, in one pass: ``out[k][t] = sources[k][slots[t]]``, zeros where the slot is
    outside the source (a map's -1).  slots int64 [n] (``SlotMap.slots``); sources [rows, ...] of any type, a row in one piece.
    Returns a tuple of dense tensors.  Not differentiable: for data, not for features."""
    import torch
    what = "take_rows"
    _slots(what, "slots", slots)
    sources = _rows_of(what, "sources", sources)
    n = slots.shape[0]
    with on_device_of(what, slots, *sources):
        outs = tuple([t.new_empty((n, *t.shape[1:])) for t in sources])
        if n:
            if sources[0].shape[0] == 0:
                return tuple(o.zero_() for o in outs)
            _move(what, sources, outs, slots, None, n)
    return outs


def put_rows(slots, rows, dests, source_slots=None):
    """The other way, in place: ``dests[k][slots[t]] = rows[k][t]`` -- or ``rows[k][source_slots[t]]`` -- for up to four pairs of
    tensors in one pass.  Nothing is written where either slot is outside (a map's -1): rows that no slot names stay as they
    were.  The slots must be distinct; which of two equal ones wins is not defined, nor is a row read that the same call writes.
    Returns dests."""
    import torch
    what = "put_rows"
    _slots(what, "slots", slots)
    rows, dests = _rows_of(what, "rows", rows), _rows_of(what, "dests", dests)
    if len(rows) != len(dests) or any(r.dtype != d.dtype or r.shape[1:] != d.shape[1:] for r, d in zip(rows, dests)):
        raise ValueError(f"{what}: rows and dests must match in number, type and shape of a row")
    n = slots.shape[0]
    if source_slots is not None:
        _slots(what, "source_slots", source_slots)
        if source_slots.shape[0] != n:
            raise ValueError(f"{what}: as many source_slots as slots")
    elif rows[0].shape[0] < n:
        raise ValueError(f"{what}: {n} slots for {rows[0].shape[0]} rows")
    for d in dests:
        if d.shape[0] > 1 and d.stride(0) < d[0].numel():
            raise ValueError(f"{what}: the rows of dests overlap")
    with on_device_of(what, slots, *rows, *dests, *(() if source_slots is None else (source_slots,))):
        if n and rows[0].shape[0] and dests[0].shape[0]:
            _move(what, rows, dests, source_slots, slots, n)
            torch.autograd.graph.increment_version(dests)      # (autograd sees a tensor that it has kept change)
    return dests


class PackedScenes(NamedTuple):
    xyzi: object      # float32 [tokens, 4]
    label: object     # int32 [tokens], the bits of the batch's uint32 labels
    offsets: object   # int64 [scenes + 1]
    sequence: object  # int32 [tokens]: number within the request, -1 behind the last point
    slots: object     # int64 [tokens]


def _with_index(device):
    """This device by its number: "cuda" is the current one, now (and stays it when another becomes current)."""
    import torch
    device = torch.device(device)
    return device if device.type != "cuda" or device.index is not None else torch.device("cuda", torch.cuda.current_device())


class ScenePool:
    """Up to ``max_scenes`` augmented scenes resident on one GPU, in ``n_blocks`` pages of ``block_size`` points.

    ``add(batch)`` takes the scenes of a finished ``SceneBatch`` where they stand, ``packed(scenes)`` returns the points of the
    scenes a step asks for; neither waits for the device (but see ``packed``, and numbers in a tensor are read back).  All on the
    current stream: a program that uses the pool from several orders them."""

    def __init__(self, max_scenes, max_points, n_blocks=None, block_size=2048, device="cuda:0"):
        torch = _lib.require_gpu()
        max_scenes, max_points, block_size = int(max_scenes), int(max_points), int(block_size)
        if max_scenes < 1 or max_points < 1 or block_size < 1:
            raise ValueError("ScenePool: max_scenes, max_points and block_size must be positive")
        most = -(-max_points // block_size)
        if most * block_size >= 2 ** 31:
            raise ValueError("ScenePool: a scene must have fewer than 2^31 points")
        n_blocks = max_scenes * most if n_blocks is None else int(n_blocks)
        if not 1 <= n_blocks < 2 ** 31:
            raise ValueError("ScenePool: n_blocks must be positive and below 2^31")
        self.block_size, self.max_scenes, self.max_points, self.device = block_size, max_scenes, most * block_size, _with_index(device)
        with _lib.on(self.device):
            self.xyzi = torch.zeros((n_blocks * block_size, 4), dtype=torch.float32, device=self.device)
            self.label = torch.zeros((n_blocks * block_size,), dtype=torch.int32, device=self.device)
            i32 = dict(dtype=torch.int32, device=self.device)
            self.blocks = BlockTables(torch.full((max_scenes, most), -1, **i32), torch.zeros(max_scenes, **i32),
                                      torch.arange(n_blocks - 1, -1, -1, **i32), torch.full((1,), n_blocks, **i32), torch.zeros(1, **i32))
            self._refused = torch.zeros(1, **i32)      # bits of every ``resize`` since ``raise_on_status`` last looked

    def _rows(self, scenes):
        import torch
        if isinstance(scenes, torch.Tensor):
            scenes = scenes.tolist()
        scenes = [int(s) for s in scenes]
        if any(not 0 <= s < self.max_scenes for s in scenes):
            raise ValueError(f"ScenePool: scenes are numbered 0 to {self.max_scenes - 1}")
        return scenes

    def _on_device(self, scenes):
        """Scene numbers on the device; from pinned memory, which no call waits for."""
        import torch
        return torch.tensor(scenes, dtype=torch.int32, pin_memory=True).to(self.device, non_blocking=True)

    @property
    def lengths(self):
        """Points of every scene (int32 [max_scenes], on the device; 0: no scene)."""
        return self.blocks.held

    @_lib.on_own_device
    def resize(self, lengths):
        """New lengths for all scenes (int32 [max_scenes] on the device): pages given back and taken (``block_tables``).  What a
        scene's first points are stays; new ones are whatever the page held."""
        import torch
        b, stream = self.blocks, torch.cuda.current_stream()
        for t in b:      # (made on another stream, they would be handed out there while this one still reads them)
            t.record_stream(stream)
        self.blocks = block_tables(lengths, self.block_size, b.tables, b.held, b.free_blocks, b.n_free)
        self._refused.bitwise_or_(self.blocks.status)

    def check_scenes(self, scenes, n):
        """The distinct scene numbers of a batch of n (None: 0 .. n-1); raises where they are not that."""
        scenes = list(range(n)) if scenes is None else self._rows(scenes)
        if len(scenes) != n or len(set(scenes)) != n or n > self.max_scenes:
            raise ValueError(f"ScenePool: {n} distinct scene numbers below {self.max_scenes}")
        return scenes

    def check_device(self, device):
        """Raises where scenes on this device cannot go into the pool."""
        if _with_index(device) != self.device:
            raise ValueError(f"ScenePool: the batch is on {device}, the pool on {self.device}")

    @_lib.on_own_device
    def add(self, batch, scenes=None):
        """The merged clouds of a finished batch (``SceneBatch.finish``) become scenes ``scenes`` (distinct numbers, one per scene of
        the batch; default 0 .. B-1), replacing what was there.  A scene the pool has no room for keeps its old points.
        Returns an int32 tensor [B] on the device: 1 where the scene was taken."""
        import torch
        scenes = self.check_scenes(scenes, batch.B)
        self.check_device(batch.device)
        rows = self._on_device(scenes)
        self.resize(self.blocks.held.index_copy(0, rows.long(), batch.n_out))
        taken = self.blocks.held[rows.long()] == batch.n_out
        new = torch.where(taken, batch.n_out, 0)
        capacity = batch.B * batch.cap
        at = slot_map(torch.zeros_like(self.blocks.held).index_copy_(0, rows.long(), new), self.block_size, self.blocks.tables, rows, capacity)
        put_rows(at.slots, (batch.out_xyzi.view(-1, 4), batch.out_label.view(-1)), (self.xyzi, self.label),
                 source_slots=slot_map(new, batch.cap, capacity=capacity).slots)
        return taken.to(torch.int32)

    @_lib.on_own_device
    def remove(self, scenes):
        """These scenes' pages are free again."""
        self.resize(self.blocks.held.index_fill(0, self._on_device(self._rows(scenes)).long(), 0))

    @_lib.on_own_device
    def packed(self, scenes, capacity=None):
        """The points and labels of these scenes (any order, repeats allowed), one scene after the other (``PackedScenes``).
        ``capacity``: room for that many points, zeros behind the last one (None: exactly as many as there are, which
        reads the lengths back)."""
        rows = self._on_device(self._rows(scenes))
        m = slot_map(self.blocks.held, self.block_size, self.blocks.tables, rows, capacity)
        xyzi, label = take_rows(m.slots, (self.xyzi, self.label))
        return PackedScenes(xyzi, label, m.offsets, m.sequence, m.slots)

    @_lib.on_own_device
    def raise_on_status(self):
        """Waits for the device; raises where any ``add`` / ``resize`` since the last call of this did not find room for a scene
        (and forgets it: the next call asks about what comes after)."""
        if int(self._refused.item()):
            self._refused.zero_()
            raise _lib.R3DError("ScenePool: no room for a scene (out of pages, or more points than max_points)")
