"""The `hip` runtime's entries for operators of language models: rotary positions, the 8-bit key/value cache
and the adjustment of logits.  Checks of shapes and addresses, choice of the kernel variant, launch -- the
kernels are in codegen/lm_kernel.py."""
from __future__ import annotations

import numpy as np

from dlgrad_amd.buffer import Buffer
from dlgrad_amd.codegen import lm_kernel as K
from dlgrad_amd.device import Device
from dlgrad_amd.dispatch import dispatcher
from dlgrad_amd.helpers import CustomOps
from dlgrad_amd.runtime.hip import DevicePtr, _addr, _upload, alloc, kernel, launch, props

EXACT_WHOLE = 1 << 24        # whole numbers up to here are exact in fp32


def _on_device(what: str, **tensors) -> None:
    for name, t in tensors.items():
        if t is not None and (t.is_host_scalar or t.device is not Device.HIP):
            raise ValueError(f"{what}: {name} is not a tensor on the hip device")


def _aligned(*addrs: int) -> bool:
    return not any(a & 15 for a in addrs)


class Cache8:
    """One layer of an 8-bit key/value cache in device memory: codes, scales and the fp32 tails."""
    __slots__ = ("batch", "heads", "d", "width", "blocks", "kc", "vc", "scales", "tail_k", "tail_v")

    def __init__(self, batch: int, heads: int, d: int, blocks: int) -> None:
        self.batch, self.heads, self.d, self.blocks = batch, heads, d, blocks
        self.width = K.cache8_width(d)
        n = batch * heads * blocks
        codes = n * K.CACHE8_BLOCK * self.width // 4                       # in units of 4 bytes, as everything is allocated
        self.kc, self.vc = alloc(codes), alloc(codes)                        # (a block is written whole before its first read)
        self.scales = Buffer.full((n, 2), 0.0, Device.HIP)
        # tails are read in whole blocks: columns beyond d, and rows not written yet, are zeros from the start
        self.tail_k, self.tail_v = (Buffer.full((2, batch * heads, K.CACHE8_BLOCK, self.width), 0.0, Device.HIP) for _ in range(2))

    @property
    def nbytes(self) -> int:
        return self.kc.nbytes + self.vc.nbytes + self.scales.nbytes + self.tail_k.nbytes + self.tail_v.nbytes


class HIPLM:
    """Dispatch-table entries for Device.HIP."""

    # workgroups the 8-bit attention aims for when it splits the tokens of a sequence
    ATTEND_WORKGROUPS_PER_CU = 4

    @staticmethod
    def words(a: np.ndarray) -> Buffer:
        """A host array of 64-bit words in device memory, as a Buffer of twice as many floats that nothing does arithmetic on."""
        a = np.ascontiguousarray(a, dtype=np.uint64)
        p = alloc(2 * a.size)
        _upload(p.addr, a)
        return Buffer(p, (2 * a.size,), Device.HIP)

    # ---- rotary positions ------------------------------------------------------------------------
    @staticmethod
    @dispatcher.register(CustomOps.ROTARY, Device.HIP)
    def rotary(parts: list, freq: Buffer, rows: int, T: int, per: int, d: int, rot: int, half: bool, back: bool, gain: float,
               positions: Buffer | None = None, start: Buffer | None = None, inplace: bool = False) -> list:
        """parts: one or two (Buffer, heads, pitch): `rows` rows of `heads` heads of d, `pitch` floats apart.  Row i is position
        i % T of sequence i // T // per.  Returns the turned tensors' pointers (rows * heads * d floats each), or writes
        the parts themselves when `inplace`."""
        _on_device("rotary", positions=positions, start=start, **{f"x{i}": p[0] for i, p in enumerate(parts)})
        if not 1 <= len(parts) <= 2 or not 0 < rot <= d or rot % 2 or freq.numel != rot:
            raise ValueError(f"rotary: {len(parts)} tensors, {rot} of {d} elements turned, {freq.numel // 2} frequencies")
        if rows == 0:
            return [x.ptr if inplace else alloc(0) for x, _, _ in parts]
        if T < 1 or per < 1 or rows % (T * per) or T > EXACT_WHOLE:
            raise ValueError(f"rotary: {rows} rows are not whole sequences of {T}")
        batch = rows // (T * per)
        for x, heads, pitch in parts:
            if heads < 1 or pitch < heads * d or x.numel < (rows - 1) * pitch + heads * d:
                raise ValueError(f"rotary: {rows} rows of {heads} heads of {d} are not in a tensor of {x.numel} elements with rows {pitch} apart")
            if pitch >= 2 ** 32:
                raise ValueError(f"rotary: rows {pitch} elements apart exceed the kernel's 32-bit pitch")
        if positions is not None and positions.numel not in (T, batch * T):
            raise ValueError(f"rotary: {positions.numel} positions for {batch} sequences of {T}")
        if start is not None and start.numel not in (1, batch):
            raise ValueError(f"rotary: {start.numel} starts for {batch} sequences")
        outs = [x.ptr if inplace else alloc(rows * heads * d) for x, heads, _ in parts]
        out_pitch = [p if inplace else h * d for _, h, p in parts]
        addrs = [_addr(x) for x, _, _ in parts]
        unit = 8 if half else 4                                        # elements of a unit of pairs in 16-byte accesses
        vec = rot % unit == 0 and d % 4 == 0 and all(p % 4 == 0 for _, _, p in parts) and _aligned(*addrs, *[o.addr for o in outs])
        units = rot // unit if vec else rot // 2
        if not inplace:
            units += (d - rot) // (4 if vec else 1)
        most = max(rows * -(-h // K.ROTARY_HEADS) * units for _, h, _ in parts)
        if (most + 255) // 256 >= 2 ** 31:
            raise ValueError(f"rotary: {rows} rows exceed the grid")
        two = len(parts) - 1
        launch(kernel(K.rotary_kernel, half, vec), ((most + 255) // 256, 1, 1 + two), 256, addrs[0], outs[0].addr, addrs[two], outs[two].addr,
               _addr(freq), _addr(positions) if positions is not None else 0, _addr(start) if start is not None else 0,
               rows, T, per, parts[0][1], parts[two][1], d, rot, parts[0][2], parts[two][2], out_pitch[0], out_pitch[two],
               T if positions is not None and positions.numel == batch * T else 0,
               1 if start is not None and start.numel == batch else 0, int(back), float(gain))
        return outs

    # ---- the 8-bit cache ---------------------------------------------------------------------------
    @staticmethod
    def _cache8_lengths(what: str, c: Cache8, lengths: Buffer, counts: Buffer | None) -> None:
        _on_device(what, lengths=lengths, counts=counts)
        if lengths.numel != c.batch or (counts is not None and counts.numel != c.batch):
            raise ValueError(f"{what}: {lengths.numel} lengths and {'no' if counts is None else counts.numel} counts for {c.batch} sequences")

    @staticmethod
    @dispatcher.register(CustomOps.CACHE8_WRITE, Device.HIP)
    def cache8_write(cache: Cache8, k: Buffer, v: Buffer, lengths: Buffer, counts: Buffer | None = None) -> None:
        c = cache
        _on_device("cache8_write", k=k, v=v)
        HIPLM._cache8_lengths("cache8_write", c, lengths, counts)
        C = c.heads * c.d
        if k.ndim != 3 or k.shape != v.shape or k.shape[0] != c.batch or k.shape[2] != C:
            raise ValueError(f"cache8_write: keys {k.shape} and values {v.shape} for {c.batch} sequences of {c.heads} heads of {c.d}")
        T = k.shape[1]
        if T > c.blocks * K.CACHE8_BLOCK:
            raise ValueError(f"cache8_write: {T} tokens for a cache of {c.blocks * K.CACHE8_BLOCK}")
        if T == 0:
            return
        vec = C % 4 == 0 and c.d % 4 == 0 and _aligned(_addr(k), _addr(v))
        # a call may complete the block it starts in and ceil(T / 64) more
        launch(kernel(K.cache8_write_kernel, c.width, vec), (1 + -(-T // K.CACHE8_BLOCK), c.heads, c.batch), 256, _addr(k), _addr(v),
               _addr(lengths), _addr(counts) if counts is not None else 0, c.kc.addr, c.vc.addr, _addr(c.scales), _addr(c.tail_k), _addr(c.tail_v),
               T, c.heads, c.d, c.blocks, C, C)

    @staticmethod
    def attend_splits(groups: int, blocks: int, compute_units: int) -> int:
        """Into how many parts the blocks of a sequence are cut when one part makes `groups` workgroups: enough to fill the
        device, and four blocks a part at least, one for each wavefront.  The length is device data, so the capacity
        stands for it; a part whose blocks are not there yet costs its launch."""
        return max(1, min(HIPLM.ATTEND_WORKGROUPS_PER_CU * compute_units // max(groups, 1), (blocks + 3) // 4))

    @staticmethod
    @dispatcher.register(CustomOps.CACHE8_ATTEND, Device.HIP)
    def cache8_attend(cache: Cache8, q: Buffer, scale: float, lengths: Buffer, counts: Buffer | None = None) -> DevicePtr:
        c = cache
        _on_device("cache8_attend", q=q)
        HIPLM._cache8_lengths("cache8_attend", c, lengths, counts)
        if q.ndim != 3 or q.shape[0] != c.batch or q.shape[2] == 0 or q.shape[2] % (c.heads * c.d):
            raise ValueError(f"cache8_attend: queries {q.shape} for {c.batch} sequences with {c.heads} key heads of {c.d}")
        T, group = q.shape[1], q.shape[2] // (c.heads * c.d)
        if T > c.blocks * K.CACHE8_BLOCK:
            raise ValueError(f"cache8_attend: {T} positions for a cache of {c.blocks * K.CACHE8_BLOCK}")
        y = alloc(q.numel)
        if q.numel == 0:
            return y
        rows, pairs = T * group, c.batch * c.heads
        tiles = -(-rows // 16)
        splits = HIPLM.attend_splits(pairs * tiles, c.blocks, props()["compute_units"])
        if pairs * tiles * splits >= 2 ** 31 or pairs * rows >= 2 ** 31:
            raise ValueError(f"cache8_attend: {pairs} heads of {rows} query rows exceed the grid")
        part = alloc(pairs * rows * splits * (c.width + 2)) if splits > 1 else None
        launch(kernel(K.cache8_attend_kernel, c.width), pairs * tiles * splits, 256, _addr(q), c.kc.addr, c.vc.addr, _addr(c.scales), _addr(c.tail_k),
               _addr(c.tail_v), _addr(lengths), _addr(counts) if counts is not None else 0, y.addr, part.addr if part is not None else 0,
               c.batch, T, c.heads, group, c.d, c.blocks, tiles, splits, float(scale))
        if part is not None:
            launch(kernel(K.cache8_join_kernel, c.width), (pairs * rows + 3) // 4, 256, part.addr, y.addr, pairs * rows, T, c.heads, group, c.d, splits)
        return y

    @staticmethod
    @dispatcher.register(CustomOps.CACHE8_READ, Device.HIP)
    def cache8_read(cache: Cache8, n: int, lengths: Buffer, counts: Buffer | None = None, extra: int = 0) -> tuple[DevicePtr, DevicePtr]:
        c = cache
        HIPLM._cache8_lengths("cache8_read", c, lengths, counts)
        if not 0 <= n <= c.blocks * K.CACHE8_BLOCK or not 0 <= extra <= c.blocks * K.CACHE8_BLOCK:
            raise ValueError(f"cache8_read: {n} positions (and {extra} new ones) of a cache of {c.blocks * K.CACHE8_BLOCK}")
        size = c.batch * n * c.heads * c.d
        k, v = alloc(size), alloc(size)
        if size:
            launch(kernel(K.cache8_read_kernel, c.width), (-(-n // K.CACHE8_BLOCK), c.heads, c.batch), 256, c.kc.addr, c.vc.addr, _addr(c.scales),
                   _addr(c.tail_k), _addr(c.tail_v), _addr(lengths), _addr(counts) if counts is not None else 0, k.addr, v.addr,
                   n, c.heads, c.d, c.blocks, extra)
        return k, v

    # ---- logits ----------------------------------------------------------------------------------------
    @staticmethod
    def adjust_items(B: int, V: int, compute_units: int) -> int:
        """Logits per thread of the adjustment: every block walks its row's whole history, so long slices of the vocabulary save
        walks -- as long as there are two blocks for every compute unit."""
        for items in (32, 16, 8):
            if B * -(-V // (256 * items)) >= 2 * compute_units:
                return items
        return 4

    @staticmethod
    @dispatcher.register(CustomOps.ADJUST_LOGITS, Device.HIP)
    def adjust_logits(logits: Buffer, history: Buffer | None, lengths: Buffer | None, penalties: tuple, bias: Buffer | None, hidden: Buffer | None) -> DevicePtr:
        """logits (B, V); history (B, L); lengths B; penalties: (repetition, presence, frequency), each a float or a Buffer of B;
        bias and hidden: V or (B, V)."""
        pen = [p if isinstance(p, Buffer) else None for p in penalties]
        _on_device("adjust_logits", logits=logits, history=history, lengths=lengths, bias=bias, hidden=hidden, repetition=pen[0], presence=pen[1], frequency=pen[2])
        if logits.ndim != 2 or logits.shape[1] > EXACT_WHOLE:
            raise ValueError(f"adjust_logits: logits {logits.shape} are not rows of at most {EXACT_WHOLE} tokens")
        B, V = logits.shape
        if history is not None and (history.ndim != 2 or history.shape[0] != B or history.shape[1] > EXACT_WHOLE):
            raise ValueError(f"adjust_logits: a history {history.shape} for {B} rows")
        if lengths is not None and (history is None or lengths.numel != B):
            raise ValueError(f"adjust_logits: {lengths.numel} lengths for {'no history' if history is None else f'{B} rows'}")
        for name, t in (("bias", bias), ("hidden", hidden)):
            if t is not None and (t.shape[-1:] != (V,) or t.numel not in (V, B * V)):
                raise ValueError(f"adjust_logits: {name} {t.shape} for logits {logits.shape}")
        for name, p in zip(("repetition", "presence", "frequency"), pen):
            if p is not None and p.numel != B:
                raise ValueError(f"adjust_logits: {p.numel} values of {name} for {B} rows")
        y = alloc(B * V)
        if B * V == 0:
            return y
        if B > 65535:
            raise ValueError(f"adjust_logits: {B} rows, at most 65535 in one call")
        addr = lambda t: 0 if t is None else _addr(t)                     # noqa: E731
        vec = V % 4 == 0 and _aligned(_addr(logits), addr(bias), addr(hidden), y.addr)
        items = HIPLM.adjust_items(B, V, props()["compute_units"])
        launch(kernel(K.adjust_logits_kernel, items, vec), (-(-V // (256 * items)), B, 1), 256, _addr(logits), addr(history), addr(lengths),
               addr(bias), addr(hidden), y.addr, *[addr(p) for p in pen], V, 0 if history is None else history.shape[1],
               V if bias is not None and bias.numel == B * V else 0, V if hidden is not None and hidden.numel == B * V else 0,
               *[0.0 if isinstance(p, Buffer) else float(p) for p in penalties])
        return y
