"""The `hip` runtime's entries for operators of language models: rotary positions, the 8-bit key/value cache
and the adjustment of logits.  Checks of shapes and addresses, choice of the kernel variant, launch -- the
kernels are in codegen/lm_kernel.py."""
from __future__ import annotations

import math

import numpy as np

from dlgrad_amd.buffer import Buffer
from dlgrad_amd.codegen import lm_kernel as K
from dlgrad_amd.device import Device
from dlgrad_amd.dispatch import dispatcher
from dlgrad_amd.helpers import CustomOps
from dlgrad_amd.runtime.hip import DevicePtr, _addr, _PlanCache, _upload, alloc, field_offset, kernel, launch, launch_out, props

STREAM_BYTES = 1 << 28       # the Infinity Cache
# elements from which rotary positions bypass the caches.  Queries and keys with an addition in front of each and one of both behind, against the
# same through the caches: 16 x 128 x 4 heads of 32 (2^19 elements) 11.7 us, 11.4; 2 x 512 x 12 heads of 64 (1.5 2^20) 15.4, 15.8; 2 x 1024 18.5, 21.3; 4 x 1024
# 30.8, 32.5; 8 x 1024 54.6, 53.3; 16 x 1024 105.7, 106.8; 32 x 1024 223, 231.  Alone, from inputs that no cache holds: 2 x 1024 7.1, 8.3; 8 x 1024 19.7, 21.7.
ROTARY_STREAM_ELEMENTS = 1 << 20
EXACT_WHOLE = 1 << 24        # whole numbers up to here are exact in fp32
_rotary_plans: dict = _PlanCache()     # what a call looked at -> the launch that its checks ended in


def _on_device(what: str, **tensors) -> None:
    for name, t in tensors.items():
        if t is not None and (t.is_host_scalar or t.device is not Device.HIP):
            raise ValueError(f"{what}: {name} is not a tensor on the hip device")


class Cache8:
    """One layer of an 8-bit key/value cache in device memory: codes, scales, the fp32 tails and what each tail holds."""
    __slots__ = ("batch", "heads", "d", "width", "blocks", "layers", "kc", "vc", "scales", "tail_k", "tail_v", "marks", "wrote", "writers", "attenders")

    def __init__(self, batch: int, heads: int, d: int, blocks: int, layers: int, wrote: Buffer) -> None:
        """layers: how many of these a step reads one after the other.  wrote: rows of each sequence that the last write to any of them brought."""
        self.wrote = wrote
        self.batch, self.heads, self.d, self.blocks, self.layers = batch, heads, d, blocks, layers
        self.width = K.cache8_width(d)
        self.writers, self.attenders = _PlanCache(), _PlanCache()            # shape of a call -> the launch that its checks ended in
        n = batch * heads * blocks
        codes = n * K.CACHE8_BLOCK * self.width // 4                       # in units of 4 bytes, as everything is allocated
        self.kc, self.vc = alloc(codes), alloc(codes)                        # (a block is written whole before its first read)
        self.scales = Buffer.full((n, 2), 0.0, Device.HIP)
        # tails are read in whole blocks: columns beyond d, and rows not written yet, are zeros from the start
        self.tail_k, self.tail_v = (Buffer.full((2, batch * heads, K.CACHE8_BLOCK, self.width), 0.0, Device.HIP) for _ in range(2))
        self.marks = Buffer.full((batch * heads, 32), 0.0, Device.HIP)        # (two whole numbers of 32 bits at the front of each row, 0: nothing)

    @property
    def nbytes(self) -> int:
        """Bytes of codes, scales and tails (the marks are 128 more for each sequence and head)."""
        return self.kc.nbytes + self.vc.nbytes + self.scales.nbytes + self.tail_k.nbytes + self.tail_v.nbytes


class HIPLM:
    """Dispatch-table entries for Device.HIP."""

    @staticmethod
    def words(a: np.ndarray) -> Buffer:
        """A host array of 64-bit words in device memory, as a Buffer of twice as many floats that nothing does arithmetic on."""
        a = np.ascontiguousarray(a, dtype=np.uint64)
        p = alloc(2 * a.size)
        _upload(p.addr, a)
        return Buffer(p, (2 * a.size,), Device.HIP)

    # ---- rotary positions ------------------------------------------------------------------------
    @staticmethod
    def rotary_plan(sizes: list, n_words: int, rows: int, T: int, per: int, d: int, rot: int, half: bool, back: bool, gain: float,
                    n_positions: int, n_starts: int, inplace: bool):
        """The checks of a call that depend on sizes alone, and the launch of everything else.  sizes: one or two (elements, heads,
        pitch): `rows` rows of `heads` heads of d, `pitch` floats apart.  Row i is position i % T of sequence i // T // per.
        Returns run(pointer, second pointer, addresses of the frequencies, the positions and the starts) -> two pointers, or None where there
        is nothing to do."""
        if not 1 <= len(sizes) <= 2 or not 0 < rot <= d or rot % 2 or n_words != rot:
            raise ValueError(f"rotary: {len(sizes)} tensors, {rot} of {d} elements turned, {n_words // 2} frequencies")
        if rows == 0:
            return None
        if T < 1 or per < 1 or rows % (T * per) or T > EXACT_WHOLE:
            raise ValueError(f"rotary: {rows} rows are not whole sequences of {T}")
        batch = rows // (T * per)
        for numel, heads, pitch in sizes:
            if heads < 1 or pitch < heads * d or numel < (rows - 1) * pitch + heads * d:
                raise ValueError(f"rotary: {rows} rows of {heads} heads of {d} are not in a tensor of {numel} elements with rows {pitch} apart")
            if pitch >= 2 ** 32:
                raise ValueError(f"rotary: rows {pitch} elements apart exceed the kernel's 32-bit pitch")
        if n_positions not in (0, T, batch * T):
            raise ValueError(f"rotary: {n_positions} positions for {batch} sequences of {T}")
        if n_starts not in (0, 1, batch):
            raise ValueError(f"rotary: {n_starts} starts for {batch} sequences")
        two = len(sizes) - 1
        numel0, numel1 = rows * sizes[0][1] * d, rows * sizes[two][1] * d
        out_pitch = [p if inplace else h * d for _, h, p in sizes]
        unit = 8 if half else 4                                        # elements of a unit of pairs in 16-byte accesses
        wide = rot % unit == 0 and d % 4 == 0 and all(p % 4 == 0 for _, _, p in sizes)

        def grid(vec: bool) -> tuple:
            units = (rot // unit if vec else rot // 2) + (0 if inplace else (d - rot) // (4 if vec else 1))
            blocks = (max(rows * -(-h // K.ROTARY_HEADS) * units for _, h, _ in sizes) + 255) // 256
            if blocks >= 2 ** 31:
                raise ValueError(f"rotary: {rows} rows exceed the grid")
            return (blocks, 1, 1 + two)
        stream = not inplace and numel0 + two * numel1 >= ROTARY_STREAM_ELEMENTS

        def variant(vec: bool) -> list:
            v = [None, grid(vec), None]

            def load():
                v[0] = kernel(K.rotary_kernel, half, vec, stream and vec)
                return v[0]
            v[2] = load
            return v
        narrow = variant(False)
        first = variant(True) if wide else narrow
        tail = (rows, T, per, sizes[0][1], sizes[two][1], d, rot, sizes[0][2], sizes[two][2], out_pitch[0], out_pitch[two],
                T if n_positions == batch * T else 0, 1 if n_starts == batch else 0, int(back), float(gain))
        def run(x0: DevicePtr, x1: DevicePtr | None, table: int, pos: int, start: int) -> tuple:
            a0 = x0.addr
            a1 = x1.addr if two else a0
            y0 = x0 if inplace else alloc(numel0)
            y1 = y0 if not two else x1 if inplace else alloc(numel1)
            v = narrow if (a0 | a1) & 15 else first                  # (fresh blocks are aligned)
            k = v[0] or v[2]()
            launch(k, v[1], 256, a0, y0.addr, a1, y1.addr, table, pos, start, *tail)
            return y0, y1
        return run

    @staticmethod
    @dispatcher.register(CustomOps.ROTARY, Device.HIP)
    def rotary(parts: list, freq: Buffer, rows: int, T: int, per: int, d: int, rot: int, half: bool, back: bool, gain: float,
               positions: Buffer | None = None, start: Buffer | None = None, inplace: bool = False) -> list:
        """parts: one or two (Buffer, heads, pitch), see rotary_plan.  Returns the turned tensors' pointers (rows * heads * d floats
        each), or writes the parts themselves when `inplace`."""
        bufs = [p[0] for p in parts]
        key = (freq.numel, rows, T, per, d, rot, half, back, gain, inplace, *[(b.numel, h, p, b.device, b.ptr.__class__) for b, h, p in parts],
               None if positions is None else (positions.numel, positions.device, positions.ptr.__class__),
               None if start is None else (start.numel, start.device, start.ptr.__class__))
        plan = _rotary_plans.get(key, _rotary_plans)
        if plan is _rotary_plans:
            _on_device("rotary", positions=positions, start=start, **{f"x{i}": b for i, b in enumerate(bufs)})
            plan = _rotary_plans[key] = HIPLM.rotary_plan([(b.numel, h, p) for b, h, p in parts], freq.numel, rows, T, per, d, rot, half, back, gain,
                                                          0 if positions is None else positions.numel, 0 if start is None else start.numel, inplace)
        if plan is None:
            return [b.ptr if inplace else alloc(0) for b in bufs]
        return plan(bufs[0].ptr, bufs[-1].ptr, freq.ptr.addr, positions.ptr.addr if positions is not None else 0,
                    start.ptr.addr if start is not None else 0)[:len(parts)]

    # ---- the 8-bit cache ---------------------------------------------------------------------------
    @staticmethod
    def _cache8_lengths(what: str, c: Cache8, lengths: Buffer, counts: Buffer | None) -> None:
        _on_device(what, lengths=lengths, counts=counts)
        if lengths.numel != c.batch or (counts is not None and counts.numel != c.batch):
            raise ValueError(f"{what}: {lengths.numel} lengths and {'no' if counts is None else counts.numel} counts for {c.batch} sequences")

    @staticmethod
    def cache8_writer(c: Cache8, shape: tuple):
        """The checks of cache8_write that depend on the shape of the keys alone, and run(addresses of keys, values, lengths, counts)."""
        C = c.heads * c.d
        if len(shape) != 3 or shape[0] != c.batch or shape[2] != C:
            raise ValueError(f"cache8_write: keys {shape} for {c.batch} sequences of {c.heads} heads of {c.d}")
        T = shape[1]
        if T > c.blocks * K.CACHE8_BLOCK:
            raise ValueError(f"cache8_write: {T} tokens for a cache of {c.blocks * K.CACHE8_BLOCK}")
        if not T:
            return lambda ka, va, la, ca: None
        grid, wide, kernels = (-(-T // K.CACHE8_BLOCK), c.heads, c.batch), C % 4 == 0 and c.d % 4 == 0, [None, None]
        tail = (c.kc.addr, c.vc.addr, _addr(c.scales), _addr(c.tail_k), _addr(c.tail_v), _addr(c.marks), _addr(c.wrote), T, c.heads, c.d, c.blocks, C, C)

        def run(ka: int, va: int, la: int, ca: int) -> None:
            vec = wide and not (ka | va) & 15
            k = kernels[vec]
            if k is None:
                k = kernels[vec] = kernel(K.cache8_write_kernel, c.width, vec)
            # a call completes at most ceil(T / 64) blocks, the one it starts in among them
            launch(k, grid, K.CACHE8_WRITE_THREADS, ka, va, la, ca, *tail)
        return run

    @staticmethod
    @dispatcher.register(CustomOps.CACHE8_WRITE, Device.HIP)
    def cache8_write(cache: Cache8, k: Buffer, v: Buffer, lengths: Buffer, counts: Buffer | None = None) -> None:
        _on_device("cache8_write", k=k, v=v)
        HIPLM._cache8_lengths("cache8_write", cache, lengths, counts)
        if v.shape != k.shape:
            raise ValueError(f"cache8_write: keys {k.shape} and values {v.shape}")
        run = cache.writers.get(k.shape)
        if run is None:
            run = cache.writers[k.shape] = HIPLM.cache8_writer(cache, k.shape)
        run(_addr(k), _addr(v), _addr(lengths), 0 if counts is None else _addr(counts))

    @staticmethod
    def attend_tiles(rows: int, pairs: int, width: int, compute_units: int) -> int:
        """Tiles of 16 query rows that a wavefront of the 8-bit attention holds.  Two share the widening of the codes (4 x 12 heads of 64,
        512 rows after 4096 tokens: 79 us against 88; 8 x 12 heads, 1024 after 1024: 123 against 133) but halve the
        workgroups, of which there should be three for every compute unit (the same with 256 rows: 52 us against 47); heads wider
        than 64 have no registers for them (2 x 8 heads of 128, 512 after 2048: 52 us against 35).  Up to 16 rows are one tile
        (64 x 12 heads of 64 over 2000 tokens, 16 rows: 37 us against 45; 32 rows: 50 against 47)."""
        return 2 if width <= 64 and rows > 16 and pairs * -(-rows // 32) >= 3 * compute_units else 1

    @staticmethod
    def attend_waves(rows: int, blocks: int, width: int) -> int:
        """Wavefronts of a workgroup of the 8-bit attention.  With one tile of 16 query rows, eight halve the blocks that each goes through
        (16 x 12 heads of 64 over 4096 tokens: 20.9 us against 24.8 with four); heads wider than 64 fill the registers with four
        (4 x 8 heads of 128 over 8192: 24.7 us, 25.5 with eight), few blocks leave the others idle (1 x 12 heads of 64, two blocks: 5.0 us with four, 5.3
        with eight; four: 5.95, 5.75; six: 6.1, 5.8), and rows that two tiles share have workgroups enough (64 x 12 heads of 64 over 2000 tokens,
        32 rows: 47 us with four, 61 with eight).  It does not look at the batch: with more workgroups than compute units four are ahead for short
        caches (40 x 12 heads of 64 over 738 tokens: 13.1 us, 14.1 with eight)."""
        return 8 if rows <= 16 and width <= 64 and blocks > 4 else 4

    @staticmethod
    def attend_streams(c: Cache8, tiles: int) -> bool:
        """Whether the codes bypass the caches: they are read once by a call, and the cache as a whole, all layers of it, is larger than
        the 256 MiB that a later step might find them in (16 x 8 heads of 128 over 32768 tokens, 1.07 GB: 168 us against 193;
        4 x 8 heads, 0.27 GB: 53 against 59; 16 x 12 heads of 64 over 8192, 0.2 GB, again and again: 40.4 us against 35.7)."""
        return tiles == 1 and c.layers * (c.kc.nbytes + c.vc.nbytes) > STREAM_BYTES

    @staticmethod
    def attend_splits(groups: int, blocks: int, waves: int, compute_units: int) -> int:
        """Into how many parts the blocks of a sequence are cut when one part makes `groups` workgroups of `waves` wavefronts.  A wavefront
        takes 0.8 us for a block when there are few, the second launch that joins the parts 3.5 us and 0.1 us for each:
        sqrt(blocks / 2) parts from 8 blocks a wavefront on (1 x 12 heads of 64 over 4096 tokens: 17.0 us with one part, 11.3 with 4, 11.1 with
        8, 12.5 with 16; 1 x 8 heads of 128 over 32768: 35 us with 8, 30 with 16, 34 with 32), and no more than
        eight wavefronts for every compute unit (16 x 12 heads of 64 over 4096: 19.4 us with one part, 25.0 with 2, 29.6 with 8).  The length is
        device data; the capacity stands for it."""
        if blocks < 8 * waves:
            return 1
        return max(1, min(8 * compute_units // (waves * max(groups, 1)), math.isqrt(blocks // 2), K.CACHE8_MAX_SPLITS))

    @staticmethod
    def cache8_attender(c: Cache8, shape: tuple):
        """The checks of cache8_attend that depend on the shape of the queries alone, and run(addresses of queries, lengths, counts,
        scale) -> pointer."""
        if len(shape) != 3 or shape[0] != c.batch or shape[2] == 0 or shape[2] % (c.heads * c.d):
            raise ValueError(f"cache8_attend: queries {shape} for {c.batch} sequences with {c.heads} key heads of {c.d}")
        T, group = shape[1], shape[2] // (c.heads * c.d)
        if T > c.blocks * K.CACHE8_BLOCK:
            raise ValueError(f"cache8_attend: {T} positions for a cache of {c.blocks * K.CACHE8_BLOCK}")
        rows, pairs, numel = T * group, c.batch * c.heads, shape[0] * T * shape[2]
        if not rows:
            return lambda qa, la, ca, scale: alloc(0)
        nq = HIPLM.attend_tiles(rows, pairs, c.width, props()["compute_units"])
        tiles = -(-rows // (16 * nq))
        waves = HIPLM.attend_waves(rows, c.blocks, c.width)
        splits = HIPLM.attend_splits(pairs * tiles, c.blocks, waves, props()["compute_units"])
        grid = pairs * tiles * splits
        if grid >= 2 ** 31 or pairs * rows >= 2 ** 31:
            raise ValueError(f"cache8_attend: {pairs} heads of {rows} query rows exceed the grid")
        k, join = kernel(K.cache8_attend_kernel, c.width, nq, waves, HIPLM.attend_streams(c, tiles)), kernel(K.cache8_join_kernel, c.width) if splits > 1 else None
        held = (c.kc.addr, c.vc.addr, _addr(c.scales), _addr(c.tail_k), _addr(c.tail_v), _addr(c.marks), _addr(c.wrote))
        sizes = (c.batch, T, c.heads, group, c.d, c.blocks, tiles, splits)
        wide = c.d % 4 == 0                                              # (then the rows of the queries are whole 16-byte items)
        n_part, join_grid, join_sizes = pairs * rows * splits * (c.width + 2), (pairs * rows + 3) // 4, (pairs * rows, T, c.heads, group, c.d, splits)

        def run(qa: int, la: int, ca: int, scale: float) -> DevicePtr:
            y = alloc(numel)
            if join is None:
                launch(k, grid, 64 * waves, qa, *held, la, ca, y.addr, 0, *sizes, int(wide and not qa & 15), scale)
                return y
            part = alloc(n_part)
            launch(k, grid, 64 * waves, qa, *held, la, ca, y.addr, part.addr, *sizes, int(wide and not qa & 15), scale)
            launch(join, join_grid, 256, part.addr, y.addr, *join_sizes)
            return y
        return run

    @staticmethod
    @dispatcher.register(CustomOps.CACHE8_ATTEND, Device.HIP)
    def cache8_attend(cache: Cache8, q: Buffer, scale: float, lengths: Buffer, counts: Buffer | None = None) -> DevicePtr:
        _on_device("cache8_attend", q=q)
        HIPLM._cache8_lengths("cache8_attend", cache, lengths, counts)
        run = cache.attenders.get(q.shape)
        if run is None:
            run = cache.attenders[q.shape] = HIPLM.cache8_attender(cache, q.shape)
        return run(_addr(q), _addr(lengths), 0 if counts is None else _addr(counts), float(scale))

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
                   _addr(c.tail_k), _addr(c.tail_v), _addr(c.marks), _addr(c.wrote), _addr(lengths), _addr(counts) if counts is not None else 0, k.addr, v.addr,
                   n, c.heads, c.d, c.blocks, extra)
        return k, v

    @staticmethod
    @dispatcher.register(CustomOps.CACHE8_ADVANCE, Device.HIP)
    def cache8_advance(cache: Cache8, lengths: Buffer, by: "Buffer | int", reset: bool = False) -> None:
        """by: rows of every sequence, or a number for each."""
        counts = by if isinstance(by, Buffer) else None
        HIPLM._cache8_lengths("cache8_advance", cache, lengths, counts)
        if counts is None and not 0 <= by < 2 ** 32:
            raise ValueError(f"cache8_advance: {by} rows")
        launch(kernel(K.cache8_advance_kernel), -(-cache.batch // 256), 256, _addr(lengths), 0 if counts is None else _addr(counts), _addr(cache.wrote),
               cache.batch, cache.blocks * K.CACHE8_BLOCK, by if counts is None else 0, int(reset))

    # ---- logits ----------------------------------------------------------------------------------------
    @staticmethod
    def adjust_items(B: int, V: int, compute_units: int) -> int:
        """Logits per thread of the adjustment: every block walks its row's whole history, so long slices of the vocabulary save
        walks -- as long as there are blocks enough, four for every compute unit with 16 (32 x 128256 logits, 4000 said, 4 a unit: 10.1 us with 16,
        10.4 with 8; 256 x 128256, 32 a unit: 47.3, 48.7; 16 x 128256, 300 said, 2 a unit: 7.0, 6.7; 64 x 50257, 3.3 a unit: 12.3, 11.0), two with 8
        (32 x 50304, 3.1 a unit: 6.6 us with 8, 7.3 with 4; 8 x 50304, 0.8 a unit: 5.1, 4.6)."""
        for items, blocks in ((16, 4), (8, 2)):
            if B * -(-V // (256 * items)) >= blocks * compute_units:
                return items
        return 4

    @staticmethod
    @dispatcher.register(CustomOps.ADJUST_LOGITS, Device.HIP)
    def logits_plan(logits: Buffer, history: Buffer | None, lengths: Buffer | None, penalties: tuple, bias: Buffer | None, hidden: Buffer | None):
        """The checks of a call, which depend on shapes alone, and run(the same arguments) -> pointer for every call that agrees in them.
        logits (B, V); history (B, L); lengths B; penalties: (repetition, presence, frequency), each a float or a Buffer of B;
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
        if B > 65535:
            raise ValueError(f"adjust_logits: {B} rows, at most 65535 in one call")
        items = HIPLM.adjust_items(B, V, props()["compute_units"])
        if B * V == 0:
            return lambda *given: alloc(0)
        wide, grid, kernels, out_at = V % 4 == 0, (-(-V // (256 * items)), B, 1), [None, None], field_offset("@" + "P" * 6, 5)
        sizes = (V, 0 if history is None else history.shape[1], V if bias is not None and bias.numel == B * V else 0,
                 V if hidden is not None and hidden.numel == B * V else 0)

        def run(logits, history, lengths, penalties, bias, hidden) -> DevicePtr:
            la, ba, ha = logits.ptr.addr, 0 if bias is None else bias.ptr.addr, 0 if hidden is None else hidden.ptr.addr
            vec = wide and not (la | ba | ha) & 15
            k = kernels[vec]
            if k is None:
                k = kernels[vec] = kernel(K.adjust_logits_kernel, items, vec, sizes[1] <= K.LOGITS_PACKED_L)
            r, p, f = penalties
            ra = pa = fa = 0
            if isinstance(r, Buffer):
                ra, r = r.ptr.addr, 1.0
            if isinstance(p, Buffer):
                pa, p = p.ptr.addr, 0.0
            if isinstance(f, Buffer):
                fa, f = f.ptr.addr, 0.0
            return launch_out(k, grid, 256, out_at, B * V, la, 0 if history is None else history.ptr.addr, 0 if lengths is None else lengths.ptr.addr,
                              ba, ha, 0, ra, pa, fa, *sizes, r, p, f)
        return run
