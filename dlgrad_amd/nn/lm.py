"""Operators of language models beside the ones in nn/__init__.py: rotary positions (instead of a learned position
table), a key/value cache held in 8 bits with the attention that reads it (instead of fp32 stores and
cached_attention), and the adjustment of logits before a token is chosen (in front of decode_append and
decode_sample)."""
from __future__ import annotations

import math

import numpy as np

import dlgrad_amd.nn as _nn
from dlgrad_amd import ops
from dlgrad_amd.buffer import Buffer, HostScalar, _dispatch_table
from dlgrad_amd.device import Device, as_device
from dlgrad_amd.helpers import CustomOps
from dlgrad_amd.tensor import Tensor


def _result(buf: Buffer) -> Tensor:
    """A tensor without a tape around a buffer (what Tensor(buf) makes)."""
    t = Tensor.__new__(Tensor)
    t.data, t.requires_grad, t._ctx, t.grad = buf, False, None, None
    return t


def _no_tape(what: str) -> None:
    """Refuses a call, made with a tensor that requires a gradient, whose result would silently stop that gradient."""
    if not _nn._inference_depth:
        raise ValueError(f"{what} has no gradient: call it inside nn.inference(), or with detach()ed tensors")


def rotary_frequencies(rotated: int, base: float = 10000.0, scaling: str | None = None, factor: float = 1.0,
                       trained: int | None = None) -> tuple[np.ndarray, float]:
    """(radians per position of each of the rotated / 2 pairs in float64, the factor of the turned elements).

    Pair i turns by base^(-2 i / rotated) per position.  For contexts longer than the trained ones by `factor`:
      "linear"  every frequency over factor;
      "base"    base * factor^(rotated / (rotated - 2)) as the base: the fastest pair keeps its frequency and the slowest is
                slowed by factor;
      "parts"   a pair that makes 32 turns or more within `trained` positions keeps its frequency, one that makes at most one
                is slowed by factor, those between are mixed in proportion; the elements are multiplied by 0.1 ln(factor) + 1."""
    if scaling not in (None, "linear", "base", "parts"):
        raise ValueError(f"rotary: no scaling {scaling!r} (None, 'linear', 'base' or 'parts')")
    if rotated < 2 or rotated % 2 or not base > 0 or not math.isfinite(base) or not factor > 0 or not math.isfinite(factor):
        raise ValueError(f"rotary: {rotated} elements, base {base}, factor {factor}")
    if scaling is None and factor != 1.0:
        raise ValueError(f"rotary: a factor of {factor} and no scaling to take it")
    if scaling == "base":
        if rotated == 2:
            raise ValueError("rotary: one pair has no slowest one apart from the fastest: scaling 'base' needs four elements")
        base = base * factor ** (rotated / (rotated - 2))
    f = float(base) ** (-2.0 * np.arange(rotated // 2, dtype=np.float64) / rotated)
    if scaling == "linear":
        return f / factor, 1.0
    if scaling == "parts":
        if trained is None or trained < 1 or factor < 1:
            raise ValueError("rotary: scaling 'parts' needs the trained length and a factor of at least 1")
        keep = np.clip((trained * f / (2 * math.pi) - 1.0) / 31.0, 0.0, 1.0)
        return keep * f + (1.0 - keep) * (f / factor), 0.1 * math.log(factor) + 1.0
    return f, 1.0


def _copied(b: Buffer | None) -> Buffer | None:
    """A copy on the hip device."""
    if b is None:
        return None
    from dlgrad_amd.runtime.hip import alloc
    own = Buffer.fresh(alloc(b.numel), b.shape, Device.HIP)
    own.copy_(b)
    return own


def _on_hip(b: Buffer) -> bool:
    return b.device is Device.HIP and b.ptr.__class__ is not HostScalar


class Rotary:
    """Rotary positions for heads of `head_dim` elements, the first `rotated` of which turn (all by default):

        rope = nn.Rotary(64)
        q, k = rope.pair(q, k, n_head)                       # (B, T, n_head * 64) projections, positions 0 .. T - 1

    layout "half": pair i is elements i and i + rotated / 2 of a head; "interleaved": 2 i and 2 i + 1.  base, scaling,
    factor, trained: see rotary_frequencies.  Positions are whole numbers of magnitude up to 2^24; angles are exact
    modulo one turn at any of them (a fixed-point product, lm_kernel.rotary_kernel)."""

    def __init__(self, head_dim: int, rotated: int | None = None, base: float = 10000.0, layout: str = "half", scaling: str | None = None,
                 factor: float = 1.0, trained: int | None = None, device: Device | str = "hip") -> None:
        rotated = head_dim if rotated is None else rotated
        if layout not in ("half", "interleaved"):
            raise ValueError(f"rotary: no layout {layout!r} ('half' or 'interleaved')")
        if not 0 < rotated <= head_dim:
            raise ValueError(f"rotary: {rotated} of {head_dim} elements cannot turn")
        device = as_device(device)
        if device is None:
            raise ValueError("rotary: no such device")
        self.head_dim, self.rotated, self.half = head_dim, rotated, layout == "half"
        self.frequencies, self.gain = rotary_frequencies(rotated, base, scaling, factor, trained)
        self._words, self._plans = None, {}
        if device is Device.HIP:
            self._table()

    def _table(self) -> Buffer:
        """The frequencies in turns per position as fractions of 2^64, on the device."""
        if self._words is None:
            from dlgrad_amd.runtime.hip import capturing
            from dlgrad_amd.runtime.hip_lm import HIPLM
            if capturing():
                raise RuntimeError("rotary: made for another device, its table cannot be uploaded inside a capture")
            turns = [int(round(float(f) / (2 * math.pi) % 1.0 * 2.0 ** 64)) % 2 ** 64 for f in self.frequencies]
            self._words = HIPLM.words(np.array(turns, dtype=np.uint64))
        return self._words

    def _geometry(self, x, n_head: int) -> tuple[int, int, int]:
        """(rows, T, rows of T per sequence): x is (B, T, n_head * d), or (B, heads, T, d) with n_head = 1."""
        if x.ndim not in (3, 4) or n_head < 1 or x.shape[-1] != n_head * self.head_dim or (x.ndim == 4 and n_head != 1):
            raise ValueError(f"rotary: {x.shape} is neither (B, T, {n_head} * {self.head_dim}) nor (B, heads, T, {self.head_dim}) with n_head = 1")
        return x.numel // x.shape[-1] if x.shape[-1] else 0, x.shape[-2], x.shape[1] if x.ndim == 4 else 1

    def __call__(self, x: Tensor, n_head: int = 1, positions: Tensor | None = None, start: Tensor | None = None, transpose: bool = False) -> Tensor:
        """x, (B, T, n_head * head_dim) or (B, heads, T, head_dim), turned by its positions: `positions` (T,) or (B, T), or 0 .. T - 1
        without them, plus `start` (one number, or one per sequence: a device tensor, so a captured step may move it).
        transpose: the transposed map, which turns the other way -- it takes a gradient of the result to one of x."""
        xd, p, s0 = x.data, None if positions is None else positions.data, None if start is None else start.data
        key = (xd.shape, n_head, None if p is None else p.shape, None if s0 is None else s0.shape, transpose)
        plan = self._plans.get(key) if ops.FUSED and not x.requires_grad else None
        if plan is None or not (_on_hip(xd) and (p is None or _on_hip(p)) and (s0 is None or _on_hip(s0))):
            out = self._turn([x], [n_head], positions, start, transpose)
            self._remember(key, [x], [n_head], p, s0, transpose)
            return out[0]
        return _result(xd._like(plan(xd.ptr, None, self._words.ptr.addr, 0 if p is None else p.ptr.addr, 0 if s0 is None else s0.ptr.addr)[0]))

    def pair(self, q: Tensor, k: Tensor, n_head: int, n_kv_head: int | None = None, positions: Tensor | None = None, start: Tensor | None = None,
             transpose: bool = False) -> tuple[Tensor, Tensor]:
        """(self(q), self(k)) with n_head and n_kv_head heads, in one launch on the hip device."""
        qd, kd = q.data, k.data
        p, s0 = None if positions is None else positions.data, None if start is None else start.data
        key = (qd.shape, kd.shape, n_head, n_kv_head, None if p is None else p.shape, None if s0 is None else s0.shape, transpose)
        plan = self._plans.get(key) if ops.FUSED and not (q.requires_grad or k.requires_grad) else None
        if plan is None or not (_on_hip(qd) and _on_hip(kd) and (p is None or _on_hip(p)) and (s0 is None or _on_hip(s0))):
            heads = [n_head, n_head if n_kv_head is None else n_kv_head]
            out = self._turn([q, k], heads, positions, start, transpose)
            self._remember(key, [q, k], heads, p, s0, transpose)
            return out[0], out[1]
        y0, y1 = plan(qd.ptr, kd.ptr, self._words.ptr.addr, 0 if p is None else p.ptr.addr, 0 if s0 is None else s0.ptr.addr)
        return _result(qd._like(y0)), _result(kd._like(y1))

    def _remember(self, key: tuple, xs: list, heads: list, p: Buffer | None, s0: Buffer | None, back: bool) -> None:
        """Keeps the launch of a call that has just passed its checks for calls of the same shapes."""
        shapes = [self._geometry(x, h) for x, h in zip(xs, heads)]
        if not ops.FUSED or not _on_hip(xs[0].data) or shapes[0][2] != shapes[-1][2] or key in self._plans:
            return
        from dlgrad_amd.runtime.hip_lm import HIPLM
        if len(self._plans) >= 1024:                                   # (a workload whose shapes never repeat)
            self._plans.clear()
        plan = HIPLM.rotary_plan([(x.data.numel, h, h * self.head_dim) for x, h in zip(xs, heads)], self._words.numel, *shapes[0], self.head_dim,
                                 self.rotated, self.half, bool(back), self.gain, 0 if p is None else p.numel, 0 if s0 is None else s0.numel, False)
        if plan is not None:
            self._plans[key] = plan

    def _turn(self, xs: list, heads: list, positions, start, back: bool) -> list:
        shapes = self._check(xs, heads, positions, start)
        if not ops.FUSED or xs[0].data.device is not Device.HIP:
            return [self._composed(x, h, s, positions, start, back) for x, h, s in zip(xs, heads, shapes)]
        back, p, s0 = bool(back), None if positions is None else positions.data, None if start is None else start.data
        d = self.head_dim
        if len(xs) == 1 or shapes[0][2] == shapes[1][2]:                # rows map to sequences alike: one launch
            out = self._launch([(x.data, h, h * d) for x, h in zip(xs, heads)], shapes[0], back, p, s0)
        else:
            out = [self._launch([(x.data, h, h * d)], s, back, p, s0)[0] for x, h, s in zip(xs, heads, shapes)]
        if any(x.requires_grad for x in xs):                            # (the backward pass turns by the angles of this call, wherever the tensors have moved by then)
            p, s0 = _copied(p), _copied(s0)
        return [ops.Rotary.execute(x, turned=y, rope=self, n_head=h, geometry=s, positions=p, start=s0, back=back) if x.requires_grad else Tensor(y)
                for x, y, h, s in zip(xs, out, heads, shapes)]

    def _check(self, xs: list, heads: list, positions, start) -> list:
        """Refuses shapes and devices that do not fit together; the geometry of each tensor."""
        shapes = [self._geometry(x, h) for x, h in zip(xs, heads)]
        x = xs[0]
        if any(t.device is not x.device for t in xs[1:] + [t for t in (positions, start) if t is not None]):
            raise ValueError("rotary: the tensors are on different devices")
        if len({(x.shape[0], s[1]) for x, s in zip(xs, shapes)}) > 1:
            raise ValueError(f"rotary: {' and '.join(str(x.shape) for x in xs)} have different sequences")
        B, T = x.shape[0], shapes[0][1]
        if positions is not None and positions.shape not in ((T,), (1, T), (B, T)):
            raise ValueError(f"rotary: positions {positions.shape} for {B} sequences of {T}")
        if start is not None and start.numel != 1 and start.shape not in ((B,), (B, 1)):
            raise ValueError(f"rotary: starts {start.shape} for {B} sequences")
        return shapes

    def _launch(self, parts: list, geometry: tuple, back: bool, positions: Buffer | None, start: Buffer | None, inplace: bool = False) -> list:
        rows, T, per = geometry
        return Buffer.rotary(parts, freq=self._words or self._table(), rows=rows, T=T, per=per, d=self.head_dim, rot=self.rotated, half=self.half,
                             back=back, gain=self.gain, positions=positions, start=start, inplace=inplace)

    def turn_back(self, g: Buffer, n_head: int, geometry: tuple, positions: Buffer | None, start: Buffer | None, back: bool) -> Buffer:
        """The transposed map of a gradient."""
        return self._launch([(g, n_head, n_head * self.head_dim)], geometry, not back, positions, start)[0]

    def turn_qkv_(self, qkv: Buffer, n_head: int, back: bool = False) -> None:
        """In place, positions 0 .. T - 1: the query and key heads of a (B, T, 3 C) projection, C = n_head * head_dim."""
        B, T, C3 = qkv.shape
        if C3 != 3 * n_head * self.head_dim:
            raise ValueError(f"rotary: a projection {qkv.shape} for {n_head} heads of {self.head_dim}")
        self._launch([(qkv, 2 * n_head, C3)], (B * T, T, 1), back, None, None, inplace=True)

    def _composed(self, x: Tensor, n_head: int, geometry: tuple, positions, start, back: bool) -> Tensor:
        """The same as x * cos + (x @ J) * sin with J the signed permutation that takes (a, b) of a pair to (-b, a): existing
        ops, with the angles computed on the host."""
        B, T, d, r = x.shape[0], geometry[1], self.head_dim, self.rotated
        p = np.arange(T, dtype=np.float64)[None] if positions is None else np.trunc(positions.numpy().astype(np.float64)).reshape(-1, T)
        if start is not None:
            p = p + np.trunc(start.numpy().astype(np.float64)).reshape(-1, 1)
        w = p[:, :, None] * self.frequencies
        first, second = (np.arange(r // 2), np.arange(r // 2) + r // 2) if self.half else (2 * np.arange(r // 2), 2 * np.arange(r // 2) + 1)
        cos, sin = np.ones(p.shape + (d,)), np.zeros(p.shape + (d,))
        for at in (first, second):
            cos[..., at], sin[..., at] = self.gain * np.cos(w), self.gain * np.sin(w) * (-1.0 if back else 1.0)
        J = np.zeros((d, d), np.float32)
        J[second, first], J[first, second] = -1.0, 1.0
        shape = (p.shape[0], 1, T, d) if x.ndim == 4 else (p.shape[0], T, 1, d)
        cos, sin = (Tensor(np.ascontiguousarray(t.reshape(shape), dtype=np.float32), device=x.device) for t in (cos, sin))
        h = x if x.ndim == 4 else x.reshape((B, T, n_head, d))
        y = h * cos + (h @ Tensor(J, device=x.device)) * sin
        return y.reshape(x.shape)


class QuantizedKVCache:
    """The keys and values of every position so far, in 8 bits with a scale for each block of 64 tokens and head; for inference.

        cache = nn.QuantizedKVCache(batch, capacity, n_kv_head, head_dim, layers=n_layer)
        cache.write(k, v, layer)              # (B, T, n_kv_head * head_dim): the new positions' keys and values
        y = cache.attend(q, scale, layer)     # (B, T, n_head * head_dim): they attend to everything before them and themselves
        cache.advance(T)                      # once all layers have done so

    A block is quantised when it is full: code = x / scale to the nearest whole number in -127 .. 127 with scale = max |x| / 127.
    The tokens of the block that is not full are kept as they came, so what is held depends on the tokens and not on
    the calls that brought them.  Memory: 2 * head_dim bytes a token and key head (head_dim rounded up to a multiple of 32), where two fp32
    stores take 8, and for each sequence and key head two blocks of fp32 rows, as much as 512 tokens: more than fp32 stores for a capacity
    of 128 tokens (125 %), less from 192 on (92 %), 38 % of them at 1024 and 25.5 % at 32768; heads of 40 take 60 and 41 %, heads of 16 51 % at 32768.

    lengths (B, 1), tokens held per sequence, is a device tensor (one of the caller's if given), so a captured step works at
    any length.  counts (B, 1): how many of the T rows of each sequence are tokens (a padded batch); the rest is neither
    written nor seen, and their rows of the result are zeros.  Rows that do not fit into the capacity (rounded up to whole blocks) are
    dropped the same way.  Until advance(), a write of at most 64 rows may be repeated or replaced, and advance() may be given
    less than was written.  After a longer one a sequence goes on from all that was written or from a whole block of it, and it can be
    repeated where the sequence holds whole blocks: the tokens of any other block that is opened again are gone, and every result
    that sees it is NaN (a batch of padded prompts therefore gives write() its counts).  A row with a NaN or an infinity makes
    every result that sees its block, once that is full, or itself, before, NaN.  Values are to stay below 2^88 in
    magnitude.  Results carry no tape.

    Query heads share key heads in order: query heads h * G .. h * G + G - 1 read key head h, G = n_head / n_kv_head."""

    BLOCK = 64

    def __init__(self, batch: int, capacity: int, n_kv_head: int, head_dim: int, layers: int = 1, device: Device | str = "hip",
                 lengths: Tensor | None = None) -> None:
        if as_device(device) is not Device.HIP:
            raise ValueError("QuantizedKVCache is provided on the hip device")
        from dlgrad_amd.codegen.lm_kernel import CACHE8_BLOCK, CACHE8_MAX_D
        from dlgrad_amd.runtime.hip_lm import EXACT_WHOLE, Cache8
        assert CACHE8_BLOCK == self.BLOCK
        if not (0 < batch <= 65535 and 0 < n_kv_head <= 65535 and 0 < head_dim <= CACHE8_MAX_D and layers > 0 and 0 < capacity <= EXACT_WHOLE):
            raise ValueError(f"QuantizedKVCache: {layers} layers, {batch} sequences of {capacity} tokens, {n_kv_head} key heads of {head_dim} "
                             f"(heads of at most {CACHE8_MAX_D}, at most {EXACT_WHOLE} tokens)")
        if lengths is not None and (lengths.device is not Device.HIP or lengths.numel != batch or lengths.data.is_host_scalar):
            raise ValueError(f"QuantizedKVCache: lengths {lengths.shape} for {batch} sequences")
        self.batch, self.n_kv_head, self.head_dim = batch, n_kv_head, head_dim
        blocks = -(-capacity // self.BLOCK)
        self.capacity = blocks * self.BLOCK
        self.lengths = Tensor.full((batch, 1), 0.0, device="hip") if lengths is None else lengths
        wrote = Buffer.full((batch, 1), 0.0, Device.HIP)                        # (whole numbers of 32 bits)
        self.layers = [Cache8(batch, n_kv_head, head_dim, blocks, layers, wrote) for _ in range(layers)]
        self._most = 0                                                          # rows of the longest write so far

    @property
    def nbytes(self) -> int:
        return sum(c.nbytes for c in self.layers)

    def _run(self, op, layer: int, counts: Tensor | None, **kw):
        if not 0 <= layer < len(self.layers):
            raise IndexError(f"layer {layer} of a cache of {len(self.layers)}")
        if counts is not None:
            if counts.__class__ is not Tensor:
                raise TypeError("counts is a tensor with a number per sequence")
            counts = counts.data
        return _dispatch_table[(op, Device.HIP)](cache=self.layers[layer], lengths=self.lengths.data, counts=counts, **kw)

    def _sized(self, counts: Tensor | None) -> bool:
        """Whether the lengths and counts of a call are what the launch of an earlier call may read."""
        n = self.lengths.data
        if n.numel != self.batch or n.device is not Device.HIP or n.ptr.__class__ is HostScalar:
            return False
        return counts is None or (counts.__class__ is Tensor and counts.data.numel == self.batch and _on_hip(counts.data))

    def write(self, k: Tensor, v: Tensor, layer: int = 0, counts: Tensor | None = None) -> None:
        """k, v (B, T, n_kv_head * head_dim): keys and values of positions lengths[b] .. of each sequence."""
        if k.requires_grad or v.requires_grad:
            _no_tape("QuantizedKVCache.write")
        kd, vd = k.data, v.data
        run = self.layers[layer].writers.get(kd.shape) if 0 <= layer < len(self.layers) else None
        if run is not None and kd.shape == vd.shape and _on_hip(kd) and _on_hip(vd) and self._sized(counts):
            run(kd.ptr.addr, vd.ptr.addr, self.lengths.data.ptr.addr, 0 if counts is None else counts.data.ptr.addr)
        else:
            self._run(CustomOps.CACHE8_WRITE, layer, counts, k=kd, v=vd)
            self._most = max(self._most, kd.shape[1])

    def attend(self, q: Tensor, scale: float | None = None, layer: int = 0, counts: Tensor | None = None) -> Tensor:
        """q (B, T, n_head * head_dim): the queries of positions lengths[b] .., whose keys and values write() has stored; each sees
        the positions up to its own.  Rows beyond those that the last write brought, its counts included, are zeros.  scale: of the scores, head_dim ** -0.5 without one."""
        if q.requires_grad:
            _no_tape("QuantizedKVCache.attend")
        scale = self.head_dim ** -0.5 if scale is None else float(scale)
        qd = q.data
        run = self.layers[layer].attenders.get(qd.shape) if 0 <= layer < len(self.layers) else None
        if run is not None and _on_hip(qd) and self._sized(counts):
            y = run(qd.ptr.addr, self.lengths.data.ptr.addr, 0 if counts is None else counts.data.ptr.addr, scale)
        else:
            y = self._run(CustomOps.CACHE8_ATTEND, layer, counts, q=qd, scale=scale)
        return _result(Buffer.fresh(y, qd.shape, Device.HIP))

    def read(self, n: int, layer: int = 0, new: int = 0, counts: Tensor | None = None) -> tuple[Tensor, Tensor]:
        """(k, v), both (B, n, n_kv_head * head_dim): the values that the first n positions stand for, zeros where a sequence is
        shorter.  new, or counts: rows that were written since the last advance() and belong to it, as many as there are."""
        k, v = self._run(CustomOps.CACHE8_READ, layer, counts, n=int(n), extra=self.capacity if counts is not None else int(new))
        shape = (self.batch, int(n), self.n_kv_head * self.head_dim)
        return _result(Buffer.fresh(k, shape, Device.HIP)), _result(Buffer.fresh(v, shape, Device.HIP))

    def advance(self, n: "int | Tensor") -> None:
        """The rows written become part of the sequences: n of each, or n (B, 1) of them, taken as write() takes its counts.  A sequence goes on
        by no more rows than the last write brought it, and never back."""
        if isinstance(n, Tensor):
            if n.numel != self.batch or n.device is not Device.HIP or n.data.is_host_scalar:
                raise ValueError(f"advance: counts {n.shape} for {self.batch} sequences")
            by = n.data
        elif not 0 <= n <= self._most or n != int(n):
            raise ValueError(f"advance: {n} tokens after writes of at most {self._most} (a cache does not go back; see reset())")
        else:
            by = int(n)
        self._move(by)

    def reset(self) -> None:
        """Forgets every token."""
        self._move(0, reset=True)

    def _move(self, by: "Buffer | int", reset: bool = False) -> None:
        self.lengths.data._writable("advance")
        _dispatch_table[(CustomOps.CACHE8_ADVANCE, Device.HIP)](cache=self.layers[0], lengths=self.lengths.data, by=by, reset=reset)


_adjust_plans: dict = {}       # shapes and numbers that _check_adjust has let through -> the launch


def _check_adjust(logits, history, lengths, repetition, presence, frequency, bias, hidden) -> None:
    if logits.ndim != 2:
        raise ValueError(f"adjust_logits: logits {logits.shape} are not (B, V)")
    for name, p in (("repetition", repetition), ("presence", presence), ("frequency", frequency)):
        if not isinstance(p, Tensor) and not (1e-38 if name == "repetition" else -3.4e38) <= p <= 3.4e38:      # (what fp32 holds, not a denormal)
            raise ValueError(f"adjust_logits: {name} = {p}")
    given = [t for t in (history, lengths, repetition, presence, frequency, bias, hidden) if isinstance(t, Tensor)]
    if any(t.device is not logits.device or t.data.is_host_scalar for t in given):
        raise ValueError("adjust_logits: the tensors are on different devices")
    B, V = logits.shape
    if history is not None and (history.ndim != 2 or history.shape[0] != B):
        raise ValueError(f"adjust_logits: a history {history.shape} for {B} rows")
    if lengths is not None and (history is None or lengths.numel != B):
        raise ValueError(f"adjust_logits: {lengths.numel} lengths for {'no history' if history is None else f'{B} rows'}")
    for name, t in (("bias", bias), ("hidden", hidden)):
        if t is not None and (t.shape[-1:] != (V,) or t.numel not in (V, B * V)):
            raise ValueError(f"adjust_logits: {name} {t.shape} for logits {logits.shape}")
    for name, p in (("repetition", repetition), ("presence", presence), ("frequency", frequency)):
        if isinstance(p, Tensor) and p.numel != B:
            raise ValueError(f"adjust_logits: {p.numel} values of {name} for {B} rows")


def adjust_logits(logits: Tensor, history: Tensor | None = None, lengths: Tensor | None = None, repetition: "float | Tensor" = 1.0,
                  presence: "float | Tensor" = 0.0, frequency: "float | Tensor" = 0.0, bias: Tensor | None = None,
                  hidden: Tensor | None = None) -> Tensor:
    """logits (B, V) before a token is chosen from them (decode_append, decode_sample, argmax): a new tensor without a tape.

    history (B, L): token ids said so far, the first lengths[b] of each row (all without lengths); ids outside [0, V) count for
    nothing.  A token that occurs c > 0 times there becomes x / repetition if x > 0 and x * repetition otherwise, less
    presence + frequency * c; the three are numbers, or tensors with one per row (taken as they are).  Then bias, (V,) or
    (B, V), is added, and tokens that hidden, (V,) or (B, V), marks (> 0: a grammar's mask) become -inf whatever they were; a row
    may be hidden whole.  One launch on the hip device; elsewhere on the host, from the downloaded logits."""
    for t in (logits, repetition, presence, frequency, bias):
        if t.__class__ is Tensor and t.requires_grad:
            _no_tape("adjust_logits")
    x, h, n = logits.data, None if history is None else history.data, None if lengths is None else lengths.data
    b, m = None if bias is None else bias.data, None if hidden is None else hidden.data
    r, p, f = (t.data if t.__class__ is Tensor else t for t in (repetition, presence, frequency))
    given = (h, n, b, m, r, p, f)
    key = (x.shape, *[(t.shape, t.device, t.ptr.__class__) if isinstance(t, Buffer) else t for t in given])
    plan = _adjust_plans.get(key) if ops.FUSED and _on_hip(x) else None
    if plan is not None:
        return _result(x._like(plan(x, h, n, (r, p, f), b, m)))
    _check_adjust(logits, history, lengths, repetition, presence, frequency, bias, hidden)
    if ops.FUSED and logits.device is Device.HIP:
        plan = _dispatch_table[(CustomOps.ADJUST_LOGITS, Device.HIP)](x, h, n, (r, p, f), b, m)
        if len(_adjust_plans) >= 1024:                                  # (a workload whose shapes never repeat)
            _adjust_plans.clear()
        _adjust_plans[key] = plan
        return _result(x._like(plan(x, h, n, (r, p, f), b, m)))
    (B, V), x = logits.shape, logits.numpy().astype(np.float32, copy=True)
    rows = lambda p: p.numpy().reshape(B) if isinstance(p, Tensor) else np.full(B, p, np.float32)      # noqa: E731
    rep, pre, fre = rows(repetition), rows(presence), rows(frequency)
    if history is not None and history.shape[1]:
        ids, L = history.numpy(), history.shape[1]
        n = np.full(B, float(L)) if lengths is None else np.nan_to_num(lengths.numpy().reshape(B).astype(np.float64), nan=0.0)
        for b in range(B):
            row = ids[b, :int(min(max(n[b], 0), L))]
            row = row[(row >= 0) & (row < V)].astype(np.int64)
            count = np.bincount(row, minlength=V)[:V].astype(np.float32)
            with np.errstate(all="ignore"):
                said = np.where(x[b] > 0, x[b] / rep[b], x[b] * rep[b]) - (pre[b] + fre[b] * count)
            x[b] = np.where(count > 0, said, x[b])
    if bias is not None:
        x = x + bias.numpy().reshape(-1, V)
    if hidden is not None:
        x = np.where(hidden.numpy().reshape(-1, V) > 0, np.float32(-np.inf), x)
    return Tensor(np.ascontiguousarray(x, dtype=np.float32), device=logits.device)
