"""What the language-model operators of this package are timed on: rotary positions, a key/value cache held in 8 bits
with the attention that reads it, and the adjustment of logits before a token is chosen.

`own` chooses between the package's kernels and the operators' plain forms (elementary torch operations).  A case is a
dict of plain values; prepare() makes what a program holds before the call, run() is one pass, exact() the same results
in 64 bits.
"""
import math

import numpy as np
import torch

own = False

BLOCK = 64          # tokens that share a scale in the 8-bit cache


# ---------------------------------------------------------------- cases
def listed():
    def rotary(name, batch, tokens, heads, kv_heads, dim, rotated, layout, scaling, first, grad):
        return dict(name=name, op="rotary", batch=batch, tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim,
                    rotated=rotated, layout=layout, scaling=scaling, first=first, grad=grad)

    def attend(name, batch, heads, kv_heads, dim, held, new, ragged):
        return dict(name=name, op="attend", batch=batch, heads=heads, kv_heads=kv_heads, dim=dim, held=held, new=new, ragged=ragged)

    def fill(name, batch, kv_heads, dim, new):
        return dict(name=name, op="fill", batch=batch, kv_heads=kv_heads, dim=dim, new=new)

    def logits(name, batch, vocab, history, hidden, bias):
        return dict(name=name, op="logits", batch=batch, vocab=vocab, history=history, hidden=hidden, bias=bias)

    return [
        # one token of the char-level model (4 heads of 32): the smallest call there is, all latency
        rotary("rotary_one_token", 1, 1, 4, 4, 32, 32, "half", "none", 100, False),
        # a training step's q and k of the char-level model (batch 16, 128 tokens), neighbouring elements as pairs
        rotary("rotary_train_char", 16, 128, 4, 4, 32, 32, "interleaved", "none", 0, True),
        # a training step's q and k of the scaled model (batch 8, 1024 tokens, 12 heads of 64)
        rotary("rotary_train_scaled", 8, 1024, 12, 12, 64, 64, "half", "none", 0, True),
        # one long sequence far beyond the trained length: half of each head is turned, frequencies scaled by parts, shared key heads
        rotary("rotary_long_partial", 1, 30001, 32, 8, 128, 64, "half", "parts", 100000, False),
        # decoding with the char-level model: one sequence, one block of 8-bit tokens and a tail
        attend("attend_char", 1, 4, 4, 32, 100, 1, False),
        # decoding with the scaled model: 8 sequences, the step that completes a block
        attend("attend_scaled", 8, 12, 12, 64, 1023, 1, False),
        # serving: 16 sequences of different lengths up to 32768, 32 query heads on 8 key heads of 128
        attend("attend_long_shared", 16, 32, 8, 128, 32768, 1, True),
        # a prompt that arrives in pieces: 256 new tokens per sequence after 4096
        attend("attend_piece", 4, 12, 12, 64, 4096, 256, False),
        # the scaled model's prompt of 1024 tokens, written to the cache and read back as values
        fill("fill_scaled", 8, 12, 64, 1024),
        # one sequence of the char-level model: 65 logits, 128 tokens so far
        logits("logits_char", 1, 65, 128, False, False),
        # the scaled model's vocabulary, 8 sequences, with a grammar's mask and a bias row
        logits("logits_scaled", 8, 50304, 1024, True, True),
        # a large batch of requests over a large vocabulary with long histories
        logits("logits_batch", 256, 128256, 4000, False, True),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "attend", "attend", "fill", "logits"])
    kv = rng.choice([1, 2, 3, 4, 5, 8, 12])
    if op == "rotary":
        dim = rng.choice([16, 20, 32, 64, 80, 96, 128])
        rotated = rng.choice([dim, dim, dim // 2 // 2 * 2])
        heads = kv * rng.choice([1, 1, 2, 4])
        room = 30001 * 40 * 128 // (2 * (heads + kv) * dim)
        batch = _spread(rng, 1, 16)
        return dict(op=op, batch=batch, tokens=_spread(rng, 1, max(2, room // batch)), heads=heads, kv_heads=kv, dim=dim,
                    rotated=rotated, layout=rng.choice(["half", "interleaved"]), scaling=rng.choice(["none", "linear", "base", "parts"]),
                    first=_spread(rng, 1, 200000), grad=rng.random() < 0.5)
    if op == "attend":
        dim = rng.choice([16, 32, 40, 64, 80, 128])
        heads = kv * rng.choice([1, 1, 2, 3, 4, 7])
        batch = _spread(rng, 1, 16)
        new = rng.choice([1, 1, 1, _spread(rng, 2, 48), _spread(rng, 65, 300)])
        most = min(40000, 8 * 16 * 32768 * 128 // (batch * kv * dim * (1 if new == 1 else 16)))
        held = _spread(rng, 2, max(3, most // (1 if new <= 48 else 4)))
        ragged = new <= 48 and rng.random() < 0.5
        return dict(op=op, batch=batch, heads=heads, kv_heads=kv, dim=dim, held=held if new <= 48 else held // BLOCK * BLOCK, new=new, ragged=ragged)
    if op == "fill":
        dim = rng.choice([16, 24, 32, 64, 80, 128])
        batch = _spread(rng, 1, 16)
        return dict(op=op, batch=batch, kv_heads=kv, dim=dim, new=_spread(rng, 1, max(2, min(20000, 8 * 12 * 64 * 4096 // (batch * kv * dim)))))
    batch = _spread(rng, 1, 200)
    return dict(op=op, batch=batch, vocab=_spread(rng, 50, min(150000, 256 * 120000 // batch)), history=_spread(rng, 1, 4000),
                hidden=rng.random() < 0.5, bias=rng.random() < 0.5)


def work(case):
    if case["op"] == "rotary":
        n = case["batch"] * case["tokens"] * (case["heads"] + case["kv_heads"]) * case["dim"]
        passes = 2 if case["grad"] else 1
        return {"bytes": passes * (8 * n + 4 * case["batch"] * case["tokens"]), "flops": passes * 3 * n}
    if case["op"] == "attend":
        b, kv, d, t = case["batch"], case["kv_heads"], case["dim"], case["new"]
        held = int(_lengths(case).sum())
        seen = sum(t * int(n) + t * (t + 1) // 2 for n in _lengths(case))
        read = 2 * held * kv * d + 8 * kv * (held // BLOCK)
        return {"bytes": read + 8 * b * t * case["heads"] * d + 8 * b * t * kv * d, "flops": 4 * seen * case["heads"] * d}
    if case["op"] == "fill":
        n = 2 * case["batch"] * case["new"] * case["kv_heads"] * case["dim"]
        return {"bytes": n * (4 + 1 + 4), "flops": 3 * n}           # read, held as 8 bits, read back as values
    n = case["batch"] * case["vocab"]
    return {"bytes": 8 * n + (4 * n if case["hidden"] else 0) + (4 * case["vocab"] if case["bias"] else 0) + 4 * case["batch"] * case["history"],
            "flops": 4 * n}


# ---------------------------------------------------------------- inputs
def _device():
    return torch.device("cuda" if torch.cuda.is_available() else "cpu")


def _maker(seed):
    g = torch.Generator(device=_device())
    g.manual_seed(seed)
    return g


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device=_device(), dtype=torch.float32)


def _lengths(case):
    """Tokens that each sequence holds before the call: the same for all, or falling from `held` to a little over a half of it."""
    b, n = case["batch"], case["held"]
    return np.array([n - (i * n) // (2 * b) if case["ragged"] else n for i in range(b)], dtype=np.int64)


def _frequencies(case):
    """Radians per position of each pair of a head, and the factor of the result."""
    r, base, factor, trained = case["rotated"], 10000.0, 8.0, 8192
    i = np.arange(r // 2, dtype=np.float64)
    if case["scaling"] == "base":
        base = base * factor ** (r / (r - 2))
    f = base ** (-2.0 * i / r)
    if case["scaling"] == "linear":
        return f / factor, 1.0
    if case["scaling"] == "parts":
        turns = trained * f / (2 * math.pi)
        keep = np.clip((turns - 1.0) / (32.0 - 1.0), 0.0, 1.0)
        return keep * f + (1.0 - keep) * f / factor, 0.1 * math.log(factor) + 1.0
    return f, 1.0


def _rotary_inputs(case, seed):
    g = _maker(seed)
    b, t, d = case["batch"], case["tokens"], case["dim"]
    names = ("q", "k", "gq", "gk") if case["grad"] else ("q", "k")
    x = {n: _normal(g, b, t, (case["kv_heads"] if n.endswith("k") else case["heads"]) * d) for n in names}
    x["positions"] = (case["first"] + torch.arange(b, device=_device())[:, None] * 3 + torch.arange(t, device=_device())[None, :]).to(torch.float32)
    return x


def _attend_inputs(case, seed):
    """The keys and values so far (b, held, kv_heads * d), and the new q, k, v."""
    g = _maker(seed)
    b, kv, d, t = case["batch"], case["kv_heads"], case["dim"], case["new"]
    wide = 0.5 + torch.rand((kv * d,), generator=g, device=_device())          # channels differ in spread
    hold = case.get("held", 0)
    return {"old_k": _normal(g, b, hold, kv * d) * wide, "old_v": _normal(g, b, hold, kv * d),
            "q": _normal(g, b, t, case.get("heads", 1) * d), "k": _normal(g, b, t, kv * d) * wide, "v": _normal(g, b, t, kv * d)}


def _logits_inputs(case, seed):
    g = _maker(seed)
    b, v, n = case["batch"], case["vocab"], case["history"]
    u = torch.rand((b, n), generator=g, device=_device())
    x = {"logits": 4.0 * _normal(g, b, v),
         "history": (u * u * u * v).floor().clamp(max=v - 1),                      # low ids come often, as in text
         "lengths": torch.tensor([[n - (i * n) // (2 * b)] for i in range(b)], dtype=torch.float32, device=_device())}
    if case["bias"]:
        x["bias"] = 0.5 * _normal(g, v)
    if case["hidden"]:
        x["hidden"] = (torch.rand((b, v), generator=g, device=_device()) < 0.4).to(torch.float32)
    return x


REPETITION, PRESENCE, FREQUENCY = 1.3, 0.25, 0.125


class _Memory:
    """A tensor of this package as torch sees device memory; keeps the tensor alive."""

    def __init__(self, t):
        self.t = t
        self.__cuda_array_interface__ = {"shape": tuple(t.shape), "typestr": "<f4", "data": (t.data.ptr.addr, False), "version": 2}


def _seen(t):
    return torch.as_tensor(_Memory(t), device="cuda")


def _given(x):
    """torch tensors as tensors of this package, copied on the device."""
    from dlgrad_amd import Tensor
    from dlgrad_amd.runtime import hip
    mine = {n: Tensor.full(tuple(t.shape), 0.0, device="hip") for n, t in x.items()}
    hip.lib().sync()
    for n, t in x.items():
        if t.numel():
            _seen(mine[n]).copy_(t)
    torch.cuda.synchronize()
    return mine


def prepare(case, seed):
    if case["op"] == "rotary":
        x = _rotary_inputs(case, seed)
        f, gain = _frequencies(case)
        if own:
            from dlgrad_amd import nn
            rope = nn.Rotary(case["dim"], case["rotated"], layout=case["layout"], scaling=None if case["scaling"] == "none" else case["scaling"],
                             factor=8.0 if case["scaling"] != "none" else 1.0, trained=8192, device="hip")
            return {"case": case, "x": _given(x), "rope": rope}
        return {"case": case, "x": x, "f": torch.tensor(f, device=_device()), "gain": gain}
    if case["op"] == "logits":
        x = _logits_inputs(case, seed)
        return {"case": case, "x": _given(x) if own else x}
    x = _attend_inputs(case, seed)
    b, kv, d = case["batch"], case["kv_heads"], case["dim"]
    lens = _lengths(case) if case["op"] == "attend" else np.zeros(b, np.int64)
    blocks = (int(lens.max()) + case["new"]) // BLOCK + 1
    if own:
        from dlgrad_amd import Tensor, nn
        cache = nn.QuantizedKVCache(b, blocks * BLOCK, kv, d, device="hip")
        mine = _given(x)
        if lens.max():
            counts = Tensor(lens.astype(np.float32).reshape(b, 1), device="hip")
            cache.write(mine["old_k"], mine["old_v"], counts=counts)
            cache.advance(counts)
        return {"case": case, "cache": cache, "x": {n: mine[n] for n in ("q", "k", "v")}}
    old = {}
    for n in ("k", "v"):
        full = torch.zeros((b, blocks * BLOCK, kv * d), device=_device())
        full[:, :x["old_" + n].shape[1]] = x["old_" + n]
        old[n] = full.view(b, blocks, BLOCK, kv, d).permute(0, 3, 1, 2, 4).contiguous()
    at = torch.tensor(lens, device=_device())
    state = {"case": case, "at": at, "x": {n: x[n] for n in ("q", "k", "v")}}
    for n in ("k", "v"):
        codes, scale = _quantised(old[n])
        state["codes_" + n], state["scale_" + n] = codes.to(torch.int8), scale
        state["tail_" + n] = old[n][torch.arange(b, device=_device()), :, at // BLOCK]        # the block that is not full yet, unquantised
    return state


# ---------------------------------------------------------------- plain forms
def _turned(x, cos, sin, case, back):
    """x (b, t, heads * d) with the first `rotated` elements of each head turned, pair by pair."""
    r = case["rotated"]
    h = x.reshape(x.shape[0], x.shape[1], -1, case["dim"])
    if case["layout"] == "half":
        a, b = h[..., :r // 2], h[..., r // 2:r]
    else:
        a, b = h[..., 0:r:2], h[..., 1:r:2]
    c, s = cos[:, :, None, :], (-sin if back else sin)[:, :, None, :]
    ya, yb = a * c - b * s, a * s + b * c
    y = torch.cat((ya, yb), -1) if case["layout"] == "half" else torch.stack((ya, yb), -1).flatten(-2)
    return torch.cat((y, h[..., r:]), -1).reshape(x.shape)


def _quantised(x):
    """Whole numbers in -127 .. 127 of the blocks x (..., BLOCK, d) and their scales (...): scale = largest magnitude / 127
    as a 32-bit number, x / scale rounded to the nearest, ties to even (in 64 bits: a quotient next to a half must not cross it)."""
    scale = (x.abs().amax((-1, -2)).double() / 127.0).float()
    wide = scale.double()[..., None, None]
    return torch.where(wide > 0, x.double() / wide, 0.0).round().clamp(-127, 127), scale


def _written(codes, scale, tail, new, at, case):
    """The cache's values (b, kv, blocks, BLOCK, d) after the rows `new` (b, t, kv * d) went to positions at[b] ..: the blocks that are
    full by then quantised, the rest as they came."""
    b, kv, d, t = case["batch"], case["kv_heads"], case["dim"], case["new"]
    rows = torch.arange(b, device=new.device)
    values = codes.float() * scale[..., None, None]
    values[rows, :, at // BLOCK] = tail
    where = at[:, None] + torch.arange(t, device=new.device)                                   # (b, t)
    values[rows[:, None], :, where // BLOCK, where % BLOCK] = new.view(b, t, kv, d)
    touched = (at // BLOCK)[:, None] + torch.arange((t + BLOCK - 1) // BLOCK, device=new.device)
    touched = touched.clamp(max=values.shape[2] - 1)
    now = values[rows[:, None], :, touched]                                                      # (b, blocks touched, kv, BLOCK, d)
    q, s = _quantised(now)
    full = (touched + 1) * BLOCK <= (at + t)[:, None]
    values[rows[:, None], :, touched] = torch.where(full[:, :, None, None, None], q.float() * s[..., None, None], now)
    return values


def _attended(state):
    case, x, at = state["case"], state["x"], state["at"]
    b, kv, d, t = case["batch"], case["kv_heads"], case["dim"], case["new"]
    g = case["heads"] // kv
    k, v = (_written(state["codes_" + n], state["scale_" + n], state["tail_" + n], x[n], at, case).flatten(2, 3) for n in ("k", "v"))
    q = x["q"].view(b, t, kv, g, d).permute(0, 2, 3, 1, 4).reshape(b, kv, g * t, d)
    s = torch.matmul(q, k.transpose(2, 3).contiguous()) * (d ** -0.5)                            # (b, kv, g * t, positions)
    late = torch.arange(k.shape[2], device=k.device) > (at[:, None] + torch.arange(t, device=k.device))[:, :, None]      # (b, t, positions)
    s = s.view(b, kv, g, t, -1).masked_fill(late[:, None, None], float("-inf"))
    e = torch.exp(s - s.amax(-1, keepdim=True))
    p = (e / e.sum(-1, keepdim=True)).view(b, kv, g * t, -1)
    y = torch.matmul(p, v)
    return y.view(b, kv, g, t, d).permute(0, 3, 1, 2, 4).reshape(b, t, kv * g * d)


def _adjusted(x):
    logits, history = x["logits"], x["history"].long()
    valid = torch.arange(history.shape[1], device=logits.device) < x["lengths"]
    count = torch.zeros_like(logits).scatter_add_(1, history, valid.float())
    y = torch.where(logits > 0, logits / REPETITION, logits * REPETITION) - (PRESENCE + FREQUENCY * count)
    y = torch.where(count > 0, y, logits)
    if "bias" in x:
        y = y + x["bias"]
    return y.masked_fill(x["hidden"] > 0, float("-inf")) if "hidden" in x else y


def run(state):
    case = state["case"]
    if case["op"] == "rotary":
        x = state["x"]
        if own:
            rope, heads, kv = state["rope"], case["heads"], case["kv_heads"]
            q, k = rope.pair(x["q"], x["k"], heads, kv, positions=x["positions"])
            if not case["grad"]:
                return {"q": _seen(q), "k": _seen(k)}
            dq, dk = rope.pair(x["gq"], x["gk"], heads, kv, positions=x["positions"], transpose=True)
            return {"q": _seen(q), "k": _seen(k), "dq": _seen(dq), "dk": _seen(dk)}
        angle = x["positions"].double()[:, :, None] * state["f"]
        cos, sin = (torch.cos(angle) * state["gain"]).float(), (torch.sin(angle) * state["gain"]).float()
        y = {"q": _turned(x["q"], cos, sin, case, False), "k": _turned(x["k"], cos, sin, case, False)}
        if case["grad"]:
            y["dq"], y["dk"] = _turned(x["gq"], cos, sin, case, True), _turned(x["gk"], cos, sin, case, True)
        return y
    if case["op"] == "attend":
        if own:
            cache, x = state["cache"], state["x"]
            cache.write(x["k"], x["v"])
            return {"y": _seen(cache.attend(x["q"]))}
        return {"y": _attended(state)}
    if case["op"] == "fill":
        x, t = state["x"], case["new"]
        if own:
            cache = state["cache"]
            cache.write(x["k"], x["v"])
            k, v = cache.read(t, new=t)
            return {"k": _seen(k), "v": _seen(v)}
        got = {n: _written(state["codes_" + n], state["scale_" + n], state["tail_" + n], x[n], state["at"], case) for n in ("k", "v")}
        return {n: y.permute(0, 2, 3, 1, 4).reshape(case["batch"], -1, case["kv_heads"] * case["dim"])[:, :t] for n, y in got.items()}
    x = state["x"]
    if own:
        from dlgrad_amd import nn
        return {"logits": _seen(nn.adjust_logits(x["logits"], x["history"], x["lengths"], repetition=REPETITION, presence=PRESENCE,
                                                 frequency=FREQUENCY, bias=x.get("bias"), hidden=x.get("hidden")))}
    return {"logits": _adjusted(x)}


# ---------------------------------------------------------------- 64 bits
def _rotated_64(x, angles, gain, case, sign):
    """Each pair as one complex number, times gain * exp(i angle)."""
    r = case["rotated"]
    y = x.double().reshape(x.shape[0], x.shape[1], -1, case["dim"]).clone()
    first, second = (slice(0, r // 2), slice(r // 2, r)) if case["layout"] == "half" else (slice(0, r, 2), slice(1, r, 2))
    z = torch.complex(y[..., first].contiguous(), y[..., second].contiguous()) * torch.polar(torch.full_like(angles, gain), sign * angles)[:, :, None]
    y[..., first], y[..., second] = z.real, z.imag
    return y.reshape(x.shape)


def _held_64(rows, whole):
    """rows (n, d) of one head: the first `whole` of them, in blocks, as the 8-bit cache stands for them; the rest as they are."""
    rows = rows.double()
    head = rows[:whole].reshape(-1, BLOCK, rows.shape[1])
    step = (head.abs().flatten(1).max(1).values / 127).float().double()[:, None, None] if whole else head.new_zeros(0, 1, 1)
    n = torch.where(step == 0, torch.zeros_like(head), torch.round(head / torch.where(step == 0, 1.0, step)))
    return torch.cat((torch.clamp(n, -127, 127).mul(step).reshape(whole, rows.shape[1]), rows[whole:]))


def exact(case, seed):
    if case["op"] == "rotary":
        x = _rotary_inputs(case, seed)
        f, gain = _frequencies(case)
        angles = x["positions"].double()[..., None] * torch.from_numpy(f).to(x["positions"].device)
        got = {n: _rotated_64(x[n], angles, gain, case, 1.0) for n in ("q", "k")}
        if case["grad"]:
            got.update(dq=_rotated_64(x["gq"], angles, gain, case, -1.0), dk=_rotated_64(x["gk"], angles, gain, case, -1.0))
        return got
    if case["op"] == "logits":
        x = _logits_inputs(case, seed)
        y = x["logits"].double()
        for i in range(case["batch"]):
            ids, times = torch.unique(x["history"][i, :int(x["lengths"][i, 0])].long(), return_counts=True)
            z = y[i, ids]
            y[i, ids] = torch.where(z > 0, z / REPETITION, z * REPETITION) - PRESENCE - FREQUENCY * times.double()
        if "bias" in x:
            y += x["bias"].double()
        if "hidden" in x:
            y[x["hidden"] != 0] = -math.inf
        return {"logits": y}
    x = _attend_inputs(case, seed)
    b, kv, d, t = case["batch"], case["kv_heads"], case["dim"], case["new"]
    if case["op"] == "fill":
        return {n: torch.stack([torch.cat([_held_64(x[n][i, :, h * d:(h + 1) * d], t // BLOCK * BLOCK) for h in range(kv)], 1) for i in range(b)]) for n in ("k", "v")}
    g = case["heads"] // kv
    y = torch.empty((b, t, kv * g * d), dtype=torch.float64, device=x["q"].device)
    for i, n in enumerate(_lengths(case).tolist()):
        whole = (n + t) // BLOCK * BLOCK
        for h in range(kv):
            at = slice(h * d, (h + 1) * d)
            k, v = (_held_64(torch.cat((x["old_" + w][i, :n, at], x[w][i, :, at])), whole) for w in ("k", "v"))
            for j in range(g):
                here = slice((h * g + j) * d, (h * g + j + 1) * d)
                s = x["q"][i, :, here].double() @ k.T / math.sqrt(d)
                if t > 1:
                    s[torch.ones_like(s, dtype=torch.bool).triu(n + 1)] = -math.inf
                y[i, :, here] = torch.softmax(s, 1) @ v
    return {"y": y}
