"""Rotary positions, the 8-bit key/value cache and the adjustment of logits against plain float64 formulas.

Tolerances count roundings.  An fp32 operation is off by at most EPS = 2^-24 of its result."""
import math

import numpy as np
import pytest

import oracle.cpu_runtime  # noqa: F401  (the CPU column of the dispatch table)
from dlgrad_amd import Tensor, nn, ops
from dlgrad_amd.buffer import Buffer
from dlgrad_amd.device import Device
from dlgrad_amd.runtime import hip
from dlgrad_amd.runtime.hip_lm import HIPLM
from hip_util import require_gpu

EPS = 2.0 ** -24
BLOCK = 64
f32 = np.float32


def hip_tensor(a, requires_grad=False):
    return Tensor(np.ascontiguousarray(a, dtype=np.float32), device="hip", requires_grad=requires_grad)


def within(got, want, tol, what=""):
    """|got - want| <= tol elementwise; NaN and infinities in the same places."""
    if hip.COMPILE_ONLY:
        return
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    assert got.shape == want.shape, f"{what}: {got.shape} vs {want.shape}"
    if not want.size:
        return
    odd = ~np.isfinite(want)
    np.testing.assert_array_equal(got[odd], want[odd], err_msg=what)
    assert np.isfinite(got[~odd]).all(), f"{what}: not finite where it should be"
    d = np.abs(got[~odd] - want[~odd])
    t = np.broadcast_to(tol, want.shape)[~odd]
    assert (d <= t).all(), f"{what}: off by {d.max():.3e}, {float((d / np.maximum(t, 1e-300)).max()):.2f} of what is allowed"


def same(got, want, what=""):
    if not hip.COMPILE_ONLY:
        np.testing.assert_array_equal(np.asarray(got), np.asarray(want), err_msg=what)


# ================================================================ rotary positions
def turned(x, n_head, rope, p, back=False):
    """float64; p broadcasts against (B, T)."""
    d, r = rope.head_dim, rope.rotated
    four = x.ndim == 4
    h = np.array(x, np.float64) if four else np.array(x, np.float64).reshape(x.shape[0], x.shape[1], n_head, d)
    w = np.asarray(p, np.float64)[..., None] * rope.frequencies
    w = w[:, None] if four else w[:, :, None]
    z = (h[..., :r // 2] + 1j * h[..., r // 2:r]) if rope.half else (h[..., 0:r:2] + 1j * h[..., 1:r:2])
    z = z * rope.gain * np.exp((-1j if back else 1j) * w)
    out = h.copy()
    if rope.half:
        out[..., :r // 2], out[..., r // 2:r] = z.real, z.imag
    else:
        out[..., 0:r:2], out[..., 1:r:2] = z.real, z.imag
    return out.reshape(x.shape)


def turned_tol(x, rope):
    """Per element: |x| of the pair times (angle 2^-24 of a radian each way after a 30-bit turn and its fp32 polynomial, at most
    4 EPS for sine and cosine together with the Taylor remainder of 2.5e-8, times the gain), two products and a sum."""
    return np.abs(x).max() * 2 * rope.gain * (4 * EPS + 2.5e-8 + 3 * EPS)


ROTARY = [  # head_dim, rotated, n_head, B, T
    (32, 32, 4, 16, 128), (64, 64, 12, 2, 33), (64, 64, 1, 1, 1), (128, 64, 5, 3, 7), (20, 20, 3, 2, 9), (80, 40, 9, 1, 65),
    (6, 2, 2, 2, 5), (2, 2, 7, 1, 3), (256, 256, 2, 1, 11), (12, 4, 1, 4, 300),
]


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("d,r,h,B,T", ROTARY)
def test_rotary_turns_every_pair_by_its_angle(d, r, h, B, T, layout):
    require_gpu()
    rng = np.random.default_rng(d * 7 + T)
    rope = nn.Rotary(d, r, layout=layout)
    x = rng.standard_normal((B, T, h * d)).astype(f32)
    p = rng.integers(0, 5000, (B, T)).astype(f32)
    tol = turned_tol(x, rope)
    y = rope(hip_tensor(x), h)
    within(y.numpy(), turned(x, h, rope, np.arange(T)[None]), tol, "positions 0 ..")
    within(rope(hip_tensor(x), h, positions=hip_tensor(p)).numpy(), turned(x, h, rope, p), tol, "positions (B, T)")
    within(rope(hip_tensor(x), h, positions=hip_tensor(p[0]), transpose=True).numpy(), turned(x, h, rope, p[:1], True), tol, "positions (T,)")
    start = np.arange(B, dtype=f32).reshape(B, 1) * 17
    within(rope(hip_tensor(x), h, start=hip_tensor(start)).numpy(), turned(x, h, rope, start + np.arange(T)), tol, "a start each")
    within(rope(hip_tensor(x), h, positions=hip_tensor(p), start=hip_tensor(np.full((1, 1), 100, f32))).numpy(), turned(x, h, rope, p + 100), tol, "one start")
    if not hip.COMPILE_ONLY:
        rest = y.numpy().reshape(B, T, h, d)[..., r:]
        same(rest, x.reshape(B, T, h, d)[..., r:], "elements that do not turn")


@pytest.mark.gpu
def test_rotary_at_far_and_negative_positions():
    """2^24 - 1 radians would be off by a whole radian as an fp32 product.  float64 holds the angle to 2^24 * 2^-53 * 2 pi."""
    require_gpu()
    rng = np.random.default_rng(3)
    for layout in ("half", "interleaved"):
        rope = nn.Rotary(64, layout=layout)
        x = rng.standard_normal((1, 6, 3 * 64)).astype(f32)
        p = np.array([[-1, -(2 ** 24) + 1, 2 ** 24 - 1, 2 ** 24, 131071, 0]], f32)
        within(rope(hip_tensor(x), 3, positions=hip_tensor(p)).numpy(), turned(x, 3, rope, p), turned_tol(x, rope), layout)


@pytest.mark.gpu
@pytest.mark.parametrize("scaling,factor", [("linear", 4.0), ("base", 8.0), ("parts", 16.0)])
def test_rotary_scaled_for_long_contexts(scaling, factor):
    require_gpu()
    rng = np.random.default_rng(5)
    rope = nn.Rotary(64, 32, scaling=scaling, factor=factor, trained=2048)
    x = rng.standard_normal((2, 50, 2 * 64)).astype(f32)
    p = rng.integers(0, 2048 * 16, (2, 50)).astype(f32)
    within(rope(hip_tensor(x), 2, positions=hip_tensor(p)).numpy(), turned(x, 2, rope, p), turned_tol(x, rope))


def test_rotary_frequencies():
    f, gain = nn.rotary_frequencies(8)
    np.testing.assert_allclose(f, [1.0, 0.1, 0.01, 0.001], rtol=1e-12)
    assert gain == 1.0
    np.testing.assert_allclose(nn.rotary_frequencies(8, scaling="linear", factor=4.0)[0], f / 4, rtol=1e-15)
    g = nn.rotary_frequencies(8, scaling="base", factor=4.0)[0]
    np.testing.assert_allclose([g[0], g[-1]], [f[0], f[-1] / 4], rtol=1e-12)
    g, gain = nn.rotary_frequencies(128, scaling="parts", factor=4.0, trained=4096)
    f = nn.rotary_frequencies(128)[0]
    turns = 4096 * f / (2 * math.pi)
    np.testing.assert_allclose(g[turns >= 32], f[turns >= 32], rtol=1e-15)
    np.testing.assert_allclose(g[turns <= 1], f[turns <= 1] / 4, rtol=1e-15)
    assert np.all(np.diff(g) < 0) and gain == pytest.approx(0.1 * math.log(4) + 1)


@pytest.mark.gpu
def test_rotary_pair_and_four_dimensions():
    """One launch for queries and keys of different head counts gives the bits of two; (B, heads, T, d) those of (B, T, heads * d)."""
    require_gpu()
    rng = np.random.default_rng(9)
    for layout in ("half", "interleaved"):
        for d, r in ((64, 64), (40, 20)):
            rope = nn.Rotary(d, r, layout=layout)
            q, k = rng.standard_normal((2, 19, 8 * d)).astype(f32), rng.standard_normal((2, 19, 3 * d)).astype(f32)
            p = hip_tensor(rng.integers(0, 999, (2, 19)))
            qt, kt = rope.pair(hip_tensor(q), hip_tensor(k), 8, 3, positions=p)
            same(qt.numpy(), rope(hip_tensor(q), 8, positions=p).numpy())
            same(kt.numpy(), rope(hip_tensor(k), 3, positions=p).numpy())
            q4 = np.ascontiguousarray(q.reshape(2, 19, 8, d).transpose(0, 2, 1, 3))
            y4 = rope(hip_tensor(q4), positions=p, start=hip_tensor(np.zeros((2, 1)))).numpy()
            same(y4.transpose(0, 2, 1, 3).reshape(2, 19, 8 * d), qt.numpy())
            k4 = np.ascontiguousarray(k.reshape(2, 19, 3, d).transpose(0, 2, 1, 3))
            a, b = rope.pair(hip_tensor(q4), hip_tensor(k4), 1, positions=p)                  # per-sequence rows differ: two launches
            same(a.numpy(), y4)
            same(b.numpy().transpose(0, 2, 1, 3).reshape(2, 19, 3 * d), kt.numpy())


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotary_beyond_the_caches_has_the_same_bits(layout, monkeypatch):
    """The form for large tensors, which bypasses the caches, forced on a small one."""
    require_gpu()
    from dlgrad_amd.runtime import hip_lm
    rng = np.random.default_rng(12)
    q, k = rng.standard_normal((2, 33, 6 * 48)).astype(f32), rng.standard_normal((2, 33, 2 * 48)).astype(f32)
    want = [t.numpy() for t in nn.Rotary(48, 32, layout=layout).pair(hip_tensor(q), hip_tensor(k), 6, 2)]
    monkeypatch.setattr(hip_lm, "ROTARY_STREAM_ELEMENTS", 1)
    monkeypatch.setattr(hip_lm, "_rotary_plans", {})
    for a, b in zip(nn.Rotary(48, 32, layout=layout).pair(hip_tensor(q), hip_tensor(k), 6, 2), want):
        same(a.numpy(), b)


@pytest.mark.gpu
def test_rotary_by_size_has_the_bits_of_its_pieces():
    """Enough elements to bypass the caches, against pieces that do not."""
    require_gpu()
    from dlgrad_amd.runtime import hip_lm
    rng = np.random.default_rng(15)
    q, k = (rng.standard_normal((1, 700, 12 * 64)).astype(f32) for _ in range(2))
    assert q.size + k.size >= hip_lm.ROTARY_STREAM_ELEMENTS > 2 * q[:, :300].size
    rope = nn.Rotary(64)
    got = [t.numpy() for t in rope.pair(hip_tensor(q), hip_tensor(k), 12)]
    for at in range(0, 700, 300):
        rows = slice(at, at + 300)
        for a, b in zip(got, rope.pair(hip_tensor(q[:, rows]), hip_tensor(k[:, rows]), 12, start=hip_tensor([[at]]))):
            same(a[:, rows], b.numpy())


@pytest.mark.gpu
def test_rotary_of_unaligned_views_and_of_nothing():
    require_gpu()
    rng = np.random.default_rng(2)
    rope = nn.Rotary(64)
    x = rng.standard_normal((1, 7, 128)).astype(f32)
    room = Buffer.from_numpy(np.concatenate([np.zeros(1, f32), x.reshape(-1)]), Device.HIP)
    view = Tensor(Buffer(room.ptr + 1, (1, 7, 128), Device.HIP))
    same(rope(view, 2).numpy(), rope(hip_tensor(x), 2).numpy())
    assert rope(Tensor.full((2, 0, 128), 0.0, device="hip"), 2).shape == (2, 0, 128)


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotary_gradient(layout):
    """Against the transposed formula, and against differences of the loss along the gradient."""
    require_gpu()
    rng = np.random.default_rng(11)
    rope = nn.Rotary(12, 8, layout=layout, scaling="parts", factor=4.0, trained=64)
    q, k = rng.standard_normal((2, 5, 36)).astype(f32), rng.standard_normal((2, 5, 12)).astype(f32)
    gq, gk = rng.standard_normal((2, 5, 36)).astype(f32), rng.standard_normal((2, 5, 12)).astype(f32)
    p = rng.integers(0, 200, (2, 5)).astype(f32)
    qt, kt = hip_tensor(q, True), hip_tensor(k, True)
    yq, yk = rope.pair(qt, kt, 3, 1, positions=hip_tensor(p))
    loss = (yq * hip_tensor(gq)).sum() + (yk * hip_tensor(gk)).sum()
    loss.backward()
    within(qt.grad.numpy(), turned(gq, 3, rope, p, True), turned_tol(gq, rope), "dq")
    within(kt.grad.numpy(), turned(gk, 1, rope, p, True), turned_tol(gk, rope), "dk")
    if hip.COMPILE_ONLY:
        return
    step = 0.125
    at = lambda s: float((turned(q + s * qt.grad.numpy(), 3, rope, p) * gq).sum())      # noqa: E731
    norm = float((qt.grad.numpy().astype(np.float64) ** 2).sum())
    assert abs((at(step) - at(-step)) / (2 * step) - norm) <= 1e-5 * norm       # linear: differences are exact but for the gradient's own roundings


@pytest.mark.parametrize("device", ["cpu", pytest.param("hip", marks=pytest.mark.gpu)])
def test_rotary_gradient_turns_back_by_the_positions_of_its_forward(device):
    """Positions and starts that have moved on by the time of the backward pass."""
    if device == "hip":
        require_gpu()
    rng = np.random.default_rng(14)
    rope = nn.Rotary(8, device=device)
    q, k, gq, gk = (rng.standard_normal((2, 3, n)).astype(f32) for n in (16, 8, 16, 8))
    p, s0 = rng.integers(0, 50, (2, 3)).astype(f32), np.array([[4], [9]], f32)
    make = lambda a, **kw: Tensor(np.array(a), device=device, **kw)              # noqa: E731
    qt, kt, pt, st = make(q, requires_grad=True), make(k, requires_grad=True), make(p), make(s0)
    y, z = rope.pair(qt, kt, 2, 1, positions=pt, start=st)
    loss = (y * make(gq)).sum() + (z * make(gk)).sum()
    for t in (pt, st):
        t.data.copy_(make(np.full(t.shape, 31.0, f32)).data)
    loss.backward()
    within(qt.grad.numpy(), turned(gq, 2, rope, p + s0, True), turned_tol(gq, rope), "dq")
    within(kt.grad.numpy(), turned(gk, 1, rope, p + s0, True), turned_tol(gk, rope), "dk")


@pytest.mark.gpu
def test_rotary_gradient_in_a_captured_step_follows_its_start():
    """The copies of the positions are part of the step: each replay turns back by the start it turned by."""
    require_gpu()
    if hip.COMPILE_ONLY:
        return
    rng = np.random.default_rng(16)
    rope = nn.Rotary(8)
    q, k, gq, gk = (rng.standard_normal((2, 3, n)).astype(f32) for n in (16, 8, 16, 8))
    qt, kt, gqt, gkt, st = hip_tensor(q, True), hip_tensor(k, True), hip_tensor(gq), hip_tensor(gk), hip_tensor([[0], [0]])

    def step():
        qt.grad = kt.grad = None
        y, z = rope.pair(qt, kt, 2, 1, start=st)
        loss = (y * gqt).sum() + (z * gkt).sum()
        st.data.copy_((st + 5.0).data)                                       # the next call's
        loss.backward()
        return y
    run = hip.CapturedStep(step)
    p = np.arange(3) + np.zeros((2, 1))
    for i in range(6):
        y = run().numpy()
        within(y, turned(q, 2, rope, p + 5 * i), turned_tol(q, rope), f"step {i}")
        within(qt.grad.numpy(), turned(gq, 2, rope, p + 5 * i, True), turned_tol(gq, rope), f"dq of step {i}")
        within(kt.grad.numpy(), turned(gk, 1, rope, p + 5 * i, True), turned_tol(gk, rope), f"dk of step {i}")
        rope(hip_tensor(q), 2).numpy()                                        # work of its own between the replays
    run.close()


def test_rotary_composed_of_existing_ops_on_the_cpu():
    rng = np.random.default_rng(1)
    for layout in ("half", "interleaved"):
        rope = nn.Rotary(12, 8, layout=layout, device="cpu")
        x = rng.standard_normal((2, 5, 24)).astype(f32)
        p = rng.integers(0, 50, (2, 5)).astype(f32)
        t = Tensor(x, requires_grad=True)
        y = rope(t, 2, positions=Tensor(p), start=Tensor(np.array([[3.0]], f32)))
        within(y.numpy(), turned(x, 2, rope, p + 3), turned_tol(x, rope))
        g = rng.standard_normal(x.shape).astype(f32)
        (y * Tensor(g)).sum().backward()
        within(t.grad.numpy(), turned(g, 2, rope, p + 3, True), turned_tol(g, rope))
        x4 = np.ascontiguousarray(x.reshape(2, 5, 2, 12).transpose(0, 2, 1, 3))
        within(rope(Tensor(x4), positions=Tensor(p)).numpy(), turned(x4, 1, rope, p), turned_tol(x, rope))


@pytest.mark.gpu
def test_rotary_composition_and_kernel_agree(monkeypatch):
    require_gpu()
    rng = np.random.default_rng(1)
    rope = nn.Rotary(16)
    x, p = hip_tensor(rng.standard_normal((2, 9, 64))), hip_tensor(rng.integers(0, 70, (2, 9)))
    a = rope(x, 4, positions=p).numpy()
    monkeypatch.setattr(ops, "FUSED", False)
    within(rope(x, 4, positions=p).numpy(), a, 2 * turned_tol(x.numpy(), rope))


def test_rotary_refusals():
    for bad in (dict(head_dim=8, rotated=10), dict(head_dim=8, rotated=3), dict(head_dim=8, rotated=0), dict(head_dim=8, layout="other"),
                dict(head_dim=8, scaling="other"), dict(head_dim=8, scaling="parts"), dict(head_dim=8, scaling="parts", trained=64, factor=0.5),
                dict(head_dim=8, base=0.0), dict(head_dim=8, factor=-1.0, scaling="linear"), dict(head_dim=2, scaling="base", factor=2.0),
                dict(head_dim=8, base=float("inf"))):
        with pytest.raises(ValueError):
            nn.Rotary(device="cpu", **bad)
    rope = nn.Rotary(8, device="cpu")
    x = Tensor(np.zeros((2, 3, 16), f32))
    for call in (lambda: rope(x, 3), lambda: rope(x, 0), lambda: rope(Tensor(np.zeros((2, 2, 3, 16), f32)), 1), lambda: rope(Tensor(np.zeros((3, 16), f32)), 2),
                 lambda: rope(x, 2, positions=Tensor(np.zeros((2, 2), f32))), lambda: rope(x, 2, start=Tensor(np.zeros((3, 1), f32))),
                 lambda: rope(x, 2, positions=Tensor(np.zeros((3, 2), f32))),
                 lambda: rope.pair(x, Tensor(np.zeros((2, 4, 16), f32)), 2), lambda: rope.pair(x, Tensor(np.zeros((1, 3, 16), f32)), 2)):
        with pytest.raises(ValueError):
            call()


def test_rotary_refuses_a_factor_without_a_scaling():
    for call in (lambda: nn.Rotary(8, factor=8.0, device="cpu"), lambda: nn.rotary_frequencies(8, factor=0.5)):
        with pytest.raises(ValueError, match="no scaling"):
            call()
    assert nn.Rotary(8, factor=1, trained=64, device="cpu").gain == 1.0


def test_rotary_runtime_refuses_what_does_not_fit():
    """Host checks of the launch, before any device is touched."""
    class Ptr:
        addr, nbytes = 256, 1 << 40
    b = lambda n: Buffer(Ptr(), (n,), Device.HIP)                  # noqa: E731
    good = dict(parts=[(b(96), 2, 16)], freq=b(8), rows=6, T=3, per=1, d=8, rot=8, half=True, back=False, gain=1.0)
    for bad in (dict(rot=10), dict(rot=7), dict(freq=b(6)), dict(rows=7), dict(rows=6, T=4), dict(parts=[(b(95), 2, 16)]), dict(parts=[(b(96), 2, 15)]),
                dict(parts=[(b(96), 0, 16)]), dict(parts=[]), dict(positions=b(5)), dict(start=b(3)), dict(per=4),
                dict(positions=Buffer.from_scalar(1.0))):
        with pytest.raises(ValueError):
            HIPLM.rotary(**{**good, **bad})


# ================================================================ logits
def adjusted(x, history, n, rep, pre, fre, bias=None, hidden=None):
    y = np.array(x, np.float64)
    for b in range(x.shape[0]):
        ids = [int(i) for i in history[b, :n[b]] if 0 <= i < x.shape[1]]
        for i in set(ids):
            z = y[b, i]
            y[b, i] = (z / rep[b] if z > 0 else z * rep[b]) - (pre[b] + fre[b] * ids.count(i))
    if bias is not None:
        y = y + bias
    if hidden is not None:
        y = np.where(np.broadcast_to(hidden, y.shape) > 0, -np.inf, y)
    return y


LOGITS = [(1, 65, 128), (1, 1, 3), (3, 7, 1), (2, 1000, 50), (8, 50304, 1024), (5, 4097, 300), (2, 1024, 0), (64, 32768, 70), (300, 2052, 9), (17, 33333, 5000), (1, 700, 70000)]


@pytest.mark.gpu
@pytest.mark.parametrize("B,V,L", LOGITS)
def test_adjust_logits(B, V, L):
    """Each result is at most four fp32 operations away: quotient or product, presence + frequency * count, difference, bias."""
    require_gpu()
    rng = np.random.default_rng(V + L)
    x = (4 * rng.standard_normal((B, V))).astype(f32)
    history = np.floor(rng.random((B, L)) ** 3 * V).astype(f32)
    if L > 4:
        history[:, :4] = [V - 1, 0, V, -1]                                  # the ends of the table and beyond them
    n = rng.integers(0, L + 1, B)
    n[0] = L
    rep, pre, fre = (rng.uniform(1, 2, B).astype(f32), rng.uniform(-1, 1, B).astype(f32), rng.uniform(-1, 1, B).astype(f32))
    bias, hidden = rng.standard_normal(V).astype(f32), (rng.random((B, V)) < 0.3).astype(f32)
    want = adjusted(x, history, n, rep, pre, fre, bias, hidden)
    most = np.abs(x).max() * 2 + 1 + L + np.abs(bias).max()
    y = nn.adjust_logits(hip_tensor(x), hip_tensor(history), hip_tensor(n.reshape(B, 1)), hip_tensor(rep), hip_tensor(pre), hip_tensor(fre.reshape(B, 1)),
                         hip_tensor(bias), hip_tensor(hidden))
    within(y.numpy(), want, 5 * EPS * most, "a penalty per row")
    full = np.full(B, L)
    y = nn.adjust_logits(hip_tensor(x), hip_tensor(history), None, 1.3, 0.2, 0.1, hip_tensor(np.tile(bias, (B, 1))), hip_tensor(hidden[0]))
    c = np.ones(B)
    within(y.numpy(), adjusted(x, history, full, f32(1.3) * c, f32(0.2) * c, f32(0.1) * c, bias, hidden[:1]), 5 * EPS * most, "numbers")
    same(nn.adjust_logits(hip_tensor(x)).numpy(), x, "nothing asked")


@pytest.mark.gpu
@pytest.mark.parametrize("B,V,L,items", [(3, 701, 66000, 4), (24, 50257, 9, 8), (24, 50256, 66000, 8), (24, 50257, 66000, 8), (100, 50257, 70, 16), (100, 50256, 66000, 16), (100, 50257, 66000, 16)])
def test_adjust_logits_in_every_form(B, V, L, items):
    """8 and 16 logits a thread with and without 16-byte accesses, and counters of 32 bits for long histories; bounds as above."""
    require_gpu()
    assert HIPLM.adjust_items(B, V, 256) == items
    rng = np.random.default_rng(L + B)
    x = (4 * rng.standard_normal((B, V))).astype(f32)
    history = np.floor(rng.random((B, L), dtype=f32) ** 3 * (V + 2)).astype(f32) - 1              # from -1 to V
    n = rng.integers(0, L + 1, B)
    n[0] = L
    history[0] = V - 1                                                      # one token, more often than 16 bits count
    bias = rng.standard_normal(V).astype(f32)
    want = x.astype(np.float64)
    for b in range(B):
        ids = history[b, :n[b]]
        c = np.bincount(ids[(ids >= 0) & (ids < V)].astype(np.int64), minlength=V)
        want[b] = np.where(c > 0, np.where(want[b] > 0, want[b] / f32(1.3), want[b] * f32(1.3)) - (float(f32(0.2)) + float(f32(0.1)) * c), want[b])
    y = nn.adjust_logits(hip_tensor(x), hip_tensor(history), hip_tensor(n.reshape(B, 1)), 1.3, 0.2, 0.1, hip_tensor(bias))
    within(y.numpy(), want + bias, 5 * EPS * (np.abs(x).max() * 2 + 1 + 0.1 * L + np.abs(bias).max()))


@pytest.mark.gpu
def test_adjust_logits_masks_and_special_values():
    require_gpu()
    x = np.array([[1.0, np.nan, np.inf, -np.inf, -2.0, 3.4e38, -3.4028235e38, 0.0]], f32).repeat(3, 0)
    history = np.array([[0, 1, 2, 3, 4, 5, 6, 7]] * 3, f32)
    hidden = np.zeros((3, 8), f32)
    hidden[1] = 1.0                                                         # a row hidden whole
    hidden[2, [1, 2]] = 1.0                                                 # a NaN and an infinity hidden
    y = nn.adjust_logits(hip_tensor(x), hip_tensor(history), None, 2.0, hidden=hip_tensor(hidden)).numpy()
    if hip.COMPILE_ONLY:
        return
    want = np.array([0.5, np.nan, np.inf, -np.inf, -4.0, 1.7e38, -np.inf, 0.0])
    np.testing.assert_array_equal(y[0], want.astype(f32))
    assert (y[1] == -np.inf).all()
    np.testing.assert_array_equal(y[2], np.where(hidden[2] > 0, -np.inf, want).astype(f32))


@pytest.mark.gpu
def test_adjust_logits_lengths_beyond_the_history():
    require_gpu()
    x = np.arange(40, dtype=f32).reshape(4, 10) + 1
    history = np.array([[1, 2, 3]] * 4, f32)
    n = np.array([[-5], [100], [np.nan], [1.9]], f32)
    y = nn.adjust_logits(hip_tensor(x), hip_tensor(history), hip_tensor(n), 2.0).numpy()
    want = x.copy()
    want[1, 1:4] /= 2
    want[3, 1] /= 2
    same(y, want)


@pytest.mark.gpu
def test_adjust_logits_on_host_and_device_agree(monkeypatch):
    require_gpu()
    rng = np.random.default_rng(4)
    x, history = rng.standard_normal((3, 130)).astype(f32), rng.integers(-2, 140, (3, 60)).astype(f32)
    kw = dict(repetition=1.5, presence=0.25, frequency=0.5)               # (exact in fp32, so that the order of operations does not matter)
    a = nn.adjust_logits(hip_tensor(x), hip_tensor(history), hip_tensor([[60], [3], [0]]), **kw).numpy()
    b = nn.adjust_logits(Tensor(x), Tensor(history), Tensor(np.array([[60], [3], [0]], f32)), **kw).numpy()
    within(a, b, 4 * EPS * 40)
    within(b, adjusted(x, history, [60, 3, 0], [1.5] * 3, [0.25] * 3, [0.5] * 3), 4 * EPS * 40)


def test_adjust_logits_on_the_cpu_and_refusals():
    x = np.array([[1.0, -1.0, 2.0]], f32)
    y = nn.adjust_logits(Tensor(x), Tensor(np.array([[0, 1, 1]], f32)), repetition=2.0, frequency=0.5, hidden=Tensor(np.array([0, 0, 1], f32)))
    np.testing.assert_array_equal(y.numpy(), np.array([[0.0, -3.0, -np.inf]], f32))
    t, z = Tensor(x), lambda *s: Tensor(np.zeros(s, f32))          # noqa: E731
    for bad in (dict(repetition=0.0), dict(repetition=-1.0), dict(repetition=float("nan")), dict(presence=float("inf")), dict(history=z(2, 3)),
                dict(history=z(3)), dict(lengths=z(1)), dict(history=z(1, 3), lengths=z(2)), dict(bias=z(4)), dict(hidden=z(3, 1)), dict(bias=z(2, 3)),
                dict(repetition=z(2)), dict(history=Tensor(1.0))):
        with pytest.raises(ValueError):
            nn.adjust_logits(t, **bad)
    with pytest.raises(ValueError):
        nn.adjust_logits(z(3))
    with pytest.raises(ValueError, match="no gradient"):
        nn.adjust_logits(Tensor(x, requires_grad=True))
    with nn.inference():
        nn.adjust_logits(Tensor(x, requires_grad=True))


def test_adjust_logits_refuses_numbers_that_fp32_does_not_hold():
    x, h = Tensor(np.ones((1, 3), f32)), Tensor(np.zeros((1, 1), f32))
    for bad in (dict(repetition=1e-50), dict(repetition=1e300), dict(presence=1e39), dict(frequency=-1e39), dict(presence=float("nan")), dict(frequency=float("-inf"))):
        with pytest.raises(ValueError, match=next(iter(bad))):
            nn.adjust_logits(x, h, **bad)
    nn.adjust_logits(x, h, repetition=2, presence=-3, frequency=np.float32(0.5))


@pytest.mark.parametrize("which", ["repetition", "presence", "frequency", "bias"])
def test_adjust_logits_refuses_to_stop_a_gradient(which):
    x, h = Tensor(np.ones((2, 3), f32)), Tensor(np.zeros((2, 1), f32))
    t = Tensor(np.ones((2, 3) if which == "bias" else (2, 1), f32), requires_grad=True)
    with pytest.raises(ValueError, match="no gradient"):
        nn.adjust_logits(x, h, **{which: t})
    with nn.inference():
        nn.adjust_logits(x, h, **{which: t})
    nn.adjust_logits(x, h, **{which: t.detach()})


# ================================================================ the 8-bit cache
def held(rows, whole):
    """rows (n, H, d) as the cache stands for them: the first `whole` tokens in blocks of 64 per head, scale = max / 127 in fp32,
    the quotient in float64 to the nearest whole number; the rest as they are."""
    out = np.array(rows, f32)
    for at in range(0, whole, BLOCK):
        blk = rows[at:at + BLOCK]
        s = (np.abs(blk).max((0, 2)) / f32(127)).astype(f32)[None, :, None]
        with np.errstate(all="ignore"):
            q = np.where(s > 0, np.rint(blk.astype(np.float64) / s.astype(np.float64)), 0.0)
        with np.errstate(over="ignore"):                                     # (127 scales of the largest number may round beyond it)
            out[at:at + BLOCK] = np.clip(q, -127, 127).astype(f32) * s
    return out


def attended(q, k, v, first, scale, H):
    """float64: q (T, Hq, d) at positions first .. over k, v (n, H, d); also the bound on the result's error.

    A score is a sum of d products in fp32 accumulators, off by at most d roundings of sum |q k| scale, and by 2^-22 of it for the
    two 16-bit floats of a query element; a probability is off by twice that and 2^-22 for the exponential, its two 16-bit floats
    and the running maximum's factors; the sums over the tokens go block by block: 64 + n / 64 + 40 roundings of max |v|."""
    T, Hq, d = q.shape
    y, tol = np.zeros((T, Hq, d)), np.zeros((T, Hq, d))
    G = Hq // H
    for j in range(Hq):
        for t in range(T):
            n = first + t + 1
            kk, vv, qq = k[:n, j // G].astype(np.float64), v[:n, j // G].astype(np.float64), q[t, j].astype(np.float64)
            s = kk @ qq * scale
            p = np.exp(s - s.max())
            p /= p.sum()
            y[t, j] = p @ vv
            ds = (np.abs(kk) @ np.abs(qq) * scale).max() * (d * EPS + 2.0 ** -22)
            tol[t, j] = np.abs(vv).max() * (2 * ds + 2.0 ** -21 + (64 + n / 64 + 40) * EPS)
    return y, tol


def filled(B, cap, H, d, hist, counts=None, **kw):
    cache = nn.QuantizedKVCache(B, cap, H, d, **kw)
    k, v = hist
    if k.shape[1]:
        c = None if counts is None else hip_tensor(np.asarray(counts).reshape(B, 1))
        cache.write(hip_tensor(k), hip_tensor(v), counts=c)
        cache.advance(k.shape[1] if c is None else c)
    return cache


def rows_of(rng, B, n, C):
    wide = 0.25 + rng.random(C)
    return (rng.standard_normal((B, n, C)) * wide).astype(f32), rng.standard_normal((B, n, C)).astype(f32)


@pytest.mark.gpu
@pytest.mark.parametrize("H,d", [(2, 64), (1, 32), (3, 40), (2, 128), (1, 7), (2, 96), (1, 256), (1, 130)])
def test_cache_holds_the_same_however_the_tokens_arrive(H, d):
    """All at once, in uneven pieces, one at a time, padded: bit for bit what the definition gives."""
    require_gpu()
    rng = np.random.default_rng(d)
    B, n, C = 2, 203, H * d
    k, v = rows_of(rng, B, n, C)
    want = [np.stack([held(a[b].reshape(n, H, d), n // BLOCK * BLOCK).reshape(n, C) for b in range(B)]) for a in (k, v)]
    for pieces in ([203], [1, 62, 1, 1, 64, 74], [65, 130, 8], [64, 64, 75], [100, 103], [20, 128 + 10, 45]):
        cache, at = nn.QuantizedKVCache(B, 256, H, d), 0
        for m in pieces:
            kk, vv = hip_tensor(k[:, at:at + m]), hip_tensor(v[:, at:at + m])
            cache.write(kk, vv)
            if at % 64 == 0 or m <= 64:
                cache.write(kk, vv)                                         # a write may be repeated
            got = cache.read(at + m, new=m)
            cache.advance(m)
            at += m
            for a, b in zip(got, cache.read(at)):
                same(a.numpy(), b.numpy(), "before and after advance")
        for a, b, name in zip(cache.read(n), want, "kv"):
            same(a.numpy(), b, f"{name} in pieces {pieces}")
        wide = cache.read(256)[0].numpy()
        if not hip.COMPILE_ONLY:
            assert (wide[:, n:] == 0).all()
    cache, at = nn.QuantizedKVCache(B, 256, H, d), 0                         # sequences that grow at different speeds, padded rows between
    done = np.zeros(B, int)
    while done.min() < 130:
        m = np.minimum(rng.integers(0, 48, B), n - done)
        T = 48
        kk, vv = np.full((B, T, C), 9e9, f32), np.full((B, T, C), np.nan, f32)
        for b in range(B):
            kk[b, :m[b]], vv[b, :m[b]] = k[b, done[b]:done[b] + m[b]], v[b, done[b]:done[b] + m[b]]
        c = hip_tensor(m.reshape(B, 1))
        cache.write(hip_tensor(kk), hip_tensor(vv), counts=c)
        cache.advance(c)
        done += m
    for a, src in zip(cache.read(256), (k, v)):
        for b in range(B):
            if not hip.COMPILE_ONLY:
                same(a.numpy()[b, :done[b]], held(src[b, :done[b]].reshape(-1, H, d), done[b] // BLOCK * BLOCK).reshape(-1, C))
                assert (a.numpy()[b, done[b]:] == 0).all()


@pytest.mark.gpu
def test_cache_rounds_exactly():
    """Ties, neighbours of ties, denormal and huge blocks, and blocks of zeros."""
    require_gpu()
    rng = np.random.default_rng(0)
    d, blocks = 32, []
    for unit in (1.0, 0.1, 3.0, 1e-30, 1e-41, 2.5e36, 7.0 / 127):
        s = f32(f32(127 * unit) / f32(127))
        b = ((rng.integers(-127, 127, (BLOCK, d)) + 0.5) * np.float64(s)).astype(f32)      # halves, or as near as fp32 comes
        b[::3] = np.nextafter(b[::3], f32(0))
        b[1::3] = np.nextafter(b[1::3], f32(np.inf))
        b = np.clip(b, -f32(127 * unit), f32(127 * unit))
        b[0, 0] = f32(127 * unit)
        blocks.append(b)
    blocks += [np.zeros((BLOCK, d), f32), np.full((BLOCK, d), 1e-45, f32), np.full((BLOCK, d), 3.4028235e38, f32), -np.full((BLOCK, d), 9e-44, f32)]
    x = np.concatenate(blocks)[None]
    cache = filled(1, x.shape[1], 1, d, (x, -x))
    k, v = cache.read(x.shape[1])
    want = held(x[0].reshape(-1, 1, d), x.shape[1]).reshape(x.shape)
    same(k.numpy(), want)
    same(v.numpy(), -want)


ATTEND = [  # B, H, G, d, tokens held, new, capacity
    (1, 4, 1, 32, 0, 1, 64), (1, 1, 1, 64, 62, 1, 128), (2, 3, 1, 64, 63, 1, 128), (2, 2, 2, 64, 64, 1, 200), (1, 2, 3, 40, 129, 1, 256),
    (3, 2, 8, 128, 500, 1, 512), (1, 1, 17, 64, 200, 1, 256), (1, 2, 1, 256, 100, 1, 128), (2, 1, 2, 7, 77, 1, 128),
    (1, 1, 1, 64, 5000, 1, 5056), (1, 2, 4, 96, 3000, 3, 3200), (2, 2, 1, 64, 0, 150, 256), (1, 2, 2, 32, 64, 130, 256), (2, 1, 3, 64, 45, 37, 128),
    (1, 1, 5, 130, 60, 9, 128), (1, 1, 1, 16, 1, 63, 64),
]


@pytest.mark.gpu
@pytest.mark.parametrize("B,H,G,d,n,T,cap", ATTEND)
def test_cache_attention(B, H, G, d, n, T, cap):
    require_gpu()
    rng = np.random.default_rng(n + d)
    k, v = rows_of(rng, B, n + T, H * d)
    q = rng.standard_normal((B, T, H * G * d)).astype(f32) * f32(1.5)
    lens = [n - (b * n) // (2 * B) for b in range(B)] if T <= 64 else [n] * B
    cache = filled(B, cap, H, d, (k[:, :n], v[:, :n]), lens)
    new = [np.stack([a[b, lens[b]:lens[b] + T] for b in range(B)]) for a in (k, v)]
    cache.write(hip_tensor(new[0]), hip_tensor(new[1]))
    scale = 0.7 * d ** -0.5
    y = cache.attend(hip_tensor(q), scale).numpy()
    assert y.shape == q.shape
    for b in range(B):
        m = lens[b] + T
        kk, vv = (held(a[b, :m].reshape(m, H, d), m // BLOCK * BLOCK) for a in (k, v))
        want, tol = attended(q[b].reshape(T, H * G, d), kk, vv, lens[b], scale, H)
        within(y[b].reshape(T, H * G, d), want, tol, f"sequence {b}")
    same(cache.attend(hip_tensor(q), scale).numpy(), y, "again")


@pytest.mark.gpu
@pytest.mark.parametrize("tiles,waves,splits,stream", [(2, 4, 1, False), (2, 4, 3, False), (1, 8, 1, True), (1, 8, 2, False), (1, 4, 64, True)])
@pytest.mark.parametrize("B,H,G,d,n,T,cap", [(2, 2, 1, 64, 70, 150, 256), (1, 2, 3, 32, 300, 21, 512), (2, 1, 1, 64, 200, 1, 256), (1, 1, 2, 128, 700, 1, 768), (1, 2, 1, 40, 0, 33, 64)])
def test_cache_attention_in_every_form(B, H, G, d, n, T, cap, tiles, waves, splits, stream, monkeypatch):
    """The forms that the sizes choose between, forced on sizes where the others would run."""
    if d > 64 and (tiles > 1 or waves > 4):
        tiles, waves = 1, 4
    monkeypatch.setattr(HIPLM, "attend_tiles", staticmethod(lambda *a: tiles))
    monkeypatch.setattr(HIPLM, "attend_waves", staticmethod(lambda *a: waves))
    monkeypatch.setattr(HIPLM, "attend_splits", staticmethod(lambda *a: splits))
    monkeypatch.setattr(HIPLM, "attend_streams", staticmethod(lambda *a: stream))
    if n % 64 and T > 64:
        n = n // 64 * 64
    test_cache_attention(B, H, G, d, n, T, cap)


@pytest.mark.gpu
@pytest.mark.parametrize("H,d", [(1, 192), (2, 161), (1, 224), (2, 200)])
def test_cache_of_wide_heads(H, d):
    test_cache_holds_the_same_however_the_tokens_arrive(H, d)
    test_cache_attention(1, H, 2, d, 200, 3, 256)


@pytest.mark.gpu
@pytest.mark.parametrize("splits,stream", [(1, True), (3, False), (2, True)])
@pytest.mark.parametrize("d", [96, 130, 192, 224, 256])
def test_cache_attention_of_wide_heads_in_every_form(d, splits, stream, monkeypatch):
    """Parts joined and loads past the caches, which long caches of such heads take."""
    require_gpu()
    monkeypatch.setattr(HIPLM, "attend_splits", staticmethod(lambda *a: splits))
    monkeypatch.setattr(HIPLM, "attend_streams", staticmethod(lambda *a: stream))
    test_cache_attention(1, 2, 3, d, 300, 21, 512)


@pytest.mark.gpu
def test_cache_attention_of_many_rows():
    """Enough query rows for two tiles a wavefront: the bits that a launch of its own, one tile a wavefront, gives for each sequence."""
    require_gpu()
    rng = np.random.default_rng(31)
    B, H, d, T = 8, 12, 32, 256
    assert HIPLM.attend_tiles(T, B * H, 32, 256) == 2 and HIPLM.attend_tiles(T, H, 32, 256) == 1
    k, v = rows_of(rng, B, T, H * d)
    q = rng.standard_normal((B, T, H * d)).astype(f32)
    cache = nn.QuantizedKVCache(B, T, H, d)
    cache.write(hip_tensor(k), hip_tensor(v))
    y = cache.attend(hip_tensor(q)).numpy()
    for b in range(0, B, 3):
        one = nn.QuantizedKVCache(1, T, H, d)
        one.write(hip_tensor(k[b:b + 1]), hip_tensor(v[b:b + 1]))
        same(y[b:b + 1], one.attend(hip_tensor(q[b:b + 1])).numpy(), f"sequence {b}")
    kk, vv = (held(a[0].reshape(T, H, d), T) for a in (k, v))
    want, tol = attended(q[0].reshape(T, H, d), kk, vv, 0, d ** -0.5, H)
    within(y[0].reshape(T, H, d), want, tol)


@pytest.mark.gpu
def test_cache_attention_of_extreme_queries():
    """Scores far apart (one token takes all the weight), tiny and huge queries, zeros."""
    require_gpu()
    rng = np.random.default_rng(8)
    n, d = 300, 64
    k, v = rows_of(rng, 1, n, d)
    cache = filled(1, 320, 1, d, (k[:, :-1], v[:, :-1]))
    cache.write(hip_tensor(k[:, -1:]), hip_tensor(v[:, -1:]))
    kk, vv = (held(a[0].reshape(n, 1, d), n // BLOCK * BLOCK) for a in (k, v))
    for size in (0.0, 1e-38, 1e-20, 1.0, 30.0):
        q = (rng.standard_normal((1, 1, d)) * size).astype(f32)
        want, tol = attended(q.reshape(1, 1, d), kk, vv, n - 1, 0.125, 1)
        within(cache.attend(hip_tensor(q)).numpy().reshape(1, 1, d), want, tol, f"queries of {size}")


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [-0.3, 0.0, 1e-30, 4.0])
def test_cache_attention_with_any_scale(scale):
    require_gpu()
    rng = np.random.default_rng(18)
    n, d = 150, 64
    k, v = rows_of(rng, 1, n, d)
    cache = filled(1, 192, 1, d, (k[:, :-1], v[:, :-1]))
    cache.write(hip_tensor(k[:, -1:]), hip_tensor(v[:, -1:]))
    kk, vv = (held(a[0].reshape(n, 1, d), n // BLOCK * BLOCK) for a in (k, v))
    q = rng.standard_normal((1, 1, 2 * d)).astype(f32)
    want, tol = attended(q.reshape(1, 2, d), kk, vv, n - 1, scale, 1)
    if scale < 0:
        tol = attended(q.reshape(1, 2, d), -kk, vv, n - 1, -scale, 1)[1]       # the same scores, a bound of the right sign
    within(cache.attend(hip_tensor(q), scale).numpy().reshape(1, 2, d), want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 40])
def test_cache_of_unaligned_views(d):
    """Queries, keys and values four bytes off a 16-byte boundary: the same bits."""
    require_gpu()
    rng = np.random.default_rng(19)
    k, v = rows_of(rng, 2, 70, 2 * d)
    q = rng.standard_normal((2, 70, 4 * d)).astype(f32)

    def off(a):
        room = Buffer.from_numpy(np.concatenate([np.zeros(1, f32), a.reshape(-1)]), Device.HIP)
        return Tensor(Buffer(room.ptr + 1, a.shape, Device.HIP))
    got = []
    for make in (hip_tensor, off):
        cache = nn.QuantizedKVCache(2, 128, 2, d)
        cache.write(make(k), make(v))
        got.append([cache.attend(make(q)).numpy(), *[t.numpy() for t in cache.read(70, new=70)]])
    for a, b in zip(*got):
        same(a, b)


@pytest.mark.gpu
def test_cache_padding_and_empty_sequences():
    """Rows beyond counts give zeros and are not seen; a sequence without tokens gives zeros."""
    require_gpu()
    rng = np.random.default_rng(6)
    B, H, G, d, T = 4, 2, 2, 64, 40
    k, v = rows_of(rng, B, T, H * d)
    q = rng.standard_normal((B, T, H * G * d)).astype(f32)
    n = np.array([40, 7, 0, 1])
    for b in range(B):
        k[b, n[b]:], v[b, n[b]:], q[b, n[b]:] = np.nan, np.inf, np.nan
    cache, c = nn.QuantizedKVCache(B, 128, H, d), hip_tensor(n.reshape(B, 1))
    cache.write(hip_tensor(k), hip_tensor(v), counts=c)
    y = cache.attend(hip_tensor(q), counts=c).numpy()
    if hip.COMPILE_ONLY:
        return
    for b in range(B):
        assert (y[b, n[b]:] == 0).all()
        if n[b]:
            want, tol = attended(q[b, :n[b]].reshape(n[b], H * G, d), k[b, :n[b]].reshape(-1, H, d), v[b, :n[b]].reshape(-1, H, d), 0, d ** -0.5, H)
            within(y[b, :n[b]].reshape(want.shape), want, tol, f"sequence {b}")
    zero = hip_tensor(np.zeros((B, 1)))
    assert (nn.QuantizedKVCache(B, 64, H, d).attend(hip_tensor(np.ones((B, 1, H * G * d))), counts=zero).numpy() == 0).all()
    assert cache.attend(Tensor.full((B, 0, H * d), 0.0, device="hip")).shape == (B, 0, H * d)


@pytest.mark.gpu
def test_cache_keeps_a_nan_to_those_who_see_it():
    """A poisoned row in the tail: the queries before it are as if it were not there, it and those after are NaN; once its block is
    full, everything that sees the block is NaN -- in its own head only."""
    require_gpu()
    rng = np.random.default_rng(7)
    H, d, T = 2, 32, 30
    for poison in (np.nan, np.inf, -np.inf):
        for which in (0, 1):
            k, v = rows_of(rng, 1, 140, H * d)
            q = rng.standard_normal((1, 140, H * d)).astype(f32)
            (k, v)[which][0, 20, 5] = poison                                    # head 0, position 20
            cache = nn.QuantizedKVCache(1, 192, H, d)
            cache.write(hip_tensor(k[:, :T]), hip_tensor(v[:, :T]))
            y = cache.attend(hip_tensor(q[:, :T])).numpy()
            if hip.COMPILE_ONLY:
                continue
            assert np.isnan(y[0, 20:, :d]).all() and np.isfinite(y[0, :20]).all() and np.isfinite(y[0, :, d:]).all()
            want, tol = attended(q[0, :20].reshape(20, H, d), k[0, :20].reshape(20, H, d), v[0, :20].reshape(20, H, d), 0, d ** -0.5, H)
            within(y[0, :20].reshape(20, H, d), want, tol)
            cache.advance(T)
            cache.write(hip_tensor(k[:, T:140]), hip_tensor(v[:, T:140]))
            y = cache.attend(hip_tensor(q[:, T:140])).numpy()
            assert np.isnan(y[0, :, :d]).all() and np.isfinite(y[0, :, d:]).all()
            got = cache.read(140, new=110)
            assert np.isnan(got[0].numpy()[0, :64, :d]).all() and np.isfinite(got[0].numpy()[0, 64:]).all() and np.isfinite(got[1].numpy()[0, :, d:]).all()


@pytest.mark.gpu
def test_cache_that_is_full_drops_the_rest():
    require_gpu()
    rng = np.random.default_rng(1)
    k, v = rows_of(rng, 2, 200, 32)
    cache = nn.QuantizedKVCache(2, 100, 1, 32)                                  # 128 in whole blocks
    assert cache.capacity == 128
    c = hip_tensor([[100], [20]])
    cache.write(hip_tensor(k[:, :100]), hip_tensor(v[:, :100]), counts=c)
    cache.advance(c)
    cache.write(hip_tensor(k[:, 100:]), hip_tensor(v[:, 100:]))
    y = cache.attend(hip_tensor(k[:, 100:])).numpy()
    cache.advance(100)
    got = cache.read(128)[0].numpy()
    if hip.COMPILE_ONLY:
        return
    same(got[0], held(k[0, :128].reshape(-1, 1, 32), 128).reshape(128, 32))
    same(got[1, :120], held(np.concatenate([k[1, :20], k[1, 100:]])[:120].reshape(-1, 1, 32), 64).reshape(120, 32))
    assert cache.lengths.numpy().reshape(-1).tolist() == [128, 120]
    assert (y[0, 28:] == 0).all() and (y[0, :28] != 0).all() and (y[1] != 0).all()


@pytest.mark.gpu
def test_cache_goes_back_over_rows_that_were_not_kept():
    """Sixty-four rows are tried, some are kept, others take their place: as if only the kept ones had been written."""
    require_gpu()
    rng = np.random.default_rng(12)
    k, v = rows_of(rng, 1, 230, 64)
    bad = rows_of(rng, 1, 64, 64)
    cache, at = nn.QuantizedKVCache(1, 256, 2, 32), 0
    for keep, tried in ((50, 64), (0, 64), (14, 30), (33, 64), (63, 64), (1, 1), (40, 64), (29, 50)):
        kk, vv = (np.concatenate([a[:, at:at + keep], w[:, keep:tried]], 1) for a, w in ((k, bad[0]), (v, bad[1])))
        cache.write(hip_tensor(kk), hip_tensor(vv))
        cache.advance(keep)
        at += keep
        same(cache.read(at)[0].numpy()[0], held(k[0, :at].reshape(-1, 2, 32), at // 64 * 64).reshape(at, 64), f"after {at}")
    assert at == 230
    same(cache.read(at)[1].numpy()[0], held(v[0].reshape(-1, 2, 32), at // 64 * 64).reshape(at, 64))


@pytest.mark.gpu
def test_cache_goes_on_from_less_than_a_long_write():
    """Rows that a long write did not leave in fp32 are NaN where they are needed, and not the rows of other tokens."""
    require_gpu()
    rng = np.random.default_rng(40)
    k, v = rows_of(rng, 1, 200, 32)
    q = rng.standard_normal((1, 1, 32)).astype(f32)
    one = lambda: [hip_tensor(a) for a in rows_of(rng, 1, 1, 32)]                                   # noqa: E731

    def check(cache, n, right, what):
        got = [t.numpy()[0] for t in cache.read(n)]
        cache.write(*one())
        y = cache.attend(hip_tensor(q)).numpy()
        if hip.COMPILE_ONLY:
            return
        for a, src in zip(got, (k, v)):
            want = held(src[0, :n].reshape(n, 1, 32), n // 64 * 64).reshape(n, 32)
            same(a[:n // 64 * 64], want[:n // 64 * 64], what)
            if right:
                same(a, want, what)
            else:
                assert np.isnan(a[n // 64 * 64:]).all(), what
        assert np.isfinite(y).all() if right else np.isnan(y).all(), what

    for tried, n, right in ((200, 70, False), (200, 128, True), (200, 192, True), (200, 195, True), (130, 100, False), (130, 10, False), (128, 64, True), (100, 70, True), (100, 3, True)):
        cache = nn.QuantizedKVCache(1, 256, 1, 32)
        cache.write(hip_tensor(k[:, :tried]), hip_tensor(v[:, :tried]))
        cache.advance(n)
        check(cache, n, right, f"{tried} tried, {n} kept")
    cache = filled(1, 256, 1, 32, (k[:, :10], v[:, :10]))
    for time, right in (("once", True), ("twice", False)):                      # the second time the ten rows before it are gone
        cache.write(hip_tensor(k[:, 10:140]), hip_tensor(v[:, 10:140]))
        got = cache.read(140, new=130)[0].numpy()[0]
        if not hip.COMPILE_ONLY:
            same(got[64:], held(k[0, :140].reshape(140, 1, 32), 128).reshape(140, 32)[64:], time)
            assert np.isfinite(got[:64]).all() if right else np.isnan(got[:64]).all(), time
    cache = filled(1, 256, 1, 32, (k[:, :10], v[:, :10]))
    cache.write(hip_tensor(k[:, 50:70]), hip_tensor(v[:, 50:70]))                # tried, and given up for a longer one
    cache.write(hip_tensor(k[:, 10:200]), hip_tensor(v[:, 10:200]))
    cache.advance(15)
    got = cache.read(25)[0].numpy()[0]
    if not hip.COMPILE_ONLY:
        assert np.isnan(got).all()


@pytest.mark.gpu
def test_cache_advances_over_what_was_written():
    """Counts below zero, beyond the rows of the write, between two whole numbers and without a value are what write() takes them for."""
    require_gpu()
    rng = np.random.default_rng(43)
    B = 6
    k, v = rows_of(rng, B, 5, 32)
    c = np.array([[-3], [2.75], [9], [np.nan], [5], [0]], f32)
    for brought in (True, False):
        cache = nn.QuantizedKVCache(B, 128, 1, 32)
        cache.write(hip_tensor(k), hip_tensor(v))
        cache.advance(1)
        cache.write(hip_tensor(k), hip_tensor(v), counts=hip_tensor(c) if brought else None)
        cache.advance(hip_tensor(c))
        same(cache.lengths.numpy().reshape(-1), [1, 3, 6, 1, 6, 1])
        cache.advance(hip_tensor(np.full((B, 1), -1.0)))
        same(cache.lengths.numpy().reshape(-1), [1, 3, 6, 1, 6, 1], "never back")
        cache.advance(4)                                                      # what the write brought and was not taken yet
        same(cache.lengths.numpy().reshape(-1), [1, 3, 6, 1, 6, 1] if brought else [5, 6, 6, 5, 6, 5])
        got = cache.read(8)[0].numpy()
        if not hip.COMPILE_ONLY:
            for b, n in enumerate([1, 3, 6, 1, 6, 1] if brought else [5, 6, 6, 5, 6, 5]):
                same(got[b, :n], np.concatenate([k[b, :1], k[b]])[:n])
                assert (got[b, n:] == 0).all()
    whole = nn.QuantizedKVCache(1, 64, 1, 32, lengths=hip_tensor([[7.0]]))
    with pytest.raises(ValueError):
        whole.advance(1)                                                       # nothing was ever written
    whole.write(hip_tensor(k[:1, :2]), hip_tensor(v[:1, :2]))
    for bad in (3, float("inf"), float("nan"), -1, 0.5):
        with pytest.raises(ValueError):
            whole.advance(bad)
    whole.advance(1)
    same(whole.lengths.numpy(), [[8.0]])
    whole.reset()
    whole.advance(2)
    same(whole.lengths.numpy(), [[0.0]], "a reset forgets what was written")


def test_cache_runtime_refuses_to_advance_by_what_does_not_fit():
    """Host checks, before any device is touched."""
    from dlgrad_amd.runtime.hip_lm import Cache8

    class Ptr:
        addr, nbytes = 256, 1 << 40
    b = lambda *s: Buffer(Ptr(), s, Device.HIP)                  # noqa: E731
    c = Cache8.__new__(Cache8)
    c.batch, c.blocks, c.wrote = 2, 2, b(2, 1)
    for lengths, by in ((b(2), b(3)), (b(3), 1), (b(2), -1), (b(2), 2 ** 32), (b(2), Buffer.from_scalar(1.0)), (Buffer.from_scalar(1.0), 1)):
        with pytest.raises(ValueError):
            HIPLM.cache8_advance(c, lengths, by)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [40, 150])
def test_cache_attends_to_what_was_written(T):
    """Counts that only write() was given, more queries than rows, none written at all: what is there is attended to and read, the rest is zeros."""
    require_gpu()
    if hip.COMPILE_ONLY:
        return
    rng = np.random.default_rng(46)
    B, d, n = 4, 32, np.array([T, 30, 0, 1])
    k, v = rows_of(rng, B, T, d)
    q = rng.standard_normal((B, T, d)).astype(f32)
    cache, c = nn.QuantizedKVCache(B, 192, 1, d), hip_tensor(n.reshape(B, 1))
    assert (cache.attend(hip_tensor(q)).numpy() == 0).all() and (cache.read(T, new=T)[0].numpy() == 0).all()
    cache.write(hip_tensor(k), hip_tensor(v), counts=c)
    want = cache.attend(hip_tensor(q), counts=c).numpy()
    same(cache.attend(hip_tensor(q)).numpy(), want)
    for b in range(B):
        assert np.isfinite(want[b]).all() and (want[b, n[b]:] == 0).all()
        if n[b]:
            y, tol = attended(q[b, :n[b]].reshape(n[b], 1, d), *(held(a[b, :n[b]].reshape(n[b], 1, d), n[b] // 64 * 64) for a in (k, v)), 0, d ** -0.5, 1)
            within(want[b, :n[b]].reshape(y.shape), y, tol, f"sequence {b}")
    for a, z, w in zip(cache.read(T, new=T), cache.read(T, counts=c), (k, v)):
        same(a.numpy(), z.numpy())
        for b in range(B):
            same(a.numpy()[b, :n[b]], held(w[b, :n[b]].reshape(n[b], 1, d), n[b] // 64 * 64).reshape(n[b], d))
    cache.advance(c)
    assert (cache.attend(hip_tensor(q)).numpy() == 0).all()
    same(cache.read(192, new=5)[0].numpy(), cache.read(192)[0].numpy())


@pytest.mark.gpu
@pytest.mark.parametrize("seed", range(6))
def test_cache_gives_its_own_tokens_or_nan(seed):
    """Writes of any length, replaced and advanced over by any part of them: every position reads as its token, or as NaN in a block that
    the documentation says is gone."""
    require_gpu()
    if hip.COMPILE_ONLY:
        return
    rng = np.random.default_rng(seed)
    B, H, d, cap = 3, 2, 32, 1024
    C, at, gone = H * d, np.zeros(B, int), [set() for _ in range(B)]
    truth = np.zeros((2, B, cap, C), f32)
    cache = nn.QuantizedKVCache(B, cap, H, d)
    while at.max() < cap - 320:
        for again in range(rng.integers(1, 3)):
            T = int(rng.choice([1, 7, 64, 65, 130, 200, 300]))
            n = np.where(rng.random(B) < 0.5, T, rng.integers(0, T + 1, B))
            new = rows_of(rng, B, T, C)
            if again:
                for b in range(B):
                    if at[b] % 64 and before[b] > 64:
                        gone[b].add(at[b] // 64)
            cache.write(hip_tensor(new[0]), hip_tensor(new[1]), counts=hip_tensor(n.reshape(B, 1)))
            before = n
            for b in range(B):
                truth[:, b, at[b]:at[b] + n[b]] = [a[b, :n[b]] for a in new]
        m = np.where(rng.random(B) < 0.5, n, rng.integers(0, n + 1))
        for b in range(B):
            if n[b] > 64 and m[b] < n[b] and (at[b] + m[b]) % 64 and (at[b] + m[b]) // 64 != (at[b] + n[b]) // 64:
                gone[b].add((at[b] + m[b]) // 64)
        cache.advance(hip_tensor(m.reshape(B, 1)))
        at += m
        for name, a, src in zip("kv", cache.read(cap), truth):
            a = a.numpy()
            for b in range(B):
                want = held(src[b, :at[b]].reshape(-1, H, d), at[b] // 64 * 64).reshape(-1, C)
                for blk in range(-(-at[b] // 64)):
                    rows = slice(blk * 64, min(blk * 64 + 64, at[b]))
                    if not (blk in gone[b] and np.isnan(a[b, rows]).any()):
                        same(a[b, rows], want[rows], f"{name} of sequence {b}, block {blk}")
                assert (a[b, at[b]:] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("gap", [14, 24, 30, 36])
def test_cache_attention_adds_up_many_small_weights(gap):
    """2^20 tokens of weight 2^-gap beside one of weight 1, values around 1: together they move the result by up to 2^(20 - gap)."""
    require_gpu()
    rng = np.random.default_rng(gap)
    n, d = 1 << 20, 32
    k, v = np.zeros((1, n, d), f32), (1 + 0.25 * rng.standard_normal((1, n, d))).astype(f32)
    q, last = np.zeros((1, 1, d), f32), rng.standard_normal((1, 1, d)).astype(f32)
    q[0, 0, 3] = 2.0
    key = np.zeros((1, 1, d), f32)
    key[0, 0, 3] = gap * math.log(2) / 2                                  # the score of the last token: gap ln 2
    cache = filled(1, n + 64, 1, d, (k, v))
    cache.write(hip_tensor(key), hip_tensor(last))
    y = cache.attend(hip_tensor(q), 1.0).numpy().reshape(1, 1, d)
    want, tol = attended(q, np.concatenate([k[0], key[0]])[:, None], np.concatenate([held(v[0][:, None], n), last[0][:, None]]), n, 1.0, 1)
    # the sums over the tokens: a term is off by 2^-22 of itself, a partial sum by a rounding of the whole
    small = n * 2.0 ** -gap
    tol = np.abs(want) * (64 * EPS + 2 * gap * EPS) + small / (1 + small) * (2.0 ** -20 + (64 + n / 64 / 4) * EPS) * np.abs(v).max() + 16 * EPS * np.abs(last).max()
    within(y, want, tol, f"weights of 2^-{gap}")


@pytest.mark.gpu
@pytest.mark.parametrize("tiles,waves,splits", [(1, 4, 1), (2, 4, 1), (1, 8, 1), (1, 4, 3)])
@pytest.mark.parametrize("gap", [18.3, 26.7, 38.45])
def test_cache_attention_keeps_weights_far_below_the_largest(gap, tiles, waves, splits, monkeypatch):
    """2^18 tokens of weights around 2^-gap, no power of two among them, behind some of weight 1, one in each wavefront's first block, whose
    values are 0: all of the result is the others'.  A weight is off by 2^-22 of itself for the two 16-bit floats, or 2^-51 of the largest;
    by 2 roundings of its score; each partial sum by a rounding, of at most 64 + a wavefront's n / 256 blocks."""
    require_gpu()
    monkeypatch.setattr(HIPLM, "attend_tiles", staticmethod(lambda *a: tiles))
    monkeypatch.setattr(HIPLM, "attend_waves", staticmethod(lambda *a: waves))
    monkeypatch.setattr(HIPLM, "attend_splits", staticmethod(lambda *a: splits))
    rng = np.random.default_rng(44)
    n, d = 1 << 18, 32
    k, v = np.zeros((1, n, d), f32), (1 + 0.25 * rng.standard_normal((1, n, d))).astype(f32)
    k[0, :, 3] = -np.repeat(rng.uniform(0, 0.5, n // 64), 64)                 # scores down to -1, the same in a block
    for s in range(splits):
        for block in range(n // 64 * s // splits, n // 64 * s // splits + waves):
            k[0, block * 64 + 7, 3] = gap * math.log(2) / 2
            v[0, block * 64 + 7] = 0
    q = np.zeros((1, 1, d), f32)
    q[0, 0, 3] = 2.0
    cache = filled(1, n, 1, d, (k[:, :-1], v[:, :-1]))
    cache.write(hip_tensor(k[:, -1:]), hip_tensor(v[:, -1:]))
    y = cache.attend(hip_tensor(q), 1.0).numpy().reshape(d)
    kk, vv = held(k[0][:, None], n)[:, 0].astype(np.float64), held(v[0][:, None], n)[:, 0].astype(np.float64)
    w = np.exp(2 * (kk[:, 3] - kk[:, 3].max()))
    want, small = w @ vv / w.sum(), w[w < 0.5].sum()
    assert (w >= 0.5).sum() == splits * waves and small <= 4 * n * 2.0 ** -gap
    tol = np.abs(vv).max() / w.sum() * (small * (2.0 ** -22 + 2 * (gap + 2) * EPS + (64 + n / 256) * EPS) + n * 2.0 ** -51)
    within(y, want, tol, f"weights of 2^-{gap}")


@pytest.mark.gpu
@pytest.mark.parametrize("tiles,waves,splits", [(1, 4, 1), (2, 4, 1), (1, 8, 1), (1, 4, 3)])
@pytest.mark.parametrize("d", [32, 64])
def test_cache_attention_of_a_query_with_one_huge_element(d, tiles, waves, splits, monkeypatch):
    """An element 2^30 times the others, in a column where the keys are nothing: the others make the scores.  They are off by 2^-22 of
    themselves (in the common bound) or 2^-50 of the largest, 2^-20 here."""
    require_gpu()
    monkeypatch.setattr(HIPLM, "attend_tiles", staticmethod(lambda *a: tiles))
    monkeypatch.setattr(HIPLM, "attend_waves", staticmethod(lambda *a: waves))
    monkeypatch.setattr(HIPLM, "attend_splits", staticmethod(lambda *a: splits))
    rng = np.random.default_rng(45)
    n = 400
    k, v = rows_of(rng, 1, n, d)
    k[:, :, 5] = 0
    q = rng.standard_normal((1, 1, d)).astype(f32)
    q[0, 0, 5] = 2.0 ** 30
    cache = filled(1, n, 1, d, (k[:, :-1], v[:, :-1]))
    cache.write(hip_tensor(k[:, -1:]), hip_tensor(v[:, -1:]))
    kk, vv = (held(a[0].reshape(n, 1, d), n // 64 * 64) for a in (k, v))
    want, tol = attended(q.reshape(1, 1, d), kk, vv, n - 1, 0.2, 1)
    tol = tol + np.abs(vv).max() * 2 * np.abs(kk).sum(2).max() * 0.2 * 2.0 ** (30 - 50)
    within(cache.attend(hip_tensor(q), 0.2).numpy().reshape(1, 1, d), want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("tiles,waves,splits", [(1, 4, 1), (2, 4, 1), (1, 8, 1), (1, 4, 3)])
@pytest.mark.parametrize("G,later", [(1, 0.0), (3, 0.0), (1, 1e-36)])
def test_cache_attention_beside_a_block_of_zero_keys(G, later, tiles, waves, splits, monkeypatch):
    """Scores far below zero in the first block, keys of nothing (or next to it) in the second: a query that sees none of the second is
    not moved by its scores, though it shares a tile with queries that do."""
    require_gpu()
    monkeypatch.setattr(HIPLM, "attend_tiles", staticmethod(lambda *a: tiles))
    monkeypatch.setattr(HIPLM, "attend_waves", staticmethod(lambda *a: waves))
    monkeypatch.setattr(HIPLM, "attend_splits", staticmethod(lambda *a: splits))
    rng = np.random.default_rng(17)
    first, T, d = 8, 130, 64
    n = first + T
    k, v = rows_of(rng, 1, n, d)
    k = (-5 + 0.125 * k).astype(f32)                                      # scores around -320: exp of them is nothing in 32 bits
    k[:, 64:] = later
    q = np.ones((1, T, G * d), f32)
    cache = filled(1, n, 1, d, (k[:, :first], v[:, :first]))
    cache.write(hip_tensor(k[:, first:]), hip_tensor(v[:, first:]))
    y = cache.attend(hip_tensor(q), 1.0).numpy().reshape(T, G, d)
    kk, vv = (held(a[0].reshape(n, 1, d), n // 64 * 64) for a in (k, v))
    want, tol = attended(q[0].reshape(T, G, d), kk, vv, first, 1.0, 1)
    within(y, want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("tiles,waves,splits", [(1, 4, 1), (2, 4, 1), (1, 8, 1), (1, 4, 2)])
@pytest.mark.parametrize("size", [1e4, 1e6, 1e8, 1e10, 1e16])
@pytest.mark.parametrize("T", [1, 70])
def test_cache_attention_of_scores_beyond_whole_numbers(T, size, tiles, waves, splits, monkeypatch):
    """Scores so large that neighbouring numbers of 32 bits lie far apart: one token takes all the weight, and nothing overflows."""
    require_gpu()
    monkeypatch.setattr(HIPLM, "attend_tiles", staticmethod(lambda *a: tiles))
    monkeypatch.setattr(HIPLM, "attend_waves", staticmethod(lambda *a: waves))
    monkeypatch.setattr(HIPLM, "attend_splits", staticmethod(lambda *a: splits))
    rng = np.random.default_rng(41)
    first, d = 600, 64
    n = first + T
    k, v = rows_of(rng, 1, n, d)
    q = (rng.standard_normal((1, T, 4 * d)) * size).astype(f32)
    cache = filled(1, n, 1, d, (k[:, :first], v[:, :first]))
    cache.write(hip_tensor(k[:, first:]), hip_tensor(v[:, first:]))
    y = cache.attend(hip_tensor(q), 0.125).numpy().reshape(T, 4, d)
    assert np.isfinite(y).all()
    kk, vv = (held(a[0].reshape(n, 1, d), n // 64 * 64)[:, 0] for a in (k, v))
    alone = 0
    for t in range(T):
        for j in range(4):
            s = kk[:first + t + 1].astype(np.float64) @ q[0, t, j * d:(j + 1) * d].astype(np.float64) * 0.125
            # a score is off by (d + 4) roundings of the largest sum of |q k|; where the best one leads by more than 40 and that, it is alone
            off = (np.abs(kk[:first + t + 1]) @ np.abs(q[0, t, j * d:(j + 1) * d])).max() * 0.125 * (d + 4) * EPS
            two = np.partition(s, -2)[-2:]
            if two[1] - two[0] > 40 + 4 * off:
                alone += 1
                # exp(-40) of 670 others is nothing; the weight and its reciprocal are off by 2^-21 and four roundings
                within(y[t, j], vv[s.argmax()], np.abs(vv).max() * (2.0 ** -21 + 4 * EPS), f"row {t}, head {j}")
    assert alone >= 3 * T


@pytest.mark.gpu
def test_cache_beyond_four_gigabytes():
    """Offsets past 32 bits: blocks that were never written have scale 0, so their tokens weigh exp(0) and add nothing."""
    require_gpu()
    rng = np.random.default_rng(2)
    H, d, cap = 3, 128, 1 << 24
    if hip.COMPILE_ONLY:
        return
    cache = nn.QuantizedKVCache(1, cap, H, d)
    assert cache.layers[0].kc.nbytes > 1 << 32
    n = cap - 130
    k, v = rows_of(rng, 1, 131, H * d)
    cache.lengths.data.upload_(np.array([[n - n % 64]], f32))
    first = n - n % 64
    cache.write(hip_tensor(k[:, :130]), hip_tensor(v[:, :130]))
    cache.advance(130)
    cache.write(hip_tensor(k[:, 130:]), hip_tensor(v[:, 130:]))
    q = rng.standard_normal((1, 1, H * d)).astype(f32)
    y = cache.attend(hip_tensor(q)).numpy().reshape(H, d)
    kk, vv = (held(a[0].reshape(-1, H, d), 128) for a in (k, v))
    for h in range(H):
        s = kk[:, h].astype(np.float64) @ q.reshape(H, d)[h] * d ** -0.5
        want = (np.exp(s) @ vv[:, h].astype(np.float64)) / (np.exp(s).sum() + first)
        tol = np.abs(vv).max() * np.exp(s).sum() / first * (2 * np.abs(s).max() * 130 * EPS + 2.0 ** -20) + np.abs(want) * (64 + first / 64) * EPS
        within(y[h], want, tol, f"head {h}")


@pytest.mark.gpu
def test_cache_steps_in_a_captured_graph():
    """Two graphs over one cache, replayed in turns with eager calls and synchronizations between: every replay as the eager step."""
    require_gpu()
    if hip.COMPILE_ONLY:
        return
    rng = np.random.default_rng(5)
    B, H, G, d, total = 2, 2, 2, 64, 150
    k, v = rows_of(rng, B, total, H * d)
    q = rng.standard_normal((B, total, H * G * d)).astype(f32)
    plain, cache = nn.QuantizedKVCache(B, 256, H, d), nn.QuantizedKVCache(B, 256, H, d)
    kt, vt, qt = (hip_tensor(np.zeros((B, 1, a.shape[2]))) for a in (k, v, q))

    def step():
        cache.write(kt, vt)
        return cache.attend(qt)

    def both():
        y = step()
        cache.advance(1)
        return y
    graphs = []
    for fn in (step, both):
        g = hip.Graph()
        with g.arena():
            fn()
        with g.capture():
            out = fn()
        graphs.append((g, out))
    cache.reset()
    for t in range(total):
        kk, vv, qq = k[:, t:t + 1], v[:, t:t + 1], q[:, t:t + 1]
        plain.write(hip_tensor(kk), hip_tensor(vv))
        want = plain.attend(hip_tensor(qq)).numpy()
        plain.advance(1)
        for dst, src in ((kt, kk), (vt, vv), (qt, qq)):
            dst.data.upload_(np.ascontiguousarray(src))
        for g, out in graphs:
            g.replay()
            if t % 7 == 0:
                hip.lib().sync()
            same(out.numpy(), want, f"token {t}")
        assert cache.lengths.numpy().reshape(-1).tolist() == [t + 1] * B
    for g, _ in graphs:
        g.close()


@pytest.mark.gpu
def test_cache_takes_the_memory_that_is_documented():
    """Percent of the bytes of two fp32 stores of the same tokens."""
    require_gpu()
    for tokens, d, percent in ((128, 32, 125), (128, 64, 125), (192, 64, 92), (1024, 64, 37.5), (32768, 128, 25.5), (1024, 40, 60), (32768, 40, 41), (32768, 16, 51)):
        cache = nn.QuantizedKVCache(2, tokens, 3, d)
        assert abs(100 * cache.nbytes / (2 * 3 * tokens * 8 * d) - percent) < 0.6, (tokens, d)


@pytest.mark.gpu
def test_cache_of_several_layers_and_shared_lengths():
    require_gpu()
    rng = np.random.default_rng(3)
    slot = Tensor.full((1, 1), 0.0, device="hip")
    cache = nn.QuantizedKVCache(1, 64, 1, 32, layers=3, lengths=slot)
    data = [rows_of(rng, 1, 5, 32) for _ in range(3)]
    for i, (k, v) in enumerate(data):
        cache.write(hip_tensor(k), hip_tensor(v), layer=i)
    slot.data.upload_(np.array([[5.0]], f32))
    for i, (k, v) in enumerate(data):
        same(cache.read(5, layer=i)[0].numpy(), k)
        same(cache.read(5, layer=i)[1].numpy(), v)
    with pytest.raises(IndexError):
        cache.read(5, layer=3)
    assert cache.nbytes == 3 * (2 * 64 * 32 + 8 + 2 * 2 * 64 * 32 * 4)


@pytest.mark.gpu
def test_cache_refusals():
    require_gpu()
    cache = nn.QuantizedKVCache(2, 64, 2, 32)
    z = lambda *s: Tensor.full(s, 0.0, device="hip")                       # noqa: E731
    for call in (lambda: cache.write(z(2, 1, 64), z(2, 1, 32)), lambda: cache.write(z(1, 1, 64), z(1, 1, 64)), lambda: cache.write(z(2, 64), z(2, 64)),
                 lambda: cache.write(z(2, 65, 64), z(2, 65, 64)), lambda: cache.attend(z(2, 1, 96)), lambda: cache.attend(z(3, 1, 64)),
                 lambda: cache.attend(z(2, 65, 64)), lambda: cache.attend(z(2, 1, 64), counts=z(3, 1)), lambda: cache.read(65), lambda: cache.read(-1),
                 lambda: cache.advance(-1), lambda: cache.advance(0.5), lambda: cache.advance(z(3, 1)), lambda: cache.write(Tensor(np.zeros((2, 1, 64), f32)), z(2, 1, 64)),
                 lambda: cache.attend(Tensor(np.zeros((2, 1, 64), f32))), lambda: cache.attend(Tensor.full((2, 1, 64), 0.0, device="hip", requires_grad=True)),
                 lambda: cache.attend(z(2, 1, 0))):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        cache.write(z(2, 1, 64), z(2, 1, 64), counts=3)
    with pytest.raises(IndexError):
        cache.write(z(2, 1, 64), z(2, 1, 64), layer=1)
    for bad in (dict(batch=0), dict(capacity=0), dict(n_kv_head=0), dict(head_dim=257), dict(layers=0), dict(capacity=2 ** 24 + 1), dict(lengths=z(3, 1))):
        with pytest.raises(ValueError):
            nn.QuantizedKVCache(**{**dict(batch=2, capacity=64, n_kv_head=2, head_dim=32), **bad})


def test_cache_runtime_refuses_what_does_not_fit():
    """Host checks of the launches, before any device is touched."""
    from dlgrad_amd.runtime.hip_lm import Cache8

    class Ptr:
        addr, nbytes = 256, 1 << 40
    b = lambda *s: Buffer(Ptr(), s, Device.HIP)                  # noqa: E731
    c = Cache8.__new__(Cache8)
    c.batch, c.heads, c.d, c.width, c.blocks, c.layers, c.kc, c.vc = 2, 3, 40, 64, 2, 1, Ptr(), Ptr()
    c.scales = c.tail_k = c.tail_v = b(1)
    c.writers, c.attenders = {}, {}
    for shape in ((2, 1, 121), (1, 1, 120), (2, 120), (2, 129, 120), (2, 1, 1, 120)):
        with pytest.raises(ValueError):
            HIPLM.cache8_write(c, b(*shape), b(*shape), b(2))
    for shape in ((2, 1, 121), (2, 1, 0), (3, 1, 120), (2, 129, 120), (2, 240)):
        with pytest.raises(ValueError):
            HIPLM.cache8_attend(c, b(*shape), 1.0, b(2))
    good = b(2, 1, 120)
    for call in (lambda: HIPLM.cache8_write(c, good, b(2, 2, 120), b(2)), lambda: HIPLM.cache8_write(c, good, good, b(3)), lambda: HIPLM.cache8_write(c, good, good, b(2), b(1)),
                 lambda: HIPLM.cache8_write(c, good, Buffer.from_scalar(1.0), b(2)), lambda: HIPLM.cache8_attend(c, good, 1.0, Buffer.from_scalar(1.0)),
                 lambda: HIPLM.cache8_attend(c, good, 1.0, b(2), b(5)), lambda: HIPLM.cache8_read(c, 129, b(2)), lambda: HIPLM.cache8_read(c, 1, b(2), None, 129),
                 lambda: HIPLM.cache8_read(c, 1, b(1))):
        with pytest.raises(ValueError):
            call()
    assert HIPLM.cache8_writer(c, (2, 0, 120))(0, 0, 0, 0) is None                # nothing to write: nothing launched
    assert not c.writers and not c.attenders


def test_adjust_logits_runtime_refuses_what_does_not_fit():
    class Ptr:
        addr, nbytes = 256, 1 << 40
    b = lambda *s: Buffer(Ptr(), s, Device.HIP)                  # noqa: E731
    good = dict(logits=b(4, 10), history=b(4, 3), lengths=b(4), penalties=(1.0, 0.0, 0.0), bias=b(10), hidden=b(4, 10))
    for bad in (dict(logits=b(40)), dict(logits=b(4, (1 << 24) + 1)), dict(history=b(3, 3)), dict(history=b(12)), dict(history=None), dict(lengths=b(3)),
                dict(bias=b(4)), dict(hidden=b(2, 10)), dict(hidden=b(4, 10, 1)), dict(penalties=(b(3), 0.0, 0.0)), dict(penalties=(1.0, 0.0, Buffer.from_scalar(2.0))),
                dict(logits=b(70000, 10), history=b(70000, 3), lengths=None, hidden=None)):
        with pytest.raises(ValueError):
            HIPLM.logits_plan(**{**good, **bad})


def test_cache_layout_puts_every_byte_in_one_place():
    """The places of a block's 64 x DP keys and values, restated: a permutation, and what each lane's load is meant to find there."""
    for DP in (32, 64, 96, 128, 160, 192, 224, 256):
        Q4 = DP // 4
        w = 16 if Q4 % 16 == 0 else 8
        row, c = (a.reshape(-1) for a in np.meshgrid(np.arange(64), np.arange(DP), indexing="ij"))
        g, i = c // Q4, c % Q4
        key = ((row >> 2) & 3) * 64 * Q4 + i // w * 64 * w + (g * 16 + ((row >> 4) << 2) + (row & 3)) * w + i % w
        value = (c >> 4) * 1024 + ((row >> 4) * 16 + (c & 15)) * 16 + (row & 15)
        for at in (key, value):
            assert np.array_equal(np.sort(at), np.arange(64 * DP))
        owner, column = np.empty(64 * DP, int), np.empty(64 * DP, int)
        owner[key], column[key] = row, c
        for u in range(4):                                          # lane r + 16 g of token tile u: the g-th quarter of token 16 (r / 4) + 4 u + r % 4
            for lane in range(64):
                r, q = lane % 16, lane // 16
                at = np.concatenate([u * 64 * Q4 + x * 64 * w + lane * w + np.arange(w) for x in range(Q4 // w)])
                assert (owner[at] == 16 * (r // 4) + 4 * u + r % 4).all() and np.array_equal(column[at], q * Q4 + np.arange(Q4))
        owner[value], column[value] = row, c
        for dt in range(DP // 16):                                  # ... and of column tile dt: tokens 16 g .. of column 16 dt + r
            for lane in range(64):
                at = dt * 1024 + lane * 16 + np.arange(16)
                assert np.array_equal(owner[at], 16 * (lane // 16) + np.arange(16)) and (column[at] == 16 * dt + lane % 16).all()


def test_cache_is_refused_off_the_device():
    with pytest.raises(ValueError, match="hip device"):
        nn.QuantizedKVCache(1, 64, 1, 32, device="cpu")


def test_splits_and_slices():
    """Parts are made from 8 blocks a wavefront on, their number grows with the root of the blocks, and they fill the device, not more."""
    assert HIPLM.attend_splits(4, 2, 4, 256) == 1 and HIPLM.attend_splits(4, 31, 4, 256) == 1 and HIPLM.attend_splits(4, 63, 8, 256) == 1
    assert HIPLM.attend_splits(1, 2048, 4, 256) == 32 and HIPLM.attend_splits(1, 1 << 18, 4, 256) == 64
    assert HIPLM.attend_splits(128, 512, 4, 256) == 4 and HIPLM.attend_splits(192, 64, 8, 256) == 1
    assert HIPLM.attend_splits(5000, 512, 4, 256) == 1
    assert HIPLM.adjust_items(1, 65, 256) == 4 and HIPLM.adjust_items(256, 128256, 256) == 16
    for B, V in ((1, 50304), (8, 50304), (64, 32000)):
        items = HIPLM.adjust_items(B, V, 256)
        assert items == 4 or B * -(-V // (256 * items)) >= 512


def test_adjust_items_by_blocks():
    """Sixteen logits a thread from four blocks a compute unit on, eight from two."""
    for B, V in ((1, 65), (8, 50304), (16, 128256), (32, 50304), (32, 128256), (64, 50257), (64, 32000), (100, 50257), (65535, 1)):
        items = HIPLM.adjust_items(B, V, 256)
        blocks = lambda n: B * -(-V // (256 * n))                          # noqa: E731
        assert items == (16 if blocks(16) >= 1024 else 8 if blocks(8) >= 512 else 4), (B, V)
    assert [HIPLM.adjust_items(B, V, 256) for B, V in ((8, 50304), (16, 128256), (64, 50257), (32, 128256))] == [4, 8, 8, 16]


def test_attention_forms_by_rows():
    """No tile of query rows is all padding, and eight wavefronts come with one tile, as the kernels are made for."""
    for pairs in (1, 96, 768, 5000):
        for rows in (1, 2, 15, 16, 17, 31, 32, 33, 500):
            for width in (32, 64, 128):
                nq, waves = HIPLM.attend_tiles(rows, pairs, width, 256), HIPLM.attend_waves(rows, 40, width)
                assert nq == 1 or rows > 16
                assert waves == 4 or (nq == 1 and rows <= 16 and width <= 64)
    assert HIPLM.attend_tiles(1, 768, 64, 256) == 1 and HIPLM.attend_waves(1, 40, 64) == 8 and HIPLM.attend_tiles(17, 768, 64, 256) == 2


# ================================================================ in the GPT of the examples
TINY = dict(vocab_size=33, block_size=96, n_layer=2, n_head=2, n_embd=64, batch_size=3)


def gpt(device, seed=3, std=0.2, **kw):
    from examples import gpt as G
    model = G.GPT(G.GPTConfig(device=device, **{**TINY, **kw}))
    G.init_weights_(model, seed, std)
    return model


def test_gpt_options_and_parameters():
    from examples import gpt as G
    for bad in (dict(positions="other"), dict(cache="int4")):
        with pytest.raises(ValueError):
            G.GPTConfig(**bad)
    learned, rotary = gpt("cpu"), gpt("cpu", positions="rotary")
    names = set(nn.utils.get_state_dict(learned))
    assert names - set(nn.utils.get_state_dict(rotary)) == {"wpe.weight"}
    assert len(nn.utils.get_parameters(rotary)) == len(names) - 1


def test_rotary_gpt_decodes_as_it_recomputes_on_the_cpu():
    """The cached, the fixed-shape and the recomputing decoders agree, with penalties too, inside the window and beyond it."""
    from examples import gpt as G
    model = gpt("cpu", positions="rotary", block_size=16)
    want = model.generate_greedy(3, 12)
    assert model.generate_greedy_cached(3, 12) == want
    assert G.StaticDecoder(model).generate(3, 22)[:13] == want
    kw = dict(repetition=1.7, presence=0.3, frequency=0.2)
    got = G.StaticDecoder(model, penalties=kw).generate(3, 22)
    assert got[:13] == model.generate_greedy_cached(3, 12, penalties=kw) != want
    hidden = np.ones(33, f32)
    hidden[[5, 6]] = 0
    assert set(model.generate(3, 12, u=np.linspace(0, 0.99, 12), penalties=dict(hidden=Tensor(hidden)))[1:]) <= {5, 6}


@pytest.mark.gpu
@pytest.mark.parametrize("T", [64, 96])
def test_rotary_gpt_trains_as_on_the_cpu(T):
    """Loss and every gradient of a step against the CPU composition: 1e-4, what this package asks of a whole step in fp32."""
    require_gpu()
    rng = np.random.default_rng(T)
    ids, targets = (rng.integers(0, 33, (3, T)).astype(f32) for _ in range(2))
    got = {}
    for device in ("cpu", "hip"):
        model = gpt(device, positions="rotary", std=0.05)
        _, loss = model(Tensor(ids, device=device), Tensor(targets, device=device))
        loss.backward()
        got[device] = (float(loss.numpy()), {k: p.grad.numpy() for k, p in nn.utils.get_state_dict(model).items()})
    if hip.COMPILE_ONLY:
        return
    assert abs(got["hip"][0] - got["cpu"][0]) <= 1e-4 * abs(got["cpu"][0])
    for name, want in got["cpu"][1].items():
        assert np.abs(got["hip"][1][name] - want).max() <= 1e-4 * np.abs(want).max(), name


@pytest.mark.gpu
def test_rotary_gpt_steps_in_a_captured_graph():
    """Forward, backward and the optimizer's step recorded once: every replay leaves the weights of an eager step, bit for bit."""
    require_gpu()
    if hip.COMPILE_ONLY:
        return
    rng = np.random.default_rng(8)
    ids, targets = (rng.integers(0, 33, (3, 96)).astype(f32) for _ in range(2))
    weights = []
    for captured in (False, True):
        model = gpt("hip", positions="rotary", std=0.05)
        opt = nn.optim.Adam(nn.utils.get_parameters(model), lr=1e-3)
        it, tt = hip_tensor(ids), hip_tensor(targets)

        def step():
            for p in nn.utils.get_parameters(model):
                p.grad = None
            _, loss = model(it, tt)
            loss.backward()
            opt.step()
            return loss
        run = hip.CapturedStep(step, before_replay=opt.advance) if captured else step
        losses = []
        for i in range(6):
            losses.append(float(run().numpy()))
            if i == 3:
                nn.adjust_logits(hip_tensor(rng.standard_normal((2, 9)))).numpy()         # work of its own between the replays
        weights.append((losses, [p.numpy() for p in nn.utils.get_parameters(model)]))
        if captured:
            run.close()
    assert weights[0][0] == weights[1][0]
    for a, b in zip(weights[0][1], weights[1][1]):
        same(a, b)


@pytest.mark.gpu
def test_rotary_inside_the_projection_is_rotary_after_it(monkeypatch):
    """Turned in place in the stacked projection: the context has the bits of three projections turned as tensors; and the
    gradient of x is that of the same composition to the rounding of one accumulator against three."""
    require_gpu()
    rng = np.random.default_rng(2)
    B, T, h, d = 2, 40, 4, 16
    C = h * d
    rope = nn.Rotary(d, layout="interleaved")
    x = rng.standard_normal((B, T, C)).astype(f32)
    w = [(rng.standard_normal((C, C)) * C ** -0.5).astype(f32) for _ in range(3)]
    g = rng.standard_normal((B, T, C)).astype(f32)
    out = []
    for stacked in (True, False):
        xt, ws = hip_tensor(x, True), [hip_tensor(a, True) for a in w]
        if stacked:
            nn.stack_parameters(ws)
            assert ops.use_fused_qkv_attention(xt, *ws, h)
        else:
            monkeypatch.setattr(ops, "use_fused_qkv_attention", lambda *a: False)
        y = nn.self_attention_qkv(xt, *ws, h, d ** -0.5, rotary=rope)
        (y * hip_tensor(g)).sum().backward()
        out.append([y.numpy(), xt.grad.numpy(), *[a.grad.numpy() for a in ws]])
    if hip.COMPILE_ONLY:
        return
    same(out[0][0], out[1][0], "context")
    for a, b in zip(out[0][1:], out[1][1:]):
        assert np.abs(a - b).max() <= 3 * C * EPS * np.abs(b).max()


@pytest.mark.gpu
@pytest.mark.parametrize("positions", ["learned", "rotary"])
@pytest.mark.parametrize("cache", ["float32", "int8"])
def test_gpt_decodes_with_every_combination(positions, cache):
    """Rotary positions, the 8-bit cache and penalties together, as a decoder uses them: eager steps, a captured graph and -- while no block of
    the cache is full, so that it holds what the fp32 cache holds -- the CPU's decoder give the same tokens."""
    require_gpu()
    from examples import gpt as G
    penalties = dict(repetition=1.3, presence=0.2, frequency=0.1)
    model = gpt("hip", positions=positions, cache=cache)
    eager = model.generate_greedy_cached(7, 90, False, penalties=penalties)
    for temperature in (None, 0.8):
        u = np.random.default_rng(1).random(120).astype(f32)
        dec = G.StaticDecoder(model, reference_positions=False, capacity=121, temperature=temperature, penalties=penalties)
        plain = dec.generate(7, 110, u) if temperature else dec.generate(7, 110)
        dec.capture()
        for _ in range(2):
            tokens = dec.generate(7, 110, u) if temperature else dec.generate(7, 110)
            if not hip.COMPILE_ONLY:
                assert tokens == plain
        dec.close()
        if not temperature and not hip.COMPILE_ONLY:
            assert tokens[:91] == eager
    if not hip.COMPILE_ONLY:
        cpu = gpt("cpu", positions=positions).generate_greedy_cached(7, 60, False, penalties=penalties)
        assert tokens is not None and eager[:61] == cpu


@pytest.mark.gpu
@pytest.mark.parametrize("first", [20, 64, 70])
def test_gpt_prompt_into_the_quantized_cache(first):
    """A batch of prompts, then single tokens, against an fp32 cache that holds the values the 8-bit one stands for: 1e-4, what this
    package asks of a whole pass in fp32."""
    require_gpu()
    from examples import gpt as G
    rng = np.random.default_rng(4)
    ids = rng.integers(0, 33, (3, 90)).astype(f32)
    model, plain = gpt("hip", cache="int8", positions="rotary"), gpt("hip", positions="rotary")
    got, cache = model.prefill(hip_tensor(ids[:, :first]))
    want, _ = plain.prefill(hip_tensor(ids[:, :first]))
    same(got.numpy(), want.numpy(), "the prompt itself attends in fp32")
    wide = G.KVCache(plain.config, 3)
    for layer in range(2):
        wide.write(layer, *cache.store.read(first, layer), 0)
    wide.advance(first)
    for t in range(first, first + 20 if first < 64 else 90):
        got, want = (m.forward_incremental(hip_tensor(ids[:, t:t + 1]), hip_tensor([[t]]), c).numpy() for m, c in ((model, cache), (plain, wide)))
        if not hip.COMPILE_ONLY:
            assert np.abs(got - want).max() <= 1e-4 * np.abs(want).max(), t
