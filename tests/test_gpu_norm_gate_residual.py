"""GPU: the join of two blocks (norm, gate, residual scale, residual, norm) against the formulas in 64
bits: every norm, gate and storage type, group counts, channel counts from one to the largest, strides,
in place, infinities, the calls that are refused, and a run of the causal-context operators as a block."""

import ctypes
import time

import numpy as np
import pytest

from devbuf import HALF_STEP, DevBuf, from_raw, to_raw
from linear_attention_oracle import oracle
from zenjpegai_amd import _lib, nn

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
POST_EPS, PRE_EPS = 1e-5, 1e-3


@pytest.fixture(scope="module")
def eng():
    e = nn.Engine(0)
    yield e
    e.close()


def norm(x, kind, groups, eps, w, b, err):
    """The norm of x [n][c] whose elements are off by at most err, and what the result is off by: the
    statistics' f32 sums of m = c / groups values take at most m / 64 + 16 roundings one after another."""
    n, c = x.shape
    k = (c // groups / 64 + 16) * U
    x, err = x.reshape(n, groups, c // groups), err.reshape(n, groups, c // groups)
    if kind != "none":
        mean = x.mean(-1, keepdims=True) if kind == "layer" else 0.0
        if kind == "layer":
            err = err + err.mean(-1, keepdims=True) + k * np.abs(x).mean(-1, keepdims=True) + U * np.abs(x - mean)
        d = x - mean
        inv = 1.0 / np.sqrt((d * d).mean(-1, keepdims=True) + eps)
        rel = inv ** 2 * (np.abs(d) * err + err ** 2).mean(-1, keepdims=True) + k
        x, err = d * inv, err * inv * (1 + rel) + np.abs(d) * inv * rel
    x, err = x.reshape(n, c), err.reshape(n, c)
    if w is not None:
        x, err = x * w, err * np.abs(w) + U * np.abs(x * w)
    if b is not None:
        x, err = x + b, err + U * (np.abs(x) + np.abs(b))
    return x, err


def oracle_join(x, y, gate, act, post, groups, pre, w1, b1, s, w2, b2):
    u, err = norm(y, post, groups, POST_EPS, w1, b1, np.zeros_like(y))
    if gate is not None:
        sig = 1.0 / (1.0 + np.exp(-gate))
        a = {"linear": gate, "sigmoid": sig, "silu": gate * sig}[act]
        # exp(-g) is off by the rounding of its argument (|g| log2 e) and two steps, the quotient by two more.
        u, err = u * a, err * np.abs(a) + np.abs(u * a) * U * (1 if act == "linear" else 8 + 3 * np.abs(gate))
    if s is not None:
        u, err = u * s, err * np.abs(s) + U * np.abs(u * s)
    xo, err = x + u, err + U * (np.abs(x) + np.abs(u))
    h, eh = norm(xo, pre, 1, PRE_EPS, w2, b2, err) if pre != "none" else (None, None)
    return (xo, err), (h, eh)


def near(raw, prec, want, err):
    got = from_raw(raw, prec).reshape(want.shape)
    tol = err + HALF_STEP[prec] * (np.abs(want) + err) + 2.0 ** -25 * (prec == "f16") + 1e-38
    off = np.abs(got - want)
    assert (off <= tol).all(), (float((off / tol).max()), np.unravel_index(np.argmax(off / tol), off.shape))


def run(eng, prec, n, c, groups=1, post="layer", act="linear", gate=True, pre="rms", weights=True, place=None, gap=0,
        offset=0, seed=0):
    rng = np.random.default_rng(seed + c)
    st = c + gap

    def rows(dev, mean=0.0):
        return to_raw(mean + dev * rng.standard_normal((n, st)), prec)

    x, y = rows(2.0), rows(1.0, 0.4)
    g = rows(2.0) if gate else None
    vec = [(m + d * rng.standard_normal(c)).astype(np.float32) if weights else None
           for m, d in ((1.0, 0.2), (0.0, 0.3), (0.5, 0.2), (1.0, 0.2), (0.0, 0.3))]
    if post == "none":
        vec[0] = vec[1] = None
    if pre == "none":
        vec[3] = vec[4] = None
    fill = to_raw(np.full((n, st), 9.0), prec)
    dx, dy, dg, dxo, dh = (None if a is None else DevBuf(a, offset) for a in (x, y, g, fill, fill if pre != "none" else None))
    before_x, before_h = fill, fill
    if place:
        dxo, before_x = dx, x
        if pre != "none":
            dh, before_h = (dy, y) if place == "y" else (dg, g)
    d = [None if a is None else DevBuf(a) for a in vec]
    nn.norm_gate_residual_noalloc(eng, nn.norm_gate_residual_desc(
        prec, dx, dy, dg, dxo, dh, positions=n, channels=c, gate_act=act if gate else "linear", post_norm=post,
        post_groups=groups, post_eps=POST_EPS, post_weight=d[0], post_bias=d[1], residual_scale=d[2], pre_norm=pre,
        pre_eps=PRE_EPS, pre_weight=d[3], pre_bias=d[4], **{k + "_stride": st for k in ("x", "y", "gate", "x_out", "h")}))
    eng.sync()
    f = [None if a is None else from_raw(a, prec)[:, :c] for a in (x, y, g)]
    v = [None if a is None else a.astype(np.float64) for a in vec]
    (xo, ex), (h, eh) = oracle_join(*f, act, post, groups, pre, *v)
    got = dxo.get()
    near(got[:, :c], prec, xo, ex)
    assert np.array_equal(got[:, c:], before_x[:, c:])
    if pre != "none":
        got = dh.get()
        near(got[:, :c], prec, h, eh)
        assert np.array_equal(got[:, c:], before_h[:, c:])


@pytest.mark.parametrize("prec", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("post", ["none", "layer", "rms"])
@pytest.mark.parametrize("act", [None, "linear", "sigmoid", "silu"])
@pytest.mark.parametrize("pre", ["none", "layer", "rms"])
def test_every_norm_and_gate(eng, prec, post, act, pre):
    run(eng, prec, 5, 96, groups=4, post=post, act=act or "linear", gate=act is not None, pre=pre)


@pytest.mark.parametrize("prec", ["f32", "bf16"])
@pytest.mark.parametrize("c,groups", [(1, 1), (3, 1), (7, 7), (8, 2), (20, 5), (64, 1), (96, 8), (100, 4), (128, 4), (129, 3),
                                      (192, 12), (250, 5), (512, 16), (1000, 8), (1024, 1), (1536, 4), (2048, 128), (4096, 1),
                                      (5000, 5), (8192, 64), (16384, 2), (16380, 1), (16383, 3), (9000, 45)])
def test_channel_and_group_counts(eng, prec, c, groups):
    run(eng, prec, 3, c, groups=groups, act="sigmoid", pre="layer")
    run(eng, prec, 1, c, groups=groups, post="rms", act="silu", weights=False)


@pytest.mark.parametrize("prec", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("c,gap,offset", [(96, 1, 0), (128, 8, 0), (100, 3, 4), (512, 0, 4), (160, 5, 8)])
def test_strides_and_buffers_off_16_bytes(eng, prec, c, gap, offset):
    run(eng, prec, 6, c, groups=2, act="silu", gap=gap, offset=offset)


@pytest.mark.parametrize("prec", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("c", [128, 100, 4096])
@pytest.mark.parametrize("place", ["y", "gate"])
def test_in_place(eng, prec, c, place):
    run(eng, prec, 9, c, groups=4, act="sigmoid", place=place)


@pytest.mark.parametrize("n,c", [(0, 64), (1, 128), (4097, 24), (70001, 8), (3001, 512)])
def test_position_counts(eng, n, c):
    run(eng, "bf16", n, c, act="silu")


@pytest.mark.parametrize("prec", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,c", [(700, 64), (33, 1000), (1, 24)])
def test_one_gate_for_all_positions_and_interleaved_outputs(eng, prec, n, c):
    """x and the gate are one row each (stride 0); x_out and h alternate in one buffer."""
    rng = np.random.default_rng(c)
    x, g = (to_raw(rng.standard_normal((1, c)), prec) for _ in range(2))
    y = to_raw(rng.standard_normal((n, c)), prec)
    dx, dg, dy = DevBuf(x), DevBuf(g), DevBuf(y)
    both = DevBuf(to_raw(np.zeros((n, 2, c)), prec))
    es = 4 if prec == "f32" else 2
    nn.norm_gate_residual_noalloc(eng, nn.norm_gate_residual_desc(
        prec, dx, dy, dg, both, both.address + c * es, positions=n, channels=c, gate_act="sigmoid", post_norm="rms",
        post_eps=POST_EPS, pre_norm="layer", pre_eps=PRE_EPS, x_stride=0, gate_stride=0, x_out_stride=2 * c, h_stride=2 * c))
    eng.sync()
    f = [np.broadcast_to(from_raw(a, prec), (n, c)) for a in (x, y, g)]
    (xo, ex), (h, eh) = oracle_join(*f, "sigmoid", "rms", 1, "layer", None, None, None, None, None)
    got = both.get()
    near(got[:, 0], prec, xo, ex)
    near(got[:, 1], prec, h, eh)


@pytest.mark.parametrize("prec", ["f32", "bf16"])
@pytest.mark.parametrize("n,c", [(700, 64), (40, 2000)])
def test_h_in_the_place_of_x(eng, prec, n, c):
    rng = np.random.default_rng(c + 1)
    x, y = (to_raw(rng.standard_normal((n, c)), prec) for _ in range(2))
    dx, dy, dxo = DevBuf(x), DevBuf(y), DevBuf(y)
    nn.norm_gate_residual_noalloc(eng, nn.norm_gate_residual_desc(prec, dx, dy, None, dxo, dx, positions=n, channels=c,
                                                                  post_norm="layer", post_eps=POST_EPS, pre_norm="rms", pre_eps=PRE_EPS))
    eng.sync()
    (xo, ex), (h, eh) = oracle_join(from_raw(x, prec), from_raw(y, prec), None, "linear", "layer", 1, "rms", None, None, None, None, None)
    near(dxo.get(), prec, xo, ex)
    near(dx.get(), prec, h, eh)


def test_a_position_with_an_infinity_leaves_the_others_alone(eng):
    n, c, prec = 40, 96, "f32"
    rng = np.random.default_rng(3)
    x, y = (rng.standard_normal((n, c)).astype(np.float32) for _ in range(2))
    y[17, 5], x[21, 0] = np.inf, np.nan
    b = [DevBuf(a) for a in (x, y, x, x)]
    nn.norm_gate_residual_noalloc(eng, nn.norm_gate_residual_desc(prec, b[0], b[1], None, b[2], b[3], positions=n, channels=c,
                                                                  post_norm="layer", post_eps=POST_EPS, pre_norm="layer",
                                                                  pre_eps=PRE_EPS))
    eng.sync()
    xo, h = b[2].get(), b[3].get()
    assert not np.isfinite(h[17]).any() and not np.isfinite(h[21]).any() and np.isnan(xo[21, 0])
    ok = np.ones(n, bool)
    ok[[17, 21]] = False
    (wx, ex), (wh, eh) = oracle_join(*(a[ok].astype(np.float64) for a in (x, y)), None, "linear", "layer", 1, "layer", *[None] * 5)
    near(xo[ok], prec, wx, ex)
    near(h[ok], prec, wh, eh)


def test_a_constant_position_and_large_gates(eng):
    """A position without variance is normed to its bias; gates at the ends of the range stay finite."""
    c = 64
    x, y = np.zeros((2, c), np.float32), np.full((2, c), 3.0, np.float32)
    gate = np.full((2, c), -3e38, np.float32)
    gate[1] = 3e38
    b = [DevBuf(a) for a in (x, y, gate, x, x)]
    for act, want in (("sigmoid", [0.0, 3.0]), ("silu", [0.0, None])):
        nn.norm_gate_residual_noalloc(eng, nn.norm_gate_residual_desc(
            "f32", b[0], b[1], b[2], b[3], b[4], positions=2, channels=c, gate_act=act, pre_norm="layer", pre_eps=PRE_EPS))
        eng.sync()
        xo, h = b[3].get(), b[4].get()
        assert (xo[0] == want[0]).all() and (h[0] == 0.0).all()
        if want[1] is not None:
            assert (xo[1] == want[1]).all() and (h[1] == 0.0).all()


@pytest.mark.parametrize("prec", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("crop", [False, True])
def test_tensor_form(prec, crop):
    e = nn.Engine(0, prec)
    c, h, w = 36, 7, 9
    rng = np.random.default_rng(1)
    raw = [to_raw(rng.standard_normal((c, h + crop, w + 2 * crop)), prec) for _ in range(3)]
    vec = [rng.standard_normal(c).astype(np.float32) for _ in range(5)]
    t = [nn.BTensor.from_planar(e, from_raw(a, prec).astype(np.float32)) for a in raw]
    if crop:
        t, raw = [a.crop(h, w) for a in t], [a[:, :h, :w] for a in raw]
    xo, hh = nn.norm_gate_residual(e, *t, gate_act="sigmoid", post_norm="layer", post_groups=3, post_eps=POST_EPS,
                                   post_weight=vec[0], post_bias=vec[1], residual_scale=vec[2], pre_norm="rms",
                                   pre_eps=PRE_EPS, pre_weight=vec[3], pre_bias=vec[4])
    flat = [from_raw(a, prec).reshape(c, h * w).T for a in raw]
    (wx, ex), (wh, eh) = oracle_join(*flat, "sigmoid", "layer", 3, "rms", *[a.astype(np.float64) for a in vec])
    near(to_raw(xo.to_planar().reshape(c, -1).T, prec), prec, wx, ex)
    near(to_raw(hh.to_planar().reshape(c, -1).T, prec), prec, wh, eh)
    xo, none = nn.norm_gate_residual(e, t[0], t[1])
    assert none is None
    near(to_raw(xo.to_planar().reshape(c, -1).T, prec), prec, flat[0] + flat[1], U * (np.abs(flat[0]) + np.abs(flat[1])))
    del t, xo, hh
    e.close()


def test_refused_calls(eng):
    b = {n: DevBuf(np.zeros(4096, np.float32)) for n in ("x", "y", "g", "xo", "h", "w")}
    good = dict(positions=4, channels=16, post_norm="layer", pre_norm="rms")

    def code(prec="f32", edit=None, **kw):
        d = nn.norm_gate_residual_desc(prec, b["x"], b["y"], b["g"], b["xo"], b["h"], **{**good, **kw})
        for n, v in (edit or {}).items():
            setattr(d, n, v)
        return _lib.lib().zjai_norm_gate_residual_noalloc(eng.handle, ctypes.byref(d))

    bad = _lib.E_INVALID_ARGUMENT
    assert code() == _lib.OK and code(positions=0) == _lib.OK
    assert code(channels=16385) == _lib.E_UNSUPPORTED
    for e in ({"precision": -1}, {"gate_act": 3}, {"gate_act": -1}, {"post_norm": 3}, {"pre_norm": -1}, {"post_groups": 0},
              {"post_groups": 3}, {"channels": 0}, {"positions": -1}, {"x": None}, {"y": None}, {"x_out": None}, {"h": None},
              {"pre_norm": 0}, {"post_eps": 0.0}, {"pre_eps": -1.0}, {"pre_eps": float("nan")}, {"post_eps": float("inf")},
              {"gate": None, "gate_act": 1}, {"x": b["x"].address + 2}, {"post_weight": b["w"].address + 1},
              {"x_stride": -16}, {"x_out_stride": 15}, {"h_stride": 15}, {"h": b["xo"].address}, {"x_out": b["y"].address},
              {"x_out": b["g"].address}, {"x_out": b["x"].address, "x_out_stride": 20}, {"h": b["y"].address, "y_stride": 32},
              {"h": b["g"].address, "h_stride": 24}, {"post_norm": 0, "post_weight": b["w"].address},
              {"pre_norm": 0, "h": None, "pre_bias": b["w"].address}):
        assert code(edit=e) == bad, e
    assert _lib.lib().zjai_norm_gate_residual_noalloc(None, None) == bad
    t = [nn.BTensor.from_planar(eng, np.zeros((8, 2, k), np.float32)) for k in (2, 2, 3)]
    for kw in (dict(x=t[0], y=t[2]), dict(x=t[0], y=t[1], gate=t[2]), dict(x=t[0], y=t[1], post_norm="rms", post_groups=3),
               dict(x=t[0], y=t[1], gate_act="silu"), dict(x=t[0], y=t[1], post_weight=np.ones(8))):
        with pytest.raises(_lib.HipError) as err:
            nn.norm_gate_residual(eng, **kw)
        assert err.value.kind == "InvalidArgument"
    eng.sync()


@pytest.mark.parametrize("prec", ["f32", "f16", "bf16"])
def test_a_causal_context_block(prec):
    """norm -> 1x1 to q, k, v -> linear attention -> 1x1 -> post norm, residual scale, residual and the next
    block's norm, as a context model chains them, against the same chain in 64 bits on rounded weights.
    The bound: each of the five stored maps is rounded to the storage type once, which the two 1x1
    products and the norms of a random block carry on at about their own size (factor 4 in all)."""
    c, heads, h, w = 64, 2, 12, 10
    d = c // heads
    rng = np.random.default_rng(7)
    e = nn.Engine(0, prec)

    def rounded(a):
        return from_raw(to_raw(a, prec), prec)

    x = rounded(rng.standard_normal((c, h, w)))
    w_in = rounded(rng.standard_normal((3 * c, c)) / np.sqrt(c))
    w_out = rounded(rng.standard_normal((c, c)) / np.sqrt(c))
    ln = [(1 + 0.1 * rng.standard_normal(c)).astype(np.float32), (0.1 * rng.standard_normal(c)).astype(np.float32)]
    post_w, scale = (1 + 0.1 * rng.standard_normal((2, c))).astype(np.float32)
    decay = np.array([0.9, 0.99], np.float32)

    t = nn.BTensor.from_planar(e, x.astype(np.float32))
    conv = [nn.ConvLayer(nn.Conv2d(m.shape[1], m.shape[0], (1, 1), 1, (0, 0), 1, m.astype(np.float32)), e) for m in (w_in, w_out)]
    qkv = conv[0].forward(e, nn.layer_norm_channels(e, t, *ln))
    y = conv[1].forward(e, nn.linear_attention(e, qkv, heads, d, decay, d ** -0.5))
    xo, hh = nn.norm_gate_residual(e, t, y, post_norm="rms", post_groups=heads, post_weight=post_w, residual_scale=scale,
                                   pre_norm="layer", pre_weight=ln[0], pre_bias=ln[1])

    def layer(a):
        return (a - a.mean(1, keepdims=True)) / np.sqrt(a.var(1, keepdims=True) + 1e-5) * ln[0] + ln[1]

    f = x.reshape(c, -1).T
    p = layer(f) @ w_in.T
    q, k, v = (p[:, i * c:(i + 1) * c].reshape(-1, heads, d) for i in range(3))
    (o, _, _), _ = oracle(q, k, v, decay, d ** -0.5, h * w)
    u = (o.reshape(-1, c) @ w_out.T).reshape(-1, heads, d)
    u = (u / np.sqrt((u * u).mean(-1, keepdims=True) + 1e-5)).reshape(-1, c) * post_w
    wx = f + scale * u
    for got, want in ((xo, wx), (hh, layer(wx))):
        got = got.to_planar().reshape(c, -1).T
        rel = np.linalg.norm(got - want) / np.linalg.norm(want)
        assert rel <= 5 * 4 * HALF_STEP[prec], rel
    del t, conv, qkv, y, xo, hh
    e.close()


@pytest.mark.parametrize("prec", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("c,groups", [(9, 3), (100, 4), (250, 5), (999, 333), (1001, 7), (1400, 7), (1536, 6), (2600, 200), (4096, 2),
                                      (8190, 10), (8190, 2730), (9002, 2), (12000, 3), (16383, 5461), (16380, 1365)])
@pytest.mark.parametrize("post", ["layer", "rms"])
def test_groups_that_are_no_power_of_two(eng, prec, c, groups, post):
    """Few long groups, many short ones, and several positions to a workgroup and one after another."""
    run(eng, prec, 37 if c < 2000 else 3, c, groups=groups, post=post, act="silu", pre="rms", seed=5)


def test_odd_groups_take_no_longer_than_the_size_accounts_for(eng):
    """Two groups of 4501 channels, 600 positions: some 60 us of work (with every lane adding its whole group up 60 ms)."""
    n, c = 600, 9002
    rng = np.random.default_rng(6)
    b = [DevBuf(to_raw(rng.standard_normal((n, c)), "bf16")) for _ in range(4)]
    d = nn.norm_gate_residual_desc("bf16", b[0], b[1], None, b[2], b[3], positions=n, channels=c, post_norm="layer", post_groups=2,
                                   pre_norm="rms")
    for _ in range(3):  # the first call loads the kernel
        eng.sync()
        t = time.perf_counter()
        for _ in range(5):
            nn.norm_gate_residual_noalloc(eng, d)
        eng.sync()
        t = time.perf_counter() - t
    assert t < 0.05, t
