"""GPU: the operators of a state-space context model as they are used together: a rotated linear attention and a
convolved scan, joined into a block; a prompt continued position by position; calls on another stream's buffers, captured into a
graph and replayed, on two contexts at once, and on buffers that share a context's scratch."""

import ctypes
from types import SimpleNamespace

import numpy as np
import pytest

from devbuf import DevBuf, from_raw, hip, to_raw
from linear_attention_oracle import oracle as attention
from state_space_oracle import conv, rotary, scan
from zenjpegai_amd import _lib, nn

pytestmark = pytest.mark.gpu
NON_BLOCKING, CAPTURE_GLOBAL = 1, 0
SEQS, HEADS, D = 2, 2, 32
C, N, TAPS = HEADS * D, 16, 4


@pytest.fixture(scope="module")
def eng():
    e = nn.Engine(0)
    yield e
    e.close()


@pytest.fixture()
def stream():
    s = ctypes.c_void_p()
    assert hip().hipStreamCreateWithFlags(ctypes.byref(s), NON_BLOCKING) == 0
    yield s
    assert hip().hipStreamDestroy(s) == 0


def weights(seed=0):
    rng = np.random.default_rng(seed)
    return SimpleNamespace(
        freq=nn.rotary_frequencies(D)[0], decay=np.array([0.9, 0.99], np.float32),
        cw=(0.5 * rng.standard_normal((C, TAPS))).astype(np.float32), cb=rng.standard_normal(C).astype(np.float32),
        a=(-np.arange(1, N + 1) * rng.uniform(0.8, 1.2, (C, N))).astype(np.float32), d=rng.standard_normal(C).astype(np.float32),
        bias=np.full(C, -3.0, np.float32))


def inputs(seed, prec, seqs, length):
    rng = np.random.default_rng(seed)
    return {n: to_raw(rng.standard_normal((seqs, length, w)), prec) for n, w in (("qkv", 3 * C), ("xz", 2 * C), ("delta", C), ("bc", 2 * N))}


class Block:
    """The buffers and calls of a block on `length` positions: rotary, attention; convolution, scan; their join."""

    def __init__(self, prec, length, w, states=None, starts=None, seqs=SEQS):
        es = 4 if prec == "f32" else 2
        self.prec, self.length, self.step = prec, length, states is not None
        z = lambda n: DevBuf(to_raw(np.zeros((seqs, length, n)), prec))  # noqa: E731
        self.buf = {n: z(k) for n, k in (("qkv", 3 * C), ("xz", 2 * C), ("delta", C), ("bc", 2 * N), ("att", C), ("conv", C), ("scan", C),
                                         ("x_out", C), ("h", C))}
        self.w = {n: DevBuf(v) for n, v in vars(w).items()}
        self.states = states or {"att": DevBuf(np.zeros((seqs, HEADS, D, D), np.float32)),
                                 "conv": DevBuf(to_raw(np.zeros((seqs, TAPS - 1, C)), prec)),
                                 "scan": DevBuf(np.zeros((seqs, C, N), np.float32))}
        self.starts = starts
        b, s, k = self.buf, self.states, self.w
        common = dict(sequences=seqs, length=length)
        self.rotary = nn.rotary_desc(prec, b["qkv"], b["qkv"], heads=2 * HEADS, head_dim=D, frequencies=k["freq"], starts=starts,
                                     x_position=3 * C, out_position=3 * C, x_sequence=3 * C * length, out_sequence=3 * C * length, **common)
        self.att = nn.linear_attention_desc(prec, b["qkv"], b["att"], heads=HEADS, key_dim=D, value_dim=D, decay=k["decay"], scale=0.2,
                                            state_in=s["att"], state_out=s["att"], **common)
        self.conv = nn.causal_conv_desc(prec, b["xz"], b["conv"], channels=C, taps=TAPS, weight=k["cw"], bias=k["cb"], act="silu",
                                        state_in=s["conv"], state_out=s["conv"], x_position=2 * C, x_sequence=2 * C * length, **common)
        self.scan = nn.selective_scan_desc(
            prec, b["conv"], b["delta"], b["bc"], b["bc"].address + N * es, b["scan"], channels=C, state_dim=N, a=k["a"], d=k["d"],
            delta_bias=k["bias"], z=b["xz"].address + C * es, state_in=s["scan"], state_out=s["scan"], z_position=2 * C,
            z_sequence=2 * C * length, b_position=2 * N, c_position=2 * N, b_sequence=2 * N * length, c_sequence=2 * N * length, **common)
        self.join = nn.norm_gate_residual_desc(prec, b["att"], b["scan"], None, b["x_out"], b["h"], positions=seqs * length, channels=C,
                                               post_norm="rms", post_groups=HEADS, pre_norm="layer")

    def put(self, values, at=slice(None)):
        for n, v in values.items():
            self.buf[n].put(np.ascontiguousarray(v[:, at]))

    def calls(self, eng):
        nn.rotary_noalloc(eng, self.rotary)
        (nn.linear_attention_step if self.step else nn.linear_attention_noalloc)(eng, self.att)
        (nn.causal_conv_step if self.step else nn.causal_conv_noalloc)(eng, self.conv)
        (nn.selective_scan_step if self.step else nn.selective_scan_noalloc)(eng, self.scan)
        nn.norm_gate_residual_noalloc(eng, self.join)

    def results(self):
        return {n: self.buf[n].get() for n in ("att", "conv", "scan", "x_out", "h")} | {"state_" + n: b.get() for n, b in self.states.items()}

    def clear(self):
        for b in self.states.values():
            b.put(np.zeros(b.shape, b.dtype))


@pytest.mark.parametrize("prec", ["f32", "f16", "bf16"])
def test_a_block_equals_its_parts_in_64_bits(eng, prec):
    """Every part against the formula on the inputs that the part before it wrote."""
    length, w = 77, weights()
    b, v = Block(prec, length, w), inputs(1, prec, SEQS, length)
    b.put(v)
    b.calls(eng)
    eng.sync()
    got, turned = b.results(), b.buf["qkv"].get()
    for s in range(SEQS):
        qk = from_raw(v["qkv"][s], prec)[:, :2 * C].reshape(length, 2 * HEADS, D)
        want, tol = rotary(prec, qk, np.arange(length), w.freq, "interleaved", 1.0)
        t = from_raw(turned[s], prec)
        assert (np.abs(t[:, :2 * C].reshape(want.shape) - want) <= tol).all()
        q, k, val = (t[:, i * C:(i + 1) * C].reshape(length, HEADS, D) for i in range(3))
        (o, _, _), (state, _, _) = attention(q, k, val, w.decay, 0.2, length)
        assert np.allclose(from_raw(got["att"][s], prec).reshape(o.shape), o, rtol=2e-2 if prec != "f32" else 1e-4, atol=2e-2 if prec != "f32" else 1e-4)
        xz = from_raw(v["xz"][s], prec)
        y, tol, last = conv(prec, xz[:, :C], w.cw, w.cb, "silu", length)
        assert (np.abs(from_raw(got["conv"][s], prec) - y) <= tol).all()
        assert np.array_equal(from_raw(got["state_conv"][s], prec), last)
        bc = from_raw(v["bc"][s], prec).reshape(length, 2, 1, N)
        y, tol, h, htol = scan(prec, from_raw(got["conv"][s], prec), from_raw(v["delta"][s], prec), bc[:, 0], bc[:, 1], xz[:, C:], w.a, w.d,
                               w.bias, True, length)
        assert (np.abs(from_raw(got["scan"][s], prec) - y) <= tol).all() and (np.abs(got["state_scan"][s] - h) <= htol).all()


@pytest.mark.parametrize("prec", ["f32", "f16", "bf16"])
def test_a_prompt_goes_on_position_by_position(eng, prec):
    """The first positions at once and the rest one by one, from the same states: what all of them at once give, to the types'
    rounding (the intermediate results are rounded alike, their f32 sums are formed in another order)."""
    first, rest, w = 50, 6, weights(2)
    v = inputs(3, prec, SEQS, first + rest)
    whole = Block(prec, first + rest, w)
    whole.put(v)
    whole.calls(eng)
    eng.sync()
    want = whole.results()
    b = Block(prec, first, w)
    b.put(v, slice(0, first))
    b.calls(eng)
    eng.sync()
    outs = [b.results()]
    one = Block(prec, 1, w, states=b.states, starts=DevBuf(np.full(SEQS, first, np.int32)))
    for t in range(first, first + rest):
        one.starts.put(np.full(SEQS, t, np.int32))
        one.put(v, slice(t, t + 1))
        one.calls(eng)
        eng.sync()
        outs.append(one.results())
    # A rounding may fall to the other side at each of the two stored results in front of the last ones.
    tol = {"f32": 1e-5, "f16": 4 * 2.0 ** -10, "bf16": 4 * 2.0 ** -7}[prec]
    for n in ("att", "conv", "scan"):
        got, ref = from_raw(np.concatenate([o[n] for o in outs], axis=1), prec), from_raw(want[n], prec)
        assert (np.abs(got - ref) <= tol * (np.abs(ref) + np.sqrt((ref ** 2).mean()))).all(), n
    for n in ("state_att", "state_scan"):
        assert (np.abs(outs[-1][n] - want[n]) <= tol * (np.abs(want[n]) + np.sqrt((want[n] ** 2).mean()))).all(), n
    assert np.array_equal(outs[-1]["state_conv"], want["state_conv"])


@pytest.mark.parametrize("length", [1, 40, 900])
def test_calls_captured_into_a_graph_and_replayed(eng, stream, length):
    """Each replay, on inputs of its own and with eager calls of the same context between, gives the eager call's bits."""
    w = weights(4)
    b, other = Block("bf16", length, w), Block("bf16", length, w)
    graph, runnable = ctypes.c_void_p(), ctypes.c_void_p()
    assert hip().hipStreamBeginCapture(stream, CAPTURE_GLOBAL) == 0
    eng.order_after(stream)
    b.calls(eng)
    eng.order_before(stream)
    assert hip().hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
    assert hip().hipGraphInstantiate(ctypes.byref(runnable), graph, None, None, ctypes.c_size_t(0)) == 0
    try:
        for i in range(4):
            v = inputs(10 + i, "bf16", SEQS, length)
            for t in (b, other):
                t.put(v)  # the states go on from replay to replay
            eng.order_before(stream)  # the context's scratch is the graph's too
            assert hip().hipGraphLaunch(runnable, stream) == 0
            eng.order_after(stream)
            other.calls(eng)
            eng.sync()
            assert hip().hipStreamSynchronize(stream) == 0
            got, want = b.results(), other.results()
            for n in got:
                assert np.array_equal(got[n], want[n]), (i, n)
            assert (want["scan"] != 0).any()
    finally:
        assert hip().hipGraphExecDestroy(runnable) == 0
        assert hip().hipGraphDestroy(graph) == 0


def test_two_contexts_at_once():
    """Calls in flight on two contexts of a device, each with its own scratch."""
    engines = [nn.Engine(0), nn.Engine(0)]
    w = weights(5)
    blocks = [Block("f16", 1500, w) for _ in engines]
    vs = [inputs(20 + i, "f16", SEQS, 1500) for i in range(2)]
    want = []
    for e, b, v in zip(engines, blocks, vs):
        b.put(v)
        b.calls(e)
        e.sync()
        want.append(b.results())
        b.clear()
        b.put(v)
    for b, v in zip(blocks, vs):
        b.put(v)
    for e, b in zip(engines, blocks):
        b.calls(e)
    for e in engines:
        e.sync()
    for b, r in zip(blocks, want):
        got = b.results()
        for n in got:
            assert np.array_equal(got[n], r[n]), n
    for e in engines:
        e.close()


def test_calls_in_flight_share_a_scratch(eng):
    """Long and short scans and attentions enqueued behind one another, none waited for, give the bits of each alone."""
    w = weights(6)
    blocks = [Block("bf16", n, w) for n in (2000, 40, 700, 2000)]
    vs = [inputs(30 + i, "bf16", SEQS, b.length) for i, b in enumerate(blocks)]
    want = []
    for b, v in zip(blocks, vs):
        b.put(v)
        b.calls(eng)
        eng.sync()
        want.append(b.results())
        b.clear()
        b.put(v)
    for b in blocks:
        b.calls(eng)
    eng.sync()
    for b, r in zip(blocks, want):
        got = b.results()
        for n in got:
            assert np.array_equal(got[n], r[n]), n


def test_a_failed_launch_is_reported_and_the_next_call_works(eng):
    w = weights(7)
    b, v = Block("f32", 600, w), inputs(40, "f32", SEQS, 600)
    b.put(v)
    b.calls(eng)
    eng.sync()
    want = b.results()
    for after in range(3):  # the scan's three launches
        b.clear()
        b.put(v)
        nn.rotary_noalloc(eng, b.rotary)
        nn.causal_conv_noalloc(eng, b.conv)
        eng.inject_failure(_lib.FAIL_LAUNCH, after)
        with pytest.raises(_lib.HipError) as e:
            nn.selective_scan_noalloc(eng, b.scan)
        assert e.value.kind == "Device"
        eng.sync()
    b.clear()
    b.put(v)
    b.calls(eng)
    eng.sync()
    got = b.results()
    for n in got:
        assert np.array_equal(got[n], want[n]), n
