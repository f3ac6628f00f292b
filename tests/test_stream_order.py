"""Order between a context's stream and a caller's (``zjai_order_after``, ``zjai_order_before``): buffers that another
stream fills and reads, and enqueued calls as part of a graph that it is captured into."""

import ctypes
from types import SimpleNamespace

import numpy as np
import pytest

from devbuf import DevBuf, hip, to_raw
from zenjpegai_amd import _lib, nn

NON_BLOCKING, D2D, CAPTURE_GLOBAL = 1, 3, 0
SEQS, HEADS, DK, DV = 2, 2, 32, 32


def test_a_null_context_is_refused():
    assert _lib.lib().zjai_order_after(None, None) == _lib.E_INVALID_ARGUMENT
    assert _lib.lib().zjai_order_before(None, None) == _lib.E_INVALID_ARGUMENT


@pytest.fixture(scope="module")
def eng():
    e = nn.Engine(0, "bf16")
    yield e
    e.close()


@pytest.fixture()
def stream():
    s = ctypes.c_void_p()
    assert hip().hipStreamCreateWithFlags(ctypes.byref(s), NON_BLOCKING) == 0
    yield s
    assert hip().hipStreamDestroy(s) == 0


def channels(seed, length):
    return to_raw(np.random.default_rng(seed).standard_normal((SEQS, length, HEADS * (2 * DK + DV))), "bf16")


def block(length):
    """Buffers and descriptors of a block's calls: sequences, a step on their states, a join."""
    rng = np.random.default_rng(1)
    c = HEADS * DV
    b = SimpleNamespace(
        qkv=DevBuf(channels(0, length)), out=DevBuf(to_raw(np.zeros((SEQS, length, c)), "bf16")),
        one=DevBuf(channels(99, 1)), one_out=DevBuf(to_raw(np.zeros((SEQS, 1, c)), "bf16")),
        decay=DevBuf(np.array([0.9, 0.999], np.float32)), state=DevBuf(np.zeros((SEQS, HEADS, DK, DV), np.float32)),
        x=DevBuf(to_raw(rng.standard_normal((SEQS, length, c)), "bf16")), x_out=DevBuf(to_raw(np.zeros((SEQS, length, c)), "bf16")),
        h=DevBuf(to_raw(np.zeros((SEQS, length, c)), "bf16")))
    common = dict(heads=HEADS, key_dim=DK, value_dim=DV, sequences=SEQS, decay=b.decay, scale=0.2)
    b.whole = nn.linear_attention_desc("bf16", b.qkv, b.out, length=length, state_out=b.state, **common)
    b.step = nn.linear_attention_desc("bf16", b.one, b.one_out, length=1, state_in=b.state, state_out=b.state, **common)
    b.join = nn.norm_gate_residual_desc("bf16", b.x, b.out, None, b.x_out, b.h, positions=SEQS * length, channels=c,
                                        post_norm="rms", post_groups=HEADS, pre_norm="layer")
    return b


def calls(eng, b):
    nn.linear_attention_noalloc(eng, b.whole)
    nn.linear_attention_step(eng, b.step)
    nn.norm_gate_residual_noalloc(eng, b.join)


def results(b):
    return [a.get() for a in (b.out, b.one_out, b.state, b.x_out, b.h)]


@pytest.mark.gpu
@pytest.mark.parametrize("wrapped", [False, True])
def test_inputs_from_and_outputs_to_another_stream(eng, stream, wrapped):
    """The other stream is milliseconds behind when a call is made, and overwrites its input when it has been used."""
    length = 700
    theirs = SimpleNamespace(cuda_stream=stream.value) if wrapped else stream
    b = block(length)
    inputs = [channels(s, length) for s in range(4)]
    want = []
    for x in inputs:
        b.qkv.put(x)
        calls(eng, b)
        eng.sync()
        want.append(results(b)[0])
    sources, sinks = [DevBuf(x) for x in inputs], [DevBuf(np.zeros_like(w)) for w in want]
    big = [DevBuf(np.zeros(1 << 28, np.uint8)) for _ in range(2)]
    b.qkv.put(np.zeros_like(inputs[0]))
    for src, dst in zip(sources, sinks):
        for _ in range(16):
            assert hip().hipMemcpyAsync(ctypes.c_void_p(big[0].address), ctypes.c_void_p(big[1].address), ctypes.c_size_t(1 << 28),
                                        D2D, stream) == 0
        assert hip().hipMemcpyAsync(ctypes.c_void_p(b.qkv.address), ctypes.c_void_p(src.address),
                                    ctypes.c_size_t(inputs[0].nbytes), D2D, stream) == 0
        eng.order_after(theirs)
        calls(eng, b)
        eng.order_before(theirs)
        assert hip().hipMemcpyAsync(ctypes.c_void_p(dst.address), ctypes.c_void_p(b.out.address), ctypes.c_size_t(want[0].nbytes),
                                    D2D, stream) == 0
    assert hip().hipStreamSynchronize(stream) == 0
    for dst, w in zip(sinks, want):
        assert np.array_equal(dst.get(), w)


@pytest.mark.gpu
def test_the_default_stream(eng):
    b = block(64)
    calls(eng, b)
    eng.sync()
    want = results(b)
    for a in (b.out, b.one_out, b.x_out, b.h):
        a.put(np.zeros(a.shape, a.dtype))
    eng.order_after()
    calls(eng, b)
    eng.order_before()
    assert hip().hipStreamSynchronize(None) == 0
    for got, w in zip(results(b), want):
        assert np.array_equal(got, w)


@pytest.mark.gpu
@pytest.mark.parametrize("length", [40, 900])
def test_calls_captured_into_a_graph_and_replayed(eng, stream, length):
    """Each replay, on inputs of its own and with eager calls of the same context between, gives the eager call's bits."""
    b, other = block(length), block(length)
    graph, runnable = ctypes.c_void_p(), ctypes.c_void_p()
    assert hip().hipStreamBeginCapture(stream, CAPTURE_GLOBAL) == 0
    eng.order_after(stream)
    calls(eng, b)
    eng.order_before(stream)
    assert hip().hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
    assert hip().hipGraphInstantiate(ctypes.byref(runnable), graph, None, None, ctypes.c_size_t(0)) == 0
    try:
        for i in range(4):
            x = channels(10 + i, length)
            for t in (b, other):
                t.qkv.put(x)
                t.out.put(np.zeros(t.out.shape, t.out.dtype))
            eng.order_before(stream)  # the context's scratch is the graph's too
            assert hip().hipGraphLaunch(runnable, stream) == 0
            eng.order_after(stream)
            calls(eng, other)
            eng.sync()
            assert hip().hipStreamSynchronize(stream) == 0
            for got, want in zip(results(b), results(other)):
                assert np.array_equal(got, want), i
            assert (results(other)[0] != 0).any()
    finally:
        assert hip().hipGraphExecDestroy(runnable) == 0
        assert hip().hipGraphDestroy(graph) == 0
