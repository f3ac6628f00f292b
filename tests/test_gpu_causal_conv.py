"""GPU: the short causal convolution against its sum in 64 bits: every number of taps, odd channel counts, lengths from
none to several runs, kept states (in place, too), strides, slots, infinities, and the calls that are refused."""

import numpy as np
import pytest

from devbuf import DevBuf, from_raw, to_raw
from state_space_oracle import conv
from zenjpegai_amd import _lib, nn

pytestmark = pytest.mark.gpu
PRECS = ["f32", "f16", "bf16"]


@pytest.fixture(scope="module")
def eng():
    e = nn.Engine(0)
    yield e
    e.close()


def inputs(seed, prec, seqs, length, channels, taps):
    rng = np.random.default_rng(seed)
    return (to_raw(rng.standard_normal((seqs, length, channels)), prec), rng.standard_normal((channels, taps)).astype(np.float32),
            rng.standard_normal(channels).astype(np.float32), to_raw(rng.standard_normal((seqs, taps - 1, channels)), prec))


def check(prec, got, x, w, b, act, n, state, fill, final):
    y, tol, last = conv(prec, from_raw(x, prec), w, b, act, n, None if state is None else from_raw(state, prec))
    err = np.abs(from_raw(got, prec) - y)[:n]
    assert (err <= tol[:n]).all(), (float((err - tol[:n]).max()), np.unravel_index(np.argmax(err - tol[:n]), err.shape))
    assert np.array_equal(got[n:], fill[n:])
    if final is not None:
        assert np.array_equal(from_raw(final, prec), last)


def run(eng, prec, seqs, length, channels, taps, act="silu", lengths=None, keep=(True, True), bias=True, in_place=False, seed=1,
        offset=0):
    x, w, b, state = inputs(seed, prec, seqs, length, channels, taps)
    fill = to_raw(np.full(x.shape, 7.0), prec)
    dx, do, dw, db, ds, df = (DevBuf(v, o) for v, o in (
        (x, offset), (fill, offset), (w, 0), (b, 0), (state, offset), (to_raw(np.full(state.shape, 9.0), prec), offset)))
    nn.causal_conv_noalloc(eng, nn.causal_conv_desc(
        prec, dx, do, channels=channels, taps=taps, sequences=seqs, length=length, weight=dw, bias=db if bias else None, act=act,
        lengths=None if lengths is None else DevBuf(np.asarray(lengths, np.int32)), state_in=ds if keep[0] else None,
        state_out=(ds if in_place else df) if keep[1] else None))
    eng.sync()
    got, fin = do.get(), (ds if in_place else df).get()
    for s in range(seqs):
        n = length if lengths is None else min(max(lengths[s], 0), length)
        check(prec, got[s], x[s], w, b if bias else None, act, n, state[s] if keep[0] else None, fill[s], fin[s] if keep[1] else None)
    if not keep[1]:
        assert (from_raw(df.get(), prec) == 9.0).all()


@pytest.mark.parametrize("prec", PRECS)
@pytest.mark.parametrize("taps", range(1, 9))
@pytest.mark.parametrize("channels", [1, 6, 100, 257])
def test_equals_the_sum(eng, prec, taps, channels):
    for length in (1, 5, 33, 70):
        run(eng, prec, 2, length, channels, taps, seed=length)


@pytest.mark.parametrize("prec", PRECS)
@pytest.mark.parametrize("act", ["linear", "sigmoid", "silu"])
def test_activations_and_an_absent_bias(eng, prec, act):
    for bias in (False, True):
        run(eng, prec, 3, 50, 64, 4, act=act, bias=bias)


@pytest.mark.parametrize("prec", PRECS)
@pytest.mark.parametrize("keep", [(False, False), (False, True), (True, False)])
@pytest.mark.parametrize("taps", [1, 2, 8])
def test_absent_states_are_zeros_and_not_written(eng, prec, keep, taps):
    run(eng, prec, 3, 70, 40, taps, keep=keep, lengths=[70, 3, 0])


@pytest.mark.parametrize("prec", PRECS)
@pytest.mark.parametrize("taps", [2, 4, 8])
@pytest.mark.parametrize("in_place", [False, True])
def test_ragged_lengths_and_states_in_place(eng, prec, taps, in_place):
    """Lengths shorter than the taps keep a part of the state that was; far runs of a sequence do not see the new one."""
    run(eng, prec, 11, 150, 72, taps, lengths=[0, 1, 2, 3, 6, 7, 150, 99, 64, -5, 1000], in_place=in_place)


@pytest.mark.parametrize("prec", PRECS)
@pytest.mark.parametrize("in_place", [False, True])
def test_long_sequences_and_many(eng, prec, in_place):
    run(eng, prec, 1, 20001, 24, 4, in_place=in_place)
    run(eng, prec, 300, 40, 16, 3, in_place=in_place)


@pytest.mark.parametrize("prec", PRECS)
def test_buffers_off_16_bytes(eng, prec):
    es = 4 if prec == "f32" else 2
    for offset in (es, 2 * es, 8):
        run(eng, prec, 2, 45, 64, 4, offset=offset)


def test_no_positions_pass_the_state_on(eng):
    run(eng, "bf16", 3, 0, 24, 4)
    run(eng, "f32", 3, 0, 24, 4, in_place=True)
    run(eng, "f32", 0, 40, 24, 4)


@pytest.mark.parametrize("prec", PRECS)
def test_packed_channels_and_gaps(eng, prec):
    seqs, length, c, taps = 2, 40, 30, 4
    x, w, b, state = inputs(3, prec, seqs, length, c, taps)
    for xp, op in ((2 * c, c), (c + 1, c + 3), (2 * c + 4, 2 * c + 4)):
        full = to_raw(np.full((seqs, length * xp + 3), 100.0), prec)
        for s in range(seqs):
            full[s, :length * xp].reshape(length, xp)[:, :c] = x[s]
        fill = to_raw(np.full((seqs, length * op + 5), 7.0), prec)
        dx, do, dw, db, ds = (DevBuf(v) for v in (full, fill, w, b, state))
        nn.causal_conv_noalloc(eng, nn.causal_conv_desc(
            prec, dx, do, channels=c, taps=taps, sequences=seqs, length=length, weight=dw, bias=db, act="silu", state_in=ds,
            x_position=xp, x_sequence=length * xp + 3, out_position=op, out_sequence=length * op + 5))
        eng.sync()
        got = do.get()
        for s in range(seqs):
            rows = got[s, :length * op].reshape(length, op)
            check(prec, rows[:, :c], x[s], w, b, "silu", length, state[s], rows[:, :c], None)
            assert (rows[:, c:] == fill[0, 0]).all() and (got[s, length * op:] == fill[0, 0]).all()


@pytest.mark.parametrize("prec", PRECS)
@pytest.mark.parametrize("taps,channels", [(1, 20), (2, 64), (4, 300), (5, 33), (8, 1000)])
@pytest.mark.parametrize("in_place", [False, True])
def test_steps_equal_whole_sequences(eng, prec, taps, channels, in_place):
    seqs, length = 3, 12
    x, w, b, state = inputs(5, prec, seqs, length, channels, taps)
    dw, db = DevBuf(w), DevBuf(b)
    cur, new = DevBuf(state), DevBuf(np.zeros_like(state))
    one, out = DevBuf(x[:, :1]), DevBuf(np.zeros_like(x[:, :1]))
    for t in range(length):
        one.put(x[:, t:t + 1])
        nn.causal_conv_step(eng, nn.causal_conv_desc(
            prec, one, out, channels=channels, taps=taps, sequences=seqs, length=1, weight=dw, bias=db, act="silu",
            state_in=cur if taps > 1 else None, state_out=(cur if in_place else new) if taps > 1 else None))
        eng.sync()
        for s in range(seqs):
            y, tol, _ = conv(prec, from_raw(x[s], prec), w, b, "silu", length, from_raw(state[s], prec))
            assert (np.abs(from_raw(out.get()[s, 0], prec) - y[t]) <= tol[t]).all()
        if not in_place:
            cur, new = new, cur
    for s in range(seqs):
        want = np.concatenate([state[s], x[s]])[length:]
        assert np.array_equal(cur.get()[s], want)


@pytest.mark.parametrize("prec", PRECS)
@pytest.mark.parametrize("in_place", [False, True])
def test_slots_idle_and_repeated(eng, prec, in_place):
    """Idle sequences and other slots' states stay as they were; sequences of one slot are consecutive positions."""
    slots = np.array([4, -1, 2, 7, 4, 100, 0, 4, 2], np.int32)
    seqs, channels, taps, num = len(slots), 70, 4, 7
    x, w, b, _ = inputs(6, prec, seqs, 1, channels, taps)
    state = inputs(7, prec, num, 1, channels, taps)[3]
    fill = to_raw(np.full(x.shape, 7.0), prec)
    dx, do, dw, db, di, dn, sl = (DevBuf(v) for v in (x, fill, w, b, state, np.zeros_like(state), slots))
    to = di if in_place else dn
    before = to.get()
    nn.causal_conv_step(eng, nn.causal_conv_desc(prec, dx, do, channels=channels, taps=taps, sequences=seqs, length=1, weight=dw, bias=db,
                                                 act="silu", slots=sl, num_slots=num, state_in=di, state_out=to))
    eng.sync()
    got, fin = do.get(), to.get()
    for slot in range(-1, 101):
        at = np.flatnonzero(slots == slot)
        if not 0 <= slot < num:
            assert np.array_equal(got[at], fill[at])
        elif not len(at):
            assert np.array_equal(fin[slot], before[slot])
        else:
            check(prec, got[at, 0], x[at, 0], w, b, "silu", len(at), state[slot], fill[at, 0], fin[slot])


@pytest.mark.parametrize("prec", PRECS)
def test_non_finite_inputs_reach_the_taps_that_see_them(eng, prec):
    length, channels, taps = 40, 16, 3
    x, w, b, state = inputs(8, prec, 1, length, channels, taps)
    v = from_raw(x, prec).astype(np.float32)
    v[0, 10, 3], v[0, 30, 5], v[0, 39, 7] = np.inf, np.nan, -np.inf
    raw = to_raw(v, prec)
    dx, do, dw, db, ds, df = (DevBuf(a) for a in (raw, np.zeros_like(raw), w, b, state, np.zeros_like(state)))
    nn.causal_conv_noalloc(eng, nn.causal_conv_desc(prec, dx, do, channels=channels, taps=taps, sequences=1, length=length, weight=dw,
                                                    bias=db, state_in=ds, state_out=df))
    eng.sync()
    bad = ~np.isfinite(from_raw(do.get(), prec)[0])
    want = np.zeros_like(bad)
    want[10:13, 3] = want[30:33, 5] = want[39, 7] = True
    assert np.array_equal(bad, want)
    assert np.array_equal(~np.isfinite(from_raw(df.get(), prec)[0]), ~np.isfinite(v[0, -2:]))


@pytest.mark.parametrize("prec", PRECS)
def test_offsets_past_32_bits(eng, prec):
    import ctypes
    from devbuf import hip
    c, taps, far, es = 8, 3, 3 * 2 ** 30, 4 if prec == "f32" else 2
    x, w, b, _ = inputs(9, prec, 1, 2, c, taps)
    base = ctypes.c_void_p()
    assert hip().hipMalloc(ctypes.byref(base), ctypes.c_size_t((far + 64) * es)) == 0
    try:
        for i in range(2):
            assert hip().hipMemcpy(base.value + i * far * es, x[0, i].ctypes.data, x[0, i].nbytes, 1) == 0
        out, dw, db = DevBuf(np.zeros_like(x[0])), DevBuf(w), DevBuf(b)
        for seqs, length in ((1, 2), (2, 1)):
            nn.causal_conv_noalloc(eng, nn.causal_conv_desc(prec, base.value, out, channels=c, taps=taps, sequences=seqs, length=length,
                                                            weight=dw, bias=db, x_position=far, x_sequence=far, out_position=c,
                                                            out_sequence=c))
            eng.sync()
            for s in range(seqs):
                at = slice(s, s + 1) if length == 1 else slice(0, 2)
                check(prec, out.get()[at], x[0, at], w, b, "linear", length, None, out.get()[at], None)
    finally:
        hip().hipFree(base)


@pytest.mark.parametrize("prec", PRECS)
@pytest.mark.parametrize("rows", [False, True])
def test_a_map(prec, rows):
    e = nn.Engine(0, prec)
    c, h, w, taps = 20, 6, 9, 4
    rng = np.random.default_rng(10)
    x, wt, b = rng.standard_normal((c, h, w)).astype(np.float32), rng.standard_normal((c, taps)), rng.standard_normal(c)
    wt, b = wt.astype(np.float32), b.astype(np.float32)
    big = np.full((c, h + 1, w + 2), 50.0, np.float32)
    big[:, :h, :w] = x
    for t in (nn.BTensor.from_planar(e, x), nn.BTensor.from_planar(e, big).crop(h, w)):
        v = to_raw(t.to_planar(), prec).reshape(c, h, w).transpose(1, 2, 0)
        got = to_raw(nn.causal_conv(e, t, wt, b, act="silu", rows=rows).to_planar(), prec).transpose(1, 2, 0)
        seqs = (h, w) if rows else (1, h * w)
        for xs, gs in zip(np.ascontiguousarray(v).reshape(*seqs, c), np.ascontiguousarray(got).reshape(*seqs, c)):
            check(prec, gs, xs, wt, b, "silu", seqs[1], None, gs, None)
        del t
    e.close()


def test_refusals(eng):
    x, o, w, s = (DevBuf(np.zeros(n, np.float32)) for n in (2 * 4 * 16, 2 * 4 * 16, 64, 512))
    good = dict(channels=16, taps=4, sequences=2, length=4, weight=w)

    def refused(kind="InvalidArgument", call=nn.causal_conv_noalloc, x=x, out=o, prec="f32", **kw):
        desc = nn.causal_conv_desc(prec, x, out, **{**good, **{k: v for k, v in kw.items() if k != "fields"}})
        for k, v in kw.get("fields", {}).items():
            setattr(desc, k, v)
        with pytest.raises(_lib.HipError) as e:
            call(eng, desc)
        assert e.value.kind == kind, e.value

    refused(channels=0)
    refused(kind="Unsupported", channels=2 ** 20 + 1)
    refused(taps=0)
    refused(kind="Unsupported", taps=9)
    refused(fields={"act": 3})
    refused(fields={"act": -1})
    refused(fields={"precision": 3})
    refused(fields={"reserved": 1})
    refused(fields={"num_slots": 1})
    refused(sequences=-1)
    refused(length=-1)
    refused(kind="LimitExceeded", length=2 ** 30 + 1)
    refused(weight=None)
    refused(weight=w.address + 2)
    refused(bias=w.address + 1)
    refused(lengths=w.address + 2)
    refused(x=None)
    refused(out=None)
    refused(x=x.address + 2)
    refused(out=x)
    refused(x_position=-1)
    refused(out_position=15)
    refused(out_sequence=15)
    refused(out_position=16, out_sequence=16)
    refused(slots=w, num_slots=2)
    refused(state_in=s.address + 2)
    refused(state_in=s, state_out=s.address + 64)
    step = dict(call=nn.causal_conv_step, length=1)
    refused(**step)
    refused(**step, state_in=s)
    refused(**step, state_in=s, state_out=s, lengths=w)
    refused(call=nn.causal_conv_step, state_in=s, state_out=s)
    refused(**step, state_in=s, state_out=s, slots=w)
    refused(**step, state_in=s, state_out=s, slots=w, num_slots=-1)
    refused(**step, state_in=s, state_out=s, fields={"num_slots": 1})
    refused(**step, state_in=s, state_out=s, slots=w.address + 2, num_slots=2)
    refused(kind="LimitExceeded", **{**step, "sequences": 2 ** 24}, state_in=s, state_out=s)
    t = nn.BTensor.from_planar(eng, np.zeros((16, 2, 2), np.float32))
    for weight, bias, kw in ((np.zeros((15, 4)), None, {}), (np.zeros(64), None, {}), (np.zeros((16, 4)), np.zeros(15), {}),
                             (np.zeros((16, 0)), None, {})):
        with pytest.raises(_lib.HipError) as e:
            nn.causal_conv(eng, t, weight, bias, **kw)
        assert e.value.kind == "InvalidArgument"
    nn.causal_conv_noalloc(eng, nn.causal_conv_desc("f32", x, o, **good))
    eng.sync()
