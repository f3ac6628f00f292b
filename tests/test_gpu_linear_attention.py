"""GPU: decayed linear attention against the recurrence in 64 bits: whole sequences and single positions, every
storage type, head sizes with and without whole 16 bytes, lengths from none to several chunks, kept
states, strides, idle and repeated slots, infinities, and the calls that are refused."""

import ctypes

import numpy as np
import pytest

from devbuf import DevBuf, from_raw, hip, to_raw
from linear_attention_oracle import oracle, out_bound, state_bound
from zenjpegai_amd import _lib, nn

pytestmark = pytest.mark.gpu

DECAYS = np.array([0.97, 1.0, 0.5, 0.0, 0.999, 0.875, 0.25, 0.99], np.float32)


@pytest.fixture(scope="module")
def eng():
    e = nn.Engine(0)
    yield e
    e.close()


def inputs(seed, prec, seqs, length, heads, dk, dv, fill=7.0):
    """Packed channels in the storage type and an output buffer of a known value."""
    rng = np.random.default_rng(seed)
    qkv = to_raw(rng.standard_normal((seqs, length, heads * (2 * dk + dv))), prec)
    out = to_raw(np.full((seqs, length, heads * dv), fill), prec)
    decay = np.resize(DECAYS, heads)
    state = (2 * rng.standard_normal((seqs, heads, dk, dv))).astype(np.float32)
    return qkv, out, decay, state


def parts(qkv, prec, heads, dk, dv):
    x = from_raw(qkv, prec)
    t, n = x.shape[0], heads * dk
    return x[:, :n].reshape(t, heads, dk), x[:, n:2 * n].reshape(t, heads, dk), x[:, 2 * n:].reshape(t, heads, dv)


def check_sequence(prec, heads, dk, dv, qkv, decay, scale, length, state, out, before, final):
    """One sequence's outputs and final state (None: not kept) against the oracle."""
    (o, oa, ob), (S, sa, sb) = oracle(*parts(qkv, prec, heads, dk, dv), decay, scale, length, state)
    got = from_raw(out, prec).reshape(o.shape)[:length]
    err, tol = np.abs(got - o[:length]), out_bound(prec, dk, o, oa, ob)[:length]
    assert (err <= tol).all(), (float((err / tol).max()), np.unravel_index(np.argmax(err / tol), err.shape))
    assert np.array_equal(out[length:], before[length:])
    if final is not None:
        err, tol = np.abs(final - S), state_bound(S, sa, sb)
        assert (err <= tol).all(), float((err / tol).max())


def run_whole(eng, prec, seqs, length, heads, dk, dv, lengths=None, keep=(True, True), scale=0.5, seed=1, offset=0):
    qkv, out, decay, state = inputs(seed, prec, seqs, length, heads, dk, dv)
    b = {n: DevBuf(a, offset if n in ("qkv", "out") else 0) for n, a in
         {"qkv": qkv, "out": out, "decay": decay, "in": state, "fin": np.full_like(state, 5.0)}.items()}
    d_len = None if lengths is None else DevBuf(np.asarray(lengths, np.int32))
    nn.linear_attention_noalloc(eng, nn.linear_attention_desc(
        prec, b["qkv"], b["out"], heads=heads, key_dim=dk, value_dim=dv, sequences=seqs, length=length,
        decay=b["decay"], scale=scale, lengths=d_len, state_in=b["in"] if keep[0] else None,
        state_out=b["fin"] if keep[1] else None))
    eng.sync()
    got, fin = b["out"].get(), b["fin"].get()
    for s in range(seqs):
        n = length if lengths is None else min(max(lengths[s], 0), length)
        check_sequence(prec, heads, dk, dv, qkv[s], decay, scale, n, state[s] if keep[0] else None, got[s], out[s],
                       fin[s] if keep[1] else None)
    if not keep[1]:
        assert (fin == 5.0).all()


@pytest.mark.parametrize("prec", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,dk,dv", [(1, 1, 1), (4, 32, 32), (3, 24, 40), (2, 20, 30), (2, 64, 128), (1, 128, 64),
                                         (2, 128, 256), (5, 16, 8)])
@pytest.mark.parametrize("length", [1, 5, 6, 31, 64, 193])
def test_whole_sequences_equal_the_recurrence(eng, prec, heads, dk, dv, length):
    run_whole(eng, prec, 2, length, heads, dk, dv, seed=length)


@pytest.mark.parametrize("prec", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("keep", [(False, False), (False, True), (True, False)])
def test_absent_states_are_zeros_and_not_written(eng, prec, keep):
    run_whole(eng, prec, 3, 70, 2, 32, 32, keep=keep, seed=3)


@pytest.mark.parametrize("prec", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dk,dv", [(32, 32), (64, 30), (128, 128)])
def test_ragged_lengths_leave_the_rest_as_it_was(eng, prec, dk, dv):
    run_whole(eng, prec, 7, 150, 2, dk, dv, lengths=[0, 1, 64, 150, 99, -5, 1000], seed=4)


@pytest.mark.parametrize("prec", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("seqs,length,heads,dk,dv", [(1, 3000, 4, 32, 32), (1, 2111, 1, 128, 128), (2, 2500, 3, 64, 48),
                                                     (40, 100, 8, 16, 16)])
def test_long_sequences_and_many(eng, prec, seqs, length, heads, dk, dv):
    run_whole(eng, prec, seqs, length, heads, dk, dv, seed=5)


@pytest.mark.parametrize("prec", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dk,dv", [(32, 32), (128, 96)])
def test_buffers_off_16_bytes(eng, prec, dk, dv):
    run_whole(eng, prec, 2, 130, 3, dk, dv, seed=6, offset=4 if prec == "f32" else 2)


def test_no_positions_pass_the_state_on(eng):
    run_whole(eng, "bf16", 3, 0, 2, 32, 32)
    run_whole(eng, "f32", 3, 40, 2, 32, 32, lengths=[0, 0, 0])
    run_whole(eng, "f32", 0, 40, 2, 32, 32)


@pytest.mark.parametrize("prec", ["f32", "bf16"])
def test_separate_buffers_with_gaps_between_positions_and_sequences(eng, prec):
    seqs, length, heads, dk, dv, scale = 3, 90, 2, 32, 64, 1.5
    qkv, _, decay, state = inputs(8, prec, seqs, length, heads, dk, dv)
    kc, vc = heads * dk, heads * dv
    width = {"q": kc + 8, "k": kc + 16, "v": vc + 3, "out": vc + 5}
    extra = {"q": 40, "k": 8, "v": 1, "out": 17}
    full = {n: np.zeros((seqs, length * w + extra[n]), qkv.dtype) + to_raw(np.float32(3), prec) for n, w in width.items()}
    for n, (lo, c) in {"q": (0, kc), "k": (kc, kc), "v": (2 * kc, vc)}.items():
        for s in range(seqs):
            full[n][s, :length * width[n]].reshape(length, width[n])[:, :c] = qkv[s, :, lo:lo + c]
    b = {n: DevBuf(a) for n, a in full.items()}
    d_decay, d_in = DevBuf(decay), DevBuf(state)
    st = {n + "_position": w for n, w in width.items()} | {n + "_sequence": a.shape[1] for n, a in full.items()}
    nn.linear_attention_noalloc(eng, nn.linear_attention_desc(
        prec, (b["q"], b["k"], b["v"]), b["out"], heads=heads, key_dim=dk, value_dim=dv, sequences=seqs, length=length,
        decay=d_decay, scale=scale, state_in=d_in, state_out=d_in, **st))
    eng.sync()
    got, fin, w = b["out"].get(), d_in.get(), width["out"]
    for s in range(seqs):
        rows = got[s, :length * w].reshape(length, w)
        check_sequence(prec, heads, dk, dv, qkv[s], decay, scale, length, state[s], rows[:, :vc], rows[:, :vc], fin[s])
        assert (rows[:, vc:] == full["out"][0, 0]).all() and (got[s, length * w:] == full["out"][0, 0]).all()


@pytest.mark.parametrize("prec", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dk,dv", [(32, 32), (128, 64)])
def test_an_infinity_reaches_only_its_position_and_later_ones(eng, prec, dk, dv):
    """One value channel of one position is infinite, a key of another position's NaN."""
    seqs, length, heads = 2, 140, 2
    qkv, out, decay, _ = inputs(9, prec, seqs, length, heads, dk, dv)
    decay[:] = [0.9, 1.0]
    x = from_raw(qkv, prec).astype(np.float32)
    x[0, 70, 2 * heads * dk + 3] = np.inf
    x[1, 90, heads * dk + dk + 5] = np.nan
    qkv = to_raw(x, prec)
    clean = x.copy()
    clean[0, 70, 2 * heads * dk + 3] = clean[1, 90, heads * dk + dk + 5] = 0.0
    b = [DevBuf(a) for a in (qkv, out, decay)]
    nn.linear_attention_noalloc(eng, nn.linear_attention_desc(prec, b[0], b[1], heads=heads, key_dim=dk, value_dim=dv,
                                                              sequences=seqs, length=length, decay=b[2]))
    eng.sync()
    got = from_raw(b[1].get(), prec).reshape(seqs, length, heads, dv)
    hit = np.zeros(got.shape, bool)
    hit[0, 70:, 0, 3] = True
    hit[1, 90:, 1, :] = True
    assert not np.isfinite(got[hit]).any()
    for s in range(seqs):
        (o, oa, ob), _ = oracle(*parts(to_raw(clean[s], prec), prec, heads, dk, dv), decay, 1.0, length)
        ok = ~hit[s]
        assert (np.abs(got[s] - o) <= out_bound(prec, dk, o, oa, ob))[ok].all()


@pytest.mark.parametrize("prec", ["f32", "f16", "bf16"])
def test_a_memory_of_a_million_positions(eng, prec):
    """Decays next to one, over many segments."""
    seqs, length, heads, dk, dv = 1, 6001, 2, 16, 16
    qkv, out, _, state = inputs(20, prec, seqs, length, heads, dk, dv)
    decay = np.array([1 - 2.0 ** -20, 1 - 2.0 ** -24], np.float32)
    b = [DevBuf(a) for a in (qkv, out, decay, state)]
    nn.linear_attention_noalloc(eng, nn.linear_attention_desc(prec, b[0], b[1], heads=heads, key_dim=dk, value_dim=dv, sequences=1,
                                                              length=length, decay=b[2], state_in=b[3], state_out=b[3]))
    eng.sync()
    check_sequence(prec, heads, dk, dv, qkv[0], decay, 1.0, length, state[0], b[1].get()[0], out[0], b[3].get()[0])


@pytest.mark.parametrize("dk,dv", [(32, 32), (64, 64), (128, 128)])
@pytest.mark.parametrize("k_size,v_size", [(200.0, 20000.0), (20000.0, 200.0), (1e-3, 1e-4)])
def test_f16_values_at_the_ends_of_their_range(eng, dk, dv, k_size, v_size):
    """Products and states far beyond f16's range, outputs back in it by the scale; and small ones."""
    prec, length, heads = "f16", 100, 2
    qkv, out, decay, _ = inputs(21, prec, 1, length, heads, dk, dv)
    x = from_raw(qkv, prec)
    x[..., heads * dk:2 * heads * dk] *= k_size
    x[..., 2 * heads * dk:] *= v_size
    qkv = to_raw(np.clip(x, -6e4, 6e4), prec)
    scale = 1.0 / (k_size * v_size)
    b = [DevBuf(a) for a in (qkv, out, decay)]
    fin = DevBuf(np.zeros((1, heads, dk, dv), np.float32))
    nn.linear_attention_noalloc(eng, nn.linear_attention_desc(prec, b[0], b[1], heads=heads, key_dim=dk, value_dim=dv, sequences=1,
                                                              length=length, decay=b[2], scale=scale, state_out=fin))
    eng.sync()
    check_sequence(prec, heads, dk, dv, qkv[0], decay, scale, length, None, b[1].get()[0], out[0], fin.get()[0])


@pytest.mark.parametrize("prec", ["f32", "bf16"])
def test_two_contexts_and_other_calls_in_flight_together(prec):
    """Calls of two contexts that nothing orders, each between channel-attention calls that use its scratch too."""
    engs = [nn.Engine(0, prec) for _ in range(2)]
    seqs, length, heads, dk, dv = 1, 1500, 2, 32, 32
    runs = []
    for i, e in enumerate(engs):
        qkv, out, decay, state = inputs(30 + i, prec, seqs, length, heads, dk, dv)
        b = [DevBuf(a) for a in (qkv, out, decay, state)]
        other = DevBuf(np.random.default_rng(i).standard_normal((20, 24, 3 * 64)).astype(np.float32))
        y = DevBuf(np.zeros((20, 24, 64), np.float32))
        temp = DevBuf(np.ones(4, np.float32))
        d = nn.linear_attention_desc(prec, b[0], b[1], heads=heads, key_dim=dk, value_dim=dv, sequences=1, length=length,
                                     decay=b[2], scale=0.5)
        runs.append((e, b, d, qkv, out, decay, other, y, temp))
    for _ in range(3):
        for e, _, d, _, _, _, other, y, temp in runs:
            _lib.check(_lib.lib().zjai_channel_attention_noalloc(e.handle, other.address, 192, 20, 24, 4, temp.address,
                                                                 _lib.F32, y.address), e.handle)
            nn.linear_attention_noalloc(e, d)
    for e, b, _, qkv, out, decay, *_ in runs:
        e.sync()
        check_sequence(prec, heads, dk, dv, qkv[0], decay, 0.5, length, None, b[1].get()[0], out[0], None)
    del runs, b
    for e in engs:
        e.close()


def test_offsets_that_pass_32_bits(eng):
    """Two sequences 2^31 + 64 elements apart, and a state slot whose offset passes 2^31 floats."""
    prec, heads, dk, dv, length = "bf16", 1, 32, 32, 70
    qkv, out, decay, _ = inputs(40, prec, 2, length, heads, dk, dv)
    gap, width = (1 << 31) + 64, heads * (2 * dk + dv)
    big = ctypes.c_void_p()
    assert hip().hipMalloc(ctypes.byref(big), 2 * (2 * gap + length * width)) == 0
    try:
        d_decay = DevBuf(decay)
        for s in range(2):
            at = big.value + 2 * s * gap
            assert hip().hipMemcpy(at, np.ascontiguousarray(qkv[s]).ctypes.data, qkv[s].nbytes, 1) == 0
        out_at = big.value + 2 * length * width  # behind the first sequence's inputs, and behind the second's
        nn.linear_attention_noalloc(eng, nn.linear_attention_desc(
            prec, big.value, out_at, heads=heads, key_dim=dk, value_dim=dv, sequences=2, length=length, decay=d_decay,
            q_sequence=gap, k_sequence=gap, v_sequence=gap, out_sequence=gap))
        eng.sync()
        for s in range(2):
            got = np.empty((length, heads * dv), np.uint16)
            assert hip().hipMemcpy(got.ctypes.data, out_at + 2 * s * gap, got.nbytes, 2) == 0
            check_sequence(prec, heads, dk, dv, qkv[s], decay, 1.0, length, None, got, got, None)
    finally:
        hip().hipFree(big)
    heads, dk, dv, slots = 1, 128, 1024, 16386  # 2^17 floats a state
    qkv, out, decay, state = inputs(41, "f32", 1, 1, heads, dk, dv)
    assert hip().hipMalloc(ctypes.byref(big), 4 * slots * dk * dv) == 0
    try:
        at = big.value + 4 * (slots - 1) * dk * dv
        assert hip().hipMemcpy(at, state.ctypes.data, state.nbytes, 1) == 0
        b = [DevBuf(a) for a in (qkv, out, decay, np.array([slots - 1], np.int32))]
        nn.linear_attention_step(eng, nn.linear_attention_desc("f32", b[0], b[1], heads=heads, key_dim=dk, value_dim=dv, sequences=1,
                                                               length=1, decay=b[2], slots=b[3], num_slots=slots,
                                                               state_in=big.value, state_out=big.value))
        eng.sync()
        fin = np.empty_like(state[0])
        assert hip().hipMemcpy(fin.ctypes.data, at, fin.nbytes, 2) == 0
        check_sequence("f32", heads, dk, dv, qkv[0], decay, 1.0, 1, state[0], b[1].get()[0], out[0], fin)
    finally:
        hip().hipFree(big)


@pytest.mark.parametrize("what,after", [(_lib.FAIL_LAUNCH, 0), (_lib.FAIL_LAUNCH, 1), (_lib.FAIL_LAUNCH, 2), (_lib.FAIL_ALLOC, 0),
                                        (_lib.FAIL_ALLOC, 1)])
def test_an_injected_failure_is_reported_and_the_context_goes_on(what, after):
    e = nn.Engine(0)
    x = np.random.default_rng(0).standard_normal((96, 40, 50)).astype(np.float32)
    t = nn.BTensor.from_planar(e, x)
    want = nn.linear_attention(e, t, 1, 32, [0.9]).to_planar()
    e.inject_failure(what, after)
    with pytest.raises(_lib.HipError) as err:
        nn.linear_attention(e, t, 1, 32, [0.9])
    assert err.value.kind == ("Device" if what == _lib.FAIL_LAUNCH else "LimitExceeded")
    assert np.array_equal(nn.linear_attention(e, t, 1, 32, [0.9]).to_planar(), want)
    del t
    e.close()


def test_repeated_calls_give_the_same_bits(eng):
    for prec, seqs, length, dk, dv in (("bf16", 1, 5000, 64, 64), ("f32", 3, 700, 32, 48)):
        qkv, out, decay, state = inputs(50, prec, seqs, length, 2, dk, dv)
        b = [DevBuf(a) for a in (qkv, out, decay, state)]
        fin = [DevBuf(np.zeros_like(state)) for _ in range(2)]
        got = []
        for f in fin:
            nn.linear_attention_noalloc(eng, nn.linear_attention_desc(prec, b[0], b[1], heads=2, key_dim=dk, value_dim=dv, sequences=seqs,
                                                                      length=length, decay=b[2], state_in=b[3], state_out=f))
            eng.sync()
            got.append((b[1].get(), f.get()))
        assert np.array_equal(got[0][0], got[1][0]) and np.array_equal(got[0][1], got[1][1])


@pytest.mark.parametrize("prec", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dk,dv", [(32, 32), (64, 40), (128, 128)])
def test_what_lies_behind_a_sequence_is_not_read(eng, prec, dk, dv):
    """NaN in q, k and v past the lengths."""
    lengths, length, heads = [1, 31, 33, 0, 64], 70, 2
    qkv, out, decay, state = inputs(60, prec, len(lengths), length, heads, dk, dv)
    clean = qkv.copy()
    for s, n in enumerate(lengths):
        qkv[s, n:] = to_raw(np.full(qkv[s, n:].shape, np.nan), prec)
    b = [DevBuf(a) for a in (qkv, out, decay, state, np.zeros_like(state), np.asarray(lengths, np.int32))]
    nn.linear_attention_noalloc(eng, nn.linear_attention_desc(prec, b[0], b[1], heads=heads, key_dim=dk, value_dim=dv,
                                                              sequences=len(lengths), length=length, decay=b[2], state_in=b[3],
                                                              state_out=b[4], lengths=b[5]))
    eng.sync()
    got, fin = b[1].get(), b[4].get()
    for s, n in enumerate(lengths):
        check_sequence(prec, heads, dk, dv, clean[s], decay, 1.0, n, state[s], got[s], out[s], fin[s])


@pytest.mark.parametrize("prec", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("length", [3, 100, 2500])
def test_one_query_for_all_positions_and_keys_that_sequences_share(eng, prec, length):
    heads, dk, dv, seqs = 2, 32, 64, 2
    qkv, out, decay, _ = inputs(61, prec, 1, length, heads, dk, dv)
    n = heads * dk
    b = [DevBuf(a) for a in (qkv, np.repeat(out, seqs, 0), decay)]
    nn.linear_attention_noalloc(eng, nn.linear_attention_desc(prec, b[0], b[1], heads=heads, key_dim=dk, value_dim=dv, sequences=seqs,
                                                              length=length, decay=b[2], q_position=0, q_sequence=0,
                                                              k_sequence=0, v_sequence=0))
    eng.sync()
    same = qkv[0].copy()
    same[:, :n] = same[:1, :n]
    got = b[1].get()
    for s in range(seqs):
        check_sequence(prec, heads, dk, dv, same, decay, 1.0, length, None, got[s], out[0], None)


def test_more_than_a_launch_takes_is_refused_before_anything_is_read(eng):
    b = {n: DevBuf(np.zeros(64, np.float32)) for n in ("qkv", "out", "decay", "s0")}
    still = dict.fromkeys(("q_position", "k_position", "v_position", "q_sequence", "k_sequence", "v_sequence"), 0)

    def code(heads, sequences, length, step=False, **kw):
        d = nn.linear_attention_desc("f32", b["qkv"], b["out"], heads=heads, key_dim=1, value_dim=1, sequences=sequences,
                                     length=length, decay=b["decay"], **{**still, **kw})
        f = _lib.lib().zjai_linear_attention_step if step else _lib.lib().zjai_linear_attention_noalloc
        return f(eng.handle, ctypes.byref(d))

    assert code(1, 1, (1 << 30) + 1) == _lib.E_LIMIT
    for length in (1, 6):
        assert code(1, (1 << 22) + 1, length) == _lib.E_LIMIT
        assert code(1 << 12, (1 << 10) + 1, length) == _lib.E_LIMIT
        assert code(2**31 - 1, 2**31 - 1, length, out_sequence=2**40) == _lib.E_LIMIT
    assert code(1, (1 << 22) + 1, 1, step=True, state_in=b["s0"], state_out=b["s0"]) == _lib.E_LIMIT
    eng.sync()


@pytest.mark.parametrize("prec", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("keep", [(False, False), (False, True), (True, False), (True, True)])
@pytest.mark.parametrize("length", [2, 3, 4, 5, 6])
def test_short_sequences_with_and_without_states(eng, prec, keep, length):
    run_whole(eng, prec, 3, length, 2, 24, 40, lengths=[length, 1, length - 1], keep=keep, seed=70 + length)


# ------------------------------------------------------------------------- single positions
def run_step(eng, prec, n, heads, dk, dv, num_slots, slots, in_place, seed=11):
    qkv, out, decay, _ = inputs(seed, prec, n, 1, heads, dk, dv)
    state = np.random.default_rng(seed).standard_normal((num_slots, heads, dk, dv)).astype(np.float32)
    b = [DevBuf(a) for a in (qkv, out, decay, state)]
    d_out = b[3] if in_place else DevBuf(np.full_like(state, 5.0))
    d_slots = None if slots is None else DevBuf(np.asarray(slots, np.int32))
    nn.linear_attention_step(eng, nn.linear_attention_desc(
        prec, b[0], b[1], heads=heads, key_dim=dk, value_dim=dv, sequences=n, length=1, decay=b[2], scale=0.25,
        slots=d_slots, num_slots=num_slots, state_in=b[3], state_out=d_out))
    eng.sync()
    got, fin = b[1].get(), d_out.get()
    order = list(range(n)) if slots is None else slots
    for slot in range(num_slots):
        mine = [i for i in range(n) if order[i] == slot]
        if not mine:
            assert np.array_equal(fin[slot], state[slot] if in_place else np.full_like(state[slot], 5.0))
            continue
        check_sequence(prec, heads, dk, dv, qkv[mine, 0], decay, 0.25, len(mine), state[slot], got[mine, 0],
                       out[mine, 0], fin[slot])
    for i in range(n):
        if not 0 <= order[i] < num_slots:
            assert np.array_equal(got[i], out[i])


@pytest.mark.parametrize("prec", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,dk,dv", [(1, 1, 1), (4, 32, 32), (3, 24, 40), (2, 20, 30), (2, 64, 128), (1, 128, 64),
                                         (1, 128, 1000)])
@pytest.mark.parametrize("n", [1, 5])
def test_single_positions_equal_the_recurrence(eng, prec, heads, dk, dv, n):
    run_step(eng, prec, n, heads, dk, dv, n, None, in_place=n == 5)


@pytest.mark.parametrize("in_place", [False, True])
def test_slots_may_be_out_of_order_idle_and_repeated(eng, in_place):
    run_step(eng, "bf16", 9, 2, 32, 48, 12, [3, 0, -1, 7, 3, 12, 11, 3, 1 << 30], in_place)
    run_step(eng, "f32", 300, 1, 16, 16, 40, [(i * 7) % 43 for i in range(300)], in_place)
    run_step(eng, "f16", 6, 2, 128, 128, 4, [2] * 6, in_place)


@pytest.mark.parametrize("prec", ["f32", "f16", "bf16"])
def test_a_prompt_and_then_single_positions_continue_one_sequence(eng, prec):
    seqs, length, heads, dk, dv, cut = 2, 100, 2, 32, 64, 83
    qkv, out, decay, state = inputs(13, prec, seqs, length, heads, dk, dv)
    b = [DevBuf(a) for a in (qkv, out, decay, state)]
    width, ow = heads * (2 * dk + dv), heads * dv
    es = qkv.itemsize
    common = dict(heads=heads, key_dim=dk, value_dim=dv, sequences=seqs, decay=b[2], scale=0.5, state_in=b[3], state_out=b[3])
    strides = {n + "_sequence": width * length for n in "qkv"} | {"out_sequence": ow * length}
    nn.linear_attention_noalloc(eng, nn.linear_attention_desc(prec, b[0], b[1], length=cut, **common, **strides))
    for t in range(cut, length):
        nn.linear_attention_step(eng, nn.linear_attention_desc(
            prec, b[0].address + t * width * es, b[1].address + t * ow * es, length=1, **common, **strides))
    eng.sync()
    got, fin = b[1].get(), b[3].get()
    for s in range(seqs):
        check_sequence(prec, heads, dk, dv, qkv[s], decay, 0.5, length, state[s], got[s], out[s], fin[s])


# ------------------------------------------------------------------------------- tensor form
@pytest.mark.parametrize("prec", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,dk,dv,h,w", [(4, 32, 32, 9, 13), (3, 8, 12, 1, 1), (2, 64, 64, 20, 11)])
@pytest.mark.parametrize("rows", [False, True])
@pytest.mark.parametrize("crop", [False, True])
def test_maps_in_raster_order_and_row_by_row(prec, heads, dk, dv, h, w, rows, crop):
    e = nn.Engine(0, prec)
    c = heads * (2 * dk + dv)
    x = np.random.default_rng(h).standard_normal((c, h + 2 * crop, w + 3 * crop)).astype(np.float32)
    raw = to_raw(x, prec)
    t = nn.BTensor.from_planar(e, from_raw(raw, prec).astype(np.float32))
    if crop:
        t, raw = t.crop(h, w), raw[:, :h, :w]
    decay = np.resize(DECAYS, heads)
    y = nn.linear_attention(e, t, heads, dk, decay, 0.5, rows)
    assert y.shape == (heads * dv, h, w)
    got = to_raw(y.to_planar(), prec)
    seqs = raw.transpose(1, 2, 0) if rows else raw.transpose(1, 2, 0).reshape(1, h * w, c)
    outs = got.transpose(1, 2, 0).reshape(seqs.shape[0], seqs.shape[1], heads * dv)
    for s in range(seqs.shape[0]):
        check_sequence(prec, heads, dk, dv, seqs[s], decay, 0.5, seqs.shape[1], None, outs[s], outs[s], None)
    del y, t
    e.close()


def test_refused_calls(eng):
    b = {n: DevBuf(np.zeros(4096, np.float32)) for n in ("qkv", "out", "decay", "s0", "s1", "len")}
    good = dict(heads=2, key_dim=8, value_dim=8, sequences=2, length=4, decay=b["decay"])

    def code(step=False, prec="f32", qkv=b["qkv"], out=b["out"], edit=None, **kw):
        d = nn.linear_attention_desc(prec, qkv, out, **{**good, **kw})
        for n, v in (edit or {}).items():
            setattr(d, n, v)
        f = _lib.lib().zjai_linear_attention_step if step else _lib.lib().zjai_linear_attention_noalloc
        return f(eng.handle, ctypes.byref(d))

    bad = _lib.E_INVALID_ARGUMENT
    assert code() == _lib.OK
    assert code(edit={"precision": 3}) == bad
    for n in ("heads", "key_dim", "value_dim"):
        assert code(**{n: 0}) == bad
    assert code(sequences=-1) == bad and code(length=-1) == bad
    assert code(key_dim=129) == _lib.E_UNSUPPORTED and code(value_dim=1025) == _lib.E_UNSUPPORTED
    assert code(decay=None) == bad and code(scale=float("nan")) == bad and code(scale=float("inf")) == bad
    for n in ("q", "k", "v", "out"):
        assert code(edit={n: None}) == bad
        assert code(edit={n: b["s0"].address + 2}) == bad
    assert code(out=b["qkv"]) == bad
    assert code(q_position=-8) == bad and code(out_position=15) == bad and code(out_sequence=15) == bad
    assert code(edit={"slots": b["len"].address, "num_slots": 2}) == bad
    assert code(state_in=b["s0"], state_out=b["s0"].address + 64) == bad
    assert code(state_in=b["s0"].address + 2) == bad
    # The recurrent form's.
    step = dict(step=True, length=1, state_in=b["s0"], state_out=b["s1"])
    assert code(**step) == _lib.OK
    assert code(**{**step, "length": 2}) == bad and code(**step, lengths=b["len"]) == bad
    assert code(**{**step, "state_in": None}) == bad and code(**{**step, "state_out": None}) == bad
    assert code(**step, slots=b["len"]) == bad
    assert code(**step, edit={"num_slots": 1}) == bad
    assert _lib.lib().zjai_linear_attention_noalloc(None, None) == bad
    assert _lib.lib().zjai_linear_attention_step(eng.handle, None) == bad
    # The tensor form's.
    t = nn.BTensor.from_planar(eng, np.zeros((24, 2, 2), np.float32))
    for heads, dk, decay, rows in ((0, 4, [], 0), (5, 1, [0.5] * 5, 0), (2, 6, [0.5] * 2, 0), (2, 4, [0.5, 1.5], 0),
                                   (2, 4, [0.5, float("nan")], 0), (2, 4, [0.5, 0.5], 2), (2, 0, [0.5, 0.5], 0)):
        out = ctypes.c_void_p()
        d = (ctypes.c_float * 8)(*decay)
        assert _lib.lib().zjai_linear_attention(eng.handle, t._h, heads, dk, d, 1.0, rows, ctypes.byref(out)) == bad
    eng.sync()
