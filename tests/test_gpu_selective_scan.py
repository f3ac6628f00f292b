"""GPU: the selective state-space scan against its recurrence in 64 bits: state and channel counts with and without whole
vectors, groups, lengths from none to many segments, kept states (in place, too), ragged lengths, single
positions in slots, strides, infinities, extreme steps, and the calls that are refused."""

import numpy as np
import pytest

from devbuf import DevBuf, from_raw, to_raw
from state_space_oracle import scan
from zenjpegai_amd import _lib, nn

pytestmark = pytest.mark.gpu
PRECS = ["f32", "f16", "bf16"]


@pytest.fixture(scope="module")
def eng():
    e = nn.Engine(0)
    yield e
    e.close()


class Case:
    """Inputs of a call. Steps after the softplus lie around `step`, the decays of a state go from -1 to -n."""

    def __init__(self, seed, prec, seqs, length, channels, n, groups=1, softplus=True, step=0.03):
        rng = np.random.default_rng(seed)
        self.prec, self.softplus, self.shape = prec, softplus, (seqs, length, channels, n, groups)
        raw = lambda *s: to_raw(rng.standard_normal(s), prec)  # noqa: E731
        self.x, self.z = raw(seqs, length, channels), raw(seqs, length, channels)
        self.b, self.c = raw(seqs, length, groups * n), raw(seqs, length, groups * n)
        self.delta = raw(seqs, length, channels) if softplus else to_raw(step * rng.uniform(0.1, 2.0, (seqs, length, channels)), prec)
        self.a = (-np.arange(1, n + 1) * rng.uniform(0.8, 1.2, (channels, n))).astype(np.float32)
        self.d = rng.standard_normal(channels).astype(np.float32)
        self.bias = (np.log(np.expm1(step)) + 0.5 * rng.standard_normal(channels)).astype(np.float32) if softplus else np.zeros(channels, np.float32)
        self.state = rng.standard_normal((seqs, channels, n)).astype(np.float32)

    def check(self, s, got, n, fill, state, final, gate=True, skip=True, bias=True, what=slice(None)):
        """Sequence s (positions `what` of it) against the oracle."""
        _, _, _, m, g = self.shape
        x, delta, z, b, c = (from_raw(v[s][what], self.prec) for v in (self.x, self.delta, self.z, self.b, self.c))
        b, c = b.reshape(-1, g, m), c.reshape(-1, g, m)
        y, tol, h, htol = scan(self.prec, x, delta, b, c, z if gate else None, self.a, self.d if skip else None,
                               self.bias if bias else None, self.softplus, n, state)
        err = np.abs(from_raw(got, self.prec) - y)[:n]
        assert (err <= tol[:n]).all(), (float((err / tol[:n]).max()), np.unravel_index(np.argmax(err / tol[:n]), err.shape))
        assert np.array_equal(got[n:], fill[n:])
        if final is not None:
            err = np.abs(final - h)
            assert (err <= htol).all(), float((err / htol).max())


def run(eng, k, lengths=None, keep=(True, True), gate=True, skip=True, bias=True, in_place=False, offset=0, only=None):
    seqs, length, channels, n, groups = k.shape
    fill = to_raw(np.full(k.x.shape, 7.0), k.prec)
    dx, dd, dz, db, dc, do = (DevBuf(v, offset) for v in (k.x, k.delta, k.z, k.b, k.c, fill))
    da, dk, dbias = DevBuf(k.a), DevBuf(k.d), DevBuf(k.bias)
    ds, df = DevBuf(k.state), DevBuf(np.full_like(k.state, 5.0))
    nn.selective_scan_noalloc(eng, nn.selective_scan_desc(
        k.prec, dx, dd, db, dc, do, channels=channels, state_dim=n, sequences=seqs, length=length, a=da, z=dz if gate else None,
        groups=groups, d=dk if skip else None, delta_bias=dbias if bias else None, softplus=k.softplus,
        lengths=None if lengths is None else DevBuf(np.asarray(lengths, np.int32)), state_in=ds if keep[0] else None,
        state_out=(ds if in_place else df) if keep[1] else None))
    eng.sync()
    got, fin = do.get(), (ds if in_place else df).get()
    for s in range(seqs) if only is None else only:
        m = length if lengths is None else min(max(lengths[s], 0), length)
        k.check(s, got[s], m, fill[s], k.state[s] if keep[0] else None, fin[s] if keep[1] else None, gate, skip, bias)
    if not keep[1]:
        assert (df.get() == 5.0).all()
    return got, fin


@pytest.mark.parametrize("prec", PRECS)
@pytest.mark.parametrize("channels,n,groups", [(1, 1, 1), (64, 16, 1), (100, 16, 2), (70, 1, 1), (40, 3, 1), (129, 5, 3), (48, 8, 4),
                                               (66, 24, 2), (20, 64, 1), (9, 256, 3), (7, 100, 7), (320, 12, 1), (16, 2, 1), (128, 32, 1)])
def test_whole_sequences_equal_the_recurrence(eng, prec, channels, n, groups):
    for length in (1, 8, 9, 63):
        run(eng, Case(length, prec, 2, length, channels, n, groups))


@pytest.mark.parametrize("prec", PRECS)
@pytest.mark.parametrize("channels,n,groups", [(64, 16, 1), (24, 64, 2), (100, 4, 1), (33, 20, 1)])
@pytest.mark.parametrize("seqs,length", [(1, 1500), (3, 777), (2, 64), (1, 65)])
def test_sequences_cut_into_segments(eng, prec, channels, n, groups, seqs, length):
    run(eng, Case(7, prec, seqs, length, channels, n, groups))


@pytest.mark.parametrize("prec", PRECS)
def test_one_long_sequence(eng, prec):
    run(eng, Case(8, prec, 1, 12001, 16, 16, step=0.002))


@pytest.mark.parametrize("prec", PRECS)
def test_many_sequences(eng, prec):
    run(eng, Case(9, prec, 300, 40, 64, 16), only=[0, 1, 150, 299])


@pytest.mark.parametrize("prec", PRECS)
@pytest.mark.parametrize("softplus", [False, True])
@pytest.mark.parametrize("gate,skip,bias", [(False, False, False), (True, False, True), (False, True, False), (False, False, True)])
def test_absent_parts(eng, prec, softplus, gate, skip, bias):
    for length in (20, 400):
        run(eng, Case(10, prec, 2, length, 40, 16, softplus=softplus), gate=gate, skip=skip, bias=bias)


@pytest.mark.parametrize("prec", PRECS)
@pytest.mark.parametrize("keep", [(False, False), (False, True), (True, False)])
@pytest.mark.parametrize("length", [30, 500])
def test_absent_states_are_zeros_and_not_written(eng, prec, keep, length):
    run(eng, Case(11, prec, 3, length, 64, 16), keep=keep)


@pytest.mark.parametrize("prec", PRECS)
@pytest.mark.parametrize("channels,n", [(64, 16), (40, 5), (16, 64)])
@pytest.mark.parametrize("in_place", [False, True])
def test_ragged_lengths_and_states_in_place(eng, prec, channels, n, in_place):
    run(eng, Case(12, prec, 9, 300, channels, n), lengths=[0, 1, 8, 300, 99, -5, 1000, 64, 257], in_place=in_place)


@pytest.mark.parametrize("prec", PRECS)
def test_states_updated_in_place_over_many_segments(eng, prec):
    """A sequence's first segment starts from the states that its last replaces: the same bits as with states of their own."""
    k = Case(13, prec, 12, 2001, 128, 16)
    lengths = np.random.default_rng(14).integers(0, 2002, 12)
    want = run(eng, k, lengths=lengths, only=[0])
    for _ in range(3):
        got = run(eng, k, lengths=lengths, in_place=True, only=[])
        assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


@pytest.mark.parametrize("prec", PRECS)
@pytest.mark.parametrize("channels,n", [(300, 16), (515, 8), (70, 64), (257, 1)])
def test_states_in_place_with_workgroups_of_part_of_the_channels(eng, prec, channels, n):
    """The lanes of a channel's last workgroup that have no channel leave the first one, whose state has been replaced, alone:
    the same bits as with states of their own, in sequences whose workgroups do not all run at once."""
    k = Case(25, prec, 600, 33, channels, n)
    want = run(eng, k, only=[0, 599])
    for _ in range(2):
        got = run(eng, k, in_place=True, only=[])
        assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


@pytest.mark.parametrize("prec", PRECS)
def test_buffers_off_16_bytes(eng, prec):
    run(eng, Case(15, prec, 2, 45, 64, 16), offset=4 if prec == "f32" else 2)


def test_no_positions_pass_the_state_on(eng):
    run(eng, Case(16, "bf16", 3, 0, 24, 16))
    run(eng, Case(16, "f32", 3, 0, 24, 16), in_place=True)
    run(eng, Case(16, "f32", 3, 40, 24, 16), lengths=[0, 0, 0])
    run(eng, Case(16, "f32", 0, 40, 24, 16))


@pytest.mark.parametrize("prec", PRECS)
@pytest.mark.parametrize("length", [30, 300])
def test_packed_channels_and_gaps(eng, prec, length):
    """x and z as halves of packed channels, b and c of others, steps shared by all sequences, positions before sequences."""
    seqs, channels, n, groups = 2, 24, 16, 2
    k = Case(17, prec, seqs, length, channels, n, groups)
    k.delta[1] = k.delta[0]
    es, gn = (4 if prec == "f32" else 2), groups * n
    xz = np.concatenate([k.x, k.z], axis=2).transpose(1, 0, 2)  # [position][sequence][2 channels]
    bc = np.concatenate([k.b, k.c], axis=2)
    op = channels + 3
    fill = to_raw(np.full((seqs, length * op + 1), 7.0), prec)
    dxz, dbc, dd, do, da, dk, dbias = (DevBuf(v) for v in (xz, bc, k.delta[0], fill, k.a, k.d, k.bias))
    two = 2 * channels
    nn.selective_scan_noalloc(eng, nn.selective_scan_desc(
        prec, dxz, dd, dbc, dbc.address + gn * es, do, channels=channels, state_dim=n, sequences=seqs, length=length, a=da,
        z=dxz.address + channels * es, groups=groups, d=dk, delta_bias=dbias, x_position=seqs * two, z_position=seqs * two, x_sequence=two,
        z_sequence=two, delta_sequence=0, b_position=2 * gn, c_position=2 * gn, b_sequence=2 * gn * length,
        c_sequence=2 * gn * length, out_position=op, out_sequence=length * op + 1))
    eng.sync()
    got = do.get()
    for s in range(seqs):
        rows = got[s, :length * op].reshape(length, op)
        k.check(s, rows[:, :channels], length, rows[:, :channels], None, None)
        assert (rows[:, channels:] == fill[0, 0]).all() and (got[s, length * op:] == fill[0, 0]).all()


def step(eng, k, t, state_in, state_out, slots=None, num_slots=0, out=None):
    """The positions t of the case's sequences."""
    seqs, _, channels, n, groups = k.shape
    bufs = [DevBuf(np.ascontiguousarray(v[:, t:t + 1])) for v in (k.x, k.delta, k.z, k.b, k.c)]
    do = DevBuf(to_raw(np.full((seqs, 1, channels), 7.0), k.prec))
    da, dk, dbias = DevBuf(k.a), DevBuf(k.d), DevBuf(k.bias)
    nn.selective_scan_step(eng, nn.selective_scan_desc(
        k.prec, bufs[0], bufs[1], bufs[3], bufs[4], do, channels=channels, state_dim=n, sequences=seqs, length=1, a=da, z=bufs[2],
        groups=groups, d=dk, delta_bias=dbias, softplus=k.softplus, slots=slots, num_slots=num_slots, state_in=state_in,
        state_out=state_out))
    eng.sync()
    return do.get()


@pytest.mark.parametrize("prec", PRECS)
@pytest.mark.parametrize("channels,n,groups", [(64, 16, 1), (1, 1, 1), (70, 2, 1), (40, 3, 2), (33, 5, 1), (100, 16, 4), (66, 24, 2), (20, 64, 1),
                                               (9, 256, 3), (320, 12, 1), (17, 130, 1)])
@pytest.mark.parametrize("in_place", [False, True])
def test_steps_equal_whole_sequences(eng, prec, channels, n, groups, in_place):
    seqs, length = 3, 7
    k = Case(18, prec, seqs, length, channels, n, groups)
    cur, new = DevBuf(k.state), DevBuf(np.zeros_like(k.state))
    outs = []
    for t in range(length):
        outs.append(step(eng, k, t, cur, cur if in_place else new))
        if not in_place:
            cur, new = new, cur
    got = np.concatenate(outs, axis=1)
    for s in range(seqs):
        k.check(s, got[s], length, got[s], k.state[s], cur.get()[s])


@pytest.mark.parametrize("prec", PRECS)
@pytest.mark.parametrize("in_place", [False, True])
def test_slots_idle_and_repeated(eng, prec, in_place):
    slots = np.array([4, -1, 2, 7, 4, 100, 0, 4, 2], np.int32)
    seqs, num = len(slots), 7
    k = Case(19, prec, seqs, 1, 70, 16)
    state = np.random.default_rng(20).standard_normal((num, 70, 16)).astype(np.float32)
    di, dn = DevBuf(state), DevBuf(np.zeros_like(state))
    to = di if in_place else dn
    before = to.get()
    got, fin = step(eng, k, 0, di, to, DevBuf(slots), num), to.get()
    # The sequences of a slot as positions of one.
    for slot in range(-1, 101):
        at = np.flatnonzero(slots == slot)
        if not 0 <= slot < num:
            assert (from_raw(got[at], prec) == 7.0).all()
        elif not len(at):
            assert np.array_equal(fin[slot], before[slot])
        else:
            one = Case(19, prec, seqs, 1, 70, 16)
            for name in ("x", "delta", "z", "b", "c"):
                setattr(one, name, getattr(k, name)[at].transpose(1, 0, 2))
            one.check(0, got[at, 0], len(at), got[at, 0], state[slot], fin[slot])


@pytest.mark.parametrize("prec", PRECS)
@pytest.mark.parametrize("length", [40, 400])
def test_a_non_finite_input_reaches_only_later_outputs(eng, prec, length):
    seqs, channels, n, groups = 2, 32, 16, 2
    at = length // 2 + 3
    for name, ch, reach in (("x", 5, "channel"), ("delta", 6, "channel"), ("z", 7, "position"), ("b", 3, "group"), ("c", 17, "group position")):
        k = Case(21, prec, seqs, length, channels, n, groups)
        v = from_raw(getattr(k, name), prec).astype(np.float32)
        v[0, at, ch] = np.nan
        setattr(k, name, to_raw(v, prec))
        got, fin = run(eng, k, only=[1])
        bad, want = ~np.isfinite(from_raw(got, prec)), np.zeros(got.shape, bool)
        chans = slice(ch, ch + 1) if "group" not in reach else slice(0, 16) if ch < 16 else slice(16, 32)
        want[0, slice(at, at + 1) if "position" in reach else slice(at, None), chans] = True
        assert np.array_equal(bad, want), name
        assert np.isfinite(fin).all() == ("position" in reach), name


@pytest.mark.parametrize("prec", PRECS)
@pytest.mark.parametrize("length", [9, 200])
def test_extreme_steps(eng, prec, length):
    """Steps of the softplus far to both sides: none at all, and ones that forget everything; and decays of none."""
    k = Case(22, prec, 2, length, 16, 16)
    v = from_raw(k.delta, prec).astype(np.float32)
    v[:, 2::5], v[:, 3::5], v[:, 4::7], v[:, 5::7] = -200.0, 60.0, 15.0, -12.0
    v[1, 6] = -np.inf
    k.delta = to_raw(v, prec)
    k.a[3], k.a[4, ::2] = 0.0, -1e-8
    run(eng, k)


@pytest.mark.parametrize("prec", PRECS)
@pytest.mark.parametrize("rows", [False, True])
def test_a_map(prec, rows):
    e = nn.Engine(0, prec)
    c, n, g, h, w = 24, 8, 2, 6, 9
    k = Case(23, prec, 1, h * w, c, n, g)
    planar = [from_raw(v[0], prec).astype(np.float32).T.reshape(-1, h, w) for v in (k.x, k.delta, np.concatenate([k.b, k.c], axis=2), k.z)]

    def tensors(crop):
        for p in planar:
            big = np.full((p.shape[0], h + 1, w + 2), 50.0, np.float32)
            big[:, :h, :w] = p
            yield nn.BTensor.from_planar(e, big).crop(h, w) if crop else nn.BTensor.from_planar(e, p)

    for crop in (False, True):
        x, delta, bc, z = tensors(crop)
        got = nn.selective_scan(e, x, delta, bc, k.a, z, groups=g, d=k.d, delta_bias=k.bias, rows=rows).to_planar()
        got = to_raw(got, prec).reshape(c, h * w).T
        for s in range(h) if rows else [0]:
            what = slice(s * w, (s + 1) * w) if rows else slice(None)
            k.check(0, got[what], w if rows else h * w, got[what], None, None, what=what)
        del x, delta, bc, z
    e.close()


@pytest.mark.parametrize("prec", PRECS)
def test_offsets_past_32_bits(eng, prec):
    import ctypes
    from devbuf import hip
    far, es, c, n = 3 * 2 ** 30, 4 if prec == "f32" else 2, 8, 16
    k = Case(24, prec, 1, 2, c, n)
    base = ctypes.c_void_p()
    assert hip().hipMalloc(ctypes.byref(base), ctypes.c_size_t((far + 256) * es)) == 0
    try:
        places = {}
        for name, at in (("x", 0), ("delta", 32), ("z", 64), ("b", 96), ("c", 128)):
            places[name] = base.value + at * es
            for i in range(2):
                row = np.ascontiguousarray(getattr(k, name)[0, i])
                assert hip().hipMemcpy(places[name] + i * far * es, row.ctypes.data, row.nbytes, 1) == 0
        out, da, dk, db = DevBuf(np.zeros_like(k.x[0])), DevBuf(k.a), DevBuf(k.d), DevBuf(k.bias)
        far_apart = {m + end: far for m in places for end in ("_position", "_sequence")}
        for seqs, length in ((1, 2), (2, 1)):
            nn.selective_scan_noalloc(eng, nn.selective_scan_desc(
                prec, places["x"], places["delta"], places["b"], places["c"], out, channels=c, state_dim=n, sequences=seqs,
                length=length, a=da, z=places["z"], d=dk, delta_bias=db, out_position=c, out_sequence=c, **far_apart))
            eng.sync()
            for s in range(seqs):
                what = slice(0, 2) if seqs == 1 else slice(s, s + 1)
                k.check(0, out.get()[what], length, out.get()[what], None, None, what=what)
    finally:
        hip().hipFree(base)


def test_refusals(eng):
    x, o, b, w, s = (DevBuf(np.zeros(m, np.float32)) for m in (128, 128, 256, 1024, 2048))
    good = dict(channels=16, state_dim=16, sequences=2, length=4, a=w)

    def refused(kind="InvalidArgument", call=nn.selective_scan_noalloc, x=x, delta=x, b=b, c=b, out=o, prec="f32", **kw):
        desc = nn.selective_scan_desc(prec, x, delta, b, c, out, **{**good, **{k: v for k, v in kw.items() if k != "fields"}})
        for k, v in kw.get("fields", {}).items():
            setattr(desc, k, v)
        with pytest.raises(_lib.HipError) as e:
            call(eng, desc)
        assert e.value.kind == kind, e.value

    refused(channels=0)
    refused(kind="Unsupported", channels=2 ** 20 + 1)
    refused(groups=0)
    refused(groups=3)
    refused(state_dim=0)
    refused(kind="Unsupported", state_dim=257)
    refused(fields={"softplus": 2})
    refused(fields={"precision": 3})
    refused(fields={"num_slots": 1})
    refused(sequences=-1)
    refused(length=-1)
    refused(kind="LimitExceeded", length=2 ** 30 + 1)
    refused(kind="LimitExceeded", sequences=2 ** 22 + 1, length=1)
    refused(a=None)
    refused(a=w.address + 2)
    refused(d=w.address + 1)
    refused(delta_bias=w.address + 2)
    refused(lengths=w.address + 2)
    for name in ("x", "delta", "b", "c", "out"):
        refused(**{name: None})
        refused(**{name: o.address + 2})
    for name in ("x", "delta", "b", "c", "z"):
        refused(**{name: o})
        refused(**{name + "_position": -1}, **({"z": x} if name == "z" else {}))
        refused(**{name + "_sequence": -1}, **({"z": x} if name == "z" else {}))
    refused(z=x.address + 1)
    refused(out_position=15)
    refused(out_sequence=15)
    refused(out_position=16, out_sequence=16)
    refused(slots=w, num_slots=2)
    refused(state_in=s.address + 2)
    refused(state_in=s, state_out=s.address + 64)
    step = dict(call=nn.selective_scan_step, length=1)
    refused(**step)
    refused(**step, state_in=s)
    refused(**step, state_in=s, state_out=s, lengths=w)
    refused(call=nn.selective_scan_step, state_in=s, state_out=s)
    refused(**step, state_in=s, state_out=s, slots=w)
    refused(**step, state_in=s, state_out=s, slots=w, num_slots=-1)
    refused(**step, state_in=s, state_out=s, fields={"num_slots": 1})
    refused(**step, state_in=s, state_out=s, slots=w.address + 2, num_slots=2)
    refused(kind="LimitExceeded", **{**step, "sequences": 2 ** 26}, state_in=s, state_out=s)
    t, bc = (nn.BTensor.from_planar(eng, np.zeros((c, 2, 2), np.float32)) for c in (16, 64))
    small = nn.BTensor.from_planar(eng, np.zeros((16, 2, 1), np.float32))
    a = np.zeros((16, 16), np.float32)
    for args, kw in (((t, t, bc, a[:15]), {}), ((t, t, bc, a[:, :8]), {}), ((t, small, bc, a), {"groups": 2}), ((t, t, bc, a, small), {"groups": 2}),
                     ((t, t, bc, a), {"groups": 3}), ((t, t, bc, a), {"groups": 2, "d": np.zeros(3)})):
        with pytest.raises(_lib.HipError) as e:
            nn.selective_scan(eng, *args, **kw)
        assert e.value.kind == "InvalidArgument"
    nn.selective_scan_noalloc(eng, nn.selective_scan_desc("f32", x, x, b, b, o, **good))
    eng.sync()
