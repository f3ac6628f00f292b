"""GPU: rotary positions against sines and cosines in 64 bits: both layouts, part of a head, odd sizes, far and given
positions, rows and columns of a map, strides, in place, ragged lengths, and the calls that are refused."""

import numpy as np
import pytest

from devbuf import DevBuf, from_raw, to_raw
from state_space_oracle import rotary
from zenjpegai_amd import _lib, nn

pytestmark = pytest.mark.gpu
PRECS = ["f32", "f16", "bf16"]


@pytest.fixture(scope="module")
def eng():
    e = nn.Engine(0)
    yield e
    e.close()


def values(seed, prec, *shape):
    return to_raw(np.random.default_rng(seed).standard_normal(shape), prec)


def check(prec, got, x, places, freq, layout, magnitude=1.0, inverse=False):
    want, tol = rotary(prec, from_raw(x, prec), places, freq, layout, magnitude, inverse)
    err = np.abs(from_raw(got, prec) - want)
    assert (err <= tol).all(), (float((err - tol).max()), np.unravel_index(np.argmax(err - tol), err.shape))


def run(eng, prec, x, out, **kw):
    """x, out: [sequences][length][heads][dim] arrays."""
    n, t, h, d = x.shape
    dx, do = DevBuf(x, kw.pop("offset", 0)), DevBuf(out)
    bufs = {k: DevBuf(np.asarray(kw[k], np.int32)) for k in ("positions", "starts", "lengths") if kw.get(k) is not None}
    f = DevBuf(np.asarray(kw.pop("freq"), np.float64))
    in_place = kw.pop("in_place", False)
    desc = nn.rotary_desc(prec, dx, dx if in_place else do, heads=h, head_dim=d, rotary_dim=2 * f.shape[0], sequences=n, length=t,
                          frequencies=f, **{**kw, **bufs})
    nn.rotary_noalloc(eng, desc)
    eng.sync()
    return (dx if in_place else do).get()


@pytest.mark.parametrize("prec", PRECS)
@pytest.mark.parametrize("layout", ["interleaved", "halves"])
@pytest.mark.parametrize("heads,dim,turned", [(1, 2, 2), (3, 32, 32), (2, 20, 12), (5, 128, 64), (1, 1024, 1024), (7, 6, 2), (2, 9, 4)])
@pytest.mark.parametrize("length", [1, 37])
def test_equals_sines_and_cosines(eng, prec, layout, heads, dim, turned, length):
    x = values(1, prec, 2, length, heads, dim)
    freq = nn.rotary_frequencies(turned)[0]
    got = run(eng, prec, x, np.zeros_like(x), freq=freq, layout=layout)
    for s in range(2):
        check(prec, got[s], x[s], np.arange(length), freq, layout)
    assert np.array_equal(got[..., turned:], x[..., turned:])


@pytest.mark.parametrize("prec", PRECS)
@pytest.mark.parametrize("layout", ["interleaved", "halves"])
def test_far_positions_and_every_eighth_of_a_turn(eng, prec, layout):
    """Positions up to 2^31, before the first, and angles around all multiples of an eighth of a turn."""
    places = np.array([0, 1, 1000000, 2 ** 31 - 1, -1, -2 ** 31, 123456789, 65535], np.int32)
    freq = nn.rotary_frequencies(64, scaling="yarn", factor=16.0, trained_length=4096.0)[0]
    x = values(2, prec, 1, len(places), 3, 64)
    got = run(eng, prec, x, np.zeros_like(x), freq=freq, layout=layout, positions=places, magnitude=1.25)
    check(prec, got[0], x[0], places, freq, layout, 1.25)
    eighths = np.arange(-9, 10) * (np.pi / 4)
    freq = np.concatenate([eighths, eighths + 1e-6, eighths - 1e-6, eighths * (1 + 2 ** -30)])
    x = values(3, prec, 1, 2, 2, 2 * freq.size)
    check(prec, run(eng, prec, x, np.zeros_like(x), freq=freq, layout=layout)[0], x[0], [0, 1], freq, layout)


@pytest.mark.parametrize("prec", PRECS)
def test_starts_add_to_positions_modulo_2_32(eng, prec):
    n, t = 3, 5
    freq = nn.rotary_frequencies(16)[0]
    x = values(4, prec, n, t, 2, 16)
    places = np.random.default_rng(5).integers(-100, 100, (n, t))
    for positions in (None, places):
        for starts in ([7, 2 ** 31 - 3, -50], [0, 1, 99999]):
            got = run(eng, prec, x, np.zeros_like(x), freq=freq, starts=starts, positions=positions)
            at = (np.arange(t) + np.zeros((n, 1)) if positions is None else places) + np.array(starts)[:, None]
            at = (at.astype(np.int64) + 2 ** 31) % 2 ** 32 - 2 ** 31
            for s in range(n):
                check(prec, got[s], x[s], at[s], freq, "interleaved")


@pytest.mark.parametrize("prec", PRECS)
@pytest.mark.parametrize("layout", ["interleaved", "halves"])
@pytest.mark.parametrize("width", [1, 7, 300])
def test_half_of_the_pairs_by_row_and_half_by_column(eng, prec, layout, width):
    t, freq = 40, np.tile(nn.rotary_frequencies(16)[0], 2)
    x = values(6, prec, 2, t, 2, 40)
    starts = np.array([0, -20], np.int32)
    got = run(eng, prec, x, np.zeros_like(x), freq=freq, layout=layout, width=width, starts=starts)
    for s in range(2):
        at = np.arange(t) + starts[s]
        places = np.concatenate([np.repeat((at // width)[:, None], 8, 1), np.repeat((at % width)[:, None], 8, 1)], axis=1)
        check(prec, got[s], x[s], places, freq, layout)


@pytest.mark.parametrize("prec", PRECS)
@pytest.mark.parametrize("layout", ["interleaved", "halves"])
@pytest.mark.parametrize("turned", [24, 64])
def test_in_place_in_packed_channels_and_back(eng, prec, layout, turned):
    """Queries and keys of packed channels in place: the rest stays; the same call the other way round undoes it to rounding."""
    n, t, h, d = 2, 19, 4, 64
    packed = values(7, prec, n, t, 3 * h * d // 2 + 8)
    freq = DevBuf(nn.rotary_frequencies(turned)[0])
    buf, p = DevBuf(packed), packed.shape[2]
    kw = dict(heads=h, head_dim=d, rotary_dim=turned, layout=layout, sequences=n, length=t, frequencies=freq,
              x_position=p, out_position=p, x_sequence=p * t, out_sequence=p * t)
    nn.rotary_noalloc(eng, nn.rotary_desc(prec, buf, buf, **kw))
    eng.sync()
    got = buf.get()
    x = packed[..., :h * d].reshape(n, t, h, d)
    y = got[..., :h * d].reshape(n, t, h, d)
    for s in range(n):
        check(prec, y[s], x[s], np.arange(t), freq.get(), layout)
        check_back, _ = rotary(prec, from_raw(y[s], prec), np.arange(t), freq.get(), layout, 1.0, inverse=True)
    assert np.array_equal(got[..., h * d:], packed[..., h * d:]) and np.array_equal(y[..., turned:], x[..., turned:])
    nn.rotary_noalloc(eng, nn.rotary_desc(prec, buf, buf, inverse=True, **kw))
    eng.sync()
    back = buf.get()[..., :h * d].reshape(n, t, h, d)
    for s in range(n):
        check(prec, back[s], y[s], np.arange(t), freq.get(), layout, inverse=True)
    assert np.abs(check_back - from_raw(x[n - 1], prec)).max() < 0.1


@pytest.mark.parametrize("prec", PRECS)
@pytest.mark.parametrize("layout", ["interleaved", "halves"])
def test_strides_and_buffers_off_16_bytes(eng, prec, layout):
    n, t, h, d = 2, 11, 3, 16
    es = 4 if prec == "f32" else 2
    freq = nn.rotary_frequencies(8)[0]
    for xp, op, offset in ((h * d + 1, h * d + 3, 0), (h * d + 8, h * d, es), (h * d + 2, h * d + 4, 0), (h * d, h * d, 8)):
        full = values(8, prec, n, t * xp + 5)
        x = np.stack([full[s, :t * xp].reshape(t, xp)[:, :h * d] for s in range(n)]).reshape(n, t, h, d)
        fill = to_raw(np.full((n, t * op + 7), 3.0), prec)
        bx, bo, f = DevBuf(full, offset), DevBuf(fill, offset), DevBuf(freq)
        nn.rotary_noalloc(eng, nn.rotary_desc(prec, bx, bo, heads=h, head_dim=d, rotary_dim=8, layout=layout, sequences=n, length=t,
                                              frequencies=f, x_position=xp, x_sequence=t * xp + 5, out_position=op,
                                              out_sequence=t * op + 7))
        eng.sync()
        got = bo.get()
        for s in range(n):
            rows = got[s, :t * op].reshape(t, op)
            check(prec, rows[:, :h * d].reshape(t, h, d), x[s], np.arange(t), freq, layout)
            assert (rows[:, h * d:] == fill[0, 0]).all() and (got[s, t * op:] == fill[0, 0]).all()


@pytest.mark.parametrize("prec", PRECS)
def test_positions_first_and_sequences_between_them(eng, prec):
    """[position][sequence][channels], and one input row for all sequences (a stride of none)."""
    n, t, h, d = 3, 9, 2, 16
    freq = nn.rotary_frequencies(16)[0]
    x = values(9, prec, t, n, h, d)
    bx, bo, f = DevBuf(x), DevBuf(np.zeros_like(x)), DevBuf(freq)
    kw = dict(heads=h, head_dim=d, sequences=n, length=t, frequencies=f, out_position=n * h * d, out_sequence=h * d)
    nn.rotary_noalloc(eng, nn.rotary_desc(prec, bx, bo, x_position=n * h * d, x_sequence=h * d, **kw))
    eng.sync()
    got = bo.get()
    for s in range(n):
        check(prec, got[:, s], x[:, s], np.arange(t), freq, "interleaved")
    nn.rotary_noalloc(eng, nn.rotary_desc(prec, bx, bo, x_position=0, x_sequence=0, **kw))
    eng.sync()
    got = bo.get()
    for s in range(n):
        check(prec, got[:, s], np.broadcast_to(x[0, 0], (t, h, d)), np.arange(t), freq, "interleaved")


@pytest.mark.parametrize("prec", PRECS)
@pytest.mark.parametrize("heads,dim", [(2, 32), (32, 128)])
def test_ragged_lengths_leave_the_rest_as_it_was(eng, prec, heads, dim):
    t, lengths = 41, [0, 1, 41, 20, -3, 1000]
    x = values(10, prec, len(lengths), t, heads, dim)
    fill = to_raw(np.full(x.shape, 5.0), prec)
    freq = nn.rotary_frequencies(dim)[0]
    got = run(eng, prec, x, fill, freq=freq, lengths=lengths, layout="halves")
    for s, n in enumerate(min(max(v, 0), t) for v in lengths):
        check(prec, got[s, :n], x[s, :n], np.arange(n), freq, "halves")
        assert np.array_equal(got[s, n:], fill[s, n:])


def test_long_sequences_and_none(eng):
    x = values(11, "bf16", 1, 70001, 1, 8)
    freq = nn.rotary_frequencies(8)[0]
    check("bf16", run(eng, "bf16", x, np.zeros_like(x), freq=freq)[0], x[0], np.arange(70001), freq, "interleaved")
    for shape in ((0, 5, 1, 8), (3, 0, 1, 8)):
        x = values(12, "bf16", *shape)
        run(eng, "bf16", x, x, freq=freq)


@pytest.mark.parametrize("prec", PRECS)
def test_offsets_past_32_bits(eng, prec):
    """The second of two positions lies 2^32 elements behind the first (two sequences, too): only what is read is there."""
    h, d = 2, 16
    far = 3 * 2 ** 30  # elements: past 2^32 bytes in every type, and past 2^31 elements
    es = 4 if prec == "f32" else 2
    import ctypes
    from devbuf import hip
    base = ctypes.c_void_p()
    assert hip().hipMalloc(ctypes.byref(base), ctypes.c_size_t((far + 64) * es)) == 0
    try:
        x = values(13, prec, 2, h, d)
        for i in range(2):
            assert hip().hipMemcpy(base.value + i * far * es, x[i].ctypes.data, x[i].nbytes, 1) == 0
        out, f = DevBuf(np.zeros_like(x)), DevBuf(nn.rotary_frequencies(d)[0])
        for kw, places in (({"sequences": 1, "length": 2}, [0, 1]), ({"sequences": 2, "length": 1}, [0, 0])):
            nn.rotary_noalloc(eng, nn.rotary_desc(prec, base.value, out, heads=h, head_dim=d, frequencies=f, x_position=far,
                                                  x_sequence=far, out_position=h * d, out_sequence=h * d, **kw))
            eng.sync()
            check(prec, out.get(), x, places, f.get(), "interleaved")
    finally:
        hip().hipFree(base)


@pytest.mark.parametrize("prec", PRECS)
def test_non_finite_values_stay_in_their_pair(eng, prec):
    x = np.random.default_rng(14).standard_normal((1, 6, 2, 16)).astype(np.float32)
    x[0, 2, 1, 3], x[0, 4, 0, 0] = np.inf, np.nan
    raw = to_raw(x, prec)
    freq = nn.rotary_frequencies(16)[0]
    got = from_raw(run(eng, prec, raw, np.zeros_like(raw), freq=freq), prec)
    bad = ~np.isfinite(got)
    want = np.zeros_like(bad)
    want[0, 2, 1, 2:4] = want[0, 4, 0, 0:2] = True
    assert np.array_equal(bad, want)


@pytest.mark.parametrize("prec", PRECS)
@pytest.mark.parametrize("layout", ["interleaved", "halves"])
@pytest.mark.parametrize("by", ["raster", "column", "both"])
def test_a_map(eng, prec, layout, by):
    """The tensor form, over a whole map and over a corner of a larger one."""
    e = nn.Engine(0, prec)
    heads, dim, h, w = 4, 16, 5, 7
    x = np.random.default_rng(15).standard_normal((heads * dim + 12, h, w)).astype(np.float32)
    freq = nn.rotary_frequencies(8)[0]
    for crop in (False, True):
        big = np.zeros((x.shape[0], h + 2, w + 3), np.float32)
        big[:, :h, :w] = x
        t = nn.BTensor.from_planar(e, big).crop(h, w) if crop else nn.BTensor.from_planar(e, x)
        before = to_raw(t.to_planar(), prec)
        nn.rotary(e, t, heads, dim, freq, layout=layout, by=by, magnitude=0.5)
        got = to_raw(t.to_planar(), prec)
        y, xx = np.mgrid[:h, :w].reshape(2, -1)
        places = {"raster": np.arange(h * w), "column": xx,
                  "both": np.stack([y, y, xx, xx], axis=1)}[by]
        flat = [np.ascontiguousarray(v[:heads * dim].reshape(heads, dim, -1).transpose(2, 0, 1)) for v in (got, before)]
        check(prec, flat[0], flat[1], places, freq, layout, 0.5)
        assert np.array_equal(got[heads * dim:], before[heads * dim:])
        del t
    e.close()


def test_refusals(eng):
    x, f = DevBuf(np.zeros((2, 4, 64), np.float32)), DevBuf(np.zeros(8))
    out = DevBuf(np.zeros((2, 4, 64), np.float32))
    good = dict(heads=4, head_dim=16, sequences=2, length=4, frequencies=f)

    def refused(kind="InvalidArgument", a=x, o=out, prec="f32", **kw):
        desc = nn.rotary_desc(prec, a, o, **{**good, **kw})
        with pytest.raises(_lib.HipError) as e:
            nn.rotary_noalloc(eng, desc)
        assert e.value.kind == kind, e.value

    refused(heads=0)
    refused(head_dim=0)
    refused(kind="Unsupported", head_dim=1026, rotary_dim=2)
    refused(kind="LimitExceeded", heads=2 ** 21, head_dim=1024, rotary_dim=2)
    refused(rotary_dim=3)
    refused(rotary_dim=0)
    refused(rotary_dim=18)
    refused(rotary_dim=6, width=4)
    refused(width=-1)
    refused(sequences=-1)
    refused(length=-1)
    refused(kind="LimitExceeded", length=2 ** 30 + 1)
    refused(magnitude=float("nan"))
    refused(frequencies=None)
    refused(frequencies=f.address + 4)
    refused(a=None)
    refused(o=None)
    refused(a=x.address + 2)
    refused(starts=x.address + 1)
    refused(lengths=x.address + 2)
    refused(positions=x.address + 2)
    refused(x_position=-1)
    refused(out_position=63)
    refused(out_sequence=63)
    refused(out_sequence=64, out_position=64)
    refused(a=x, o=x, x_position=128)
    refused(a=x, o=x, x_sequence=512)
    for field, value in (("layout", 2), ("layout", -1), ("inverse", 2), ("precision", 3), ("precision", -1)):
        desc = nn.rotary_desc("f32", x, out, **good)
        setattr(desc, field, value)
        with pytest.raises(_lib.HipError) as e:
            nn.rotary_noalloc(eng, desc)
        assert e.value.kind == "InvalidArgument"
    t = nn.BTensor.from_planar(eng, np.zeros((32, 2, 2), np.float32))
    for heads, dim, freq, kw in ((3, 16, np.ones(8), {}), (2, 16, np.ones(9), {}), (2, 16, np.ones(3), {"by": "both"}),
                                 (2, 16, np.ones(0), {})):
        with pytest.raises(_lib.HipError) as e:
            nn.rotary(eng, t, heads, dim, freq, **kw)
        assert e.value.kind == "InvalidArgument"
    nn.rotary_noalloc(eng, nn.rotary_desc("f32", x, out, **good))
    eng.sync()
