"""GPU: every form of the selective scan's kernels, each chosen by sizes and named by the profile so that a change of the rules
cannot leave one untested; and steps and convolution steps of more sequences than a workgroup has lanes, slots shared far apart."""

import numpy as np
import pytest

from devbuf import DevBuf, from_raw, to_raw
from state_space_oracle import conv
from test_gpu_selective_scan import PRECS, Case, eng, run, step  # noqa: F401  (eng: the fixture)
from zenjpegai_amd import nn

pytestmark = pytest.mark.gpu
TYPES = {"f32": "float", "f16": "_Float16", "bf16": "__bf16"}


def launched(e, call):
    e.profile_begin()
    try:
        call()
    finally:
        names = [r[0] for r in e.profile_end()]
    return names


class Wide(Case):
    """Many channels of which only a few are computed in 64 bits: the channels `seen` of each group's."""

    seen = slice(None)

    def check(self, s, got, n, fill, state, final, *parts):
        seqs, length, channels, m, g = self.shape
        part = Case.__new__(Case)
        at = np.arange(channels).reshape(g, -1)[:, self.seen].ravel()
        part.prec, part.softplus, part.shape = self.prec, self.softplus, (seqs, length, len(at), m, g)
        part.b, part.c = self.b, self.c
        part.x, part.delta, part.z = (v[..., at] for v in (self.x, self.delta, self.z))
        part.a, part.d, part.bias = self.a[at], self.d[at], self.bias[at]
        part.check(s, got[:, at], n, fill[:, at], None if state is None else state[at], None if final is None else final[at], *parts)


# (states a lane, lanes), states, channels, groups, sequences, positions: plans that keep a sequence whole, and that cut it.
WHOLE = [(1, 1, 1, 70, 1, 2, 40), (4, 1, 3, 100, 2, 2, 40), (4, 4, 10, 48, 2, 2, 40), (8, 1, 7, 129, 1, 2, 40), (12, 1, 9, 130, 1, 700, 40),
         (12, 1, 12, 64, 2, 600, 60), (12, 2, 20, 66, 2, 2, 40), (12, 4, 33, 30, 2, 2, 50), (12, 4, 48, 20, 1, 3, 40),
         (16, 1, 13, 70, 1, 700, 60), (16, 1, 16, 128, 2, 600, 60), (16, 2, 30, 50, 1, 2, 40), (16, 4, 50, 24, 2, 2, 40),
         (16, 8, 100, 21, 3, 2, 40), (16, 16, 129, 9, 1, 2, 40), (16, 16, 256, 10, 2, 1, 40)]
CUT = [(1, 1, 1, 70, 1, 2, 700), (4, 1, 4, 65, 1, 1, 700), (4, 4, 16, 40, 2, 1, 700), (8, 1, 8, 100, 1, 2, 700), (12, 1, 11, 128, 1, 8, 4100),
       (12, 2, 24, 33, 1, 2, 700), (12, 4, 40, 40, 2, 2, 700), (12, 4, 48, 17, 1, 1, 1500), (16, 1, 16, 128, 2, 8, 4100),
       (16, 1, 14, 1024, 1, 1, 4100), (16, 2, 32, 40, 2, 1, 700), (16, 4, 64, 24, 1, 2, 700), (16, 8, 128, 12, 2, 1, 700),
       (16, 16, 200, 9, 3, 1, 400), (16, 16, 256, 5, 1, 2, 300)]


@pytest.mark.parametrize("prec", PRECS)
@pytest.mark.parametrize("plan", WHOLE)
def test_whole_sequences_in_every_form(eng, prec, plan):  # noqa: F811
    ns, lanes, n, channels, groups, seqs, length = plan
    k = Wide(51, prec, seqs, length, channels, n, groups)
    only = [0, seqs // 2, seqs - 1]
    names = launched(eng, lambda: run(eng, k, only=only, in_place=True))
    assert names == [f"k_scan<{TYPES[prec]}, {ns}, {lanes}, true>"]


@pytest.mark.parametrize("prec", PRECS)
@pytest.mark.parametrize("plan", CUT)
def test_segments_in_every_form(eng, prec, plan):  # noqa: F811
    ns, lanes, n, channels, groups, seqs, length = plan
    k = Wide(52, prec, seqs, length, channels, n, groups, step=0.01)
    if length * channels > 4e5:
        k.seen = [0, 63, 64 % (channels // groups), channels // groups - 1]
    form = f"k_scan<{TYPES[prec]}, {ns}, {lanes}, "
    names = launched(eng, lambda: run(eng, k, only=[0, seqs - 1]))
    assert names == [form + "false>", "k_scan_starts", form + "true>"]


@pytest.mark.parametrize("prec", PRECS)
@pytest.mark.parametrize("plan", [p for p in CUT if p[0] >= 12])
def test_ragged_segments_in_every_form(eng, prec, plan):  # noqa: F811
    ns, lanes, n, channels, groups, seqs, length = plan
    seqs = max(seqs, 4)
    k = Wide(53, prec, seqs, length, channels, n, groups, step=0.01)
    if length * channels > 4e5:
        k.seen = [0, channels // groups - 1]
    lengths = np.resize([length - 1, 0, 1, length // 2 + 3], seqs)
    names = launched(eng, lambda: run(eng, k, lengths=lengths, only=range(4), in_place=True))
    assert names[0].startswith(f"k_scan<{TYPES[prec]}, {ns}, {lanes}, ") and len(names) == 3


@pytest.mark.parametrize("channels", [3, 64, 65, 128, 130, 190, 200, 256, 257, 320, 385, 449])
@pytest.mark.parametrize("n,lanes", [(1, 1), (4, 1), (8, 1), (12, 4)])
def test_workgroups_of_one_to_four_waves(eng, n, lanes, channels):  # noqa: F811
    for length in (30, 200):
        k = Wide(54, "f16", 2, length, channels, n)
        names = launched(eng, lambda: run(eng, k))  # noqa: B023
        assert names[-1].startswith(f"k_scan<_Float16, {n if n < 12 else 4}, {lanes}, ")


def spread_slots(seqs, num):
    """Slots of which some are shared, next to one another and more than 256 and 512 sequences apart, and some are none."""
    rng = np.random.default_rng(55)
    slots = np.resize(rng.permutation(num), seqs).astype(np.int32)
    slots[[0, 300, 301, 515, seqs - 1]] = 5
    slots[[1, 258, 514]] = 6
    slots[[2, 255, 256, 257, 511, 512, 513]] = 7
    slots[10::37] = -1
    slots[11::53] = num + 3
    slots[400] = num - 1
    return slots


@pytest.mark.parametrize("prec", PRECS)
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("seqs,num,channels,n", [(700, 400, 70, 16), (1300, 1000, 9, 5), (520, 300, 6, 64)])
def test_steps_of_slots_shared_far_apart(eng, prec, in_place, seqs, num, channels, n):  # noqa: F811
    slots = spread_slots(seqs, num)
    k = Case(56, prec, seqs, 1, channels, n)
    state = np.random.default_rng(57).standard_normal((num, channels, n)).astype(np.float32)
    di, dn = DevBuf(state), DevBuf(np.full_like(state, 4.0))
    to = di if in_place else dn
    got, fin = step(eng, k, 0, di, to, DevBuf(slots), num), to.get()
    live = (slots >= 0) & (slots < num)
    assert (from_raw(got[~live], prec) == 7.0).all()
    for slot in range(num):
        at = np.flatnonzero(slots == slot)
        if not len(at):
            assert np.array_equal(fin[slot], state[slot] if in_place else np.full_like(fin[slot], 4.0))
            continue
        one = Case.__new__(Case)
        one.__dict__.update(vars(k))
        for name in ("x", "delta", "z", "b", "c"):
            setattr(one, name, getattr(k, name)[at].transpose(1, 0, 2))
        one.check(0, got[at, 0], len(at), got[at, 0], state[slot], fin[slot])


@pytest.mark.parametrize("prec", PRECS)
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("seqs,num,channels", [(700, 400, 70), (1300, 1000, 512), (520, 300, 1)])
def test_convolution_steps_of_slots_shared_far_apart(eng, prec, in_place, seqs, num, channels):  # noqa: F811
    taps, slots, rng = 4, spread_slots(seqs, num), np.random.default_rng(58)
    x, state = to_raw(rng.standard_normal((seqs, 1, channels)), prec), to_raw(rng.standard_normal((num, taps - 1, channels)), prec)
    w, b = rng.standard_normal((channels, taps)).astype(np.float32), rng.standard_normal(channels).astype(np.float32)
    fill, rest = to_raw(np.full(x.shape, 7.0), prec), to_raw(np.full(state.shape, 4.0), prec)
    dx, do, dw, db, di, dn, sl = (DevBuf(v) for v in (x, fill, w, b, state, rest, slots))
    to = di if in_place else dn
    nn.causal_conv_step(eng, nn.causal_conv_desc(prec, dx, do, channels=channels, taps=taps, sequences=seqs, length=1, weight=dw, bias=db,
                                                 act="silu", slots=sl, num_slots=num, state_in=di, state_out=to))
    eng.sync()
    got, fin = do.get(), to.get()
    live = (slots >= 0) & (slots < num)
    assert np.array_equal(got[~live], fill[~live])
    for slot in range(num):
        at = np.flatnonzero(slots == slot)
        if not len(at):
            assert np.array_equal(fin[slot], (state if in_place else rest)[slot])
            continue
        y, tol, last = conv(prec, from_raw(x[at, 0], prec), w, b, "silu", len(at), from_raw(state[slot], prec))
        assert (np.abs(from_raw(got[at, 0], prec) - y) <= tol).all(), slot
        assert np.array_equal(from_raw(fin[slot], prec), last)


def test_a_convolution_of_more_items_than_32_bits_count(eng):  # noqa: F811
    """2^20 channels one by one (x off 4 bytes), 2 x 1100 runs: 2^31 and more items, of which the lengths leave a few."""
    channels, taps, length, lengths = 2 ** 20, 3, 17600, [18, 3]
    rng = np.random.default_rng(59)
    x = to_raw(rng.standard_normal((2, 20, channels)), "f16")
    w, b = rng.standard_normal((channels, taps)).astype(np.float32), rng.standard_normal(channels).astype(np.float32)
    fill = to_raw(np.full((20, 2, channels), 7.0), "f16")
    dx, do, dw, db, dl = DevBuf(x, 2), DevBuf(fill), DevBuf(w), DevBuf(b), DevBuf(np.array(lengths, np.int32))
    nn.causal_conv_noalloc(eng, nn.causal_conv_desc("f16", dx, do, channels=channels, taps=taps, sequences=2, length=length, weight=dw, bias=db,
                                                    lengths=dl, x_position=channels, x_sequence=20 * channels, out_position=2 * channels,
                                                    out_sequence=channels))
    eng.sync()
    got = do.get()
    at = np.concatenate([np.arange(1000), np.arange(channels - 1000, channels), rng.integers(0, channels, 2000)])
    for s, n in enumerate(lengths):
        y, tol, _ = conv("f16", from_raw(x[s, :n, at].T, "f16"), w[at], b[at], "linear", n)
        assert (np.abs(from_raw(got[:n, s, at], "f16") - y) <= tol).all()
        assert np.array_equal(got[n:, s], fill[n:, s])
