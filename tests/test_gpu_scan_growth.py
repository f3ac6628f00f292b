"""GPU: selective scans whose states grow (a above zero, or negative steps without the softplus): what the recurrence keeps in
f32's range stays in it however the sequence is cut, and a state of zero stays zero."""

import numpy as np
import pytest

from devbuf import DevBuf, to_raw
from test_gpu_selective_scan import PRECS, Case, eng, run  # noqa: F401  (eng: the fixture)
from zenjpegai_amd import nn

pytestmark = pytest.mark.gpu


def growing(prec, length, seqs=1, channels=16, n=16, sign=1):
    """Steps of 1 (or -1), states that grow by e^3 to e^4 a position: 32 positions by 2^138 at least. No inputs but at the end."""
    k = Case(31, prec, seqs, length, channels, n, softplus=False)
    k.a = (sign * (3.0 + np.arange(n) / n) * np.ones((channels, n))).astype(np.float32)
    k.delta = to_raw(np.full(k.delta.shape, float(sign)), prec)
    k.x[:, :-2] = 0
    k.state[:] = 0.0
    return k


@pytest.mark.parametrize("prec", PRECS)
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("length", [20, 64, 700, 6000])
@pytest.mark.parametrize("keep", [(False, True), (True, True)])
def test_a_state_of_zero_stays_zero(eng, prec, sign, length, keep):  # noqa: F811
    run(eng, growing(prec, length, sign=sign), keep=keep)


@pytest.mark.parametrize("prec", PRECS)
def test_ragged_sequences_and_more_states(eng, prec):  # noqa: F811
    lengths = [700, 0, 1, 65, 333, 699]
    for n in (1, 24, 40, 64):
        k = growing(prec, 700, seqs=len(lengths), n=n)
        for s, m in enumerate(lengths):
            k.x[s] = 0
            k.x[s, max(m - 2, 0):m] = to_raw(np.ones((min(m, 2), 16)), prec)
        run(eng, k, lengths=lengths)


@pytest.mark.parametrize("prec", PRECS)
def test_steps_of_the_softplus(eng, prec):  # noqa: F811
    k = growing(prec, 700)
    k.softplus = True  # ln(1 + e) = 1.3
    run(eng, k, bias=False)


@pytest.mark.parametrize("first,last", [(64, 64), (700, 64), (2000, 700)])
def test_growth_and_decay_past_the_range_of_one_factor(eng, first, last):  # noqa: F811
    """States of 2^-120 grow by 2^200 over the first 32 positions and go back by 2^-200 over others: each factor of a stretch is past
    what f32 holds, no state is."""
    for back in (32, first - 32):
        length = first + last
        k = Case(32, "f32", 1, length, 16, 16, softplus=False)
        k.a = np.ones((16, 16), np.float32)
        k.delta[:] = 0.0
        k.delta[0, :32] = 200 * np.log(2.0) / 32
        k.delta[0, first - back:first] -= np.float32(200 * np.log(2.0) / back)
        k.delta[0, first:] = 1e-3
        k.x[0, :first] = 0.0
        k.state = (k.state * 2.0 ** -120).astype(np.float32)
        run(eng, k)


@pytest.mark.parametrize("prec", PRECS)
def test_position_by_position_the_same(eng, prec):  # noqa: F811
    """The step form of such a sequence and the whole one give the same states but for rounding."""
    length, channels, n = 96, 16, 16
    k = growing(prec, length)
    k.x[:, -2:], k.b = to_raw(np.ones((1, 2, channels)), prec), to_raw(np.full(k.b.shape, 0.75), prec)  # sums of one sign
    whole, cur = run(eng, k, keep=(False, True))[1], DevBuf(np.zeros((1, channels, n), np.float32))
    da, dk, db = DevBuf(k.a), DevBuf(k.d), DevBuf(k.bias)
    for t in range(length):
        one = [DevBuf(np.ascontiguousarray(v[:, t:t + 1])) for v in (k.x, k.delta, k.z, k.b, k.c, k.x)]
        nn.selective_scan_step(eng, nn.selective_scan_desc(
            prec, one[0], one[1], one[3], one[4], one[5], channels=channels, state_dim=n, sequences=1, length=1, a=da, z=one[2],
            d=dk, delta_bias=db, softplus=False, state_in=cur, state_out=cur))
        eng.sync()
    # Three factors and sums of up to three roundings, exponents of 3 to 4 with two of their own.
    assert np.allclose(cur.get(), whole, rtol=2.0 ** -24 * 40, atol=0)
