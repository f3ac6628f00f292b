"""GPU: rotary positions over more tiles than there are workgroups, and counts of accesses that do not fill one."""

import numpy as np
import pytest

from test_gpu_rotary import PRECS, check, eng, run, values  # noqa: F401  (eng: the fixture)
from zenjpegai_amd import nn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("prec", PRECS)
@pytest.mark.parametrize("seqs,length,in_place", [(70001, 1, False), (140003, 1, True), (33000, 5, False)])
def test_more_tiles_than_workgroups(eng, prec, seqs, length, in_place):  # noqa: F811
    x, starts = values(61, prec, seqs, length, 1, 4), np.random.default_rng(62).integers(0, 100000, seqs)
    freq = nn.rotary_frequencies(4)[0]
    lengths = np.where(np.arange(seqs) % 7 == 3, 0, length)
    fill = np.zeros_like(x)
    got = run(eng, prec, x, fill, freq=freq, starts=starts, lengths=lengths, in_place=in_place)
    on = np.flatnonzero(lengths)
    places = (starts[on, None] + np.arange(length)).ravel()
    check(prec, got[on].reshape(-1, 1, 4), x[on].reshape(-1, 1, 4), places, freq, "interleaved")
    off = np.flatnonzero(lengths == 0)
    assert np.array_equal(got[off], (x if in_place else fill)[off])


@pytest.mark.parametrize("prec", PRECS)
@pytest.mark.parametrize("layout", ["interleaved", "halves"])
@pytest.mark.parametrize("heads,dim,turned", [(13, 80, 80), (13, 40, 40), (129, 8, 8), (257, 8, 4), (65, 16, 16), (43, 12, 6), (5, 1024, 512), (300, 2, 2)])
def test_accesses_that_leave_lanes_idle(eng, prec, layout, heads, dim, turned):  # noqa: F811
    freq = nn.rotary_frequencies(turned)[0]
    for length in (1, 40, 3000 if heads * dim < 2000 else 300):
        x = values(63, prec, 1, length, heads, dim)
        check(prec, run(eng, prec, x, np.zeros_like(x), freq=freq, layout=layout)[0], x[0], np.arange(length), freq, layout)
