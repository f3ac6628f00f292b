"""GPU: states of decayed linear attention: updated in place over many segments, what they keep of small and
single terms, and how fast they forget."""

import numpy as np
import pytest

from devbuf import DevBuf, from_raw, to_raw
from linear_attention_oracle import U, oracle
from test_gpu_linear_attention import check_sequence, eng, inputs  # noqa: F401 (eng: the fixture)
from zenjpegai_amd import _lib, nn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("prec,seqs,length,heads,dk,dv", [
    ("f16", 24, 3001, 2, 32, 32),   # 2256 workgroups of outputs, of which the card holds 1536 at a time
    ("bf16", 12, 3001, 8, 64, 64),  # 1824, of which it holds 768
    ("f32", 12, 3001, 8, 64, 40),
    ("bf16", 3, 9001, 1, 128, 128),  # 57 segments a sequence: a scan in four parts
    ("f16", 3, 9001, 1, 100, 96)])
def test_states_updated_in_place_over_many_segments(eng, prec, seqs, length, heads, dk, dv):  # noqa: F811
    """A sequence's first segment starts from the states that its last segment replaces: the same bits as with
    states of their own, whichever of the two runs first, and the recurrence in 64 bits for the
    first sequences."""
    qkv, out, decay, state = inputs(80, prec, seqs, length, heads, dk, dv)
    lengths = np.random.default_rng(81).integers(0, length + 1, seqs).astype(np.int32)
    lengths[:3] = [length, 0, length - 1]
    if seqs > 4:
        lengths[4:8] = [1, 0, 33, 0]
    b = [DevBuf(a) for a in (qkv, out, decay, state, lengths)]
    fin = DevBuf(np.zeros_like(state))

    def call(state_in, state_out):
        b[1].put(out)
        nn.linear_attention_noalloc(eng, nn.linear_attention_desc(
            prec, b[0], b[1], heads=heads, key_dim=dk, value_dim=dv, sequences=seqs, length=length, decay=b[2], scale=0.5,
            lengths=b[4], state_in=state_in, state_out=state_out))
        eng.sync()
        return b[1].get(), state_out.get()

    want = call(b[3], fin)
    for s in range(3):
        check_sequence(prec, heads, dk, dv, qkv[s], decay, 0.5, int(lengths[s]), state[s], want[0][s], out[s], want[1][s])
    for _ in range(4):
        b[3].put(state)
        got = call(b[3], b[3])
        assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


def packed(prec, q, k, v):
    """[t][h][d] arrays as one sequence of packed channels in the storage type."""
    t = q.shape[0]
    return to_raw(np.concatenate([a.reshape(t, -1) for a in (q, k, v)], axis=1), prec)[None]


@pytest.mark.parametrize("prec", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dk,dv", [(32, 32), (64, 40), (128, 128)])
@pytest.mark.parametrize("length,every", [(32, 32), (70, 32), (330, 16)])
@pytest.mark.parametrize("size", [1.0, 1e-4, 1e-6])
def test_a_value_followed_by_zeros_stays_in_the_state(eng, prec, dk, dv, length, every, size):  # noqa: F811
    """Values at every 32nd or 16th position, zeros between: what is left of them has decayed by up to 2^-62 (2^-82 at a
    decay of 0.4 and 63 positions), and nothing newer covers what is lost of it. The scale brings the
    outputs right after a value back to about one."""
    heads = 4
    rng = np.random.default_rng(82)
    q, k = (rng.standard_normal((length, heads, dk)) for _ in range(2))
    v = np.zeros((length, heads, dv))
    v[::every] = size * rng.uniform(1.0, 2.0, v[::every].shape)
    decay = np.array([0.5, 0.25, 0.4, 0.97], np.float32)
    scale = float(np.float32(0.1 / size))
    qkv = packed(prec, q, k, v)
    out = to_raw(np.zeros((1, length, heads * dv)), prec)
    b = [DevBuf(a) for a in (qkv, out, decay, np.zeros((1, heads, dk, dv), np.float32))]
    nn.linear_attention_noalloc(eng, nn.linear_attention_desc(prec, b[0], b[1], heads=heads, key_dim=dk, value_dim=dv, sequences=1,
                                                              length=length, decay=b[2], scale=scale, state_out=b[3]))
    eng.sync()
    check_sequence(prec, heads, dk, dv, qkv[0], decay, scale, length, None, b[1].get()[0], out[0], b[3].get()[0])


@pytest.mark.parametrize("prec", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("size", [1.0, 1e-4, 1e-6])
def test_positions_with_key_channels_of_their_own(eng, prec, d, size):  # noqa: F811
    """Every key has one channel, which no other position of its run of d positions has: every state row is one decayed
    value, beside far larger ones in the other rows. Values of one head are dense and small."""
    heads, length = 3, d + 32
    rng = np.random.default_rng(83)
    q, k, v = (np.zeros((length, heads, d)) for _ in range(3))
    k[np.arange(length), :, np.arange(length) % d] = rng.uniform(1.0, 2.0, (length, heads))
    q[:] = rng.standard_normal(q.shape)
    v[:] = size * rng.standard_normal(v.shape)
    decay = np.array([0.5, 0.8, 0.97], np.float32)
    qkv = packed(prec, q, k, v)
    out = to_raw(np.zeros((1, length, heads * d)), prec)
    scale = float(np.float32(0.1 / size))
    b = [DevBuf(a) for a in (qkv, out, decay, np.zeros((1, heads, d, d), np.float32))]
    nn.linear_attention_noalloc(eng, nn.linear_attention_desc(prec, b[0], b[1], heads=heads, key_dim=d, value_dim=d, sequences=1,
                                                              length=length, decay=b[2], scale=scale, state_out=b[3]))
    eng.sync()
    check_sequence(prec, heads, d, d, qkv[0], decay, scale, length, None, b[1].get()[0], out[0], b[3].get()[0])


def rounds_from_within(got, want, tol, prec):
    """Every stored value is the rounding of some value within tol of the wanted one."""
    lo, hi = (from_raw(to_raw((want + s * tol).astype(np.float32), prec), prec) for s in (-1, 1))
    bad = (got < lo) | (got > hi)
    assert not bad.any(), (int(bad.sum()), bad.size, float((np.abs(got - want) / want)[bad].max()))


@pytest.mark.parametrize("prec", ["f16", "bf16"])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("path", ["state", "values"])
def test_what_16_bits_leave_of_the_products_before_an_output(eng, prec, d, path):  # noqa: F811
    """A state or a weighted query product enters the product with f16 queries or values, or bf16 ones, as two bf16
    pieces, the first cut off and the second rounded: 2^-16 of it at most, and the other operand is exact. The
    operands are powers of two with ones in every bit behind the eighth, which makes what is left out as large as it
    gets, with one sign. (f32's sums: d + 96 roundings of the term at most, 33 products of a chunk among them.)"""
    length, heads = 32, 2
    rng = np.random.default_rng(84)
    in16 = 1.0 + 2.0 ** -7 - 2.0 ** -10 if prec == "f16" else 1.0  # as far as 16 bits go
    in32 = 1.0 + 2.0 ** -7 - 2.0 ** -20

    def powers(*shape):
        return 0.5 ** rng.integers(0, 4, shape)

    q, k, state = np.zeros((length, heads, d)), np.zeros((length, heads, d)), None
    if path == "state":
        q[:], v, scale = in16 * powers(*q.shape), np.zeros(q.shape), 1.0 / d
        state = (in32 * powers(heads, d, d)).astype(np.float32)
    else:  # the query products are the keys times the scale
        q[:, :, 0], k[:, :, 0], v = 1.0, in16 * powers(length, heads), in16 * powers(length, heads, d)
        scale = 1.0 if prec == "f16" else in32
    decay = np.ones(heads, np.float32)
    qkv = packed(prec, q, k, v)
    b = [DevBuf(a) for a in (qkv, to_raw(np.zeros((1, length, heads * d)), prec), decay)]
    d_state = None if state is None else DevBuf(state[None])
    nn.linear_attention_noalloc(eng, nn.linear_attention_desc(prec, b[0], b[1], heads=heads, key_dim=d, value_dim=d, sequences=1,
                                                              length=length, decay=b[2], scale=scale, state_in=d_state))
    eng.sync()
    (o, oa, _), _ = oracle(q, k, v, decay, scale, length, state)
    got = from_raw(b[1].get(), prec).reshape(o.shape)
    rounds_from_within(got, o, (2.0 ** -16 + (d + 96) * U) * oa, prec)


@pytest.mark.parametrize("prec", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("seqs,length,d", [(1, 6001, 16), (1, 6001, 128), (600, 1000, 16)])
@pytest.mark.parametrize("what", ["first position", "state", "all positions"])
def test_decays_next_to_one_are_told_from_one(eng, prec, seqs, length, d, what):  # noqa: F811
    """What a memory of a thousand, of a million and of 16 million positions keeps of a one at the first position, of a
    state of ones, and of a one at every position, split into up to 188 segments or (600 sequences) in one.
    A chunk's power g^32 comes from 2^x, off by a step (2 U of a value above a half), at an exponent 32 log2 g
    off by 8 U of itself, and joins the state with one rounding, where ones come in at every position with up
    to 32 more: m chunks are off by m (3 + 8 * 32 |ln g|) U, or m 32 U more; 64 U for the first one's products."""
    decay = np.array([1 - 2.0 ** -10, 1 - 2.0 ** -20, 1 - 2.0 ** -24], np.float32)
    heads, g = 3, decay.astype(np.float64)
    q, k, v = (np.zeros((length, heads, d)) for _ in range(3))
    if what != "state":
        k[0], v[0] = 1.0, 1.0
    if what == "all positions":
        k[:], v[:] = 1.0, 1.0
    state = np.ones((seqs, heads, d, d), np.float32) if what == "state" else None
    b = [DevBuf(a) for a in (packed(prec, q, k, v), to_raw(np.zeros((seqs, length, heads * d)), prec), decay)]
    fin = DevBuf(np.zeros((seqs, heads, d, d), np.float32))
    d_state = None if state is None else DevBuf(state)
    nn.linear_attention_noalloc(eng, nn.linear_attention_desc(
        prec, b[0], b[1], heads=heads, key_dim=d, value_dim=d, sequences=seqs, length=length, decay=b[2], state_in=d_state,
        state_out=fin, q_sequence=0, k_sequence=0, v_sequence=0))
    eng.sync()
    n = {"first position": length - 1, "state": length}.get(what)
    keep = -np.expm1(length * np.log(g)) / (1 - g) if n is None else np.exp(n * np.log(g))
    m = -(-length // 32)
    rel = U * (m * (3 + 8 * 32 * np.abs(np.log(g)) + (32 if n is None else 0)) + 64)
    assert (np.abs(keep - (length if n is None else 1.0)) > 2 * rel * keep)[:2 if n is None or length < 6001 else 3].all()
    err = np.abs(fin.get() - keep[:, None, None]) / keep[:, None, None]
    assert (err <= rel[:, None, None]).all(), (err.max((0, 2, 3)) / U, rel / U)


@pytest.mark.parametrize("prec", ["f32", "bf16"])
def test_calls_that_share_a_scratch_keep_their_results(prec):
    """Linear attention in segments and channel attention work in the scratch of their context, one after the other; two
    contexts' calls overlap. Every output is that of the same call by itself."""
    engs = [nn.Engine(0, prec) for _ in range(2)]
    length, heads, d = 1500, 2, 32
    runs = []
    for i, e in enumerate(engs):
        qkv, out, decay, _ = inputs(30 + i, prec, 1, length, heads, d, d)
        b = [DevBuf(a) for a in (qkv, out, decay)]
        other = DevBuf(np.random.default_rng(i).standard_normal((20, 24, 3 * 64)).astype(np.float32))
        y, temp = DevBuf(np.zeros((20, 24, 64), np.float32)), DevBuf(np.ones(4, np.float32))
        desc = nn.linear_attention_desc(prec, b[0], b[1], heads=heads, key_dim=d, value_dim=d, sequences=1, length=length, decay=b[2])
        runs.append((e, desc, b, other, y, temp))

    def channel(e, other, y, temp):
        _lib.check(_lib.lib().zjai_channel_attention_noalloc(e.handle, other.address, 192, 20, 24, 4, temp.address, _lib.F32,
                                                             y.address), e.handle)

    want = []
    for e, desc, b, other, y, temp in runs:
        channel(e, other, y, temp)
        e.sync()
        nn.linear_attention_noalloc(e, desc)
        e.sync()
        want.append((y.get(), b[1].get()))
        y.put(np.zeros(y.shape, y.dtype))
        b[1].put(np.zeros(b[1].shape, b[1].dtype))
    assert not np.array_equal(want[0][0], want[1][0])
    for _ in range(5):
        for e, desc, b, other, y, temp in runs:
            nn.linear_attention_noalloc(e, desc)
            channel(e, other, y, temp)
            nn.linear_attention_noalloc(e, desc)
    for (e, _, b, _, y, _), w in zip(runs, want):
        e.sync()
        assert np.array_equal(y.get(), w[0]) and np.array_equal(b[1].get(), w[1])
    del runs, b, other, y, temp, desc
    for e in engs:
        e.close()


@pytest.mark.parametrize("prec", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,dk,dv", [(2, 64, 66), (1, 33, 1023), (3, 128, 70), (2, 100, 34), (1, 128, 129)])
@pytest.mark.parametrize("offset", [0, 4])
def test_steps_on_states_that_are_not_whole_16_bytes(eng, prec, heads, dk, dv, offset):  # noqa: F811
    """Rows whose length or place is not a multiple of four floats, with up to 16 of them to a lane."""
    n = 3
    qkv, out, decay, state = inputs(90, prec, n, 1, heads, dk, dv)
    b = [DevBuf(a) for a in (qkv, out, decay)]
    d_in, d_out = DevBuf(state, offset), DevBuf(np.zeros_like(state), offset)
    nn.linear_attention_step(eng, nn.linear_attention_desc(prec, b[0], b[1], heads=heads, key_dim=dk, value_dim=dv, sequences=n,
                                                           length=1, decay=b[2], state_in=d_in, state_out=d_out))
    eng.sync()
    got, fin = b[1].get(), d_out.get()
    for s in range(n):
        check_sequence(prec, heads, dk, dv, qkv[s], decay, 1.0, 1, state[s], got[s], out[s], fin[s])
