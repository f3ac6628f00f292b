"""GPU: states of decayed linear attention: updated in place over many segments, what they keep of small and
single terms, and how fast they forget."""

import numpy as np
import pytest

from devbuf import DevBuf
from test_gpu_linear_attention import check_sequence, eng, inputs  # noqa: F401 (eng: the fixture)
from zenjpegai_amd import nn

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
