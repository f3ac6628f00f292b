"""CPU: a descriptor of a call on device buffers keeps the objects that it was made of, so that a buffer which nothing else
refers to is still there when the call is enqueued."""

import gc
import weakref

import pytest

from zenjpegai_amd import nn


class Buffer:
    def __init__(self, address):
        self.address = address

    def data_ptr(self):
        return self.address


SEQUENCES = dict(sequences=2, length=4)
KEPT = ["lengths", "slots", "state_in", "state_out"]
# Each helper's positional buffers, its other buffers, and what it needs besides.
HELPERS = {
    "linear_attention_desc": (["qkv", "out"], ["decay", *KEPT], dict(heads=2, key_dim=8, value_dim=8, num_slots=3, **SEQUENCES)),
    "rotary_desc": (["x", "out"], ["frequencies", "positions", "starts", "lengths"], dict(heads=2, head_dim=8, **SEQUENCES)),
    "causal_conv_desc": (["x", "out"], ["weight", "bias", *KEPT], dict(channels=8, taps=4, num_slots=3, **SEQUENCES)),
    "selective_scan_desc": (["x", "delta", "b", "c", "out"], ["a", "z", "d", "delta_bias", *KEPT],
                            dict(channels=8, state_dim=4, num_slots=3, **SEQUENCES)),
    "norm_gate_residual_desc": (["x", "y", "gate", "x_out", "h"],
                                ["post_weight", "post_bias", "residual_scale", "pre_weight", "pre_bias"], dict(positions=4, channels=8)),
}


def made(helper, buffers):
    first, others, kw = HELPERS[helper]
    return getattr(nn, helper)("f32", *(buffers[n] for n in first), **{n: buffers[n] for n in others}, **kw)


@pytest.mark.parametrize("helper", HELPERS)
def test_a_descriptor_keeps_its_buffers(helper):
    names = HELPERS[helper][0] + HELPERS[helper][1]
    buffers = {n: Buffer(4096 * (i + 1)) for i, n in enumerate(names)}
    refs = {n: weakref.ref(b) for n, b in buffers.items()}
    desc = made(helper, buffers)
    buffers.clear()
    gc.collect()
    assert [n for n, r in refs.items() if r() is None] == []
    for n in names:
        assert getattr(desc, "q" if n == "qkv" else n) == refs[n]().address
    del desc
    gc.collect()
    assert all(r() is None for r in refs.values())


def test_queries_keys_and_values_of_their_own_are_kept():
    qkv = [Buffer(4096 * (i + 1)) for i in range(3)]
    refs = [weakref.ref(b) for b in qkv]
    desc = made("linear_attention_desc", {"qkv": tuple(qkv), "out": 64, **dict.fromkeys(HELPERS["linear_attention_desc"][1])})
    qkv.clear()
    gc.collect()
    assert all(r() is not None for r in refs) and (desc.q, desc.k, desc.v, desc.out) == (4096, 8192, 12288, 64)


@pytest.mark.parametrize("helper", HELPERS)
def test_addresses_and_absent_buffers_need_no_object(helper):
    first, others, _ = HELPERS[helper]
    desc = made(helper, {n: 64 for n in first} | dict.fromkeys(others))
    assert all(getattr(desc, n) is None for n in others)
