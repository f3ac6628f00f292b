"""Decayed linear attention in 64 bits, position after position, with bounds on what f32 arithmetic may
differ by."""

import numpy as np

from devbuf import HALF_STEP

U = 2.0 ** -24


def oracle(q, k, v, decay, scale, length, state=None):
    """One sequence: q, k [t][h][dk], v [t][h][dv], state [h][dk][dv] -> (out [t][h][dv], state),
    each with an array of the magnitudes (A, B) that the bounds are made of:
    A_t = scale |q_t| sum_j g^(t-j) |k_j| |v_j|   (what the terms of the sum add up to),
    B_t = the same with the j-th term counted t - j + 1 times (the roundings it goes through)."""
    t, h, dk = q.shape
    dv = v.shape[2]
    S = np.zeros((h, dk, dv)) if state is None else state.astype(np.float64).copy()
    A, B = np.abs(S), np.abs(S)
    g = decay.astype(np.float64)[:, None, None]
    out, oa, ob = (np.zeros((t, h, dv)) for _ in range(3))
    with np.errstate(invalid="ignore", over="ignore"):
        for i in range(length):
            kv = k[i][:, :, None] * v[i][:, None, :]
            S = g * S + kv
            A = g * A + np.abs(kv)
            B = g * B + A
            out[i] = scale * np.matmul(q[i][:, None, :], S)[:, 0]
            oa[i] = abs(scale) * np.matmul(np.abs(q[i])[:, None, :], A)[:, 0]
            ob[i] = abs(scale) * np.matmul(np.abs(q[i])[:, None, :], B)[:, 0]
    return (out, oa, ob), (S, A, B)


def out_bound(prec, dk, out, A, B):
    """f32 sums: two roundings for each position a term stays in the state, dk of the query's products,
    64 of a chunk's; in the 16-bit types the intermediate products and states enter the matrix cores
    as two bf16 pieces (2^-16 of them each); and the rounding of the result (2^-25: f16's smallest step halved)."""
    f32 = U * (2 * B + (dk + 96) * A)
    pieces = 0.0 if prec == "f32" else 2 * 2.0 ** -16 * A
    return f32 + pieces + HALF_STEP[prec] * (np.abs(out) + f32 + pieces) + 2.0 ** -25 * (prec == "f16")


def state_bound(S, A, B):
    return U * (2 * B + 96 * A) + 1e-37
