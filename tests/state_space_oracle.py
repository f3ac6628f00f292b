"""Rotary positions, short causal convolution and selective scan in 64 bits, one position after another, with bounds on what
f32 arithmetic and the rounding of the results may differ by.

U is f32's half step. The hardware's 2^x and 1 / x are taken to be off by a step (2 U) at most."""

import numpy as np

from devbuf import HALF_STEP

U = 2.0 ** -24


def rounded(prec, value, err):
    """The bound `err` on a value, with its rounding to the storage type (f16: half of the smallest step, too)."""
    return err + HALF_STEP[prec] * (np.abs(value) + err) + (2.0 ** -25 if prec == "f16" else 1e-37)


# ------------------------------------------------------------------------------------- rotary

def rotary(prec, x, places, freq, layout, magnitude, inverse=False, turned=None):
    """x [t][heads][dim], places [t] or [t][pairs] -> (out, bound). An angle is off by 2^-51 of itself and by the rounding
    of what is left of it (an eighth of a turn at most: 2^-25), sine and cosine by that, 2^-27 of their series and
    two roundings; the magnitude is one rounding, the products and their sum three."""
    t, _, dim = x.shape
    r = 2 * len(freq) if turned is None else turned
    p = np.broadcast_to(np.asarray(places, np.float64).reshape(t, max(1, np.size(places) // max(t, 1))), (t, r // 2))
    angle = p * np.asarray(freq, np.float64)
    # Angles whose double is off by more than the bound: whole turns taken off in wider arithmetic.
    turns = np.asarray(p, np.longdouble) * np.asarray(freq, np.float64).astype(np.longdouble)
    rest = np.fmod(turns, 2 * np.pi * np.longdouble(1) + np.longdouble(2.4492935982947064e-16)).astype(np.float64)
    c, s = magnitude * np.cos(rest)[:, None], magnitude * np.sin(rest)[:, None]
    if inverse:
        s = -s
    a, b = (x[..., :r // 2], x[..., r // 2:r]) if layout == "halves" else (x[..., 0:r:2], x[..., 1:r:2])
    off = abs(magnitude) * (2.0 ** -51 * np.abs(angle)[:, None] + 2.0 ** -25 + 2.0 ** -27 + 2 * U)
    e = off * (np.abs(a) + np.abs(b)) + 4 * U * (np.abs(a * c) + np.abs(b * s))
    e2 = off * (np.abs(a) + np.abs(b)) + 4 * U * (np.abs(a * s) + np.abs(b * c))
    out, tol = x.copy(), np.zeros_like(x)
    u, v = a * c - b * s, a * s + b * c
    at = (slice(0, r // 2), slice(r // 2, r)) if layout == "halves" else (slice(0, r, 2), slice(1, r, 2))
    out[..., at[0]], out[..., at[1]] = u, v
    tol[..., at[0]], tol[..., at[1]] = rounded(prec, u, e), rounded(prec, v, e2)
    return out, tol


# --------------------------------------------------------------------------------- convolution

def activation(act, v, e):
    """act(v) and the bound on it for an argument that is off by e: both activations' slopes are 1.1 at most, the exponential is off
    by |v| + 2 roundings and what follows by five."""
    with np.errstate(over="ignore"):
        s = 1.0 / (1.0 + np.exp(-v))
    y = {"linear": v, "sigmoid": s, "silu": v * s}[act]
    return (y, e) if act == "linear" else (y, 1.1 * e + U * (np.abs(v) + 7) * np.abs(y) + 1e-36)


def conv(prec, x, weight, bias, act, length, before=None):
    """x [t][c], weight [c][taps], before [taps - 1][c] -> (out, bound, the last taps - 1 inputs)."""
    t, c = x.shape
    k = weight.shape[1]
    full = np.concatenate([np.zeros((k - 1, c)) if before is None else before, x])
    w = weight.astype(np.float64)
    v = np.zeros((t, c)) if bias is None else np.broadcast_to(bias.astype(np.float64), (t, c)).copy()
    m = np.abs(v)
    with np.errstate(invalid="ignore"):
        for j in range(k):
            v = v + w[:, j] * full[j:j + t]
            m = m + np.abs(w[:, j] * full[j:j + t])
        y, e = activation(act, v, U * k * m)
        return y, rounded(prec, y, e), full[length:length + k - 1]


# ---------------------------------------------------------------------------------------- scan

def scan(prec, x, delta, b, c, z, a, d, delta_bias, softplus, length, state=None):
    """x, delta, z [t][ch], b, c [t][groups][n], a [ch][n] -> (out, bound, state, its bound). Of a position's step: its
    argument is off by a rounding, e^s by |s| + 2, what makes it the softplus by nine; of its decay: the rate by two, its
    product by one, 2^x by two. A state collects the roundings of every step's decay, product and sum; the
    pieces that a long sequence is computed in add fewer of them than the steps they stand for."""
    t, ch = x.shape
    g, n = b.shape[1:]
    spread = np.arange(ch) // (ch // g)
    A64 = a.astype(np.float64)
    s = delta + (0.0 if delta_bias is None else delta_bias.astype(np.float64))
    es = U * np.ones_like(s)
    if softplus:
        es = np.where(s == -np.inf, 0.0, U * (2 * np.abs(s) + 12))  # e^-inf is 0 without an error, and so is the step
        s = np.maximum(s, 0) + np.log1p(np.exp(-np.abs(s)))
    h = np.zeros((ch, n)) if state is None else state.astype(np.float64).copy()
    mag, err = np.abs(h), np.zeros((ch, n))
    y, e = np.zeros((t, ch)), np.zeros((t, ch))
    with np.errstate(invalid="ignore", over="ignore"):
        for i in range(length):
            sa = s[i][:, None] * A64
            keep = np.exp(sa)
            new = s[i][:, None] * x[i][:, None] * b[i][spread]
            err = keep * err + keep * mag * (U * 4 + np.abs(sa) * (4 * U + es[i][:, None])) + np.abs(new) * (3 * U + es[i][:, None])
            mag = keep * mag + np.abs(new)
            h = keep * h + new
            cc = c[i][spread]
            y[i] = (cc * h).sum(1)
            e[i] = (np.abs(cc) * (err + (n + 6) * U * mag)).sum(1)
        if d is not None:
            dx = d.astype(np.float64) * x
            y, e = y + dx, e + U * (2 * np.abs(dx) + np.abs(y))
        if z is not None:
            gate, ge = activation("silu", z, 0.0)
            e = e * np.abs(gate) + np.abs(y) * (ge + 2 * U * np.abs(gate))
            y = y * gate
        return y, rounded(prec, y, e), h, err + U * mag + 1e-37
