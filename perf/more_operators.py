"""The operators of a state-space context model over latents, as measurable cases.

``rotary`` turns the queries and keys of an attention by their positions, ``conv`` is the short causal convolution
in front of a scan, ``scan`` the selective state-space scan itself: each over whole maps or batches of sequences
(what an encoder, which has every latent, runs) and for one position of each of several sequences (what a decoder
runs, its states in slots).
"""

from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda:0"
STORAGE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def _rotary(prec, seqs, length, heads, dim, turned, layout, width=0, starts=False):
    return {"kind": "rotary", "prec": prec, "seqs": seqs, "length": length, "heads": heads, "dim": dim, "turned": turned,
            "layout": layout, "width": width, "starts": starts}


def _conv(prec, seqs, length, channels, taps, act, ragged=False, state=False, slots=0):
    return {"kind": "conv", "prec": prec, "seqs": seqs, "length": length, "channels": channels, "taps": taps, "act": act,
            "ragged": ragged, "state": state, "slots": slots}


def _scan(prec, seqs, length, channels, groups, states, gate=True, skip=True, ragged=False, state=False, slots=0):
    return {"kind": "scan", "prec": prec, "seqs": seqs, "length": length, "channels": channels, "groups": groups,
            "states": states, "gate": gate, "skip": skip, "ragged": ragged, "state": state, "slots": slots}


def listed():
    return [
        # One position of each of some dozens of pictures being decoded: the queries and keys of 8 heads each.
        {"name": "rotary_step_50_bf16", **_rotary("bf16", 50, 1, 16, 64, 64, "interleaved", starts=True)},
        # The latent map of the 1 MP picture, five heads; half of the pairs turn by row, half by column.
        {"name": "rotary_64x64_f32", **_rotary("f32", 1, 4096, 10, 32, 32, "halves", width=64)},
        # One very long sequence, continued far from its beginning; half of each head is turned.
        {"name": "rotary_long_bf16", **_rotary("bf16", 1, 65536, 32, 128, 64, "halves", starts=True)},
        # The latent of a 4K picture, every row a sequence of its own.
        {"name": "conv_rows_135x240_bf16", **_conv("bf16", 135, 240, 384, 4, "silu")},
        # A batch of latents of different sizes, continued from kept states.
        {"name": "conv_ragged_f16", **_conv("f16", 12, 3001, 2048, 4, "silu", ragged=True, state=True)},
        # A decoder server: one position of each of hundreds of pictures.
        {"name": "conv_step_257_f16", **_conv("f16", 257, 1, 2048, 4, "silu", state=True, slots=300)},
        # The latent of a 64 x 96 thumbnail, 4 x 6 positions: launches count.
        {"name": "scan_4x6_f32", **_scan("f32", 1, 24, 64, 1, 16)},
        # The latent map of the 1 MP picture in raster order, twice its 160 channels.
        {"name": "scan_64x64_f32", **_scan("f32", 1, 4096, 320, 1, 16)},
        # Latents of different sizes with large states, whose inputs and outputs four groups of channels have their own of.
        {"name": "scan_ragged_f16", **_scan("f16", 12, 3001, 1024, 4, 64, ragged=True, state=True)},
        # One very long sequence, which has to be split to fill the card.
        {"name": "scan_long_bf16", **_scan("bf16", 1, 65536, 2048, 1, 16, state=True)},
        # One position of one picture being decoded: latency.
        {"name": "scan_step_1_f32", **_scan("f32", 1, 1, 320, 1, 16, state=True, slots=1)},
        # ... and of hundreds: the states' traffic.
        {"name": "scan_step_257_f16", **_scan("f16", 257, 1, 2048, 1, 16, state=True, slots=300)},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, uniform in its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rotary", "conv", "scan", "scan"])
    prec = rng.choice(["f32", "f16", "bf16"])
    seqs = rng.choice([1, 1, 1, 2, 3, 8, 17, 64, 135])
    step = rng.random() < 0.3
    if step:
        seqs = _log(rng, 1, 300)
    if kind == "rotary":
        heads, dim = rng.choice([1, 2, 4, 5, 8, 10, 16, 32]), rng.choice([8, 20, 24, 32, 36, 64, 80, 100, 128, 256])
        width = 0 if step else rng.choice([0, 0, rng.randrange(1, 300)])
        turned = rng.choice([d for d in (dim, dim // 2, dim // 4) if d >= 4 and d % (4 if width else 2) == 0])
        room = 65536 * 32 * 128 * 2 // (SIZE[prec] * heads * dim * seqs)
        length = 1 if step else _log(rng, 1, max(1, min(65536, room)))
        return _rotary(prec, seqs, length, heads, dim, turned, rng.choice(["interleaved", "halves"]), width,
                       step or (not width and rng.random() < 0.5))
    channels = rng.choice([64, 96, 100, 160, 250, 320, 384, 512, 1000, 1001, 2048, 4096])
    slots = seqs + rng.randrange(40) if step else 0
    ragged, state = not step and rng.random() < 0.4, step or rng.random() < 0.5
    if kind == "conv":
        room = 12 * 3001 * 2048 * 2 // (SIZE[prec] * channels * seqs)
        length = 1 if step else _log(rng, 1, max(1, min(65536, room)))
        return _conv(prec, seqs, length, channels, rng.choice([2, 3, 4, 4, 5, 8]), rng.choice(["linear", "silu", "silu"]), ragged,
                     state, slots)
    groups = rng.choice([g for g in (1, 1, 1, 2, 4, 5, 7) if channels % g == 0])
    states = rng.choice([1, 2, 4, 8, 12, 16, 16, 16, 24, 32, 64])
    room = 65536 * 2048 * 16 * 2 // (SIZE[prec] * channels * max(states, 8) * seqs)
    length = 1 if step else _log(rng, 1, max(1, min(65536, room)))
    return _scan(prec, seqs, length, channels, groups, states, rng.random() < 0.7, rng.random() < 0.8, ragged, state, slots)


# ------------------------------------------------------------------------------------- inputs

def _inputs(case, seed):
    g = torch.Generator(DEVICE).manual_seed(seed)
    dt, n, t = STORAGE[case["prec"]], case["seqs"], case["length"]

    def normal(*shape, mean=0.0, dev=1.0, dtype=torch.float32):
        return (mean + dev * torch.randn(shape, generator=g, device=DEVICE)).to(dtype)

    def whole(lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=g, device=DEVICE, dtype=torch.int32)

    if case["kind"] == "rotary":
        h, d, r = case["heads"], case["dim"], case["turned"]
        # The queries and keys at the front of packed channels, the values behind them.
        x = {"x": normal(n, t, h * d + max(1, h // 2) * d, dtype=dt), "out": torch.zeros(n, t, h * d, dtype=dt, device=DEVICE),
             "starts": whole(0, 200000, n) if case["starts"] else None}
        pairs = r // 4 if case["width"] else r // 2
        f = 10000.0 ** (-torch.arange(pairs, dtype=torch.float64, device=DEVICE) / pairs)
        x["frequencies"] = torch.cat([f, f]) if case["width"] else f
        return x
    c = case["channels"]
    x = {"lengths": whole(0, t + 1, n) if case["ragged"] else None,
         "slots": torch.randperm(case["slots"], generator=g, device=DEVICE)[:n].to(torch.int32) if case["slots"] else None,
         "out": torch.zeros(n, t, c, dtype=dt, device=DEVICE)}
    kept = case["slots"] or n
    if case["kind"] == "conv":
        k = case["taps"]
        # The first half of packed channels: the others are a scan's gate.
        return {**x, "xz": normal(n, t, 2 * c, dtype=dt), "weight": normal(c, k, dev=k ** -0.5), "bias": normal(c, dev=0.2),
                "state_in": normal(kept, k - 1, c, dtype=dt) if case["state"] else None,
                "state_out": torch.zeros(kept, k - 1, c, dtype=dt, device=DEVICE) if case["state"] else None}
    m, gr = case["states"], case["groups"]
    # Steps between 0.001 and 0.1 on the whole, and decays of a state from -1 to -states.
    step = torch.exp(math.log(1e-3) + math.log(100.0) * torch.rand(c, generator=g, device=DEVICE))
    rates = torch.arange(1, m + 1, device=DEVICE) * torch.exp(normal(c, m, dev=0.1))
    return {**x, "u": normal(n, t, c, dtype=dt), "delta": normal(n, t, c, dev=0.5, dtype=dt), "bc": normal(n, t, 2 * gr * m, dtype=dt),
            "z": normal(n, t, 2 * c, dtype=dt) if case["gate"] else None, "a": -rates,
            "d": normal(c, mean=1.0, dev=0.1) if case["skip"] else None, "delta_bias": step + torch.log(-torch.expm1(-step)),
            "state_in": normal(kept, c, m) if case["state"] else None,
            "state_out": torch.zeros(kept, c, m, device=DEVICE) if case["state"] else None}


_engines = []


def _engine():
    """The process's one engine."""
    if not _engines:
        from zenjpegai_amd import nn
        _engines.append(nn.Engine(0))
    return _engines[0]


def _plan(case, x):
    """The descriptor of a call, which a program fills in once for its buffers."""
    from zenjpegai_amd import nn
    n, t = case["seqs"], case["length"]
    if case["kind"] == "rotary":
        p = x["x"].shape[2]
        return nn.rotary_desc(case["prec"], x["x"], x["out"], heads=case["heads"], head_dim=case["dim"], rotary_dim=case["turned"],
                              layout=case["layout"], width=case["width"], sequences=n, length=t, frequencies=x["frequencies"],
                              starts=x["starts"], x_position=p, x_sequence=p * t)
    c = case["channels"]
    common = dict(channels=c, sequences=n, length=t, lengths=x["lengths"], slots=x["slots"], num_slots=case["slots"],
                  state_in=x["state_in"], state_out=x["state_out"])
    if case["kind"] == "conv":
        return nn.causal_conv_desc(case["prec"], x["xz"], x["out"], taps=case["taps"], weight=x["weight"], bias=x["bias"],
                                   act=case["act"], x_position=2 * c, x_sequence=2 * c * t, **common)
    m, gr = case["states"], case["groups"]
    b = x["bc"].data_ptr()
    packed = 2 * gr * m
    strides = {"b_position": packed, "c_position": packed, "b_sequence": packed * t, "c_sequence": packed * t}
    z = None
    if x["z"] is not None:  # the other half of packed channels
        z = x["z"].data_ptr() + c * SIZE[case["prec"]]
        strides.update(z_position=2 * c, z_sequence=2 * c * t)
    return nn.selective_scan_desc(case["prec"], x["u"], x["delta"], b, b + gr * m * SIZE[case["prec"]], x["out"], z=z, groups=gr,
                                  state_dim=m, a=x["a"], d=x["d"], delta_bias=x["delta_bias"], softplus=True, **strides, **common)


def prepare(case, seed):
    state = {"case": case, **_inputs(case, seed)}
    if own:
        state["engine"], state["plan"] = _engine(), _plan(case, state)
        torch.cuda.current_stream(DEVICE).synchronize()  # the engine's stream is ordered with no other one
    return state


def run(state):
    """One pass. The engine's calls go on its own stream: their outputs are there, and the state's buffers free,
    when the engine or the device has been waited for (or a stream that the engine has ordered behind them)."""
    case = state["case"]
    kind, step = case["kind"], case.get("slots", 0) > 0
    if own:
        from zenjpegai_amd import nn
        if kind == "rotary":
            nn.rotary_noalloc(state["engine"], state["plan"])
            return [state["out"]]
        if kind == "conv":
            (nn.causal_conv_step if step else nn.causal_conv_noalloc)(state["engine"], state["plan"])
        else:
            (nn.selective_scan_step if step else nn.selective_scan_noalloc)(state["engine"], state["plan"])
        return [state["out"]] if state["state_out"] is None else [state["out"], state["state_out"]]
    if kind == "rotary":
        return _rotary_plain(state)
    if kind == "conv":
        return (_conv_step_plain if step else _conv_plain)(state)
    return (_scan_step_plain if step else _scan_plain)(state)


# -------------------------------------------------------------------------------- plain forms

def _rotary_plain(s):
    case, x, t = s["case"], s["x"], s["x"].shape[1]
    h, d, r = case["heads"], case["dim"], case["turned"]
    x = x[..., :h * d].reshape(x.shape[0], t, h, d).float()
    at = torch.arange(t, device=x.device, dtype=torch.float64)
    if case["width"]:
        row = torch.floor(at / case["width"])
        at = torch.stack([row, at - row * case["width"]], dim=1).repeat_interleave(r // 4, dim=1)[None]
    else:
        at = at[None, :, None] if s["starts"] is None else (s["starts"][:, None] + at)[..., None]
    angle = (at * s["frequencies"])[:, :, None]  # in 64 bits: far positions
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    if case["layout"] == "halves":
        a, b = x[..., :r // 2], x[..., r // 2:r]
        turned = [a * cos - b * sin, a * sin + b * cos]
    else:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        turned = [torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2)]
    return [torch.cat([*turned, x[..., r:]], dim=-1).reshape(s["out"].shape).to(s["out"].dtype)]


def _activate(x, act):
    return x * torch.sigmoid(x) if act == "silu" else x


def _valid(s):
    """Which positions a sequence has: [sequences][length]."""
    n, t = s["out"].shape[:2]
    at = torch.arange(t, device=s["out"].device)
    return (at < s["lengths"][:, None]) if s["lengths"] is not None else (at < t).expand(n, t)


def _windows(x, k):
    """[n][t + k - 1][c] -> [n][t][c][k]: the k positions that end at each."""
    return x.unfold(1, k, 1)


def _conv_plain(s):
    case, c, k = s["case"], s["case"]["channels"], s["case"]["taps"]
    x = s["xz"][..., :c]
    n, t = x.shape[:2]
    before = torch.zeros(n, k - 1, c, dtype=x.dtype, device=x.device) if s["state_in"] is None else s["state_in"]
    x = torch.cat([before, x], dim=1)
    y = _activate((_windows(x.float(), k) * s["weight"]).sum(-1) + s["bias"], case["act"])
    out = torch.where(_valid(s)[..., None], y.to(s["out"].dtype), s["out"])
    if s["state_out"] is None:
        return [out]
    first = torch.full((n,), t, device=x.device) if s["lengths"] is None else s["lengths"].long()
    rows = first[:, None] + torch.arange(k - 1, device=x.device)
    return [out, x.gather(1, rows[..., None].expand(-1, -1, c))]


def _conv_step_plain(s):
    case, c = s["case"], s["case"]["channels"]
    at = s["slots"].long()
    x = torch.cat([s["state_in"][at], s["xz"][..., :c]], dim=1)
    y = _activate((x.float() * s["weight"].t()).sum(1) + s["bias"], case["act"])
    s["state_out"].index_copy_(0, at, x[:, 1:])
    return [y[:, None].to(s["out"].dtype), s["state_out"]]


def _softplus(x):
    return x.clamp(min=0) + torch.log1p(torch.exp(-x.abs()))


def _finish(s, y):
    """Skip and gate: y [n][t][c] in f32 -> the outputs."""
    c = s["case"]["channels"]
    if s["d"] is not None:
        y = y + s["d"] * s["u"].float()
    if s["z"] is not None:
        y = y * _activate(s["z"][..., c:].float(), "silu")
    return y.to(s["out"].dtype)


def _recur(h, dt, a, x, b, c):
    """The recurrence over the positions (dimension 2 of dt, x [n][m][t][g][w], b, c [n][m][t][g][s]; h [n][m][g][w][s]):
    the last state and, where c is given, the outputs [n][m][t][g][w]. Each step depends on the one before."""
    y = None if c is None else torch.empty_like(dt)
    for i in range(dt.shape[2]):
        h = torch.exp(dt[:, :, i, ..., None] * a) * h + (dt[:, :, i] * x[:, :, i])[..., None] * b[:, :, i, :, None]
        if c is not None:
            torch.sum(h * c[:, :, i, :, None], -1, out=y[:, :, i])
    return h, y


def _scan_plain(s):
    case = s["case"]
    g, m, w = case["groups"], case["states"], case["channels"] // case["groups"]
    n, t, c = s["u"].shape
    dt = torch.where(_valid(s)[..., None], _softplus(s["delta"].float() + s["delta_bias"]), 0.0)  # no step, no change
    # Pieces of a square root's length: all of them at once without what comes before, that from piece to piece, and all
    # of them again with it.
    size = math.isqrt(t - 1) + 1 if t > 64 else t
    pieces = -(-t // size)

    def cut(x, *shape):
        return torch.nn.functional.pad(x, (0, 0, 0, pieces * size - t)).reshape(n, pieces, size, *shape)

    dt, x = cut(dt, g, w), cut(s["u"].float(), g, w)
    b, o = (cut(v, g, m) for v in s["bc"].float().split(g * m, dim=2))
    a = s["a"].reshape(g, w, m)
    h = torch.zeros(n, 1, g, w, m, device=x.device) if s["state_in"] is None else s["state_in"].reshape(n, 1, g, w, m)
    if pieces > 1:
        ends, _ = _recur(torch.zeros(n, pieces, g, w, m, device=x.device), dt, a, x, b, None)
        keep = torch.exp(dt.sum(2)[..., None] * a)
        starts = [h[:, 0]]
        for i in range(pieces - 1):
            starts.append(keep[:, i] * starts[-1] + ends[:, i])
        h = torch.stack(starts, dim=1)
    h, y = _recur(h, dt, a, x, b, o)
    out = _finish(s, y.reshape(n, pieces * size, c)[:, :t])
    out = torch.where(_valid(s)[..., None], out, s["out"])
    return [out] if s["state_out"] is None else [out, h[:, -1].reshape(n, c, m)]


def _scan_step_plain(s):
    case = s["case"]
    g, m, w = case["groups"], case["states"], case["channels"] // case["groups"]
    n = case["seqs"]
    at = s["slots"].long()
    dt = _softplus(s["delta"].float() + s["delta_bias"]).reshape(n, g, w, 1)
    b, o = (v.reshape(n, g, 1, m) for v in s["bc"].float().split(g * m, dim=2))
    h = torch.exp(dt * s["a"].reshape(g, w, m)) * s["state_in"][at].reshape(n, g, w, m) + dt * s["u"].float().reshape(n, g, w, 1) * b
    s["state_out"].index_copy_(0, at, h.reshape(n, g * w, m))
    return [_finish(s, (h * o).sum(-1).reshape(n, 1, g * w)), s["state_out"]]


# ---------------------------------------------------------------------------------- 64 bits

def exact(case, seed):
    s = {k: v.double() if isinstance(v, torch.Tensor) and v.dtype.is_floating_point else v for k, v in _inputs(case, seed).items()}
    n, t = case["seqs"], case["length"]
    device = s["out"].device

    if case["kind"] == "rotary":
        h, d, r = case["heads"], case["dim"], case["turned"]
        x = s["x"][..., :h * d].reshape(n, t, h, d)
        place = torch.arange(t, device=device)
        if case["width"]:
            axes = torch.cat([(place // case["width"])[:, None].expand(t, r // 4), (place % case["width"])[:, None].expand(t, r // 4)], dim=1)
            angle = axes.double().expand(n, t, r // 2) * s["frequencies"]
        else:
            place = place.expand(n, t) if s["starts"] is None else place + s["starts"].long()[:, None]
            angle = place.double()[..., None] * s["frequencies"]
        turn = torch.polar(torch.ones_like(angle), angle)[:, :, None]
        y = x.clone()
        if case["layout"] == "halves":
            z = torch.complex(x[..., :r // 2], x[..., r // 2:r]) * turn
            y[..., :r // 2], y[..., r // 2:r] = z.real, z.imag
        else:
            z = torch.complex(x[..., 0:r:2].contiguous(), x[..., 1:r:2].contiguous()) * turn
            y[..., 0:r:2], y[..., 1:r:2] = z.real, z.imag
        return [y.reshape(n, t, h * d)]

    c = case["channels"]
    ends = torch.full((n,), t, device=device) if s["lengths"] is None else s["lengths"].long()
    live = (torch.arange(t, device=device) < ends[:, None])[..., None]

    def states(new):
        """The states of all slots with those of the sequences put in."""
        if s["slots"] is None:
            return new
        kept = s["state_out"].clone()
        kept[s["slots"].long()] = new
        return kept

    def begin(*shape):
        if s["state_in"] is None:
            return torch.zeros(n, *shape, dtype=torch.float64, device=device)
        return s["state_in"].clone() if s["slots"] is None else s["state_in"][s["slots"].long()]

    if case["kind"] == "conv":
        k = case["taps"]
        x = torch.cat([begin(k - 1, c), s["xz"][..., :c]], dim=1)
        y = s["bias"].expand(n, t, c).clone()
        for j in range(k):
            y += s["weight"][:, j] * x[:, j:j + t]
        if case["act"] == "silu":
            y = y / (1.0 + torch.exp(-y))
        y = torch.where(live, y, s["out"])
        if s["state_out"] is None:
            return [y]
        return [y, states(torch.stack([x[i, e:e + k - 1] for i, e in enumerate(ends.tolist())]))]

    g, m = case["groups"], case["states"]
    delta = s["delta"] + s["delta_bias"]
    delta = torch.where(delta > 30.0, delta, torch.log1p(torch.exp(delta)))
    spread = torch.arange(c, device=device) // (c // g)  # each channel's group
    b, o = s["bc"][..., :g * m].reshape(n, t, g, m), s["bc"][..., g * m:].reshape(n, t, g, m)
    S, y = begin(c, m), torch.empty(n, t, c, dtype=torch.float64, device=device)
    for j in range(t):
        step = delta[:, j, :, None]
        new = torch.exp(step * s["a"]) * S + step * s["u"][:, j, :, None] * b[:, j, spread]
        y[:, j] = torch.einsum("ncs,ncs->nc", new, o[:, j, spread])
        S = new if s["lengths"] is None else torch.where(live[:, j, :, None], new, S)
    if s["d"] is not None:
        y += s["d"] * s["u"]
    if s["z"] is not None:
        z = s["z"][..., c:]
        y *= z / (1.0 + torch.exp(-z))
    y = torch.where(live, y, s["out"])
    return [y] if s["state_out"] is None else [y, states(S)]


def work(case):
    e, n = SIZE[case["prec"]], case["seqs"] * case["length"] * (0.5 if case.get("ragged") else 1.0)  # lengths are uniform
    if case["kind"] == "rotary":
        return {"bytes": 2.0 * e * n * case["heads"] * case["dim"] + 8.0 * (case["turned"] // 2),
                "flops": n * (3.0 * case["heads"] * case["turned"] + 20.0 * case["turned"])}
    c = case["channels"]
    if case["kind"] == "conv":
        states = 2.0 * e * case["seqs"] * (case["taps"] - 1) * c if case["state"] else 0.0
        return {"bytes": 2.0 * e * n * c + 4.0 * c * (case["taps"] + 1) + states, "flops": n * c * (2.0 * case["taps"] + 6.0)}
    m = case["states"]
    states = 8.0 * case["seqs"] * c * m if case["state"] else 0.0
    return {"bytes": e * n * ((3 + case["gate"]) * c + 2 * case["groups"] * m) + 4.0 * c * (m + 2) + states,
            "flops": n * c * (7.0 * m + 20.0)}
