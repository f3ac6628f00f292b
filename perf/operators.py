"""The operators of a causal context model over latents, as measurable cases.

Three ways in which a program uses them: ``attend``, decayed linear attention over whole maps or
batches of sequences (what an encoder, which has every latent, runs); ``step``, its recurrent form
for one position of each of several sequences (what a decoder runs); ``join``, the end of a block
and the start of the next: norm, gate, residual scale, residual and norm in one pass.
"""

from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda:0"
STORAGE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
POST_EPS, PRE_EPS = 1e-5, 1e-6


def _attend(prec, seqs, length, heads, dk, dv, ragged=False, state=False):
    return {"kind": "attend", "prec": prec, "seqs": seqs, "length": length, "heads": heads, "dk": dk, "dv": dv,
            "ragged": ragged, "state": state}


def _step(prec, tokens, heads, dk, dv, slots):
    return {"kind": "step", "prec": prec, "tokens": tokens, "heads": heads, "dk": dk, "dv": dv, "slots": slots}


def _join(prec, positions, channels, groups, post, gate, pre):
    return {"kind": "join", "prec": prec, "positions": positions, "channels": channels, "groups": groups,
            "post": post, "gate": gate, "pre": pre}


def listed():
    return [
        # The latent of a 64 x 96 thumbnail, 4 x 6 positions: launches count.
        {"name": "attend_4x6_f32", **_attend("f32", 1, 24, 4, 32, 32)},
        # The latent map of the 1 MP picture in raster order, 160 channels in five heads.
        {"name": "attend_64x64_f32", **_attend("f32", 1, 4096, 5, 32, 32)},
        # The latent of a 4K picture, every row a sequence of its own; heads of 24 channels.
        {"name": "attend_rows_135x240_bf16", **_attend("bf16", 135, 240, 8, 24, 24)},
        # A batch of latents of different sizes, continued from kept states, values wider than keys.
        {"name": "attend_ragged_f16", **_attend("f16", 12, 3001, 8, 64, 128, ragged=True, state=True)},
        # One very long sequence, which has to be split to fill the card.
        {"name": "attend_long_bf16", **_attend("bf16", 1, 65536, 16, 128, 128, state=True)},
        # One position of one picture being decoded: latency.
        {"name": "step_1_f32", **_step("f32", 1, 4, 32, 32, 1)},
        # A decoder server: one position of each of some dozens of pictures, their states in slots.
        {"name": "step_50_bf16", **_step("bf16", 50, 16, 64, 64, 64)},
        # ... and of hundreds, with large heads: the states' traffic.
        {"name": "step_257_f16", **_step("f16", 257, 16, 128, 128, 300)},
        # The block join of a single position.
        {"name": "join_1x1024_bf16", **_join("bf16", 1, 1024, 8, "rms", "silu", "rms")},
        # The map of a 4K tile at the attention blocks' 128 channels, normed head by head.
        {"name": "join_215x216x128_bf16", **_join("bf16", 215 * 216, 128, 4, "layer", "sigmoid", "layer")},
        # A preview-sized map in f32, without a gate.
        {"name": "join_203x301x192_f32", **_join("f32", 203 * 301, 192, 1, "layer", "none", "layer")},
        # Wide channels over many positions: bandwidth.
        {"name": "join_16385x4096_f16", **_join("f16", 16385, 4096, 16, "rms", "silu", "rms")},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, uniform in its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "step", "join"])
    prec = rng.choice(["f32", "f16", "bf16"])
    if kind == "join":
        channels = rng.choice([96, 100, 128, 160, 192, 250, 512, 1000, 2048, 4096])
        groups = rng.choice([g for g in (1, 2, 4, 5, 8, 16) if channels % g == 0])
        positions = _log(rng, 1, min(1 << 18, 16384 * 4096 * 2 // SIZE[prec] // channels))
        return _join(prec, positions, channels, groups, rng.choice(["none", "layer", "rms"]),
                     rng.choice(["none", "linear", "sigmoid", "silu"]), rng.choice(["none", "layer", "rms"]))
    heads = rng.choice([1, 2, 4, 5, 8, 12, 16])
    dk, dv = rng.choice([8, 16, 20, 24, 32, 48, 64, 80, 128]), rng.choice([8, 16, 24, 30, 32, 64, 96, 128, 256])
    if kind == "step":
        tokens = _log(rng, 1, min(1024, 257 * 16 * 128 * 128 // (heads * dk * dv)))
        return _step(prec, tokens, heads, dk, dv, tokens + rng.randrange(40))
    seqs = rng.choice([1, 1, 1, 2, 3, 8, 17, 64, 135])
    room = 65536 * 16 * 128 * 2 * 2 // (SIZE[prec] * heads * (dk + dv) * seqs)
    return _attend(prec, seqs, _log(rng, 1, max(1, min(65536, room))), heads, dk, dv, rng.random() < 0.4,
                   rng.random() < 0.5)


# ------------------------------------------------------------------------------------- inputs

def _decays(heads):
    """From a memory of two positions in the first head to one of a thousand in the last."""
    return 1.0 - 2.0 ** -torch.linspace(1.0, 10.0, heads, dtype=torch.float64)


def _inputs(case, seed):
    g = torch.Generator(DEVICE).manual_seed(seed)
    dt = STORAGE[case["prec"]]

    def normal(*shape, mean=0.0, dev=1.0, dtype=torch.float32):
        return (mean + dev * torch.randn(shape, generator=g, device=DEVICE)).to(dtype)

    if case["kind"] == "join":
        n, c = case["positions"], case["channels"]
        x = {"x": normal(n, c, dev=2.0, dtype=dt), "y": normal(n, c, mean=0.3, dtype=dt),
             "gate": None if case["gate"] == "none" else normal(n, c, dtype=dt),
             "post_weight": normal(c, mean=1.0, dev=0.1), "post_bias": normal(c, dev=0.1),
             "scale": normal(c, mean=0.5, dev=0.2),
             "pre_weight": normal(c, mean=1.0, dev=0.1), "pre_bias": normal(c, dev=0.1),
             "x_out": torch.empty(n, c, dtype=dt, device=DEVICE),
             "h": None if case["pre"] == "none" else torch.empty(n, c, dtype=dt, device=DEVICE)}
        unused = {"layer": [], "rms": ["_bias"], "none": ["_weight", "_bias"]}
        x.update({p + name: None for p in ("post", "pre") for name in unused[case[p]]})
        return x
    h, dk, dv = case["heads"], case["dk"], case["dv"]
    decay = _decays(h).float().to(DEVICE)
    if case["kind"] == "step":
        n, m = case["tokens"], case["slots"]
        return {"qkv": normal(n, 1, h * (2 * dk + dv), dtype=dt), "decay": decay,
                "slots": torch.randperm(m, generator=g, device=DEVICE)[:n].to(torch.int32),
                "state_in": normal(m, h, dk, dv, dev=2.0), "state_out": torch.zeros(m, h, dk, dv, device=DEVICE),
                "out": torch.zeros(n, 1, h * dv, dtype=dt, device=DEVICE)}
    n, t = case["seqs"], case["length"]
    return {"qkv": normal(n, t, h * (2 * dk + dv), dtype=dt), "decay": decay,
            "lengths": torch.randint(0, t + 1, (n,), generator=g, device=DEVICE, dtype=torch.int32) if case["ragged"] else None,
            "state_in": normal(n, h, dk, dv, dev=2.0) if case["state"] else None,
            "state_out": torch.empty(n, h, dk, dv, device=DEVICE) if case["state"] else None,
            "out": torch.zeros(n, t, h * dv, dtype=dt, device=DEVICE)}


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
    if case["kind"] == "join":
        return nn.norm_gate_residual_desc(
            case["prec"], x["x"], x["y"], x["gate"], x["x_out"], x["h"], positions=case["positions"],
            channels=case["channels"], post_norm=case["post"], post_groups=case["groups"], post_eps=POST_EPS,
            post_weight=x["post_weight"], post_bias=x["post_bias"],
            gate_act="linear" if case["gate"] == "none" else case["gate"], residual_scale=x["scale"],
            pre_norm=case["pre"], pre_eps=PRE_EPS, pre_weight=x["pre_weight"], pre_bias=x["pre_bias"])
    return nn.linear_attention_desc(
        case["prec"], x["qkv"], x["out"], heads=case["heads"], key_dim=case["dk"], value_dim=case["dv"],
        sequences=x["qkv"].shape[0], length=x["qkv"].shape[1], decay=x["decay"], scale=case["dk"] ** -0.5,
        lengths=x.get("lengths"), slots=x.get("slots"), num_slots=case.get("slots", 0),
        state_in=x["state_in"], state_out=x["state_out"])


def prepare(case, seed):
    state = {"case": case, **_inputs(case, seed)}
    if own:
        state["engine"], state["plan"] = _engine(), _plan(case, state)
        torch.cuda.current_stream(DEVICE).synchronize()  # the engine's stream is ordered with no other one
    return state


def run(state):
    """One pass. The engine's calls go on its own stream: their outputs are there, and the state's buffers free,
    when the engine or the device has been waited for (or a stream that the engine has ordered behind them)."""
    kind = state["case"]["kind"]
    if own:
        from zenjpegai_amd import nn
        if kind == "join":
            nn.norm_gate_residual_noalloc(state["engine"], state["plan"])
        elif kind == "step":
            nn.linear_attention_step(state["engine"], state["plan"])
        else:
            nn.linear_attention_noalloc(state["engine"], state["plan"])
    else:
        return {"attend": _attend_plain, "step": _step_plain, "join": _join_plain}[kind](state)
    if kind == "join":
        return [state["x_out"]] if state["h"] is None else [state["x_out"], state["h"]]
    return [state["out"]] if state["state_out"] is None else [state["out"], state["state_out"]]


# -------------------------------------------------------------------------------- plain forms

def _split(case, qkv):
    """The packed channels as f32 q, k [n][h][t][dk] and v [n][h][t][dv]."""
    h, dk, dv = case["heads"], case["dk"], case["dv"]
    n, t, _ = qkv.shape
    q, k, v = qkv.float().split([h * dk, h * dk, h * dv], dim=2)
    return tuple(a.reshape(n, t, h, -1).transpose(1, 2) for a in (q, k, v))


def _powers(decay, exponents):
    """decay[h] ** exponents, [h][...] in f32, by way of 64 bits; a negative exponent's is zero."""
    e = exponents.clamp(min=0).double()
    p = decay.double().reshape(-1, *[1] * e.dim()) ** e
    return (p * (exponents >= 0)).float()


def _attend_plain(s):
    case, decay = s["case"], s["decay"]
    h, dk, dv = case["heads"], case["dk"], case["dv"]
    q, k, v = _split(case, s["qkv"])
    n, _, t, _ = q.shape
    at = torch.arange(t, device=q.device)
    lengths = s["lengths"]
    if lengths is None:
        lengths = torch.full((n,), t, device=q.device, dtype=torch.int32)
    valid = at < lengths[:, None]
    k = torch.where(valid[:, None, :, None], k, 0.0)
    v = torch.where(valid[:, None, :, None], v, 0.0)
    state_out = None
    if s["state_out"] is not None:
        ahead = lengths[:, None] - 1 - at  # positions still to come after this one
        w = _powers(decay, ahead).transpose(0, 1)
        state_out = (k * w[..., None]).transpose(2, 3) @ v
        if s["state_in"] is not None:
            state_out = state_out + _powers(decay, lengths).t()[:, :, None, None] * s["state_in"]
    # Chunks of c positions: within one by its own products, across chunks by the state before it.
    c = 64 if t <= 8192 else 128
    m = -(-t // c)
    pad = (0, 0, 0, m * c - t)
    q, k, v = (torch.nn.functional.pad(a, pad).reshape(n, h, m, c, -1) for a in (q, k, v))
    i = torch.arange(c, device=q.device)
    a = torch.arange(m, device=q.device)
    kv = (k * _powers(decay, c - 1 - i)[:, None, :, None]).transpose(3, 4) @ v
    before = _powers(decay, c * (a[:, None] - 1 - a)) @ kv.reshape(n, h, m, dk * dv)
    if s["state_in"] is not None:
        before = before + _powers(decay, c * a)[:, :, None] * s["state_in"].reshape(n, h, 1, dk * dv)
    o = (q * _powers(decay, i + 1)[:, None, :, None]) @ before.reshape(n, h, m, dk, dv)
    o = o + ((q @ k.transpose(3, 4)) * _powers(decay, i[:, None] - i)[:, None]) @ v
    o = (o * dk ** -0.5).reshape(n, h, m * c, dv)[:, :, :t].transpose(1, 2).reshape(n, t, h * dv)
    out = torch.where(valid[..., None], o.to(s["out"].dtype), s["out"])
    return [out] if state_out is None else [out, state_out]


def _step_plain(s):
    case = s["case"]
    q, k, v = (a[:, :, 0] for a in _split(case, s["qkv"]))
    at = s["slots"].long()
    new = s["decay"][:, None, None] * s["state_in"][at] + k[..., None] * v[:, :, None]
    o = (q[..., None] * new).sum(2) * case["dk"] ** -0.5
    s["state_out"].index_copy_(0, at, new)
    return [o.reshape(o.shape[0], 1, -1).to(s["out"].dtype), s["state_out"]]


def _norm(x, kind, eps):
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps)


def _join_plain(s):
    case, dt = s["case"], s["x"].dtype
    y = s["y"].float()
    if case["post"] != "none":
        y = _norm(y.reshape(y.shape[0], case["groups"], -1), case["post"], POST_EPS).reshape(y.shape) * s["post_weight"]
        if s["post_bias"] is not None:
            y = y + s["post_bias"]
    if s["gate"] is not None:
        g = s["gate"].float()
        y = y * (g if case["gate"] == "linear" else torch.sigmoid(g) if case["gate"] == "sigmoid" else g * torch.sigmoid(g))
    x = s["x"].float() + s["scale"] * y
    if case["pre"] == "none":
        return [x.to(dt)]
    h = _norm(x, case["pre"], PRE_EPS) * s["pre_weight"]
    if s["pre_bias"] is not None:
        h = h + s["pre_bias"]
    return [x.to(dt), h.to(dt)]


# ---------------------------------------------------------------------------------- 64 bits

def exact(case, seed):
    s = _inputs(case, seed)

    def recurrence(qkv, decay, scale, lengths, state, heads, dk, dv, out):
        """S = decay S + k v^T; o = scale q S, position after position; rows past a length keep out's."""
        n, t, _ = qkv.shape
        x = qkv.double()
        q = x[..., :heads * dk].reshape(n, t, heads, dk)
        k = x[..., heads * dk:2 * heads * dk].reshape(n, t, heads, dk)
        v = x[..., 2 * heads * dk:].reshape(n, t, heads, dv)
        S = torch.zeros(n, heads, dk, dv, dtype=torch.float64, device=x.device) if state is None else state.double().clone()
        g = decay.double()[:, None, None]
        o = out.double().reshape(n, t, heads, dv)
        for j in range(t):
            new = g * S + k[:, j, :, :, None] * v[:, j, :, None, :]
            y = scale * torch.einsum("nhk,nhkv->nhv", q[:, j], new)
            if lengths is None:
                S = new
                o[:, j] = y
            else:
                live = (lengths > j)[:, None, None]
                S = torch.where(live[..., None], new, S)
                o[:, j] = torch.where(live, y, o[:, j])
        return o.reshape(n, t, heads * dv), S

    if case["kind"] == "attend":
        o, S = recurrence(s["qkv"], s["decay"], case["dk"] ** -0.5, s["lengths"], s["state_in"], case["heads"],
                           case["dk"], case["dv"], s["out"])
        return [o] if s["state_out"] is None else [o, S]
    if case["kind"] == "step":
        at = s["slots"].long()
        o, S = recurrence(s["qkv"], s["decay"], case["dk"] ** -0.5, None, s["state_in"][at], case["heads"], case["dk"],
                           case["dv"], s["out"])
        state = s["state_out"].double()
        state[at] = S
        return [o, state]
    d = {k: v.double() if isinstance(v, torch.Tensor) else v for k, v in s.items()}

    def norm(x, kind, eps, groups, weight, bias):
        if kind == "none":
            return x
        parts = []
        for p in x.chunk(groups, dim=1):
            var, mean = torch.var_mean(p, dim=1, correction=0, keepdim=True)
            parts.append((p - mean) / (var + eps).sqrt() if kind == "layer" else p / (var + mean ** 2 + eps).sqrt())
        x = torch.cat(parts, dim=1) * weight
        return x if bias is None else x + bias

    u = norm(d["y"], case["post"], POST_EPS, case["groups"], d["post_weight"], d["post_bias"])
    if d["gate"] is not None:
        one = 1.0 / (1.0 + (-d["gate"]).exp())
        u = u * {"linear": d["gate"], "sigmoid": one, "silu": d["gate"] * one}[case["gate"]]
    x = d["x"] + d["scale"] * u
    return [x] if case["pre"] == "none" else [x, norm(x, case["pre"], PRE_EPS, 1, d["pre_weight"], d["pre_bias"])]


def work(case):
    e = SIZE[case["prec"]]
    if case["kind"] == "join":
        arrays = 3 + (case["gate"] != "none") + (case["pre"] != "none")
        n = case["positions"] * case["channels"]
        return {"bytes": arrays * e * n + 4.0 * 5 * case["channels"], "flops": 20.0 * n}
    h, dk, dv = case["heads"], case["dk"], case["dv"]
    if case["kind"] == "step":
        n = case["tokens"] * h
        return {"bytes": n * (8.0 * dk * dv + e * (2 * dk + 2 * dv)), "flops": 5.0 * n * dk * dv}
    positions = case["seqs"] * case["length"] * (0.5 if case["ragged"] else 1.0)  # lengths are uniform
    states = 8.0 * case["seqs"] * h * dk * dv if case["state"] else 0.0
    return {"bytes": positions * h * e * (2 * dk + 2 * dv) + states, "flops": positions * h * 4.0 * dk * dv}
