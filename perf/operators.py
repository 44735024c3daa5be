"""Timed cases of the streaming operators: rotary positions and linear attention with a
decay for each head (its chunked form for prompts and its recurrent form for single tokens).

``run`` computes one pass: with ``own`` false in elementary torch operations in FP32 (angles
and decay sums in 64 bits), with ``own`` true through ``trifusion_b200``.
"""

import math
import os
import sys

import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "trifusion-fp-kernel_b200")
_TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _framework():
    if "trifusion_b200" not in sys.modules and _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import trifusion_b200

    return trifusion_b200


# ---- cases ---------------------------------------------------------------------------------

def _rotary(name, batch, time, heads, kv_heads, dim, rotary_dim, layout, dtype, scaling, first, packed):
    """``first``: the first position of row 0 (row b starts b * 977 later); ``packed``: q and k are
    views of one projection row [q heads, k heads, v heads]."""
    return dict(name=name, op="rotary", batch=batch, time=time, heads=heads, kv_heads=kv_heads, dim=dim,
                rotary_dim=rotary_dim, layout=layout, dtype=dtype, scaling=scaling, first=first, packed=packed)


def _prompt(name, batch, time, heads, groups, n, p, ragged, carried):
    """``ragged``: rows of different lengths; ``carried``: a state from an earlier piece of the
    prompt goes in, in slots of a pool, and comes out."""
    return dict(name=name, op="prompt", batch=batch, time=time, heads=heads, groups=groups, n=n, p=p,
                ragged=ragged, carried=carried, dtype="bf16")


def _step(name, batch, padded, heads, groups, n, p, dtype):
    """``padded``: rows behind the live ones whose slot is -1 (a batch padded for a captured graph)."""
    return dict(name=name, op="step", batch=batch, padded=padded, heads=heads, groups=groups, n=n, p=p, dtype=dtype)


def listed():
    return [
        # One new token for each of 48 streams at far positions, frequencies scaled by parts.
        _rotary("rotary step", 48, 1, 32, 8, 128, 128, "half", "bf16", "parts", 70001, False),
        # The pooled attention's heads (6 x 64) over a padded batch of odd length, FP32.
        _rotary("rotary f32 odd", 16, 451, 6, 6, 64, 64, "interleaved", "f32", "none", 0, False),
        # Long clips (3600 steps), half of each head rotated, read from the projection's rows.
        _rotary("rotary partial", 2, 3600, 12, 12, 64, 32, "interleaved", "bf16", "linear", 3, True),
        # A long prompt of shared key heads.
        _rotary("rotary long", 1, 32768, 32, 8, 128, 128, "half", "bf16", "base", 0, True),
        # A very short clip: one tile, little to share out.
        _prompt("prompt 26", 2, 26, 4, 1, 128, 64, False, False),
        # The batch of 4 s clips of the recurrence benchmark, lengths 120..200.
        _prompt("prompt 16x200", 16, 200, 12, 1, 128, 64, True, False),
        # The 72 s clips of the recurrence benchmark: few rows, long.
        _prompt("prompt 2x3600", 2, 3600, 12, 1, 128, 64, True, True),
        # One long stream: few heads, every head with its own keys, state carried on.
        _prompt("prompt 1x32768", 1, 32768, 16, 16, 128, 128, False, True),
        # Many rows of an odd length, small heads, keys shared by four heads.
        _prompt("prompt 8x4097", 8, 4097, 32, 8, 64, 64, True, True),
        # One stream, one token: the latency of a step.
        _step("step 1", 1, 0, 12, 1, 128, 64, "bf16"),
        # FP32 operands, a batch padded with rows that have no slot.
        _step("step f32 padded", 19, 13, 12, 12, 64, 128, "f32"),
        # A full serving batch, the states alone are 268 MB read and written.
        _step("step 64", 64, 0, 32, 8, 128, 128, "bf16"),
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["rotary", "prompt", "prompt", "step"])
    if op == "rotary":
        heads = rng.randint(1, 32)
        kv = rng.choice([h for h in range(1, heads + 1) if heads % h == 0])
        dim = rng.choice([32, 64, 80, 96, 128, 256])
        rotary_dim = rng.choice([dim, dim, dim // 2])
        dtype = rng.choice(["bf16", "bf16", "f32"])
        batch = _log(rng, 1, 64)
        most = 32768 * 40 * 128 // (batch * (heads + kv) * dim * (2 if dtype == "f32" else 1))
        time = 1 if rng.random() < 0.25 else _log(rng, 2, max(2, min(32768, most)))
        c = _rotary("", batch, time, heads, kv, dim, rotary_dim, rng.choice(["half", "interleaved"]), dtype,
                    rng.choice(["none", "linear", "base", "parts"]), _log(rng, 1, 1000000) - 1, rng.random() < 0.5)
    elif op == "prompt":
        heads = rng.randint(1, 32)
        groups = rng.choice([h for h in range(1, heads + 1) if heads % h == 0])
        n, p = rng.choice([32, 64, 96, 128]), rng.choice([32, 64, 96, 128])
        batch = _log(rng, 1, 32)
        most = 32768 * 16 * 128 * 4 // (batch * 2 * (groups * n + heads * p))
        c = _prompt("", batch, _log(rng, 1, max(1, min(32768, most))), heads, groups, n, p, rng.random() < 0.5,
                    rng.random() < 0.5)
    else:
        heads = rng.randint(1, 32)
        groups = rng.choice([h for h in range(1, heads + 1) if heads % h == 0])
        n, p = rng.choice([32, 64, 96, 128]), rng.choice([32, 64, 96, 128])
        c = _step("", _log(rng, 1, 64), rng.choice([0, 0, rng.randint(1, 16)]), heads, groups, n, p,
                  rng.choice(["bf16", "bf16", "f32"]))
    del c["name"]
    return c


# ---- inputs --------------------------------------------------------------------------------

_SCALE, _TRAINED = 8.0, 4096  # of the long-context scalings


def _frequencies(rotary_dim, scaling):
    """(inverse frequencies [rotary_dim / 2] in 64 bits, amplitude)."""
    base = 10000.0
    if scaling == "base" and rotary_dim > 2:
        base *= _SCALE ** (rotary_dim / (rotary_dim - 2))
    i = torch.arange(0, rotary_dim, 2, dtype=torch.float64)
    f = base ** (-i / rotary_dim)
    if scaling == "linear":
        return f / _SCALE, 1.0
    if scaling == "parts":
        # Full turns within the trained length: below 1 interpolated, above 32 kept, blended between.
        turns = _TRAINED * f / (2 * math.pi)
        keep = ((turns - 1.0) / 31.0).clamp(0, 1)
        return f * keep + f / _SCALE * (1 - keep), 0.1 * math.log(_SCALE) + 1.0
    return f, 1.0


def _lengths(case):
    """Row lengths of a ragged batch: from three fifths of the time to all of it, the first row full."""
    t = case["time"]
    return [t - (2 * t * i) // (5 * case["batch"]) for i in range(case["batch"])]


def _slots(rows, pool, g):
    return torch.randperm(pool, generator=g, device="cuda")[:rows]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _TYPES[case["dtype"]]
    s = {"case": case}

    def randn(*shape, dtype=dtype, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)

    b = case["batch"]
    if case["op"] == "rotary":
        t, h, kv, d = case["time"], case["heads"], case["kv_heads"], case["dim"]
        if case["packed"]:
            rows = randn(b, t, (h + 2 * kv) * d)
            s["q"] = rows[..., : h * d].unflatten(-1, (h, d))
            s["k"] = rows[..., h * d: (h + kv) * d].unflatten(-1, (kv, d))
        else:
            s["q"], s["k"] = randn(b, t, h, d), randn(b, t, kv, d)
        start = case["first"] + 977 * torch.arange(b, device="cuda")
        s["positions"] = start[:, None] + torch.arange(t, device="cuda")
        f, s["amplitude"] = _frequencies(case["rotary_dim"], case["scaling"])
        s["inv_freq"] = f.cuda()
        return s
    h, hq, n, p = case["heads"], case["groups"], case["n"], case["p"]
    # Decay rates per head from slow (a memory of some hundred tokens) to fast, as the recurrence's
    # benchmark draws them: -dt * A with dt log-uniform in [1e-3, 1e-1] and A in [1, 16].
    rate = torch.exp(torch.rand(h, generator=g, device="cuda") * math.log(16.0))
    if case["op"] == "prompt":
        t = case["time"]
        s["q"], s["k"], s["v"] = randn(b, t, hq, n), randn(b, t, hq, n), randn(b, t, h, p)
        dt = torch.exp(math.log(1e-3) + math.log(100.0) * torch.rand(b, h, t, generator=g, device="cuda"))
        s["decay"] = -rate[None, :, None] * dt
        s["lengths"] = torch.tensor(_lengths(case), device="cuda") if case["ragged"] else None
        if case["carried"]:
            pool = b + 3
            s["state"] = randn(pool, h, n, p, dtype=torch.float32, scale=4.0)
            s["slots"] = _slots(b, pool, g)
        return s
    live, rows = b, b + case["padded"]
    s["q"], s["k"], s["v"] = randn(rows, hq, n), randn(rows, hq, n), randn(rows, h, p)
    s["decay"] = -rate * torch.exp(math.log(1e-3) + math.log(100.0) * torch.rand(rows, h, generator=g, device="cuda"))
    pool = live + 3
    s["state"] = randn(pool, h, n, p, dtype=torch.float32, scale=4.0)
    s["slots"] = torch.cat([_slots(live, pool, g), torch.full((case["padded"],), -1, device="cuda")])
    s["live"] = live
    return s


# ---- one pass ------------------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if own:
        tf = _framework()
        if op == "rotary":
            return tf.apply_rotary(state["q"], state["k"], state["positions"], state["inv_freq"],
                                   layout=state["case"]["layout"], amplitude=state["amplitude"])
        if op == "prompt":
            return tf.linear_attention(state["q"], state["k"], state["v"], state["decay"], state.get("state"),
                                       slots=state.get("slots"), lengths=state["lengths"])
        out = tf.linear_attention_step(state["q"], state["k"], state["v"], state["decay"], state["state"],
                                       slots=state["slots"])
        return out, state["state"]
    return {"rotary": _plain_rotary, "prompt": _plain_prompt, "step": _plain_step}[op](state)


def _plain_rotary(s):
    c = s["case"]
    r = c["rotary_dim"]
    angle = (s["positions"].double()[..., None] * s["inv_freq"])[:, :, None]
    cos, sin = (angle.cos() * s["amplitude"]).float(), (angle.sin() * s["amplitude"]).float()

    def turn(x):
        xf = x.float()
        y = xf.clone()
        if c["layout"] == "half":
            a, z = xf[..., : r // 2], xf[..., r // 2: r]
            y[..., : r // 2], y[..., r // 2: r] = a * cos - z * sin, z * cos + a * sin
        else:
            a, z = xf[..., 0:r:2], xf[..., 1:r:2]
            y[..., 0:r:2], y[..., 1:r:2] = a * cos - z * sin, z * cos + a * sin
        return y.to(x.dtype)

    return turn(s["q"]), turn(s["k"])


_CHUNK = 256


def _plain_prompt(s):
    """Chunks of 256 steps: scores within a chunk with the decay between two steps, one state sum
    for each chunk, and the chunks' states joined by the matrix of decays between chunks."""
    c = s["case"]
    b, t, h, hq, n, p = (c[x] for x in ("batch", "time", "heads", "groups", "n", "p"))
    size = min(_CHUNK, t)
    m = (t + size - 1) // size
    pad = m * size - t
    at = torch.arange(m * size, device="cuda")
    end = s["lengths"] if s["lengths"] is not None else torch.full((b,), t, device="cuda")
    live = at < end[:, None]                                                    # [B, M*C]

    def rows(x, heads):  # [B, T, heads, w] -> [B, H, M, C, w], zero past each length
        x = torch.nn.functional.pad(x.float(), (0, 0, 0, 0, 0, pad))
        x = torch.where(live[:, :, None, None], x, 0.0).transpose(1, 2).unflatten(2, (m, size))
        return x if heads == h else x.repeat_interleave(h // heads, dim=1)

    q, k, v = rows(s["q"], hq), rows(s["k"], hq), rows(s["v"], h)
    g = torch.where(live[:, None], torch.nn.functional.pad(s["decay"], (0, pad)), 0.0)
    sums = g.double().cumsum(-1).unflatten(2, (m, size))                        # from the first step on
    ahead = at[:size, None] >= at[None, :size]
    within = torch.where(ahead, sums[..., :, None] - sums[..., None, :], -math.inf).float().exp()
    out = ((q @ k.transpose(-1, -2)) * within) @ v
    last = sums[..., -1:]                                                       # [B, H, M, 1]
    added = (k * (last - sums).float().exp()[..., None]).transpose(-1, -2) @ v  # [B, H, M, N, P]
    # State before chunk i: sum over j < i of e^(last[i-1] - last[j]) added[j], and the carried one.
    before = torch.nn.functional.pad(last[..., 0], (1, 0))                      # [B, H, M+1]
    order = torch.arange(m + 1, device="cuda")
    between = torch.where(order[:, None] > order[None, :m], before[..., :, None] - last[..., None, :, 0],
                          -math.inf).float().exp()                              # [B, H, M+1, M]
    states = (between @ added.flatten(-2)).unflatten(-1, (n, p))                # [B, H, M+1, N, P]
    if "state" in s:
        states = states + before.float().exp()[..., None, None] * s["state"][s["slots"]][:, :, None]
    out = out + (q * (sums - before[..., :m, None]).float().exp()[..., None]) @ states[:, :, :m]
    out = (out * n ** -0.5).flatten(2, 3)[:, :, :t].transpose(1, 2).to(s["v"].dtype)
    if "state" not in s:
        return out, states[:, :, m]
    s["state"][s["slots"]] = states[:, :, m]
    return out, s["state"]


def _plain_step(s):
    c, live = s["case"], s["live"]
    share = c["heads"] // c["groups"]
    slots = s["slots"][:live]
    q, k = (s[x][:live].float().repeat_interleave(share, dim=1) for x in ("q", "k"))
    new = s["state"][slots] * s["decay"][:live].exp()[..., None, None]
    new = new + k[..., :, None] * s["v"][:live].float()[..., None, :]
    s["state"][slots] = new
    out = torch.zeros_like(s["v"])
    out[:live] = ((q[..., :, None] * new).sum(-2) * c["n"] ** -0.5).to(out.dtype)
    return out, s["state"]


# ---- what a pass cannot do without -----------------------------------------------------------

def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    b = case["batch"]
    if case["op"] == "rotary":
        tokens = b * case["time"]
        values = tokens * (case["heads"] + case["kv_heads"]) * case["dim"]
        return {"bytes": 2 * size * values + 8 * tokens + 4 * case["rotary_dim"],
                "flops": 3 * tokens * (case["heads"] + case["kv_heads"]) * case["rotary_dim"]}
    h, hq, n, p = case["heads"], case["groups"], case["n"], case["p"]
    states = 4 * b * h * n * p
    if case["op"] == "prompt":
        tokens = sum(_lengths(case)) if case["ragged"] else b * case["time"]
        read = tokens * (2 * size * hq * n + size * h * p + 4 * h)
        write = b * case["time"] * size * h * p
        states *= 2 if case["carried"] else 1
        return {"bytes": read + write + states, "flops": 4 * tokens * h * n * p}
    rows = b + case["padded"]
    return {"bytes": b * (2 * size * hq * n + size * h * p + 4 * h) + rows * (size * h * p + 8) + 2 * states,
            "flops": 5 * b * h * n * p}


# ---- the definitions in 64 bits ----------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        r, f = case["rotary_dim"], s["inv_freq"]
        turn = torch.polar(torch.full_like(f, s["amplitude"]).expand(*s["positions"].shape, -1).contiguous(),
                           s["positions"].double()[..., None] * f)[:, :, None]
        done = []
        for x in (s["q"], s["k"]):
            y, head = x.double(), x[..., :r].double()
            if case["layout"] == "half":
                z = torch.complex(head[..., : r // 2], head[..., r // 2:]) * turn
                z = torch.cat([z.real, z.imag], -1)
            else:
                z = torch.view_as_real(torch.view_as_complex(head.unflatten(-1, (r // 2, 2)).contiguous()) * turn)
                z = z.flatten(-2)
            done.append(torch.cat([z, y[..., r:]], -1))
        return tuple(done)
    h, n, p = case["heads"], case["n"], case["p"]
    share = h // case["groups"]
    if case["op"] == "prompt":
        b, t = case["batch"], case["time"]
        state = (s["state"][s["slots"]] if "state" in s else torch.zeros(b, h, n, p, device="cuda")).double()
        out = torch.zeros(b, t, h, p, dtype=torch.float64, device="cuda")
        lengths = _lengths(case) if case["ragged"] else [t] * b  # the longest first
        factor = s["decay"].double().exp()
        for i in range(t):
            rows = sum(length > i for length in lengths)
            q, k = (s[x][:rows, i].double().repeat_interleave(share, dim=1) for x in ("q", "k"))
            now = state[:rows]
            now.mul_(factor[:rows, :, i, None, None])
            now.add_(k[..., :, None] * s["v"][:rows, i].double()[..., None, :])
            torch.matmul(q[..., None, :], now, out=out[:rows, i].unsqueeze(-2))
        out *= n ** -0.5
        if "state" not in s:
            return out, state
        pool = s["state"].double()
        pool[s["slots"]] = state
        return out, pool
    pool = s["state"].double()
    out = torch.zeros(s["v"].shape, dtype=torch.float64, device="cuda")
    for row, slot in enumerate(s["slots"][: case["batch"]].tolist()):
        for head in range(h):
            k, q = (s[x][row, head // share].double() for x in ("k", "q"))
            pool[slot, head] = pool[slot, head] * s["decay"][row, head].double().exp() + torch.outer(k, s["v"][row, head].double())
            out[row, head] = n ** -0.5 * (q @ pool[slot, head])
    return out, pool
