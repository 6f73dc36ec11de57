"""Workloads of the token-major operators: ``ops.linear`` (matrix product with bias, activation and residual in its
epilogue) and ``ops.attention`` (packed sequences of different lengths, grouped heads, causal or not).

Every workload exists twice: as plain torch arithmetic in float32, rounded once at the end (``own`` false), and as the
one call a user of this package makes (``own`` true).  ``exact`` is the definition in float64, written on its own.
"""
from __future__ import annotations

import math
import random

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def _device():
    return torch.device("cuda", torch.cuda.current_device()) if torch.cuda.is_available() else torch.device("cpu")


# ------------------------------------------------------------------------------------------------------- the cases

def _linear(name, rows, features, outputs, dtype, activation="none", residual=False):
    return {"name": name, "op": "linear", "rows": rows, "features": features, "outputs": outputs, "dtype": dtype,
            "activation": activation, "residual": residual}


def _attention(name, sequences, longest_q, longest_k, heads, kv_heads, dim, dtype, causal, ragged, one_buffer=False):
    """``longest_k`` 0: every sequence attends to itself.  ``one_buffer``: q, k and v are slices of one projection."""
    return {"name": name, "op": "attention", "sequences": sequences, "longest_q": longest_q, "longest_k": longest_k,
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "causal": causal, "ragged": ragged,
            "one_buffer": one_buffer}


def listed():
    return [
        # one new token through a square projection: latency and the read of the weights
        _linear("linear_one_row", 1, 4096, 4096, "bf16", "none", True),
        # a batch of new tokens through the widening half of a perceptron: still the read of the weights
        _linear("linear_few_rows", 37, 4096, 16384, "bf16", "silu"),
        # the correlation window of one 640x480 frame (4 levels of 9x9, 324 values a pixel: rows of no 16-byte multiple)
        # into 256 features, as the flow network's motion encoder widens it
        _linear("linear_window", 4800, 324, 256, "f16", "relu"),
        # eight frames' 256 features a pixel at 1/8 resolution through a square layer with its residual, in float32
        _linear("linear_frames", 38400, 256, 256, "f32", "none", True),
        # a long prompt through both halves of a perceptron
        _linear("linear_widen", 16384, 4096, 16384, "bf16", "gelu"),
        _linear("linear_narrow", 8191, 8192, 4096, "f16", "none", True),
        # one new token over a short history: latency
        _attention("attention_one_token", 1, 1, 777, 32, 8, 128, "bf16", True, False),
        # one new token for each of 32 sequences over histories of up to 32768 tokens: the read of the cache
        _attention("attention_long_caches", 32, 1, 32768, 32, 8, 128, "bf16", True, True),
        # a short continuation behind a long history: few rows, many keys
        _attention("attention_continue", 1, 96, 30001, 32, 4, 128, "f16", True, False),
        # the epipolar lines of eight 640x480 stereo pairs at 1/4 resolution, 256 features in four heads: a match lies
        # never right of its pixel
        _attention("attention_lines", 960, 160, 0, 4, 4, 64, "f16", True, False),
        # all pixels of one 640x480 frame at 1/8 resolution among themselves, in float32
        _attention("attention_frame", 1, 4800, 0, 4, 4, 64, "f32", False, False),
        # prompts of different lengths packed behind one another, straight from their fused projection
        _attention("attention_prompts", 8, 8192, 0, 32, 8, 128, "bf16", True, True, True),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.5)))))))


def _odd_or_round(rng, n, step):
    """Half of the sizes as drawn, half at a multiple of ``step``."""
    return n if rng.random() < 0.5 else max(step, n // step * step)


def draw(rng):
    """One more case.  float32 runs on a sixteenth of the 16-bit matrix rate, so its cases get a sixteenth of the work."""
    dearest = {op: max(work(c)["flops"] for c in listed() if c["op"] == op) for op in ("linear", "attention")}
    most_bytes = {op: max(work(c)["bytes"] for c in listed() if c["op"] == op) for op in ("linear", "attention")}
    op = rng.choice(["linear", "attention"])
    while True:
        dtype = rng.choice(["bf16", "bf16", "f16", "f16", "f32"])
        if op == "linear":
            case = {"op": op, "rows": _log_int(rng, 1, 16384),
                    "features": _odd_or_round(rng, _log_int(rng, 24, 8192), 8),
                    "outputs": _odd_or_round(rng, _log_int(rng, 24, 16384), 8), "dtype": dtype,
                    "activation": rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"]), "residual": rng.random() < 0.5}
        else:
            group, kv_heads = rng.choice([1, 1, 2, 4, 8]), rng.choice([1, 2, 4, 8])
            form = rng.choice(["token", "continue", "self", "self"])
            longest_q = {"token": 1, "continue": _log_int(rng, 2, 256), "self": _log_int(rng, 2, 8192)}[form]
            longest_k = 0 if form == "self" else max(longest_q, _log_int(rng, 16, 32768))
            case = {"op": op, "sequences": _log_int(rng, 1, 64), "longest_q": longest_q, "longest_k": longest_k,
                    "heads": group * kv_heads, "kv_heads": kv_heads, "dim": rng.choice([32, 64, 64, 72, 96, 128, 128, 256]),
                    "dtype": dtype, "causal": rng.random() < 0.7, "ragged": rng.random() < 0.7,
                    "one_buffer": form == "self" and rng.random() < 0.5}
        share = 16 if dtype == "f32" else 1
        w = work(case)
        if w["flops"] * share <= dearest[op] and w["bytes"] <= most_bytes[op]:
            return case


def _lengths(case):
    """(query lengths, key lengths) of the case's sequences, from the case alone."""
    n, q, k = case["sequences"], case["longest_q"], case["longest_k"]
    rng = random.Random(n * 1000003 + q * 1009 + k)
    qs = [q if (i == 0 or not case["ragged"]) else rng.randint(1, q) for i in range(n)]
    if k == 0:
        return qs, list(qs)
    return qs, [k if (i == 0 or not case["ragged"]) else rng.randint(min(qs[i], k), k) for i in range(n)]


def work(case):
    e = _BYTES[case["dtype"]]
    if case["op"] == "linear":
        m, c, k = case["rows"], case["features"], case["outputs"]
        return {"bytes": e * (m * c + k * c + m * k * (2 if case["residual"] else 1)) + 4 * k, "flops": 2 * m * c * k}
    qs, ks = _lengths(case)
    pairs = 0
    for a, b in zip(qs, ks):
        # row i of a sees the keys 0 .. i + b - a
        pairs += (a * (b - a) + a * (a + 1) // 2) if case["causal"] else a * b
    d = case["dim"]
    return {"bytes": e * d * (2 * sum(qs) * case["heads"] + 2 * sum(ks) * case["kv_heads"]) + 8 * (len(qs) + 1),
            "flops": 4 * d * case["heads"] * pairs}


# ------------------------------------------------------------------------------------------------------ the inputs

def prepare(case, seed):
    dev, dt = _device(), _TYPES[case["dtype"]]
    gen = torch.Generator(device=dev).manual_seed(int(seed) % (2 ** 63))

    def normal(*shape, scale=1.0, dtype=dt):
        return (torch.randn(*shape, generator=gen, device=dev, dtype=torch.float32) * scale).to(dtype)

    if case["op"] == "linear":
        m, c, k = case["rows"], case["features"], case["outputs"]
        return {"case": case, "x": normal(m, c), "weight": normal(k, c, scale=c ** -0.5),
                "bias": normal(k, scale=0.1, dtype=torch.float32), "residual": normal(m, k) if case["residual"] else None}
    qs, ks = _lengths(case)
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    if case["one_buffer"]:
        qkv = normal(sum(qs), h + 2 * hk, d)
        q, k, v = qkv[:, :h], qkv[:, h:h + hk], qkv[:, h + hk:]
    else:
        q, k, v = normal(sum(qs), h, d), normal(sum(ks), hk, d), normal(sum(ks), hk, d)

    def offsets(lengths):
        return torch.tensor([0] + lengths, dtype=torch.int64).cumsum(0).to(torch.int32).to(dev)

    return {"case": case, "q": q, "k": k, "v": v, "q_lengths": qs, "k_lengths": ks, "q_offsets": offsets(qs), "k_offsets": offsets(ks)}


# -------------------------------------------------------------------------------------------------- one plain pass

def _activate(z, name):
    if name == "relu":
        return torch.clamp(z, min=0.0)
    if name == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if name == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)))
    if name == "silu":
        return z / (1.0 + torch.exp(-z))
    return z


def _plain_linear(s):
    y = _activate(torch.matmul(s["x"].float(), s["weight"].float().t()) + s["bias"], s["case"]["activation"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(s["x"].dtype)


def _plain_attention(s):
    """Sequences of equal lengths are taken together; scores, softmax and the weighted sum each as they are written."""
    case, q, k, v = s["case"], s["q"], s["k"], s["v"]
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    out = torch.empty(q.shape, device=q.device, dtype=q.dtype)
    groups, q0, k0 = {}, 0, 0
    for lq, lk in zip(s["q_lengths"], s["k_lengths"]):
        groups.setdefault((lq, lk), []).append((q0, k0))
        q0, k0 = q0 + lq, k0 + lk
    for (lq, lk), starts in groups.items():
        n = len(starts)
        if n == 1:
            rows_q, rows_k = slice(starts[0][0], starts[0][0] + lq), slice(starts[0][1], starts[0][1] + lk)
        else:
            rows_q = (torch.tensor([a for a, _ in starts]).to(q.device)[:, None] + torch.arange(lq, device=q.device)).reshape(-1)
            rows_k = (torch.tensor([b for _, b in starts]).to(q.device)[:, None] + torch.arange(lk, device=q.device)).reshape(-1)
        # (n, hk, group, lq, d) against (n, hk, 1, lk, d)
        qg = q[rows_q].float().reshape(n, lq, hk, h // hk, d).permute(0, 2, 3, 1, 4).reshape(n * hk, h // hk * lq, d).contiguous()
        kg = k[rows_k].float().reshape(n, lk, hk, d).permute(0, 2, 3, 1).reshape(n * hk, d, lk).contiguous()
        vg = v[rows_k].float().reshape(n, lk, hk, d).permute(0, 2, 1, 3).reshape(n * hk, lk, d).contiguous()
        scores = torch.matmul(qg, kg) * d ** -0.5
        if case["causal"]:
            last = torch.arange(lq, device=q.device) + (lk - lq)
            hidden = torch.arange(lk, device=q.device)[None, :] > last[:, None]
            scores = scores.reshape(n * hk, h // hk, lq, lk).masked_fill(hidden, float("-inf")).reshape(n * hk, h // hk * lq, lk)
        weights = torch.exp(scores - scores.amax(dim=-1, keepdim=True))
        mean = torch.matmul(weights, vg) / weights.sum(dim=-1, keepdim=True)
        out[rows_q] = mean.reshape(n, hk, h // hk, lq, d).permute(0, 3, 1, 2, 4).reshape(n * lq, h, d).to(q.dtype)
    return out


def run(state):
    case = state["case"]
    if own:
        from visual_odometry_amd import ops
        if case["op"] == "linear":
            activation = None if case["activation"] == "none" else case["activation"]
            return ops.linear(state["x"], state["weight"], state["bias"], activation=activation, residual=state["residual"])
        return ops.attention(state["q"], state["k"], state["v"], state["q_offsets"], state["k_offsets"], causal=case["causal"])
    return _plain_linear(state) if case["op"] == "linear" else _plain_attention(state)


# ------------------------------------------------------------------------------------------- the definition, 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "linear":
        w = s["weight"].double()
        parts = []
        for x in s["x"].split(2048):
            z = x.double().matmul(w.t().contiguous())
            z += s["bias"].double()
            a = case["activation"]
            if a == "relu":
                z = torch.where(z > 0, z, torch.zeros_like(z))
            elif a == "gelu":                                    # z times the normal distribution function
                z = z * torch.special.ndtr(z)
            elif a == "gelu_tanh":                               # (1 + tanh u) / 2 = 1 / (1 + exp(-2u))
                z = z * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (z + 0.044715 * z ** 3))
            elif a == "silu":
                z = z * torch.sigmoid(z)
            parts.append(z)
        y = torch.cat(parts)
        return y if s["residual"] is None else y + s["residual"].double()
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    out = torch.zeros((sum(s["q_lengths"]), h, d), device=s["q"].device, dtype=torch.float64)
    a = b = 0
    for lq, lk in zip(s["q_lengths"], s["k_lengths"]):
        q = s["q"][a:a + lq].double().transpose(0, 1).contiguous()                     # (h, lq, d)
        k = s["k"][b:b + lk].double().permute(1, 2, 0).contiguous()                    # (hk, d, lk)
        v = s["v"][b:b + lk].double().transpose(0, 1).contiguous()                     # (hk, lk, d)
        per = h // hk
        step = max(1, 2 ** 26 // max(1, per * lk))                                     # rows at a time: at most 2^26 scores
        for g in range(hk):
            for r in range(0, lq, step):
                n = min(step, lq - r)
                z = q[g * per:(g + 1) * per, r:r + n].reshape(per * n, d).matmul(k[g]).view(per, n, lk) / math.sqrt(d)
                if case["causal"]:
                    below = torch.ones((n, lk), device=z.device, dtype=torch.bool).tril(lk - lq + r)
                    z = torch.where(below, z, torch.full_like(z, -math.inf))
                p = torch.exp(z - torch.logsumexp(z, dim=-1, keepdim=True))
                out[a + r:a + r + n, g * per:(g + 1) * per] = p.view(per * n, lk).matmul(v[g]).view(per, n, d).transpose(0, 1)
        a, b = a + lq, b + lk
    return out
