"""Cases of the general int8 products and of the query / key norm with rotation.

Three operators, reached through ``arctic_embed_s_int8.Engine``:

``matmul_i8``      int8 activations with a scale for each token, int8 weights with a scale for each output channel:
                   out[m, n] = (sum_k a[m, k] w[n, k]) * (a_scale[m] * w_scale[n]) + bias[n]
``linear_i8``      the same product from float activations, which are smoothed and quantized per token on the way:
                   y = x * inv_smooth,  top = max_k |y|,  a = round_half_even(y * (127 / top)),  a_scale = top / 127
``qk_norm_rope``   RMS norm of every query and key head and the rotation of its first `rotary` dims, in one pass:
                   y = x / sqrt(mean(x^2) + eps) * weight,  (y_i, y_j) -> (y_i c - y_j s, y_j c + y_i s)

``run`` computes them in elementary torch operations in 32 bits, or, where ``own`` is true, by the framework's calls.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"i8": 1, "f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-6
TINY = 2.0 ** -119  # a token whose largest |y| is below this quantizes to zero: 127 / top would not be finite
MOST_WORK = 16384 * 8192 * 4096  # products of the largest listed case
MOST_HEADS = 16384 * 40 * 128    # elements of the largest listed norm and rotation

_engine = None


def listed():
    return [
        # one token through the encoder's own QKV projection: latency
        {"name": "matmul-1x1152x384", "op": "matmul", "m": 1, "n": 1152, "k": 384, "out": "f32", "bias": True},
        # a few rows against the word table as an output matrix: a column count that no tile divides
        {"name": "matmul-33x30522x384", "op": "matmul", "m": 33, "n": 30522, "k": 384, "out": "f32", "bias": False},
        # the benchmark's batch of 512 sequences of 128 tokens through the FFN's first projection
        {"name": "matmul-65536x1536x384", "op": "matmul", "m": 65536, "n": 1536, "k": 384, "out": "bf16", "bias": True},
        # a long batch through a projection of a larger encoder: the tensor cores' rate
        {"name": "matmul-16384x8192x4096", "op": "matmul", "m": 16384, "n": 8192, "k": 4096, "out": "bf16", "bias": False},
        # one token of a larger model, activations as they come: the weights' bytes
        {"name": "linear-1x4096x4096", "op": "linear", "m": 1, "n": 4096, "k": 4096, "x": "bf16", "out": "bf16",
         "bias": True, "smooth": False},
        # one full-length sequence through the encoder's FFN, float in and out as its row kernels keep them
        {"name": "linear-512x384x1536", "op": "linear", "m": 512, "n": 384, "k": 1536, "x": "f32", "out": "f32",
         "bias": True, "smooth": True},
        # odd everything: rows, channels and a depth that ends inside a 16-byte piece
        {"name": "linear-509x1001x1003", "op": "linear", "m": 509, "n": 1001, "k": 1003, "x": "f16", "out": "f16",
         "bias": True, "smooth": False},
        # a long batch of a larger model with smoothing
        {"name": "linear-16384x4096x4096", "op": "linear", "m": 16384, "n": 4096, "k": 4096, "x": "bf16", "out": "bf16",
         "bias": True, "smooth": True},
        # one token, grouped heads
        {"name": "qk-1x32+8x128", "op": "qk", "tokens": 1, "q_heads": 32, "k_heads": 8, "dim": 128, "rotary": 128,
         "type": "bf16", "pairs": "halves", "seqs": 0, "rows": 32768},
        # an odd count of tokens, heads of 80 with 64 rotated dims in neighbouring pairs
        {"name": "qk-777x10+5x80", "op": "qk", "tokens": 777, "q_heads": 10, "k_heads": 5, "dim": 80, "rotary": 64,
         "type": "f16", "pairs": "neighbours", "seqs": 0, "rows": 4096},
        # the benchmark's batch in the encoder's own head layout, ragged sequences that restart at position 0
        {"name": "qk-65536x12+12x32", "op": "qk", "tokens": 65536, "q_heads": 12, "k_heads": 12, "dim": 32, "rotary": 32,
         "type": "f32", "pairs": "halves", "seqs": 512, "rows": 512},
        # a long batch of a larger model
        {"name": "qk-16384x32+8x128", "op": "qk", "tokens": 16384, "q_heads": 32, "k_heads": 8, "dim": 128,
         "rotary": 128, "type": "bf16", "pairs": "halves", "seqs": 0, "rows": 32768},
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _size(rng, lo, hi, step):
    """Of a model's own kind (a multiple of `step`) three times in four, any number otherwise."""
    v = _spread(rng, lo, hi)
    return v if rng.random() < 0.25 else max(step, v // step * step)


def draw(rng):
    kind = rng.choice(["matmul", "linear", "qk"])
    types = ["f32", "f16", "bf16"]
    if kind == "qk":
        q = rng.choice([1, 4, 8, 12, 15, 16, 32])
        kv = rng.choice([h for h in (1, 2, 3, 4, 5, 8, 12, 16, 32) if q % h == 0])
        dim = rng.choice([32, 64, 80, 96, 128, 128, 256])
        tokens = _spread(rng, 1, max(1, min(65536, MOST_HEADS // ((q + kv) * dim))))
        seqs = rng.choice([0, min(tokens, _spread(rng, 1, 512))])
        return {"op": "qk", "tokens": tokens, "q_heads": q, "k_heads": kv, "dim": dim,
                "rotary": rng.choice([dim, dim, dim // 2, dim // 4]), "type": rng.choice(types),
                "pairs": rng.choice(["halves", "halves", "neighbours"]), "seqs": seqs,
                "rows": max(tokens if seqs else 1, rng.choice([512, 4096, 32768]))}
    n, k = _size(rng, 64, 32768, 64), _size(rng, 64, 8192, 64)
    m = _spread(rng, 1, max(1, min(65536, MOST_WORK // 2 // (n * k), 2 ** 28 // n)))
    c = {"op": kind, "m": m, "n": n, "k": k, "out": rng.choice(types), "bias": rng.random() < 0.5}
    if kind == "linear":
        c.update(x=rng.choice(types), smooth=rng.random() < 0.5)
    return c


def _rows(values, step):
    """The same matrix in rows that start at multiples of `step` elements, as a program lays out what it keeps."""
    r, c = values.shape
    if c % step == 0:
        return values
    wide = torch.zeros(r, -(-c // step) * step, dtype=values.dtype, device=values.device)
    wide[:, :c] = values
    return wide[:, :c]


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*size):
        return torch.randn(*size, generator=g, device="cuda")

    def uniform(*size):
        return torch.rand(*size, generator=g, device="cuda")

    if case["op"] == "qk":
        t, hq, hk, d, r = (case[x] for x in ("tokens", "q_heads", "k_heads", "dim", "rotary"))
        # a packed projection, queries | keys | values, of which the operator reads the first two
        qkv = (normal(t, (hq + 2 * hk) * d) * torch.exp(normal(t, 1) * 0.5)).to(TYPES[case["type"]])
        angle = torch.outer(torch.arange(case["rows"], dtype=torch.float64, device="cuda"),
                            10000.0 ** (-torch.arange(0, r, 2, dtype=torch.float64, device="cuda") / r))
        s = {"q": qkv[:, :hq * d].view(t, hq, d), "k": qkv[:, hq * d:(hq + hk) * d].view(t, hk, d),
             "q_weight": 1 + 0.2 * normal(d), "k_weight": 1 + 0.2 * normal(d),
             "table": torch.cat([angle.cos(), angle.sin()], 1).float(), "positions": None, "cu": None}
        if case["seqs"]:
            # sequence i ends inside the i-th of equal steps, so lengths run from none to twice the step
            step = t / case["seqs"]
            cut = ((torch.arange(case["seqs"] - 1, device="cuda") + uniform(case["seqs"] - 1).double()) * step).long()
            ends = torch.tensor([0], device="cuda"), torch.tensor([t], device="cuda")
            s["cu"] = torch.cat([ends[0], cut, ends[1]]).int()
        else:
            s["positions"] = (uniform(t) * case["rows"]).long().clamp(max=case["rows"] - 1).int()
        return s
    m, n, k = case["m"], case["n"], case["k"]
    s = {"w": _rows((normal(n, k) * 40).round_().clamp_(-127, 127).to(torch.int8), 16),
         "w_scale": 5e-4 + 1e-3 * uniform(n), "bias": 0.05 * normal(n) if case["bias"] else None}
    if case["op"] == "matmul":
        s["a"] = _rows((normal(m, k) * 32).round_().clamp_(-127, 127).to(torch.int8), 16)
        s["a_scale"] = 5e-3 + 2e-2 * uniform(m)
    else:
        # channels of unlike size, as the activations of an encoder have them
        s["x"] = _rows((normal(m, k) * torch.exp(0.7 * normal(k))).to(TYPES[case["x"]]), 8)
        s["inv_smooth"] = torch.exp(0.5 * normal(k)) if case["smooth"] else None
    return s


def prepare(case, seed):
    global _engine
    state = {"case": case, **_inputs(case, seed)}
    if own:
        if _engine is None:
            import os
            import sys

            sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                            "snowflake-arctic-embed-s-rust_b200"))
            from arctic_embed_s_int8 import Engine

            _engine = Engine(0)
        state["engine"] = _engine
    return state


def _product(a, a_scale, w, w_scale, bias, out):
    y = (a @ w.float().t()) * (a_scale[:, None] * w_scale)
    if bias is not None:
        y = y + bias
    return y.to(out)


def _plain_qk(x, weight, cos, sin, neighbours):
    y = x.float()
    y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + EPS) * weight
    r = 2 * cos.shape[-1]
    rot, rest = y[..., :r], y[..., r:]
    c, s = cos[:, None], sin[:, None]
    if neighbours:
        a, b = rot[..., 0::2], rot[..., 1::2]
        rot = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    else:
        a, b = rot[..., :r // 2], rot[..., r // 2:]
        rot = torch.cat([a * c - b * s, b * c + a * s], -1)
    return torch.cat([rot, rest], -1).to(x.dtype)


def run(state):
    case = state["case"]
    if case["op"] == "qk":
        q, k = state["q"], state["k"]
        neighbours = case["pairs"] == "neighbours"
        if own:
            q_out, k_out = torch.empty_like(q, memory_format=torch.contiguous_format), torch.empty_like(
                k, memory_format=torch.contiguous_format)
            state["engine"].qk_norm_rope(q, k, q_out, k_out, state["table"], positions=state["positions"],
                                         cu=state["cu"], q_weight=state["q_weight"], k_weight=state["k_weight"],
                                         eps=EPS, neighbours=neighbours)
            return {"q": q_out, "k": k_out}
        at = state["positions"]
        if at is None:
            t = torch.arange(q.shape[0], dtype=torch.int32, device=q.device)
            at = t - state["cu"][torch.searchsorted(state["cu"], t, right=True) - 1]
        cos, sin = state["table"][at.long()].chunk(2, -1)
        return {"q": _plain_qk(q, state["q_weight"], cos, sin, neighbours),
                "k": _plain_qk(k, state["k_weight"], cos, sin, neighbours)}
    out_type = TYPES[case["out"]]
    w, w_scale, bias = state["w"], state["w_scale"], state["bias"]
    if own:
        out = torch.empty(case["m"], case["n"], dtype=out_type, device=w.device)
        if case["op"] == "matmul":
            state["engine"].matmul_i8(state["a"], state["a_scale"], w, w_scale, out, bias=bias)
        else:
            state["engine"].linear_i8(state["x"], w, w_scale, out, bias=bias, inv_smooth=state["inv_smooth"])
        return out
    if case["op"] == "matmul":
        return _product(state["a"].float(), state["a_scale"], w, w_scale, bias, out_type)
    y = state["x"].float()
    if state["inv_smooth"] is not None:
        y = y * state["inv_smooth"]
    top = y.abs().amax(1, keepdim=True)
    most = torch.full_like(top, 127.0)  # as a tensor, so that both quotients are rounded once
    a = (y * torch.where(top >= TINY, most / top, 0.0)).round()
    return _product(a, torch.where(top >= TINY, top / most, 0.0)[:, 0], w, w_scale, bias, out_type)


def work(case):
    if case["op"] == "qk":
        t, d = case["tokens"], case["dim"]
        n = t * (case["q_heads"] + case["k_heads"]) * d
        table = min(t, case["rows"]) * case["rotary"] * 4
        where = 4 * (case["seqs"] + 1 if case["seqs"] else t)
        return {"bytes": 2 * n * BYTES[case["type"]] + table + where + 8 * d, "flops": 8 * n}
    m, n, k = case["m"], case["n"], case["k"]
    rows = m * k * BYTES[case.get("x", "i8")] + (4 * m if case["op"] == "matmul" else 0)
    rows += 4 * k if case.get("smooth") else 0
    return {"bytes": rows + n * k + (8 if case["bias"] else 4) * n + m * n * BYTES[case["out"]], "flops": 2 * m * n * k}


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "qk":
        t = case["tokens"]
        if s["cu"] is not None:
            cu = s["cu"].long()
            at = torch.arange(t, device="cuda") - torch.repeat_interleave(cu[:-1], cu[1:] - cu[:-1])
        else:
            at = s["positions"].long()
        half = case["rotary"] // 2
        turn = torch.complex(s["table"][at, :half].double(), s["table"][at, half:].double())[:, None]

        def one(x, weight):
            y = x.double()
            y = y * (y.square().sum(-1, keepdim=True) / y.shape[-1] + EPS).rsqrt() * weight.double()
            head = y[..., :2 * half]
            if case["pairs"] == "neighbours":
                z = torch.view_as_complex(head.reshape(*head.shape[:-1], half, 2).contiguous()) * turn
                y[..., :2 * half] = torch.view_as_real(z).flatten(-2)
            else:
                z = torch.complex(head[..., :half].contiguous(), head[..., half:].contiguous()) * turn
                y[..., :half], y[..., half:2 * half] = z.real, z.imag
            return y

        return {"q": one(s["q"], s["q_weight"]), "k": one(s["k"], s["k_weight"])}
    if case["op"] == "matmul":
        a, scale = s["a"].double(), s["a_scale"].double()
    else:
        y = s["x"].double()
        if s["inv_smooth"] is not None:
            y *= s["inv_smooth"].double()
        scale = y.abs().max(dim=1).values / 127
        a = torch.where(scale[:, None] > 0, y / scale[:, None], torch.zeros_like(y)).round_()
    out = torch.mm(a, s["w"].double().T)
    out *= scale[:, None]
    out *= s["w_scale"].double()
    return out if s["bias"] is None else out.add_(s["bias"].double())
