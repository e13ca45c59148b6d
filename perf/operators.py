"""The dense path of a transformer layer, as cases to be timed: the product of activations with a
weight and what follows it (bias, activation or gate, residual), rotary positions on the heads of
a packed query / key / value row, and the same with the queries' and keys' norm in front.

``run`` computes a case either in plain torch operations (``own`` false) or through the
framework's compiled kernels (``own`` true): the package builders of ``thompiler.synth`` and
``thompiler.device.DeviceKernel``, as INTEGRATION.md shows them.  A compiled kernel belongs to a
set of sizes and types, so a program keeps one for each and calls it with pointers.
"""

import math
import os
import sys
import tempfile

import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
BYTES = {"f16": 2, "bf16": 2, "f32": 4}


# ---- the cases --------------------------------------------------------------------

def _linear(name, m, n, k, dtype, bias=False, act="", residual=False, gated=False):
    return {"name": name, "op": "linear", "m": m, "n": n, "k": k, "dtype": dtype, "bias": bias, "act": act,
            "residual": residual, "gated": gated}


def _rope(name, b, s, heads, kv, d, rotary, dtype, interleaved=False, values=False, heads_first=False,
          inverse=False, norm=False, table=4096, first=0, padded=0):
    return {"name": name, "op": "qk_norm_rope" if norm else "rope", "b": b, "s": s, "heads": heads, "kv": kv, "d": d,
            "rotary": rotary, "dtype": dtype, "interleaved": interleaved, "values": values,
            "heads_first": heads_first, "inverse": inverse, "table": table, "first": first, "padded": padded}


def listed():
    return [
        # one new token through an attention block's output projection, added to its residual stream
        _linear("linear_one_token", 1, 4096, 4096, "bf16", residual=True),
        # sixteen sequences' new tokens through the gated half of a feed-forward block
        _linear("linear_decode_gated", 16, 8192, 4096, "bf16", act="silu", gated=True),
        # a ragged batch of prompts' tokens through a small model's feed-forward block
        _linear("linear_ragged_gelu", 333, 1000, 1032, "f16", bias=True, act="gelu_tanh", residual=True),
        # a prompt through the query, key and value projection
        _linear("linear_qkv_bias", 2048, 6144, 4096, "bf16", bias=True),
        # long prompts through the down projection of a feed-forward block
        _linear("linear_down_residual", 4096, 4096, 8192, "f16", residual=True),
        # the same batch through the gated projection: the largest product of a layer
        _linear("linear_gated_large", 8192, 8192, 4096, "bf16", act="silu", gated=True),
        # one new token far into a long context, heads in halves
        _rope("rope_one_token", 1, 1, 32, 8, 128, 128, "bf16", values=True, table=131072, first=131000),
        # prompts whose heads rotate only half of their elements, in pairs, laid out for the attention kernel
        _rope("rope_prompt_pairs", 4, 4096, 32, 8, 128, 64, "f16", interleaved=True, values=True, heads_first=True),
        # the gradient of a rotation, in the type that gradients are kept in
        _rope("rope_gradient_f32", 2, 1777, 16, 0, 96, 96, "f32", inverse=True),
        # a decode step of 48 sequences, a third of its slots empty
        _rope("qk_norm_rope_decode", 48, 1, 32, 8, 128, 128, "bf16", norm=True, table=32768, first=20000, padded=16),
        # prompts of an odd length with small heads
        _rope("qk_norm_rope_odd", 3, 1021, 12, 4, 80, 40, "f16", norm=True, values=True, heads_first=True),
        # a long prompt: the queries, keys and values of one layer
        _rope("qk_norm_rope_long", 1, 32768, 64, 8, 128, 128, "bf16", norm=True, values=True, heads_first=True,
              table=32768),
    ]


def _log(rng, low, high, step=1):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high))) / step)) * step))


def draw(rng):
    if rng.random() < 0.5:
        gated = rng.random() < 0.3
        act = rng.choice(("silu", "gelu_tanh")) if gated else rng.choice(("", "", "relu", "silu", "gelu_tanh"))
        c = _linear("", _log(rng, 1, 8192), _log(rng, 256, 8192, 8), _log(rng, 256, 4096, 8),
                    rng.choice(("f16", "bf16")), rng.random() < 0.5, act, rng.random() < 0.5, gated)
    else:
        d = rng.choice((32, 64, 80, 96, 128, 128, 256))
        heads = rng.choice((4, 8, 12, 16, 32))
        kv = rng.choice((0, 1, 2, 4, 8))
        tokens = _log(rng, 1, 16384)
        b = rng.choice((1, 1, 2, 3, 7))
        s = max(1, tokens // b)
        first = rng.choice((0, 0, 777, 100000))
        heads_first = rng.random() < 0.5
        c = _rope("", b, s, heads, kv, d, rng.choice((d, d, d // 2)), rng.choice(("f16", "bf16", "f32")),
                  rng.random() < 0.5, kv > 0 and rng.random() < 0.5, heads_first,
                  False, rng.random() < 0.5, first + s, first, rng.randrange(0, max(1, b * s // 4)))
    del c["name"]
    return c


# ---- what a program has in hand -----------------------------------------------------

_kernels = {}


def _kernel(case):
    """The framework's compiled kernel for the sizes and types of ``case``."""
    key = tuple(sorted((k, v) for k, v in case.items() if k not in ("name", "first", "padded")))
    if key not in _kernels:
        root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "thompiler-emmy-hackathon_b200")
        if root not in sys.path:
            sys.path.insert(0, root)
        from thompiler import synth
        from thompiler.device import DeviceKernel
        with tempfile.TemporaryDirectory() as tmp:
            if case["op"] == "linear":
                d = synth.linear_package(tmp, case["m"], case["n"], case["k"], dtype=case["dtype"],
                                         bias=case["bias"], activation=case["act"] or None,
                                         residual=case["residual"], gated=case["gated"])
                _kernels[key] = DeviceKernel(d / "k_linear.ir.json")
            else:
                build = synth.qk_norm_rope_package if case["op"] == "qk_norm_rope" else synth.rope_package
                more = {} if case["op"] == "qk_norm_rope" else {"inverse": case["inverse"]}
                d = build(tmp, case["b"], case["s"], case["heads"], case["kv"], case["d"], rotary=case["rotary"],
                          interleaved=case["interleaved"], dtype=case["dtype"], table=case["table"],
                          values=case["values"], heads_first=case["heads_first"], **more)
                _kernels[key] = DeviceKernel(d / f"k_{case['op']}.ir.json")
    return _kernels[key]


def _tables(rows, rotary, device):
    """cos and sin of position * 10000^(-2 i / rotary), formed in 64 bits."""
    i = torch.arange(rotary // 2, dtype=torch.float64, device=device)
    a = torch.arange(rows, dtype=torch.float64, device=device)[:, None] * torch.pow(10000.0, -2.0 * i / rotary)
    return torch.cos(a).float(), torch.sin(a).float()


def prepare(case, seed):
    dev, t = "cuda", TYPES[case["dtype"]]
    g = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, device=dev, generator=g) * scale).to(t)

    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        rows = 2 * n if case["gated"] else n
        st = {"x": normal(m, k), "w": normal(rows, k, scale=k ** -0.5)}
        if case["bias"]:
            st["bias"] = normal(rows, scale=0.2)
        if case["residual"]:
            st["res"] = normal(m, n)
        st["linear"] = torch.zeros(m, n, device=dev, dtype=t)
    else:
        b, s, h, kv, d = (case[x] for x in ("b", "s", "heads", "kv", "d"))
        st = {"qkv": normal(b, s, h + kv * (2 if case["values"] else 1), d)}
        st["cos"], st["sin"] = _tables(case["table"], case["rotary"], dev)
        pos = (case["first"] + torch.arange(s, device=dev, dtype=torch.int32)).repeat(b, 1)
        if s == 1 and case["first"]:            # sequences of their own lengths
            pos = pos - torch.randint(0, case["first"], (b, s), device=dev, generator=g, dtype=torch.int32) // 2
        if case["padded"]:                      # empty slots at the batch's end
            pos.view(-1)[b * s - case["padded"]:] = -1
        st["pos"] = pos.contiguous()
        if case["op"] == "qk_norm_rope":
            st["wq"] = (1 + normal(d, scale=0.2).float()).to(t)
            if kv:
                st["wk"] = (1 + normal(d, scale=0.2).float()).to(t)
        for name, n in (("q", h), ("k", kv), ("v", kv if case["values"] else 0)):
            if n:
                shape = (b, n, s, d) if case["heads_first"] else (b, s, n, d)
                st[name] = torch.zeros(shape, device=dev, dtype=t)
    st = {"case": dict(case), "buffers": st}
    if own:
        st["kernel"] = _kernel(case)
    return st


def _outputs(case):
    if case["op"] == "linear":
        return ("linear",)
    return ("q",) + (("k",) if case["kv"] else ()) + (("v",) if case["kv"] and case["values"] else ())


# ---- one pass -------------------------------------------------------------------------

def run(state):
    case, x = state["case"], state["buffers"]
    if own:
        state["kernel"]({n: t.data_ptr() for n, t in x.items()}, torch.cuda.current_stream().cuda_stream)
        return {n: x[n] for n in _outputs(case)}
    return _plain_linear(case, x) if case["op"] == "linear" else _plain_heads(case, x)


def _activate(z, act):
    if act == "relu":
        return torch.clamp(z, min=0)
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu_tanh":
        u = math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)
        return 0.5 * z * (1 + torch.tanh(u))
    return z


def _plain_linear(case, x):
    z = x["x"].float() @ x["w"].float().t()
    if case["bias"]:
        z = z + x["bias"].float()
    if case["gated"]:
        n = case["n"]
        z = _activate(z[:, :n], case["act"]) * z[:, n:]
    else:
        z = _activate(z, case["act"])
    if case["residual"]:
        z = z + x["res"].float()
    return {"linear": z.to(TYPES[case["dtype"]])}


def _turn(y, cos, sin, case):
    """Rotate the leading ``rotary`` elements of each head of y[b, s, heads, d]."""
    r = case["rotary"]
    a, rest = y[..., :r], y[..., r:]
    if case["inverse"]:
        sin = -sin
    if case["interleaved"]:
        a0, a1 = a[..., 0::2], a[..., 1::2]
        a = torch.stack((a0 * cos - a1 * sin, a1 * cos + a0 * sin), -1).flatten(-2)
    else:
        a0, a1 = a[..., :r // 2], a[..., r // 2:]
        a = torch.cat((a0 * cos - a1 * sin, a1 * cos + a0 * sin), -1)
    return torch.cat((a, rest), -1)


def _plain_heads(case, x):
    h, kv, t = case["heads"], case["kv"], TYPES[case["dtype"]]
    live = x["pos"] >= 0
    at = x["pos"].clamp(min=0).long()
    cos, sin = x["cos"][at][:, :, None], x["sin"][at][:, :, None]
    y = x["qkv"].float()
    parts = {"q": (y[:, :, :h], "wq"), "k": (y[:, :, h:h + kv], "wk")}
    out = {}
    for name in _outputs(case):
        if name == "v":
            z = y[:, :, h + kv:]
        else:
            z, w = parts[name]
            if case["op"] == "qk_norm_rope":
                z = z * torch.rsqrt((z * z).mean(-1, keepdim=True) + 1e-6) * x[w].float()
            z = _turn(z, cos, sin, case)
        z = z.to(t)
        keep = live[:, :, None, None]
        if case["heads_first"]:
            z, keep = z.transpose(1, 2), live[:, None, :, None]
        out[name] = torch.where(keep, z, x[name])
    return out


# ---- what a pass cannot do without --------------------------------------------------------

def work(case):
    e = BYTES[case["dtype"]]
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        rows = 2 * n if case["gated"] else n
        nbytes = e * (m * k + rows * k + m * n + (rows if case["bias"] else 0) + (m * n if case["residual"] else 0))
        return {"bytes": nbytes, "flops": 2 * m * rows * k}
    live = case["b"] * case["s"] - case["padded"]
    heads = case["heads"] + case["kv"] * (2 if case["values"] else 1)
    turned = case["heads"] + case["kv"]
    nbytes = 2 * e * live * heads * case["d"] + 4 * case["b"] * case["s"]
    # the rows of the tables that are read: no more than there are positions
    nbytes += 4 * case["rotary"] * min(live, case["s"] if case["s"] > 1 else live)
    flops = live * turned * (3 * case["rotary"] + (4 * case["d"] if case["op"] == "qk_norm_rope" else 0))
    return {"bytes": nbytes, "flops": flops}


# ---- the definition, in 64 bits -------------------------------------------------------------

def exact(case, seed):
    x = {n: t.double() if t.is_floating_point() else t for n, t in prepare(case, seed)["buffers"].items()}
    if case["op"] == "linear":
        z = torch.matmul(x["x"], x["w"].transpose(0, 1))
        if case["bias"]:
            z += x["bias"]
        gate = z[:, :case["n"]]
        if case["act"] == "relu":
            gate = torch.where(gate > 0, gate, torch.zeros_like(gate))
        elif case["act"] == "silu":
            gate = gate * torch.sigmoid(gate)
        elif case["act"] == "gelu_tanh":
            gate = gate * torch.sigmoid(math.sqrt(8 / math.pi) * (gate + 0.044715 * gate ** 3))
        if case["gated"]:
            gate = gate * z[:, case["n"]:]
        return {"linear": gate + x["res"] if case["residual"] else gate}
    h, kv, r = case["heads"], case["kv"], case["rotary"]
    turn = torch.complex(x["cos"], -x["sin"] if case["inverse"] else x["sin"])[x["pos"].clamp(min=0).long()]
    out = {}
    for name, lo, hi in (("q", 0, h), ("k", h, h + kv), ("v", h + kv, h + 2 * kv)):
        if name not in _outputs(case):
            continue
        y = x["qkv"][:, :, lo:hi].clone()
        if name != "v":
            if case["op"] == "qk_norm_rope":
                y /= torch.sqrt(y.square().sum(-1, keepdim=True) / case["d"] + 1e-6)
                y *= x["wq" if name == "q" else "wk"]
            i = torch.arange(r // 2, device=y.device)
            first, second = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + r // 2)
            z = torch.complex(y[..., first], y[..., second]) * turn[:, :, None]
            y[..., first], y[..., second] = z.real, z.imag
        y *= (x["pos"] >= 0)[:, :, None, None]          # the outputs hold zeros where a slot is empty
        out[name] = y.transpose(1, 2) if case["heads_first"] else y
    return out
