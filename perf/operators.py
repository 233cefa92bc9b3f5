"""Timed cases of the operators in 8-bit floating point (e4m3) with a scale for each block of 128 values:
the residual's addition with the root-mean-square norm and an 8-bit output, the quantisers, the routed matrix
product, and the gated feed-forward block made of them.

A quantised tensor is q (e4m3) with one exponent byte s for each row and block of 128 columns; it stands for
q * 2^(s - 127). s is the smallest byte with max|v| <= 448 * 2^(s - 127) over the block (a weight's block spans
128 rows too, which then hold the same s). The bytes are packed in tiles of 128 rows x 4 blocks: row r's byte for
block b is at ((r // 128) * G + b // 4) * 512 + (r % 32) * 16 + (r % 128) // 32 * 4 + b % 4, with G groups of
four blocks in a row.
"""
import math
import os
import sys

import torch

own = False

EPS = 1e-6
HIDDEN, INTER, QKV = 4096, 12288, 6144      # the full model's layer (u15b200.model.FULL)
E4M3_MAX = 448.0


def listed():
    return [
        # a text prompt's next token: the norm before a layer's projections, where only latency counts
        {"name": "norm_1", "op": "norm", "rows": 1, "cols": HIDDEN, "first": 1, "add": True},
        # the generation pass: 512 text rows by one expert, 3584 image rows by the other
        {"name": "norm_4096_routed", "op": "norm", "rows": 4096, "cols": HIDDEN, "first": 512, "add": True},
        # an odd prompt at a width that ends inside a block, no residual to add
        {"name": "norm_1537_narrow", "op": "norm", "rows": 1537, "cols": 1552, "first": 100, "add": False},
        # the feed-forward's wide activations of an odd number of rows
        {"name": "quant_333_wide", "op": "quant", "rows": 333, "cols": INTER},
        # binding a layer's weights: both experts' query, key and value rows
        {"name": "weight_qkv", "op": "weight", "rows": QKV, "cols": HIDDEN},
        # one token through the query, key and value projection: the weights' bytes
        {"name": "qkv_1", "op": "linear", "rows": 1, "k": HIDDEN, "n": QKV, "first": 1, "add": False},
        # a few tokens through the output projection, with the residual
        {"name": "o_17_residual", "op": "linear", "rows": 17, "k": HIDDEN, "n": HIDDEN, "first": 17, "add": True},
        # a ragged prompt through the down projection, both experts
        {"name": "down_1000_residual", "op": "linear", "rows": 1000, "k": INTER, "n": HIDDEN, "first": 77, "add": True},
        # text and image rows together through the query, key and value projection
        {"name": "qkv_4416_routed", "op": "linear", "rows": 4416, "k": HIDDEN, "n": QKV, "first": 320, "add": False},
        # the whole feed-forward block for one token, a ragged prompt, and the generation pass
        {"name": "ffn_1", "op": "ffn", "rows": 1, "hidden": HIDDEN, "inter": INTER, "first": 1},
        {"name": "ffn_333_routed", "op": "ffn", "rows": 333, "hidden": HIDDEN, "inter": INTER, "first": 41},
        {"name": "ffn_4096_routed", "op": "ffn", "rows": 4096, "hidden": HIDDEN, "inter": INTER, "first": 512},
    ]


def draw(rng):
    def log(lo, hi, step=1):
        return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step) * step))

    op = rng.choice(["norm", "norm", "quant", "weight", "linear", "linear", "linear", "ffn", "ffn"])
    rows = log(1, 4096 if op == "ffn" else 4416)
    first = rng.choice([rows, rows, rng.randint(0, rows)])
    if op == "norm":
        return {"op": op, "rows": rows, "cols": log(64, INTER, 16), "first": first, "add": rng.random() < 0.7}
    if op == "quant":
        return {"op": op, "rows": rows, "cols": log(64, INTER, 16)}
    if op == "weight":
        return {"op": op, "rows": log(64, 8192), "cols": log(64, INTER, 16)}
    if op == "linear":
        n = log(64, 8192, rng.choice([1, 8, 128]))
        return {"op": op, "rows": rows, "k": log(128, INTER, 16), "n": n, "first": first, "add": rng.random() < 0.5}
    return {"op": op, "rows": rows, "hidden": log(256, HIDDEN, 16), "inter": log(256, INTER, 128), "first": first}


# ------------------------------------------------------------------ inputs
def _groups(cols):
    return -(-cols // 512)


def _places(rows, cols, device="cuda"):
    """Where the packed scale bytes of [rows][blocks] are."""
    r = torch.arange(rows, device=device)[:, None]
    b = torch.arange(-(-cols // 128), device=device)[None, :]
    return ((r // 128) * _groups(cols) + b // 4) * 512 + (r % 32) * 16 + (r % 128) // 32 * 4 + b % 4


def _scale_bytes(amax):
    """The smallest byte s with amax <= 448 * 2^(s - 127): 448 = 1.75 * 2^8."""
    u = amax.float().contiguous().view(torch.int32)
    return ((u >> 23) - 8 + ((u & 0x7FFFFF) > 0x600000).int()).clamp(min=0)


def _quantised(v, rows_too=False):
    """v [rows][cols] in 32 bits -> (e4m3 values, packed scale bytes)."""
    rows, cols = v.shape
    nb = -(-cols // 128)
    a = torch.nn.functional.pad(v.abs(), (0, nb * 128 - cols)).reshape(rows, nb, 128).amax(2)
    if rows_too:
        nr = -(-rows // 128)
        a = torch.nn.functional.pad(a, (0, 0, 0, nr * 128 - rows)).reshape(nr, 128, nb).amax(1)
        a = a.repeat_interleave(128, 0)[:rows]
    s = _scale_bytes(a)
    q = (v * torch.exp2(127.0 - s.float()).repeat_interleave(128, 1)[:, :cols]).to(torch.float8_e4m3fn)
    packed = torch.full((-(-rows // 128) * _groups(cols) * 512,), 127, dtype=torch.uint8, device=v.device)
    packed[_places(rows, cols, v.device)] = s.to(torch.uint8)
    return q, packed


def _values(q, packed):
    """What a quantised tensor stands for, in 32 bits."""
    rows, cols = q.shape
    s = packed[_places(rows, cols, q.device)].float() - 127.0
    return q.float() * torch.exp2(s).repeat_interleave(128, 1)[:, :cols]


def _activations(g, rows, cols):
    """Tokens whose channels differ in size, a few of them by much."""
    gain = torch.exp(0.5 * torch.randn(cols, generator=g, device="cuda"))
    gain[torch.randint(0, cols, (max(1, cols // 512),), generator=g, device="cuda")] *= 12.0
    return (torch.randn(rows, cols, generator=g, device="cuda") * gain).bfloat16()


def _weight(g, n, k):
    """Two experts' [n][k], quantised in blocks of 128 x 128, each expert's scales packed apart."""
    both = [_quantised(0.02 * torch.randn(n, k, generator=g, device="cuda"), True) for _ in range(2)]
    return torch.stack([q for q, _ in both]), torch.cat([s for _, s in both])


def _segments(rows, first):
    """The first rows go to expert 0, the others to expert 1."""
    return [(a, b, e) for a, b, e in ((0, first, 0), (first, rows, 1)) if b > a]


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    op, rows, st = case["op"], case["rows"], dict(case)
    if op == "ffn":
        h, i = case["hidden"], case["inter"]
        st["x"], st["d"] = _activations(g, rows, h), _activations(g, rows, h)
        st["w"] = (1 + 0.1 * torch.randn(2, h, generator=g, device="cuda")).bfloat16()
        st["gu"], st["gu_s"] = _weight(g, 2 * i, h)
        st["down"], st["down_s"] = _weight(g, h, i)
        st["y"] = torch.empty(rows, h, dtype=torch.bfloat16, device="cuda")
        # what the block's steps leave to one another: quantised rows and packed scales
        size = rows * h + rows * i + -(-rows // 128) * 512 * (_groups(h) + _groups(i)) + 1024
        st["ws"] = torch.empty(size, dtype=torch.uint8, device="cuda")
    elif op == "linear":
        k, n = case["k"], case["n"]
        st["xq"], st["xs"] = _quantised(_activations(g, rows, k).float())
        st["wq"], st["ws"] = _weight(g, n, k)
        st["r"] = torch.randn(rows, n, generator=g, device="cuda").bfloat16() if case["add"] else None
        st["y"] = torch.empty(rows, n, dtype=torch.bfloat16, device="cuda")
    else:
        cols = case["cols"]
        st["x"] = _weight_source(g, rows, cols) if op == "weight" else _activations(g, rows, cols)
        if op == "norm":
            st["d"] = _activations(g, rows, cols) if case["add"] else None
            st["w"] = (1 + 0.1 * torch.randn(2, cols, generator=g, device="cuda")).bfloat16()
            st["sum"] = torch.empty_like(st["x"]) if case["add"] else None
        count = 2 if op == "weight" else 1
        st["q"] = torch.empty(count * rows, cols, dtype=torch.float8_e4m3fn, device="cuda")
        st["s"] = torch.empty(count * -(-rows // 128) * _groups(cols) * 512, dtype=torch.uint8, device="cuda")
        st["values"] = torch.empty(count * rows, cols, dtype=torch.bfloat16, device="cuda")
    if "first" in st:
        st["segments"] = _segments(rows, st["first"])
    return st


def _weight_source(g, rows, cols):
    return (0.02 * torch.randn(2 * rows, cols, generator=g, device="cuda")).bfloat16()


# ------------------------------------------------------------------ the operators
_ops = []


def _framework():
    if not _ops:
        root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        sys.path.insert(0, os.path.join(root, "vpipe-sensenova-u1.5_b200"))
        import u15b200
        _ops.append(u15b200.CudaOps(0))
    return _ops[0]


def run(st):
    return _run_own(st) if own else _run_plain(st)


def _run_own(st):
    o, op, rows = _framework(), st["op"], st["rows"]
    if op == "norm":
        cols = st["cols"]
        o.mot_add_rms_norm_quant_fp8(st["x"], st["d"], st["w"], st["segments"], st["sum"], st["q"], st["s"], rows,
                                     cols, EPS)
        o.dequant_fp8(st["q"], st["s"], st["values"], rows, cols)
        return {"sum": st["sum"], "values": st["values"]}
    if op == "quant":
        o.quant_rows_fp8(st["x"], st["q"], st["s"], rows, st["cols"])
        o.dequant_fp8(st["q"], st["s"], st["values"], rows, st["cols"])
        return {"values": st["values"]}
    if op == "weight":
        o.quant_weight_fp8(st["x"], st["q"], st["s"], 2, rows, st["cols"])
        o.dequant_fp8(st["q"], st["s"], st["values"], rows, st["cols"], n_experts=2)
        return {"values": st["values"]}
    if op == "linear":
        o.mot_linear_fp8(st["xq"], st["xs"], st["wq"], st["ws"], st["segments"], st["y"], rows, st["k"], st["n"],
                         epilogue=1 if st["add"] else 0, resid=st["r"])
        return {"y": st["y"]}
    o.mot_ffn_fp8(st["x"], st["d"], st["w"], st["gu"], st["gu_s"], st["down"], st["down_s"], st["segments"],
                  st["y"], st["ws"], rows, st["hidden"], st["inter"], EPS)
    return {"y": st["y"]}


def _normed(st, x):
    v = x * torch.rsqrt((x * x).mean(1, keepdim=True) + EPS)
    gain = torch.cat([st["w"][e].float().expand(b - a, -1) for a, b, e in st["segments"]])
    return v * gain


def _product(xq, xs, wq, ws, segments):
    x, per = _values(xq, xs), ws.numel() // 2
    parts = [x[a:b] @ _values(wq[e], ws[e * per:(e + 1) * per]).T for a, b, e in segments]
    return torch.cat(parts)


def _gate_up(v):
    """Weight rows come in blocks of 128 gate rows and the 128 up rows that go with them."""
    v = v.reshape(v.shape[0], -1, 2, 128)
    gate, up = v[:, :, 0].flatten(1), v[:, :, 1].flatten(1)
    return gate / (1 + torch.exp(-gate)) * up


def _run_plain(st):
    op, rows = st["op"], st["rows"]
    if op in ("norm", "ffn"):
        x = st["x"].float()
        total = None
        if st["d"] is not None:
            total = (x + st["d"].float()).bfloat16()
            x = total.float()
        q, s = _quantised(_normed(st, x))
        if op == "norm":
            return {"sum": total, "values": _values(q, s).bfloat16()}
        h, hs = _quantised(_gate_up(_product(q, s, st["gu"], st["gu_s"], st["segments"])))
        return {"y": (x + _product(h, hs, st["down"], st["down_s"], st["segments"])).bfloat16()}
    if op == "quant":
        return {"values": _values(*_quantised(st["x"].float())).bfloat16()}
    if op == "weight":
        both = [_values(*_quantised(w.float(), True)) for w in st["x"].split(rows)]
        return {"values": torch.cat(both).bfloat16()}
    y = _product(st["xq"], st["xs"], st["wq"], st["ws"], st["segments"])
    if st["add"]:
        y = st["r"].float() + y
    return {"y": y.bfloat16()}


# ------------------------------------------------------------------ the work
def work(case):
    """Bytes of the inputs and outputs once, weights of the experts that rows go to, and a product's operations."""
    op, rows = case["op"], case["rows"]
    if op == "norm":
        cols = case["cols"]
        return {"bytes": rows * cols * (7 if case["add"] else 3) + rows * -(-cols // 128) + 2 * cols, "flops": 6 * rows * cols}
    if op in ("quant", "weight"):
        n = rows * case["cols"] * (2 if op == "weight" else 1)
        return {"bytes": 3 * n + n // 128, "flops": 3 * n}
    if op == "linear":
        k, n = case["k"], case["n"]
        experts = len(_segments(rows, case["first"]))
        return {"bytes": (rows + experts * n) * (k + k // 128) + rows * n * (4 if case["add"] else 2),
                "flops": 2 * rows * n * k}
    h, i = case["hidden"], case["inter"]
    experts = len(_segments(rows, case["first"]))
    return {"bytes": experts * 3 * h * i * (1 + 1 / 128) + rows * h * 6, "flops": 6 * rows * h * i}


# ------------------------------------------------------------------ the definition, in 64 bits
def _rounded(v):
    """Nearest e4m3 value, ties to even: three bits after the leading one, steps of 2^-9 below 2^-6."""
    _, e = torch.frexp(v)
    step = torch.exp2((e.double() - 4).clamp(min=-9))
    return torch.round(v / step) * step


def _stands_for(v, tall):
    """The values that v has after quantisation in blocks of tall x 128."""
    r, c = v.shape
    p = torch.nn.functional.pad(v, (0, -c % 128, 0, -r % tall)).reshape(-(-r // tall), tall, -(-c // 128), 128)
    m, e = torch.frexp(p.abs().amax((1, 3), keepdim=True))    # amax = m * 2^e, and 448 = 0.875 * 2^9
    scale = torch.exp2((e.double() - 9 + (m > 0.875)).clamp(min=-127))
    return (_rounded(p / scale) * scale).flatten(2).flatten(0, 1)[:r, :c]


def _wide(q, packed):
    """A quantised tensor in 64 bits: the packed tiles as [row tile][group][32][4 rows][4 blocks]."""
    r, c = q.shape
    e = packed.reshape(-1, _groups(c), 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(-(-r // 128) * 128, -1)
    scale = torch.exp2(e[:r, :-(-c // 128)].double() - 127)
    v = torch.nn.functional.pad(q.double(), (0, -c % 128)).reshape(r, -1, 128) * scale[:, :, None]
    return v.flatten(1)[:, :c]


def exact(case, seed):
    st = prepare(case, seed)
    op, rows = case["op"], case["rows"]
    if op == "quant":
        return {"values": _stands_for(st["x"].double(), 1)}
    if op == "weight":
        return {"values": torch.cat([_stands_for(w.double(), 128) for w in st["x"].split(rows)])}
    expert = torch.ones(rows, dtype=torch.long, device="cuda")
    expert[:st["first"]] = 0

    def times(x, wq, ws):
        ws = ws.reshape(2, -1)
        y = x.new_empty(rows, wq.shape[1])
        for e in set(expert.tolist()):
            y[expert == e] = torch.mm(x[expert == e], _wide(wq[e], ws[e]).t())
        return y

    if op == "linear":
        y = times(_wide(st["xq"], st["xs"]), st["wq"], st["ws"])
        return {"y": y if st["r"] is None else y + st["r"].double()}
    x = st["x"] if st["d"] is None else st["x"] + st["d"]     # held in 16 bits, by the definition
    v = x.double()
    v = v / (v.pow(2).sum(1, keepdim=True) / v.shape[1] + EPS).sqrt() * st["w"].double()[expert]
    v = _stands_for(v, 1)
    if op == "norm":
        return {"sum": None if st["d"] is None else st["x"].double() + st["d"].double(), "values": v}
    p = times(v, st["gu"], st["gu_s"]).unflatten(1, (-1, 2, 128))
    gate, up = p.unbind(2)
    act = (gate * torch.sigmoid(gate) * up).flatten(1)
    return {"y": x.double() + times(_stands_for(act, 1), st["down"], st["down_s"])}
