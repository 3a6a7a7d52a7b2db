"""The 4-bit floating-point products and the rules between logits and token, as cases to time.

- `quantise`: rows of weights or activations to MXFP4 (32 elements of e2m1 under one power-of-two scale), with the values that the codes
  stand for.
- `product`: Y = X . W^T of two quantised operands.
- `decode`: Y = X . W^T of 1 to 16 rows of 16-bit activations with a quantised weight matrix.
- `answer`: penalties for repeated tokens, biases and a grammar's mask on the logits of a step, and the token that wins.

`run` computes them in plain torch operations, or with the library's doors where `own` is true.
"""
from __future__ import annotations

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODE = {"f32": 0, "f16": 1, "bf16": 2}   # the library's element types
GEMM_WORKSPACE = 64 << 20                # what a program sets aside for the products' K ranges


def listed():
    return [
        # one token's hidden row in front of a quantised projection: latency
        {"name": "quantise_row", "op": "quantise", "rows": 1, "k": 5120, "ld": 5120, "dtype": "f16"},
        # rows of a wider fp32 tensor, an odd number of blocks each
        {"name": "quantise_ragged", "op": "quantise", "rows": 333, "k": 2080, "ld": 2112, "dtype": "f32"},
        # a projection's weights at load time
        {"name": "quantise_weights", "op": "quantise", "rows": 17408, "k": 5120, "ld": 5120, "dtype": "bf16"},
        # a small projection of a few rows: latency
        {"name": "product_small", "op": "product", "m": 16, "n": 640, "k": 1024, "y": "bf16"},
        # a short prompt, with odd rows, columns and blocks
        {"name": "product_ragged", "op": "product", "m": 77, "n": 1003, "k": 1056, "y": "f32"},
        # a long prompt on a square projection
        {"name": "product_prompt", "op": "product", "m": 4096, "n": 5120, "k": 5120, "y": "bf16"},
        # a long prompt on a wide feed-forward projection: the largest product
        {"name": "product_wide", "op": "product", "m": 4096, "n": 17408, "k": 5120, "y": "f16"},
        # a token on a wide feed-forward projection
        {"name": "decode_row", "op": "decode", "m": 1, "n": 17408, "k": 5120, "x": "bf16", "y": "f16"},
        # a verify window of eight tokens on the projection back
        {"name": "decode_window", "op": "decode", "m": 8, "n": 5120, "k": 17408, "x": "f16", "y": "f32"},
        # a token's logits
        {"name": "decode_head", "op": "decode", "m": 1, "n": 151936, "k": 5120, "x": "bf16", "y": "f32"},
        # one request's step, under a grammar
        {"name": "answer_row", "op": "answer", "rows": 1, "n": 151936, "history": 4096, "prompt": 1024, "biases": 16, "masks": 1, "dtype": "f32"},
        # a step of a full batch, a quarter of it under grammars
        {"name": "answer_batch", "op": "answer", "rows": 256, "n": 151936, "history": 2048, "prompt": 1500, "biases": 8, "masks": 64, "dtype": "f32"},
    ]


def draw(rng):
    def spread(lo, hi):
        return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))

    op = rng.choice(["quantise", "product", "decode", "answer"])
    if op == "quantise":
        k = 32 * spread(1, 544)
        return {"op": op, "rows": spread(1, min(17408, 17408 * 5120 // k)), "k": k, "ld": k + rng.choice([0, 0, 32, 1024]), "dtype": rng.choice(["f32", "f16", "bf16"])}
    if op == "product":
        n, k = spread(1, 17408), 32 * spread(1, 544)
        return {"op": op, "m": spread(1, min(8192, 4096 * 17408 * 5120 // (n * k))), "n": n, "k": k, "y": rng.choice(["f32", "f16", "bf16"])}
    if op == "decode":
        k = 32 * spread(1, 544)
        return {"op": op, "m": rng.randint(1, 16), "n": spread(1, min(151936, 151936 * 5120 // k)), "k": k, "x": rng.choice(["f16", "bf16"]), "y": rng.choice(["f16", "f32"])}
    n = spread(64, 151936)
    rows, history = spread(1, 256), spread(1, 4096)
    return {"op": op, "rows": rows, "n": n, "history": history, "prompt": rng.randint(0, history), "biases": rng.randint(0, 32),
            "masks": rng.choice([0, rows, (rows + 3) // 4]), "dtype": rng.choice(["f32", "f32", "f16", "bf16"])}


def _normal(shape, g, std=1.0, outliers=0.0):
    x = torch.randn(shape, device="cuda", generator=g) * std
    if outliers:   # a few channels that are far larger, as activations have them
        x = torch.where(torch.rand(shape, device="cuda", generator=g) < outliers, x * 20.0, x)
    return x


# ---- MXFP4 in plain torch --------------------------------------------------------------------------------------------------------
def _quantise(x):
    """x f32 [rows, k] -> codes u8 [rows, k / 2] (the even element in the low half), scales u8 [rows, k / 32], values f32 [rows, k]."""
    rows, k = x.shape
    v = x.contiguous().view(rows, k // 32, 32)
    field = (v.abs().amax(2).view(torch.int32) >> 23) & 0xFF                          # exponent field of the largest magnitude
    broken = ~torch.isfinite(v).all(2)
    scale = torch.where(broken, 255, torch.clamp(field - 2, min=0))                   # floor(log2) less e2m1's largest exponent
    inverse = ((254 - torch.where(broken, 127, scale)) << 23).view(torch.float32)     # 2^(127 - scale), exact
    t = torch.where(broken[:, :, None], 0.0, v * inverse[:, :, None])
    a = torch.clamp(t.abs(), max=6.0)
    step = torch.where(a < 2.0, 0.5, torch.where(a < 4.0, 1.0, 2.0))
    q = torch.round(a / step) * step                                                  # to even: the even code
    code = torch.where(q < 2.0, 2.0 * q, torch.where(q < 4.0, q + 2.0, q * 0.5 + 4.0)).to(torch.int32)
    code = code | ((t.view(torch.int32) >> 28) & 8)
    code = code.view(rows, k // 2, 2)
    packed = (code[:, :, 0] | (code[:, :, 1] << 4)).to(torch.uint8)
    return packed, scale.to(torch.uint8), _values(packed, scale.to(torch.uint8))


def _values(codes, scales):
    """What the codes stand for, f32 [rows, k]."""
    rows, half = codes.shape
    c = torch.stack((codes & 15, codes >> 4), 2).view(rows, half // 16, 32).to(torch.int32)
    m = (c & 7).to(torch.float32)
    a = torch.where(m < 4.0, 0.5 * m, torch.where(m < 6.0, m - 2.0, 2.0 * m - 8.0))
    a = torch.where(c >= 8, -a, a)
    e = scales.to(torch.int32)
    s = torch.where(e == 0, 0x00400000, torch.where(e == 255, 0x7FC00000, e << 23)).view(torch.float32)   # 2^(e - 127), 255: NaN
    return (a * s[:, :, None]).view(rows, 2 * half)


def _quantised(shape, g, std, outliers=0.0):
    codes, scales = [], []
    for part in torch.split(torch.arange(shape[0]), 8192):   # large matrices by pieces: less memory
        c, s, _ = _quantise(_normal((len(part), shape[1]), g, std, outliers))
        codes.append(c)
        scales.append(s)
    return torch.cat(codes), torch.cat(scales)


# ---- states ----------------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = dict(case)
    if case["op"] == "quantise":
        rows, k, ld = case["rows"], case["k"], case["ld"]
        t = TYPES[case["dtype"]]
        s["x"] = _normal((rows, ld), g, 0.02 if rows > 4096 else 1.0, 0.0 if rows > 4096 else 0.001).to(t)
        s["codes"] = torch.empty(rows, k // 2, dtype=torch.uint8, device="cuda")
        s["scales"] = torch.empty(rows, k // 32, dtype=torch.uint8, device="cuda")
        s["values"] = torch.empty(rows, k, dtype=t, device="cuda")
    elif case["op"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        s["wc"], s["ws"] = _quantised((n, k), g, 0.02)
        s["xc"], s["xs"] = _quantised((m, k), g, 1.0, 0.001)
        s["out"] = torch.empty(m, n, dtype=TYPES[case["y"]], device="cuda")
        s["workspace"] = torch.empty(GEMM_WORKSPACE, dtype=torch.uint8, device="cuda")
    elif case["op"] == "decode":
        m, n, k = case["m"], case["n"], case["k"]
        s["wc"], s["ws"] = _quantised((n, k), g, 0.02)
        s["rows_x"] = _normal((m, k), g, 1.0, 0.001).to(TYPES[case["x"]])
        s["out"] = torch.empty(m, n, dtype=TYPES[case["y"]], device="cuda")
    else:
        rows, n, hist = case["rows"], case["n"], case["history"]
        r = lambda *shape: torch.rand(shape, device="cuda", generator=g)  # noqa: E731
        s["logits"] = _normal((rows, n), g, 3.0).to(TYPES[case["dtype"]])
        s["tokens_seen"] = (r(rows, hist) ** 3 * n).to(torch.int32).clamp_(max=n - 1)       # some tokens far more often than others
        s["total"] = (hist - r(rows) * 0.25 * hist).to(torch.int32)                         # requests are of different lengths
        s["prompt_len"] = torch.minimum(s["total"], torch.full_like(s["total"], case["prompt"]))
        s["repetition"], s["presence"], s["frequency"] = 1.0 + 0.3 * r(rows), 0.5 * r(rows), 0.2 * r(rows)
        s["bias_off"] = torch.arange(rows + 1, dtype=torch.int32, device="cuda") * case["biases"]
        s["bias_tok"] = (r(rows * case["biases"]) * n).to(torch.int32).clamp_(max=n - 1)
        s["bias_val"] = 4.0 * r(rows * case["biases"]) - 2.0
        words = (n + 31) // 32
        mask = torch.randint(-(1 << 31), 1 << 31, (case["masks"], words), device="cuda", generator=g).to(torch.int32)
        mask &= torch.randint(-(1 << 31), 1 << 31, (case["masks"], words), device="cuda", generator=g).to(torch.int32)
        if case["masks"] > 3:
            mask[3] = 0                                                                     # a grammar at a dead end
        s["allowed"] = mask
        at = torch.arange(rows, dtype=torch.int32, device="cuda")
        s["allowed_row"] = torch.where(at < case["masks"], at, torch.full_like(at, -1))     # which mask a request has, -1: none
        s["out"] = torch.empty(rows, n, dtype=s["logits"].dtype, device="cuda")
        s["tokens"] = torch.empty(rows, dtype=torch.int32, device="cuda")
        s["workspace"] = torch.empty(rows * (n // 1024 + 1) * 8, dtype=torch.uint8, device="cuda")
    return s


# ---- one pass --------------------------------------------------------------------------------------------------------------------
def run(state):
    if own:
        return _own(state)
    if state["op"] == "quantise":
        _, scales, values = _quantise(state["x"][:, : state["k"]].float())
        return {"scales": scales, "values": values.to(state["x"].dtype)}
    if state["op"] == "product":
        return {"y": (_values(state["xc"], state["xs"]) @ _values(state["wc"], state["ws"]).t()).to(state["out"].dtype)}
    if state["op"] == "decode":
        return {"y": (state["rows_x"].float() @ _values(state["wc"], state["ws"]).t()).to(state["out"].dtype)}
    return _answer(state)


def _answer(s):
    l = s["logits"].float()
    rows, n = l.shape
    at = torch.arange(s["tokens_seen"].shape[1], device="cuda")[None, :]
    tok = s["tokens_seen"].long()
    seen = torch.zeros(rows, n, dtype=torch.int32, device="cuda").scatter_add_(1, tok, (at < s["total"][:, None]).to(torch.int32))
    count = torch.zeros(rows, n, dtype=torch.int32, device="cuda").scatter_add_(
        1, tok, ((at >= s["prompt_len"][:, None]) & (at < s["total"][:, None])).to(torch.int32))
    r = s["repetition"][:, None]
    l = torch.where(seen > 0, torch.where(l > 0, l / r, l * r), l)
    l = l - s["frequency"][:, None] * count.float()
    l = torch.where(count > 0, l - s["presence"][:, None], l)
    if s["bias_tok"].numel():
        entry = torch.arange(s["bias_tok"].numel(), device="cuda")
        row = entry // s["biases"]
        last = torch.full((rows * n,), -1, dtype=torch.int64, device="cuda").scatter_reduce_(0, row * n + s["bias_tok"].long(), entry, "amax").view(rows, n)
        l = torch.where(last >= 0, l + s["bias_val"][last.clamp(min=0)], l)
    if s["masks"]:
        i = torch.arange(n, device="cuda")
        free = ((s["allowed"][:, i >> 5] >> (i & 31)[None, :]) & 1) != 0
        l[: s["masks"]] = torch.where(free, l[: s["masks"]], float("-inf"))
    top = l.amax(1, keepdim=True)
    first = torch.where(l == top, torch.arange(n, device="cuda")[None, :], n).amin(1)
    return {"logits": l.to(s["logits"].dtype), "tokens": torch.where(top[:, 0] == float("-inf"), -1, first).to(torch.int32)}


_kept = {}


def _library():
    if not _kept:
        from qwegn_amd import qwhip

        dev = qwhip.Device(torch.cuda.current_device())
        _kept.update(q=qwhip, dev=dev, lib=dev.lib, stream=dev.stream.handle)
    return _kept["q"], _kept["lib"], _kept["stream"]


def _own(s):
    q, lib, st = _library()
    if "call" not in s:   # the addresses and the views that a program keeps beside its buffers
        s["call"] = _call_of(s, q, lib, st)
    fn, args, out = s["call"]
    status = fn(*args)
    if status:
        q.check(status)
    return out


def _call_of(s, q, lib, st):
    if s["op"] == "quantise":
        return lib.qwhip_quantize_mxfp4, (st, s["x"].data_ptr(), CODE[s["dtype"]], s["rows"], s["k"], s["ld"], s["codes"].data_ptr(), s["scales"].data_ptr(),
                                          s["values"].data_ptr()), {"scales": s["scales"], "values": s["values"]}
    if s["op"] == "answer":
        rules = q.LogitsRules(history=s["tokens_seen"].data_ptr(), ld_history=s["history"], prompt_len=s["prompt_len"].data_ptr(), total_len=s["total"].data_ptr(),
                              repetition=s["repetition"].data_ptr(), presence=s["presence"].data_ptr(), frequency=s["frequency"].data_ptr(),
                              bias_off=s["bias_off"].data_ptr(), bias_tok=s["bias_tok"].data_ptr(), bias_val=s["bias_val"].data_ptr(), bias_count=s["bias_tok"].numel(),
                              allowed=s["allowed"].data_ptr(), allowed_rows=s["masks"], ld_allowed=s["allowed"].shape[1], allowed_row=s["allowed_row"].data_ptr())
        return lib.qwhip_logits_process, (st, q.C.byref(rules), s["logits"].data_ptr(), CODE[s["dtype"]], s["rows"], s["n"], 0, s["out"].data_ptr(), 0, s["tokens"].data_ptr(),
                                          s["workspace"].data_ptr(), s["workspace"].numel()), {"logits": s["out"], "tokens": s["tokens"]}
    w = q.Mxfp4View(s["wc"].data_ptr(), s["ws"].data_ptr(), s["wc"].numel(), s["ws"].numel(), s["n"], s["k"], 0)
    if s["op"] == "product":
        x = q.Mxfp4View(s["xc"].data_ptr(), s["xs"].data_ptr(), s["xc"].numel(), s["xs"].numel(), s["m"], s["k"], 0)
        return lib.qwhip_mxfp4_gemm, (st, q.C.byref(w), q.C.byref(x), s["out"].data_ptr(), CODE[s["y"]], 0, s["workspace"].data_ptr(), GEMM_WORKSPACE), {"y": s["out"]}
    y16, y32 = (s["out"].data_ptr(), None) if s["y"] == "f16" else (None, s["out"].data_ptr())
    return lib.qwhip_mxfp4_gemv, (st, q.C.byref(w), s["rows_x"].data_ptr(), CODE[s["x"]], s["m"], y16, y32), {"y": s["out"]}


# ---- what a pass cannot do without -----------------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "quantise":
        size, e = TYPES[case["dtype"]].itemsize, case["rows"] * case["k"]
        return {"bytes": e * size * 2 + e * 17 // 32, "flops": 4 * e}
    if case["op"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": (m + n) * k * 17 // 32 + m * n * TYPES[case["y"]].itemsize, "flops": 2 * m * n * k}
    if case["op"] == "decode":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": n * k * 17 // 32 + m * k * 2 + m * n * TYPES[case["y"]].itemsize, "flops": 2 * m * n * k}
    rows, n = case["rows"], case["n"]
    return {"bytes": 2 * rows * n * TYPES[case["dtype"]].itemsize + case["masks"] * ((n + 31) // 32) * 4 + rows * (case["history"] * 4 + case["biases"] * 8 + 28),
            "flops": 6 * rows * n}


# ---- the definitions, in 64 bits ---------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "quantise":
        x = s["x"][:, : case["k"]].double().reshape(case["rows"], -1, 32)
        top = x.abs().amax(2, keepdim=True)
        unit = torch.exp2(torch.clamp(torch.frexp(top).exponent - 3, min=-127).double())        # frexp's mantissa is in [1/2, 1)
        unit = torch.where(top > 0, unit, torch.full_like(unit, 2.0 ** -127))
        grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device="cuda")
        between = 0.5 * (grid[1:] + grid[:-1])
        a = x.abs() / unit
        below, above = torch.bucketize(a, between, right=False), torch.bucketize(a, between, right=True)
        near = torch.where(below % 2 == 0, below, above)                                        # they differ on a border: the even one
        return {"scales": None, "values": (grid[near] * torch.sign(x) * unit).reshape(case["rows"], case["k"])}
    if case["op"] in ("product", "decode"):
        w = _wide(s["wc"], s["ws"])
        x = _wide(s["xc"], s["xs"]) if case["op"] == "product" else s["rows_x"].double()
        return {"y": torch.mm(x, w.t())}
    l = s["logits"].double()
    rows, n = l.shape
    places = torch.arange(rows, device="cuda")
    both, answer = torch.zeros(rows * n, dtype=torch.float64, device="cuda"), torch.zeros(rows * n, dtype=torch.float64, device="cuda")
    row, col = torch.nonzero(torch.arange(case["history"], device="cuda")[None] < s["total"][:, None], as_tuple=True)
    spot, one = row * n + s["tokens_seen"][row, col].long(), torch.ones(len(row), dtype=torch.float64, device="cuda")
    both.index_add_(0, spot, one)
    answer.index_add_(0, spot, (col >= s["prompt_len"][row]).double())
    both, answer = both.view(rows, n), answer.view(rows, n)
    rep = s["repetition"].double()[:, None].expand(rows, n)
    factor = torch.where(both > 0, torch.where(l > 0, 1.0 / rep, rep), torch.ones_like(l))
    l = l * factor - s["frequency"].double()[:, None] * answer - s["presence"].double()[:, None] * (answer > 0)
    for j in range(case["biases"]):   # in order: of two entries for a token the later one holds
        t = s["bias_tok"].view(rows, -1)[:, j].long()
        again = (s["bias_tok"].view(rows, -1)[:, j + 1:] == t[:, None]).any(1)
        l[places, t] += torch.where(again, 0.0, s["bias_val"].view(rows, -1)[:, j].double())
    if case["masks"]:
        bits = (s["allowed"].long() & 0xFFFFFFFF)[:, :, None] // (2 ** torch.arange(32, device="cuda"))[None, None] % 2
        l[: case["masks"]][bits.reshape(case["masks"], -1)[:, :n] == 0] = float("-inf")
    return {"logits": l, "tokens": None}


def _wide(codes, scales):
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0], dtype=torch.float64, device="cuda")
    v = torch.empty(codes.shape[0], codes.shape[1] * 2, dtype=torch.float64, device="cuda")
    v[:, 0::2], v[:, 1::2] = table[(codes % 16).int()], table[(codes // 16).int()]
    return v * torch.exp2(scales.double() - 127.0).repeat_interleave(32, 1)
