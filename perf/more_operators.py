"""What stands between the q|k|v projection and the output projection, as cases to time.

- `heads`: queries and keys of a prompt or a step normed head by head, their positions' rotation, and the 32-point transform.
- `append`: a step's or a prompt's keys and values into a paged cache of 4-bit floats, rotated on the way; the queries with them.
- `attend`: attention over that cache: single tokens, windows of a few tokens, whole prompts and chunks of them.

`run` computes them in plain torch operations, or with the library's doors where `own` is true.
"""
from __future__ import annotations

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODE = {"f32": 0, "f16": 1, "bf16": 2}   # the library's element types
PLUS_ONE, PAIRS, FWHT_QK, FWHT_V = 1, 2, 4, 8   # the library's flags for a layer's head rules
ATTEND_WORKSPACE = 128 << 20             # what a program sets aside for partial results over long sequences
INV_SQRT32 = 0.17677669529663687


def listed():
    return [
        # a token's queries and keys: latency
        {"name": "heads_token", "op": "heads", "rows": 1, "q_heads": 40, "k_heads": 8, "d": 128, "rope": 128, "flags": PLUS_ONE, "dtype": "f16", "out": "f16"},
        # a verify window's fp32 rows: few heads, part of a head rotated in neighbouring pairs
        {"name": "heads_ragged", "op": "heads", "rows": 333, "q_heads": 6, "k_heads": 3, "d": 96, "rope": 48, "flags": PAIRS | FWHT_QK, "dtype": "f32", "out": "bf16"},
        # a long prompt
        {"name": "heads_prompt", "op": "heads", "rows": 8192, "q_heads": 40, "k_heads": 8, "d": 128, "rope": 128, "flags": PLUS_ONE, "dtype": "bf16", "out": "bf16"},
        # a token of one request: latency
        {"name": "append_token", "op": "append", "rows": 1, "q_heads": 40, "kv_heads": 8, "d": 128, "rope": 128, "norm": True, "flags": PLUS_ONE | FWHT_QK | FWHT_V, "page": 64, "dtype": "f16"},
        # a token of each request of a batch, some of its rows padding
        {"name": "append_batch", "op": "append", "rows": 250, "q_heads": 16, "kv_heads": 2, "d": 256, "rope": 64, "norm": True, "flags": PLUS_ONE, "page": 16, "dtype": "bf16"},
        # a long prompt
        {"name": "append_prompt", "op": "append", "rows": 8192, "q_heads": 40, "kv_heads": 8, "d": 128, "rope": 128, "norm": False, "flags": FWHT_QK | FWHT_V, "page": 64, "dtype": "bf16"},
        # a token of one request: latency
        {"name": "attend_token", "op": "attend", "seqs": 1, "rows": 1, "length": 4096, "q_heads": 40, "kv_heads": 8, "d": 128, "page": 64, "window": 0, "dtype": "f16"},
        # a token behind a very long context
        {"name": "attend_long", "op": "attend", "seqs": 1, "rows": 1, "length": 131077, "q_heads": 40, "kv_heads": 8, "d": 128, "page": 256, "window": 0, "dtype": "bf16"},
        # a token of each request of a batch of all lengths
        {"name": "attend_batch", "op": "attend", "seqs": 64, "rows": 1, "length": 8192, "q_heads": 40, "kv_heads": 8, "d": 128, "page": 64, "window": 0, "dtype": "bf16"},
        # verify windows of up to eight tokens, wide heads that see the last 1000 tokens, small pages
        {"name": "attend_window", "op": "attend", "seqs": 16, "rows": 8, "length": 5000, "q_heads": 16, "kv_heads": 2, "d": 256, "page": 16, "window": 1000, "dtype": "f16"},
        # a whole prompt
        {"name": "attend_prompt", "op": "attend", "seqs": 1, "rows": 4096, "length": 4096, "q_heads": 40, "kv_heads": 8, "d": 128, "page": 64, "window": 0, "dtype": "bf16"},
        # chunks of several prompts behind what they have cached, all ragged
        {"name": "attend_chunk", "op": "attend", "seqs": 6, "rows": 700, "length": 6001, "q_heads": 24, "kv_heads": 4, "d": 64, "page": 32, "window": 0, "dtype": "f16"},
    ]


def draw(rng):
    def spread(lo, hi):
        return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))

    op = rng.choice(["heads", "append", "attend", "attend"])
    flags = rng.choice([0, PLUS_ONE]) | rng.choice([0, 0, PAIRS])
    if op == "heads":
        d = 32 * rng.choice([1, 2, 3, 4, 4, 6, 8])
        k_heads = rng.randint(1, 16)
        q_heads = k_heads * rng.randint(1, 8)
        most = 8192 * 48 * 128 // ((q_heads + k_heads) * d)
        return {"op": op, "rows": spread(1, min(8192, most)), "q_heads": q_heads, "k_heads": k_heads, "d": d, "rope": rng.choice([0, 16 * rng.randint(1, d // 16), d]),
                "flags": flags | rng.choice([0, FWHT_QK]), "dtype": rng.choice(["f32", "f16", "bf16"]), "out": rng.choice(["f16", "bf16", "f32"])}
    d, kv_heads, page = rng.choice([64, 128, 128, 256]), rng.choice([1, 2, 3, 4, 8]), rng.choice([16, 32, 64, 128, 256])
    q_heads = kv_heads * rng.randint(1, 10)
    if op == "append":
        most = 8192 * 56 * 128 // ((q_heads + 2 * kv_heads) * d)
        return {"op": op, "rows": spread(1, min(8192, most)), "q_heads": rng.choice([0, q_heads]), "kv_heads": kv_heads, "d": d, "rope": rng.choice([0, 16 * rng.randint(1, d // 16), d]),
                "norm": rng.random() < 0.5, "flags": flags | rng.choice([0, FWHT_QK, FWHT_V, FWHT_QK | FWHT_V]), "page": page, "dtype": rng.choice(["f32", "f16", "bf16"])}
    kind = rng.choice(["token", "window", "chunk"])
    rows = 1 if kind == "token" else rng.randint(2, 16) if kind == "window" else spread(17, 4096)
    seqs = spread(1, 64) if kind != "chunk" else rng.randint(1, 8)
    rows = max(1, min(rows, 4096 // seqs))
    most = min(131072 if kind != "chunk" else 16384, 64 * 8192 * 8 * 128 // (seqs * kv_heads * d), 40 * 4096 * 4096 // (seqs * rows * q_heads))
    length = spread(rows, max(rows, most))
    return {"op": op, "seqs": seqs, "rows": rows, "length": length, "q_heads": q_heads, "kv_heads": kv_heads, "d": d, "page": page,
            "window": rng.choice([0, 0, 0, spread(1, length)]), "dtype": rng.choice(["f16", "bf16"])}


def _normal(shape, g, std=1.0):
    return torch.randn(shape, device="cuda", generator=g) * std


# ---- 4-bit floats and pages in plain torch ---------------------------------------------------------------------------------------
def _quantise(x):
    """x f32 [..., d] -> codes u8 [..., d / 2] (the even element in the low half), scales u8 [..., d / 32]: e2m1 elements under 2^(byte - 127)."""
    v = x.contiguous().view(*x.shape[:-1], -1, 32)
    field = (v.abs().amax(-1).view(torch.int32) >> 23) & 0xFF                         # exponent field of the largest magnitude
    broken = ~torch.isfinite(v).all(-1)
    scale = torch.where(broken, 255, torch.clamp(field - 2, min=0))                   # floor(log2) less e2m1's largest exponent
    inverse = ((254 - torch.where(broken, 127, scale)) << 23).view(torch.float32)     # 2^(127 - scale), exact
    t = torch.where(broken[..., None], 0.0, v * inverse[..., None])
    a = torch.clamp(t.abs(), max=6.0)
    step = torch.where(a < 2.0, 0.5, torch.where(a < 4.0, 1.0, 2.0))
    q = torch.round(a / step) * step                                                  # to even: the even code
    code = torch.where(q < 2.0, 2.0 * q, torch.where(q < 4.0, q + 2.0, q * 0.5 + 4.0)).to(torch.int32) | ((t.view(torch.int32) >> 28) & 8)
    code = code.view(*x.shape[:-1], x.shape[-1] // 2, 2)
    return (code[..., 0] | (code[..., 1] << 4)).to(torch.uint8), scale.to(torch.uint8)


def _values(codes, scales):
    """What the codes stand for, f32 [..., d]."""
    c = torch.stack((codes & 15, codes >> 4), -1).view(*scales.shape, 32).to(torch.int32)
    m = (c & 7).to(torch.float32)
    a = torch.where(m < 4.0, 0.5 * m, torch.where(m < 6.0, m - 2.0, 2.0 * m - 8.0))
    a = torch.where(c >= 8, -a, a)
    e = scales.to(torch.int32)
    s = torch.where(e == 0, 0x00400000, torch.where(e == 255, 0x7FC00000, e << 23)).view(torch.float32)
    return (a * s[..., None]).view(*scales.shape[:-1], -1)


# A page holds for each head: the keys' codes token by token, their scale bytes token by token; the values' codes in words of eight elements, the
# words of eight tokens side by side, and their scale bytes, eight tokens side by side too.
def _pages_of(k, v, page):
    """k, v f32 [pages, heads, page, d] -> u8 [pages, heads, bytes]."""
    (kc, ks), (vc, vs) = _quantise(k), _quantise(v)
    n, h, _, d = k.shape
    vc = vc.view(n, h, page // 8, 8, d // 8, 4).transpose(3, 4)
    vs = vs.view(n, h, page // 8, 8, d // 32).transpose(3, 4)
    return torch.cat([t.reshape(n, h, -1) for t in (kc, ks, vc, vs)], 2)


def _planes(pages, page, d):
    """u8 [..., bytes] -> codes and scales of keys and of values, token by token."""
    at = pages.shape[:-1]
    kc, ks, vc, vs = torch.split(pages, [page * d // 2, page * d // 32, page * d // 2, page * d // 32], -1)
    kc, ks = kc.reshape(*at, page, d // 2), ks.reshape(*at, page, d // 32)
    vc = vc.reshape(*at, page // 8, d // 8, 8, 4).transpose(-3, -2).reshape(*at, page, d // 2)
    vs = vs.reshape(*at, page // 8, d // 32, 8).transpose(-2, -1).reshape(*at, page, d // 32)
    return kc, ks, vc, vs


# ---- states ----------------------------------------------------------------------------------------------------------------------
def _rules(s, case, g, table, normed):
    """What a layer's program keeps for its heads: gammas and the table of cosines and sines."""
    d, rope = case["d"], case["rope"]
    centre = 0.0 if case["flags"] & PLUS_ONE else 1.0
    s["q_gamma"] = (centre + _normal((d,), g, 0.1)).half() if normed else None
    s["k_gamma"] = (centre + _normal((d,), g, 0.1)).half() if normed else None
    s["table"], s["eps"] = None, 1e-6
    if rope:
        angle = torch.arange(table, device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, rope, 2, device="cuda", dtype=torch.float64) / rope)
        s["table"] = torch.cat((torch.cos(angle), torch.sin(angle)), 1).float()


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s, d = dict(case), case["d"]
    pick = lambda n: torch.randperm(n, device="cuda", generator=g).to(torch.int32)  # noqa: E731
    if case["op"] == "heads":
        rows, width = case["rows"], (case["q_heads"] + 2 * case["k_heads"]) * d      # the projection's rows: q, k, v
        s["qkv"] = _normal((rows, width), g).to(TYPES[case["dtype"]])
        _rules(s, case, g, rows + 1000, True)
        s["position"] = pick(rows + 1000)[:rows].clone()
        s["q_out"] = torch.empty(rows, case["q_heads"], d, dtype=TYPES[case["out"]], device="cuda")
        s["k_out"] = torch.empty(rows, case["k_heads"], d, dtype=TYPES[case["out"]], device="cuda")
    elif case["op"] == "append":
        rows, heads, page = case["rows"], case["kv_heads"], case["page"]
        s["qkv"] = _normal((rows, (case["q_heads"] + 2 * heads) * d), g).to(TYPES[case["dtype"]])
        _rules(s, case, g, rows + 1000, case["norm"])
        s["position"] = pick(rows + 1000)[:rows].clone()
        s["page_count"] = (rows + 1000) // page + 1
        slots = pick(s["page_count"] * page)[:rows].clone()
        if rows > 1000:                                                              # a prompt: token after token, page after page
            at = torch.arange(rows, device="cuda")
            slots = (pick(s["page_count"])[at // page] * page + at % page).to(torch.int32)
        s["slots"] = torch.where(torch.rand(rows, device="cuda", generator=g) < (0.1 if 10 < rows < 1000 else 0.0), torch.full_like(slots, -1), slots)
        s["pages"] = torch.zeros(s["page_count"], heads, page * d * 34 // 32, dtype=torch.uint8, device="cuda")
        out = TYPES[case["dtype"]]
        s["q_out"] = torch.zeros(rows, case["q_heads"], d, dtype=out, device="cuda")
        s["k_values"], s["v_values"] = (torch.zeros(rows, heads, d, dtype=out, device="cuda") for _ in range(2))
    else:
        seqs, most, longest, heads, page = case["seqs"], case["rows"], case["length"], case["kv_heads"], case["page"]
        of = lambda n: torch.rand(seqs, generator=torch.Generator().manual_seed(n))  # noqa: E731
        rows = (most * (1.0 - 0.5 * of(seqs))).ceil().long().clamp(1, most)          # the step's plan: requests bring different numbers of rows
        if seqs > 8 and most > 1:
            rows[3] = 0                                                              # one that has nothing to do in this step
        rows[0] = most
        lengths = torch.maximum((longest * (1.0 - 0.9 * of(seed) ** 2)).long().clamp(1, longest), rows)
        lengths[0] = longest
        start = torch.cat((torch.zeros(1, dtype=torch.int64), rows.cumsum(0)))
        total = int(start[-1]) + (1 if seqs > 1 else 0)                              # and a row of padding behind the last
        s["row_start"], s["lengths"] = start.to(torch.int32).cuda(), lengths.to(torch.int32).cuda()
        s["q"] = _normal((total, case["q_heads"], d), g, 1.5).to(TYPES[case["dtype"]])
        each = (longest + page - 1) // page
        s["table"] = pick(seqs * each).view(seqs, each)
        s["pages"] = torch.empty(seqs * each, heads, page * d * 34 // 32, dtype=torch.uint8, device="cuda")
        step = max(1, (1 << 25) // (heads * page * d))
        for i in range(0, seqs * each, step):                                        # large caches by pieces: less memory
            n = min(step, seqs * each - i)
            s["pages"][i:i + n] = _pages_of(_normal((n, heads, page, d), g), _normal((n, heads, page, d), g), page)
        s["scale"] = d ** -0.5
        s["out"], s["lse"] = torch.zeros_like(s["q"]), torch.zeros(total, case["q_heads"], device="cuda")
        s["workspace"] = torch.empty(ATTEND_WORKSPACE, dtype=torch.uint8, device="cuda")
    return s


# ---- one pass --------------------------------------------------------------------------------------------------------------------
def run(state):
    if own:
        return _own(state)
    if state["op"] == "heads":
        q, k, _ = _split(state, state["k_heads"])
        out = TYPES[state["out"]]
        return {"q": _head(q, state, state["q_gamma"], FWHT_QK).to(out), "k": _head(k, state, state["k_gamma"], FWHT_QK).to(out)}
    if state["op"] == "append":
        return _append(state)
    return _attend(state)


def _split(s, k_heads):
    x = s["qkv"].view(s["rows"], -1, s["d"]).float()
    return x[:, : s["q_heads"]], x[:, s["q_heads"] : s["q_heads"] + k_heads], x[:, s["q_heads"] + k_heads :]


def _halve(t):
    """The sum over the last axis as a tree, halves onto halves."""
    while t.shape[-1] > 1:
        h = t.shape[-1] // 2
        t = t[..., :h] + t[..., h:]
    return t[..., 0]


def _head(x, s, gamma, fwht, rope=True):
    """Norm, rotation and transform of x f32 [rows, heads, d], an operation and its rounding after the other: what comes out may be next to a border of
    the 4-bit grid.  The squares' sum goes by eights first, as a tree, then over the eights."""
    d = s["d"]
    if gamma is not None:
        sums = _halve((x * x).view(*x.shape[:-1], d // 8, 8))
        room = 1 << (d // 8 - 1).bit_length()
        sums = _halve(torch.cat((sums, sums.new_zeros(*sums.shape[:-1], room - d // 8)), -1))
        inv = 1.0 / torch.sqrt(sums / d + s["eps"])
        g = gamma.float() + 1.0 if s["flags"] & PLUS_ONE else gamma.float()
        x = (x * inv[..., None]) * g
    if rope and s["rope"]:
        n = s["rope"]
        c, sn = s["table"][s["position"].long()][:, None].split(n // 2, -1)
        if s["flags"] & PAIRS:
            a, b = x[..., 0:n:2], x[..., 1:n:2]
            x = torch.cat((torch.stack((a * c - b * sn, b * c + a * sn), -1).flatten(-2), x[..., n:]), -1)
        else:
            a, b = x[..., : n // 2], x[..., n // 2 : n]
            x = torch.cat((a * c - b * sn, b * c + a * sn, x[..., n:]), -1)
    if s["flags"] & fwht:
        y = x.reshape(-1, 32)
        y = _butterfly(_butterfly(_butterfly(_butterfly(_butterfly(y, 1), 2), 4), 8), 16)
        x = (y * INV_SQRT32).view(x.shape)
    return x


def _butterfly(y, h):
    p = y.view(-1, 16 // h, 2, h)
    return torch.stack((p[:, :, 0] + p[:, :, 1], p[:, :, 0] - p[:, :, 1]), 2).view(-1, 32)


def _append(s):
    q, k, v = _split(s, s["kv_heads"])
    out, page, d = s["q_out"].dtype, s["page"], s["d"]
    q, k, v = _head(q, s, s["q_gamma"], FWHT_QK), _head(k, s, s["k_gamma"], FWHT_QK), _head(v, s, None, FWHT_V, False)
    (kc, ks), (vc, vs) = _quantise(k), _quantise(v)
    there = s["slots"] >= 0
    # the pages: a row of padding goes to a page behind the last
    at = torch.where(there, s["slots"], s["page_count"] * page).long()
    p, t = at // page, at % page
    rows, heads = s["rows"], s["kv_heads"]
    pages = torch.cat((s["pages"], s["pages"].new_zeros(1, heads, s["pages"].shape[2])))
    a, b = page * d // 2, page * d // 32
    pages[:, :, :a].view(-1, heads, page, d // 2)[p, :, t] = kc
    pages[:, :, a : a + b].view(-1, heads, page, d // 32)[p, :, t] = ks
    pages[:, :, a + b : 2 * a + b].view(-1, heads, page // 8, d // 8, 8, 4)[p, :, t // 8, :, t % 8] = vc.view(rows, heads, d // 8, 4)
    pages[:, :, 2 * a + b :].view(-1, heads, page // 8, d // 32, 8)[p, :, t // 8, :, t % 8] = vs
    s["pages"].copy_(pages[:-1])
    m = there[:, None, None]
    return {"q": torch.where(m, q, 0.0).to(out), "k": torch.where(m, _values(kc, ks), 0.0).to(out), "v": torch.where(m, _values(vc, vs), 0.0).to(out)}


def _attend(s):
    seqs, most, heads, d, page, q_heads = s["seqs"], s["rows"], s["kv_heads"], s["d"], s["page"], s["q_heads"]
    shared, total = q_heads // heads, s["q"].shape[0]
    kc, ks, vc, vs = _planes(s["pages"][s["table"].long()].transpose(1, 2), page, d)         # [seqs, heads, pages, page, ..]
    k, v = (_values(c, e).view(seqs, heads, -1, d) for c, e in ((kc, ks), (vc, vs)))
    long = k.shape[2]
    start, n = s["row_start"][:-1].long(), (s["row_start"][1:] - s["row_start"][:-1]).long()
    i = torch.arange(most, device="cuda")
    q = s["q"].float()[(start[:, None] + i).clamp(max=total - 1)]                            # [seqs, most, q_heads, d]
    q = q.view(seqs, most, heads, shared, d).permute(0, 2, 1, 3, 4).reshape(seqs, heads, most * shared, d)
    l = (q @ k.transpose(2, 3)).view(seqs, heads, most, shared, long) * s["scale"]
    at = (s["lengths"].long() - n)[:, None] + i                                              # a row's position
    j = torch.arange(long, device="cuda")
    sees = j <= at[:, :, None]
    if s["window"]:
        sees = sees & (j > at[:, :, None] - s["window"])
    l = torch.where(sees[:, None, :, None], l, float("-inf"))
    top = l.amax(-1, keepdim=True)
    top = torch.where(top == float("-inf"), 0.0, top)
    p = torch.exp(l - top)
    del l
    sum_ = p.sum(-1, keepdim=True)
    o = (p.view(seqs, heads, most * shared, long) @ v).view(seqs, heads, most, shared, d) / torch.where(sum_ > 0, sum_, 1.0)
    lse = (top + torch.log(sum_))[..., 0]
    r = torch.arange(total, device="cuda")                                                   # back to packed rows
    seq = (torch.searchsorted(s["row_start"].long(), r, right=True) - 1).clamp(max=seqs - 1)
    row, there = (r - start[seq]).clamp(max=most - 1), r < s["row_start"][-1]
    o = o.permute(0, 2, 1, 3, 4).reshape(seqs, most, q_heads, d)[seq, row]
    lse = lse.permute(0, 2, 1, 3).reshape(seqs, most, q_heads)[seq, row]
    return {"out": torch.where(there[:, None, None], o, 0.0).to(s["q"].dtype), "lse": torch.where(there[:, None], lse, 0.0)}


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
    at = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    d = s["d"]
    if s["op"] == "attend":
        cache = q.KvCache(at(s["pages"]), s["pages"].numel(), s["pages"].shape[0], s["page"], s["kv_heads"], d)
        batch = q.KvBatch(row_start=at(s["row_start"]), lengths=at(s["lengths"]), block_table=at(s["table"]), ld_table=s["table"].shape[1], seqs=s["seqs"], max_rows=s["rows"],
                          max_length=s["length"])
        return lib.qwhip_kv_attention_mxfp4, (st, q.C.byref(cache), q.C.byref(batch), at(s["q"]), CODE[s["dtype"]], s["q_heads"], 0, s["q"].shape[0], s["scale"], s["window"],
                                              at(s["out"]), 0, at(s["lse"]), at(s["workspace"]), ATTEND_WORKSPACE), {"out": s["out"], "lse": s["lse"]}
    rules = q.HeadRules(position=at(s["position"]), cos_sin=at(s["table"]), q_gamma=at(s["q_gamma"]), k_gamma=at(s["k_gamma"]), positions=0 if s["table"] is None else s["table"].shape[0],
                        rope_dims=s["rope"], eps=s["eps"], flags=s["flags"])
    rows, ld, size = s["rows"], s["qkv"].shape[1], s["qkv"].element_size()
    k = at(s["qkv"]) + s["q_heads"] * d * size
    if s["op"] == "heads":
        return lib.qwhip_head_norm_rope, (st, q.C.byref(rules), rows, d, at(s["qkv"]), s["q_heads"], ld, k, s["k_heads"], ld, CODE[s["dtype"]], at(s["q_out"]), 0, at(s["k_out"]), 0,
                                          CODE[s["out"]]), {"q": s["q_out"], "k": s["k_out"]}
    cache = q.KvCache(at(s["pages"]), s["pages"].numel(), s["page_count"], s["page"], s["kv_heads"], d)
    return lib.qwhip_kv_append_mxfp4, (st, q.C.byref(cache), q.C.byref(rules), rows, at(s["slots"]), k, ld, k + s["kv_heads"] * d * size, ld, CODE[s["dtype"]],
                                       at(s["qkv"]), s["q_heads"], ld, at(s["q_out"]), 0, CODE[s["dtype"]], at(s["k_values"]), at(s["v_values"])), {
                                           "q": s["q_out"], "k": s["k_values"], "v": s["v_values"]}


# ---- what a pass cannot do without -----------------------------------------------------------------------------------------------
def work(case):
    d = case["d"]
    if case["op"] == "heads":
        e = case["rows"] * (case["q_heads"] + case["k_heads"]) * d
        return {"bytes": e * (TYPES[case["dtype"]].itemsize + TYPES[case["out"]].itemsize) + case["rows"] * case["rope"] * 4, "flops": 10 * e}
    if case["op"] == "append":
        e, q, size = case["rows"] * 2 * case["kv_heads"] * d, case["rows"] * case["q_heads"] * d, TYPES[case["dtype"]].itemsize
        return {"bytes": 2 * (e + q) * size + e * 17 // 32 + case["rows"] * case["rope"] * 4, "flops": 12 * (e + q)}
    # of sequences that are 0.7 of the longest on average, and 0.75 of the most rows
    some, more = (1.0, 1.0) if case["seqs"] == 1 else (0.7, 0.75 if case["rows"] > 1 else 1.0)
    length, rows = some * case["length"], more * case["rows"]
    seen = min(length, case["window"] + rows) if case["window"] else length
    pairs = rows * (min(length, case["window"]) if case["window"] else length - min(rows, length) / 2)
    return {"bytes": int(case["seqs"] * (seen * case["kv_heads"] * d * 34 // 32 + rows * case["q_heads"] * (4 * d + 4))), "flops": int(case["seqs"] * pairs * case["q_heads"] * 4 * d)}


# ---- the definitions, in 64 bits ---------------------------------------------------------------------------------------------------
GRID = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _wide_head(x, s, gamma, fwht, rope=True):
    x = x.double()
    if x.numel() == 0:
        return x
    if gamma is not None:
        x = x * (x.square().mean(-1, keepdim=True) + s["eps"]).rsqrt() * (gamma.double() + (1.0 if s["flags"] & PLUS_ONE else 0.0))
    if rope and s["rope"]:
        n = s["rope"]
        turn = torch.complex(*(t.contiguous().double() for t in s["table"][s["position"].long()][:, None].chunk(2, -1)))
        part = x[..., :n].unflatten(-1, (n // 2, 2)) if s["flags"] & PAIRS else x[..., :n].unflatten(-1, (2, n // 2)).transpose(-1, -2)
        part = torch.view_as_real(torch.view_as_complex(part.contiguous()) * turn)
        x = torch.cat(((part if s["flags"] & PAIRS else part.transpose(-1, -2)).flatten(-2), x[..., n:]), -1)
    if s["flags"] & fwht:
        h = torch.ones(1, 1, dtype=torch.float64, device="cuda")
        for _ in range(5):
            h = torch.cat((torch.cat((h, h), 1), torch.cat((h, -h), 1)))
        x = (x.reshape(-1, 32) @ h / 32.0 ** 0.5).view(x.shape)
    return x


def _wide_nearest(x):
    b = x.reshape(-1, 32)
    top = b.abs().amax(1, keepdim=True)
    unit = torch.exp2(torch.clamp(torch.frexp(top).exponent - 3, min=-127).double())
    grid = torch.tensor(GRID, dtype=torch.float64, device="cuda")
    between = 0.5 * (grid[1:] + grid[:-1])
    a = b.abs() / unit
    low, high = torch.bucketize(a, between, right=False), torch.bucketize(a, between, right=True)
    return (grid[torch.where(low % 2 == 0, low, high)] * torch.sign(b) * unit).view(x.shape)


def _wide_values(codes, scales):
    table = torch.tensor(GRID + [-x for x in GRID], dtype=torch.float64, device="cuda")
    v = torch.empty(*codes.shape[:-1], codes.shape[-1] * 2, dtype=torch.float64, device="cuda")
    v[..., 0::2], v[..., 1::2] = table[(codes % 16).int()], table[(codes // 16).int()]
    return v * torch.exp2(scales.double() - 127.0).repeat_interleave(32, -1)


def exact(case, seed):
    s, d = prepare(case, seed), case["d"]
    if case["op"] in ("heads", "append"):
        heads = case["k_heads"] if case["op"] == "heads" else case["kv_heads"]
        q, k, v = s["qkv"].view(case["rows"], -1, d).split([case["q_heads"], heads, heads], 1)
        q, k = _wide_head(q, s, s["q_gamma"], FWHT_QK), _wide_head(k, s, s["k_gamma"], FWHT_QK)
        if case["op"] == "heads":
            return {"q": q, "k": k}
        v = _wide_head(v, s, None, FWHT_V, False)
        there = (s["slots"] >= 0).double()[:, None, None]
        return {"q": q * there, "k": _wide_nearest(k) * there, "v": _wide_nearest(v) * there}
    page, heads, shared = case["page"], case["kv_heads"], case["q_heads"] // case["kv_heads"]
    out, lse = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), torch.zeros(s["lse"].shape, dtype=torch.float64, device="cuda")
    start, lengths = s["row_start"].tolist(), s["lengths"].tolist()
    for i in range(case["seqs"]):
        n, long = start[i + 1] - start[i], lengths[i]
        if n == 0:
            continue
        mine = s["pages"][s["table"][i, : (long + page - 1) // page].long()]
        first = torch.arange(long, device="cuda")
        row = torch.arange(long - n, long, device="cuda")[:, None]
        hidden = (first > row) | ((first <= row - case["window"]) if case["window"] else torch.zeros_like(first > row))
        for h in range(heads):
            kc, ks, vc, vs = _planes(mine[:, h], page, d)
            k, v = (_wide_values(c.reshape(-1, d // 2)[:long], e.reshape(-1, d // 32)[:long]) for c, e in ((kc, ks), (vc, vs)))
            for a in range(h * shared, (h + 1) * shared):
                x = torch.mm(s["q"][start[i] : start[i + 1], a].double(), k.t()) * s["scale"]
                x = x.masked_fill(hidden, float("-inf"))
                lse[start[i] : start[i + 1], a] = torch.logsumexp(x, 1)
                out[start[i] : start[i + 1], a] = torch.mm(torch.softmax(x, 1), v)
    return {"out": out, "lse": lse}
