"""What the operators of an autoregressive acoustic model's step cost: rotary positions, appending to a paged key/value cache,
attention over that cache, and products with 4-bit weights.

The step is the one a streaming speech model takes between its text and the vocoder: a stack of decoder layers (1024 channels in 16
heads is the size this package's streaming vocoder is fed by) reads a prompt of text tokens in one chunk, then makes one audio token
at a time for every request in flight.  `run` computes a case either in plain torch (`own` false) or through tts_amd.ops."""
import math

import torch

own = False
DEV = "cuda:0"
TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


# ---------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # the queries of one step of 24 streaming requests
        dict(name="rotary_step", op="rotary", dtype="bfloat16", tokens=24, heads=16, head_dim=64, rotary_dim=64, interleaved=False,
             scaling="none", factor=1.0, far=1000),
        # long documents read at far positions: pairs side by side in half of the head, frequencies stretched for a longer context
        dict(name="rotary_prompt", op="rotary", dtype="float32", tokens=8192, heads=32, head_dim=128, rotary_dim=64, interleaved=True,
             scaling="ramp", factor=8.0, far=120000),
        # one step of 48 requests: a key, a value and a query each
        dict(name="append_step", op="append", dtype="float16", seqs=48, new=1, ragged=False, ctx=1007, kv_heads=16, heads=16, head_dim=64,
             page=16, rotary_dim=64, interleaved=False, scaling="none", factor=1.0),
        # ragged prompts of a few requests, keys shared by groups of four heads
        dict(name="append_prompt", op="append", dtype="bfloat16", seqs=6, new=1500, ragged=True, ctx=2000, kv_heads=8, heads=32,
             head_dim=128, page=64, rotary_dim=128, interleaved=False, scaling="linear", factor=4.0),
        # one streaming request, one token: latency alone
        dict(name="attend_one", op="attend", dtype="float32", seqs=1, new=1, ragged=False, ctx=605, kv_heads=16, heads=16, head_dim=64,
             page=16, window=0),
        # one step of 48 requests of all lengths
        dict(name="attend_step", op="attend", dtype="float16", seqs=48, new=1, ragged=False, ctx=1007, kv_heads=16, heads=16, head_dim=64,
             page=16, window=0),
        # a few very long conversations, one token each, eight heads to a key
        dict(name="attend_far", op="attend", dtype="bfloat16", seqs=3, new=1, ragged=False, ctx=65537, kv_heads=4, heads=32, head_dim=128,
             page=64, window=0),
        # text prompts of two requests, in the package's own type
        dict(name="attend_prompt", op="attend", dtype="float32", seqs=2, new=437, ragged=True, ctx=437, kv_heads=16, heads=16, head_dim=64,
             page=32, window=0),
        # a chunk of a long prompt behind what earlier chunks left in the cache
        dict(name="attend_chunk", op="attend", dtype="bfloat16", seqs=2, new=2048, ragged=False, ctx=8191, kv_heads=8, heads=32,
             head_dim=128, page=64, window=0),
        # the first product of a layer's feed-forward part, one request
        dict(name="w4_one", op="w4", dtype="bfloat16", rows=1, inner=1024, outer=4096, group=64, zeros=False),
        # its second product, 24 requests in the package's own type, weights with zero points
        dict(name="w4_step", op="w4", dtype="float32", rows=24, inner=4096, outer=1024, group=32, zeros=True),
        # a wide layer, one request
        dict(name="w4_wide", op="w4", dtype="float16", rows=1, inner=8192, outer=8192, group=128, zeros=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "append", "attend", "attend", "w4"])
    dtype = rng.choice(sorted(TYPES))
    if op == "w4":
        group = rng.choice([32, 64, 128])
        inner, outer = group * _log(rng, 2, 8192 // group), _log(rng, 64, 8192)
        return dict(op=op, dtype=dtype, rows=_log(rng, 1, 64), inner=inner, outer=outer, group=group, zeros=rng.random() < 0.5)
    head_dim = 8 * rng.choice([4, 6, 8, 8, 10, 12, 16, 16, 24, 32])
    turn = dict(rotary_dim=rng.choice([head_dim, head_dim, head_dim // 2]), interleaved=rng.random() < 0.5,
                scaling=rng.choice(["none", "linear", "base", "ramp"]), factor=rng.choice([2.0, 4.0, 8.0, 32.0]))
    kv_heads = rng.choice([1, 2, 4, 8, 16])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 8] if kv_heads < 8 else [1, 2, 4])
    if op == "rotary":
        tokens = _log(rng, 1, max(1, (1 << 24) // (heads * head_dim)))
        return dict(op=op, dtype=dtype, tokens=tokens, heads=heads, head_dim=head_dim, far=_log(rng, 1, 1000000), **turn)
    page = rng.choice([1, 8, 16, 16, 24, 32, 64, 128])
    if rng.random() < 0.5:                                  # a step of many requests
        new, ragged = 1, False
        ctx = _log(rng, 1, 32768)
        seqs = _log(rng, 1, max(1, min(96, (1 << 25) // (ctx * kv_heads * head_dim))))
    else:                                                   # chunks of a prompt
        new = _log(rng, 2, 1500 if dtype != "float32" else 700)
        ragged = rng.random() < 0.7
        ctx = new + _log(rng, 1, 4096) - 1
        while new * ctx * heads * head_dim > 1 << 35:
            new, ctx = max(2, new // 2), max(2, ctx // 2)
        seqs = _log(rng, 1, max(1, min(6, (1 << 35) // (new * ctx * heads * head_dim))))
    case = dict(op=op, dtype=dtype, seqs=seqs, new=new, ragged=ragged, ctx=ctx, kv_heads=kv_heads, heads=heads, head_dim=head_dim, page=page)
    return dict(case, **turn) if op == "append" else dict(case, window=rng.choice([0, 0, _log(rng, 1, ctx)]))


# --------------------------------------------------------------------------------------------------------------- inputs
def _lengths(case):
    """New tokens and tokens in all of every sequence: the same for every seed, so that a case is one amount of work."""
    new, ctx = [], []
    for b in range(case["seqs"]):
        n = case["new"] if not case["ragged"] else max(1, case["new"] - (b * 7919) % max(1, case["new"] * 3 // 4))
        spread = case["ctx"] if case["seqs"] == 1 else max(n, case["ctx"] - (b * 104729) % max(1, case["ctx"] // 2))
        new.append(n)
        ctx.append(max(n, spread))
    return new, ctx


def _frequencies(case):
    """Radians a position for every rotated pair, and the factor on the rotated values."""
    rd, f, kind = case["rotary_dim"], case["factor"], case["scaling"]
    base = 10000.0 * f ** (rd / (rd - 2.0)) if kind == "base" else 10000.0
    freq = base ** (-torch.arange(0, rd, 2, dtype=torch.float64) / rd)
    if kind == "linear":
        return freq / f, 1.0
    if kind == "ramp":                 # by how often a pair turned round within the length that was trained on
        keep = ((4096 * freq / (2 * math.pi) - 1.0) / (32.0 - 1.0)).clamp(0, 1)
        return freq / f * (1 - keep) + freq * keep, 0.1 * math.log(f) + 1.0
    return freq, 1.0


def _scaling(case):
    if case["scaling"] == "none":
        return None
    extra = dict(trained_len=4096, low=1.0, high=32.0) if case["scaling"] == "ramp" else {}
    return dict(kind=case["scaling"], factor=case["factor"], **extra)


def _rotary_plan(case):
    from tts_amd import ops

    return ops.Rotary(case["head_dim"], case["rotary_dim"], interleaved=case["interleaved"], scaling=_scaling(case), device=DEV)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    dt = TYPES[case["dtype"]]
    new = lambda *shape: torch.randn(shape, generator=g, device=DEV).to(dt)  # noqa: E731
    s = dict(case=case)
    if case["op"] == "w4":
        n, k, grp = case["outer"], case["inner"], case["group"]
        s["x"] = new(case["rows"], k)
        s["q"] = torch.randint(0, 256, (n, k // 2), generator=g, device=DEV, dtype=torch.uint8)      # two levels a byte, the even one low
        s["scales"] = ((torch.rand((n, k // grp), generator=g, device=DEV) + 0.5) * (0.25 / math.sqrt(k))).to(dt)
        s["zeros"] = torch.randint(5, 11, (n, k // grp), generator=g, device=DEV, dtype=torch.uint8) if case["zeros"] else None
        s["bias"] = new(n)
        if own:
            from tts_amd import ops

            s["weights"] = ops.PackedW4(s["q"], s["scales"], zeros=s["zeros"], bias=s["bias"])
        return s
    if case["op"] in ("rotary", "append"):
        freq, s["amplitude"] = _frequencies(case)
        s["freq"] = freq.to(DEV)
        if own:
            s["plan"] = _rotary_plan(case)
    if case["op"] == "rotary":
        start = torch.randint(0, case["far"], (1,), generator=g, device=DEV)
        s["positions"] = start + torch.arange(case["tokens"], device=DEV)
        s["x"] = new(case["tokens"], case["heads"], case["head_dim"])
        return s
    n, ctx = _lengths(case)
    b, ps, width = case["seqs"], case["page"], -(-max(ctx) // case["page"])
    owned = [-(-c // ps) for c in ctx]
    pages = sum(owned) + 3
    order = torch.randperm(pages, generator=g, device=DEV, dtype=torch.int32)
    have = torch.tensor(owned, device=DEV)
    first = torch.cumsum(have, 0) - have
    col = torch.arange(width, device=DEV)
    s["table"] = torch.where(col < have[:, None], order[(first[:, None] + col).clamp(max=pages - 1)], -1).to(torch.int32)
    s["lens"] = torch.tensor(ctx, device=DEV, dtype=torch.int32)
    s["starts"] = torch.cumsum(torch.tensor([0] + n, device=DEV), 0).to(torch.int32)
    s["k_cache"], s["v_cache"] = (new(pages, case["kv_heads"], ps, case["head_dim"]) for _ in range(2))
    s["max_new"], s["max_len"] = max(n), max(ctx)
    s["q"] = new(sum(n), case["heads"], case["head_dim"])
    if case["op"] == "append":
        s["k"], s["v"] = (new(sum(n), case["kv_heads"], case["head_dim"]) for _ in range(2))
    if own:
        from tts_amd import ops

        s["cache"] = ops.PagedKV(s["k_cache"], s["v_cache"])
        s["batch"] = ops.PagedBatch(s["table"], s["lens"], s["starts"], max_new=s["max_new"], max_len=s["max_len"])
    return s


# ----------------------------------------------------------------------------------------------------------- plain forms
def _turned(x, positions, freq, amplitude, interleaved):
    rd = 2 * freq.numel()
    angle = positions.double()[:, None] * freq
    c, s = (angle.cos() * amplitude).float()[:, None, :], (angle.sin() * amplitude).float()[:, None, :]
    x32 = x.float()
    out = x32.clone()
    if interleaved:
        x1, x2 = x32[..., 0:rd:2], x32[..., 1:rd:2]
        out[..., 0:rd:2], out[..., 1:rd:2] = x1 * c - x2 * s, x2 * c + x1 * s
    else:
        x1, x2 = x32[..., : rd // 2], x32[..., rd // 2: rd]
        out[..., : rd // 2], out[..., rd // 2: rd] = x1 * c - x2 * s, x2 * c + x1 * s
    return out.to(x.dtype)


def _plain_rotary(s):
    return _turned(s["x"], s["positions"], s["freq"], s["amplitude"], s["case"]["interleaved"])


def _plain_append(s):
    case = s["case"]
    token = torch.arange(s["k"].shape[0], device=DEV)
    seq = (token[:, None] >= s["starts"][None, 1:]).sum(1)
    pos = s["lens"].long()[seq] - s["starts"].long()[seq + 1] + token
    page, row = s["table"].long()[seq, pos // case["page"]], pos % case["page"]
    s["k_cache"][page, :, row] = _turned(s["k"], pos, s["freq"], s["amplitude"], case["interleaved"])
    s["v_cache"][page, :, row] = s["v"]
    return s["k_cache"], s["v_cache"], _turned(s["q"], pos, s["freq"], s["amplitude"], case["interleaved"])


def _plain_attend(s):
    case = s["case"]
    b, hk, d, n, top = case["seqs"], case["kv_heads"], case["head_dim"], s["max_new"], s["max_len"]
    g = case["heads"] // hk
    starts, lens = s["starts"].long(), s["lens"].long()
    count = starts[1:] - starts[:-1]
    pages = s["table"].long().clamp(min=0)
    key = torch.arange(top, device=DEV)
    there = key < lens[:, None]                                                              # [b, top]
    k, v = (c[pages].transpose(2, 3).reshape(b, -1, hk, d)[:, :top].transpose(1, 2).float() for c in (s["k_cache"], s["v_cache"]))
    v = torch.where(there[:, None, :, None], v, 0.0)
    i = torch.arange(n, device=DEV)
    token = (starts[:-1, None] + i).clamp(max=s["q"].shape[0] - 1)
    q = s["q"][token].float().reshape(b, n, hk, g, d).permute(0, 2, 1, 3, 4).reshape(b, hk, n * g, d)
    pos = lens[:, None] - count[:, None] + i                                                 # [b, n]
    seen = there[:, None, :] & (key <= pos[:, :, None])
    if case["window"]:
        seen = seen & (key > pos[:, :, None] - case["window"])
    seen = seen.repeat_interleave(g, 1)[:, None]                                             # [b, 1, n * g, top]
    w = torch.where(seen, torch.matmul(q, k.transpose(2, 3).contiguous()) * (1.0 / math.sqrt(d)), -math.inf)
    w = torch.where(seen, torch.exp(w - w.amax(-1, keepdim=True).clamp(min=-3e38)), 0.0)
    o = torch.matmul(w, v) / w.sum(-1, keepdim=True).clamp(min=1e-37)
    o = o.reshape(b, hk, n, g, d).permute(0, 2, 1, 3, 4).reshape(b, n, hk * g, d)
    return o[i < count[:, None]].to(s["q"].dtype)


def _plain_w4(s):
    grp = s["case"]["group"]
    n, half = s["q"].shape
    levels = torch.stack([s["q"] & 15, s["q"] >> 4], -1).reshape(n, 2 * half // grp, grp).float()
    zeros = 8.0 if s["zeros"] is None else s["zeros"].float()[..., None]
    w = ((levels - zeros) * s["scales"].float()[..., None]).reshape(n, 2 * half)
    return (torch.matmul(s["x"].float(), w.t().contiguous()) + s["bias"].float()).to(s["x"].dtype)


def run(s):
    op = s["case"]["op"]
    if own:
        from tts_amd import ops

        if op == "rotary":
            return ops.rotary(s["plan"], s["x"], s["positions"])
        if op == "append":
            q = ops.kv_append(s["cache"], s["batch"], s["k"], s["v"], rotary=s["plan"], q=s["q"])
            return s["k_cache"], s["v_cache"], q
        if op == "attend":
            return ops.paged_attention(s["q"], s["cache"], s["batch"], window=s["case"]["window"])
        return ops.linear_w4(s["weights"], s["x"])
    if op == "rotary":
        return _plain_rotary(s)
    if op == "append":
        return _plain_append(s)
    return _plain_attend(s) if op == "attend" else _plain_w4(s)


# ------------------------------------------------------------------------------------------------------------ the work
def work(case):
    e = torch.empty((), dtype=TYPES[case["dtype"]]).element_size()
    if case["op"] == "w4":
        n, k, m = case["outer"], case["inner"], case["rows"]
        groups = n * (k // case["group"])
        return {"bytes": n * k / 2 + groups * (e + (1 if case["zeros"] else 0)) + e * (m * k + m * n + n), "flops": 2.0 * m * n * k}
    if case["op"] == "rotary":
        x = case["tokens"] * case["heads"] * case["head_dim"]
        return {"bytes": 2 * e * x + 8 * case["tokens"], "flops": 3.0 * x * case["rotary_dim"] / case["head_dim"]}
    n, ctx = _lengths(case)
    d, hq, hk = case["head_dim"], case["heads"], case["kv_heads"]
    table = 4 * sum(-(-c // case["page"]) for c in ctx)
    if case["op"] == "append":
        return {"bytes": sum(n) * (4 * hk + 2 * hq) * d * e + table, "flops": 3.0 * sum(n) * (hk + hq) * case["rotary_dim"]}
    pairs = read = 0
    for a, c in zip(n, ctx):
        win = case["window"] or c
        pairs += sum(min(win, c - a + i + 1) for i in range(a))
        read += min(c, win + a - 1)
    return {"bytes": 2 * e * read * hk * d + 2 * e * sum(n) * hq * d + table, "flops": 4.0 * pairs * hq * d}


# ------------------------------------------------------------------------------------------------ the definition, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    up = lambda t: t.to(torch.float64)  # noqa: E731

    def spin(x, pos):
        """Every pair as a complex number times its own unit one."""
        half = case["rotary_dim"] // 2
        i = torch.arange(half, device=DEV, dtype=torch.float64)
        f = torch.exp(i * (-2.0 * math.log(10000.0) / case["rotary_dim"]))
        gain, c = 1.0, case["factor"]
        if case["scaling"] == "base":
            f = torch.exp(i * (-2.0 * (math.log(10000.0) + math.log(c) * half / (half - 1.0)) / case["rotary_dim"]))
        elif case["scaling"] == "linear":
            f = f / c
        elif case["scaling"] == "ramp":
            keep = torch.clamp((4096 * f / (2 * math.pi) - 1) / 31, 0, 1)
            f, gain = f * (keep + (1 - keep) / c), 1 + math.log(c) / 10
        unit = torch.polar(torch.full_like(f, gain)[None].repeat(pos.numel(), 1), up(pos)[:, None] * f[None])[:, None]
        head, rest = up(x[..., : 2 * half]), up(x[..., 2 * half:])
        two = head.unflatten(-1, (half, 2)) if case["interleaved"] else head.unflatten(-1, (2, half)).transpose(-1, -2)
        two = torch.view_as_real(torch.view_as_complex(two.contiguous()) * unit)
        two = two if case["interleaved"] else two.transpose(-1, -2)
        return torch.cat([two.flatten(-2), rest], -1)

    if case["op"] == "rotary":
        return spin(s["x"], s["positions"])
    if case["op"] == "w4":
        q = up(s["q"]).reshape(case["outer"], -1, 1)
        levels = torch.cat([torch.remainder(q, 16), torch.floor(q / 16)], -1).flatten(1)
        each = torch.arange(case["inner"], device=DEV) // case["group"]
        zeros = torch.full_like(s["scales"], 8) if s["zeros"] is None else s["zeros"]
        w = up(s["scales"])[:, each] * (levels - up(zeros)[:, each])
        return torch.addmm(up(s["bias"])[None], up(s["x"]), w.T)
    starts, lens, table, ps = s["starts"].tolist(), s["lens"].tolist(), s["table"].tolist(), case["page"]
    if case["op"] == "append":
        kc, vc, turned = up(s["k_cache"]), up(s["v_cache"]), []
        for b in range(case["seqs"]):
            mine = slice(starts[b], starts[b + 1])
            pos = torch.arange(lens[b] - (starts[b + 1] - starts[b]), lens[b], device=DEV)
            slot = torch.tensor(table[b], device=DEV)[pos // ps] * ps + pos % ps
            for c, x in ((kc, spin(s["k"][mine], pos)), (vc, up(s["v"][mine]))):
                c.transpose(1, 2)[slot // ps, slot % ps] = x
            turned.append(spin(s["q"][mine], pos))
        return kc, vc, torch.cat(turned)
    out = []
    g = case["heads"] // case["kv_heads"]
    for b in range(case["seqs"]):
        q = up(s["q"][starts[b]: starts[b + 1]])
        n, c = q.shape[0], lens[b]
        pages = torch.tensor(table[b][: -(-c // ps)], device=DEV)
        k, v = (up(t[pages]).permute(1, 0, 2, 3).flatten(1, 2)[:, :c] for t in (s["k_cache"], s["v_cache"]))
        gap = torch.arange(c - n, c, device=DEV)[:, None] - torch.arange(c, device=DEV)[None]
        dark = (gap < 0) | (gap >= (case["window"] or c))
        heads = []
        for h in range(case["heads"]):
            p = torch.softmax((q[:, h] @ k[h // g].T / math.sqrt(case["head_dim"])).masked_fill(dark, -math.inf), -1)
            heads.append(p @ v[h // g])
        out.append(torch.stack(heads, 1))
    return torch.cat(out)
