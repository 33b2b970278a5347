"""The attention half of a decoder layer, measured: per-head norm + rotation of queries and keys, appending to a paged cache held
in 4 bits (and reading it back), and attention over that cache for single tokens, verifier rows and prefill chunks.

Cache format: pool[page][kv_head] is one block of page_size * (head_dim + head_dim / 8) bytes:
  K codes [page_size][head_dim / 2] | K scales FP16 [page_size][head_dim / 32] | V codes | V scales, as for K.
A row's head_dim / 8 little-endian words hold eight 4-bit codes each, dimension i of the word's eight in bits [4 i, 4 i + 4); the
word at place c * groups + g (groups = head_dim / 32, c = 0..3) holds dimensions 32 g + 8 c .. 32 g + 8 c + 7.  The value of a code
is (code - 8) * scale of its group of 32 dimensions; scale = FP16(max |x| / 7), code = clamp(round(x / scale), -7, 7) + 8.
Sequence s of a call owns rows row_begin[s] .. row_begin[s + 1] - 1; its last row is at position context[s] - 1."""
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EPS = 1e-6


def listed():
    return [
        # one row of one sequence between the QKV projection and the attention: nothing but latency
        dict(name="rope_step", op="rope", rows=1, heads=32, kv_heads=4, dim=128, rotary=128, interleaved=False, dtype="bf16", norm=True, far=5000, factor=1.0),
        # rows of many prompts in one pass, rotation in pairs over half of the head, positions far into a stretched context
        dict(name="rope_chunk", op="rope", rows=16384, heads=32, kv_heads=4, dim=128, rotary=64, interleaved=True, dtype="f16", norm=True, far=131072, factor=8.0),
        # a decode step of 64 sequences that have just begun: K normed, rotated and appended, Q beside it; the cache read back
        dict(name="append_step", op="append", mix=1, sequences=64, rows=1, least=1, context=256, heads=32, kv_heads=4, dim=128, page=64, rotary=128, interleaved=False, dtype="bf16", norm=True, factor=1.0),
        # ragged prompts of a prefill batch, decode-side FP32 rows, small heads and small pages
        dict(name="append_chunk", op="append", mix=2, sequences=5, rows=2047, least=1, context=4000, heads=16, kv_heads=8, dim=64, page=16, rotary=64, interleaved=True, dtype="f32", norm=False, factor=4.0),
        # one user, one token after a prompt of ordinary length: latency
        dict(name="decode_one", op="attend", mix=3, sequences=1, rows=1, least=4097, context=4097, heads=32, kv_heads=4, dim=128, page=64, window=0, dtype="bf16"),
        # a serving batch, lengths spread from a few tokens to 16384
        dict(name="decode_batch", op="attend", mix=4, sequences=64, rows=1, least=1, context=16384, heads=32, kv_heads=4, dim=128, page=64, window=0, dtype="bf16"),
        # one user at the longest context: the axis has to be split
        dict(name="decode_long", op="attend", mix=5, sequences=1, rows=1, least=131072, context=131072, heads=32, kv_heads=4, dim=128, page=64, window=0, dtype="bf16"),
        # draft tokens checked in one step: five rows for each sequence
        dict(name="verify_rows", op="attend", mix=6, sequences=8, rows=5, least=3000, context=32000, heads=32, kv_heads=4, dim=128, page=32, window=0, dtype="bf16"),
        # layers with a local window: only the last 1024 tokens count, whatever the context
        dict(name="decode_window", op="attend", mix=7, sequences=32, rows=1, least=1, context=9000, heads=16, kv_heads=8, dim=64, page=16, window=1024, dtype="f16"),
        # the first chunk of a prompt
        dict(name="prefill_first", op="attend", mix=8, sequences=1, rows=2048, least=2048, context=2048, heads=32, kv_heads=4, dim=128, page=64, window=0, dtype="bf16"),
        # a later chunk of a long prompt
        dict(name="prefill_history", op="attend", mix=9, sequences=1, rows=2048, least=34815, context=34815, heads=32, kv_heads=4, dim=128, page=64, window=0, dtype="bf16"),
        # chunks of several prompts at once, odd lengths, local window, small heads
        dict(name="prefill_ragged", op="attend", mix=10, sequences=6, rows=1023, least=1, context=4095, heads=16, kv_heads=4, dim=64, page=16, window=1024, dtype="f16"),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["rope", "append", "attend", "attend", "attend"])
    mix = rng.randrange(1 << 20)
    dim = rng.choice([64, 128])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 7, 8])
    dtype = rng.choice(["bf16", "f16"])
    rotary = rng.choice([dim, dim // 2])
    if op == "rope":
        return dict(op=op, rows=_spread(rng, 1, 16384), heads=heads, kv_heads=kv_heads, dim=dim, rotary=rotary, interleaved=rng.random() < 0.5, dtype=dtype,
                    norm=rng.random() < 0.7, far=_spread(rng, 16, 131072), factor=rng.choice([1.0, 4.0, 8.0]))
    page = rng.choice([16, 32, 64, 128])
    if op == "append":
        rows = _spread(rng, 1, 2048)
        context = min(4096, _spread(rng, rows, 16 * rows + 16))
        return dict(op=op, mix=mix, sequences=rng.randint(1, 8) if rows > 16 else _spread(rng, 1, 128), rows=rows, least=1, context=context, heads=heads,
                    kv_heads=kv_heads, dim=dim, page=page, rotary=rotary, interleaved=rng.random() < 0.5, dtype=rng.choice(["bf16", "f16", "f32"]), norm=rng.random() < 0.7,
                    factor=rng.choice([1.0, 4.0]))
    rows = rng.choice([1, 1, rng.randint(2, 16), _spread(rng, 17, 2048)])
    context = max(rows, _spread(rng, 64, 131072 if rows <= 16 else 32768))
    sequences = _spread(rng, 1, 64)
    while sequences > 1 and (sequences * heads * rows * context > 1 << 30 or sequences * context * kv_heads * dim > 1 << 29):
        sequences //= 2
    while heads * rows * context > 1 << 31:
        rows = max(1, rows // 2)
    return dict(op=op, mix=mix, sequences=sequences, rows=rows, least=1, context=context, heads=heads, kv_heads=kv_heads, dim=dim, page=page,
                window=rng.choice([0, 0, 1024]), dtype=dtype)


def lengths(case):
    """(rows, context) of each sequence: the case's largest, then smaller ones; context counts the call's own rows."""
    r = random.Random(case["mix"])
    got = []
    for s in range(case["sequences"]):
        rows = case["rows"] if s == 0 or case["rows"] <= 16 else r.randint(1, case["rows"])
        context = case["context"] if s == 0 else r.randint(min(case["least"], case["context"]), case["context"])
        got.append((rows, max(rows, context)))
    return got


def visible(case, rows, context):
    """Pairs (row, token) that the mask leaves, and tokens that some row sees, of one sequence."""
    first, w = context - rows, case["window"]
    pairs = rows * first + rows * (rows + 1) // 2
    if w and context > w:
        full = max(0, w - first)  # rows whose window begins before the first token
        full = min(rows, full)
        pairs = full * first + full * (full + 1) // 2 + (rows - full) * w
    return pairs, min(context, w + rows - 1) if w else context


def work(case):
    size, cached = DTYPES[case["dtype"]].itemsize, 2 * (case["dim"] // 2 + case["dim"] // 16)
    if case["op"] == "rope":
        n = case["rows"] * (case["heads"] + case["kv_heads"]) * case["dim"]
        return {"bytes": 2 * n * size + 4 * case["rows"], "flops": 10 * n}
    seq = lengths(case)
    rows = sum(n for n, _ in seq)
    tokens = sum(c for _, c in seq)
    if case["op"] == "append":  # rows in, cache out; Q in and out; the cache in and its values out
        moved = rows * case["dim"] * size * (2 * case["kv_heads"] + 2 * case["heads"]) + rows * case["kv_heads"] * cached
        moved += tokens * case["kv_heads"] * (cached + 4 * case["dim"])
        return {"bytes": moved, "flops": 10 * rows * case["dim"] * (case["heads"] + 2 * case["kv_heads"])}
    seen = [visible(case, n, c) for n, c in seq]
    return {"bytes": 2 * rows * case["heads"] * case["dim"] * size + sum(t for _, t in seen) * case["kv_heads"] * cached,
            "flops": 4 * case["dim"] * case["heads"] * sum(p for p, _ in seen)}


# ---- inputs -------------------------------------------------------------------------------------------------------

def frequencies(case):
    """Radians per position of each rotated pair, in 64 bits; the slow pairs stretched by `factor` for long contexts."""
    n = case["rotary"] // 2
    f = 500000.0 ** (-torch.arange(n, dtype=torch.float64) / n)
    if case["factor"] != 1.0:
        keep = torch.linspace(1.0, 0.0, n, dtype=torch.float64)
        f = f * keep + f / case["factor"] * (1 - keep)
    return f.cuda()


def amplitude(case):
    return 1.0 + 0.1 * math.log(case["factor"])


def step16(x):
    """Distance of FP16 values around x > 0 (64 bits)."""
    return torch.ldexp(torch.ones_like(x), torch.frexp(x)[1].clamp(min=-13) - 11)


def pack(x):
    """[..., dim] values in 64 bits -> (code words as bytes [..., dim / 2], scales FP16 [..., dim / 32])."""
    dim = x.shape[-1]
    g = x.unflatten(-1, (dim // 32, 32))
    most = g.abs().amax(-1)
    step = step16(most / 7)
    scale = torch.round(most / 7 / step) * step
    code = torch.where(scale[..., None] > 0, torch.round(g / scale[..., None]).clamp(-7, 7), 0.0).to(torch.int32) + 8
    code = code.unflatten(-1, (4, 8)).transpose(-3, -2).reshape(*x.shape[:-1], dim // 2, 2)  # word c * groups + g
    return (code[..., 0] | code[..., 1] << 4).to(torch.uint8), scale.to(torch.float16)


def unpack(codes, scales):
    """The inverse of pack, as FP32 values."""
    dim = 2 * codes.shape[-1]
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).unflatten(-1, (4, dim // 32, 8)).transpose(-3, -2)
    return ((c.float() - 8) * scales.float()[..., None, None]).flatten(-3)


def parts(pool, case):
    """Views of a pool's K codes, K scales, V codes and V scales: [pages, kv_heads, page, ...]."""
    p, d = case["page"], case["dim"]
    a, b = p * d // 2, p * d // 16
    codes = lambda at: pool[..., at:at + a].unflatten(-1, (p, d // 2))  # noqa: E731
    scales = lambda at: pool[..., at:at + b].view(torch.float16).unflatten(-1, (p, d // 32))  # noqa: E731
    return codes(0), scales(a), codes(a + b), scales(2 * a + b)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    randn = lambda *shape: torch.randn(shape, generator=g, device="cuda")  # noqa: E731
    state = {"case": case}
    if case["op"] != "attend":
        state["inv_freq"] = frequencies(case)
        for name in ("q_weight", "k_weight"):
            state[name] = (1 + 0.2 * randn(case["dim"])).bfloat16() if case["norm"] else None
    if case["op"] == "rope":
        for name, heads in (("q", case["heads"]), ("k", case["kv_heads"])):
            state[name] = randn(case["rows"], heads, case["dim"]).to(dtype)
        state["positions"] = torch.randint(0, case["far"], (case["rows"],), generator=g, device="cuda", dtype=torch.int32)
        if own:
            from padra_b200 import attention

            state["kernels"] = attention.AttentionKernels()
            state["rotary"] = attention.Rotary(state["inv_freq"], case["interleaved"], amplitude(case))
            state["out"] = torch.empty_like(state["q"]), torch.empty_like(state["k"])
        return state

    seq = lengths(case)
    need = [-(-c // case["page"]) for _, c in seq]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros((len(seq), max(need)), dtype=torch.int32, device="cuda")
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    rows = sum(n for n, _ in seq)
    begin = [0]
    for n, _ in seq:
        begin.append(begin[-1] + n)
    state |= {"table": table, "rows": rows, "most": max(n for n, _ in seq), "longest": max(c for _, c in seq),
              "row_begin": torch.tensor(begin, dtype=torch.int32, device="cuda"),
              "context": torch.tensor([c for _, c in seq], dtype=torch.int32, device="cuda")}

    # what earlier steps have left in the cache: a few loud dimensions in K, V of one size
    dim, heads = case["dim"], case["kv_heads"]
    loud = torch.exp(0.6 * randn(heads, 1, dim))
    pool = torch.zeros((pages, heads, case["page"] * (dim + dim // 8)), dtype=torch.uint8, device="cuda")
    k_codes, k_scales, v_codes, v_scales = parts(pool, case)
    piece = max(1, (1 << 25) // (heads * case["page"] * dim))
    for a in range(0, pages, piece):
        b = min(pages, a + piece)
        k_codes[a:b], k_scales[a:b] = pack((randn(b - a, heads, case["page"], dim) * loud).double())
        v_codes[a:b], v_scales[a:b] = pack(randn(b - a, heads, case["page"], dim).double())
    state["pool"] = pool

    # q, k and v as columns of one projection's rows
    q, k, v = (randn(rows, (case["heads"] + 2 * heads) * dim)).to(dtype).split([case["heads"] * dim, heads * dim, heads * dim], -1)
    state["q"] = q.unflatten(-1, (case["heads"], dim))
    if case["op"] == "append":
        state["k"], state["v"] = k.unflatten(-1, (heads, dim)), v.unflatten(-1, (heads, dim))
    else:
        state["scale"] = dim ** -0.5
    if own:
        from padra_b200 import attention

        state["kernels"] = attention.AttentionKernels()
        state["cache"] = attention.KvCache.over(pool, case["page"], dim)
        state["sequences"] = attention.Sequences(table, state["row_begin"], state["context"], rows, state["most"])
        state["out"] = torch.empty((rows, case["heads"], dim), dtype=dtype, device="cuda")
        if case["op"] == "append":
            state["rotary"] = attention.Rotary(state["inv_freq"], case["interleaved"], amplitude(case))
            # every token of every sequence, to be read back
            total = sum(c for _, c in seq)
            ends = torch.cat((torch.zeros_like(state["context"][:1]), state["context"].cumsum(0, dtype=torch.int32)))
            state["everything"] = attention.Sequences(table, ends, state["context"], total, state["longest"])
            state["back"] = torch.empty((2, total, heads, dim), dtype=torch.bfloat16, device="cuda")
    return state


# ---- plain form ---------------------------------------------------------------------------------------------------

def normed(x, weight, kind):
    x = x.to(kind)
    if weight is None:
        return x
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.to(kind)


def rotated(x, positions, state):
    """x [rows, heads, dim] in 32 or 64 bits, rotated; angles in 64 bits."""
    case, n = state["case"], state["case"]["rotary"]
    t = positions.double()[:, None] * state["inv_freq"]
    cos, sin = ((f * amplitude(case)).to(x.dtype)[:, None] for f in (t.cos(), t.sin()))
    y, rest = x[..., :n], x[..., n:]
    if case["interleaved"]:
        a, b = y[..., 0::2], y[..., 1::2]
        y = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    else:
        a, b = y[..., :n // 2], y[..., n // 2:]
        y = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    return torch.cat((y, rest), -1)


def places(state):
    """(sequence, position) of every row of the call."""
    rows = torch.arange(state["rows"], device="cuda", dtype=torch.int32)
    s = torch.searchsorted(state["row_begin"], rows, right=True) - 1
    return s, state["context"][s] - state["row_begin"][s + 1] + rows


def everywhere(state):
    """(sequence, position) of every token of every sequence, in order."""
    at = torch.arange(state["longest"], device="cuda")
    return (at < state["context"][:, None]).nonzero(as_tuple=True)


def run(state):
    case = state["case"]
    if case["op"] == "rope":
        if own:
            return state["kernels"].qk_norm_rope(state["q"], state["k"], state["positions"], state["rotary"], state["q_weight"], state["k_weight"], EPS, *state["out"])
        return [rotated(normed(state[x], state[x + "_weight"], torch.float32), state["positions"], state).to(DTYPES[case["dtype"]]) for x in ("q", "k")]
    if case["op"] == "append":
        if own:
            q = state["kernels"].append(state["cache"], state["sequences"], state["k"], state["v"], state["rotary"], state["k_weight"], EPS, state["q"], state["q_weight"],
                                        state["out"])
            return q, state["kernels"].read(state["cache"], state["everything"], state["back"][0], state["back"][1])
        s, at = places(state)
        # values next to a border between two codes are decided in 64 bits
        k = rotated(normed(state["k"], state["k_weight"], torch.float64), at, state)
        k_codes, k_scales, v_codes, v_scales = parts(state["pool"], case)
        page, slot = state["table"][s, at // case["page"]].long(), (at % case["page"]).long()
        k_codes[page, :, slot], k_scales[page, :, slot] = pack(k)
        v_codes[page, :, slot], v_scales[page, :, slot] = pack(state["v"].double())
        q = rotated(normed(state["q"], state["q_weight"], torch.float32), at, state)
        s, at = everywhere(state)
        page, slot = state["table"][s, at // case["page"]].long(), at % case["page"]
        back = [unpack(c[page, :, slot], f[page, :, slot]).bfloat16() for c, f in ((k_codes, k_scales), (v_codes, v_scales))]
        return q.to(DTYPES[case["dtype"]]), back
    if own:
        return state["kernels"].attention(state["cache"], state["sequences"], state["q"], state["scale"], case["window"], state["out"])
    # sequences side by side, padded to the longest
    count, most, longest, groups = case["sequences"], state["most"], state["longest"], case["heads"] // case["kv_heads"]
    blocks = state["pool"][state["table"].long()]
    k_codes, k_scales, v_codes, v_scales = parts(blocks, case)
    keys, values = (unpack(c, f).transpose(1, 2).flatten(2, 3)[:, :, :longest] for c, f in ((k_codes, k_scales), (v_codes, v_scales)))
    del blocks, k_codes, k_scales, v_codes, v_scales
    row = state["row_begin"][:-1, None] + torch.arange(most, device="cuda")
    there = row < state["row_begin"][1:, None]
    at = state["context"][:, None] - state["row_begin"][1:, None] + row
    q = state["q"][row.clamp(max=state["rows"] - 1).long()].float() * state["scale"]
    q = q.unflatten(2, (case["kv_heads"], groups)).permute(0, 2, 3, 1, 4).flatten(2, 3)  # [count, kv_heads, groups * most, dim]
    scores = q @ keys.transpose(-1, -2)
    token = torch.arange(longest, device="cuda")
    hidden = token > at[..., None]
    if case["window"]:
        hidden |= token <= at[..., None] - case["window"]
    scores = scores.unflatten(2, (groups, most)).masked_fill_(hidden[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=-1e30)
    scores = scores.sub_(top).exp_()
    total = scores.sum(-1, keepdim=True)
    out = (scores.flatten(2, 3) @ values).unflatten(2, (groups, most)) / total.clamp(min=1e-30)
    return out.permute(0, 3, 1, 2, 4).flatten(2, 3)[there].to(DTYPES[case["dtype"]])


# ---- the definition in 64 bits --------------------------------------------------------------------------------------

def exact(case, seed):
    """Row by row or sequence by sequence from the formulas, in 64 bits."""
    s = prepare(case, seed)

    def rms(x, w):
        x = x.double()
        return x if w is None else x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + EPS) * w.double()

    def turn(x, positions):
        # as complex numbers: the pair (a, b) is a + b i, multiplied by amplitude * e^(i angle)
        n = case["rotary"]
        pair = x[..., :n].unflatten(-1, (n // 2, 2)) if case["interleaved"] else x[..., :n].unflatten(-1, (2, n // 2)).transpose(-1, -2)
        angle = positions.double()[:, None, None] * s["inv_freq"]
        z = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * torch.polar(torch.full_like(angle, amplitude(case)), angle))
        z = z.flatten(-2) if case["interleaved"] else z.transpose(-1, -2).flatten(-2)
        return torch.cat((z, x[..., n:]), -1)

    if case["op"] == "rope":
        return [turn(rms(s[x], s[x + "_weight"]), s["positions"]) for x in ("q", "k")]

    def values(codes, scales):
        # one dimension after the other: dimension d is code d % 8 of word (d / 8 % 4) * groups + d / 32
        words = codes.contiguous().view(torch.int32)
        d = torch.arange(case["dim"], device="cuda")
        code = words[..., d // 8 % 4 * (case["dim"] // 32) + d // 32] >> (4 * (d % 8)).int() & 15
        return (code.double() - 8) * scales.double()[..., d // 32]

    def tokens(i, c):
        """K and V of sequence i, [context, kv_heads, dim]."""
        p = case["page"]
        block = s["pool"][s["table"][i, :-(-c // p)].long()]
        kc, ks, vc, vs = parts(block, case)
        return [values(a, b).transpose(1, 2).flatten(0, 1)[:c] for a, b in ((kc, ks), (vc, vs))]

    if case["op"] == "append":
        def held(x):
            """The values that 4 bits stand for, with FP16 scales by numpy's rounding."""
            g = x.unflatten(-1, (case["dim"] // 32, 32))
            scale = torch.from_numpy((g.abs().amax(-1) / 7).cpu().numpy().astype(np.float16)).cuda().double()[..., None]
            return (torch.where(scale > 0, torch.round(g / scale), 0.0).clamp(-7, 7) * scale).flatten(-2)

        q, back = [], ([], [])
        for i, (n, c) in enumerate(lengths(case)):
            own_rows = slice(int(s["row_begin"][i]), int(s["row_begin"][i]) + n)
            at = torch.arange(c - n, c, device="cuda")
            q.append(turn(rms(s["q"][own_rows], s["q_weight"]), at))
            kept = tokens(i, c)
            for x, new, to in zip(kept, (held(turn(rms(s["k"][own_rows], s["k_weight"]), at)), held(s["v"][own_rows].double())), back):
                x[c - n:] = new
                to.append(x)
        return torch.cat(q), [torch.cat(x) for x in back]

    if work(case)["flops"] > 4e12:
        return None
    out = []
    groups = case["heads"] // case["kv_heads"]
    for i, (n, c) in enumerate(lengths(case)):
        k, v = tokens(i, c)
        q = s["q"][int(s["row_begin"][i]):int(s["row_begin"][i]) + n].double()
        piece = max(1, (1 << 28) // (c * case["heads"]))
        for a in range(0, n, piece):
            b = min(n, a + piece)
            at = torch.arange(c - n + a, c - n + b, device="cuda")[:, None]
            token = torch.arange(c, device="cuda")
            seen = (token <= at) & ((token > at - case["window"]) if case["window"] else True)
            score = torch.einsum("rhgd,thd->hgrt", q[a:b].unflatten(1, (case["kv_heads"], groups)), k) * s["scale"]
            p = torch.softmax(score.masked_fill(~seen, -math.inf), -1)
            out.append(torch.einsum("hgrt,thd->rhgd", p, v).flatten(1, 2))
    return torch.cat(out)
