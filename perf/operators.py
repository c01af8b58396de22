"""Cases for the language-model operators: rotary positions, the append to the
8-bit paged key/value cache and the attention over that cache.

`run` computes a case in one of two ways: with `own` true through the
package's entry points (`infvino_b200.KvOps`), with `own` false in elementary
torch operations in 32 bits.  `exact` computes the same from the definitions
in 64 bits.

The cache: `k`, `v` int8 [pages, kv_heads, page_size, dim]; `k_scale`,
`v_scale` float32 [pages, kv_heads, page_size / 16], one power of two for each
block of 16 tokens and head; a value is code * scale.  Sequence b's token at
position p is in page `pages[b, p // page_size]`, slot `p % page_size`.
"""
import math
import random

import torch

own = False

BLOCK = 16          # tokens that share a scale
E_MIN, E_MAX = -120, 121  # exponents a scale can have
THETA = 10000.0     # base of the rotary frequencies
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
MOST_SCORES = 3.0e9     # scores of one plain attention (float32, held whole)
MOST_CACHE = 4.4e9      # cache bytes of one case

_ops = None


def listed():
    return [
        # one decode step of 16 conversations: query heads, (time, height, width) positions
        {"name": "rope_step", "op": "rope", "dtype": "f16", "tokens": 16, "heads": 32, "dim": 128, "pairs": 64, "axes": 3,
         "interleaved": False, "packed": False},
        # patches of a batch of images in a vision tower: (height, width), a slice of the packed qkv projection
        {"name": "rope_patches", "op": "rope", "dtype": "f16", "tokens": 9999, "heads": 16, "dim": 64, "pairs": 32, "axes": 2,
         "interleaved": True, "packed": True},
        # a long prompt with video frames in it
        {"name": "rope_prompt", "op": "rope", "dtype": "bf16", "tokens": 16381, "heads": 28, "dim": 128, "pairs": 64, "axes": 3,
         "interleaved": False, "packed": False},
        # one decode step of 64 conversations: queries rotated, one token of keys and values appended to each
        {"name": "append_step", "op": "append", "dtype": "bf16", "batch": 64, "new": 1, "history": 4000, "ragged": True,
         "kv_heads": 8, "group": 4, "dim": 128, "page": 64, "axes": 1},
        # three prompts, the later turns of conversations, with images among their tokens
        {"name": "append_prompt", "op": "append", "dtype": "f16", "batch": 3, "new": 4093, "history": 1003, "ragged": True,
         "kv_heads": 8, "group": 4, "dim": 128, "page": 64, "axes": 3},
        # one user's decode step on a short conversation: latency
        {"name": "step_one", "op": "attend", "dtype": "f16", "batch": 1, "new": 1, "history": 777, "ragged": False,
         "kv_heads": 4, "group": 7, "dim": 128, "page": 16, "window": 0, "sinks": 0},
        # decode step of a serving batch with conversations of all lengths
        {"name": "step_batch", "op": "attend", "dtype": "bf16", "batch": 48, "new": 1, "history": 16383, "ragged": True,
         "kv_heads": 8, "group": 4, "dim": 128, "page": 64, "window": 0, "sinks": 0},
        # decode step over long documents: the cache's offsets pass 2^31
        {"name": "step_long", "op": "attend", "dtype": "f16", "batch": 16, "new": 1, "history": 131071, "ragged": False,
         "kv_heads": 8, "group": 8, "dim": 128, "page": 128, "window": 0, "sinks": 0},
        # decode step with a sliding window and four first tokens that stay visible
        {"name": "step_window", "op": "attend", "dtype": "f16", "batch": 128, "new": 1, "history": 8190, "ragged": True,
         "kv_heads": 4, "group": 8, "dim": 64, "page": 32, "window": 1024, "sinks": 4},
        # drafted tokens checked against the cache: six queries for each sequence
        {"name": "verify_batch", "op": "attend", "dtype": "bf16", "batch": 24, "new": 6, "history": 6001, "ragged": True,
         "kv_heads": 8, "group": 5, "dim": 64, "page": 16, "window": 0, "sinks": 0},
        # a whole prompt at once
        {"name": "prompt", "op": "attend", "dtype": "f16", "batch": 1, "new": 8191, "history": 0, "ragged": False,
         "kv_heads": 8, "group": 4, "dim": 128, "page": 64, "window": 0, "sinks": 0},
        # a chunk of two long prompts, sliding window and sinks
        {"name": "chunk_window", "op": "attend", "dtype": "bf16", "batch": 2, "new": 2000, "history": 20011, "ragged": True,
         "kv_heads": 4, "group": 6, "dim": 128, "page": 64, "window": 4096, "sinks": 16},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["rope", "append", "step", "step", "few", "prompt", "prompt"])
    dtype = rng.choice(["f16", "bf16"])
    dim = rng.choice([64, 128])
    if kind == "rope":
        axes = rng.randint(1, 3)
        return {"op": "rope", "dtype": dtype, "tokens": _log(rng, 1, 16381), "heads": rng.randint(1, 28), "dim": dim,
                "pairs": dim // 2 if axes > 1 else rng.choice([dim // 2, dim // 4]), "axes": axes,
                "interleaved": rng.random() < 0.5, "packed": rng.random() < 0.5}
    heads = {"kv_heads": rng.choice([1, 2, 3, 4, 5, 8, 16]), "group": rng.randint(1, 8), "dim": dim, "page": rng.choice([16, 32, 48, 64, 128])}
    ragged = rng.random() < 0.7
    if kind == "append":
        batch = _log(rng, 1, 128)
        new = rng.choice([1, _log(rng, 1, max(1, 8192 // batch))])
        return {"op": "append", "dtype": dtype, "batch": batch, "new": new, "history": _log(rng, 1, 8192) - 1, "ragged": ragged, **heads,
                "axes": rng.randint(1, 3)}
    window = rng.choice([0, 0, _log(rng, 16, 4096)])
    sinks = rng.choice([0, 1, 4, 16]) if window else 0
    per_token = 2 * heads["kv_heads"] * dim
    if kind == "prompt":
        batch = rng.randint(1, 4)
        new = _log(rng, 9, 8191 // batch)
        history = rng.choice([0, _log(rng, 1, 20011)])
        history = min(history, int(MOST_SCORES / (batch * new * heads["kv_heads"] * heads["group"])) - new)
        if history < 0:
            history, new = 0, min(new, 2048)
    else:
        batch = _log(rng, 1, 128)
        new = 1 if kind == "step" else rng.randint(2, 8)
        history = min(_log(rng, 1, 131071), int(MOST_CACHE / (batch * per_token)), int(MOST_SCORES / (batch * new * heads["kv_heads"] * heads["group"])))
    return {"op": "attend", "dtype": dtype, "batch": batch, "new": new, "history": history, "ragged": ragged, **heads, "window": window,
            "sinks": sinks}


# ---------------------------------------------------------------- what a case stands for

def _lengths(case):
    """(tokens in the cache before the call, new tokens) of each sequence."""
    r = random.Random("%d %d %d" % (case["batch"], case["new"], case["history"]))
    n, h = case["new"], case["history"]
    hist, new = [h], [n]
    while len(new) < case["batch"]:
        hist.append(r.randint(h // 4, h) if case["ragged"] else h)
        new.append(r.randint(-(-n // 3), n) if case["ragged"] else n)
    return hist, new


def _axes_of_pairs(pairs, axes):
    """The axis of each rotated pair: contiguous sections, the first axis with the rest."""
    each = pairs // (axes + 1) if axes > 2 else pairs // axes
    count = [each] * axes
    if axes > 1:
        count = [each] * axes
        count[-1] += (pairs - each * axes) // 2
        count[0] += pairs - sum(count)
    return [a for a in range(axes) for _ in range(count[a])]


def _inv_freq(pairs):
    return [THETA ** (-i / pairs) for i in range(pairs)]


def _visible(first, count, window, sinks):
    """(query, key) pairs that `count` queries at positions first.. see."""
    total = 0
    for p in range(first, first + count):
        if not window or p < window:
            total += p + 1
        else:
            total += window + min(sinks, p - window + 1)
    return total


def _span(first, count, window, sinks):
    """Keys that at least one of those queries sees."""
    last = first + count
    if not window or first < window:
        return last
    lo = first - window + 1
    return last - lo + min(sinks, lo)


def work(case):
    if case["op"] == "rope":
        n = case["tokens"] * case["heads"]
        return {"bytes": n * case["dim"] * 4 + case["tokens"] * case["axes"] * 4, "flops": n * case["pairs"] * 6}
    hist, new = _lengths(case)
    t, hk, hq, d = sum(new), case["kv_heads"], case["kv_heads"] * case["group"], case["dim"]
    if case["op"] == "append":
        back = sum(h % BLOCK + n for h, n in zip(hist, new))  # tokens of the blocks that were touched
        blocks = sum(-(-(h % BLOCK + n) // BLOCK) for h, n in zip(hist, new))
        old = back - t
        # keys, values and queries read; queries, codes and scales written; the first blocks' codes read; the values read back
        return {"bytes": t * (2 * hk + 2 * hq) * d * 2 + (t + old) * 2 * hk * d + blocks * 8 * hk + back * 2 * hk * d * 2,
                "flops": t * (hk + hq) * d * 3 + t * hk * d * 4}
    w, s = case["window"], case["sinks"]
    pairs = sum(_visible(h, n, w, s) for h, n in zip(hist, new))
    keys = sum(_span(h, n, w, s) for h, n in zip(hist, new))
    return {"bytes": keys * 2 * hk * (d + 4 / BLOCK) + 2 * t * hq * d * 2, "flops": 4 * d * hq * pairs}


# ---------------------------------------------------------------- inputs

def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _positions(first, axes):
    """Positions [axes, tokens]: the same number on every axis, but on the last two a grid of 14 x 14 behind it."""
    first = torch.as_tensor(first, dtype=torch.int64, device="cuda")
    pos = first.repeat(axes, 1)
    if axes > 1:
        i = torch.arange(len(first), device="cuda")
        pos[-1] = first // 2 + i % 14
        pos[-2] = first // 2 + i // 14 % 14
    return pos.to(torch.int32)


def _table(positions, pairs):
    """cos and sin of every position's angle for each pair: [positions, pairs, 2] float32."""
    inv = torch.tensor(_inv_freq(pairs), dtype=torch.float64, device="cuda")
    a = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * inv
    return torch.stack([a.cos(), a.sin()], dim=-1).float().contiguous()


def _cache(pages, case, gen):
    shape = (pages, case["kv_heads"], case["page"], case["dim"])

    def codes():
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float16).mul_(30.0).round_().clamp_(-127, 127).to(torch.int8)

    def scales():
        e = torch.randint(-6, -3, (pages, case["kv_heads"], case["page"] // BLOCK), generator=gen, device="cuda")
        return torch.ldexp(torch.ones((), device="cuda"), e)

    return {"k": codes(), "v": codes(), "k_scale": scales(), "v_scale": scales()}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = TYPES[case["dtype"]]

    def normal(tokens, heads, times=1.0):
        return torch.randn((tokens, heads, case["dim"]), generator=gen, device="cuda").mul_(times).to(dt)

    if case["op"] == "rope":
        t, h = case["tokens"], case["heads"]
        x = normal(t, 3 * h if case["packed"] else h)[:, :h]
        pos = _positions(torch.arange(t) % 8192, case["axes"])
        return {"case": case, "x": x, "out": torch.empty((t, h, case["dim"]), device="cuda", dtype=dt), "pos": pos,
                "table": _table(8192 + 14, case["pairs"])}
    hist, new = _lengths(case)
    page, hk, hq = case["page"], case["kv_heads"], case["kv_heads"] * case["group"]
    need = [-(-(h + n) // page) for h, n in zip(hist, new)]
    total = sum(need) + 3
    order = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)  # a cache that has been in use: pages in any order
    first = [sum(need[:b]) for b in range(len(need))]
    at = _ints(first)[:, None] + torch.arange(max(need), dtype=torch.int32, device="cuda")
    pages = order[at.clamp(max=total - 1).long()].contiguous()
    offsets = [sum(new[:b]) for b in range(len(new) + 1)]
    t = offsets[-1]
    s = {"case": case, **_cache(total, case, gen), "pages": pages, "offsets": _ints(offsets), "max_new": max(new),
         "q": normal(t, hq, 3.0 if case["op"] == "attend" else 1.0), "out": torch.empty((t, hq, case["dim"]), device="cuda", dtype=dt)}
    if case["op"] == "attend":
        s["lens"] = _ints([h + n for h, n in zip(hist, new)])
        return s
    which = torch.repeat_interleave(torch.arange(len(new)), torch.tensor(new))
    s["pos"] = _positions(torch.tensor(hist)[which] + torch.arange(t) - torch.tensor(offsets)[which], case["axes"])
    s["starts"] = _ints(hist)
    spread = torch.exp(torch.randn((hk, case["dim"]), generator=gen, device="cuda"))  # some channels of keys are far larger than others
    s["new_k"], s["new_v"] = (normal(t, hk).float() * spread).to(dt), normal(t, hk)
    s["table"] = _table(max(h + n for h, n in zip(hist, new)) + 14, case["dim"] // 2)
    back = [h % BLOCK + n for h, n in zip(hist, new)]
    s["back_offsets"], s["back_starts"] = _ints([sum(back[:b]) for b in range(len(back) + 1)]), _ints([h - h % BLOCK for h in hist])
    s["back_k"], s["back_v"] = (torch.empty((sum(back), hk, case["dim"]), device="cuda", dtype=dt) for _ in range(2))
    return s


# ---------------------------------------------------------------- the framework's operators

def _own(s):
    import infvino_b200 as ivb
    global _ops
    if _ops is None:
        _ops = ivb.KvOps(device=0)
    c, st = s["case"], torch.cuda.current_stream().cuda_stream
    if c["op"] == "rope":
        rotary = ivb.Rotary(s["table"], _axes_of_pairs(c["pairs"], c["axes"]), c["interleaved"])
        _ops.rope(s["x"], s["out"], rotary, s["pos"], stream=st)
        return s["out"]
    cache = ivb.KvCache(s["k"], s["v"], s["k_scale"], s["v_scale"])
    if c["op"] == "append":
        rotary = ivb.Rotary(s["table"], _axes_of_pairs(c["dim"] // 2, c["axes"]))
        _ops.append(cache, s["new_k"], s["new_v"], s["offsets"], s["starts"], s["pages"], rotary=rotary, pos=s["pos"], q=s["q"], q_out=s["out"],
                    stream=st)
        _ops.read(cache, s["back_k"], s["back_v"], s["back_offsets"], s["back_starts"], s["pages"], stream=st)
        return s["out"], s["back_k"], s["back_v"]
    _ops.attend(cache, s["q"], s["out"], s["offsets"], s["lens"], s["pages"], max_new=s["max_new"], scale=c["dim"] ** -0.5, window=c["window"],
                sinks=c["sinks"], stream=st)
    return s["out"]


# ---------------------------------------------------------------- the plain forms

def _rotate(x, table, pos, axis, interleaved):
    x, pairs = x.float(), len(axis)
    at = pos.long()[axis].t()                                    # [tokens, pairs]
    cs = table[at, torch.arange(pairs, device=x.device)][:, None]  # [tokens, 1, pairs, 2]
    c, s = cs[..., 0], cs[..., 1]
    a, b = (x[..., 0:2 * pairs:2], x[..., 1:2 * pairs:2]) if interleaved else (x[..., :pairs], x[..., pairs:2 * pairs])
    y = x.clone()
    if interleaved:
        y[..., 0:2 * pairs:2], y[..., 1:2 * pairs:2] = a * c - b * s, b * c + a * s
    else:
        y[..., :pairs], y[..., pairs:2 * pairs] = a * c - b * s, b * c + a * s
    return y


def _sequence_of(offsets, tokens):
    """Each packed token's sequence and its place in it."""
    i = torch.arange(tokens, device=offsets.device)
    seq = torch.searchsorted(offsets[1:].contiguous(), i, right=True)
    return seq, i - offsets[seq]


def _append_one(codes, scales, x, seq, pos, starts, new, pages):
    """Quantises x [tokens, heads, dim] into one half of the cache."""
    ps, per = codes.shape[2], scales.shape[2]
    page, slot = pages[seq, pos // ps].long(), pos % ps
    block = page * per + slot // BLOCK
    most = torch.zeros((scales.shape[0] * per, x.shape[1]), device=x.device)
    most.index_reduce_(0, block, x.abs().amax(-1), "amax")
    most = most[block]
    m, e = torch.frexp(most)
    e = torch.where(most == 0, E_MIN, (e - 7 + (m > 127 / 128)).clamp(E_MIN, E_MAX))
    scale = torch.ldexp(torch.ones_like(most), e)                # [tokens, heads]
    held = pos // BLOCK * BLOCK < starts[seq]                    # the block held tokens before
    scale = torch.where(held[:, None], torch.maximum(scale, scales[page, :, slot // BLOCK]), scale)
    # the tokens before: at most one block of each sequence, the one where its new tokens begin
    i = torch.arange(BLOCK, device=x.device)
    at = (starts // BLOCK * BLOCK)[:, None].long() + i
    op, os = pages[torch.arange(len(starts), device=x.device)[:, None], (at // ps).clamp(max=pages.shape[1] - 1)].long(), at % ps
    before = scales[op[:, 0], :, os[:, 0] // BLOCK]
    scales[page, :, slot // BLOCK] = scale
    after = scales[op[:, 0], :, os[:, 0] // BLOCK]
    old = codes[op, :, os]                                       # [batch, 16, heads, dim]
    moved = torch.round(old.float() * (before / after)[:, None, :, None]).to(torch.int8)
    moves = (i < (starts % BLOCK)[:, None]) & (new > 0)[:, None]
    codes[op, :, os] = torch.where(moves[..., None, None], moved, old)
    codes[page, :, slot] = torch.round(x / scale[..., None]).to(torch.int8)


def _read_one(codes, scales, seq, pos, pages, dtype):
    ps = codes.shape[2]
    page, slot = pages[seq, pos // ps].long(), pos % ps
    return (codes[page, :, slot].float() * scales[page, :, slot // BLOCK][..., None]).to(dtype)


def _attend(s):
    c, q, offsets, lens = s["case"], s["q"], s["offsets"], s["lens"]
    batch, n, hk, g, d = c["batch"], s["max_new"], c["kv_heads"], c["group"], c["dim"]

    def half(codes, scales):
        x = s[codes][s["pages"].long()].unflatten(3, (-1, BLOCK)) * s[scales][s["pages"].long()][..., None, None]
        return x.flatten(3, 4).permute(0, 2, 1, 3, 4).flatten(2, 3)  # [batch, kv_heads, keys, dim] float32

    k, v = half("k", "k_scale"), half("v", "v_scale")
    i = torch.arange(n, device=q.device)
    x = q[(offsets[:-1, None] + i).clamp(max=q.shape[0] - 1)].float()      # [batch, n, heads, dim]
    x = x.view(batch, n, hk, g, d).permute(0, 2, 3, 1, 4).reshape(batch, hk, g * n, d)
    p = (lens - (offsets[1:] - offsets[:-1]))[:, None, None] + i[:, None]  # positions of the queries
    j = torch.arange(k.shape[2], device=q.device)
    seen = (j <= p) & (p < lens[:, None, None])
    if c["window"]:
        seen &= (p - j < c["window"]) | (j < c["sinks"])
    score = (x @ k.transpose(2, 3)).mul_(d ** -0.5).view(batch, hk, g, n, -1)
    score.masked_fill_(~seen[:, None, None], -math.inf)
    m = score.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    w = score.sub_(m).exp_()
    total = w.sum(-1, keepdim=True)
    y = (w.view(batch, hk, g * n, -1) @ v).view(batch, hk, g, n, d) / torch.where(total == 0, 1.0, total)
    seq, at = _sequence_of(offsets, q.shape[0])
    return y.permute(0, 3, 1, 2, 4).reshape(batch, n, hk * g, d)[seq, at].to(q.dtype)


def _plain(s):
    c = s["case"]
    if c["op"] == "rope":
        return _rotate(s["x"], s["table"], s["pos"], _axes_of_pairs(c["pairs"], c["axes"]), c["interleaved"]).to(s["x"].dtype)
    if c["op"] == "attend":
        return _attend(s)
    axis = _axes_of_pairs(c["dim"] // 2, c["axes"])
    q = _rotate(s["q"], s["table"], s["pos"], axis, False).to(s["q"].dtype)
    k, v = _rotate(s["new_k"], s["table"], s["pos"], axis, False), s["new_v"].float()
    starts, offsets = s["starts"], s["offsets"]
    seq, at = _sequence_of(offsets, k.shape[0])
    pos, new = starts[seq] + at, offsets[1:] - offsets[:-1]
    _append_one(s["k"], s["k_scale"], k, seq, pos, starts, new, s["pages"])
    _append_one(s["v"], s["v_scale"], v, seq, pos, starts, new, s["pages"])
    seq, at = _sequence_of(s["back_offsets"], s["back_k"].shape[0])
    pos = s["back_starts"][seq] + at
    return (q, _read_one(s["k"], s["k_scale"], seq, pos, s["pages"], q.dtype), _read_one(s["v"], s["v_scale"], seq, pos, s["pages"], q.dtype))


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------- the definitions in 64 bits

def _exact_rotation(x, pos, axes, pairs, interleaved):
    x = x.double()
    inv = torch.tensor(_inv_freq(pairs), dtype=torch.float64, device=x.device)
    rows = torch.tensor(_axes_of_pairs(pairs, axes), device=x.device)
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=x.device), pos.double().index_select(0, rows).t() * inv)[:, None]
    z = x[..., :2 * pairs]
    z = z.unflatten(-1, (pairs, 2)) if interleaved else z.unflatten(-1, (2, pairs)).transpose(-1, -2)
    z = torch.view_as_real(torch.view_as_complex(z.contiguous()) * turn)
    z = z if interleaved else z.transpose(-1, -2)
    return torch.cat([z.reshape(*x.shape[:-1], 2 * pairs), x[..., 2 * pairs:]], -1)


def _exact_append(s, which, x, hist, new):
    """The values that the touched blocks hold after the append, block by block."""
    codes, scales, pages, ps = s[which], s[which + "_scale"], s["pages"].tolist(), s["case"]["page"]
    got, done = [], 0
    for b, (h, n) in enumerate(zip(hist, new)):
        lo = h - h % BLOCK
        y = torch.zeros((-(-(h + n - lo) // BLOCK) * BLOCK, *x.shape[1:]), dtype=torch.float64, device=x.device)
        y[h - lo:h - lo + n] = x[done:done + n]
        done += n
        y = y.unflatten(0, (-1, BLOCK))
        most = y.abs().amax((1, 3))
        step = torch.exp2(torch.ceil(torch.log2(most / 127)).clamp(E_MIN, E_MAX))
        if h > lo:
            page, slot = pages[b][lo // ps], lo % ps
            before = scales[page, :, slot // BLOCK].double()
            held = codes[page, :, slot:slot + h - lo].double().transpose(0, 1)
            step[0] = torch.maximum(step[0], before)
            y[0, :h - lo] = torch.round(held * (before / step[0])[:, None]) * step[0][:, None]
        got.append((torch.round(y / step[:, None, :, None]) * step[:, None, :, None]).flatten(0, 1)[:h + n - lo])
    return torch.cat(got)


def _exact_attention(s, hist, new):
    c, q, got, done = s["case"], s["q"], [], 0
    for b, (h, n) in enumerate(zip(hist, new)):
        need = -(-(h + n) // c["page"])
        rows, heads = s["pages"][b, :need].long(), []
        p = torch.arange(h, h + n, device=q.device)[:, None]
        j = torch.arange(h + n, device=q.device)
        hidden = j > p
        if c["window"]:
            hidden |= (j <= p - c["window"]) & (j >= c["sinks"])
        for head in range(c["kv_heads"]):
            k, v = ((s[w][rows, head].double() * s[w + "_scale"][rows, head].double().repeat_interleave(BLOCK, 1)[..., None]).flatten(0, 1)[:h + n]
                    for w in ("k", "v"))
            for r in range(head * c["group"], (head + 1) * c["group"]):
                a = (q[done:done + n, r].double() @ k.t()) / math.sqrt(c["dim"])
                heads.append(torch.softmax(a.masked_fill_(hidden, -math.inf), -1) @ v)
        done += n
        got.append(torch.stack(heads, 1))
    return torch.cat(got)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        return _exact_rotation(s["x"], s["pos"], case["axes"], case["pairs"], case["interleaved"])
    hist, new = _lengths(case)
    if case["op"] == "attend":
        return _exact_attention(s, hist, new)
    q, k = (_exact_rotation(x, s["pos"], case["axes"], case["dim"] // 2, False) for x in (s["q"], s["new_k"]))
    return q, _exact_append(s, "k", k, hist, new), _exact_append(s, "v", s["new_v"].double(), hist, new)
