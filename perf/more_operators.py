"""Cases for further language-model operators: attention of sequences that begin
with the same pages, the choice of a token from logits, and products of matrices
in microscaled 4-bit numbers.

`run` computes a case in one of two ways: with `own` true through the
package's entry points (`infvino_b200.KvOps`), with `own` false in elementary
torch operations in 32 bits (the choice of a token in 64: which one it is goes
by sums next to a border).  `exact` computes the same from the definitions in
64 bits.

Shared beginnings: sequences groups[g] .. groups[g + 1] - 1 have their first
shared[g] tokens (whole pages) in common, in the same pages of the 8-bit cache
(`k`, `v` int8 [pages, kv_heads, page_size, dim], a power of two in `k_scale`,
`v_scale` [pages, kv_heads, page_size / 16] for each 16 tokens).

Microscaled 4-bit numbers of a [rows, width] matrix: codes uint8 [rows,
width / 2], the lower four bits first, each a sign, two bits of exponent and one
of mantissa (0, 0.5, 1, 1.5, 2, 3, 4, 6); a scale 2^(e - 127) for each block of
32 of a row, its byte e for block b of row r at scales[r // 128, b // 4, r % 32,
r % 128 // 32, b % 4] (0 where there is no such row or block).
"""
import math
import random

import torch

own = False

BLOCK = 16          # tokens that share a scale of the cache
GROUP = 32          # values that share a scale of a 4-bit matrix
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
MOST_SCORES = 6.0e8     # scores of a plain attention (float32, held whole)
MOST_CACHE = 3.0e9      # cache bytes of one case
MOST_LOGITS = 512 * 150001
MOST_PRODUCT = 4001 * 4096 * 14336
MOST_MATRIX = 8191 * 8192

_ops = None


def listed():
    return [
        # eight answers to one question about a few frames, sampled side by side: latency
        {"name": "answers_one", "op": "shared", "dtype": "f16", "batch": 8, "groups": 1, "new": 1, "shared": 784, "suffix": 60,
         "kv_heads": 4, "group": 7, "dim": 128, "page": 16},
        # many conversations about one long recording
        {"name": "answers_batch", "op": "shared", "dtype": "bf16", "batch": 64, "groups": 1, "new": 1, "shared": 32768, "suffix": 500,
         "kv_heads": 8, "group": 4, "dim": 128, "page": 64},
        # several recordings, each with its own conversations; drafted tokens are checked
        {"name": "answers_drafted", "op": "shared", "dtype": "f16", "batch": 96, "groups": 6, "new": 4, "shared": 8192, "suffix": 1023,
         "kv_heads": 4, "group": 8, "dim": 64, "page": 32},
        # questions of some hundred tokens read at once behind the same frames
        {"name": "questions", "op": "shared", "dtype": "bf16", "batch": 13, "groups": 2, "new": 211, "shared": 20000, "suffix": 0,
         "kv_heads": 8, "group": 4, "dim": 128, "page": 16},
        # one user's next token, all filters: latency
        {"name": "sample_one", "op": "sample", "dtype": "f16", "rows": 1, "vocab": 32003, "filters": "all", "masked": False},
        # a serving batch with constrained answers: most tokens are ruled out in some rows
        {"name": "sample_batch", "op": "sample", "dtype": "f32", "rows": 64, "vocab": 131072, "filters": "all", "masked": True},
        # many samples at once from the most probable tokens
        {"name": "sample_many", "op": "sample", "dtype": "bf16", "rows": 512, "vocab": 150001, "filters": "top_p", "masked": False},
        # a step's activations to 4 bits and back
        {"name": "quantize_step", "op": "quantize", "dtype": "f16", "rows": 16, "width": 4096},
        # a weight matrix, or a prompt's activations
        {"name": "quantize_large", "op": "quantize", "dtype": "bf16", "rows": 8191, "width": 8192},
        # one user's decode step: a projection for one token
        {"name": "linear_one", "op": "linear", "dtype": "f16", "rows": 1, "width": 4096, "outputs": 6144},
        # a serving batch's step through a wide projection
        {"name": "linear_batch", "op": "linear", "dtype": "bf16", "rows": 61, "width": 8192, "outputs": 28672},
        # a prompt through the feed-forward part
        {"name": "linear_prompt", "op": "linear", "dtype": "bf16", "rows": 4001, "width": 4096, "outputs": 14336},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["shared", "shared", "sample", "quantize", "linear", "linear"])
    dtype = rng.choice(["f16", "bf16"])
    if op == "sample":
        rows = _log(rng, 1, 512)
        return {"op": op, "dtype": rng.choice(["f16", "bf16", "f32"]), "rows": rows,
                "vocab": min(_log(rng, 1000, 262144), MOST_LOGITS // rows),
                "filters": rng.choice(["all", "all", "top_k", "top_p", "min_p", "none"]), "masked": rng.random() < 0.3}
    if op == "quantize":
        rows = _log(rng, 1, 8191)
        return {"op": op, "dtype": dtype, "rows": rows, "width": GROUP * _log(rng, 1, min(28672, MOST_MATRIX // rows) // GROUP)}
    if op == "linear":
        rows = rng.choice([_log(rng, 1, 64), _log(rng, 1, 4001)])
        width = GROUP * _log(rng, 4, 14336 // GROUP)
        return {"op": op, "dtype": dtype, "rows": rows, "width": width,
                "outputs": _log(rng, 65, max(65, min(28672, MOST_PRODUCT // (rows * width))))}
    new = rng.choice([1, 1, rng.randint(2, 8), _log(rng, 9, 211)])
    groups = rng.choice([1, rng.randint(1, 8)])
    batch = max(groups, _log(rng, 2, 128 if new <= 8 else 16))
    kv_heads, group, dim = rng.choice([1, 2, 3, 4, 5, 8]), rng.randint(1, 8), rng.choice([64, 128])
    page = rng.choice([16, 32, 48, 64, 128])
    suffix = rng.choice([0, _log(rng, 1, 1023)])
    room = int(MOST_SCORES / (batch * new * kv_heads * group)) - suffix - new
    shared = min(_log(rng, page, 32768), max(page, room), int(MOST_CACHE / (2 * kv_heads * dim * groups)))
    return {"op": op, "dtype": dtype, "batch": batch, "groups": groups, "new": new, "shared": shared, "suffix": suffix,
            "kv_heads": kv_heads, "group": group, "dim": dim, "page": page}


# ---------------------------------------------------------------- what a case stands for

def _lengths(case):
    """Of each group: its first sequence, shared tokens; of each sequence: its own tokens before the call, new ones."""
    r = random.Random("%d %d %d %d" % (case["batch"], case["groups"], case["new"], case["shared"]))
    batch, many, page, n = case["batch"], case["groups"], case["page"], case["new"]
    cuts = sorted(r.sample(range(1, batch), many - 1)) if many > 1 else []
    shared = [max(1, (case["shared"] if g == 0 else r.randint(case["shared"] // 4, case["shared"])) // page) * page for g in range(many)]
    mine = [r.randint(case["suffix"] // 4, case["suffix"]) for _ in range(batch)]
    new = [n] + [r.randint(-(-n // 3), n) for _ in range(batch - 1)]
    return [0] + cuts + [batch], shared, mine, new


def work(case):
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * (4 if case["dtype"] == "f32" else 2) + case["rows"] * 28, "flops": n * 16}
    if case["op"] == "quantize":
        n = case["rows"] * case["width"]
        # values read, codes and scales written; codes and scales read, values written
        return {"bytes": int(n * (2 + 2 * 17 / 32 + 2)), "flops": n * 4}
    if case["op"] == "linear":
        t, k, n = case["rows"], case["width"], case["outputs"]
        return {"bytes": int(n * k * 17 / 32) + t * (k + n) * 2, "flops": 2 * t * k * n}
    groups, shared, mine, new = _lengths(case)
    hk, hq, d = case["kv_heads"], case["kv_heads"] * case["group"], case["dim"]
    pairs, keys = 0, sum(shared)
    for g, p in enumerate(shared):
        for b in range(groups[g], groups[g + 1]):
            pairs += new[b] * (p + mine[b]) + new[b] * (new[b] + 1) // 2
            keys += mine[b] + new[b]
    return {"bytes": int(keys * 2 * hk * (d + 4 / BLOCK)) + 2 * sum(new) * hq * d * 2, "flops": 4 * d * hq * pairs}


# ---------------------------------------------------------------- inputs

def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _prepare_shared(case, gen):
    groups, shared, mine, new = _lengths(case)
    page, hk, hq, d = case["page"], case["kv_heads"], case["kv_heads"] * case["group"], case["dim"]
    lead = [p // page for p in shared]
    need = [-(-(m + n) // page) for m, n in zip(mine, new)]
    total = sum(lead) + sum(need) + 3
    order = torch.randperm(total, generator=gen, device="cuda").tolist()  # a cache that has been in use: pages in any order
    width = max(lead) + max(need)
    table, at, lens = [], sum(lead), []
    for g in range(len(lead)):
        first = sum(lead[:g])
        for b in range(groups[g], groups[g + 1]):
            row = order[first:first + lead[g]] + order[at:at + need[b]]
            at += need[b]
            table.append(row + [order[-1]] * (width - len(row)))
            lens.append(shared[g] + mine[b] + new[b])
    shape = (total, hk, page, d)

    def codes():
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float16).mul_(30.0).round_().clamp_(-127, 127).to(torch.int8)

    def scales():
        e = torch.randint(-6, -3, (total, hk, page // BLOCK), generator=gen, device="cuda")
        return torch.ldexp(torch.ones((), device="cuda"), e)

    t, dt = sum(new), TYPES[case["dtype"]]
    q = torch.randn((t, hq, d), generator=gen, device="cuda").mul_(3.0).to(dt)
    return {"case": case, "k": codes(), "v": codes(), "k_scale": scales(), "v_scale": scales(), "q": q, "out": torch.empty_like(q),
            "offsets": _ints([sum(new[:b]) for b in range(len(new) + 1)]), "lens": _ints(lens), "pages": _ints(table), "max_new": max(new),
            "groups": _ints(groups), "shared": _ints(shared), "scratch": torch.empty(t * hq * (d + 2), device="cuda")}


def _prepare_sample(case, gen):
    rows, vocab, f = case["rows"], case["vocab"], case["filters"]

    def uniform(lo, hi, n=(rows,)):
        return torch.rand(n, generator=gen, device="cuda").mul_(hi - lo).add_(lo)

    def choice(values, **kind):
        return torch.tensor(values, device="cuda", **kind)[torch.randint(len(values), (rows,), generator=gen, device="cuda")]

    # a wide heap of tokens, and some twenty that the model has in mind
    x = torch.randn((rows, vocab), generator=gen, device="cuda").mul_(2.0)
    some = torch.randint(vocab, (rows, 20), generator=gen, device="cuda")
    x.scatter_add_(1, some, uniform(2.0, 11.0, (rows, 20)))
    x = x.to(TYPES[case["dtype"]])
    if case["masked"]:
        allowed = torch.rand((rows, vocab), generator=gen, device="cuda") < torch.exp(uniform(-7.0, 0.0))[:, None]
        allowed.scatter_(1, some[:, :1], True)
        x.masked_fill_(~allowed, -math.inf)
    s = {"case": case, "logits": x, "u": torch.rand(rows, generator=gen, device="cuda"),
         "tokens": torch.empty(rows, dtype=torch.int32, device="cuda"), "probs": torch.empty(rows, device="cuda"),
         "temperature": uniform(0.4, 1.3), "top_k": None, "top_p": None, "min_p": None}
    if f == "all":
        s["temperature"] = s["temperature"] * choice([0.0, 1.0, 1.0, 1.0, 1.0])  # some rows want the most probable token
    if f in ("all", "top_k"):
        s["top_k"] = choice([0, 1, 20, 50, 1000], dtype=torch.int32)
    if f in ("all", "top_p"):
        s["top_p"] = uniform(0.7, 1.0)
    if f in ("all", "min_p"):
        s["min_p"] = choice([0.0, 0.02, 0.1])
    return s


def _activations(rows, width, dt, gen):
    spread = torch.exp(torch.randn(width, generator=gen, device="cuda"))  # some channels are far larger than others
    return torch.randn((rows, width), generator=gen, device="cuda").mul_(spread).to(dt)


def _empty(rows, width):
    return {"codes": torch.empty((rows, width // 2), dtype=torch.uint8, device="cuda"),
            "scales": torch.empty((-(-rows // 128), -(-width // 128), 32, 4, 4), dtype=torch.uint8, device="cuda")}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "shared":
        return _prepare_shared(case, gen)
    if case["op"] == "sample":
        return _prepare_sample(case, gen)
    t, k, dt = case["rows"], case["width"], TYPES[case["dtype"]]
    s = {"case": case, "x": _activations(t, k, dt, gen), "m": _empty(t, k)}
    if case["op"] == "quantize":
        s["out"] = torch.empty_like(s["x"])
        return s
    n = case["outputs"]
    w = torch.randn((n, k), generator=gen, device="cuda").mul_(k ** -0.5)
    codes, e = _quantize(w)
    s["w"] = _empty(n, k)
    s["w"]["codes"].copy_(_packed(codes))
    s["w"]["scales"].copy_(_tiled(e + 127))
    s["out"] = torch.empty((t, n), device="cuda", dtype=dt)
    return s


# ---------------------------------------------------------------- the framework's operators

def _own(s):
    import infvino_b200 as ivb
    global _ops
    if _ops is None:
        _ops = ivb.KvOps(device=0)
    c, st = s["case"], torch.cuda.current_stream().cuda_stream
    if c["op"] == "shared":
        cache = ivb.KvCache(s["k"], s["v"], s["k_scale"], s["v_scale"])
        _ops.attend_shared(cache, s["q"], s["out"], s["offsets"], s["lens"], s["pages"], s["groups"], s["shared"], s["scratch"],
                           max_new=s["max_new"], scale=c["dim"] ** -0.5, stream=st)
        return s["out"]
    if c["op"] == "sample":
        _ops.sample(s["logits"], s["u"], s["tokens"], s["probs"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                    min_p=s["min_p"], stream=st)
        return s["tokens"], s["probs"]
    m = ivb.Mx4(s["m"]["codes"], s["m"]["scales"])
    if c["op"] == "quantize":
        _ops.mx4_quantize(s["x"], m, stream=st)
        _ops.mx4_read(m, s["out"], stream=st)
        return s["out"]
    _ops.mx4_linear(s["x"], ivb.Mx4(s["w"]["codes"], s["w"]["scales"]), s["out"], scratch=m, stream=st)
    return s["out"]


# ---------------------------------------------------------------- the plain forms

def _halves(s, pages):
    """Keys and values of the pages [n] as float32 [kv_heads, n * page_size, dim]."""
    for codes in ("k", "v"):
        x = s[codes][pages].unflatten(2, (-1, BLOCK)) * s[codes + "_scale"][pages][..., None, None]
        yield x.flatten(2, 3).transpose(0, 1).flatten(1, 2)


def _attend(s):
    c, q = s["case"], s["q"].float()
    hk, g, d, page = c["kv_heads"], c["group"], c["dim"], c["page"]
    out = torch.empty_like(s["q"])
    groups, shared, mine, new = _lengths(c)
    for n, p in enumerate(shared):
        b0, b1 = groups[n], groups[n + 1]
        first, last = sum(new[:b0]), sum(new[:b1])
        x = q[first:last].view(last - first, hk, g, d).permute(1, 2, 0, 3).reshape(hk, g * (last - first), d) * d ** -0.5
        k, v = _halves(s, s["pages"][b0, :p // page].long())
        a = x @ k.transpose(1, 2)
        m = a.amax(-1, keepdim=True)
        a = a.sub_(m).exp_()
        total, y = a.sum(-1, keepdim=True), a @ v
        # the sequences' own keys, all of the group at once
        most, many = max(new[b0:b1]), max(i + j for i, j in zip(mine[b0:b1], new[b0:b1]))
        count, at, lens = s["offsets"][b0 + 1:b1 + 1] - s["offsets"][b0:b1], s["offsets"][b0:b1], s["lens"][b0:b1] - p
        need = -(-many // page)
        rows = s["pages"][b0:b1]
        rows = rows[:, p // page:p // page + need].long()
        rows = torch.nn.functional.pad(rows, (0, need - rows.shape[1]))
        k, v = (z.view(hk, b1 - b0, need * page, d) for z in _halves(s, rows.flatten()))
        i = torch.arange(most, device=q.device)
        token = (at[:, None] + i).clamp(max=q.shape[0] - 1)                 # [sequences, new]
        own = x.view(hk, g, last - first, d)[:, :, (token - first).clamp(max=last - first - 1)]  # [hk, g, sequences, new, d]
        own = own.transpose(1, 2).reshape(hk, b1 - b0, g * most, d)
        a = (own @ k.transpose(2, 3)).view(hk, b1 - b0, g, most, -1)
        j = torch.arange(need * page, device=q.device)
        seen = j <= (lens - count)[:, None, None] + i[:, None]               # [sequences, new, keys]
        a.masked_fill_(~seen[None, :, None], -math.inf)
        m2 = a.amax(-1, keepdim=True)
        a = a.sub_(m2).exp_()
        total2 = a.sum(-1, keepdim=True)
        y2 = (a.view(hk, b1 - b0, g * most, -1) @ v).view(hk, b1 - b0, g, most, d)
        seq = torch.repeat_interleave(torch.arange(b1 - b0, device=q.device), count, output_size=last - first)
        at = torch.arange(last - first, device=q.device) - (at - first)[seq]

        def packed(z):  # [hk, sequences, g, new, .] -> [hk, g, tokens, .]
            return z.transpose(1, 2)[:, :, seq, at]

        m, total, y = (z.view(hk, g, last - first, -1) for z in (m, total, y))
        m2, total2, y2 = packed(m2), packed(total2), packed(y2)
        top = torch.maximum(m, m2)
        w, w2 = torch.exp(m - top), torch.exp(m2 - top)
        y = (y * w + y2 * w2) / (total * w + total2 * w2)
        out[first:last] = y.permute(2, 0, 1, 3).reshape(last - first, hk * g, d).to(out.dtype)
    return out


def _sample(s):
    x = s["logits"].float()
    vocab, t = x.shape[1], s["temperature"][:, None].double()
    x, index = x.sort(dim=1, descending=True, stable=True)
    w = torch.exp((x.double() - x[:, :1]) / torch.where(t > 0, t, 1.0))
    place = torch.arange(vocab, device=x.device)
    keep = (place == 0) | (t > 0)
    if s["top_k"] is not None:
        k = s["top_k"][:, None]
        keep = keep & ((k <= 0) | (place < k))
    if s["top_p"] is not None:
        p = s["top_p"][:, None].double()
        c = (w * keep).cumsum(1)
        before = torch.nn.functional.pad(c, (1, 0))[:, :-1]
        keep = keep & ((before < p * c[:, -1:]) | (p >= 1))
    if s["min_p"] is not None:
        keep = keep & (w >= s["min_p"][:, None].double())
    w = torch.zeros_like(w).scatter_(1, index, w * keep)
    c = w.cumsum(1)
    token = (c <= s["u"][:, None].double() * c[:, -1:]).sum(1, keepdim=True)
    return token[:, 0].to(torch.int32), (w.gather(1, token) / c[:, -1:])[:, 0].float()


def _times_power(x, e):
    """x 2^e, e in -127..127, as products with powers of two that are made of their bits."""
    for part in (e // 2, e - e // 2):
        x = x * ((part + 127) << 23).view(torch.float32)
    return x


def _quantize(x):
    """Codes [rows, width] and exponents [rows, width / 32] of float32 values."""
    y = x.unflatten(1, (-1, GROUP))
    most = y.abs().amax(-1)
    e = (torch.frexp(most)[1] - 3).clamp(-127, 127)          # floor(log2 most) - 2
    e = torch.where(most == 0, -127, e)
    y = _times_power(y, -e[..., None])
    a = y.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    a = (torch.round(a / step) * step).clamp(max=6.0)        # ties to even multiples: the even mantissas
    code = torch.where(a < 2, a * 2, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8)
    return (code + 8 * torch.signbit(y).to(torch.uint8)).flatten(1), e


def _packed(codes):
    return codes[:, 0::2] | (codes[:, 1::2] << 4)


def _tiled(e):
    """Scale bytes [rows, blocks] in their places."""
    rows, blocks = e.shape
    e = torch.nn.functional.pad(e.to(torch.uint8), (0, -blocks % 4, 0, -rows % 128))
    return e.view(-(-rows // 128), 4, 32, -(-blocks // 4), 4).permute(0, 3, 2, 1, 4)


def _values(m, rows, width):
    """The matrix that codes and scales stand for, float32."""
    c = m["codes"].long()
    c = torch.stack([c & 15, c >> 4], -1).flatten(1)
    v = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=c.device)
    v = torch.cat([v, -v])[c]
    e = m["scales"].permute(0, 3, 2, 1, 4).flatten(0, 2).flatten(1)[:rows, :width // GROUP].int() - 127
    return _times_power(v.unflatten(1, (-1, GROUP)), e[..., None]).flatten(1)


def _quantized(s):
    codes, e = _quantize(s["x"].float())
    s["m"]["codes"].copy_(_packed(codes))
    s["m"]["scales"].copy_(_tiled(e + 127))
    return _values(s["m"], *s["x"].shape)


def _plain(s):
    c = s["case"]
    if c["op"] == "shared":
        return _attend(s)
    if c["op"] == "sample":
        return _sample(s)
    x = _quantized(s)
    if c["op"] == "quantize":
        return x.to(s["x"].dtype)
    return (x @ _values(s["w"], c["outputs"], c["width"]).t()).to(s["out"].dtype)


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------- the definitions in 64 bits

def _exact_attention(s):
    c, q, got = s["case"], s["q"], []
    groups, shared, mine, new = _lengths(c)
    first = 0
    for g, p in enumerate(shared):
        for b in range(groups[g], groups[g + 1]):
            n, length = new[b], p + mine[b] + new[b]
            rows, heads = s["pages"][b, :-(-length // c["page"])].long(), []
            hidden = torch.arange(length, device=q.device) > torch.arange(length - n, length, device=q.device)[:, None]
            for head in range(c["kv_heads"]):
                k, v = ((s[z][rows, head].double() * s[z + "_scale"][rows, head].double().repeat_interleave(BLOCK, 1)[..., None]).flatten(0, 1)[:length]
                        for z in ("k", "v"))
                a = torch.einsum("nhd,kd->hnk", q[first:first + n, head * c["group"]:(head + 1) * c["group"]].double(), k) / math.sqrt(c["dim"])
                heads.append(torch.softmax(a.masked_fill(hidden, -math.inf), -1) @ v)
            got.append(torch.cat(heads).transpose(0, 1))
            first += n
    return torch.cat(got)


def _exact_sample(s):
    tokens, probs = [], []
    off = [None] * s["logits"].shape[0]
    rows = zip(s["logits"], *(off if s[n] is None else s[n].tolist() for n in ("u", "temperature", "top_k", "top_p", "min_p")))
    for x, u, t, k, p, least in rows:
        x = x.double()
        best = int((x == x.max()).nonzero()[0])
        if not t > 0:
            tokens.append(best)
            probs.append(1.0)
            continue
        index = (x > -math.inf).nonzero()[:, 0]                # in rising order
        w = torch.exp((x[index] - x[best]) / t)
        order = torch.argsort(x[index], descending=True, stable=True)
        if k:
            order = order[:k]
        if p is not None and p < 1:
            mass = torch.cumsum(w[order], 0)
            order = order[:int(torch.searchsorted(mass, p * mass[-1])) + 1]
        order = order.sort().values
        index, w = index[order], w[order]
        if least:
            index, w = index[w >= least], w[w >= least]
        mass = torch.cumsum(w, 0)
        i = min(int(torch.searchsorted(mass, u * mass[-1], right=True)), len(index) - 1)
        tokens.append(int(index[i]))
        probs.append(float(w[i] / mass[-1]))
    device = s["logits"].device
    return torch.tensor(tokens, dtype=torch.int32, device=device), torch.tensor(probs, dtype=torch.float64, device=device)


def _exact_values(x):
    """What a matrix in 64 bits becomes in 4, by the nearest of the eight magnitudes."""
    y = x.unflatten(1, (-1, GROUP))
    most = y.abs().amax(-1, keepdim=True)
    e = ((most.view(torch.int64) >> 52) - 1023 - 2).clamp(-127, 127)
    scale = ((e + 1023) << 52).view(torch.float64)
    a = y.abs() / scale
    got = torch.zeros_like(a)
    # halfway goes to the magnitude with an even last bit
    for low, border, up in ((0.25, False, 0.5), (0.75, True, 1.0), (1.25, False, 1.5), (1.75, True, 2.0), (2.5, False, 3.0), (3.5, True, 4.0),
                            (5.0, False, 6.0)):
        got = torch.where(a >= low if border else a > low, up, got)
    return (torch.copysign(got, y) * scale).flatten(1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "shared":
        return _exact_attention(s)
    if case["op"] == "sample":
        return _exact_sample(s)
    x = _exact_values(s["x"].double())
    if case["op"] == "quantize":
        return x
    return x @ _values(s["w"], case["outputs"], case["width"]).double().t()
