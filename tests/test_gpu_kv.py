"""The language-model operators (infvino_b200.KvOps) against the definitions in
64 bits: rotation, append to the 8-bit paged cache, read, attention."""
import math

import numpy as np
import pytest
import torch

import infvino_b200 as ivb

pytestmark = pytest.mark.gpu
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
HALF_ULP = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}   # relative rounding to the type
TINY = {"f16": 2.0 ** -25, "bf16": 2.0 ** -133}     # and below its normal range
BLOCK = 16


@pytest.fixture(scope="module")
def ops():
    with ivb.KvOps(0) as o:
        yield o


def stream():
    return torch.cuda.current_stream().cuda_stream


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def offsets_of(new):
    return ints([0] + list(np.cumsum(new)))


def page_table(lens, page, spare=2, seed=0):
    """Pages in a mixed order; unused entries hold -1."""
    need = [max(1, -(-n // page)) for n in lens]
    order = np.random.default_rng(seed).permutation(sum(need) + spare)
    t = np.full((len(lens), max(need)), -1, dtype=np.int32)
    at = 0
    for b, n in enumerate(need):
        t[b, :n] = order[at:at + n]
        at += n
    return t, sum(need) + spare


# ---------------------------------------------------------------- rotation

def turned(x, table, pos, axis, interleaved):
    x, pairs = x.double(), len(axis)
    c, s = (torch.stack([table.double()[pos[a].long(), i, k] for i, a in enumerate(axis)], 1)[:, None] for k in (0, 1))
    y = x.clone()
    ai, bi = (range(0, 2 * pairs, 2), range(1, 2 * pairs, 2)) if interleaved else (range(pairs), range(pairs, 2 * pairs))
    ai, bi = list(ai), list(bi)
    y[..., ai] = x[..., ai] * c - x[..., bi] * s
    y[..., bi] = x[..., bi] * c + x[..., ai] * s
    return y


def close_rotation(got, want, x, dtype):
    # one rounding to the type, and three in f32 over terms of at most max |x| (a head's pair)
    bound = HALF_ULP[dtype] * want.abs() + TINY[dtype] + 2.0 ** -22 * x.double().abs().amax(-1, keepdim=True)
    assert ((got.double() - want).abs() <= bound).all()


def some_axes(pairs, axes):
    return sorted(i * axes // pairs for i in range(pairs)) if axes != 3 else [(i * 7 + i // 5) % 3 for i in range(pairs)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("tokens,heads,dim,pairs,axes,interleaved", [
    (1, 1, 64, 32, 1, False), (1, 1, 16, 8, 1, True), (3, 5, 128, 64, 3, False), (17, 7, 128, 64, 2, True),
    (33, 3, 80, 24, 4, False), (2000, 12, 128, 32, 3, True), (1501, 9, 256, 128, 2, False), (5, 300, 64, 8, 1, False)])
def test_rope(ops, dtype, tokens, heads, dim, pairs, axes, interleaved):
    g = torch.Generator(device="cuda").manual_seed(tokens)
    table = torch.empty((5000, pairs, 2), device="cuda")
    inv = [10000.0 ** (-i / pairs) for i in range(pairs)]
    ops.rope_table(inv, table, stream())
    a = torch.arange(5000, dtype=torch.float64, device="cuda")[:, None] * torch.tensor(inv, dtype=torch.float64, device="cuda")
    assert (table.double() - torch.stack([a.cos(), a.sin()], -1)).abs().max() <= 2.0 ** -24
    x = torch.randn((tokens, heads, dim), generator=g, device="cuda").to(TYPES[dtype])
    pos = torch.randint(0, 5000, (axes, tokens), generator=g, device="cuda", dtype=torch.int32)
    axis = some_axes(pairs, axes)
    out = torch.full_like(x, float("nan"))
    ops.rope(x, out, ivb.Rotary(table, axis, interleaved), pos, stream())
    want = turned(x, table, pos, axis, interleaved)
    close_rotation(out, want, x, dtype)
    assert torch.equal(out[..., 2 * pairs:], x[..., 2 * pairs:])
    ops.rope(x, x, ivb.Rotary(table, axis, interleaved), pos, stream())  # in place
    assert torch.equal(x, out)
    ops.synchronize(stream())


@pytest.mark.parametrize("layout", ["sliced", "heads_first", "odd_offset", "odd_stride"])
def test_rope_layouts(ops, layout):
    """Strides of a slice of a packed projection, of a transposed tensor, and rows off the 16-byte grid."""
    t, h, d = 37, 6, 64
    base = {"sliced": lambda: torch.randn(t, 3 * h, d)[:, h:2 * h], "heads_first": lambda: torch.randn(h, t, d).transpose(0, 1),
            "odd_offset": lambda: torch.randn(t * h * d + 3)[3:].view(t, h, d),
            "odd_stride": lambda: torch.randn(t, h, d + 5)[..., :d]}[layout]
    wide = base()
    dev = torch.empty_strided(wide.shape, wide.stride(), dtype=torch.float16, device="cuda")
    if layout == "odd_offset":
        dev = torch.empty(t * h * d + 3, dtype=torch.float16, device="cuda")[3:].view(t, h, d)
    dev.copy_(wide)
    table = torch.randn((64, 32, 2), device="cuda")
    pos = torch.randint(0, 64, (1, t), device="cuda", dtype=torch.int32)
    guard = torch.full((t, h + 2, d), 7.0, dtype=torch.float16, device="cuda")
    ops.rope(dev, guard[:, 1:h + 1], ivb.Rotary(table), pos, stream())
    want = turned(dev, table, pos, [0] * 32, False)
    bound = HALF_ULP["f16"] * want.abs() + TINY["f16"] + 2.0 ** -22 * (dev.double().abs().amax(-1, keepdim=True) * table.abs().max().double())
    assert ((guard[:, 1:h + 1].double() - want).abs() <= bound).all()
    assert (guard[:, 0] == 7).all() and (guard[:, -1] == 7).all()


# ---------------------------------------------------------------- append and read

class Model:
    """The cache's definition on the host: codes and exponents of each sequence and head."""

    def __init__(self, batch, heads, dim, room):
        self.codes = np.zeros((batch, room, heads, dim), dtype=np.int64)
        self.exp = np.full((batch, -(-room // BLOCK), heads), -120, dtype=np.int64)

    def append(self, b, start, x):
        """x [n, heads, dim]: f32 values (as the rotation gives them)."""
        for blk in range(start // BLOCK, -(-(start + len(x)) // BLOCK)):
            lo, hi = max(start, blk * BLOCK), min(start + len(x), blk * BLOCK + BLOCK)
            new = x[lo - start:hi - start].astype(np.float64)
            finite = np.where(np.isfinite(new), np.abs(new), 0)
            for h in range(x.shape[1]):
                m = finite[:, h].max()
                e = -120 if m == 0 else int(np.clip(math.ceil(math.log2(m / 127)), -120, 121))
                while m > 127 * 2.0 ** e and e < 121:
                    e += 1
                while e > -120 and m <= 127 * 2.0 ** (e - 1):
                    e -= 1
                if lo > blk * BLOCK:
                    old = self.exp[b, blk, h]
                    if e > old:
                        c = self.codes[b, blk * BLOCK:lo, h]
                        self.codes[b, blk * BLOCK:lo, h] = np.rint(c * 2.0 ** float(max(old - e, -60)))
                    e = max(e, old)
                self.exp[b, blk, h] = e
                v = np.nan_to_num(new[:, h] * 2.0 ** float(-e), nan=0.0, posinf=127, neginf=-127)
                self.codes[b, lo:hi, h] = np.clip(np.rint(v), -127, 127)


def new_cache(pages, heads, page, dim):
    """Codes and scales that nothing valid may come from."""
    k, v = (torch.full((pages, heads, page, dim), 99, dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.full((pages, heads, page // BLOCK), float("nan"), device="cuda") for _ in range(2))
    return k, v, ks, vs


def held(codes, scales, table, lens):
    """Codes and scales of each sequence in order, on the host."""
    page = codes.shape[2]
    c, s, got = codes.cpu().numpy(), scales.cpu().numpy(), []
    for b, n in enumerate(lens):
        pos = np.arange(n)
        got.append((c[table[b, pos // page], :, pos % page].astype(np.int64), s[table[b, pos // page], :, pos % page // BLOCK]))
    return got


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,dim,page,steps", [
    (2, 64, 16, [[5, 1, 0], [1, 1, 1], [1, 30, 16]]),
    (1, 128, 48, [[1, 1], [1, 1], [1, 1], [15, 3], [1, 1]]),
    (3, 128, 64, [[100, 17, 1, 64], [1, 1, 1, 1], [40, 0, 0, 16]]),
    (5, 64, 32, [[1] * 9] * 5),
    (2, 128, 128, [[700, 0, 600], [3, 2, 0], [300, 1200, 1]])])  # over 1024 tokens in a call too
def test_append_read(ops, dtype, heads, dim, page, steps):
    batch, dt = len(steps[0]), TYPES[dtype]
    lens = [sum(s[b] for s in steps) for b in range(batch)]
    table, pages = page_table(lens, page, seed=dim)
    cache_t = new_cache(pages, heads, page, dim)
    cache, dev_table = ivb.KvCache(*cache_t), ints(table)
    rot_table = torch.empty((4096, dim // 2, 2), device="cuda")
    ops.rope_table([100.0 ** (-i / (dim // 2)) for i in range(dim // 2)], rot_table, stream())
    axis = some_axes(dim // 2, 3)
    rotary = ivb.Rotary(rot_table, axis)
    mk, mv = (Model(batch, heads, dim, max(lens) + BLOCK) for _ in range(2))
    start = [0] * batch
    g = torch.Generator(device="cuda").manual_seed(page)
    for step, new in enumerate(steps):
        t = sum(new)
        grow = 3.0 ** step  # later tokens are larger: scales of begun blocks grow
        k, v, q = (torch.randn((t, h, dim), generator=g, device="cuda").mul_(f).to(dt) for h, f in ((heads, grow), (heads, 0.3 * grow), (2 * heads, 1)))
        pos = torch.randint(0, 4096, (3, t), generator=g, device="cuda", dtype=torch.int32)
        q_out = torch.empty_like(q)
        ops.append(cache, k, v, offsets_of(new), ints(start), dev_table, rotary=rotary, pos=pos, q=q, q_out=q_out, stream=stream())
        close_rotation(q_out, turned(q, rot_table, pos, axis, False), q, dtype)
        # the rotation in f32, rounded operation by operation
        x = k.float()
        cs = torch.stack([rot_table[pos[a].long(), i] for i, a in enumerate(axis)], 1)[:, None]
        a, b_ = x[..., :dim // 2], x[..., dim // 2:]
        kr = torch.cat([a * cs[..., 0] - b_ * cs[..., 1], b_ * cs[..., 0] + a * cs[..., 1]], -1).cpu().numpy()
        at = 0
        for b, n in enumerate(new):
            if n:
                mk.append(b, start[b], kr[at:at + n])
                mv.append(b, start[b], v[at:at + n].float().cpu().numpy())
            at += n
            start[b] += n
        for model, (codes, scales) in ((mk, cache_t[0::2]), (mv, cache_t[1::2])):
            for b, (c, s) in enumerate(held(codes, scales, table, start)):
                assert np.array_equal(s, 2.0 ** model.exp[b, np.arange(start[b]) // BLOCK].astype(np.float64)), (step, b)
                assert np.array_equal(c, model.codes[b, :start[b]]), (step, b)
    ko, vo = (torch.empty((sum(lens), heads, dim), dtype=dt, device="cuda") for _ in range(2))
    ops.read(cache, ko, vo, offsets_of(lens), ints([0] * batch), dev_table, stream())
    for model, got in ((mk, ko), (mv, vo)):
        want = np.concatenate([model.codes[b, :n] * 2.0 ** model.exp[b, np.arange(n) // BLOCK].astype(np.float64)[..., None] for b, n in enumerate(lens)])
        assert np.array_equal(got.double().cpu().numpy(), torch.tensor(want).to(dt).double().numpy())
    only = torch.empty_like(vo)
    ops.read(cache, None, only, offsets_of(lens), ints([0] * batch), dev_table, stream())
    assert torch.equal(only, vo)
    ops.synchronize(stream())


def test_append_not_finite_and_extremes(ops):
    """NaN, infinities, zeros and the type's ends: one block of one head each."""
    dim, page = 64, 16
    rows = [torch.zeros(3, dim), torch.full((3, dim), 3.38e38), torch.full((3, dim), 1e-38), torch.randn(3, dim)]
    rows[3][0, 0], rows[3][1, 5], rows[3][2, 7] = float("nan"), float("inf"), -float("inf")
    k = torch.stack(rows, 1).to(torch.bfloat16).cuda()
    table, pages = page_table([3], page)
    cache_t = new_cache(pages, 4, page, dim)
    ops.append(ivb.KvCache(*cache_t), k, k, ints([0, 3]), ints([0]), ints(table), stream=stream())
    model = Model(1, 4, dim, 16)
    model.append(0, 0, k.float().cpu().numpy())
    (c, s), = held(cache_t[0], cache_t[2], table, [3])
    assert np.array_equal(c, model.codes[0, :3]) and np.array_equal(s, 2.0 ** model.exp[0, [0, 0, 0]].astype(np.float64))
    assert c[0, 3, 0] == 0 and c[1, 3, 5] == 127 and c[2, 3, 7] == -127


def test_append_growth_error_below_one_step(ops):
    """Fifteen growths of one block's scale: no value is off by a final step or more."""
    dim, page = 64, 16
    table, pages = page_table([16], page)
    cache_t = new_cache(pages, 1, page, dim)
    cache = ivb.KvCache(*cache_t)
    x = (torch.randn((16, 1, dim), generator=torch.Generator().manual_seed(4)) * 1.9 ** torch.arange(16)[:, None, None]).half().cuda()
    for i in range(16):
        ops.append(cache, x[i:i + 1], x[i:i + 1], ints([0, 1]), ints([i]), ints(table), stream=stream())
    (c, s), = held(cache_t[0], cache_t[2], table, [16])
    assert (np.abs(c * s.astype(np.float64)[..., None] - x.double().cpu().numpy()) < s[0, 0]).all()


# ---------------------------------------------------------------- attention

def filled_cache(pages, heads, page, dim, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    k, v = (torch.randint(-127, 128, (pages, heads, page, dim), generator=g, device="cuda").to(torch.int8) for _ in range(2))
    ks, vs = (2.0 ** torch.randint(-9, -4, (pages, heads, page // BLOCK), generator=g, device="cuda").float()
              for _ in range(2))
    return k, v, ks, vs


def attention64(cache_t, table, q, new, lens, scale, window, sinks):
    """Output and error bound of each row, in 64 bits."""
    k, v, ks, vs = (c.cpu() for c in cache_t)
    page, heads, dim = k.shape[2], k.shape[1], k.shape[3]
    group, at, outs, bounds = q.shape[1] // heads, 0, [], []
    for b, n in enumerate(new):
        need = -(-lens[b] // page)
        rows = torch.from_numpy(table[b, :need]).long()
        K, V = ((c[rows].double() * s[rows].double().repeat_interleave(BLOCK, 2)[..., None]).transpose(0, 1).reshape(heads, -1, dim)[:, :lens[b]]
                for c, s in ((k, ks), (v, vs)))
        Q = q[at:at + n].double().cpu().transpose(0, 1).reshape(heads, group, n, dim)
        p, j = torch.arange(lens[b] - n, lens[b])[:, None], torch.arange(lens[b])
        seen = j <= p
        if window:
            seen &= (p - j < window) | (j < sinks)
        s = torch.einsum("hgnd,hkd->hgnk", Q, K) * scale
        big = torch.einsum("hgnd,hkd->hgnk", Q.abs(), K.abs()) * abs(scale)
        w = torch.softmax(s.masked_fill(~seen, -math.inf), -1).nan_to_num(0.0)
        o, mass = torch.einsum("hgnk,hkd->hgnd", w, V), torch.einsum("hgnk,hkd->hgnd", w, V.abs())
        # a score: dim products summed in f32, then scaled and shifted by the maximum; its error counts twice (numerator and sum)
        off = (big * (dim + 4) * 2.0 ** -24 + s.abs() * 2.0 ** -21).masked_fill(~seen, 0).amax(-1, keepdim=True) if lens[b] else torch.zeros(heads, group, n, 1)
        bounds.append((mass * (2 * off + 2.0 ** -11 + 2.0 ** -16)).permute(2, 0, 1, 3).reshape(n, heads * group, dim))  # weights are rounded to 11 bits
        outs.append(o.permute(2, 0, 1, 3).reshape(n, heads * group, dim))
        at += n
    return torch.cat(outs), torch.cat(bounds)


def check_attention(ops, dtype, new, lens, heads, group, dim, page, window=0, sinks=0, seed=0, scale=None, q=None, max_new=None):
    dt, t = TYPES[dtype], sum(new)
    table, pages = page_table(lens, page, seed=seed)
    cache_t = filled_cache(pages, heads, page, dim, seed)
    used = set(table[table >= 0].ravel())
    for s in cache_t[2:]:  # scales that no call may read: pages out of use, blocks behind the end
        for p in set(range(pages)) - used:
            s[p] = float("nan")
    for b, n in enumerate(lens):
        last = (n - 1) // page if n else 0
        first = -(-(n - last * page) // BLOCK) if n else 0
        for s in cache_t[2:]:
            s[table[b, last], :, first:] = float("nan")
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    if q is None:
        q = torch.randn((t, heads * group, dim), generator=g, device="cuda").mul_(2).to(dt)
    scale = dim ** -0.5 if scale is None else scale
    out = torch.full((t, heads * group, dim), float("nan"), dtype=dt, device="cuda")
    ops.attend(ivb.KvCache(*cache_t), q, out, offsets_of(new), ints(lens), ints(table), max_new=max_new or max(new), scale=scale, window=window,
               sinks=sinks, stream=stream())
    ops.synchronize(stream())
    want, bound = attention64(cache_t, table, q, new, lens, scale, window, sinks)
    got = out.double().cpu()
    assert torch.isfinite(got).all()
    bound = bound * 1.01 + HALF_ULP[dtype] * want.abs() + TINY[dtype]
    assert ((got - want).abs() <= bound).all(), float(((got - want).abs() / bound).max())
    return out


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new,lens,heads,group,page", [
    ([1], [1], 1, 1, 16), ([1], [16], 2, 1, 16), ([1], [17], 1, 7, 48), ([1, 1, 1], [1, 333, 64], 3, 4, 32),
    ([1] * 5, [2049, 15, 16, 31, 700], 2, 16, 64), ([1, 1], [5000, 1], 1, 17, 128), ([1], [40000], 2, 8, 64),
    ([1, 0, 1, 0], [100, 77, 5, 0], 2, 3, 16), ([1] * 40, list(range(1, 400, 10)), 4, 2, 16)])
def test_attend_one_token(ops, dtype, dim, new, lens, heads, group, page):
    check_attention(ops, dtype, new, lens, heads, group, dim, page, seed=len(lens))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new,lens,heads,group,page", [
    ([2], [2], 1, 1, 16), ([5, 3, 1], [5, 400, 1], 2, 5, 16), ([4, 4], [1000, 129], 1, 4, 64), ([7, 0, 2], [3000, 9, 18], 2, 3, 32),
    ([128], [128], 1, 1, 64), ([129], [129], 2, 1, 16), ([130, 1, 300], [400, 200, 300], 2, 3, 48), ([257], [1000], 1, 2, 128),
    ([1000], [1000], 1, 5, 64), ([33, 34], [3333, 34], 1, 8, 32), ([600], [5000], 3, 1, 64)])
def test_attend_many_tokens(ops, dtype, dim, new, lens, heads, group, page):
    check_attention(ops, dtype, new, lens, heads, group, dim, page, seed=sum(new))


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (17, 16), (100, 33), (128, 0), (255, 1), (4096, 8), (7, 1000)])
@pytest.mark.parametrize("new,lens,dim", [([1, 1, 1], [1, 300, 1111], 64), ([1], [9000], 128), ([9, 2], [500, 2], 128), ([300, 50], [300, 900], 64),
                                          ([200], [1700], 128)])
def test_attend_window(ops, new, lens, dim, window, sinks):
    check_attention(ops, "f16", new, lens, 2, 4, dim, 32, window=window, sinks=sinks, seed=window)


@pytest.mark.parametrize("new,lens", [([3], [1]), ([1], [0]), ([4, 2], [2, 0]), ([150], [20]), ([40, 300, 1], [3, 299, 0])])
@pytest.mark.parametrize("window,sinks", [(0, 0), (8, 2)])
def test_attend_rows_without_keys(ops, new, lens, window, sinks):
    """More new tokens than the cache holds: the first rows see nothing and give 0."""
    table, pages = page_table([max(1, n) for n in lens], 16)
    cache_t = filled_cache(pages, 2, 16, 64, 3)
    q = torch.randn((sum(new), 4, 64), device="cuda").half()
    out = torch.full_like(q, float("nan"))
    ops.attend(ivb.KvCache(*cache_t), q, out, offsets_of(new), ints(lens), ints(table), max_new=max(new), window=window, sinks=sinks, stream=stream())
    ops.synchronize(stream())
    at = 0
    for b, (n, have) in enumerate(zip(new, lens)):
        empty = max(0, n - have)
        assert (out[at:at + empty] == 0).all()
        if n > empty:
            want, bound = attention64(cache_t, table[b:b + 1], q[at + empty:at + n], [n - empty], [have], 64 ** -0.5, window, sinks)
            got = out[at + empty:at + n].double().cpu()
            assert ((got - want).abs() <= bound * 1.01 + HALF_ULP["f16"] * want.abs() + TINY["f16"]).all()
        at += n


@pytest.mark.parametrize("new", [[1, 1], [6, 3], [140, 20]])
def test_attend_ranges(ops, new):
    """bf16 queries far outside half precision's range, and scales of very different size within a row."""
    lens, heads, group, dim, page, t = [n + 100 for n in new], 2, 4, 128, 16, sum(new)
    table, pages = page_table(lens, page)
    for times in (1e-12, 3e7):
        cache_t = list(filled_cache(pages, heads, page, dim, 9))
        cache_t[2] = torch.full_like(cache_t[2], 0.01 / times)
        cache_t[3] = 2.0 ** torch.randint(-60, 60, cache_t[3].shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)).float()
        q = torch.randn((t, heads * group, dim), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).mul_(times).to(torch.bfloat16)
        out = torch.empty_like(q)
        ops.attend(ivb.KvCache(*cache_t), q, out, offsets_of(new), ints(lens), ints(table), max_new=max(new), stream=stream())
        ops.synchronize(stream())
        want, bound = attention64(cache_t, table, q, new, lens, dim ** -0.5, 0, 0)
        # weights and values share 11 bits relative to the row's largest value
        got = out.double().cpu()
        bound = bound.amax(-1, keepdim=True) * 1.01 + HALF_ULP["bf16"] * want.abs() + TINY["bf16"]
        assert ((got - want).abs() <= bound).all()


def test_attend_not_finite_query_stays_in_its_row(ops):
    for new in ([1, 1, 1], [5, 3, 2], [60, 100, 30]):
        t = sum(new)
        q = torch.randn((t, 8, 64), device="cuda").half()
        q[1, 3, 7], q[t - 1, 0, 0] = float("nan"), float("inf")
        lens = [n + 70 for n in new]
        table, pages = page_table(lens, 16)
        cache = ivb.KvCache(*filled_cache(pages, 2, 16, 64, 3))
        clean, out = q.clone(), torch.empty_like(q)
        clean[1, 3, 7], clean[t - 1, 0, 0] = 0, 0
        want = torch.empty_like(q)
        ops.attend(cache, q, out, offsets_of(new), ints(lens), ints(table), max_new=max(new), stream=stream())
        ops.attend(cache, clean, want, offsets_of(new), ints(lens), ints(table), max_new=max(new), stream=stream())
        same = torch.ones((t, 8), dtype=torch.bool)
        same[1, 3] = same[t - 1, 0] = False
        assert torch.equal(out.cpu()[same], want.cpu()[same])
        assert torch.isnan(out[1, 3]).all()


@pytest.mark.parametrize("new", [[1, 1], [3, 2], [100, 90]])
@pytest.mark.parametrize("layout", ["sliced", "heads_first", "odd_offset"])
def test_attend_layouts(ops, new, layout):
    t, heads, group, dim = sum(new), 2, 3, 64
    hq = heads * group
    if layout == "sliced":
        q, out = torch.randn((t, 3 * hq, dim), device="cuda").half()[:, hq:2 * hq], torch.zeros((t, hq + 2, dim), dtype=torch.float16, device="cuda")[:, 1:-1]
    elif layout == "heads_first":
        q, out = torch.randn((hq, t, dim), device="cuda").half().transpose(0, 1), torch.zeros((hq, t, dim), dtype=torch.float16, device="cuda").transpose(0, 1)
    else:
        q, out = (torch.randn(t * hq * dim + 1, device="cuda").half()[1:].view(t, hq, dim) for _ in range(2))
    lens = [n + 50 for n in new]
    table, pages = page_table(lens, 32)
    cache = ivb.KvCache(*filled_cache(pages, heads, 32, dim, 3))
    want = torch.empty((t, hq, dim), dtype=torch.float16, device="cuda")
    args = (offsets_of(new), ints(lens), ints(table))
    ops.attend(cache, q.contiguous(), want, *args, max_new=max(new), stream=stream())
    ops.attend(cache, q, out, *args, max_new=max(new), stream=stream())
    assert torch.equal(out, want)


@pytest.mark.parametrize("new", [1, 40])
def test_offsets_past_32_bits(ops, new):
    """The pages of the sequences lie behind 2^31 code bytes."""
    dim, page = 128, 16
    pages = (1 << 31) // (page * dim) + 40
    codes = [torch.empty((pages, 1, page, dim), dtype=torch.int8, device="cuda") for _ in range(2)]
    scales = [torch.empty((pages, 1, 1), device="cuda") for _ in range(2)]
    cache = ivb.KvCache(*codes, *scales)
    lens = [300, 150]
    table = (pages - 1 - np.arange(40).reshape(2, 20)).astype(np.int32)
    x = torch.randn((sum(lens), 1, dim), device="cuda").half()
    ops.append(cache, x, -x, offsets_of(lens), ints([0, 0]), ints(table), stream=stream())
    k, v = torch.empty_like(x), torch.empty_like(x)
    ops.read(cache, k, v, offsets_of(lens), ints([0, 0]), ints(table), stream())
    assert torch.equal(v, -k) and (k - x).abs().max() < 0.04
    small = [c[-40:].clone() for c in codes + scales]
    q = torch.randn((2 * new, 4, dim), device="cuda").half()
    out, want = torch.empty_like(q), torch.empty_like(q)
    args = (offsets_of([new, new]), ints(lens))
    ops.attend(cache, q, out, *args, ints(table), max_new=new, stream=stream())
    ops.attend(ivb.KvCache(*small), q, want, *args, ints(table - (pages - 40)), max_new=new, stream=stream())
    ops.synchronize(stream())
    assert torch.equal(out, want)


def test_attend_same_bits_again(ops):
    """The same call gives the same bits, alone and beside calls on another stream."""
    for new, lens in (([1] * 7, [9000, 10, 3000, 77, 1, 4000, 512]), ([300, 20], [2000, 4000])):
        table, pages = page_table(lens, 64)
        cache = ivb.KvCache(*filled_cache(pages, 4, 64, 128, 5))
        q = torch.randn((sum(new), 16, 128), device="cuda").half()
        outs = [torch.empty_like(q) for _ in range(6)]
        args = (offsets_of(new), ints(lens), ints(table))
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for i, o in enumerate(outs):
            ops.attend(cache, q, o, *args, max_new=max(new), stream=streams[i % 2].cuda_stream)
        torch.cuda.synchronize()
        assert all(torch.equal(o, outs[0]) for o in outs)


@pytest.mark.parametrize("new", [[1, 1, 1], [200, 5, 1]])
def test_graph_capture(ops, new):
    """append + attend captured once and replayed with other contents in the same tensors."""
    lens, heads, dim, page, t = [n + 90 for n in new], 2, 128, 32, sum(new)
    table, pages = page_table(lens, page)
    cache_t = filled_cache(pages, heads, page, dim, 1)
    cache, start = ivb.KvCache(*cache_t), [t.clone() for t in cache_t]
    rot = torch.empty((512, dim // 2, 2), device="cuda")
    ops.rope_table([100.0 ** (-i / 64) for i in range(64)], rot, stream())
    k, v, q = (torch.randn((t, h, dim), device="cuda").half() for h in (heads, heads, 8))
    qr, out, offs, ln, st, tb = torch.empty_like(q), torch.empty_like(q), offsets_of(new), ints(lens), ints([90] * 3), ints(table)
    pos = torch.arange(t, device="cuda", dtype=torch.int32)

    def step(s):
        ops.append(cache, k, v, offs, st, tb, rotary=ivb.Rotary(rot), pos=pos, q=q, q_out=qr, stream=s)
        ops.attend(cache, qr, out, offs, ln, tb, max_new=max(new), stream=s)

    side = torch.cuda.Stream()
    ops.reserve(side.cuda_stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step(side.cuda_stream)
    for seed in range(2):
        for x in (k, v, q):
            x.normal_(generator=torch.Generator(device="cuda").manual_seed(seed))
        for c, s in zip(cache_t, start):
            c.copy_(s)
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        for c, s in zip(cache_t, start):
            c.copy_(s)
        step(stream())
        assert torch.equal(got, out)


# ---------------------------------------------------------------- refusals

def small_call():
    table, pages = page_table([40, 40], 16)
    cache_t = filled_cache(pages, 2, 16, 64, 3)
    q = torch.zeros((2, 4, 64), dtype=torch.float16, device="cuda")
    return cache_t, q, torch.empty_like(q), ints([0, 1, 2]), ints([40, 40]), ints(table)


def test_refusals(ops):
    cache_t, q, out, offs, lens, table = small_call()
    cache = ivb.KvCache(*cache_t)
    with pytest.raises(ValueError):
        ops.attend(cache, q.float(), out, offs, lens, table, max_new=1)
    with pytest.raises(ValueError):
        ops.attend(cache, q, out[:1], offs, lens, table, max_new=1)
    with pytest.raises(ValueError):
        ops.attend(cache, q, out, offs[:2], lens, table, max_new=1)
    with pytest.raises(ValueError):
        ops.attend(cache, q, out, offs.long(), lens, table, max_new=1)
    with pytest.raises(ValueError):
        ops.attend(cache, q[..., ::2], out, offs, lens, table, max_new=1)
    for args in ((cache, q.cpu(), out, offs, lens, table), (cache, q, out.cpu(), offs, lens, table), (cache, q, out, offs, lens.cpu(), table),
                 (ivb.KvCache(*[t.cpu() for t in cache_t]), q, out, offs, lens, table)):
        with pytest.raises(ValueError):  # host memory
            ops.attend(*args, max_new=1)
    for bad in (dict(max_new=0), dict(max_new=1, window=-1), dict(max_new=1, sinks=-2)):
        with pytest.raises(ivb.NativeError) as e:
            ops.attend(cache, q, out, offs, lens, table, **bad)
        assert e.value.status == 1 and "ivc_kv_attend" in e.value.message
    with pytest.raises(ivb.NativeError) as e:  # 3 query heads over 2 kv heads
        ops.attend(cache, q[:, :3], out[:, :3], offs, lens, table, max_new=1)
    assert e.value.status == 1
    odd = filled_cache(4, 2, 16, 96, 3)
    x = torch.zeros((2, 2, 96), dtype=torch.float16, device="cuda")
    with pytest.raises(ivb.NativeError):
        ops.append(ivb.KvCache(*odd), x, x, offs, lens, table)
    rotary = ivb.Rotary(torch.zeros((8, 64, 2), device="cuda"))
    with pytest.raises(ivb.NativeError):  # 64 pairs in a head of 64
        ops.rope(q, out, rotary, ints([0, 1]))
    with pytest.raises(ValueError):
        ops.rope(q, out, rotary, ints([0, 1, 2]))
    with pytest.raises(ivb.NativeError):
        ivb.KvOps(99)
    # no tokens: nothing to do
    ops.attend(cache, q[:0], out[:0], ints([0, 0, 0]), lens, table, max_new=0)
    ops.append(cache, q[:0, :2], q[:0, :2], ints([0, 0, 0]), lens, table)


@pytest.mark.parametrize("what", ["page", "negative_page", "length", "offsets", "max_new", "position"])
@pytest.mark.parametrize("tokens", [1, 40])
def test_device_side_errors_are_reported(ops, what, tokens):
    """What only the kernels can see: they skip it, and synchronize reports it once."""
    lens_v, table = [60, 60], page_table([60, 60], 16)
    pages, table = table[1], table[0]
    cache_t = filled_cache(pages, 2, 16, 64, 3)
    q = torch.zeros((2 * tokens, 4, 64), dtype=torch.float16, device="cuda")
    offs, max_new = [0, tokens, 2 * tokens], tokens
    if what == "page":
        table[1, 2] = pages
    elif what == "negative_page":
        table[0, 0] = -5
    elif what == "length":
        lens_v[0] = 65  # five pages, the table has four
    elif what == "offsets":
        offs = [0, tokens, tokens - 1] if tokens > 1 else [1, 0, 2]
    elif what == "max_new":
        offs = [0, 0, 2 * tokens]
    if what == "position":
        rotary = ivb.Rotary(torch.zeros((100, 32, 2), device="cuda"))
        ops.rope(q, q, rotary, torch.full((2 * tokens,), 100, dtype=torch.int32, device="cuda"), stream())
    else:
        ops.attend(ivb.KvCache(*cache_t), q, torch.empty_like(q), ints(offs), ints(lens_v), ints(table), max_new=max_new, stream=stream())
    with pytest.raises(ivb.NativeError) as e:
        ops.synchronize(stream())
    assert e.value.status == 5
    ops.synchronize(stream())


@pytest.mark.parametrize("what", ["page", "start", "position"])
def test_append_device_side_errors(ops, what):
    table, pages = page_table([40, 40], 16)
    start = [0, 16]
    if what == "page":
        table[1, 1] = pages + 3
    elif what == "start":
        start[1] = 48
    cache_t = new_cache(pages, 2, 16, 64)
    x = torch.ones((8, 2, 64), dtype=torch.float16, device="cuda")
    rotary = ivb.Rotary(torch.ones((4, 32, 2), device="cuda"))
    pos = torch.full((8,), 9 if what == "position" else 1, dtype=torch.int32, device="cuda")
    ops.append(ivb.KvCache(*cache_t), x, x, ints([0, 4, 8]), ints(start), ints(table), rotary=rotary, pos=pos, stream=stream())
    with pytest.raises(ivb.NativeError) as e:
        ops.synchronize(stream())
    assert e.value.status == 5
    ops.synchronize(stream())
