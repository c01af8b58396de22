"""KvOps.attend_shared: attention of sequences that begin with the same pages,
against the definition in 64 bits and against `attend` on the same pages."""
import math

import numpy as np
import pytest
import torch

import infvino_b200 as ivb

pytestmark = pytest.mark.gpu
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
HALF_ULP = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f16": 2.0 ** -25, "bf16": 2.0 ** -134}
BLOCK = 16


@pytest.fixture(scope="module")
def ops():
    with ivb.KvOps(0) as o:
        yield o


def stream():
    return torch.cuda.current_stream().cuda_stream


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Case:
    """groups: [(common pages, [(own tokens before, new tokens), ...]), ...]"""

    def __init__(self, groups, heads, group, dim, page, dtype="f16", seed=0, spread=2.0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.heads, self.group, self.dim, self.page, self.dtype = heads, group, dim, page, dtype
        seqs = [(n, *s) for n, (_, many) in enumerate(groups) for s in many]
        self.batch, self.new = len(seqs), [s[2] for s in seqs]
        self.first = np.cumsum([0] + [len(m) for _, m in groups])
        self.common = [p * page for p, _ in groups]
        need = [-(-(m + n) // page) for _, m, n in seqs]
        total = sum(p for p, _ in groups) + sum(need) + 2
        order = np.random.default_rng(seed).permutation(total)
        width = max([1] + [groups[s[0]][0] + k for s, k in zip(seqs, need)])
        self.full = np.full((self.batch, width), -1, np.int32)  # every sequence's pages
        at = 0
        for n, (p, many) in enumerate(groups):
            self.full[self.first[n]:self.first[n + 1], :p] = order[at:at + p]
            at += p
        for b, (s, k) in enumerate(zip(seqs, need)):
            p = groups[s[0]][0]
            self.full[b, p:p + k] = order[at:at + k]
            at += k
        self.table = self.full.copy()  # where only a group's first sequence names the common pages
        for n, (p, _) in enumerate(groups):
            self.table[self.first[n] + 1:self.first[n + 1], :p] = -1
        self.lens = [self.common[n] + m + k for n, m, k in seqs]
        codes = [torch.randint(-127, 128, (total, heads, page, dim), generator=g, device="cuda").to(torch.int8) for _ in range(2)]
        scales = [2.0 ** torch.randint(-9, -4, (total, heads, page // BLOCK), generator=g, device="cuda").float() for _ in range(2)]
        self.cache_t = (*codes, *scales)
        self.q = torch.randn((sum(self.new), heads * group, dim), generator=g, device="cuda").mul_(spread).to(TYPES[dtype])
        self.out = torch.full_like(self.q, math.nan)

    def args(self, **other):
        t = self.q.shape[0]
        a = dict(cache=ivb.KvCache(*self.cache_t), q=self.q, out=self.out, offsets=ints([0] + list(np.cumsum(self.new))), lens=ints(self.lens),
                 pages=ints(self.table), groups=ints(list(self.first)), shared=ints(self.common),
                 scratch=torch.full((t * self.heads * self.group * (self.dim + 2),), math.nan, device="cuda"), max_new=max([1] + self.new))
        return {**a, **other}

    def run(self, ops, **other):
        ops.attend_shared(**self.args(**other), stream=stream())
        ops.synchronize(stream())
        return self.out

    def definition(self):
        """Output and error bound of each row, in 64 bits."""
        k, v, ks, vs = (c.cpu() for c in self.cache_t)
        at, outs, bounds, scale = 0, [], [], self.dim ** -0.5
        for b, n in enumerate(self.new):
            rows = torch.from_numpy(self.full[b, :-(-self.lens[b] // self.page)]).long()
            K, V = ((c[rows].double() * s[rows].double().repeat_interleave(BLOCK, 2)[..., None]).transpose(0, 1).reshape(self.heads, -1, self.dim)
                    [:, :self.lens[b]] for c, s in ((k, ks), (v, vs)))
            Q = self.q[at:at + n].double().cpu().transpose(0, 1).reshape(self.heads, self.group, n, self.dim)
            seen = torch.arange(self.lens[b]) <= torch.arange(self.lens[b] - n, self.lens[b])[:, None]
            s = torch.einsum("hgnd,hkd->hgnk", Q, K) * scale
            big = torch.einsum("hgnd,hkd->hgnk", Q.abs(), K.abs()) * scale
            w = torch.softmax(s.masked_fill(~seen, -math.inf), -1)
            o, mass = torch.einsum("hgnk,hkd->hgnd", w, V), torch.einsum("hgnk,hkd->hgnd", w, V.abs())
            # As for one pass over the keys: a score is dim products summed in 32 bits (its error counts twice, in the
            # numerator and in the sum), weights are rounded to 11 bits.  The step kernel's scores come from codes + 128
            # (times |q|: at most |K| + 128 scales), below 2^-21 of that; joining the parts rounds three times more in 32 bits,
            # and the difference of their references, a score's size, once.
            off = (big * (self.dim + 4) * 2.0 ** -24 + s.abs() * 2.0 ** -20).masked_fill(~seen, 0).amax(-1, keepdim=True)
            bounds.append((mass * (2 * off + 2.0 ** -11 + 2.0 ** -16)).permute(2, 0, 1, 3).reshape(n, self.heads * self.group, self.dim))
            outs.append(o.permute(2, 0, 1, 3).reshape(n, self.heads * self.group, self.dim))
            at += n
        return torch.cat(outs), torch.cat(bounds)

    def check(self, ops, **other):
        got = self.run(ops, **other).double().cpu()
        want, bound = self.definition()
        assert torch.isfinite(got).all()
        bound = bound * 1.01 + HALF_ULP[self.dtype] * want.abs() + TINY[self.dtype]
        assert ((got - want).abs() <= bound).all(), float(((got - want).abs() / bound).max())


FORMS = [
    [(1, [(0, 1)])],                                                     # one sequence, nothing of its own but the new token
    [(3, [(5, 1), (0, 1), (17, 1)])],
    [(0, [(40, 1), (3, 1)]), (2, [(9, 1)])],                             # a group without a common beginning
    [(7, [(0, 1)] * 40), (1, [(100, 1)] * 3), (30, [(33, 1), (1, 1)])],   # many rows, few, between
    [(12, [(20, 3), (0, 6), (5, 1)]), (5, [(1, 2)])],                     # drafted tokens
    [(9, [(0, 70), (31, 200), (2, 1)]), (4, [(0, 33)] * 3)],              # questions
    [(2, [(3, 1), (0, 0), (8, 2)]), (4, [(0, 0)])],                       # sequences and a group without new tokens
    [(150, [(10 * i, 1) for i in range(24)])],                           # long: items are cut over many CTAs
    [(5, [(7, 1)] * 4)] * 30,
    [(1, [(0, 300)]), (40, [(0, 150), (64, 90)])],
]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("form", range(len(FORMS)))
@pytest.mark.parametrize("heads,group,page", [(2, 4, 16), (1, 7, 48), (3, 1, 64), (1, 17, 32)])
def test_forms(ops, dtype, dim, form, heads, group, page):
    Case(FORMS[form], heads, group, dim, page, dtype, seed=form).check(ops)


@pytest.mark.parametrize("groups", [[(300, [(50, 1)] * 32)], [(600, [(0, 1), (900, 1)])], [(128, [(30, 100)] * 5)]])
def test_long(ops, groups):
    Case(groups, 2, 8, 128, 64, "bf16", seed=5).check(ops)


@pytest.mark.parametrize("form", [1, 4, 5, 7])
def test_scales_far_apart(ops, form):
    """Values of a common beginning far larger or smaller than the sequences' own."""
    for low, high in ((-30, 20), (20, -30)):
        c = Case(FORMS[form], 2, 4, 64, 16, "bf16", seed=form)
        for n, p in enumerate(c.common):
            pages = c.full[c.first[n], :p // c.page]
            c.cache_t[3][torch.from_numpy(pages).long()] *= 2.0 ** low
            for b in range(c.first[n], c.first[n + 1]):
                own = c.full[b, p // c.page:]
                c.cache_t[3][torch.from_numpy(own[own >= 0]).long()] *= 2.0 ** high
        c.check(ops)


@pytest.mark.parametrize("form", [3, 5])
@pytest.mark.parametrize("layout", ["sliced", "odd_offset"])
def test_layouts(ops, form, layout):
    c = Case(FORMS[form], 2, 4, 64, 16, "f16", seed=1)
    t, h, d = c.q.shape
    if layout == "sliced":
        q, out = torch.zeros((t, 3 * h, d), dtype=c.q.dtype, device="cuda")[:, h:2 * h], torch.zeros((h, t, d), dtype=c.q.dtype, device="cuda").transpose(0, 1)
    else:
        q, out = (torch.zeros(t * h * d + 1, dtype=c.q.dtype, device="cuda")[1:].view(t, h, d) for _ in range(2))
    q.copy_(c.q)
    c.q, c.out = q, out
    c.check(ops)


def test_shared_or_not(ops):
    """`attend` on the same pages says the same, but for the rounding of weights."""
    c = Case([(20, [(30, 1), (0, 2), (9, 5)])], 2, 4, 128, 32, "f16", seed=2)
    got = c.run(ops).double()
    plain = torch.empty_like(c.q)
    a = c.args()
    ops.attend(a["cache"], c.q, plain, a["offsets"], a["lens"], ints(c.full), max_new=a["max_new"], stream=stream())
    _, bound = c.definition()
    assert ((got - plain.double()).abs().cpu() <= 2 * bound + 2 * HALF_ULP["f16"] * plain.double().abs().cpu() + TINY["f16"]).all()


@pytest.mark.parametrize("form", [3, 5, 7])
def test_same_bits_again_and_in_a_graph(ops, form):
    c = Case(FORMS[form], 2, 4, 128, 16, "f16", seed=form)
    want = c.run(ops).clone()
    for _ in range(4):
        c.out.fill_(math.nan)
        assert torch.equal(c.run(ops), want)
    a, side = c.args(), torch.cuda.Stream()
    ops.reserve(side.cuda_stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        ops.attend_shared(**a, stream=side.cuda_stream)
    for times in (1.0, 0.5):
        c.q.mul_(times)
        c.out.fill_(math.nan)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        again = c.out.clone()
        assert torch.equal(c.run(ops), again)
    ops.release(side.cuda_stream)


def test_streams_at_once(ops):
    cases = [Case(FORMS[f], 2, 4, 64, 16, "f16", seed=f) for f in (3, 5, 7)]
    wants = [c.run(ops).clone() for c in cases]
    args, streams = [c.args() for c in cases], [torch.cuda.Stream() for _ in cases]
    outs = [[torch.empty_like(c.q) for _ in range(20)] for c in cases]
    torch.cuda.synchronize()
    for i in range(20):
        for a, st, o in zip(args, streams, outs):
            ops.attend_shared(**{**a, "out": o[i]}, stream=st.cuda_stream)
    torch.cuda.synchronize()
    for want, o in zip(wants, outs):
        assert all(torch.equal(x, want) for x in o)
    for st in streams:
        ops.release(st.cuda_stream)


@pytest.mark.parametrize("form", [1, 5])
def test_not_finite_query_stays_in_its_row(ops, form):
    c = Case(FORMS[form], 2, 4, 64, 16, "f16", seed=3)
    clean = c.run(ops).clone()
    c.q[1, 3, 7], c.q[-1, 0, 0] = math.nan, math.inf
    got = c.run(ops)
    same = torch.ones(c.q.shape[:2], dtype=torch.bool)
    same[1, 3] = same[-1, 0] = False
    assert torch.equal(got.cpu()[same], clean.cpu()[same]) and got[1, 3].isnan().all()


def test_a_row_does_not_depend_on_its_neighbours(ops):
    """The bits of one sequence stay when the others of its group have other queries."""
    for form in (3, 5):
        c = Case(FORMS[form], 2, 4, 64, 16, "f16", seed=4)
        want = c.run(ops)[:1].clone()
        c.q[1:] = c.q[1:].flip(0) * 3
        assert torch.equal(c.run(ops)[:1], want)


@pytest.mark.parametrize("what", ["length", "offsets", "common", "part_of_a_page", "negative", "first", "not_covered", "page", "max_new"])
@pytest.mark.parametrize("form", [3, 5])
def test_device_side_errors_are_reported(ops, what, form):
    """What does not fit is skipped and reported; the other groups are as they would be alone."""
    c = Case(FORMS[form], 2, 4, 64, 16, "f16", seed=6)
    want = c.run(ops).clone()
    a = c.args()
    cut = int(np.cumsum([0] + c.new)[c.first[1]])  # packed tokens of group 0
    if what == "length":
        a["lens"][0] = c.common[0] + c.new[0] - 1  # ends inside the beginning
    elif what == "offsets":
        a["offsets"][1] = 1 << 20
    elif what == "common":
        a["shared"][0] = 1 << 20
    elif what == "part_of_a_page":
        a["shared"][0] -= 1
    elif what == "negative":
        a["shared"][0] = -16
    elif what == "first":
        a["groups"][0] = -1
    elif what == "not_covered":
        a["groups"][0], a["pages"] = 1, ints(c.full)  # (the second sequence is the group's first one then, and names its pages)
    elif what == "page":
        a["pages"][0, 0] = 1 << 20
    else:
        a["max_new"] = max(c.new) - 1
    c.out.fill_(5.0)
    if a["max_new"] == 0:  # (the host sees this one)
        with pytest.raises(ivb.NativeError):
            ops.attend_shared(**a, stream=stream())
        return
    ops.attend_shared(**a, stream=stream())
    with pytest.raises(ivb.NativeError):
        ops.synchronize(stream())
    ops.synchronize(stream())  # reported once
    if what == "max_new":
        return
    # (where items are cut over CTAs goes by all of a call's keys, so that what is skipped may move a rounding of the others)
    exact, bound = c.definition()
    near = ((c.out.double().cpu() - exact).abs() <= bound * 1.01 + HALF_ULP["f16"] * exact.abs() + TINY["f16"]).all((1, 2))
    assert near[cut:].all()
    if what in ("common", "part_of_a_page", "negative", "first"):
        assert (c.out[:cut] == 5.0).all()
    if what in ("length", "not_covered"):
        assert (c.out[:c.new[0]] == 5.0).all() and near[c.new[0]:].all()
    # the handle works on
    c.out.fill_(math.nan)
    assert torch.equal(c.run(ops), want)


def test_offsets_past_32_bits(ops):
    """Common pages and own pages that lie beyond 2^31 codes."""
    page, heads, dim, pages = 128, 8, 128, 17000
    codes = [torch.zeros((pages, heads, page, dim), dtype=torch.int8, device="cuda") for _ in range(2)]
    scales = [torch.zeros((pages, heads, page // BLOCK), device="cuda") for _ in range(2)]
    c = Case([(3, [(7, 1), (90, 2)])], heads, 2, dim, page, "f16", seed=8)
    far = np.arange(pages - 12, pages)[:c.cache_t[0].shape[0]]
    for big, small in zip((*codes, *scales), c.cache_t):
        big[torch.from_numpy(far).long()] = small
    want = c.run(ops).clone()
    moved = np.where(c.table >= 0, far[c.table], -1)
    got = c.run(ops, cache=ivb.KvCache(*codes, *scales), pages=ints(moved))
    assert torch.equal(got, want)


def test_refusals(ops):
    c = Case(FORMS[1], 2, 4, 64, 16)
    a = c.args()
    for name, bad in (("scratch", a["scratch"][:-1]), ("scratch", a["scratch"][1:]), ("groups", ints([0, 3, 3, 3, 3, 3]))):
        with pytest.raises((ivb.NativeError, ValueError)):
            ops.attend_shared(**{**a, name: bad}, stream=stream())
    with pytest.raises(ivb.NativeError):  # more groups than sequences
        ops.attend_shared(**{**a, "groups": ints([0, 1, 2, 3, 3]), "shared": ints([16, 16, 16, 16])}, stream=stream())
    for name, bad in (("groups", a["groups"].long()), ("shared", a["shared"].cpu()), ("scratch", a["scratch"].half()), ("q", c.q.float()),
                      ("out", c.out[:1]), ("lens", a["lens"][:2]), ("shared", ints([16, 16]))):
        with pytest.raises(ValueError):
            ops.attend_shared(**{**a, name: bad}, stream=stream())
    with pytest.raises(ivb.NativeError):
        ops.attend_shared(**{**a, "max_new": 0}, stream=stream())
    empty = c.q[:0]
    ops.attend_shared(**{**a, "q": empty, "out": empty, "offsets": ints([0, 0, 0, 0])}, stream=stream())


def widened(c):
    """The same pages in a table with so many columns that the beginning is worth a pass of its own."""
    columns = (48 << 20) // (c.batch * c.page * c.heads * 2 * c.dim) + 2
    return ints(np.pad(c.table, ((0, 0), (0, max(0, columns - c.table.shape[1]))), constant_values=-1))


@pytest.mark.parametrize("dtype,dim,heads,group,page", [("f16", 128, 2, 4, 16), ("bf16", 64, 3, 1, 32), ("f16", 64, 1, 17, 48), ("bf16", 128, 1, 7, 16)])
@pytest.mark.parametrize("form", range(len(FORMS)))
def test_two_passes(ops, form, dtype, dim, heads, group, page):
    c = Case(FORMS[form], heads, group, dim, page, dtype, seed=form)
    c.check(ops, pages=widened(c))


@pytest.mark.parametrize("groups", [[(5, [(7, 1)] * 4)] * 40, [(20, [(3 * i, 1 + i % 3) for i in range(130)])], [(6, [(0, 1)] * 200), (8, [(700, 1)])],
                                    [(3, [(5, 1)] * 129), (40, [(900, 2)] * 3)]])
def test_many_sequences_in_two_passes(ops, groups):
    c = Case(groups, 2, 4, 128, 16, "bf16", seed=len(groups))
    c.check(ops, pages=widened(c))


@pytest.mark.parametrize("groups", [[(40, [(3 * i, 1) for i in range(12)])], [(30, [(20, 2)] * 40), (9, [(1, 1)] * 5)], [(25, [(10, 70)] * 3)]])
@pytest.mark.parametrize("captured", [False, True])
def test_calls_that_follow_at_once(ops, groups, captured):
    """Queries, lengths, tables, codes and scales that change right before each call, and outputs read right after it."""
    c = Case(groups, 2, 4, 128, 64, "f16", seed=7)
    wide, steps = widened(c), 10
    a = c.args(pages=wide.clone())
    g = torch.Generator(device="cuda").manual_seed(3)
    q = [torch.randn(c.q.shape, generator=g, device="cuda").half() for _ in range(steps)]
    new = [[t[torch.randperm(t.shape[0], generator=g, device="cuda")] for t in c.cache_t] for _ in range(steps)]
    tables = [wide.roll(0) if i % 2 else torch.where(wide >= 0, wide.max() - wide, wide) for i in range(steps)]
    lens0, lens = ints(c.lens), a["lens"]

    def run(st, wait):
        outs = []
        lens.copy_(lens0)
        for i in range(steps):
            c.q.copy_(q[i])
            for t, u in zip(c.cache_t, new[i]):
                t.copy_(u)
            a["pages"].copy_(tables[i])
            lens.add_(1)
            if wait:
                torch.cuda.synchronize()
            ops.attend_shared(**a, stream=st)
            if wait:
                torch.cuda.synchronize()
            outs.append(c.out.clone())
            c.out.fill_(math.nan)
        return torch.stack(outs)

    want = run(stream(), True)
    assert torch.isfinite(want).all()
    if captured:
        side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        ops.reserve(side.cuda_stream)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=side):
            got = run(side.cuda_stream, False)
        for _ in range(20):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, want)
        ops.release(side.cuda_stream)
    else:
        for _ in range(20):
            assert torch.equal(run(stream(), False), want)
    ops.synchronize(stream())


def test_scratch_in_others_memory_is_refused(ops):
    """Scratch that shares a byte with queries, outputs or the cache is refused; scratch between rows is not."""
    c = Case(FORMS[1], 2, 4, 64, 16)
    a = c.args()
    t, h, d = c.q.shape
    need = a["scratch"].shape[0]
    both = torch.zeros(need + t * h * d, device="cuda")  # scratch, then rows
    rows = both.view(torch.float16)[2 * need:2 * need + t * h * d].view(t, h, d)
    near = both.view(torch.float16)[2 * need - 8:2 * need - 8 + t * h * d].view(t, h, d)
    for name in ("q", "out"):
        with pytest.raises(ivb.NativeError):
            ops.attend_shared(**{**a, "scratch": both[:need], name: near}, stream=stream())
        with pytest.raises(ivb.NativeError):
            ops.attend_shared(**{**a, "scratch": both[:need], name: near.view(h, t, d).transpose(0, 1)}, stream=stream())
    codes = torch.zeros(4 * need + c.cache_t[0].numel(), dtype=torch.int8, device="cuda")
    k = codes[4 * need - 16:][:c.cache_t[0].numel()].view(c.cache_t[0].shape)
    scale = torch.zeros(need + c.cache_t[2].numel(), device="cuda")
    for at, t_ in ((0, k), (1, k), (2, scale[need - 4:][:c.cache_t[2].numel()].view(c.cache_t[2].shape)), (3, scale[need - 4:][:c.cache_t[2].numel()].view(c.cache_t[2].shape))):
        cache = list(c.cache_t)
        cache[at] = t_
        with pytest.raises(ivb.NativeError):
            ops.attend_shared(**{**a, "cache": ivb.KvCache(*cache), "scratch": codes[:4 * need].view(torch.float32) if at < 2 else scale[:need]}, stream=stream())
    rows.copy_(c.q)
    c.q = rows
    between = torch.zeros((t, need + h * d // 2), device="cuda")  # a token's rows, and room for all before the next one's
    c.q = between.view(torch.float16)[:, :h * d].view(t, h, d).copy_(rows)
    c.check(ops, scratch=between[1, h * d // 2:])


def wide(c, table):
    """`table` with the columns of `widened`."""
    columns = widened(c).shape[1]
    return ints(np.pad(table, ((0, 0), (0, columns - table.shape[1])), constant_values=-1))


# Beginnings of few rows and of many, items that are cut and whole; a sequence's own keys always for the kernel of few rows.
TWO = {n: FORMS[n] for n in (1, 3, 4, 6, 7, 8)}
TWO["long"] = [(60, [(10 * i, 1) for i in range(24)]), (40, [(5 * i, 1) for i in range(24)])]  # (the parts of cut items are added up by a launch of their own)


@pytest.mark.parametrize("form", list(TWO))
@pytest.mark.parametrize("dtype,dim,group", [("bf16", 64, 4), ("f16", 128, 4), ("bf16", 128, 17)])
@pytest.mark.parametrize("low,high", [(-30, 20), (20, -30)])
def test_scales_far_apart_in_two_passes(ops, form, dtype, dim, group, low, high):
    c = Case(TWO[form], 2, group, dim, 16, dtype, seed=7)
    for n, p in enumerate(c.common):
        c.cache_t[3][torch.from_numpy(c.full[c.first[n], :p // c.page]).long()] *= 2.0 ** low
        for b in range(c.first[n], c.first[n + 1]):
            own = c.full[b, p // c.page:]
            c.cache_t[3][torch.from_numpy(own[own >= 0]).long()] *= 2.0 ** high
    if dtype == "f16":  # (what is in the type's range)
        c.cache_t[3].mul_(2.0 ** -20)
    c.check(ops, pages=widened(c))


@pytest.mark.parametrize("form", list(TWO))
def test_zero_value_scales_in_two_passes(ops, form):
    """A beginning, or a sequence's own keys, whose values are 0."""
    for common in (True, False):
        c = Case(TWO[form], 2, 4, 64, 16, "bf16", seed=7)
        for n, p in enumerate(c.common):
            for b in range(c.first[n], c.first[n + 1]):
                some = c.full[b, :p // c.page] if common else c.full[b, p // c.page:]
                c.cache_t[3][torch.from_numpy(some[some >= 0]).long()] = 0
        c.check(ops, pages=widened(c))


@pytest.mark.parametrize("form", [3, 4, 7, "long"])
@pytest.mark.parametrize("layout", ["sliced", "odd_offset", "heads_first"])
def test_layouts_in_two_passes(ops, form, layout):
    c = Case(TWO[form], 2, 4, 64, 16, "f16", seed=1)
    t, h, d = c.q.shape
    if layout == "sliced":
        q, out = (torch.zeros((t, 3 * h, d), dtype=c.q.dtype, device="cuda")[:, h:2 * h] for _ in range(2))
    elif layout == "odd_offset":
        q, out = (torch.zeros(t * h * d + 1, dtype=c.q.dtype, device="cuda")[1:].view(t, h, d) for _ in range(2))
    else:
        q, out = (torch.zeros((h, t, d), dtype=c.q.dtype, device="cuda").transpose(0, 1) for _ in range(2))
    q.copy_(c.q)
    c.q, c.out = q, out
    c.check(ops, pages=widened(c))


@pytest.mark.parametrize("form", [1, 3, 4, 7, "long"])
def test_not_finite_query_stays_in_its_row_in_two_passes(ops, form):
    c = Case(TWO[form], 2, 4, 64, 16, "f16", seed=3)
    clean = c.run(ops, pages=widened(c)).clone()
    c.q[1, 3, 7], c.q[-1, 0, 0] = math.nan, math.inf
    got = c.run(ops, pages=widened(c))
    same = torch.ones(c.q.shape[:2], dtype=torch.bool)
    same[1, 3] = same[-1, 0] = False
    assert torch.equal(got.cpu()[same], clean.cpu()[same]) and got[1, 3].isnan().all()


@pytest.mark.parametrize("form", [3, 4, 7, "long"])
def test_a_row_does_not_depend_on_its_neighbours_in_two_passes(ops, form):
    c = Case(TWO[form], 2, 4, 64, 16, "f16", seed=4)
    want = c.run(ops, pages=widened(c))[:1].clone()
    c.q[1:] = c.q[1:].flip(0) * 3
    assert torch.equal(c.run(ops, pages=widened(c))[:1], want)


@pytest.mark.parametrize("what", ["length", "offsets", "common", "part_of_a_page", "negative", "first", "last", "not_covered", "page", "own_page", "max_new", "all"])
@pytest.mark.parametrize("form", [3, 4, 8, "long"])
def test_device_side_errors_are_reported_in_two_passes(ops, what, form):
    """What does not fit is skipped and reported; the other groups are as they would be alone, and so is the next call."""
    c = Case(TWO[form], 2, 4, 64, 16, "f16", seed=6)
    table = widened(c)
    want = c.run(ops, pages=table).clone()
    a = c.args(pages=table.clone())
    tokens = np.cumsum([0] + c.new)
    skipped, wrong = np.zeros(tokens[-1], bool), np.zeros(tokens[-1], bool)  # rows that stay as they were; rows of which nothing is said
    group0 = slice(0, tokens[c.first[1]])
    if what == "length":
        a["lens"][0] = c.common[0] + c.new[0] - 1
        skipped[:c.new[0]] = True
    elif what == "offsets":
        a["offsets"][1] = 1 << 20
        wrong[group0] = True
    elif what in ("common", "part_of_a_page", "negative"):
        a["shared"][0] = {"common": 1 << 20, "part_of_a_page": c.common[0] - 1, "negative": -16}[what]
        skipped[group0] = True
    elif what == "first":
        a["groups"][0] = -1
        skipped[group0] = True
    elif what == "last":  # the last sequence is in no group
        a["groups"][-1] -= 1
        skipped[tokens[-2]:] = True
    elif what == "not_covered":
        a["groups"][0], a["pages"] = 1, wide(c, c.full)
        skipped[:c.new[0]] = True
    elif what == "page":
        a["pages"][0, 0] = 1 << 20
        wrong[group0] = True
    elif what == "own_page":
        a["pages"][0, c.common[0] // c.page] = 1 << 20
        wrong[:c.new[0]] = True
    elif what == "max_new":
        a["max_new"] = max(c.new) - 1
        for b, n in enumerate(c.new):
            skipped[tokens[b]:tokens[b + 1]] = n == max(c.new)
    else:  # no group fits: the second pass has nothing to do
        a["shared"].fill_(-16)
        skipped[:] = True
    c.out.fill_(5.0)
    if a["max_new"] == 0:
        with pytest.raises(ivb.NativeError):
            ops.attend_shared(**a, stream=stream())
        return
    ops.attend_shared(**a, stream=stream())
    with pytest.raises(ivb.NativeError):
        ops.synchronize(stream())
    ops.synchronize(stream())
    exact, bound = c.definition()
    near = ((c.out.double().cpu() - exact).abs() <= bound * 1.01 + HALF_ULP["f16"] * exact.abs() + TINY["f16"]).all((1, 2)).numpy()
    assert near[~skipped & ~wrong].all() and (c.out.cpu().numpy()[skipped] == 5.0).all()
    # calls one behind the other, an erroneous one between
    outs = []
    for args in (c.args(pages=table), a, c.args(pages=table)):
        c.out.fill_(math.nan)
        ops.attend_shared(**args, stream=stream())
        outs.append(c.out.clone())
    with pytest.raises(ivb.NativeError):
        ops.synchronize(stream())
    assert torch.equal(outs[0], want) and torch.equal(outs[2], want)


@pytest.mark.parametrize("groups", [[(3, [(7, 1), (90, 2)])], [(6, [(5 + i, 1) for i in range(9)])], [(3, [(70, 90), (3, 20)])]])
def test_offsets_past_32_bits_in_two_passes(ops, groups):
    """Common and own pages beyond 2^31 codes: a beginning for the kernel of few rows, of many, and both passes for that one."""
    page, heads, dim, pages = 128, 8, 128, 17000
    codes = [torch.zeros((pages, heads, page, dim), dtype=torch.int8, device="cuda") for _ in range(2)]
    scales = [torch.zeros((pages, heads, page // BLOCK), device="cuda") for _ in range(2)]
    c = Case(groups, heads, 8, dim, page, "f16", seed=8)
    many = c.cache_t[0].shape[0]
    far = np.arange(pages - many, pages)
    for big, small in zip((*codes, *scales), c.cache_t):
        big[torch.from_numpy(far).long()] = small
    want = c.run(ops, pages=wide(c, c.table)).clone()
    got = c.run(ops, cache=ivb.KvCache(*codes, *scales), pages=wide(c, np.where(c.table >= 0, far[c.table], -1)))
    assert torch.equal(got, want)


@pytest.mark.parametrize("form", [3, 4, 7, "long"])
def test_same_bits_again_and_in_a_graph_in_two_passes(ops, form):
    c = Case(TWO[form], 2, 4, 128, 16, "f16", seed=7)
    table = widened(c)
    want = c.run(ops, pages=table).clone()
    for _ in range(4):
        c.out.fill_(math.nan)
        assert torch.equal(c.run(ops, pages=table), want)
    a, side = c.args(pages=table), torch.cuda.Stream()
    ops.reserve(side.cuda_stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        ops.attend_shared(**a, stream=side.cuda_stream)
    for times in (1.0, 0.5):
        c.q.mul_(times)
        c.out.fill_(math.nan)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        again = c.out.clone()
        assert torch.equal(c.run(ops, pages=table), again)
    ops.release(side.cuda_stream)


def test_streams_at_once_in_two_passes(ops):
    cases = [Case(TWO[f], 2, 4, 64, 16, "f16", seed=7) for f in (3, 4, 7, 8, "long")]
    args = [c.args(pages=widened(c)) for c in cases]
    wants = [c.run(ops, pages=widened(c)).clone() for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    outs = [[torch.empty_like(c.q) for _ in range(20)] for c in cases]
    torch.cuda.synchronize()
    for i in range(20):
        for a, st, o in zip(args, streams, outs):
            ops.attend_shared(**{**a, "out": o[i]}, stream=st.cuda_stream)
    torch.cuda.synchronize()
    for want, o in zip(wants, outs):
        assert all(torch.equal(x, want) for x in o)
    for st in streams:
        ops.release(st.cuda_stream)
