"""The language-model operators where only the device sees that input does not
fit: what is skipped stays as it was, and the rest of the call is right."""
import numpy as np
import pytest
import torch

import infvino_b200 as ivb
from test_gpu_kv import BLOCK, TYPES, Model, ints, new_cache, offsets_of, page_table, some_axes, stream

pytestmark = pytest.mark.gpu
IVC_ERR_KERNEL = 5


@pytest.fixture(scope="module")
def ops():
    with ivb.KvOps(0) as o:
        yield o


def reported(ops):
    with pytest.raises(ivb.NativeError) as e:
        ops.synchronize(stream())
    assert e.value.status == IVC_ERR_KERNEL
    ops.synchronize(stream())


def spoil(pos, tokens, positions, axis):
    """Puts the tokens' positions outside the table, on one axis."""
    for i, t in enumerate(tokens):
        pos[axis, t] = (positions, -1, 2 ** 31 - 1, -2 ** 31)[i % 4]


@pytest.mark.parametrize("tokens,heads,dim,pairs,axes,interleaved", [
    (40, 5, 128, 64, 3, False), (40, 5, 128, 64, 3, True), (33, 3, 80, 24, 4, False), (17, 300, 64, 8, 1, False), (3000, 12, 128, 32, 2, True)])
@pytest.mark.parametrize("off_grid", [False, True])
def test_rope_leaves_whole_rows_out(ops, tokens, heads, dim, pairs, axes, interleaved, off_grid):
    g = torch.Generator(device="cuda").manual_seed(tokens + dim)
    table = torch.empty((500, pairs, 2), device="cuda")
    ops.rope_table([100.0 ** (-i / pairs) for i in range(pairs)], table, stream())
    x = torch.randn(tokens * heads * dim + 8, generator=g, device="cuda").half()[int(off_grid):][:tokens * heads * dim].view(tokens, heads, dim)
    pos = torch.randint(0, 500, (axes, tokens), generator=g, device="cuda", dtype=torch.int32)
    rotary = ivb.Rotary(table, some_axes(pairs, axes), interleaved)
    want = torch.empty_like(x)
    ops.rope(x, want, rotary, pos, stream())
    ops.synchronize(stream())
    for axis in range(axes):
        bad = sorted({0, 3, 4, tokens // 2 + axis, tokens - 1})
        p = pos.clone()
        spoil(p, bad, 500, axis)
        out = torch.full_like(x, 7.0)
        ops.rope(x, out, rotary, p, stream())
        reported(ops)
        w = want.clone()
        w[bad] = 7.0
        assert torch.equal(out, w)
        y = x.clone()
        ops.rope(y, y, rotary, p, stream())  # in place: the row stays
        reported(ops)
        w[bad] = x[bad]
        assert torch.equal(y, w)
    unused = torch.cat([pos, torch.full((4 - axes, tokens), -9, dtype=torch.int32, device="cuda")])  # no pair turns by these
    out = torch.empty_like(x)
    ops.rope(x, out, rotary, unused, stream())
    ops.synchronize(stream())
    assert torch.equal(out, want)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,dim,page,axes,first,new,bad", [
    (2, 64, 16, 1, [5, 0], [30, 1], [0, 7, 29]),           # of a begun block, of whole ones
    (3, 128, 48, 3, [10, 33], [6, 20], [0, 1, 2, 3, 4, 5, 10]),  # all that a begun block gets
    (1, 128, 64, 2, [0, 16], [64, 5], list(range(16, 32)) + [64]),  # a whole new block
    (2, 64, 32, 4, [3] * 9, [1] * 9, [2, 5]),               # single tokens
    (2, 128, 64, 3, [40, 0], [2000, 900], [0, 100, 1999, 2000, 2899])])
def test_append_leaves_whole_tokens_out(ops, dtype, heads, dim, page, axes, first, new, bad):
    batch, dt, positions = len(new), TYPES[dtype], 300
    lens = [f + n for f, n in zip(first, new)]
    table, pages = page_table(lens, page, seed=dim)
    cache_t = new_cache(pages, heads, page, dim)
    cache, dev_table = ivb.KvCache(*cache_t), ints(table)
    rot_table = torch.empty((positions, dim // 2, 2), device="cuda")
    ops.rope_table([100.0 ** (-i / (dim // 2)) for i in range(dim // 2)], rot_table, stream())
    axis = some_axes(dim // 2, axes)
    rotary = ivb.Rotary(rot_table, axis)
    models = [Model(batch, heads, dim, max(lens) + BLOCK) for _ in range(2)]
    g = torch.Generator(device="cuda").manual_seed(page)
    for start, count, holes, grow in (([0] * batch, first, [], 1.0), (first, new, bad, 3.0)):
        t = sum(count)
        if t == 0:
            continue
        k, v, q = (torch.randn((t, h, dim), generator=g, device="cuda").mul_(grow).to(dt) for h in (heads, heads, 2 * heads))
        for i, h in enumerate(holes):  # what is left out would decide the scale
            k[h] *= 50.0
            v[h] *= 50.0
        pos = torch.randint(0, positions, (axes, t), generator=g, device="cuda", dtype=torch.int32)
        turned = torch.empty_like(q)
        ops.rope(q, turned, rotary, pos, stream())
        x = k.float()
        cs = torch.stack([rot_table[pos[a].long(), i] for i, a in enumerate(axis)], 1)[:, None]
        a, b_ = x[..., :dim // 2], x[..., dim // 2:]
        kr = torch.cat([a * cs[..., 0] - b_ * cs[..., 1], b_ * cs[..., 0] + a * cs[..., 1]], -1).cpu().numpy()
        spoil(pos, holes, positions, axes - 1)
        q_out, before = torch.full_like(q, 7.0), [c.clone() for c in cache_t]
        ops.append(cache, k, v, offsets_of(count), ints(start), dev_table, rotary=rotary, pos=pos, q=q, q_out=q_out, stream=stream())
        if holes:
            reported(ops)
            turned[holes] = 7.0
        else:
            ops.synchronize(stream())
        assert torch.equal(q_out, turned)
        kr[holes], vr = np.nan, v.float().cpu().numpy()  # (the model takes NaN out of the scale)
        vr[holes] = np.nan
        at = 0
        for b, n in enumerate(count):
            for model, x in zip(models, (kr, vr)):
                if n:
                    model.append(b, start[b], x[at:at + n])
            at += n
        at = 0
        for b, n in enumerate(count):
            out = np.zeros(start[b] + n, dtype=bool)
            out[[start[b] + h - at for h in holes if at <= h < at + n]] = True
            at += n
            where = np.arange(start[b] + n)
            page_of, slot = table[b, where // page], where % page
            blocks = where // BLOCK
            # a block that gets nothing keeps its scale, whatever that is
            got = np.array([(~out[(blocks == k) & (where >= start[b])]).any() for k in blocks], dtype=bool)
            touched = np.array([((blocks == k) & (where >= start[b])).any() for k in blocks], dtype=bool)
            for model, i in zip(models, (0, 1)):
                c, s = cache_t[i].cpu().numpy()[page_of, :, slot], cache_t[i + 2].cpu().numpy()[page_of, :, slot // BLOCK]
                c0, s0 = before[i].cpu().numpy()[page_of, :, slot], before[i + 2].cpu().numpy()[page_of, :, slot // BLOCK]
                want_s = 2.0 ** model.exp[b, blocks].astype(np.float64)
                same = touched & ~got
                assert np.array_equal(s[same], s0[same], equal_nan=True)
                assert np.array_equal(s[~same], want_s[~same])
                assert np.array_equal(c[~out], model.codes[b, where[~out]])
                assert np.array_equal(c[out], c0[out])


def attention_without(cache_t, table, q, new, lens, window, sinks):
    """Output and error bound of each row in 64 bits; keys in pages outside the cache are hidden (as test_gpu_kv.attention64 has it else)."""
    k, v, ks, vs = (c.cpu() for c in cache_t)
    pages, heads, page, dim = k.shape
    group, scale, at, outs, bounds = q.shape[1] // heads, dim ** -0.5, 0, [], []
    for b, n in enumerate(new):
        at += n
        if not n:
            continue
        have = np.arange(lens[b])
        page_of = table[b, have // page]
        inside = torch.from_numpy((page_of >= 0) & (page_of < pages))
        p_, s_ = np.where(inside, page_of, 0), have % page
        K, V = ((c[p_, :, s_].double() * s[p_, :, s_ // BLOCK].double()[..., None]).transpose(0, 1) for c, s in ((k, ks), (v, vs)))
        Q = q[at - n:at].double().cpu().transpose(0, 1).reshape(heads, group, n, dim)
        p, j = torch.arange(lens[b] - n, lens[b])[:, None], torch.arange(lens[b])
        seen = (j <= p) & inside
        if window:
            seen &= (p - j < window) | (j < sinks)
        s = torch.einsum("hgnd,hkd->hgnk", Q, K) * scale
        big = torch.einsum("hgnd,hkd->hgnk", Q.abs(), K.abs()) * scale
        w = torch.softmax(s.masked_fill(~seen, -torch.inf), -1).nan_to_num(0.0)
        o, mass = torch.einsum("hgnk,hkd->hgnd", w, V), torch.einsum("hgnk,hkd->hgnd", w, V.abs())
        off = (big * (dim + 4) * 2.0 ** -24 + s.abs() * 2.0 ** -21).masked_fill(~seen, 0).amax(-1, keepdim=True)
        bounds.append((mass * (2 * off + 2.0 ** -11 + 2.0 ** -16)).permute(2, 0, 1, 3).reshape(n, heads * group, dim))
        outs.append(o.permute(2, 0, 1, 3).reshape(n, heads * group, dim))
    return torch.cat(outs), torch.cat(bounds)


@pytest.mark.parametrize("tiny", [False, True])  # the least value scale beside the missing blocks
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("window,sinks", [(0, 0), (300, 20)])
@pytest.mark.parametrize("new,lens", [([1, 1, 1], [2000, 60, 700]), ([5, 0, 2], [900, 10, 300]), ([300, 40, 1], [1500, 300, 200]), ([700], [700])])
def test_attend_hides_keys_in_pages_outside_the_cache(ops, dim, window, sinks, new, lens, tiny):
    heads, group, page = 2, 4, 16
    table, pages = page_table(lens, page, seed=3)
    g = torch.Generator(device="cuda").manual_seed(dim)
    cache_t = [torch.randint(-127, 128, (pages, heads, page, dim), generator=g, device="cuda").to(torch.int8) for _ in range(2)]
    cache_t += [2.0 ** torch.randint(-9, -4, (pages, heads, 1), generator=g, device="cuda").float() for _ in range(2)]
    q = torch.randn((sum(new), heads * group, dim), generator=g, device="cuda").mul_(2).half()
    if tiny:
        cache_t[3][table[0, ::2].clip(0)] = 2.0 ** -120
    for bad in ([0], [1, 5, 6], [3, 4, 5, 6, 7, 8, 9, 10, 11, 12, 13, 14]):  # one block, some, a whole tile of 128 keys
        t = table.copy()
        for i, c in enumerate(bad):
            if c < -(-lens[0] // page):
                t[0, c] = (pages, -1, 2 ** 31 - 1, -2 ** 31)[i % 4]
        out = torch.full_like(q, float("nan"))
        ops.attend(ivb.KvCache(*cache_t), q, out, offsets_of(new), ints(lens), ints(t), max_new=max(new), window=window, sinks=sinks, stream=stream())
        want, bound = attention_without(cache_t, t, q, new, lens, window, sinks)
        got = out.double().cpu()
        assert ((got - want).abs() <= bound * 1.01 + 2.0 ** -11 * want.abs() + 2.0 ** -25).all()
        read = any((page_first <= lens[0] - 1) and (not window or page_first < sinks or (c + 1) * page - 1 > lens[0] - new[0] - window)
                   for c in bad for page_first in [c * page])
        if read:
            reported(ops)
        else:
            ops.synchronize(stream())


def test_overlapping_outputs_are_refused(ops):
    t, heads, dim = 6, 4, 64
    x = torch.randn((t, heads, dim), device="cuda").half()
    rotary, pos = ivb.Rotary(torch.zeros((8, 32, 2), device="cuda")), ints(list(range(t)))
    table, pages = page_table([t], 16)
    cache = ivb.KvCache(*[torch.zeros((pages, heads, 16, dim), dtype=torch.int8, device="cuda") for _ in range(2)],
                        *[torch.ones((pages, heads, 1), device="cuda") for _ in range(2)])
    seqs = (offsets_of([t]), ints([0]), ints(table))
    one = torch.zeros((t, heads, dim), dtype=torch.float16, device="cuda")
    for bad in (one[:1].expand(t, heads, dim), one[:, :1].expand(t, heads, dim), one.view(-1).as_strided((t, heads, dim), (heads * 32, 32, 1))):
        for call in (lambda: ops.rope(x, bad, rotary, pos, stream()), lambda: ops.read(cache, bad, None, *seqs, stream()),
                     lambda: ops.read(cache, None, bad, *seqs, stream()),
                     lambda: ops.append(cache, x, x, *seqs, rotary=rotary, pos=pos, q=x, q_out=bad, stream=stream()),
                     lambda: ops.attend(cache, x, bad, seqs[0], ints([t]), seqs[2], max_new=t, stream=stream())):
            with pytest.raises(ivb.NativeError) as e:
                call()
            assert e.value.status == 1 and "overlap" in e.value.message
    ops.rope(x[:1].expand(t, heads, dim), one, rotary, pos, stream())  # inputs may
    ops.attend(cache, x[:, :1].expand(t, heads, dim), one.transpose(0, 1).contiguous().transpose(0, 1), seqs[0], ints([t]), seqs[2], max_new=t, stream=stream())
    ops.rope(x[:1], one.expand(1, t, heads, dim)[0][:1], rotary, pos[:1], stream())
    ops.synchronize(stream())
