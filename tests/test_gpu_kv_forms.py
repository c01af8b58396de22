"""The language-model operators in the forms that test_gpu_kv.py has not: pair
layouts, parts of heads and odd strides of the append, signs of the scale,
hundreds and thousands of sequences."""
import numpy as np
import pytest
import torch

import infvino_b200 as ivb
from test_gpu_kv import TYPES, Model, check_attention, close_rotation, held, ints, new_cache, offsets_of, page_table, some_axes, stream, turned

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    with ivb.KvOps(0) as o:
        yield o


def placed(x, layout):
    """x in memory of another layout: off the 16-byte grid, between other rows, heads first."""
    t, h, d = x.shape
    if layout == "odd_offset":
        y = torch.empty(t * h * d + 1, dtype=x.dtype, device="cuda")[1:].view(t, h, d)
    elif layout == "odd_stride":
        y = torch.empty((t, h, d + 3), dtype=x.dtype, device="cuda")[..., :d]
    elif layout == "sliced":
        y = torch.empty((t, 3 * h, d), dtype=x.dtype, device="cuda")[:, h:2 * h]
    else:
        y = torch.empty((h, t, d), dtype=x.dtype, device="cuda").transpose(0, 1)
    return y.copy_(x)


def rotated_f32(k, table, pos, axis, interleaved):
    """The rotation in f32, rounded operation by operation (what the append quantises)."""
    x, pairs = k.float(), len(axis)
    cs = torch.stack([table[pos[a].long(), i] for i, a in enumerate(axis)], 1)[:, None]
    y = x.clone()
    ai, bi = (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if interleaved else (slice(0, pairs), slice(pairs, 2 * pairs))
    a, b = x[..., ai], x[..., bi]
    y[..., ai], y[..., bi] = a * cs[..., 0] - b * cs[..., 1], b * cs[..., 0] + a * cs[..., 1]
    return y


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("layout", ["sliced", "odd_offset", "odd_stride", "heads_first"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,pairs,first,new", [
    (64, 32, [3, 0], [1, 1]), (64, 8, [20, 5], [40, 17]), (128, 64, [3, 0, 31], [1, 1, 1]), (128, 24, [15, 16], [2, 90]), (128, 64, [7, 0], [900, 500])])
def test_append_and_read_forms(ops, dtype, layout, interleaved, dim, pairs, first, new):
    heads, page, batch, dt = 2, 32, len(new), TYPES[dtype]
    lens = [f + n for f, n in zip(first, new)]
    table, pages = page_table(lens, page, seed=dim)
    cache_t = new_cache(pages, heads, page, dim)
    cache, dev_table = ivb.KvCache(*cache_t), ints(table)
    rot = torch.empty((200, pairs, 2), device="cuda")
    ops.rope_table([100.0 ** (-i / pairs) for i in range(pairs)], rot, stream())
    axis = some_axes(pairs, 2)
    models = [Model(batch, heads, dim, max(lens) + 16) for _ in range(2)]
    g = torch.Generator(device="cuda").manual_seed(dim + pairs)
    for start, count, grow in (([0] * batch, first, 1.0), (first, new, 3.0)):
        t = sum(count)
        k, v, q = (torch.randn((t, h, dim), generator=g, device="cuda").mul_(grow).to(dt) for h in (heads, heads, 3))
        pos = torch.randint(0, 200, (2, t), generator=g, device="cuda", dtype=torch.int32)
        q_out = placed(torch.full_like(q, 7.0), layout)
        ops.append(cache, placed(k, layout), placed(v, layout), offsets_of(count), ints(start), dev_table,
                   rotary=ivb.Rotary(rot, axis, interleaved), pos=pos, q=placed(q, layout), q_out=q_out, stream=stream())
        close_rotation(q_out, turned(q, rot, pos, axis, interleaved), q, dtype)
        assert torch.equal(q_out[..., 2 * pairs:], q[..., 2 * pairs:])
        at = 0
        for b, n in enumerate(count):
            for model, x in zip(models, (rotated_f32(k, rot, pos, axis, interleaved), v.float())):
                if n:
                    model.append(b, start[b], x[at:at + n].cpu().numpy())
            at += n
    for model, (codes, scales) in zip(models, (cache_t[0::2], cache_t[1::2])):
        for b, (c, s) in enumerate(held(codes, scales, table, lens)):
            assert np.array_equal(s, 2.0 ** model.exp[b, np.arange(lens[b]) // 16].astype(np.float64))
            assert np.array_equal(c, model.codes[b, :lens[b]])
    seqs = (offsets_of(new), ints(first), dev_table)
    dense = [torch.empty((sum(new), heads, dim), dtype=dt, device="cuda") for _ in range(2)]
    ops.read(cache, *dense, *seqs, stream())
    other = [placed(torch.full_like(x, 7.0), layout) for x in dense]
    ops.read(cache, *other, *seqs, stream())
    mixed = [torch.empty_like(dense[0]), placed(torch.full_like(dense[1], 7.0), layout)]
    ops.read(cache, *mixed, *seqs, stream())
    ops.synchronize(stream())
    for a, b, c in zip(dense, other, mixed):
        assert torch.equal(a, b) and torch.equal(a, c)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("scale", [-0.11, 0.0, -1e-30, 1e-3])
@pytest.mark.parametrize("new,lens,dim", [([1, 1], [700, 20], 64), ([5, 3], [300, 40], 128), ([200, 1], [500, 30], 64), ([90], [400], 128)])
def test_attend_scales(ops, dtype, scale, new, lens, dim):
    check_attention(ops, dtype, new, lens, 2, 3, dim, 32, window=0, sinks=0, seed=5, scale=scale)
    check_attention(ops, dtype, new, lens, 2, 3, dim, 32, window=50, sinks=3, seed=6, scale=scale)


@pytest.mark.parametrize("batch,new_of,dim", [
    (129, lambda i: 1, 128), (700, lambda i: i % 3, 64), (1300, lambda i: 1, 64),       # the kernel for few rows
    (513, lambda i: 100 if i == 77 else 1, 64), (1100, lambda i: 70 if i % 500 == 3 else i % 2, 128),  # for many
    (8300, lambda i: 90 if i == 8000 else 1, 64)])                                       # many rows, too many sequences for it
def test_attend_many_sequences(ops, batch, new_of, dim):
    new = [new_of(i) for i in range(batch)]
    lens = [n + (i * 7) % 40 for i, n in enumerate(new)]
    check_attention(ops, "f16", new, lens, 1, 2, dim, 16, seed=batch)
    check_attention(ops, "bf16", new, lens, 1, 1, dim, 16, window=9, sinks=2, seed=batch + 1)


@pytest.mark.parametrize("batch,new_of", [(300, lambda i: 1), (900, lambda i: i % 3), (600, lambda i: 400 if i == 300 else 1)])
def test_append_and_read_many_sequences(ops, batch, new_of):
    new = [new_of(i) for i in range(batch)]
    first = [(i * 5) % 23 for i in range(batch)]
    lens, dim, page = [f + n for f, n in zip(first, new)], 64, 16
    table, pages = page_table(lens, page)
    cache_t = new_cache(pages, 1, page, dim)
    cache, dev_table = ivb.KvCache(*cache_t), ints(table)
    model = Model(batch, 1, dim, max(lens) + 16)
    g = torch.Generator(device="cuda").manual_seed(batch)
    for start, count in (([0] * batch, first), (first, new)):
        x = torch.randn((sum(count), 1, dim), generator=g, device="cuda").mul_(1 + 3 * (start is first)).half()
        ops.append(cache, x, x, offsets_of(count), ints(start), dev_table, stream=stream())
        at = 0
        for b, n in enumerate(count):
            if n:
                model.append(b, start[b], x[at:at + n].float().cpu().numpy())
            at += n
    k, v = (torch.empty((sum(lens), 1, dim), dtype=torch.float16, device="cuda") for _ in range(2))
    ops.read(cache, k, v, offsets_of(lens), ints([0] * batch), dev_table, stream())
    ops.synchronize(stream())
    want = np.concatenate([model.codes[b, :n] * 2.0 ** model.exp[b, np.arange(n) // 16].astype(np.float64)[..., None] for b, n in enumerate(lens)])
    assert np.array_equal(k.double().cpu().numpy(), torch.tensor(want).half().double().numpy())
    assert torch.equal(k, v)
