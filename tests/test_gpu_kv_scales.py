"""Attention over caches whose value scales differ much between blocks: a row's
result goes by the keys that it sees, and by those that matter among them."""
import numpy as np
import pytest
import torch

import infvino_b200 as ivb
from test_gpu_kv import BLOCK, HALF_ULP, TINY, TYPES, ints, offsets_of, page_table, stream

pytestmark = pytest.mark.gpu
PAGE = 32


@pytest.fixture(scope="module")
def ops():
    with ivb.KvOps(0) as o:
        yield o


def row_bounds(cache_t, table, q, new, lens, window, sinks):
    """Output and error bound of each row, in 64 bits.

    A weight times its value scale is rounded to 11 bits, or, far below the
    largest of the row's (T), by at most half of 2^-24 where the largest is at
    least 2^8: 2^-33 T."""
    k, v, ks, vs = (c.cpu().double() for c in cache_t)
    heads, dim = k.shape[1], k.shape[3]
    group, at, outs, bounds = q.shape[1] // heads, 0, [], []
    for b, n in enumerate(new):
        pos = np.arange(lens[b])
        page, slot = table[b, pos // PAGE], pos % PAGE
        kc, vc = (c[page, :, slot].transpose(0, 1) for c in (k, v))                     # [heads, keys, dim]
        kx, vx = (s[page, :, slot // BLOCK].transpose(0, 1)[..., None] for s in (ks, vs))  # [heads, keys, 1]
        K, V = kc * kx, vc * vx
        Q = q[at:at + n].double().cpu().transpose(0, 1).reshape(heads, group, n, dim)
        p, j = torch.arange(lens[b] - n, lens[b])[:, None], torch.arange(lens[b])
        seen = j <= p
        if window:
            seen &= (p - j < window) | (j < sinks)
        s = torch.einsum("hgnd,hkd->hgnk", Q, K) * dim ** -0.5
        # (key codes enter the products as code + 128, at most 255)
        big = torch.einsum("hgnd,hkd->hgnk", Q.abs(), (kc.abs() + 128) * kx) * dim ** -0.5
        w = torch.softmax(s.masked_fill(~seen, -torch.inf), -1)
        o, mass = torch.einsum("hgnk,hkd->hgnd", w, V), torch.einsum("hgnk,hkd->hgnd", w, V.abs())
        off = (big * (dim + 4) * 2.0 ** -24 + s.abs() * 2.0 ** -21).masked_fill(~seen, 0).amax(-1, keepdim=True)
        top = (w * vx[:, None, None, :, 0]).amax(-1, keepdim=True)
        small = torch.einsum("nk,hkd->hnd", seen.double(), vc.abs())[:, None] * top * 2.0 ** -33
        bounds.append((mass * (2 * off + 2.0 ** -11 + 2.0 ** -16) + small).permute(2, 0, 1, 3).reshape(n, heads * group, dim))
        outs.append(o.permute(2, 0, 1, 3).reshape(n, heads * group, dim))
        at += n
    return torch.cat(outs), torch.cat(bounds)


def check(ops, dtype, new, lens, dim, exponent, window=0, sinks=0, group=4, against=None, far=0.0):
    """exponent(sequence, block): of the block's value scale.  against: a block whose keys score `far` in every row."""
    heads, dt, t = 2, TYPES[dtype], sum(new)
    table, pages = page_table(lens, PAGE, seed=dim)
    g = torch.Generator(device="cuda").manual_seed(dim + t)
    k, v = (torch.randint(-127, 128, (pages, heads, PAGE, dim), generator=g, device="cuda").to(torch.int8) for _ in range(2))
    ks, vs = torch.full((pages, heads, PAGE // BLOCK), 2.0 ** -7, device="cuda"), torch.ones((pages, heads, PAGE // BLOCK), device="cuda")
    base = torch.randn(dim, generator=g, device="cuda")
    q = (base + 0.05 * torch.randn((t, heads * group, dim), generator=g, device="cuda")).to(dt)
    for b, n in enumerate(lens):
        for blk in range(-(-n // BLOCK)):
            page, part = table[b, blk * BLOCK // PAGE], blk * BLOCK % PAGE // BLOCK
            vs[page, :, part] = 2.0 ** exponent(b, blk)
            if blk == against:
                k[page, :, part * BLOCK:(part + 1) * BLOCK] = (127 * base.sign()).to(torch.int8)
                k[page, :, part * BLOCK:(part + 1) * BLOCK] *= -1 if far < 0 else 1
                ks[page, :, part] = abs(far) / (127 * float(base.abs().sum()) * dim ** -0.5)
    out = torch.full((t, heads * group, dim), float("nan"), dtype=dt, device="cuda")
    ops.attend(ivb.KvCache(k, v, ks, vs), q, out, offsets_of(new), ints(lens), ints(table), max_new=max(new), window=window, sinks=sinks, stream=stream())
    ops.synchronize(stream())
    want, bound = row_bounds((k, v, ks, vs), table, q, new, lens, window, sinks)
    bound = bound * 1.01 + HALF_ULP[dtype] * want.abs() + TINY[dtype]
    got = out.double().cpu()
    assert ((got - want).abs() <= bound).all(), float(((got - want).abs() / bound).max())


SHAPES = [([1, 1], [300, 45]), ([6, 2], [250, 130]), ([300, 90], [300, 200]), ([40], [700])]


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new,lens", SHAPES)
@pytest.mark.parametrize("step", [7, 5, -5, -7])
def test_scales_that_rise_or_fall_along_a_sequence(ops, new, lens, dim, step):
    """Rows of a tile see blocks of small values while others of the tile see blocks of far larger ones too."""
    top = max(-(-n // BLOCK) for n in lens)
    check(ops, "bf16", new, lens, dim, lambda b, blk: max(-70, min(70, step * (blk - top // 2))))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("large", [24, 40])
@pytest.mark.parametrize("new,lens,window,sinks", [
    ([1, 1], [333, 70], 40, 16), ([8, 3], [200, 75], 33, 5), ([300], [300], 40, 16), ([200, 60], [600, 90], 100, 3), ([90], [90], 17, 0)])
def test_a_block_of_large_values_between_sinks_and_window(ops, new, lens, window, sinks, dim, dtype, large):
    """Hidden from most rows, seen by some; before the window of a row in the order of the keys."""
    if dtype == "f16":
        low = -8 if large == 24 else -14  # (results stay normal halves or near)
        large = min(large, 9 - low)
    else:
        low = -20
    for at in (1, 2, 4, 11):
        check(ops, dtype, new, lens, dim, lambda b, blk: low + large if blk == at else low + blk % 3, window, sinks)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new,lens", SHAPES)
@pytest.mark.parametrize("far,large", [(-60.0, 30), (-60.0, 70), (40.0, -40), (60.0, -75)])
def test_a_block_that_does_not_matter(ops, new, lens, dim, far, large):
    """Values 2^30 larger under weights of e^-60; or the largest weights on values so small that they do not count."""
    for at in (0, 3):
        check(ops, "bf16", new, lens, dim, lambda b, blk: large if blk == at else blk % 3, against=at, far=far)


@pytest.mark.parametrize("new,lens", SHAPES)
def test_zero_values_first(ops, new, lens):
    """Sinks and a prompt's begin with values of zero (the least scale), then ordinary ones."""
    for zeros in (1, 8, 9):
        check(ops, "f16", new, lens, 64, lambda b, blk: -120 if blk < zeros else -7)
        check(ops, "bf16", new, lens, 64, lambda b, blk: -120 if blk < zeros else -7, window=40, sinks=16)


@pytest.mark.parametrize("new,lens", SHAPES)
@pytest.mark.parametrize("low,high", [(-120, 25), (-100, -7), (-40, 60)])
def test_far_apart(ops, new, lens, low, high):
    """Whole sequences' values far below or above those of their neighbours, and parts of sequences."""
    for few in (2, 8, 9, 17):
        check(ops, "bf16", new, lens, 128, lambda b, blk: low if blk < few else high)
        check(ops, "bf16", new, lens, 64, lambda b, blk: low if blk < few else high, window=100, sinks=33)
        check(ops, "bf16", new, lens, 64, lambda b, blk: high if blk < few else low, window=48, sinks=0)
