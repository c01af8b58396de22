"""Attention: a row's bits go by its own query and keys, not by its neighbours'."""
import numpy as np
import pytest
import torch

import infvino_b200 as ivb
from test_gpu_kv import HALF_ULP, TINY, TYPES, attention64, filled_cache, ints, offsets_of, page_table, stream

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("new,lens,heads,group,dim,window,sinks", [
    ([1, 1], [3000, 700], 2, 8, 64, 0, 0), ([6, 3], [900, 1200], 2, 4, 128, 0, 0), ([5, 1], [900, 400], 1, 6, 64, 200, 7),
    ([60, 100, 30], [130, 170, 100], 2, 4, 64, 0, 0), ([300], [2000], 2, 2, 128, 0, 0), ([200], [900], 1, 4, 128, 150, 20)])
def test_rows_do_not_depend_on_their_neighbours(dtype, new, lens, heads, group, dim, window, sinks):
    table, pages = page_table(lens, 32)
    t, args = sum(new), (offsets_of(new), ints(lens), ints(table))
    kw = dict(max_new=max(new), window=window, sinks=sinks)
    with ivb.KvOps(0) as ops:
        for seed in range(12):
            g = torch.Generator(device="cuda").manual_seed(seed)
            cache = ivb.KvCache(*filled_cache(pages, heads, 32, dim, seed))
            q = torch.randn((t, heads * group, dim), generator=g, device="cuda").to(TYPES[dtype])
            other = torch.rand((t, heads * group), generator=g, device="cuda") < 0.5
            changed = torch.where(other[..., None], torch.randn(q.shape, generator=g, device="cuda").mul_(3).to(q.dtype), q)
            changed[other.nonzero()[0][0], other.nonzero()[0][1], 5] = float("inf")
            out, got = torch.empty_like(q), torch.empty_like(q)
            ops.attend(cache, q, out, *args, stream=stream(), **kw)
            ops.attend(cache, changed, got, *args, stream=stream(), **kw)
            ops.synchronize(stream())
            assert torch.equal(got[~other], out[~other]), seed


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("ratio", [12, 18, 22])
def test_small_query_elements_beside_a_large_one(dim, ratio):
    """A bf16 query's largest element meets keys that are 0 there: the others, 2^-ratio of it, decide."""
    new, lens, heads, group = [200, 90], [400, 90], 2, 2
    table, pages = page_table(lens, 32)
    k, v, ks, vs = filled_cache(pages, heads, 32, dim, ratio)
    k[..., 3] = 0
    ks = torch.full_like(ks, 2.0 ** (ratio - 8))
    g = torch.Generator(device="cuda").manual_seed(dim + ratio)
    q = torch.randn((sum(new), heads * group, dim), generator=g, device="cuda") * 2.0 ** -ratio
    q[..., 3] = torch.where(torch.rand(q.shape[:2], generator=g, device="cuda") < 0.5, -1.5, 1.9)
    q = q.to(torch.bfloat16)
    out = torch.empty_like(q)
    with ivb.KvOps(0) as ops:
        ops.attend(ivb.KvCache(k, v, ks, vs), q, out, offsets_of(new), ints(lens), ints(table), max_new=max(new), stream=stream())
        ops.synchronize(stream())
    want, bound = attention64((k, v, ks, vs), table, q, new, lens, dim ** -0.5, 0, 0)
    bound = bound * 1.01 + HALF_ULP["bf16"] * want.abs() + TINY["bf16"]
    assert ((out.double().cpu() - want).abs() <= bound).all()
