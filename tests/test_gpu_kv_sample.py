"""KvOps.sample against the definition in 64 bits."""
import math

import numpy as np
import pytest
import torch

import infvino_b200 as ivb

pytestmark = pytest.mark.gpu
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
INF, NAN = math.inf, math.nan


@pytest.fixture(scope="module")
def ops():
    with ivb.KvOps(0) as o:
        yield o


def stream():
    return torch.cuda.current_stream().cuda_stream


def choose(x, u, t=1.0, k=0, p=1.0, least=0.0):
    """The token of one row of float64 logits, its probability, and how near u is to a border of it."""
    x = np.where(np.isnan(x), -INF, x) + 0.0
    top = x.max()
    if top == -INF:
        return -1, 0.0, 1.0
    best = int(np.argmax(x))
    if not t > 0:
        return best, 1.0, 1.0
    with np.errstate(all="ignore"):
        w = np.where(x == top, 1.0, np.where(x == -INF, 0.0, np.exp((x - top) / t)))
    w = np.nan_to_num(w, nan=0.0)
    w[w <= 2.0 ** -60] = 0
    order = np.lexsort((np.arange(len(x)), -x))
    if k > 0:
        order = order[:k]
    if p < 1:
        c = np.cumsum(w[order])
        order = order[:int(np.argmax(c >= max(p, 0.0) * c[-1])) + 1]
    if least > 0:
        order = order[(w[order] >= least) | (x[order] == top)]
    keep = np.zeros(len(x), bool)
    keep[order] = True
    w = w * keep
    c = np.cumsum(w)
    u = min(max(u, 0.0), 1 - 2.0 ** -24) if u == u else 0.0
    i = int(np.argmax(c > u * c[-1]))
    return i, w[i] / c[-1], min(c[i] - u * c[-1], u * c[-1] - (c[i] - w[i])) / c[-1]


def check(ops, x, u, temperature=None, top_k=None, top_p=None, min_p=None, probs=True):
    rows = x.shape[0]
    dev = {n: None if v is None else torch.tensor(v, dtype=torch.int32 if n == "k" else torch.float32, device="cuda")
           for n, v in (("u", u), ("t", temperature), ("k", top_k), ("p", top_p), ("m", min_p))}
    tokens = torch.full((rows,), -7, dtype=torch.int32, device="cuda")
    pr = torch.full((rows,), NAN, device="cuda") if probs else None
    ops.sample(x, dev["u"], tokens, pr, temperature=dev["t"], top_k=dev["k"], top_p=dev["p"], min_p=dev["m"], stream=stream())
    ops.synchronize(stream())
    host, got, f = x.double().cpu().numpy(), tokens.tolist(), {n: None if v is None else v.tolist() for n, v in dev.items()}
    for r in range(rows):
        want, share, margin = choose(host[r], f["u"][r], *(d if f[n] is None else f[n][r] for n, d in (("t", 1.0), ("k", 0), ("p", 1.0), ("m", 0.0))))
        # (sums of 500000 weights in 64 bits are good to some 2^-33 whatever their order: nearer to a border than that nothing is asked)
        assert got[r] == want or abs(margin) < 2.0 ** -33, (r, got[r], want, margin)
        if probs and got[r] == want:
            assert abs(float(pr[r]) - share) <= 2.0 ** -23 * share, (r, float(pr[r]), share)  # one rounding to f32, and 64-bit sums
    return got


def logits(rows, vocab, dtype, seed=0, spread=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((rows, vocab), generator=g, device="cuda").mul_(spread)
    some = torch.randint(vocab, (rows, 12), generator=g, device="cuda")
    return x.scatter_add_(1, some, torch.rand((rows, 12), generator=g, device="cuda") * 9).to(TYPES[dtype])


def uniform(rows, seed):
    return np.random.default_rng(seed).random(rows, dtype=np.float32)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (1, 2), (3, 31), (2, 33), (5, 1000), (1, 32003), (300, 777), (40, 50021), (2, 262144), (1, 500000)])
@pytest.mark.parametrize("filters", ["none", "temperature", "top_k", "top_p", "min_p", "all"])
def test_sample(ops, dtype, rows, vocab, filters):
    r = np.random.default_rng(rows + vocab)
    f = {}
    if filters in ("temperature", "all"):
        f["temperature"] = r.choice([0.0, 0.3, 0.7, 1.0, 1.9], rows)
    if filters in ("top_k", "all"):
        f["top_k"] = r.choice([-1, 0, 1, 2, 17, 50, 1000, 1025, 3000, 1 << 30], rows)
    if filters in ("top_p", "all"):
        f["top_p"] = r.choice([0.0, 0.1, 0.5, 0.9, 0.99, 1.0], rows)
    if filters in ("min_p", "all"):
        f["min_p"] = r.choice([0.0, 0.001, 0.05, 1.0], rows)
    check(ops, logits(rows, vocab, dtype, vocab), uniform(rows, vocab), **f)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("vocab", [40, 5000, 70000])
def test_ties(ops, dtype, vocab):
    """Few distinct logits: cuts lie inside runs of equal ones, which go by their numbers."""
    rows = 24
    g = torch.Generator(device="cuda").manual_seed(vocab)
    x = torch.randint(-2, 3, (rows, vocab), generator=g, device="cuda").to(TYPES[dtype])
    x[3] = 1.5
    x[4] = -0.0
    x[4, ::2] = 0.0
    r = np.random.default_rng(1)
    u = uniform(rows, 5)
    check(ops, x, u)
    check(ops, x, u, top_k=r.integers(1, vocab, rows))
    check(ops, x, u, top_p=r.random(rows))
    check(ops, x, u, temperature=r.random(rows) + 0.5, top_k=r.integers(1, vocab, rows), top_p=r.random(rows), min_p=r.random(rows) * 0.5)
    check(ops, x, u, temperature=[0.0] * rows)


@pytest.mark.parametrize("vocab", [3000, 60000])
def test_logits_that_one_bin_holds(ops, vocab):
    """An outlier, or values on scales that differ by many powers of two, leave most logits in one bin, again and again."""
    rows = 8
    g = torch.Generator(device="cuda").manual_seed(vocab)
    x = torch.randn((rows, vocab), generator=g, device="cuda")
    x[0] *= 1e-4
    x[0, 77] = 30.0
    x[1] = torch.exp2(-40.0 * torch.rand(vocab, generator=g, device="cuda"))
    x[2] = -torch.exp2(-60.0 * torch.rand(vocab, generator=g, device="cuda"))
    x[3] = 5.0 + 1e-6 * x[3]
    x[4] *= 1e30
    x[5] *= 1e-38
    x[6, 5:] = x[6, 5]
    t = [1000.0, 1.0, 0.5, 1e-6, 1e30, 1e-38, 1.0, INF]
    u = uniform(rows, 9)
    for k, p in ((None, None), (2000, None), (None, 0.6), (2500, 0.7), (5, 0.9)):
        check(ops, x, u, temperature=t, top_k=None if k is None else [k] * rows, top_p=None if p is None else [p] * rows)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
def test_masked_and_not_finite(ops, dtype):
    vocab = 5003
    x = logits(9, vocab, dtype, 3)
    x[0] = -INF                       # nothing is allowed
    x[1] = -INF
    x[1, 4999] = -3.0                 # one token is
    x[2, ::2] = -INF
    x[3] = torch.finfo(x.dtype).min   # a mask of the type's lowest value
    x[3, 100:110] = 1.0
    x[4, 17] = NAN
    x[4, 5:9] = NAN
    x[5] = NAN
    x[6, [30, 4000]] = INF
    x[7] = INF
    x[8] = torch.finfo(x.dtype).min
    u = uniform(9, 1)
    got = check(ops, x, u)
    assert got[0] == -1 and got[1] == 4999 and got[5] == -1 and got[6] in (30, 4000)
    check(ops, x, u, top_k=[20] * 9, top_p=[0.8] * 9, min_p=[0.01] * 9)
    check(ops, x, u, top_k=[3000] * 9, top_p=[0.99] * 9)
    check(ops, x, u, temperature=[0.0] * 9)
    check(ops, x, u, temperature=[INF] * 9)
    check(ops, x, u, temperature=[NAN] * 9, top_p=[NAN] * 9, min_p=[NAN] * 9)
    check(ops, x, u, top_p=[NAN] * 9, min_p=[NAN] * 9, top_k=[-5] * 9)


def test_borders_of_u(ops):
    x = torch.zeros((7, 1000), device="cuda")
    got = check(ops, x, [0.0, 1 - 2.0 ** -24, 0.5, 0.25, -3.0, 7.0, NAN])
    assert got == [0, 999, 500, 250, 0, 999, 0]  # equal weights: the first with more than u of them
    assert check(ops, x, [0.999, 0.0, 0.5, 0.1, 0.1, 0.1, 0.1], top_k=[10, 1, 2, 3, 4, 5, 6]) == [9, 0, 1, 0, 0, 0, 0]


def test_layouts_and_outputs(ops):
    """Rows of a wider buffer, odd strides and addresses; nothing else is written; probabilities may be left out."""
    base = logits(6, 4001, "f16", 11)
    u = uniform(6, 2)
    wide = torch.zeros((6, 5003), dtype=torch.float16, device="cuda")
    for at in (0, 1, 8):
        wide[:, at:at + 4001] = base
        check(ops, wide[:, at:at + 4001], u, top_p=[0.9] * 6, probs=at != 1)
    flipped = torch.empty_like(base)
    flipped[:] = base.flip(0)
    one = base[2:3].expand(6, -1)  # (the same row six times)
    check(ops, one, u)
    tokens = torch.full((10,), -7, dtype=torch.int32, device="cuda")
    ops.sample(base, torch.tensor(u, device="cuda"), tokens[2:8], stream=stream())
    assert tokens[:2].tolist() == [-7, -7] and tokens[8:].tolist() == [-7, -7] and (tokens[2:8] >= 0).all()
    ops.sample(base[:0], torch.empty(0, device="cuda"), tokens[:0], stream=stream())  # no rows


def test_a_row_does_not_depend_on_how_many_there_are(ops):
    x, u = logits(400, 20011, "bf16", 8), torch.tensor(uniform(400, 8), device="cuda")
    many, one = torch.empty(400, dtype=torch.int32, device="cuda"), torch.empty(400, dtype=torch.int32, device="cuda")
    p = torch.full((400,), 0.95, device="cuda")
    ops.sample(x, u, many, top_p=p, stream=stream())
    for r in range(0, 400, 13):
        ops.sample(x[r:r + 1], u[r:r + 1], one[r:r + 1], top_p=p[r:r + 1], stream=stream())
    assert torch.equal(many[::13], one[::13])


def test_same_bits_again(ops):
    x, u = logits(64, 131072, "f32", 5), torch.tensor(uniform(64, 5), device="cuda")
    k = torch.full((64,), 2000, dtype=torch.int32, device="cuda")
    p = torch.full((64,), 0.97, device="cuda")
    seen = []
    for _ in range(4):
        t, q = torch.empty(64, dtype=torch.int32, device="cuda"), torch.empty(64, device="cuda")
        ops.sample(x, u, t, q, top_k=k, top_p=p, stream=stream())
        seen.append((t, q))
    assert all(torch.equal(a, seen[0][0]) and torch.equal(b, seen[0][1]) for a, b in seen)


def test_graph_and_streams(ops):
    """Captured once (no call before it is needed) and replayed with other logits and numbers, beside calls on another stream."""
    x, u, t = logits(3, 9001, "f16", 1), torch.tensor(uniform(3, 1), device="cuda"), torch.empty(3, dtype=torch.int32, device="cuda")
    temp = torch.full((3,), 0.8, device="cuda")
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        ops.sample(x, u, t, temperature=temp, top_p=temp, stream=side.cuda_stream)
    for seed in range(3):
        x.copy_(logits(3, 9001, "f16", seed + 10))
        u.copy_(torch.tensor(uniform(3, seed + 10)))
        other = torch.empty(3, dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()
        graph.replay()
        ops.sample(x, u, other, temperature=temp, top_p=temp, stream=side.cuda_stream)
        torch.cuda.synchronize()
        assert torch.equal(t, other)
        want = [choose(x[r].double().cpu().numpy(), float(u[r]), float(temp[r]), 0, float(temp[r]))[0] for r in range(3)]
        assert t.tolist() == want


def test_how_often(ops):
    """Tokens come as often as their probabilities say."""
    rows = 20000
    x = torch.tensor([0.0, 1.0, -1.0, 2.0, -INF, 0.5], device="cuda").expand(rows, -1)
    u = torch.rand(rows, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    t = torch.empty(rows, dtype=torch.int32, device="cuda")
    ops.sample(x, u, t, stream=stream())
    p = torch.softmax(x[0].double(), 0).cpu()
    got = torch.bincount(t.long(), minlength=6).double().cpu() / rows
    assert got[4] == 0 and ((got - p).abs() <= 5 * (p * (1 - p) / rows).sqrt()).all()  # five standard deviations


def test_refusals(ops):
    x, u, t = logits(4, 100, "f16"), torch.rand(4, device="cuda"), torch.empty(4, dtype=torch.int32, device="cuda")
    for bad in (dict(logits=x.double()), dict(logits=x[0]), dict(logits=x.cpu()), dict(logits=x.t()[:4]), dict(u=u[:3]), dict(u=u.double()),
                dict(u=u.cpu()), dict(tokens=t.long()), dict(tokens=t[:3]), dict(probs=u[:2]), dict(top_k=u), dict(top_p=t), dict(min_p=u[::2]),
                dict(temperature=u.half()), dict(logits=torch.empty((4, 0), device="cuda"))):
        args = {"logits": x, "u": u, "tokens": t, **bad}
        with pytest.raises((ValueError, ivb.NativeError)):
            ops.sample(stream=stream(), **args)
    with pytest.raises(ivb.NativeError):
        ops.sample(torch.empty((1, 500001), dtype=torch.float16, device="cuda"), u[:1], t[:1], stream=stream())


@pytest.mark.parametrize("rows", [2, 120, 150])
def test_extreme_temperatures(ops, rows):
    """Logits and temperatures whose difference or quotient does not fit into 32 bits."""
    g = torch.Generator(device="cuda").manual_seed(rows)
    u, low = uniform(rows, 11), torch.finfo(torch.float32).min
    x = torch.rand((rows, 3001), generator=g, device="cuda")
    for y, t in (((x * 6 - 3) * 1e38, 1e38), ((x * 6 - 3) * 1e38, 3e38), (x * 2e-37, 1e-38), (x * -4e-44, 1e-44), (x * 1e-30, 1e-40), (x - 2.0 ** 28, 1e-40),
                 (torch.where(x > 0.5, low, -low), 3e38), (torch.where(x > 0.5, low, -low), INF)):
        for k, p in ((None, None), (40, None), (None, 0.6)):
            check(ops, y, u, temperature=[t] * rows, top_k=None if k is None else [k] * rows, top_p=None if p is None else [p] * rows)
    z = (x * 1.2e5 - 6e4).to(torch.float16)
    check(ops, z, u, temperature=[3e4] * rows, top_p=[0.7] * rows)
    check(ops, ((x * 6 - 3) * 1e38).to(torch.bfloat16), u, temperature=[1e38] * rows, top_p=[0.7] * rows)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
def test_masked_and_not_finite_in_many_rows(ops, dtype):
    vocab, times = 5003, 17
    x = logits(9, vocab, dtype, 3)
    x[0] = -INF
    x[1] = -INF
    x[1, 4999] = -3.0
    x[2, ::2] = -INF
    x[3] = torch.finfo(x.dtype).min
    x[3, 100:110] = 1.0
    x[4, 17] = NAN
    x[4, 5:9] = -NAN
    x[5] = NAN
    x[6, [30, 4000]] = INF
    x[7] = INF
    x[8] = torch.finfo(x.dtype).min
    x, rows = x.repeat(times, 1), 9 * times
    u = uniform(rows, 1)
    got = check(ops, x, u)
    assert got[::9] == [-1] * times and got[1::9] == [4999] * times and got[5::9] == [-1] * times
    check(ops, x, u, top_k=[20] * rows, top_p=[0.8] * rows, min_p=[0.01] * rows)
    check(ops, x, u, top_k=[3000] * rows, top_p=[0.99] * rows)
    check(ops, x, u, temperature=[0.0, INF, NAN] * (rows // 3), top_p=[NAN] * rows, min_p=[NAN] * rows)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("vocab", [40, 70000])
def test_ties_in_many_rows(ops, dtype, vocab):
    """Few distinct logits, some more than 65535 times in a row."""
    times = 25
    g = torch.Generator(device="cuda").manual_seed(vocab)
    x = torch.randint(-2, 3, (6, vocab), generator=g, device="cuda").to(TYPES[dtype])
    x[1] = 1.5
    x[2] = -0.0
    x[2, ::2] = 0.0
    x[3, 1:] = NAN
    x[4, 2:] = -0.0
    x, rows = x.repeat(times, 1), 6 * times
    r, u = np.random.default_rng(1), uniform(rows, 5)
    check(ops, x, u)
    check(ops, x, u, top_k=r.integers(1, vocab, rows))
    check(ops, x, u, temperature=r.random(rows) + 0.5, top_k=r.integers(1, vocab, rows), top_p=r.random(rows), min_p=r.random(rows) * 0.5)
    check(ops, x, u, top_p=r.random(rows))


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("spread", [0.05, 2.0, 5.0])
def test_cuts_far_down(ops, dtype, spread):
    """Cuts behind thousands of tokens, whose bins are guessed."""
    x, u = logits(10, 150001, dtype, 21, spread), uniform(10, 21)
    p = [0.3, 0.6, 0.9, 0.97, 0.99, 0.999, 0.9999, 0.99999, 1 - 2.0 ** -23, 0.5]
    check(ops, x, u, top_p=p)
    check(ops, x, u, top_p=p, temperature=[1.3] * 10, top_k=[100000, 800, 900, 1024, 1025, 5000, 0, 0, 0, 0])


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
def test_rows_of_clusters_that_follow_at_once(ops, dtype):
    """Rows of eight CTAs, small ones: launches of several streams, one behind the other, whose CTAs begin while others end."""
    shapes = [(18, 16500), (3, 33000), (1, 20011), (30, 17001)]
    x = [logits(*s, dtype, i) for i, s in enumerate(shapes)]
    u = [torch.tensor(uniform(r, i), device="cuda") for i, (r, _) in enumerate(shapes)]
    p = [torch.full((r,), 0.9, device="cuda") for r, _ in shapes]
    side = [torch.cuda.Stream() for _ in range(3)]
    out = [[torch.full((100, r), -7, dtype=torch.int32, device="cuda") for r, _ in shapes] for _ in side]
    torch.cuda.synchronize()
    for n in range(100):
        for st, o in zip(side, out):
            for i in range(len(shapes)):
                ops.sample(x[i], u[i], o[i][n], top_p=p[i], stream=st.cuda_stream)
    torch.cuda.synchronize()
    for i, (rows, _) in enumerate(shapes):
        want = torch.tensor(check(ops, x[i], u[i].cpu().numpy(), top_p=[0.9] * rows), dtype=torch.int32, device="cuda")
        assert all((o[i] == want).all() for o in out)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("rows", [3, 153])
def test_infinite_logits_under_min_p(ops, dtype, rows):
    """Where logits are +inf only these have a weight, whatever min_p and the cut are."""
    x, u, every = logits(rows, 5003, dtype, 4), uniform(rows, 4), np.arange(rows)
    x[::3, [30, 4000]] = INF
    x[1::3, 2500:] = INF
    x[2::9, 1] = INF
    x[5::9] = -INF
    x[5::9, 4999] = INF
    for f in (dict(), dict(top_k=[3000] * rows), dict(top_k=[1] * rows), dict(top_p=[0.99] * rows), dict(temperature=[0.5] * rows), dict(temperature=[INF] * rows),
              dict(top_k=[3000] * rows, top_p=[0.9] * rows)):
        for least in (0.01, 1.0):
            got = np.array(check(ops, x, u, min_p=[least] * rows, **f))
            assert np.isin(got[every % 3 == 0], [30, 4000]).all() and (got[every % 3 == 1] >= 2500).all()
            assert (got[2::9] == 1).all() and (got[5::9] == 4999).all()


@pytest.mark.parametrize("rows", [30, 150])
def test_cuts_at_the_end_of_a_long_run(ops, rows):
    """top_p ends within the last token of 60000 equal ones, some e^-20 of the largest each, with others behind them."""
    n, tail = 60000, 10000
    r = np.random.default_rng(7)
    near = np.float32(r.uniform(-20.3, -19.9, rows))
    w, p, u = np.exp(near.astype(np.float64)), 1 - 2.0 ** -20, [1 - 2.0 ** -24] * rows
    # p (1 + n w + tail) is what comes before the run's end but for a part of its last token
    part = np.linspace(0.05, 0.95, rows)
    far = np.float32(np.log(((1 + (n - part) * w) / p - 1 - n * w) / tail))
    x = np.full((rows, 1 + n + tail), 0, np.float32)
    x[:, 1:] = far[:, None]
    places = 1 + r.permutation(n + tail)[:n]
    x[:, places] = near[:, None]
    x[:, places[0]], x[:, 0] = 0, near  # (the largest is somewhere)
    got = check(ops, torch.tensor(x, device="cuda"), u, top_p=[p] * rows)
    assert (x[np.arange(rows), got] >= near).all()  # (what is behind the run is not kept)


@pytest.mark.parametrize("rows", [3, 150])
def test_cuts_in_long_runs_of_small_weights(ops, rows):
    """top_p ends inside 400000 equal tokens of some e^-25 each: the cut goes by sums in 64 bits."""
    n, tail = 400000, 90000
    near = np.float32(-25 + np.random.default_rng(3).uniform(-0.05, 0.05, rows))
    w, v = np.exp(near.astype(np.float64)), np.exp(np.float64(np.float32(-25.3)))
    x = torch.full((rows, 1 + n + tail), -25.3, device="cuda")
    x[:, 0] = 0
    x[:, 1:1 + n] = torch.tensor(near, device="cuda")[:, None]
    p, u = 1 - 2.0 ** -18, 1 - 2.0 ** -24
    all_ = 1 + n * w + tail * v
    kept = np.ceil((p * all_ - 1) / w)      # of the run
    assert ((kept > 1000) & (kept < n - 1000)).all()
    want = np.floor((u * (1 + kept * w) - 1) / w) + 1
    got = torch.full((rows,), -7, dtype=torch.int32, device="cuda")
    ops.sample(x, torch.full((rows,), u, device="cuda"), got, top_p=torch.full((rows,), p, device="cuda"), stream=stream())
    # three sums (all, up to the cut, up to the token), each off by at most n 2^-53 whatever its order, weights by 2^-52 of
    # themselves, and one token more or less for each border
    off = (3 * x.shape[1] * 2.0 ** -53) / w + 2 * n * 2.0 ** -52 + 2
    assert (np.abs(got.cpu().numpy() - want) <= off).all(), np.abs(got.cpu().numpy() - want).max()


def test_cuts_in_long_runs_of_near_weights(ops):
    """The same where eight values share the run, in rows enough that values are counted."""
    n, tail, distinct, times, p, u = 400000, 90000, 8, 19, 1 - 2.0 ** -19, 1 - 2.0 ** -20
    near = np.float32(-25 + np.random.default_rng(5).uniform(-0.01, 0.01, distinct))
    x = np.full((distinct, 1 + n + tail), -26.2, np.float32)
    x[:, 0] = 0
    x[:, 1:1 + n] = near[:, None] - np.float32(0.125) * (np.arange(n, dtype=np.float32) % 8)
    want = [choose(x[r].astype(np.float64), u, p=p)[0] for r in range(distinct)]
    rows = distinct * times
    got = torch.full((rows,), -7, dtype=torch.int32, device="cuda")
    ops.sample(torch.tensor(x, device="cuda").repeat(times, 1), torch.full((rows,), u, device="cuda"), got, top_p=torch.full((rows,), p, device="cuda"),
               stream=stream())
    # as above, on both sides; an eighth of the run at least is kept, so that so many tokens are at most eight times as far in numbers
    off = 8 * (2 * (3 * x.shape[1] * 2.0 ** -53) / math.exp(-25.9) + 2 * n * 2.0 ** -52 + 2)
    assert (np.abs(got.view(times, distinct).cpu().numpy() - np.array(want)) <= off).all(), (got[:distinct], want)


@pytest.mark.parametrize("seed", [10, 14, 25])
def test_a_cut_between_sums_in_two_orders(ops, seed):
    """Rows whose top_p lies, in steps of half a unit in the last place, around the weight of the same 60 tokens: sums up to
    there that are added in another order are above it or below."""
    r = np.random.default_rng(seed)
    head = np.sort(np.float16(r.uniform(3, 8, 60)))[::-1].astype(np.float64)
    top, rows = head[0], 4096
    left, tail = np.exp(head - top).sum() * (1 - 2.0 ** -42), []  # what comes behind weighs as much (p is a half)
    for y in np.arange(2.9, -22, -0.1).astype(np.float16).astype(np.float64):
        w = np.exp(y - top)
        tail += [y] * int(left / w)
        left -= int(left / w) * w
    fine = np.float64(np.float16(top - 49 * math.log(2)))
    one = np.concatenate([head, tail, np.full(rows, -INF)])
    x = np.repeat(one[None].astype(np.float16), rows, 0)
    for i in range(rows):
        x[i, len(one) - rows:len(one) - rows + i] = fine
    order = r.permutation(len(one))
    x = np.ascontiguousarray(x[:, order])
    tokens, probs = torch.full((rows,), -7, dtype=torch.int32, device="cuda"), torch.full((rows,), NAN, device="cuda")
    u = torch.full((rows,), 0.5, device="cuda")
    ops.sample(torch.tensor(x, device="cuda"), u, tokens, probs, top_p=u, stream=stream())
    # (one token more or less is kept by a rounding)
    may = [choose(x[0].astype(np.float64), 0.5, p=p)[:2] for p in (0.5 - 1e-9, 0.5 + 1e-9)]
    for got in zip(tokens.tolist(), probs.tolist()):
        assert any(got[0] == t and abs(got[1] - s) <= 2.0 ** -23 * s for t, s in may), (got, may)


@pytest.mark.parametrize("rows", [100, 1000])
def test_weights_have_the_bits_of_64(ops, rows):
    """Rows whose largest logit weighs half of all but for 2^-48 to 2^-45: u = 0.5 is at its border."""
    r, y = np.random.default_rng(2), np.float32(-0.37 * np.arange(3, 96))
    small = np.exp(y.astype(np.longdouble))
    x, first = np.full((rows, 2 + len(y)), -INF, np.float32), np.zeros(rows, bool)
    for i in range(rows):
        x[i, 0], x[i, 1] = 0, r.uniform(-0.6, -0.1)
        total = 1 + np.exp(x[i, 1].astype(np.longdouble))
        want = 2 + r.choice([-1, 1]) * r.uniform(2.0 ** -47, 2.0 ** -45)
        for j in range(len(y)):
            if total + small[j] < want:
                total, x[i, 2 + j] = total + small[j], y[j]
        # (64-bit weights and sums of them: some ten roundings of 2^-53 each)
        assert 2.0 ** -48 < abs(total - 2) < 2.0 ** -44.9
        first[i] = total < 2
    got = torch.full((rows,), -7, dtype=torch.int32, device="cuda")
    ops.sample(torch.tensor(x, device="cuda"), torch.full((rows,), 0.5, device="cuda"), got, stream=stream())
    assert (got.cpu().numpy() == np.where(first, 0, 1)).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("rows", [4, 152])
def test_min_p_above_every_weight(ops, dtype, rows):
    """The first token in order alone, of several equal ones too."""
    x = logits(rows, 3001, dtype, 6)
    x[::2, [2000, 2001, 17, 900]] = 30.0
    x[1::4] = 1.0
    x[3::8, [5, 6]] = INF
    x[7::16] = -INF
    x[7::16, 3000] = 0
    want = [int(np.argmax(v)) for v in x.double().cpu().numpy()]
    for f in (dict(), dict(top_k=[50] * rows), dict(top_p=[0.9] * rows), dict(temperature=[1.7] * rows)):
        tokens, probs = torch.full((rows,), -7, dtype=torch.int32, device="cuda"), torch.full((rows,), NAN, device="cuda")
        more = {n: torch.tensor(v, device="cuda", dtype=torch.int32 if n == "top_k" else torch.float32) for n, v in f.items()}
        ops.sample(x, torch.tensor(uniform(rows, 3), device="cuda"), tokens, probs, min_p=torch.tensor([1.5, INF] * (rows // 2), device="cuda"), stream=stream(), **more)
        assert tokens.tolist() == want and (probs == 1).all()
    one = torch.full((rows,), -7, dtype=torch.int32, device="cuda")
    ops.sample(x[:, :1], torch.rand(rows, device="cuda"), one, min_p=torch.full((rows,), 2.0, device="cuda"), stream=stream())
    assert (one == torch.where(x[:, 0] == -INF, -1, 0)).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("rows", [6, 42, 153])
@pytest.mark.parametrize("vocab", [1001, 20252])
def test_top_p_inside_the_run_that_top_k_cuts(ops, dtype, rows, vocab):
    """Equal logits behind a larger one or a few: top_k ends among them, and top_p before that."""
    r = np.random.default_rng(vocab + rows)
    x = np.repeat(r.uniform(-6, 2, (rows, 1)), vocab, 1)
    for i in range(rows):
        x[i, r.integers(0, vocab, 1 + i % 3)] += r.uniform(0.5, 12, 1 + i % 3)
    x, u = torch.tensor(x, device="cuda").to(TYPES[dtype]), uniform(rows, 9)
    for k in ([vocab - 1] * rows, [vocab - 7] * rows, r.integers(5, vocab, rows)):
        for p in ([0.9999] * rows, [0.99] * rows, r.random(rows)):
            check(ops, x, u, top_k=k, top_p=p)
            check(ops, x, np.float32(1) - u * np.float32(1e-4), top_k=k, top_p=p)
