"""Microscaled 4-bit matrices (KvOps.mx4_*) against the format's definition."""
import math

import pytest
import torch

import infvino_b200 as ivb

pytestmark = pytest.mark.gpu
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
HALF_ULP = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f16": 2.0 ** -25, "bf16": 2.0 ** -134}
MAGNITUDES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


@pytest.fixture(scope="module")
def ops():
    with ivb.KvOps(0) as o:
        yield o


def stream():
    return torch.cuda.current_stream().cuda_stream


def empty(rows, width, fill=0xAA):
    return (torch.full((rows, width // 2), fill, dtype=torch.uint8, device="cuda"),
            torch.full(ivb.Mx4.scales_shape(rows, width), fill, dtype=torch.uint8, device="cuda"))


def quantized(x):
    """Codes [rows, width] and scale bytes [rows, width / 32] of the definition, in 64 bits on the host."""
    x = x.double().cpu()
    x = torch.where(x.isnan(), 0.0, x).unflatten(1, (-1, 32))
    a = x.abs()
    most = torch.where(a.isinf(), 0.0, a).amax(-1)
    e = torch.where(most > 0, torch.frexp(most)[1] - 1 - 2, -127).clamp(min=-127)
    y = torch.ldexp(a, -e[..., None].to(torch.int32))
    m = torch.tensor(MAGNITUDES, dtype=torch.float64)
    # the nearest magnitude; of two as near the one with an even last bit (an even index)
    far = (y[..., None].clamp(max=6.0) - m).abs()
    code = (far * 16 + torch.arange(8) % 2 * 1e-9).argmin(-1)
    code = torch.where(a.isinf(), 7, code)
    return (code + 8 * torch.signbit(x).long()).flatten(1), e + 127


def spread(e):
    """Scale bytes [rows, blocks] in their places."""
    rows, blocks = e.shape
    s = torch.zeros(ivb.Mx4.scales_shape(rows, 32 * blocks), dtype=torch.uint8)
    r, b = torch.arange(rows)[:, None], torch.arange(blocks)[None]
    s[r // 128, b // 4, r % 32, r % 128 // 32, b % 4] = e.to(torch.uint8)
    return s


def values(codes, e):
    m = torch.tensor(MAGNITUDES + [-v for v in MAGNITUDES], dtype=torch.float64)
    return (m[codes].unflatten(1, (-1, 32)) * torch.exp2(e.double() - 127)[..., None]).flatten(1)


def packed(codes):
    return (codes[:, 0::2] | codes[:, 1::2] << 4).to(torch.uint8)


def inputs(rows, width, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((rows, width), generator=g, device="cuda") * torch.exp(torch.randn(width, generator=g, device="cuda") * 2)
    return x.to(TYPES[dtype])


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("rows,width", [(1, 32), (1, 4096), (3, 96), (127, 160), (128, 128), (129, 288), (300, 1056), (2, 28672)])
def test_quantize_and_read(ops, dtype, rows, width):
    x = inputs(rows, width, dtype, rows)
    x[0, :32] = 0
    x[rows // 2, -32:] = 2.0  # (a power of two is the largest)
    # every border between two magnitudes, and its neighbours
    b = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0], device="cuda")
    eps = torch.finfo(x.dtype).eps
    x[-1, :32] = torch.cat([b, b * (1 + eps), -b * (1 - eps), -b]).to(x.dtype)
    c, s = empty(rows, width)
    m = ivb.Mx4(c, s)
    ops.mx4_quantize(x, m, stream=stream())
    out = torch.full_like(x, math.nan)
    ops.mx4_read(m, out, stream=stream())
    codes, e = quantized(x)
    assert torch.equal(c.cpu(), packed(codes))
    assert torch.equal(s.cpu(), spread(e))  # (with zeros where there is no row or block)
    assert torch.equal(out.cpu().double(), values(codes, e).to(x.dtype).double())


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_quantize_extremes(ops, dtype):
    f = torch.finfo(TYPES[dtype])
    tiny = 2.0 ** -24 if dtype == "f16" else 2.0 ** -133
    x = torch.zeros((6, 64), dtype=TYPES[dtype], device="cuda")
    x[0, :4] = torch.tensor([f.max, -f.max, f.max / 2, f.tiny], device="cuda")
    x[1, :4] = torch.tensor([tiny, -tiny, 2 * tiny, 3 * tiny], device="cuda")
    x[2, :3] = torch.tensor([math.nan, math.inf, -math.inf], device="cuda")
    x[2, 3] = 1.0
    x[3, :32] = math.nan
    x[4, :32] = math.inf
    x[5] = f.tiny
    c, s = empty(6, 64)
    ops.mx4_quantize(x, ivb.Mx4(c, s), stream=stream())
    codes, e = quantized(x)
    assert torch.equal(c.cpu(), packed(codes)) and torch.equal(s.cpu(), spread(e))


@pytest.mark.parametrize("layout", ["sliced", "odd_address", "odd_stride", "more_rows"])
def test_quantize_layouts(ops, layout):
    rows, width = 40, 352
    base = inputs(rows, width, "bf16", 4)
    extra = 100 if layout == "more_rows" else 0
    c, s = empty(rows + extra, width)
    m = ivb.Mx4(c, s)
    if layout == "sliced":
        wide = torch.zeros((rows, 3 * width), dtype=base.dtype, device="cuda")
        x, out = wide[:, width:2 * width], torch.zeros_like(wide)[:, width:2 * width]
    elif layout == "odd_address":
        x, out = (torch.zeros(rows * width + 1, dtype=base.dtype, device="cuda")[1:].view(rows, width) for _ in range(2))
    elif layout == "odd_stride":
        x, out = (torch.zeros((rows, width + 3), dtype=base.dtype, device="cuda")[:, :width] for _ in range(2))
    else:
        x, out = torch.empty_like(base), torch.empty_like(base)
    x.copy_(base)
    ops.mx4_quantize(x, m, stream=stream())
    ops.mx4_read(m, out, stream=stream())
    codes, e = quantized(base)
    assert torch.equal(c[:rows].cpu(), packed(codes)) and (c[rows:] == 0xAA).all()
    assert torch.equal(out.cpu().double(), values(codes, e).to(x.dtype).double())


def linear64(x, w):
    """X W^T of the quantised matrices, and the sum of the products' magnitudes."""
    vx, vw = (values(*quantized(t)) for t in (x, w))
    return vx @ vw.t(), vx.abs() @ vw.abs().t()


def close(got, want, mass, width, dtype):
    # products of two codes and their scales are exact; width / 64 sums in 32 bits, each with at most one unit (2^-23) of the largest of what it holds, and the rounding to the type
    bound = HALF_ULP[dtype] * want.abs() + TINY[dtype] + mass * 2.0 ** -23 * (width / 32 + 4)
    got, most = got.double().cpu(), torch.finfo(TYPES[dtype]).max
    over = want.abs() - bound > most * (1 + HALF_ULP[dtype])  # what is above the type's range rounds to an infinity
    assert (got[over] == torch.sign(want[over]) * math.inf).all()
    near = over | ((want.abs() + bound > most) & got.isinf())  # (a value at the range's end may)
    off = torch.where(near, 0.0, (got - want).abs())
    assert (off <= bound).all(), float((off / bound).max())


def weights(ops, rows, width, seed):
    w = inputs(rows, width, "bf16", seed) * (width ** -0.5)
    m = ivb.Mx4(*empty(rows, width))
    ops.mx4_quantize(w, m, stream=stream())
    return w, m


SHAPES = [(1, 32, 1), (1, 64, 128), (1, 4096, 300), (2, 96, 129), (3, 2048, 1000), (8, 160, 7), (15, 1024, 640), (16, 512, 128), (17, 4128, 257),
          (33, 256, 2050), (64, 8192, 130), (65, 320, 384), (129, 1024, 1111), (192, 544, 256), (193, 128, 999), (300, 2080, 520), (1000, 768, 384),
          (4, 28672, 260), (700, 32, 200)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("rows,width,outputs", SHAPES)
def test_linear(ops, dtype, rows, width, outputs):
    x = inputs(rows, width, dtype, width)
    w, m = weights(ops, outputs, width, 3)
    out = torch.full((rows, outputs), math.nan, dtype=TYPES[dtype], device="cuda")
    ops.mx4_linear(x, m, out, scratch=ivb.Mx4(*empty(rows, width)), stream=stream())
    ops.synchronize(stream())
    want, mass = linear64(x, w)
    close(out, want, mass, width, dtype)


@pytest.mark.parametrize("rows,width,outputs", [(1, 8192, 20500), (16, 4096, 19000), (20, 14336, 4100), (1, 14336, 4096), (50, 8192, 20500), (128, 8192, 8300)])
def test_linear_long_shares(ops, rows, width, outputs):
    """Every CTA has many stages, of several tiles: rings go round, quantised on the way or before."""
    x = inputs(rows, width, "f16", 7)
    w = (torch.randn((outputs, width), generator=torch.Generator(device="cuda").manual_seed(8), device="cuda") * width ** -0.5).bfloat16()
    m, xq = ivb.Mx4(*empty(outputs, width)), ivb.Mx4(*empty(rows, width))
    ops.mx4_quantize(w, m, stream=stream())
    ops.mx4_quantize(x, xq, stream=stream())
    vx, vw = torch.empty_like(x), torch.empty_like(w)  # (their values need at most two bits: exact)
    ops.mx4_read(xq, vx, stream=stream())
    ops.mx4_read(m, vw, stream=stream())
    vx, vw = vx.double(), vw.double()
    want, mass = (vx @ vw.t()).cpu(), (vx.abs() @ vw.abs().t()).cpu()
    out, again = (torch.full((rows, outputs), math.nan, dtype=torch.float16, device="cuda") for _ in range(2))
    ops.mx4_linear(xq, m, out, stream=stream())
    ops.mx4_linear(x, m, again, scratch=ivb.Mx4(*empty(rows, width)), stream=stream())
    ops.synchronize(stream())
    close(out, want, mass, width, "f16")
    assert torch.equal(out, again)


@pytest.mark.parametrize("rows,width,outputs", [(1, 4096, 300), (20, 288, 200), (300, 2080, 520)])
def test_linear_forms(ops, rows, width, outputs):
    """A matrix that was quantised before gives the same bits; outputs of the other type; part of a larger scratch; strided outputs."""
    x = inputs(rows, width, "f16", 1)
    w, m = weights(ops, outputs, width, 2)
    out = torch.empty((rows, outputs), dtype=torch.float16, device="cuda")
    ops.mx4_linear(x, m, out, scratch=ivb.Mx4(*empty(rows, width)), stream=stream())
    xq = ivb.Mx4(*empty(rows + 200, width, fill=0xFF))  # (what lies behind the rows is NaN)
    ops.mx4_quantize(x, xq, stream=stream())
    again = torch.empty_like(out)
    ops.mx4_linear(xq, m, again, stream=stream())
    assert torch.equal(out, again)
    for pad in (1, 8):
        wide = torch.full((rows + 1, outputs + pad), 5.0, dtype=torch.bfloat16, device="cuda")
        ops.mx4_linear(x, m, wide[:rows, :outputs], scratch=xq, stream=stream())
        want, mass = linear64(x, w)
        close(wide[:rows, :outputs], want, mass, width, "bf16")
        assert (wide[rows] == 5.0).all() and (wide[:, outputs:] == 5.0).all()
    shifted = torch.full((rows * outputs + 1,), 5.0, dtype=torch.float16, device="cuda")
    ops.mx4_linear(x, m, shifted[1:].view(rows, outputs), scratch=xq, stream=stream())
    assert torch.equal(shifted[1:].view(rows, outputs), out) and shifted[0] == 5.0


def test_linear_not_finite_stays_in_its_row(ops):
    """A scale of NaN (e = 255) reaches its row's products alone."""
    x = inputs(40, 256, "f16", 1)
    w, m = weights(ops, 300, 256, 2)
    c, s = empty(40, 256)
    xq = ivb.Mx4(c, s)
    ops.mx4_quantize(x, xq, stream=stream())
    clean, out = (torch.empty((40, 300), dtype=torch.float16, device="cuda") for _ in range(2))
    ops.mx4_linear(xq, m, clean, stream=stream())
    s[0, 1, 7, 0, 2] = 255
    m._keep[1][2, 0, 3, 1, 0] = 255  # row 256 + 32 + 3 of the weights
    ops.mx4_linear(xq, m, out, stream=stream())
    bad = torch.zeros((40, 300), dtype=torch.bool, device="cuda")
    bad[7] = True
    bad[:, 291] = True
    assert out[bad].isnan().all() and torch.equal(out[~bad], clean[~bad])


@pytest.mark.parametrize("rows,width,outputs", [(1, 4096, 512), (40, 4096, 700), (500, 1024, 700)])
def test_linear_same_bits_again(ops, rows, width, outputs):
    x = inputs(rows, width, "f16", 1)
    _, m = weights(ops, outputs, width, 2)
    xq = ivb.Mx4(*empty(rows, width))
    outs = [torch.empty((rows, outputs), dtype=torch.float16, device="cuda") for _ in range(5)]
    for o in outs:
        ops.mx4_linear(x, m, o, scratch=xq, stream=stream())
    assert all(torch.equal(o, outs[0]) for o in outs)


@pytest.mark.parametrize("rows,width,outputs", [(1, 4096, 512), (300, 1024, 700)])
def test_linear_graph(ops, rows, width, outputs):
    x, out = inputs(rows, width, "f16", 1), torch.empty((rows, outputs), dtype=torch.float16, device="cuda")
    w, m = weights(ops, outputs, width, 2)
    xq = ivb.Mx4(*empty(rows, width))
    side = torch.cuda.Stream()
    ops.reserve(side.cuda_stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        ops.mx4_linear(x, m, out, scratch=xq, stream=side.cuda_stream)
        ops.mx4_linear(x, m, out, scratch=xq, stream=side.cuda_stream)  # (one behind the other)
    for seed in (5, 6):
        x.copy_(inputs(rows, width, "f16", seed))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want, mass = linear64(x, w)
        close(out, want, mass, width, "f16")
    ops.synchronize(side.cuda_stream)


def test_linear_on_streams_at_once(ops):
    """Calls on several streams do not meet in a workspace."""
    calls = []
    for seed in range(4):
        x, (_, m) = inputs(3 + seed, 4096, "f16", seed), weights(ops, 384, 4096, seed)
        calls.append((x, m, ivb.Mx4(*empty(3 + seed, 4096)), [torch.empty((3 + seed, 384), dtype=torch.float16, device="cuda") for _ in range(20)],
                      torch.cuda.Stream()))
    wants = []
    for x, m, xq, outs, _ in calls:
        o = torch.empty_like(outs[0])
        ops.mx4_linear(x, m, o, scratch=xq, stream=stream())
        wants.append(o)
    torch.cuda.synchronize()
    for i in range(20):
        for x, m, xq, outs, st in calls:
            ops.mx4_linear(x, m, outs[i], scratch=xq, stream=st.cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for (_, _, _, outs, _), want in zip(calls, wants) for o in outs)
    for c in calls:
        ops.release(c[4].cuda_stream)


def test_refusals(ops):
    c, s = empty(40, 64)
    m = ivb.Mx4(c, s)
    x, out = torch.zeros((40, 64), dtype=torch.float16, device="cuda"), torch.zeros((40, 40), dtype=torch.float16, device="cuda")
    for bad in ((c.cpu(), s), (c.char(), s), (c[:, :8], s), (c[:, ::2], s), (c, s[:, :, :16]), (c, s.char()), (c[None], s),
                (torch.zeros((4, 24), dtype=torch.uint8, device="cuda"), s)):
        with pytest.raises(ValueError):
            ivb.Mx4(*bad)
    for bad in (x.float(), x[:, :32], x.cpu(), x[0], torch.zeros((41, 64), dtype=torch.float16, device="cuda"), x.t()):
        with pytest.raises(ValueError):
            ops.mx4_quantize(bad, m, stream=stream())
        with pytest.raises(ValueError):
            ops.mx4_read(m, bad, stream=stream())
    with pytest.raises(ivb.NativeError):  # rows that are written overlap
        ops.mx4_read(m, x[:1].expand(40, -1), stream=stream())
    with pytest.raises(ivb.NativeError):
        ops.mx4_linear(m, m, out[:1].expand(40, -1), stream=stream())
    for args in (dict(x=x, w=m, out=out), dict(x=m, w=m, out=out, scratch=m), dict(x=x[:39], w=m, out=out, scratch=m), dict(x=m, w=m, out=out[:, :39]),
                 dict(x=m, w=m, out=out.float()), dict(x=m, w=ivb.Mx4(*empty(40, 96)), out=out), dict(x=x.float(), w=m, out=out, scratch=m),
                 dict(x=torch.zeros((50, 64), dtype=torch.float16, device="cuda"), w=m, out=torch.zeros((50, 40), dtype=torch.float16, device="cuda"), scratch=m)):
        with pytest.raises(ValueError):
            ops.mx4_linear(stream=stream(), **args)
    ops.mx4_quantize(x[:0], m, stream=stream())
    ops.mx4_read(m, x[:0], stream=stream())
    ops.mx4_linear(x[:0], m, out[:0], scratch=m, stream=stream())


def test_shared_memory_is_refused(ops):
    """Room for x inside the weights, or the output in x's place, would be read and written at once."""
    big, s = empty(256, 64)
    w, x = ivb.Mx4(big[:64], s[:1]), torch.zeros((16, 64), dtype=torch.float16, device="cuda")
    out = torch.zeros((16, 64), dtype=torch.float16, device="cuda")
    for room in ((big[48:64], s[1:]), (big[63:80], s[1:]), (big[128:144], s[:1])):
        with pytest.raises(ivb.NativeError):
            ops.mx4_linear(x, w, out, scratch=ivb.Mx4(*room), stream=stream())
    with pytest.raises(ivb.NativeError):
        ops.mx4_linear(x, w, x, scratch=ivb.Mx4(big[64:80], s[1:]), stream=stream())
    ops.mx4_quantize(torch.ones((64, 64), dtype=torch.float16, device="cuda"), w, stream=stream())
    ops.mx4_linear(x + 1, w, out, scratch=ivb.Mx4(big[64:80], s[1:]), stream=stream())
    xq = ivb.Mx4(big[48:64], torch.zeros_like(s[:1]))
    ops.mx4_linear(xq, w, out.clone(), stream=stream())  # (what is only read may be shared)
    ops.synchronize(stream())
    assert (out == 64).all()


@pytest.mark.parametrize("rows,more", [(1, 0), (40, 60), (100, 127), (130, 200), (128, 128), (7, 121)])
@pytest.mark.parametrize("width", [96, 4096])
def test_quantize_leaves_the_rows_behind_alone(ops, rows, more, width):
    """The first rows of a matrix that holds others: codes and scales of those stay, scale bytes without a row are 0."""
    whole, x = inputs(rows + more, width, "f16", 5), inputs(rows, width, "bf16", 6)
    c, s = empty(rows + more, width)
    m = ivb.Mx4(c, s)
    ops.mx4_quantize(whole, m, stream=stream())
    ops.mx4_quantize(x, m, stream=stream())
    (codes, e), (first, f) = quantized(whole), quantized(x)
    codes[:rows], e[:rows] = first, f
    assert torch.equal(c.cpu(), packed(codes)) and torch.equal(s.cpu(), spread(e))
    c, s = empty(rows + more, width)
    ops.mx4_quantize(x, ivb.Mx4(c, s), stream=stream())
    want = spread(torch.cat([torch.nn.functional.pad(f, (0, -(width // 32) % 4)), torch.full((more, -(-width // 128) * 4), 0xAA)]))
    touched = (rows + 127) // 128  # (128-row pieces that no row of the call is in are not looked at)
    assert torch.equal(s[:touched].cpu(), want[:touched]) and (s[touched:] == 0xAA).all()
    assert torch.equal(c[:rows].cpu(), packed(first)) and (c[rows:] == 0xAA).all()


def test_memory_that_is_read_and_written_is_refused(ops):
    """Any byte that a call both reads and writes, or writes twice; rows that lie between one another are not refused."""
    def refused(call, *args, **more):
        with pytest.raises(ivb.NativeError):
            call(*args, stream=stream(), **more)

    rows, width = 16, 64
    buf = torch.zeros(1 << 16, dtype=torch.float16, device="cuda")
    byte = buf.view(torch.uint8)
    x = buf[:rows * width].view(rows, width)
    w, room = ivb.Mx4(*empty(64, width, fill=0)), ivb.Mx4(*empty(rows, width, fill=0))
    for at in (0, 1, rows * width - 1):  # the output in x, or one element into it
        refused(ops.mx4_linear, x, w, buf[at:at + rows * 64].view(rows, 64), scratch=room)
    refused(ops.mx4_linear, x[1:], w, buf[:15 * 64].view(15, 64), scratch=room)
    refused(ops.mx4_linear, x[:8], w, torch.as_strided(buf, (8, 64), (96, 1), 511), scratch=room)
    wide = buf[:rows * 200].view(rows, 200)
    refused(ops.mx4_linear, wide[:, :64], w, wide[:, 63:127], scratch=room)
    refused(ops.mx4_linear, wide[:, :64], w, torch.as_strided(buf, (rows, 64), (264, 1), 64), scratch=room)  # (other strides: they meet further down)
    inside = ivb.Mx4(byte[1024:1024 + rows * 32].view(rows, 32), empty(rows, width)[1])
    scales = ivb.Mx4(empty(rows, width)[0], byte[512:1024].view(1, 1, 32, 4, 4))
    for m in (inside, scales):
        refused(ops.mx4_linear, x, w, torch.empty_like(x), scratch=m)                       # the room in x
        refused(ops.mx4_linear, torch.zeros_like(x), w, x, scratch=m)                       # the room in the output
        refused(ops.mx4_linear, m, w, x)                                                    # x in 4 bits in the output
        refused(ops.mx4_linear, torch.zeros_like(x), m, buf[256 if m is scales else 512:][:rows * rows].view(rows, rows), scratch=room)  # the weights
        refused(ops.mx4_quantize, x, m)
        refused(ops.mx4_read, m, x)
    # columns of one buffer, and a matrix behind the rows
    ops.mx4_quantize(torch.ones((64, width), dtype=torch.float16, device="cuda"), w, stream=stream())
    wide[:, :64] = 1
    ops.mx4_linear(wide[:, :64], w, wide[:, 64:128], scratch=room, stream=stream())
    assert (wide[:, 64:128] == 64).all() and (wide[:, :64] == 1).all() and (wide[:, 128:] == 0).all()
    ops.mx4_linear(wide[::2, :64], w, wide[::2, 128:192], scratch=room, stream=stream())
    ops.mx4_linear(wide[:4, :64], w, torch.as_strided(buf, (4, 64), (400, 1), 264), scratch=room, stream=stream())  # (every second row, the columns between)
    assert (wide[::2, 128:192] == 64).all() and (wide[1:9:2, 64:128] == 64).all() and (wide[:, :64] == 1).all()
    ops.mx4_quantize(x, ivb.Mx4(byte[2 * rows * width:2 * rows * width + rows * 32].view(rows, 32), empty(rows, width)[1]), stream=stream())
    ops.synchronize(stream())
