"""examples/video_decoder.py, several answers over the same frames: 4-bit
projections, append, attention behind shared pages and the choice of tokens, run
together, against the same decoder without a cache."""
import importlib.util
import math
import os

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def load():
    spec = importlib.util.spec_from_file_location("video_decoder", os.path.join(ROOT, "examples", "video_decoder.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def four(x):
    """What a matrix becomes in 4 bits (blocks of 32 along its rows), float32."""
    y = x.float().unflatten(-1, (-1, 32))
    most = y.abs().amax(-1, keepdim=True)
    scale = torch.exp2(torch.floor(torch.log2(most.double().clamp(min=2.0 ** -120))) - 2).float()
    a = (y / scale).abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    return torch.copysign((torch.round(a / step) * step).clamp(max=6.0) * scale, y).flatten(-2)


def plain_logits(d, x, pos):
    """Logits of every position, the whole sequence at once: halves where the decoder has halves, 4-bit products, no cache."""
    t, pairs = x.shape[0], d.head_dim // 2
    inv = torch.tensor([10000.0 ** (-i / pairs) for i in range(pairs)], dtype=torch.float64, device="cuda")
    ang = (pos.double()[d.axis_of].t() * inv)[:, None]
    c, s = ang.cos().float(), ang.sin().float()

    def turn(h):
        h = h.float()
        a, b = h[..., :pairs], h[..., pairs:]
        return torch.cat([a * c - b * s, b * c + a * s], -1)

    def linear(h, w):
        return (four(h) @ four(w.t()).t()).half()

    i = torch.arange(t, device="cuda")
    seen = i[None] <= i[:, None]
    for w in d.blocks:
        qkv = linear(torch.nn.functional.rms_norm(x, x.shape[-1:]), w["qkv"]).view(t, -1, d.head_dim)
        q, k, v = turn(qkv[:, :d.q_heads]), turn(qkv[:, d.q_heads:d.q_heads + d.kv_heads]), qkv[:, d.q_heads + d.kv_heads:].float()
        k, v = (h.repeat_interleave(d.q_heads // d.kv_heads, 1) for h in (k, v))
        a = torch.einsum("qhd,khd->hqk", q, k) / math.sqrt(d.head_dim)
        o = torch.einsum("hqk,khd->qhd", torch.softmax(a.masked_fill(~seen, -math.inf), -1), v)
        x = x + linear(o.reshape(t, -1).half(), w["o"])
        a, b = linear(torch.nn.functional.rms_norm(x, x.shape[-1:]), w["up"]).chunk(2, -1)
        x = x + linear(torch.nn.functional.silu(a) * b, w["down"])
    return linear(torch.nn.functional.rms_norm(x, x.shape[-1:]), d.head)


def choose(logits, u, t, k, p):
    x = logits.double().cpu().numpy()
    w = np.exp((x - x.max()) / t)
    order = np.lexsort((np.arange(len(x)), -x))[:k]
    c = np.cumsum(w[order])
    order = np.sort(order[:int(np.argmax(c >= p * c[-1])) + 1])
    c = np.cumsum(w[order])
    return int(order[np.argmax(c > u * c[-1])])


@pytest.mark.parametrize("frames,count", [(5, 6), (2, 1), (1, 40)])
def test_answers(tmp_path, frames, count):
    m = load()
    x = m.frame_tokens(np.random.default_rng(frames).random((frames, 3, 224, 224), dtype=np.float32), str(tmp_path))
    t, steps = x.shape[0], 12
    d = m.Decoder()
    u = torch.rand((steps, count), generator=torch.Generator(device="cuda").manual_seed(7), device="cuda")
    tokens, logits = d.answers(x, count, steps, u, temperature=0.9, top_k=40, top_p=0.9)
    assert tokens.shape == (steps, count) and logits.shape == (steps, count, 1024) and torch.isfinite(logits).all()
    # every token is the one that its logits and its random number say
    for s in range(steps):
        for b in range(count):
            assert int(tokens[s, b]) == choose(logits[s, b], float(u[s, b]), float(np.float32(0.9)), 40, float(np.float32(0.9)))
    if count > 1:
        assert len({tuple(r) for r in tokens.t().tolist()}) > 1  # the answers differ
    # the plain decoder fed an answer's tokens
    i, at = torch.arange(t, device="cuda"), max(t // 49, 7)
    for b in sorted({0, count - 1}):
        pos = torch.cat([torch.stack([i // 49, i // 7 % 7, i % 7]), (torch.arange(steps - 1, device="cuda") + at).expand(3, -1)], 1)
        whole = torch.cat([x @ d.embed_frame, d.embed[tokens[:-1, b].long()]])
        want = plain_logits(d, whole, pos)[t - 1:].float()
        got = logits[:, b].float()
        # Keys and values in 8 bits (steps of at most 2 / 127 of a block's largest element: 1.8 % of their rms) change
        # what the projections quantise: an activation that crosses a border of the 4-bit grid moves by a step there, an
        # rms error of the grid itself (steps of a quarter to a half of a value: some 11 %) for the share of values that
        # cross, at most (1.8 % * sqrt 2) / 11 % = 23 % of them for each of four layers' attention parts:
        # sqrt(4 * (0.025^2 + 0.23 * 0.11^2)) = 12 %, and as much again for what the layers between make of it.
        rel = float((got - want).norm() / want.norm())
        assert rel < 0.24, rel
        other = plain_logits(d, torch.cat([torch.zeros_like(whole[:t]), whole[t:]]), pos)[t - 1:].float()
        assert float((other - want).norm() / want.norm()) > 0.4  # (without the frames they would be others)


def test_answers_again_and_refusals(tmp_path):
    m = load()
    d = m.Decoder(layers=2, max_len=256)
    x = torch.randn((70, 576), generator=torch.Generator().manual_seed(3)).half().cuda()
    u = torch.rand((6, 5), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    tokens, logits = d.answers(x, 5, 6, u)
    again, same = d.answers(x, 5, 6, u)
    assert torch.equal(tokens, again) and torch.equal(logits, same)
    greedy, _ = d.answers(x, 5, 6, u, temperature=0.0)
    assert (greedy == greedy[:, :1]).all()  # (the same most probable token in all)
    with pytest.raises(ValueError):
        d.answers(x, 2, 200, u)
