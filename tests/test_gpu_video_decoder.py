"""examples/video_decoder.py: frames through a plan, then a decoder on the
language-model operators, against the same decoder without a cache in 32 bits."""
import importlib.util
import math
import os

import numpy as np
import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def load():
    spec = importlib.util.spec_from_file_location("video_decoder", os.path.join(ROOT, "examples", "video_decoder.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def plain_logits(d, x, pos, prompt):
    """Logits of every position from `prompt` - 1 on, the whole sequence at once, f32, no cache."""
    x, t = x.float(), x.shape[0]
    pairs = d.head_dim // 2
    inv = torch.tensor([10000.0 ** (-i / pairs) for i in range(pairs)], dtype=torch.float64, device="cuda")
    ang = (pos.double()[d.axis_of].t() * inv)[:, None]
    c, s = ang.cos().float(), ang.sin().float()

    def turn(h):
        a, b = h[..., :pairs], h[..., pairs:]
        return torch.cat([a * c - b * s, b * c + a * s], -1)

    i = torch.arange(t, device="cuda")
    seen = (i[None] <= i[:, None]) & ((i[:, None] - i[None] < d.window) | (i[None] < d.sinks))
    for w in d.blocks:
        qkv = (torch.nn.functional.rms_norm(x, x.shape[-1:]) @ w["qkv"].float()).view(t, -1, d.head_dim)
        q, k, v = turn(qkv[:, :d.q_heads]), turn(qkv[:, d.q_heads:d.q_heads + d.kv_heads]), qkv[:, d.q_heads + d.kv_heads:]
        k, v = (h.repeat_interleave(d.q_heads // d.kv_heads, 1) for h in (k, v))
        a = torch.einsum("qhd,khd->hqk", q, k) / math.sqrt(d.head_dim)
        o = torch.einsum("hqk,khd->qhd", torch.softmax(a.masked_fill(~seen, -math.inf), -1), v)
        x = x + o.reshape(t, -1) @ w["o"].float()
        a, b = (torch.nn.functional.rms_norm(x, x.shape[-1:]) @ w["up"].float()).chunk(2, -1)
        x = x + (torch.nn.functional.silu(a) * b) @ w["down"].float()
    return torch.nn.functional.rms_norm(x[prompt:], x.shape[-1:]) @ d.head.float()


@pytest.mark.gpu
def test_decoder_follows_the_plain_one(tmp_path):
    m = load()
    frames = np.random.default_rng(1).random((5, 3, 224, 224), dtype=np.float32)
    x = m.frame_tokens(frames, str(tmp_path))
    assert x.shape == (245, 576) and torch.isfinite(x).all()
    d = m.Decoder(window=100)
    steps = 40  # passes the window's end and page borders
    tokens, logits = d.generate(x, steps)
    assert len(tokens) == steps and logits.shape == (steps, 1024)
    # the plain decoder fed the same tokens
    i = torch.arange(245, device="cuda")
    pos = torch.cat([torch.stack([i // 49, i // 7 % 7, i % 7]), (torch.arange(steps, device="cuda") + 7).expand(3, steps)], 1)
    whole = torch.cat([x @ d.embed_frame, d.embed[torch.tensor(tokens, device="cuda")]])
    want = plain_logits(d, whole, pos, 245)
    # Key and value codes have steps of at most 2 / 127 of a block's largest
    # element (a scale is a power of two): with sixteen tokens x 64 elements
    # around 4 sigma, an rms error of 4 * 2 / 127 / sqrt(12) = 1.8 % of the
    # values' rms.  Every layer adds such an error twice (keys, values) to a
    # residual stream of which attention is a part: 4 layers, at most
    # 1.8 % * sqrt(2) * sqrt(4) = 5.1 %, and halves a tenth of it.
    rel = float((logits.float() - want).norm() / want.norm())
    assert rel < 0.056, rel
    # without the last tokens' attention to the frames the logits would be others
    blind = plain_logits(d, torch.cat([torch.zeros_like(x @ d.embed_frame), whole[245:]]), pos, 245)
    assert float((blind - want).norm() / want.norm()) > 0.2


@pytest.mark.gpu
def test_decoder_refuses_what_does_not_fit(tmp_path):
    m = load()
    d = m.Decoder(layers=1, max_len=64)
    with pytest.raises(ValueError):
        d.generate(torch.zeros((60, 576), dtype=torch.float16, device="cuda"), 5)


@pytest.mark.gpu
def test_decoder_is_as_before_after_a_refusal():
    """A prompt that is too long is refused before any of it runs."""
    d = load().Decoder(layers=1, max_len=64)
    x = torch.randn((40, 576), generator=torch.Generator().manual_seed(3)).half().cuda()
    tokens, logits = d.generate(x, 5)
    for count, steps in ((70, 5), (64, 1)):
        with pytest.raises(ValueError):
            d.generate(torch.zeros((count, 576), dtype=torch.float16, device="cuda"), steps)
        d.ops.synchronize(d.stream())
        again, same = d.generate(x, 5)
        assert again == tokens and torch.equal(same, logits)


@pytest.mark.gpu
def test_decoder_holds_one_capture_workspace():
    """Generation after generation takes no more memory."""
    d = load().Decoder(layers=1, max_len=64)
    x = torch.randn((20, 576), generator=torch.Generator().manual_seed(3)).half().cuda()
    d.generate(x, 2)
    torch.cuda.synchronize()
    before = torch.cuda.mem_get_info()[0]
    for _ in range(6):
        d.generate(x, 2)
    torch.cuda.synchronize()
    assert before - torch.cuda.mem_get_info()[0] < 60 << 20  # (a workspace is some 40 MB: five more were 200)
