"""Descriptors and refusals of the choice of tokens, 4-bit matrices and shared beginnings that need no GPU."""
import os
import subprocess

import pytest
import torch

import infvino_b200 as ivb
from infvino_b200 import _native, kv


def matrix(rows=130, width=160):
    return torch.zeros((rows, width // 2), dtype=torch.uint8), torch.zeros(ivb.Mx4.scales_shape(rows, width), dtype=torch.uint8)


def test_mx4_descriptor():
    codes, scales = matrix()
    m = ivb.Mx4(codes, scales)
    assert (m.rows, m.width) == (130, 160) and ivb.Mx4.scales_shape(130, 160) == (2, 2, 32, 4, 4)
    assert _native.MX4.unpack(m._m) == (codes.data_ptr(), scales.data_ptr(), 130, 160)
    assert ivb.Mx4.scales_shape(1, 32) == (1, 1, 32, 4, 4) and ivb.Mx4.scales_shape(128, 128) == (1, 1, 32, 4, 4)
    for bad in ((codes.char(), scales), (codes[:, :8], scales), (codes[:, :40], scales), (codes[:100], scales), (codes, scales[:1]), (codes, scales.char()),
                (codes.t(), scales), (codes, scales[..., :2]), (codes[:, :0], scales), (codes[None], scales)):
        with pytest.raises(ValueError):
            ivb.Mx4(*bad)


def test_host_tensors_are_refused():
    """What a handle on device 0 is given on the host is refused before any call."""
    x = torch.zeros((4, 64), dtype=torch.float16)
    with pytest.raises(ValueError):
        kv._matrix(x, "x", 0)
    assert kv._matrix(x, "x", -1)[1:] == (64, 0)
    for bad in (x.float(), x[0], x.t(), x[:, ::2]):
        with pytest.raises(ValueError):
            kv._matrix(bad, "x", -1)
    with pytest.raises(ValueError):
        kv._matrix(x, "x", -1, 4, 32)


def test_structs_match_the_header(tmp_path):
    """The packed structures have the C compiler's sizes, and every field its place."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    fields = {"ivc_kv_groups": (_native.KV_GROUPS, "count first shared"),
              "ivc_logits": (_native.LOGITS, "data dtype rows vocab row_stride"),
              "ivc_sampling": (_native.SAMPLING, "u temperature top_k top_p min_p"),
              "ivc_mx4": (_native.MX4, "codes scales rows width")}
    lines = []
    for name, (s, names) in fields.items():  # field i holds i + 1 in the struct that this prints byte by byte
        sets = "".join(f"x.{f} = (__typeof__(x.{f}))(intptr_t){i + 1};" for i, f in enumerate(names.split()))
        lines.append(f'{{ {name} x; memset(&x, 0, sizeof x); {sets} for (size_t i = 0; i < sizeof x; ++i) printf("%02x", ((unsigned char *)&x)[i]); puts(""); }}')
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include <string.h>\n#include "infvino_b200.h"\nint main(void) {' + "".join(lines) + "return 0;}")
    exe = str(tmp_path / "s")
    subprocess.run(["gcc", str(src), "-I" + os.path.join(root, "include"), "-o", exe], check=True)
    got = subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split()
    assert got == [s.pack(*range(1, len(names.split()) + 1)).hex() for s, names in fields.values()]


def test_null_handles_are_refused():
    L = _native.lib()
    assert L.ivc_kv_attend_shared(None, None, None, None, 0, 1, 1, None, None, 1.0, None, 0, None) == 1
    assert L.ivc_kv_sample(None, None, None, None, None, None) == 1
    assert L.ivc_kv_mx4_quantize(None, 0, None, 0, 0, None, None) == 1
    assert L.ivc_kv_mx4_read(None, None, 0, 0, None, 0, None) == 1
    assert L.ivc_kv_mx4_linear(None, 0, None, 0, 0, None, None, 0, None, 0, None) == 1
