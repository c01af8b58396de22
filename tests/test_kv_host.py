"""The language-model operators' descriptors and refusals that need no GPU."""
import os
import subprocess

import pytest
import torch

import infvino_b200 as ivb
from infvino_b200 import _native


def tensors(pages=3, heads=2, page=32, dim=64):
    codes = [torch.zeros((pages, heads, page, dim), dtype=torch.int8) for _ in range(2)]
    return codes + [torch.zeros((pages, heads, page // 16)) for _ in range(2)]


def test_cache_descriptor():
    c = ivb.KvCache(*tensors())
    assert (c.pages, c.kv_heads, c.page_size, c.head_dim) == (3, 2, 32, 64)
    k, v, ks, vs = tensors()
    for bad in ((k.float(), v, ks, vs), (k, v[:2], ks, vs), (k, v, ks[..., :1], vs), (k.transpose(2, 3), v, ks, vs), (k, v, ks.double(), vs)):
        with pytest.raises(ValueError):
            ivb.KvCache(*bad)


def test_rotary_descriptor():
    table = torch.zeros((10, 16, 2))
    r = ivb.Rotary(table, [0] * 8 + [2] * 8)
    assert r.axes == 3
    c = _native.ROTARY.unpack(r.at(torch.zeros((3, 5), dtype=torch.int32), 5, -1))
    assert c[1:5] == (10, 16, 3, 0) and c[6] == 5
    for pos in (torch.zeros((2, 5), dtype=torch.int32), torch.zeros(5, dtype=torch.int32), torch.zeros((3, 4), dtype=torch.int32),
                torch.zeros((3, 5), dtype=torch.int64)):
        with pytest.raises(ValueError):
            r.at(pos, 5, -1)
    with pytest.raises(ValueError):  # host memory, for a handle on device 0
        r.at(torch.zeros((3, 5), dtype=torch.int32), 5, 0)
    with pytest.raises(ValueError):
        ivb.Rotary(table, [0] * 15)
    with pytest.raises(ValueError):
        ivb.Rotary(table.double())


def test_structs_match_the_header(tmp_path):
    """The packed structures have the C compiler's sizes, and every field its place."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    fields = {"ivc_rows": (_native.ROWS, "data token_stride head_stride"),
              "ivc_kv_cache": (_native.KV_CACHE, "k v k_scale v_scale pages page_size kv_heads head_dim"),
              "ivc_kv_seqs": (_native.KV_SEQS, "batch tokens offsets at pages pages_per_seq"),
              "ivc_rotary": (_native.ROTARY, "table positions pairs axes interleaved pos pos_stride axis_of")}
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
    assert L.ivc_kv_create(0, None) == 1
    assert L.ivc_kv_synchronize(None, None) == 1
    assert L.ivc_kv_attend(None, None, None, 0, 1, 1, None, None, 1.0, 0, 0, None) == 1
    L.ivc_kv_destroy(None)
