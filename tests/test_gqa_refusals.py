"""CPU: what the grouped-query entry points refuse (C ABI, host pointers that
are never read), the ctypes structures' layout, and the oracle's own pieces."""
import ctypes
import os
import re
import subprocess
import tempfile

import numpy as np
import pytest
import torch

from oracle import gqa_oracle as G

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("name", ["GqaCache", "GqaQuery", "GqaEvictParams", "GqaPrefillParams"])
def test_layout_matches_the_header(name):
    from deepseek_v4_kernel import gqa
    cls = getattr(gqa, name)
    c_name = "dsv4b_" + re.sub(r"(?<!^)(?=[A-Z])", "_", name).lower()
    fields = "".join(f'printf("{f} %zu\\n", offsetof({c_name}, {f}));' for f, _ in cls._fields_)
    src = f'#include <stdio.h>\n#include <stddef.h>\n#include "dsv4b.h"\nint main(void) {{ printf("size %zu\\n", sizeof({c_name}));{fields} return 0; }}\n'
    with tempfile.TemporaryDirectory() as d:
        c, exe = os.path.join(d, "p.c"), os.path.join(d, "p")
        open(c, "w").write(src)
        subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), c, "-o", exe], check=True)
        got = dict(l.split() for l in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split("\n") if l)
    assert int(got.pop("size")) == ctypes.sizeof(cls)
    for f, at in got.items():
        assert int(at) == getattr(cls, f).offset, f


@pytest.fixture
def args():
    from deepseek_v4_kernel import gqa
    buf = ctypes.create_string_buffer(1 << 12)
    a = (ctypes.addressof(buf) + 15) & ~15
    cache = dict(k=a, v=a, k_scale=a, v_scale=a, stride_k_block=64 * 256, stride_k_row=256, stride_k_head=128,
                 stride_v_block=64 * 256, stride_v_row=256, stride_v_head=128, num_blocks=4, page_block_size=64, h_kv=2,
                 d=128, block_table=a, stride_block_table=4, table_width=4, b=2, context_lens=a)
    query = dict(dtype=0, s_q=1, h_q=4, sm_scale=0.1, q=a, stride_q_b=512, stride_q_s=512, stride_q_h=128)
    evict = dict(budget=64, recent=8, weights=a, stride_w_b=512, stride_w_h=256, width=256, new_width=64, new_weights=a,
                 stride_nw_b=128, stride_nw_h=64, kept=a, new_lens=a, new_table=a + 64, stride_new_table=1, new_table_width=1)
    prefill = dict(dtype=0, b=1, h_q=4, h_kv=2, d_qk=128, d_v=128, causal=1, sm_scale=0.1, total_q=8, total_k=8, q=a,
                   stride_q_t=512, stride_q_h=128, k=a, stride_k_t=256, stride_k_h=128, v=a, stride_v_t=256,
                   stride_v_h=128, cu_seqlens_q=a, cu_seqlens_k=a, out=a, stride_o_t=512, stride_o_h=128, lse=a)
    yield gqa, a, cache, query, evict, prefill
    del buf


CACHE_BAD = [("b", 0, -1), ("b", 70000, -2), ("num_blocks", 0, -1), ("page_block_size", 48, -2), ("page_block_size", 8, -2),
             ("page_block_size", 2048, -2), ("d", 96, -2), ("h_kv", 0, -1), ("table_width", 0, -1), ("k", None, -1),
             ("stride_k_row", 136, -1), ("stride_k_head", 64, -1), ("stride_k_block", -256, -1),
             ("stride_k_block", 1 << 41, -1), ("k_scale", None, -1), ("block_table", None, -1), ("context_lens", None, -1),
             ("stride_block_table", -1, -1), ("table_width", (1 << 24) + 1, -2)]


@pytest.mark.parametrize("field,value,rc", CACHE_BAD + [("v", None, -1), ("v_scale", None, -1), ("stride_v_row", 24, -1)])
def test_cache_refusals(args, field, value, rc):
    from deepseek_v4_kernel._lib import lib
    gqa, a, cache, query, evict, _ = args
    c, q, e = gqa.GqaCache(**{**cache, field: value}), gqa.GqaQuery(**query), gqa.GqaEvictParams(**evict)
    r = ctypes.byref
    assert lib.dsv4b_gqa_decode(r(c), r(q), a, 512, 512, 128, a, a, 1 << 30, None) == rc
    assert lib.dsv4b_gqa_cache_append(r(c), 0, a, 256, 128, a, 256, 128, a, 1, None) == rc
    assert lib.dsv4b_gqa_cache_evict(r(c), r(e), None) == rc
    if (field, value, rc) in CACHE_BAD:
        assert lib.dsv4b_gqa_attention_weights(r(c), r(q), a, a, 512, 256, 256, 0, None) == rc


@pytest.mark.parametrize("field,value,rc", [("s_q", 0, -1), ("h_q", 3, -1), ("h_q", 0, -1), ("sm_scale", 0.0, -1),
                                            ("sm_scale", -1.0, -1), ("sm_scale", float("nan"), -1),
                                            ("sm_scale", float("inf"), -1), ("dtype", 2, -2), ("q", None, -1),
                                            ("stride_q_h", 129, -1), ("s_q", 1 << 20, -2)])
def test_query_refusals(args, field, value, rc):
    from deepseek_v4_kernel._lib import lib
    gqa, a, cache, query, _, _ = args
    c, q = gqa.GqaCache(**cache), gqa.GqaQuery(**{**query, field: value})
    r = ctypes.byref
    assert lib.dsv4b_gqa_decode(r(c), r(q), a, 512, 512, 128, a, a, 1 << 30, None) == rc
    assert lib.dsv4b_gqa_attention_weights(r(c), r(q), a, a, 512, 256, 256, 0, None) == rc


def test_other_refusals(args):
    from deepseek_v4_kernel._lib import lib
    gqa, a, cache, query, evict, prefill = args
    c, q = gqa.GqaCache(**cache), gqa.GqaQuery(**query)
    r = ctypes.byref
    assert lib.dsv4b_gqa_decode(None, r(q), a, 512, 512, 128, a, a, 1 << 30, None) == -1
    assert lib.dsv4b_gqa_decode(r(c), None, a, 512, 512, 128, a, a, 1 << 30, None) == -1
    assert lib.dsv4b_gqa_decode(r(c), r(q), a + 8, 512, 512, 128, a, a, 1 << 30, None) == -1
    assert lib.dsv4b_gqa_decode(r(c), r(q), a, 516, 512, 128, a, a, 1 << 30, None) == -1
    assert lib.dsv4b_gqa_decode(r(c), r(q), a, 512, 512, 128, None, a, 1 << 30, None) == -1
    assert lib.dsv4b_gqa_attention_weights(r(c), r(q), None, a, 512, 256, 256, 0, None) == -1
    assert lib.dsv4b_gqa_attention_weights(r(c), r(q), a, a, 512, 256, 0, 0, None) == -1
    assert lib.dsv4b_gqa_attention_weights(r(c), r(q), a, a, 512, 256, (1 << 30) + 1, 0, None) == -2
    e = gqa.GqaEvictParams(**{**evict, "new_width": (1 << 30) + 1})
    assert lib.dsv4b_gqa_cache_evict(r(c), r(e), None) == -2
    assert lib.dsv4b_gqa_cache_append(r(c), 5, a, 256, 128, a, 256, 128, a, 1, None) == -2
    assert lib.dsv4b_gqa_cache_append(r(c), 0, a, 256, 127, a, 256, 128, a, 1, None) == -1
    assert lib.dsv4b_gqa_cache_append(r(c), 0, a, 256, 128, a, 256, 128, None, 1, None) == -1
    assert lib.dsv4b_gqa_cache_append(r(c), 0, a, 256, 128, a, 256, 128, a, -1, None) == -1
    assert lib.dsv4b_gqa_cache_append(r(c), 0, None, 256, 128, None, 256, 128, a, 0, None) == 0
    for f, x in (("budget", 0), ("recent", 65), ("recent", -1), ("new_width", 63), ("weights", None), ("kept", None),
                 ("new_table", None), ("new_table", cache["block_table"]), ("width", 0), ("new_table_width", 0)):
        e = gqa.GqaEvictParams(**{**evict, f: x})
        assert lib.dsv4b_gqa_cache_evict(r(c), r(e), None) == -1, f
    for f, x, rc in (("b", 0, -1), ("h_q", 3, -1), ("h_kv", 0, -1), ("d_qk", 96, -2), ("d_v", 64, -2), ("dtype", 3, -2),
                     ("sm_scale", 0.0, -1), ("total_q", -1, -1), ("total_q", 1 << 31, -2), ("q", a + 2, -1),
                     ("k", None, -1), ("stride_v_t", 257, -1), ("out", None, -1), ("lse", None, -1),
                     ("cu_seqlens_k", None, -1)):
        p = gqa.GqaPrefillParams(**{**prefill, f: x})
        assert lib.dsv4b_gqa_prefill(r(p), None) == rc, f
    p = gqa.GqaPrefillParams(**{**prefill, "total_q": 0})
    assert lib.dsv4b_gqa_prefill(r(p), None) == 0
    assert lib.dsv4b_gqa_prefill(None, None) == -1
    assert lib.dsv4b_gqa_status(None, None) == -1
    n = ctypes.c_size_t()
    assert lib.dsv4b_gqa_decode_workspace_bytes(0, 96, ctypes.byref(n)) == -1


def test_python_refuses_cpu_tensors():
    import deepseek_v4_kernel as dk
    q = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError):
        dk.gqa_prefill_fwd(q, q, q, torch.tensor([0, 4], dtype=torch.int32))
    cache, scale = torch.zeros(2, 16, 2, 64, dtype=torch.uint8), torch.ones(2, 2)
    with pytest.raises(RuntimeError):
        dk.gqa_decode_fwd(q[:, None], cache, cache, scale, scale, torch.zeros(4, 1, dtype=torch.int32),
                          torch.ones(4, dtype=torch.int32))


def test_oracle_e4m3():
    for b in range(256):
        x = G.E4M3[b]
        assert np.isnan(x) if b & 0x7F == 0x7F else G.e4m3_encode(np.array(x)) == b
    x = torch.randn(100000, generator=torch.Generator().manual_seed(0)).double() * 30
    want = x.clamp(-448, 448).float().to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert (G.e4m3_encode(x.float().double().numpy()) == want).all()


@pytest.mark.parametrize("amax,e", [(448.0, 0), (449.0, 1), (224.0, -1), (225.0, 0), (1.0, -8), (0.0, -100), (1e-38, -100)])
def test_oracle_block_exponent(amax, e):
    assert G.block_exponent(amax) == e
