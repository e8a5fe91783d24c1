"""The C-ABI library builds, loads without a GPU and exports every symbol the public header
declares; the ctypes table covers the header one to one; host-side argument checks work."""

import ctypes
import os
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "fast_route_sm100.h")


def header_functions():
    text = open(HEADER).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    return sorted(set(re.findall(r"\b(fr_[a-z0-9_]+)\s*\(", text)))


def test_header_symbols_exported(lib):
    names = header_functions()
    assert len(names) >= 15
    for n in names:
        assert hasattr(lib, n), f"{n} declared in the header but not exported"


def test_ctypes_table_matches_header(lib):
    from fast_route_b200 import _lib
    assert sorted(_lib.SIGNATURES) == header_functions()
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    for name, (_, args) in _lib.SIGNATURES.items():
        m = re.search(r"\b" + name + r"\s*\(([^;]*?)\)\s*;", text, flags=re.S)
        assert m, name
        params = [p for p in m.group(1).split(",") if p.strip() and p.strip() != "void"]
        assert len(params) == len(args), f"{name}: header has {len(params)} parameters, ctypes table {len(args)}"


def test_version_and_error_strings(lib):
    assert lib.fr_version() >= 100
    assert b"argument" in lib.fr_error_string(-1)
    assert b"aligned" in lib.fr_error_string(-3)
    assert lib.fr_error_string(0) == b"ok"


def test_workspace_queries_need_no_gpu(lib):
    big = lib.fr_moe_workspace_bytes(16384, 4096, 14336, 8, 2)
    small = lib.fr_moe_workspace_bytes(1, 4096, 14336, 8, 2)
    assert 1 << 30 < big < 4 << 30
    assert 0 < small < big
    assert lib.fr_moe_workspace_bytes(0, 4096, 14336, 8, 2) == 0
    assert lib.fr_gemm_splitk_workspace_bytes(32, 4096, 1) == 0
    assert lib.fr_gemm_splitk_workspace_bytes(32, 4096, 4) == 4 * 32 * 4096 * 4


def test_argument_checks_reject_before_any_launch(lib):
    null = ctypes.c_void_p(None)
    assert lib.fr_topk_softmax(null, 0, 4, 8, 8, 1, 2, 1, null, 2, null, 2, 0, null) == -1
    assert lib.fr_align(null, 8, 4, 16, null, 100, null, 100, null, null, null, null, 0, null) == -1
    assert lib.fr_moe_layer(null, null, 1, 1, null, null, 1, 4, 64, 64, 4, 2, 1, null, null, null, null, 0, null) == -1
    assert lib.fr_combine(null, 8, 1, null, 4, 2, 64, 128, null, 8, null) == -1
    # expert-parallel entry points: null tables, experts that do not divide over the ranks, misaligned capacity
    assert lib.fr_ep_experts(null, 2, 0, 0, 64, 8, 0, 0, 16, 2, null, null, null, 1, 64, 64, 8, null, 128, null, 7,
                             null, 0, null) == -1
    assert lib.fr_ep_combine(null, 2, 0, 64, 128, 1, null, null, null, 4, 2, 64, 8, null, 64, null) == -1
    assert lib.fr_ep_workspace_bytes(0, 64, 64, 8) == 0
    small, big = lib.fr_ep_workspace_bytes(1024, 4096, 14336, 8), lib.fr_ep_workspace_bytes(262272, 4096, 14336, 8)
    assert 0 < small < big and big > 9 << 30      # the operand and the activations of 262272 rows: 9.7 GB
    assert lib.fr_moe_experts_rows_cap(8 * 32768, 1) == 262272


def test_product_never_imports_the_oracle():
    pkg = os.path.join(ROOT, "fast_route_b200")
    for d, _, files in os.walk(pkg):
        for f in files:
            if f.endswith((".py", ".cu", ".cuh", ".h")):
                src = open(os.path.join(d, f)).read()
                assert not re.search(r"^\s*(from|import)\s+oracle\b", src, flags=re.M), f
                assert "oracle/" not in src, f


def test_cpu_tensors_are_rejected_loudly():
    import torch
    import fast_route_b200 as fr
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError):
        fr.route_from_logits(torch.zeros(4, 8), 2)
    with pytest.raises(RuntimeError):
        fr.fused_moe(x, torch.zeros(64, 4, dtype=torch.bfloat16), torch.zeros(4, 128, 64, dtype=torch.bfloat16),
                     torch.zeros(4, 64, 64, dtype=torch.bfloat16), 2)


def test_host_chunk_plan_covers_the_batch_exactly():
    """The chunk plan of the host-buffer entry point: contiguous, non-empty, no overlap, every row once; short first
    and last chunks when a batch is split."""
    from fast_route_b200.layers.host import _plan
    for M in (1, 5, 255, 256, 1000, 6144, 6145, 7000, 8192, 16384, 16385, 100000):
        for chunk in (256, 1024, 6144, 1 << 20):
            plan = _plan(M, chunk)
            assert plan[0][0] == 0 and plan[-1][1] == M
            assert all(a < b for a, b in plan)
            assert all(plan[i][1] == plan[i + 1][0] for i in range(len(plan) - 1))
            assert max(b - a for a, b in plan) <= chunk + max(256, chunk // 4)
            if M <= chunk:
                assert plan == [(0, M)]


def test_few_token_layer_and_fp4_checks_reject_before_any_launch(lib):
    null, p = ctypes.c_void_p(None), ctypes.c_void_p(1 << 20)        # p is never dereferenced: every call is refused

    def decode(M=2, H=64, I=64, E=4, k=2, dtype=1, block=0, x=p, w1=p, s1=p, ws=p, nbytes=1 << 30, tw=null, ti=null):
        return lib.fr_moe_decode(x, p, 1, H, w1, s1, null, p, p, null, dtype, block, M, H, I, E, k, 1, p, tw, ti, ws, nbytes,
                                 null)
    assert decode(k=5) == -1 and decode(k=0) == -1 and decode(M=-1) == -1 and decode(block=8) == -1
    assert decode(x=null) == -1 and decode(w1=null) == -1 and decode(block=16, s1=null) == -1
    assert decode(tw=p) == -1 and decode(ti=p) == -1
    assert decode(M=17) == -2 and decode(E=257) == -2 and decode(dtype=2) == -2 and decode(dtype=0, block=32) == -2
    assert decode(H=60) == -3 and decode(I=20) == -3 and decode(H=40, block=16) == -3
    assert decode(w1=ctypes.c_void_p((1 << 20) + 8)) == -3 and decode(ws=ctypes.c_void_p((1 << 20) + 128)) == -3
    assert decode(ws=null) == -4 and decode(nbytes=1000) == -4
    assert decode(M=0) == 0
    assert lib.fr_moe_decode_workspace_bytes(17, 64, 64, 4, 2) == 0
    assert lib.fr_moe_decode_workspace_bytes(16, 4096, 14336, 8, 2) < 8 << 20

    def quant(dtype=1, mats=1, rows=64, cols=1024, block=16, g=p, own=1, q=p, ws=null, nbytes=0):
        return lib.fr_fp4_quantize(p, dtype, mats, rows, cols, 0, cols, block, g, own, q, p, ws, nbytes, null)
    assert quant(block=8) == -1 and quant(cols=0) == -1 and quant(rows=-1) == -1 and quant(g=null) == -1
    assert quant(dtype=3) == -2 and quant(cols=1032) == -2 and quant(mats=65536) == -2
    assert quant(q=ctypes.c_void_p((1 << 20) + 4)) == -3
    assert quant() == -4 and quant(ws=p, nbytes=4) == -4
    assert quant(rows=0) == 0 and quant(mats=0) == 0
    assert lib.fr_fp4_dequantize(p, p, null, 1, 4, 40, 16, 1, p, null) == -2
    assert lib.fr_fp4_dequantize(p, p, null, 1, 4, 64, 16, 7, p, null) == -2
    assert lib.fr_fp4_dequantize(p, p, null, 1, 4, 64, 16, 1, null, null) == -1
    assert lib.fr_fp4_dequantize(p, p, null, 1, 4, 64, 16, 1, ctypes.c_void_p((1 << 20) + 8), null) == -3


@pytest.mark.parametrize("block", [16, 32])
def test_fp4_oracle_rounds_to_the_nearest_code(block):
    """The oracle against a search over all codes: no code is closer to x / scale than the chosen one, ties are even."""
    import numpy as np
    from oracle import fp4
    rng = np.random.default_rng(0)
    x = rng.standard_normal((8, 64)).astype(np.float32)
    x[0, :16] = [0, .25, .75, 1.25, 1.75, 2.5, 3.5, 5, 6, -.25, -.75, -1.25, -1.75, -2.5, -3.5, -5]
    code, sb, glob = fp4.quantize(x, block)
    s = fp4.e4m3(sb) if block == 16 else fp4.e8m0(sb)
    unit = np.repeat(s * (glob if glob is not None else 1.0), block, -1)
    r = np.minimum(np.abs(x / unit), 6.0)
    best = np.abs(r[..., None] - fp4.E2M1[:8]).min(-1)
    assert (np.abs(r - np.abs(fp4.E2M1[code])) <= best + 1e-6).all()
    assert (np.signbit(fp4.E2M1[code]) == np.signbit(x)).all()
    packed = (code[:, 0::2] | code[:, 1::2] << 4).astype(np.uint8)
    assert np.array_equal(fp4.unpack(packed), code)
    if block == 16:
        assert fp4.e4m3(sb).max() == 448.0               # the largest block takes the largest scale


def test_fp4_product_checks_reject_before_any_launch(lib):
    null, p = ctypes.c_void_p(None), ctypes.c_void_p(1 << 20)

    def gemm(m=4, n=8, k=64, block=16, dtype=1, a=p, c=p, ldc=8, ws=null, nbytes=0):
        return lib.fr_fp4_gemm(a, p, null, p, p, null, block, m, n, k, dtype, c, ldc, ws, nbytes, null)
    assert gemm(m=-1) == -1 and gemm(k=0) == -1 and gemm(block=8) == -1 and gemm(ldc=7) == -1
    assert gemm(a=null) == -1 and gemm(c=null) == -1
    assert gemm(k=48) == -2 and gemm(dtype=2) == -2 and gemm(m=1 << 32) == -2
    assert gemm(a=ctypes.c_void_p((1 << 20) + 8)) == -3
    assert gemm(m=0) == 0 and gemm(n=0) == 0
    need = lib.fr_fp4_gemm_workspace_bytes(200, 8, 64, 16)
    assert need == (2 + 2) * 2048 and lib.fr_fp4_gemm_workspace_bytes(128, 8, 64, 16) == 0
    assert gemm(m=200) == -4 and gemm(m=200, ws=p, nbytes=need - 1) == -4
    assert gemm(m=200, ws=ctypes.c_void_p((1 << 20) + 8), nbytes=need) == -3
