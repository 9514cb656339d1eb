"""Argument checks of the FP8 products, their quantiser and the router's balance loss, without a GPU: the
C entry points refuse before any CUDA call, the Python surface refuses host tensors."""
import pytest
import torch

E4M3 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def L():
    from sm120_nvfp4_b200 import _lib
    return _lib.lib()


def test_fp8_gemm_refuses_bad_arguments(L):
    def call(m=4, n=64, k=128, a=16, b=16, sa=16, sb=16, c=16, t=0):
        return L.b200_nvfp4_fp8_gemm(m, n, k, a, b, sa, sb, c, t, None)
    for bad in (dict(m=-1), dict(n=0), dict(n=60), dict(k=0), dict(k=120), dict(k=-16), dict(a=None), dict(b=None), dict(sa=None),
                dict(sb=None), dict(c=None), dict(a=24), dict(b=8), dict(c=2), dict(t=3), dict(t=-1)):
        assert call(**bad) == 1, bad


def test_fp8_grouped_gemm_refuses_bad_arguments(L):
    def call(y=16, x=16, w=16, s=16, cu=16, sx=16, sw=16, g=2, m=4, n=64, k=128, avg=0, t=0):
        return L.b200_nvfp4_fp8_grouped_gemm(y, x, w, s, cu, sx, sw, g, m, n, k, avg, t, None)
    for bad in (dict(g=0), dict(g=1025), dict(m=-1), dict(n=4), dict(k=8), dict(y=None), dict(x=None), dict(w=None), dict(s=None),
                dict(cu=None), dict(sx=None), dict(sw=None), dict(y=18), dict(x=17), dict(w=12), dict(t=7),
                dict(g=1024, n=1 << 22)):
        assert call(**bad) == 1, bad


def test_fp8_tile_override_takes_known_tiles_only(L):
    for bad in ((8, 0), (48, 0), (256, 0), (16, 3), (16, 16), (0, -1)):
        assert L.b200_nvfp4_fp8_set_tile(*bad) == 1
    assert L.b200_nvfp4_fp8_set_tile(32, 4) == 0 and L.b200_nvfp4_fp8_set_tile(0, 0) == 0


def test_quantiser_refuses_bad_arguments(L):
    def call(q=16, s=16, x=16, rows=4, k=128, t=0, swiglu=0):
        return L.b200_nvfp4_fp8_quantize_rows(q, s, x, rows, k, t, swiglu, None)
    for bad in (dict(q=None), dict(s=None), dict(x=None), dict(rows=-1), dict(k=0), dict(k=24), dict(t=3), dict(t=-1), dict(q=24),
                dict(x=8), dict(rows=1 << 30, k=1 << 12)):
        assert call(**bad) == 1, bad


def test_balance_loss_refuses_bad_arguments(L):
    need = L.b200_nvfp4_moe_balance_loss_workspace_bytes(100, 64, 3)
    assert need > 0 and L.b200_nvfp4_moe_balance_loss_workspace_bytes(100, 5000, 3) == 0
    assert L.b200_nvfp4_moe_balance_loss_workspace_bytes(-1, 64, 3) == 0

    def call(loss=16, counts=16, slope=16, z=16, ids=16, cu=16, t=100, e=64, k=4, s=3, dtype=2, scoring=0, ws=256, size=need):
        return L.b200_nvfp4_moe_balance_loss(loss, counts, slope, z, ids, cu, t, e, k, s, dtype, scoring, 1.0, ws, size, None)
    for bad in (dict(loss=None), dict(counts=None), dict(slope=None), dict(z=None), dict(ids=None), dict(cu=None), dict(t=-1),
                dict(e=0), dict(e=4097), dict(k=0), dict(k=65), dict(s=0), dict(s=65537), dict(dtype=3), dict(scoring=2), dict(z=18),
                dict(ws=128)):
        assert call(**bad) == 1, bad
    assert call(ws=None) == 3 and call(size=need - 1) == 3


def test_router_backward_refuses_bad_arguments(L):
    def call(out=16, z=16, ids=16, w=16, gw=16, slope=16, g=16, cu=16, t=10, e=64, k=4, s=3, dtype=2, scoring=0):
        return L.b200_nvfp4_moe_router_backward(out, z, ids, w, gw, slope, g, cu, t, e, k, s, dtype, scoring, None)
    for bad in (dict(out=None), dict(z=None), dict(ids=None), dict(w=None), dict(gw=None, slope=None), dict(g=None), dict(cu=None),
                dict(t=-1), dict(e=4097), dict(k=65), dict(s=0), dict(dtype=-1), dict(scoring=-1), dict(out=17), dict(z=2)):
        assert call(**bad) == 1, bad


def test_python_surface_refuses_host_tensors():
    import sm120_nvfp4_b200 as ops
    a, s = torch.zeros((4, 128), dtype=E4M3), torch.ones((4, 1))
    z, ids = torch.zeros((4, 8)), torch.zeros((4, 2), dtype=torch.int32)
    one = torch.ones(())
    calls = [lambda: ops.fp8_gemm(a, a, s, s), lambda: ops.quantize_fp8(torch.zeros((4, 128))),
             lambda: ops.fp8_grouped_gemm(a, a.view(1, 4, 128), ids[0], ids[0], s, s.view(1, 4, 1)),
             lambda: ops.router_balance_loss(z, ids), lambda: ops.router_topk_balanced(z, 2),
             lambda: ops.router_balance_loss(z.requires_grad_(), ids),
             lambda: ops.router_backward(z.detach(), ids, slope=z.detach()[:1], grad_loss=one)]
    for call in calls:
        with pytest.raises(RuntimeError):
            call()


def test_sizes_beyond_32_bit_arithmetic_are_refused(L):
    # K + 127, the fetches a few tokens past the end and counts of slots have to fit 32 bits
    most = 0x7fffff00
    assert L.b200_nvfp4_fp8_gemm(1, 8, most + 16, 16, 16, 16, 16, 16, 0, None) == 1
    assert L.b200_nvfp4_fp8_gemm(most + 1, 8, 16, 16, 16, 16, 16, 16, 0, None) == 1
    assert L.b200_nvfp4_fp8_grouped_gemm(16, 16, 16, 16, 16, 16, 16, 1, 1, 8, most + 16, 0, 0, None) == 1
    assert L.b200_nvfp4_fp8_quantize_rows(16, 16, 16, 1, most + 16, 0, 0, None) == 1
    for t, k in (((1 << 30) + 1, 1), (1 << 30, 2), (1 << 28, 8)):
        assert L.b200_nvfp4_moe_balance_loss(16, 16, 16, 16, 16, None, t, 8, k, 1, 2, 0, 1.0, 256, 1 << 40, None) == 1
        assert L.b200_nvfp4_moe_router_backward(16, 16, 16, 16, 16, 16, 16, None, t, 8, k, 1, 2, 0, None) == 1
    assert L.b200_nvfp4_moe_balance_loss_workspace_bytes((1 << 30) + 1, 8, 1) == 0
    assert L.b200_nvfp4_moe_balance_loss_workspace_bytes(1 << 30, 8, 1) > 0


def test_scales_and_indexes_off_their_alignment_are_refused(L):
    for i in (5, 6):
        args = [4, 64, 128, 16, 16, 16, 16, 16, 0, None]
        args[i] = 18
        assert L.b200_nvfp4_fp8_gemm(*args) == 1, i
    for i in (3, 4, 5, 6):
        args = [16] * 7 + [2, 4, 64, 128, 0, 0, None]
        args[i] = 18
        assert L.b200_nvfp4_fp8_grouped_gemm(*args) == 1, i
    assert L.b200_nvfp4_fp8_quantize_rows(16, 18, 16, 4, 128, 0, 0, None) == 1
    for i in (0, 1, 2, 4, 5):
        args = [16] * 6 + [10, 64, 4, 3, 2, 0, 1.0, 256, 1 << 30, None]
        args[i] = 18
        assert L.b200_nvfp4_moe_balance_loss(*args) == 1, i
    for i in (2, 3, 4, 5, 6, 7):
        args = [16] * 8 + [10, 64, 4, 3, 2, 0, None]
        args[i] = 18
        assert L.b200_nvfp4_moe_router_backward(*args) == 1, i


@pytest.mark.gpu
def test_python_surface_refuses_sizes_beyond_the_limits():
    import sm120_nvfp4_b200 as ops
    z = torch.empty(((1 << 30) + 1, 1), dtype=torch.float16, device="cuda")
    ids = torch.empty(((1 << 30) + 1, 1), dtype=torch.int32, device="cuda")
    for call in (lambda: ops.router_balance_loss(z, ids),
                 lambda: ops.router_backward(z, ids, slope=torch.zeros((1, 1), device="cuda"), grad_loss=torch.ones((), device="cuda"))):
        with pytest.raises(RuntimeError, match="2\\^30"):
            call()
    a = z.view(torch.uint8)[:0x7fffff10 // 2].view(1, 0x7fffff10)
    b = torch.empty((8, 0x7fffff10), dtype=torch.uint8, device="cuda")
    scales = torch.empty((1, (0x7fffff10 + 127) // 128), device="cuda")
    with pytest.raises(RuntimeError, match="0x7fffff00"):
        ops.fp8_gemm(a, b, scales, scales)
    del b
    with pytest.raises(RuntimeError, match="2\\^31"):
        ops.quantize_fp8(torch.empty((1, 0x7fffff10), dtype=torch.float16, device="cuda"))


@pytest.mark.gpu
def test_python_surface_refuses_wrong_shapes_and_types():
    import sm120_nvfp4_b200 as ops
    dev = dict(device="cuda")
    a, b = torch.zeros((4, 256), dtype=E4M3, **dev), torch.zeros((136, 256), dtype=E4M3, **dev)
    sa, sb = torch.ones((4, 2), **dev), torch.ones((2, 2), **dev)
    ops.fp8_gemm(a, b, sa, sb)
    w, sw = b.view(1, 136, 256), sb.view(1, 2, 2)
    n1, n2 = torch.tensor([4], dtype=torch.int32, **dev), torch.tensor([0, 4], dtype=torch.int32, **dev)
    ops.fp8_grouped_gemm(a, w, n1, n2, sa, sw)
    z, ids = torch.zeros((4, 8), **dev), torch.zeros((4, 2), dtype=torch.int32, **dev)
    one, slope, gw = torch.ones((), **dev), torch.zeros((1, 8), **dev), torch.zeros((4, 2), **dev)
    store = torch.zeros(4 * 256 + 8, dtype=torch.uint8, **dev)
    bad = [
        lambda: ops.fp8_gemm(a, b, sa[:, :1].contiguous(), sb), lambda: ops.fp8_gemm(a, b, sa, sb[:1]),
        lambda: ops.fp8_gemm(a, b, sa.double(), sb), lambda: ops.fp8_gemm(a.float(), b, sa, sb),
        lambda: ops.fp8_gemm(a, b[:, :128], sa, sb), lambda: ops.fp8_gemm(a, b[:132], sa, sb),
        lambda: ops.fp8_gemm(a, b, sa, sb, out_dtype=torch.float64), lambda: ops.fp8_gemm(a, b, sa.cpu(), sb),
        lambda: ops.fp8_gemm(a, b, sa, sb, output=torch.zeros((4, 128), **dev)),
        lambda: ops.fp8_gemm(a, b, sa, sb, output=torch.zeros((4, 136), **dev), out_dtype=torch.float16),
        lambda: ops.fp8_gemm(a, b, sa, sb, output=torch.zeros((136, 4), **dev).t()),
        lambda: ops.fp8_gemm(store[8:8 + 1024].view(4, 256), b, sa, sb), lambda: ops.fp8_gemm(a, w, sa, sb),
        lambda: ops.fp8_grouped_gemm(a, w, n1.long(), n2, sa, sw), lambda: ops.fp8_grouped_gemm(a, w, n2, n2, sa, sw),
        lambda: ops.fp8_grouped_gemm(a, w, n1.cpu(), n2, sa, sw), lambda: ops.fp8_grouped_gemm(a, b, n1, n2, sa, sw),
        lambda: ops.quantize_fp8(torch.zeros((4, 120), **dev)), lambda: ops.quantize_fp8(torch.zeros((4, 128), **dev).double()),
        lambda: ops.quantize_fp8(torch.zeros((128, 4), **dev).t()), lambda: ops.quantize_fp8(torch.zeros((4, 48), **dev), swiglu=True),
        lambda: ops.quantize_fp8(torch.zeros((4, 128), **dev), output=torch.zeros((4, 128), **dev)),
        lambda: ops.quantize_fp8(torch.zeros((4, 128), **dev), output_scale=torch.zeros((4, 2), **dev)),
        lambda: ops.router_balance_loss(z, ids.long()), lambda: ops.router_balance_loss(z, ids[:2]),
        lambda: ops.router_balance_loss(z.double(), ids), lambda: ops.router_balance_loss(z, ids, scoring="relu"),
        lambda: ops.router_balance_loss(z, ids, cu_seqlens=torch.zeros(1, dtype=torch.int32, **dev)),
        lambda: ops.router_balance_loss(z, ids, cu_seqlens=torch.zeros(3, dtype=torch.int64, **dev)),
        lambda: ops.router_balance_loss(z, torch.zeros((4, 9), dtype=torch.int32, **dev)),
        lambda: ops.router_backward(z, ids), lambda: ops.router_backward(z, ids, slope=slope),
        lambda: ops.router_backward(z, ids, grad_weights=gw), lambda: ops.router_backward(z, ids, slope=slope[:, :4], grad_loss=one),
        lambda: ops.router_backward(z, ids, slope=slope, grad_loss=one.cpu()),
        lambda: ops.router_backward(z, ids, topk_weights=gw, grad_weights=gw[:, :1]),
        lambda: ops.router_topk_balanced(z.half(), 2), lambda: ops.router_topk_balanced(z, 9),
        lambda: ops.router_topk_balanced(z, 2, scoring="x"),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail(f"call {i} was not refused")


def test_kernels_that_start_early_make_no_read_only_loads():
    # they run beside the kernel that still writes what they read, so nothing of it may be declared unchanging
    import re
    from pathlib import Path
    import sm120_nvfp4_b200
    sources = [p for p in sorted((Path(sm120_nvfp4_b200.__file__).parent / "csrc").glob("*.cu*")) if p.name != "ptx.cuh"]
    early = [p for p in sources if "grid_wait()" in p.read_text()]
    assert {"fp8_gemm_kernel.cuh", "fp8_quant.cu", "router_loss.cu", "router_grad.cu"} <= {p.name for p in early}
    for p in early + [p for p in sources if p.name == "router_common.cuh"]:
        code = re.sub(r"//[^\n]*", "", p.read_text())
        assert not re.search(r"__ldg|__restrict__|\.nc\b", code), p.name


def test_calls_go_through_ctypes_where_the_extension_module_is_not_to_be_had(monkeypatch):
    import importlib
    import warnings
    from sm120_nvfp4_b200 import _lib, build

    def no_compiler(force=False):
        raise FileNotFoundError("g++")

    def no_module(name, package=None):
        raise ImportError("undefined symbol")

    for patch in ((build, "build_calls", no_compiler), (importlib, "import_module", no_module)):
        with monkeypatch.context() as m:
            m.setattr(_lib, "_calls", None)
            m.setattr(*patch)
            with pytest.warns(RuntimeWarning, match="ctypes"):
                declines = _lib.calls()
            assert declines.fp8_gemm(1, 2, 3) is None and declines.balance_loss() is None
            with warnings.catch_warnings():
                warnings.simplefilter("error")
                assert _lib.calls() is declines                            # said once
    assert _lib.calls().__name__.endswith("_calls")


def test_the_extension_module_is_built_again_when_its_source_changes(monkeypatch, tmp_path):
    import os
    import subprocess
    from pathlib import Path
    from sm120_nvfp4_b200 import build
    source, runs = tmp_path / "torch_calls.cpp", []
    source.write_text("one")

    def compiler(cmd, **kwargs):
        out = Path(cmd[cmd.index("-o") + 1])
        assert out != build.CALLS and out.parent == build.CALLS.parent     # not into a file that somebody may be loading
        out.write_text(source.read_text())
        runs.append(out)
        return subprocess.CompletedProcess(cmd, int("error" in source.read_text()), "", "")

    monkeypatch.setattr(build, "CALLS", tmp_path / "_calls.so")
    monkeypatch.setattr(build, "CALLS_MADE_FROM", tmp_path / "build" / "_calls.digest")
    monkeypatch.setattr(build, "_CALLS_SOURCE", source)
    monkeypatch.setattr(build.subprocess, "run", compiler)
    assert build.build_calls().read_text() == "one" and len(runs) == 1
    os.utime(source, (2 ** 31 - 10, 2 ** 31 - 10))                          # a copy of the tree has other dates
    build.build_calls()
    assert len(runs) == 1
    source.write_text("two")
    os.utime(source, (1, 1))
    assert build.build_calls().read_text() == "two" and len(runs) == 2
    source.write_text("error")
    with pytest.raises(RuntimeError):
        build.build_calls()
    assert build.CALLS.read_text() == "two" and sorted(p.name for p in tmp_path.iterdir()) == ["_calls.so", "build", "torch_calls.cpp"]
    build.CALLS.unlink()
    source.write_text("two")
    assert build.build_calls().read_text() == "two"
