"""FP8 products with a scale per block of 128 and their quantiser, against 64-bit references.

Tolerance of a product, from its arithmetic: 128 products of a block summed in FP32 by the tensor core
(each of 128 additions may truncate: 128 * 2^-23 of the sum of absolute products S), one rounding of the
product of the two scales and one FMA per block (at most kb + 2 roundings of 2^-24 of S), the partial
sums of a split K (8 more), and half a step of the output type. Everything relative to S, so
cancellation needs no allowance of its own."""
import ctypes

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    import sm120_nvfp4_b200 as pkg
    from sm120_nvfp4_b200 import _lib
    _lib.lib().b200_nvfp4_fp8_set_tile(0, 0)
    yield pkg
    _lib.lib().b200_nvfp4_fp8_set_tile(0, 0)
    assert _lib.device_error() == 0, "a bounded wait inside a kernel timed out"


@pytest.fixture
def L(ops):
    from sm120_nvfp4_b200 import _lib
    lib = _lib.lib()
    yield lib
    lib.b200_nvfp4_fp8_set_tile(0, 0)


def blocks(k):
    return (k + 127) // 128


def codes(rows, k, seed):
    """Random finite E4M3 codes of every exponent and FP32 scales of several magnitudes."""
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn((rows, k), generator=g) * torch.exp(torch.randn((rows, 1), generator=g)) * 8).clamp(-448, 448)
    scale = torch.rand((rows, blocks(k)), generator=g) * 2.0 ** torch.randint(-6, 3, (rows, blocks(k)), generator=g)
    return x.to(E4M3).cuda(), scale.cuda()


def weight(n, k, seed):
    x, _ = codes(n, k, seed)
    g = torch.Generator().manual_seed(seed + 1)
    return x, (torch.rand((blocks(n), blocks(k)), generator=g) * 0.02 + 1e-3).cuda()


def wide(scale, rows, k, per_row):
    s = scale if per_row else scale.repeat_interleave(128, 0)[:rows]
    return s.double().repeat_interleave(128, 1)[:, :k]


def reference(a, sa, b, sb):
    """(product, sum of absolute products) in FP64, block by block as the product is defined."""
    want = torch.zeros((a.shape[0], b.shape[0]), dtype=torch.float64, device=a.device)
    total = torch.zeros_like(want)
    for j in range(sa.shape[1]):
        x, y = a[:, 128 * j:128 * j + 128].double(), b[:, 128 * j:128 * j + 128].double()
        scale = sa[:, j].double().unsqueeze(1) * sb[:, j].double().repeat_interleave(128)[:b.shape[0]]
        want += (x @ y.t()) * scale
        total += (x.abs() @ y.abs().t()) * scale
    return want, total


def check(got, want, total, k):
    assert got.dtype in (torch.float16, torch.bfloat16, torch.float32)
    tol = (128 * 2.0 ** -23 + (blocks(k) + 2 + 8) * 2.0 ** -24) * total + torch.finfo(got.dtype).eps / 2 * want.abs()
    if got.dtype == torch.float16:
        tol = tol + 2.0 ** -25          # half a step of its subnormals
    bad = (got.double() - want).abs() > tol
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} values off, worst {float(((got.double() - want).abs() / tol).max())}"


TYPES = [torch.float16, torch.bfloat16, torch.float32]


@pytest.mark.parametrize("m,n,k", [(1, 8, 16), (1, 128, 128), (2, 136, 144), (16, 256, 512), (17, 264, 1040),
                                   (33, 72, 128 * 9), (64, 1000, 656), (65, 128, 2048), (128, 384, 272), (129, 136, 96)])
def test_product_of_few_rows(ops, m, n, k):
    a, sa = codes(m, k, 10 * m + n)
    b, sb = weight(n, k, 7 * m + k)
    want, total = reference(a, sa, b, sb)
    for t in TYPES:
        check(ops.fp8_gemm(a, b, sa, sb, out_dtype=t), want, total, k)


@pytest.mark.parametrize("m,n,k", [(256, 256, 128), (300, 520, 656), (1000, 1032, 400), (2049, 2056, 144)])
@pytest.mark.parametrize("tile", [0, 512])
def test_product_of_many_rows(ops, L, m, n, k, tile):
    assert L.b200_nvfp4_fp8_set_tile(tile, 0) == 0
    a, sa = codes(m, k, m + n)
    b, sb = weight(n, k, m + k)
    want, total = reference(a, sa, b, sb)
    for t in TYPES:
        check(ops.fp8_gemm(a, b, sa, sb, out_dtype=t), want, total, k)


@pytest.mark.parametrize("tile", [16, 32, 64, 128, 512])
@pytest.mark.parametrize("m,n,k", [(5, 264, 1168), (140, 264, 2064)])
def test_every_tile_and_split(ops, L, tile, m, n, k):
    a, sa = codes(m, k, 3)
    b, sb = weight(n, k, 4)
    want, total = reference(a, sa, b, sb)
    for splits in ((1,) if tile == 512 else (1, 2, 4, 8)):
        assert L.b200_nvfp4_fp8_set_tile(tile, splits) == 0
        out = ops.fp8_gemm(a, b, sa, sb, out_dtype=torch.float32)
        check(out, want, total, k)
        assert torch.equal(out, ops.fp8_gemm(a, b, sa, sb, out_dtype=torch.float32))


def test_more_splits_than_blocks_of_k(ops, L):
    a, sa = codes(9, 144, 5)
    b, sb = weight(136, 144, 6)
    want, total = reference(a, sa, b, sb)
    for tile in (16, 32, 64, 128):
        assert L.b200_nvfp4_fp8_set_tile(tile, 8) == 0
        check(ops.fp8_gemm(a, b, sa, sb, out_dtype=torch.float32), want, total, 144)


def test_long_k_and_scales_of_every_magnitude(ops):
    m, n, k = 7, 40, 32768
    a, sa = codes(m, k, 1)
    b, sb = weight(n, k, 2)
    sa *= 2.0 ** torch.randint(-30, 30, sa.shape, device="cuda")
    want, total = reference(a, sa, b, sb)
    check(ops.fp8_gemm(a, b, sa, sb, out_dtype=torch.float32), want, total, k)
    check(ops.fp8_gemm(a, b, sa, sb, out_dtype=torch.bfloat16), want, total, k)


@pytest.mark.parametrize("m,tile", [(20, 0), (20, 16), (300, 512)])
def test_nan_and_infinity_stay_in_their_row_or_column(ops, L, m, tile):
    n, k = 264, 656
    a, sa = codes(m, k, 8)
    b, sb = weight(n, k, 9)
    a.view(torch.uint8)[3, 17] = 0x7f             # a NaN code
    sa[5, 2] = float("inf")
    b.view(torch.uint8)[130, 400] = 0xff
    assert L.b200_nvfp4_fp8_set_tile(tile, 0) == 0
    out = ops.fp8_gemm(a, b, sa, sb, out_dtype=torch.float32)
    want, total = reference(a, sa, b, sb)
    finite = torch.isfinite(want)
    assert torch.equal(torch.isfinite(out), finite)
    assert torch.equal(torch.isnan(out), torch.isnan(want))
    rows = [i for i in range(m) if i not in (3, 5)]
    cols = [i for i in range(n) if i != 130]
    check(out[rows][:, cols], want[rows][:, cols], total[rows][:, cols], k)


GROUPS = [
    ([0, 1, 127, 129], [0, 0, 1, 128, 257], 257),                  # an empty group, odd sizes
    ([3, 0, 0, 5], [0, 3, 3, 3, 8], 8),
    ([0, 0, 0], [0, 0, 0, 0], 4),                                  # nothing at all
    ([300, 2, 260], [0, 300, 302, 562], 562),
    ([4, 4, 4], [0, 10, 20, 30], 30),                              # gaps between the groups
    ([40, 70], [0, 40, 110], 90),                                  # the last group is cut off at the end of x
    ([5, 6], [0, 2000, 2006], 20),                                 # a group outside x altogether
    ([1], [0, 1], 1),
]


@pytest.mark.parametrize("seqlens,cu,rows", GROUPS)
@pytest.mark.parametrize("tile,splits", [(0, 0), (16, 1), (32, 2), (64, 4), (128, 1), (512, 1)])
def test_grouped_product(ops, L, seqlens, cu, rows, tile, splits):
    n, k, e = 264, 400, len(seqlens)
    x, sx = codes(rows, k, rows)
    pairs = [weight(n, k, 100 + i) for i in range(e)]
    w, sw = torch.stack([p[0].view(torch.uint8) for p in pairs]).view(E4M3), torch.stack([p[1] for p in pairs])
    s = torch.tensor(seqlens, dtype=torch.int32).cuda()
    c = torch.tensor(cu, dtype=torch.int32).cuda()
    assert L.b200_nvfp4_fp8_set_tile(tile, splits) == 0
    for t in TYPES:
        out = torch.full((rows, n), 7.0, dtype=t, device="cuda")
        got = ops.fp8_grouped_gemm(x, w, s, c, sx, sw, output=out)
        assert got.data_ptr() == out.data_ptr()
        untouched = torch.ones(rows, dtype=torch.bool)
        for g in range(e):
            lo, hi = cu[g], min(cu[g] + seqlens[g], rows)
            if lo >= rows or hi <= lo:
                continue
            untouched[lo:hi] = False
            want, total = reference(x[lo:hi], sx[lo:hi], w[g], sw[g])
            check(out[lo:hi], want, total, k)
        assert (out[untouched.cuda()] == 7.0).all(), "rows that belong to no group were written"


def test_grouped_product_of_many_groups_and_nan_neighbours(ops):
    """256 groups of 0 to 6 rows; the rows of one group are NaN and no other group sees them."""
    rng = np.random.default_rng(0)
    counts = rng.integers(0, 7, 256).astype(np.int32)
    counts[100] = 3
    cu = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    rows, n, k = int(cu[-1]), 136, 160
    x, sx = codes(rows, k, 1)
    x.view(torch.uint8)[cu[100]:cu[101]] = 0x7f
    g = torch.Generator().manual_seed(5)
    w = (torch.randn((256, n, k), generator=g) * 8).to(E4M3).cuda()
    sw = torch.rand((256, 2, 2), generator=g).cuda()
    out = ops.fp8_grouped_gemm(x, w, torch.from_numpy(counts).cuda(), torch.from_numpy(cu).cuda(), sx, sw, out_dtype=torch.float32)
    for e in range(256):
        lo, hi = cu[e], cu[e + 1]
        if hi == lo:
            continue
        if e == 100:
            assert torch.isnan(out[lo:hi]).all()
            continue
        want, total = reference(x[lo:hi], sx[lo:hi], w[e], sw[e])
        check(out[lo:hi], want, total, k)


def test_no_rows(ops):
    b, sb = weight(128, 256, 1)
    a, sa = codes(0, 256, 1)
    assert ops.fp8_gemm(a, b, sa, sb).shape == (0, 128)
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = ops.fp8_grouped_gemm(a, b.view(1, 128, 256), zero, torch.zeros(2, dtype=torch.int32, device="cuda"), sa, sb.view(1, 1, 2))
    assert out.shape == (0, 128)
    q, s = ops.quantize_fp8(torch.empty((0, 256), dtype=torch.bfloat16, device="cuda"))
    assert q.shape == (0, 256) and s.shape == (0, 2)


def test_raw_bytes_are_accepted(ops):
    a, sa = codes(12, 256, 1)
    b, sb = weight(64, 256, 2)
    assert torch.equal(ops.fp8_gemm(a.view(torch.uint8), b.view(torch.uint8), sa, sb), ops.fp8_gemm(a, b, sa, sb))


# --------------------------------------------------------------------------------------- quantiser


def host_quantize(x):
    """The definition, in FP32 operations of the host (IEEE): codes and scales must agree to the bit."""
    rows, k = x.shape
    pad = torch.zeros((rows, blocks(k) * 128))
    pad[:, :k] = x.float()
    b = pad.view(rows, -1, 128)
    scale = b.abs().amax(-1).clamp(min=2.0 ** -60) / 448.0
    return (b / scale.unsqueeze(-1)).view(rows, -1)[:, :k].to(E4M3), scale


def same_codes(a, b):
    a, b = a.cpu().view(torch.uint8), b.cpu().view(torch.uint8)
    nan = ((a & 0x7f) == 0x7f) & ((b & 0x7f) == 0x7f)
    return bool(((a == b) | nan).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,k", [(1, 16), (1, 128), (3, 144), (16, 7168), (130, 1040), (2500, 1296)])
def test_quantiser_is_the_definition_to_the_bit(ops, dtype, rows, k):
    g = torch.Generator().manual_seed(rows + k)
    x = (torch.randn((rows, k), generator=g) * torch.exp(3 * torch.randn((rows, 1), generator=g))).to(dtype)
    q, s = ops.quantize_fp8(x.cuda())
    wq, ws = host_quantize(x)
    assert q.dtype == E4M3 and torch.equal(s.cpu(), ws) and same_codes(q, wq)
    # and in 64 bits: half a step of E4M3 (2^-4 relative, 2^-10 below its normal numbers), in units of the
    # scale, plus the roundings of the scale and the quotient
    scale = s.cpu().double().repeat_interleave(128, 1)[:, :k]
    v = x.double() / scale
    near = (q.cpu().double() - v).abs() <= torch.clamp(v.abs() * 2.0 ** -4, min=2.0 ** -10) * (1 + 2.0 ** -20)
    assert near[torch.isfinite(scale)].all()       # (the FP16 case overflows to infinity in a few blocks)


def test_quantiser_edges(ops):
    x = torch.zeros((9, 256))
    x[0, 3] = 2.0 ** -70                       # below the floor of amax: rounds to zero
    x[1, 5], x[1, 200] = 1e38, -1e-38
    x[2, 7] = float("inf")
    x[3, 9] = float("nan")
    x[4, :128] = -0.0
    x[5] = torch.linspace(-448, 448, 256)      # scale exactly one: every code's neighbourhood
    x[6] = torch.arange(256) * 2.0 ** -9       # ties between codes
    x[7, 0], x[7, 1] = 2.0 ** -60, 2.0 ** -69
    x[8] = 3.4e38
    q, s = ops.quantize_fp8(x.cuda())
    wq, ws = host_quantize(x)
    assert torch.equal(torch.isnan(s.cpu()), torch.isnan(ws))
    ok = ~torch.isnan(ws)
    assert torch.equal(s.cpu()[ok], ws[ok]) and same_codes(q, wq)
    assert torch.isfinite(s[3, 1]) and torch.isfinite(s[2, 1])       # the neighbouring block is untouched
    value = q.float() * s.repeat_interleave(128, 1)
    assert torch.isnan(value[2, 7]) and torch.isnan(value[3, 9])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,k", [(1, 16), (5, 2048), (333, 400), (2048, 768)])
def test_quantiser_with_silu(ops, dtype, rows, k):
    g = torch.Generator().manual_seed(rows * k)
    x = (torch.randn((rows, 2 * k), generator=g) * 3).to(dtype)
    x[0, 0], x[0, 1] = -100.0, 100.0           # outside the branch-free range of the SiLU
    q, s = ops.quantize_fp8(x.cuda(), swiglu=True)
    gate, up = x[:, :k].double(), x[:, k:].double()
    v = gate * torch.sigmoid(gate) * up
    pad = torch.zeros((rows, blocks(k) * 128), dtype=torch.float64)
    pad[:, :k] = v
    scale = pad.view(rows, -1, 128).abs().amax(-1).clamp(min=2.0 ** -60) / 448.0
    # FP32 SiLU: exp 2 ulp (4 2^-24), sum, quotient, product 1/2 ulp each: 7 2^-24; one more for the scale
    assert ((s.cpu().double() - scale).abs() <= 8 * 2.0 ** -24 * scale).all()
    u = v / scale.repeat_interleave(128, 1)[:, :k]
    step = torch.clamp(u.abs() * 2.0 ** -4, min=2.0 ** -10)
    assert ((q.cpu().double() - u).abs() <= step * (1 + 2.0 ** -19) + 16 * 2.0 ** -24 * u.abs()).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_quantiser_with_silu_of_special_values(ops, dtype):
    # one special pair per block: zeros of both signs, gates around and beyond +-87, tiny ones, infinities, NaN
    tiny = float(torch.finfo(dtype).tiny)
    gates = [0.0, -0.0, 86.5, -86.5, 87.5, -87.5, 100.0, -100.0, tiny, -tiny, float("inf"), float("-inf"), float("nan"), 1.0]
    ups = [1.0, -1.0, 0.0, -0.0, 1000.0, float("inf"), float("nan")]
    pairs = [(a, b) for a in gates for b in ups]
    g = torch.Generator().manual_seed(3)
    x = torch.randn((len(pairs), 256), generator=g).to(dtype)
    x[:, 5], x[:, 128 + 5] = torch.tensor([a for a, _ in pairs]).to(dtype), torch.tensor([b for _, b in pairs]).to(dtype)
    q, s = ops.quantize_fp8(x.cuda(), swiglu=True)
    gate, up = x[:, :128].double(), x[:, 128:].double()
    v = gate / (1.0 + torch.exp(-gate)) * up
    finite = torch.isfinite(v).all(1)
    assert torch.equal(torch.isfinite(s.cpu()[:, 0]), finite)
    v, q, s = v[finite], q.cpu()[finite], s.cpu()[finite]
    scale = v.abs().amax(1, keepdim=True).clamp(min=2.0 ** -60) / 448.0
    assert ((s.double() - scale).abs() <= 8 * 2.0 ** -24 * scale).all()
    u = v / scale
    step = torch.clamp(u.abs() * 2.0 ** -4, min=2.0 ** -10)
    assert ((q.double() - u).abs() <= step * (1 + 2.0 ** -19) + 16 * 2.0 ** -24 * u.abs()).all()
    zero = v == 0
    assert torch.equal(torch.signbit(q.float())[zero], torch.signbit(v)[zero])


# ------------------------------------------------------------------------- as a user's program runs


def test_quantise_then_product_and_input_gradient(ops):
    """The forward product and the input gradient (the same product on the transposed weight) of a layer
    quantised on the way, against the FP64 product of the quantised values."""
    m, n, k = 50, 384, 640
    g = torch.Generator().manual_seed(1)
    x = torch.randn((m, k), generator=g).to(torch.bfloat16).cuda()
    w, sw = weight(n, k, 2)
    q, s = ops.quantize_fp8(x)
    want, total = reference(q, s, w, sw)
    check(ops.fp8_gemm(q, w, s, sw, out_dtype=torch.bfloat16), want, total, k)
    dy = torch.randn((m, n), generator=g).to(torch.bfloat16).cuda()
    qd, sd = ops.quantize_fp8(dy)
    wt, swt = w.view(torch.uint8).t().contiguous().view(E4M3), sw.t().contiguous()
    want, total = reference(qd, sd, wt, swt)
    dx = ops.fp8_gemm(qd, wt, sd, swt, out_dtype=torch.float32)
    check(dx, want, total, n)
    # against the exact gradient of the unquantised dy: what is left is the rounding of dy to E4M3
    exact = dy.double() @ (w.double() * wide(sw, n, k, False))
    step = (sd.double().repeat_interleave(128, 1)[:, :n] * torch.clamp(qd.double().abs() * 2.0 ** -4 * 1.07, min=2.0 ** -10))
    assert ((dx.double() - exact).abs() <= step @ (w.double() * wide(sw, n, k, False)).abs() + 2.0 ** -12 * total).all()


def test_experts_run_together(ops, L):
    """Router -> rows sorted by expert -> quantise -> gate/up -> SiLU * up -> down -> weighted sum."""
    t, e, topk, h, inter = 37, 6, 2, 256, 144
    g = torch.Generator().manual_seed(3)
    x = torch.randn((t, h), generator=g).to(torch.bfloat16).cuda()
    ids, weights, loss, counts = ops.router_topk_balanced(torch.randn((t, e), generator=g).cuda(), topk)
    order = torch.argsort(ids.flatten().long(), stable=True)
    seqlens = counts[0]
    cu = torch.zeros(e + 1, dtype=torch.int32, device="cuda")
    cu[1:] = torch.cumsum(seqlens, 0)
    gate = [weight(2 * inter, h, 20 + i) for i in range(e)]
    down = [weight(h, inter, 40 + i) for i in range(e)]
    stack = lambda p: (torch.stack([a.view(torch.uint8) for a, _ in p]).view(E4M3), torch.stack([b for _, b in p]))  # noqa: E731
    (gw, gs), (dw, ds) = stack(gate), stack(down)
    q, s = ops.quantize_fp8(x[order // topk].contiguous())
    hidden = ops.fp8_grouped_gemm(q, gw, seqlens, cu, s, gs, out_dtype=torch.bfloat16)
    q2, s2 = ops.quantize_fp8(hidden, swiglu=True)
    y = ops.fp8_grouped_gemm(q2, dw, seqlens, cu, s2, ds, out_dtype=torch.float32)
    out = torch.zeros((t, h), device="cuda")
    out.index_add_(0, order // topk, y * weights.flatten()[order].unsqueeze(1))
    assert int(seqlens.sum()) == t * topk and torch.isfinite(loss)
    # the same on dequantised values, step by step
    starts = cu.tolist()
    for i in range(e):
        lo, hi = starts[i], starts[i + 1]
        if hi > lo:
            want, total = reference(q[lo:hi], s[lo:hi], gw[i], gs[i])
            check(hidden[lo:hi], want, total, h)
            want, total = reference(q2[lo:hi], s2[lo:hi], dw[i], ds[i])
            check(y[lo:hi], want, total, inter)


def test_another_stream_and_a_captured_graph(ops):
    m, n, k = 24, 264, 1168
    a, sa = codes(m, k, 1)
    b, sb = weight(n, k, 2)
    big, sbig = codes(520, k, 3)
    x = torch.randn((m, k), device="cuda")
    eager = [ops.fp8_gemm(a, b, sa, sb), ops.fp8_gemm(big, b, sbig, sb), *ops.quantize_fp8(x)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = [ops.fp8_gemm(a, b, sa, sb), ops.fp8_gemm(big, b, sbig, sb), *ops.quantize_fp8(x)]
    torch.cuda.current_stream().wait_stream(side)
    for p, q in zip(eager, other):
        assert torch.equal(p.view(torch.uint8), q.view(torch.uint8))
    graphs = []
    for _ in range(2):                       # two graphs of the same calls
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = [ops.fp8_gemm(a, b, sa, sb), ops.fp8_gemm(big, b, sbig, sb), *ops.quantize_fp8(x)]
        graphs.append((graph, held))
    a.copy_(codes(m, k, 11)[0].view(torch.uint8).view(E4M3))
    x.mul_(3.0)
    for graph, _ in graphs:
        graph.replay()
    torch.cuda.synchronize()
    eager = [ops.fp8_gemm(a, b, sa, sb), ops.fp8_gemm(big, b, sbig, sb), *ops.quantize_fp8(x)]
    for _, held in graphs:
        for p, q in zip(eager, held):
            assert torch.equal(p.view(torch.uint8), q.view(torch.uint8))


@pytest.mark.parametrize("tile,splits,m", [(16, 1, 9), (32, 4, 9), (512, 1, 300)])
def test_a_wait_that_runs_out_is_reported(ops, L, tile, splits, m):
    from sm120_nvfp4_b200 import _lib
    n, k = 264, 2048
    a, sa = codes(m, k, 1)
    b, sb = weight(n, k, 2)
    assert L.b200_nvfp4_fp8_set_tile(tile, splits) == 0
    want = ops.fp8_gemm(a, b, sa, sb)
    try:
        assert L.b200_nvfp4_set_wait_limit(20_000_000, 1) == 0
        ops.fp8_gemm(a, b, sa, sb)
        assert _lib.device_error() & 0xff in range(1, 9)
    finally:
        L.b200_nvfp4_set_wait_limit(0, 0)
    assert torch.equal(ops.fp8_gemm(a, b, sa, sb), want)
    code = ctypes.c_int(-1)
    assert L.b200_nvfp4_device_error(ctypes.byref(code)) == 0 and code.value == 0


class _Declines:
    """Stands in for the extension module and declines every call."""

    def __getattr__(self, name):
        return lambda *args: None


def test_the_long_way_gives_the_same_results(ops, monkeypatch):
    """What the extension module declines goes through ctypes: same outputs, same `output` tensors."""
    from sm120_nvfp4_b200 import _lib
    a, sa = codes(20, 400, 1)
    b, sb = weight(136, 400, 2)
    w, sw = b.view(torch.uint8).view(1, 136, 400).view(E4M3), sb.view(1, *sb.shape)
    n = torch.tensor([15], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, 15], dtype=torch.int32, device="cuda")
    x = torch.randn((20, 800), device="cuda", dtype=torch.float16)
    z = torch.randn((20, 16), device="cuda")
    ids, weights = ops.router_topk(z, 2)

    def everything():
        held = torch.full((20, 136), 3.0, dtype=torch.float32, device="cuda")
        loss, counts, slope = ops.router_balance_loss(z, ids, alpha=0.5)
        return [ops.fp8_gemm(a, b, sa, sb), ops.fp8_gemm(a, b, sa, sb, out_dtype=torch.bfloat16),
                ops.fp8_gemm(a, b, sa, sb, output=torch.empty((20, 136), device="cuda")),
                ops.fp8_grouped_gemm(a, w, n, cu, sa, sw, output=held), *ops.quantize_fp8(x), *ops.quantize_fp8(x, swiglu=True),
                *ops.quantize_fp8(x, output=torch.empty((20, 800), dtype=torch.uint8, device="cuda")),
                loss, counts, slope, ops.router_backward(z, ids, topk_weights=weights, grad_weights=weights, slope=slope, grad_loss=loss)]

    short = everything()
    monkeypatch.setattr(_lib, "calls", lambda: _Declines())
    for p, q in zip(short, everything()):
        assert p.dtype == q.dtype and p.shape == q.shape and torch.equal(p.contiguous().view(-1).view(torch.uint8), q.contiguous().view(-1).view(torch.uint8))


@pytest.mark.parametrize("tile", [0, 16, 128])
def test_offsets_beyond_32_bits(ops, L, tile):
    # A and the output have more than 2^31 elements; only the first and the last rows are not zero
    m, n, k, ends = (1 << 20) + 5, 2056, 2064, 24
    a = torch.zeros((m, k), dtype=torch.uint8, device="cuda")
    sa = torch.ones((m, blocks(k)), device="cuda")
    b, sb = weight(n, k, 2)
    x, sx = codes(2 * ends, k, 1)
    for at, part in ((slice(0, ends), slice(0, ends)), (slice(m - ends, m), slice(ends, 2 * ends))):
        a[at] = x.view(torch.uint8)[part]
        sa[at] = sx[part]
    assert L.b200_nvfp4_fp8_set_tile(tile, 0) == 0
    out = ops.fp8_gemm(a, b, sa, sb)
    want, total = reference(x, sx, b, sb)
    check(torch.cat((out[:ends], out[m - ends:])), want, total, k)
    assert int(torch.count_nonzero(out[ends:m - ends])) == 0


def test_quantiser_offsets_beyond_32_bits(ops):
    rows, k, ends = (1 << 20) + 5, 2064, 24
    for swiglu in (False, True):
        x = torch.zeros((rows, (2 if swiglu else 1) * k), dtype=torch.float16, device="cuda")
        x[:ends].normal_()
        x[-ends:].normal_()
        q, s = ops.quantize_fp8(x, swiglu=swiglu)
        for at in (slice(0, ends), slice(rows - ends, rows)):
            wq, ws = ops.quantize_fp8(x[at].contiguous(), swiglu=swiglu)
            assert torch.equal(s[at], ws) and torch.equal(q[at].view(torch.uint8), wq.view(torch.uint8))
        assert int(torch.count_nonzero(q[ends:-ends].view(torch.uint8) & 0x7f)) == 0
        del x, q, s


def test_weights_beyond_32_bits(ops, L):
    groups, n, k = 40, 7168, 8192
    w = torch.zeros((groups, n, k), dtype=torch.uint8, device="cuda")
    sw = torch.ones((groups, blocks(n), blocks(k)), device="cuda")
    last, s_last = weight(n, k, 3)
    w[-1], sw[-1] = last.view(torch.uint8), s_last
    x, sx = codes(6, k, 4)
    n1 = torch.zeros(groups, dtype=torch.int32, device="cuda")
    n1[0], n1[-1] = 2, 4
    cu = torch.nn.functional.pad(n1.cumsum(0), (1, 0)).to(torch.int32)
    want, total = reference(x[2:], sx[2:], last, s_last)
    for tile in (0, 128, 512):
        assert L.b200_nvfp4_fp8_set_tile(tile, 0) == 0
        out = ops.fp8_grouped_gemm(x, w, n1, cu, sx, sw)
        check(out[2:], want, total, k)
        assert int(torch.count_nonzero(out[:2])) == 0


def test_several_streams_at_once(ops):
    # every kernel of this file beside the others and beside the four-bit product, whose tensor memory they share
    g = torch.Generator(device="cuda").manual_seed(7)
    a, sa = codes(24, 4096, 1)
    big, sbig = codes(1500, 4096, 2)
    b, sb = weight(2048, 4096, 3)
    x = torch.randn((3000, 2048), device="cuda", generator=g)
    four = [torch.randint(0, 256, (r, 1024), dtype=torch.uint8, device="cuda", generator=g) for r in (300, 1024)]
    fours = [torch.full((ops.scale_a_elements(300, 1024, 2048),), 0x38, dtype=torch.uint8, device="cuda"),
             torch.full((ops.scale_b_elements(300, 1024, 2048),), 0x38, dtype=torch.uint8, device="cuda")]
    calls = [lambda: ops.fp8_gemm(a, b, sa, sb), lambda: ops.fp8_gemm(big, b, sbig, sb), lambda: ops.quantize_fp8(x, swiglu=True)[0],
             lambda: ops.gemm(*four, *fours)]
    want = [call().view(torch.uint8) for call in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    got = [[] for _ in calls]
    for _ in range(20):
        for i, call in enumerate(calls):
            with torch.cuda.stream(streams[i]):
                got[i].append(call())
    torch.cuda.synchronize()
    for i, outs in enumerate(got):
        assert all(torch.equal(out.view(torch.uint8), want[i]) for out in outs), i


def test_launches_that_overlap_keep_their_order(ops):
    # Kernels may start while their predecessors drain: each reads what the one before wrote, and writes what it
    # read, over buffers used again at once; with copies and another stream between them; eagerly and captured.
    m, k, n = 48, 1024, 1024
    b, sb = weight(n, k, 5)
    g = torch.Generator(device="cuda").manual_seed(1)
    inputs = [torch.randn((m, k), device="cuda", generator=g) for _ in range(12)]
    want = []
    for x in inputs:
        y = x
        for _ in range(2):
            q, s = ops.quantize_fp8(y)
            torch.cuda.synchronize()
            y = ops.fp8_gemm(q, b, s, sb, out_dtype=torch.float32)
            torch.cuda.synchronize()
        want.append(y)
    q, s = torch.empty((m, k), dtype=E4M3, device="cuda"), torch.empty((m, blocks(k)), device="cuda")
    y, x_in = torch.empty((m, n), device="cuda"), torch.empty((m, k), device="cuda")
    side = torch.cuda.Stream()

    def chain(x, out, aside):
        if aside:                                # the input arrives through another stream
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                x_in.copy_(x)
            torch.cuda.current_stream().wait_stream(side)
        else:
            x_in.copy_(x)
        ops.quantize_fp8(x_in, output=q, output_scale=s)
        ops.fp8_gemm(q, b, s, sb, output=y)
        ops.quantize_fp8(y, output=q, output_scale=s)
        ops.fp8_gemm(q, b, s, sb, output=y)
        out.copy_(y)

    for aside in (False, True):
        outs = [torch.empty_like(y) for _ in inputs]
        for _ in range(20):
            for x, out in zip(inputs, outs):
                chain(x, out, aside)
        assert all(torch.equal(a, w) for a, w in zip(outs, want))
        graph = torch.cuda.CUDAGraph()
        held = [torch.empty_like(y) for _ in inputs]
        with torch.cuda.graph(graph):
            for x, out in zip(inputs, held):
                chain(x, out, aside)
        for _ in range(20):
            graph.replay()
        assert all(torch.equal(a, w) for a, w in zip(held, want))


def test_weights_written_by_the_kernel_before(ops):
    # unsplit few-row products ask for their weights while the kernel before them, which writes these, still runs
    n, k = 9600, 512
    a, sa = codes(5, k, 1)
    sources = [torch.randn((n, k), device="cuda", generator=torch.Generator(device="cuda").manual_seed(i)) for i in range(4)]
    sb = torch.ones((blocks(n), blocks(k)), device="cuda")
    b, scale = torch.empty((n, k), dtype=E4M3, device="cuda"), torch.empty((n, blocks(k)), device="cuda")
    want = []
    for x in sources:
        ops.quantize_fp8(x, output=b, output_scale=scale)
        torch.cuda.synchronize()
        want.append(ops.fp8_gemm(a, b, sa, sb))
        torch.cuda.synchronize()
    got = []
    for _ in range(50):
        for x in sources:
            ops.quantize_fp8(x, output=b, output_scale=scale)
            got.append(ops.fp8_gemm(a, b, sa, sb))
    for i, y in enumerate(got):
        assert torch.equal(y, want[i % 4]), i


@pytest.mark.parametrize("tile,splits,m", [(16, 8, 9), (32, 2, 30), (64, 2, 40), (64, 8, 40), (128, 1, 100), (128, 2, 100), (128, 4, 100)])
def test_clusters_leave_together_when_a_wait_runs_out(ops, L, tile, splits, m):
    # The warps of a cluster whose waits run out still meet its barriers, each warp as one: the launch ends, reports the wait,
    # and the next ones are right; for one group and for several.
    from sm120_nvfp4_b200 import _lib
    n, k = 264, 2048
    a, sa = codes(m, k, 1)
    pairs = [weight(n, k, i) for i in (2, 5)]
    b, sb = pairs[0]
    w, sw = torch.stack([p[0].view(torch.uint8) for p in pairs]).view(E4M3), torch.stack([p[1] for p in pairs])
    n1 = torch.tensor([m // 2, m - m // 2], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, m // 2, m], dtype=torch.int32, device="cuda")
    assert L.b200_nvfp4_fp8_set_tile(tile, splits) == 0
    calls = [lambda: ops.fp8_gemm(a, b, sa, sb), lambda: ops.fp8_grouped_gemm(a, w, n1, cu, sa, sw)]
    for call in calls:
        want = call()
        for _ in range(2):
            try:
                assert L.b200_nvfp4_set_wait_limit(20_000_000, 1) == 0
                call()
                assert _lib.device_error() & 0xff in range(1, 9)
            finally:
                L.b200_nvfp4_set_wait_limit(0, 0)
            assert torch.equal(call(), want) and _lib.device_error() == 0


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows", [24, 700])
def test_expert_layers_that_overlap_keep_their_order(ops, rows, dtype):
    # quantiser, gate/up products, quantiser with SiLU, down products: each starts while the one before still writes what it
    # reads, over buffers used again at once; eagerly and captured
    e, h, inter = 6, 512, 384
    g = torch.Generator(device="cuda").manual_seed(rows)
    inputs = [torch.randn((rows, h), device="cuda", generator=g).to(dtype) for _ in range(8)]
    n1 = torch.full((e,), rows // e, dtype=torch.int32, device="cuda")
    cu = torch.arange(e + 1, dtype=torch.int32, device="cuda") * (rows // e)
    stack = lambda n, k, at: [torch.stack(x) for x in zip(*((a.view(torch.uint8), b) for a, b in (weight(n, k, at + i) for i in range(e))))]  # noqa: E731
    (gw, gs), (dw, ds) = stack(2 * inter, h, 10), stack(h, inter, 30)
    x_in, mid, out = (torch.empty((rows, c), dtype=dtype, device="cuda") for c in (h, 2 * inter, h))
    q1, s1 = torch.empty((rows, h), dtype=E4M3, device="cuda"), torch.empty((rows, blocks(h)), device="cuda")
    q2, s2 = torch.empty((rows, inter), dtype=E4M3, device="cuda"), torch.empty((rows, blocks(inter)), device="cuda")
    mid.zero_(), out.zero_()

    def layer(x, to, wait):
        meet = torch.cuda.synchronize if wait else lambda: None
        x_in.copy_(x)
        for _ in range(2):                       # (the second layer reads the first one's output)
            ops.quantize_fp8(x_in, output=q1, output_scale=s1)
            meet()
            ops.fp8_grouped_gemm(q1, gw, n1, cu, s1, gs, output=mid)
            meet()
            ops.quantize_fp8(mid, swiglu=True, output=q2, output_scale=s2)
            meet()
            ops.fp8_grouped_gemm(q2, dw, n1, cu, s2, ds, output=out)
            meet()
            x_in.copy_(out)
        to.copy_(out)

    want, got, held = ([torch.empty_like(out) for _ in inputs] for _ in range(3))
    for x, to in zip(inputs, want):
        layer(x, to, True)
    for _ in range(20):
        for x, to in zip(inputs, got):
            layer(x, to, False)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for x, to in zip(inputs, held):
            layer(x, to, False)
    for _ in range(20):
        graph.replay()
    torch.cuda.synchronize()
    bits = lambda xs: [x.view(torch.int16) for x in xs]  # noqa: E731
    for a, b, c in zip(bits(got), bits(held), bits(want)):
        assert torch.equal(a, c) and torch.equal(b, c)


@pytest.mark.parametrize("dtype", TYPES)
def test_silu_does_not_depend_on_the_values_beside_it(ops, dtype):
    """Every 16-bit gate, and FP32 ones of every exponent, one per block: its scale, which shows the bits of silu(gate) * up, is
    the same with a gate of 100 in the same thread (whose values then take plain divisions) and in a batch of another size."""
    if dtype == torch.float32:
        bits = torch.randint(-2 ** 31, 2 ** 31, (1 << 18,), generator=torch.Generator().manual_seed(1)).to(torch.int32)
        gates = bits.view(torch.float32)
    else:
        gates = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(dtype)
    gates = gates[gates.float().abs() <= 87.0]
    for up in (1.0, -1.375):
        x = torch.zeros((gates.numel(), 256), dtype=dtype, device="cuda")
        x[:, 0], x[:, 128] = gates.cuda(), up
        q, s = ops.quantize_fp8(x, swiglu=True)
        parts = [ops.quantize_fp8(x[i:i + 200].contiguous(), swiglu=True) for i in range(0, min(20000, x.shape[0]), 200)]
        few = sum(p[1].shape[0] for p in parts)
        assert torch.equal(s[:few], torch.cat([p[1] for p in parts]))
        assert torch.equal(q[:few].view(torch.uint8), torch.cat([p[0].view(torch.uint8) for p in parts]))
        x[:, 1] = 100.0                                # times an up of zero
        q2, s2 = ops.quantize_fp8(x, swiglu=True)
        assert torch.equal(s, s2) and torch.equal(q.view(torch.uint8), q2.view(torch.uint8))
        # and it is the rounded value: exp 2 units, sum, quotient, product and scale half a unit each
        v = gates.double() / (1.0 + torch.exp(-gates.double())) * up
        want = v.abs().clamp(min=2.0 ** -60) / 448.0
        assert ((s[:, 0].cpu().double() - want).abs() <= 8 * 2.0 ** -24 * want).all()


def test_other_threads_run_while_a_launch_waits(ops):
    # behind a busy GPU the queue of launches fills up; whoever launches then waits, and must not hold up the other threads
    import threading
    import time
    a, sa = codes(4, 256, 1)
    b, sb = weight(64, 256, 2)
    x = torch.randn((4, 256), device="cuda")
    z = torch.randn((8, 16), device="cuda")
    ids = z.topk(2).indices.to(torch.int32)
    slope, one = torch.zeros((1, 16), device="cuda"), torch.ones((), device="cuda")
    w, sw = b.view(torch.uint8).view(1, 64, 256).view(E4M3), sb.view(1, *sb.shape)
    n1, cu = torch.tensor([4], dtype=torch.int32, device="cuda"), torch.tensor([0, 4], dtype=torch.int32, device="cuda")
    calls = [lambda: ops.fp8_gemm(a, b, sa, sb), lambda: ops.fp8_grouped_gemm(a, w, n1, cu, sa, sw), lambda: ops.quantize_fp8(x),
             lambda: ops.router_balance_loss(z, ids), lambda: ops.router_backward(z, ids, slope=slope, grad_loss=one)]
    for call in calls:
        call()
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        done = threading.Event()

        def launch():
            with torch.cuda.stream(side):
                torch.cuda._sleep(800_000_000)            # some 0.4 s
                for _ in range(2000):
                    call()
            done.set()

        worker = threading.Thread(target=launch)
        began = last = time.perf_counter()
        worst = 0.0
        worker.start()
        while not done.is_set():
            time.sleep(0.001)
            now = time.perf_counter()
            worst, last = max(worst, now - last), now
        worker.join()
        torch.cuda.synchronize()
        assert last - began > 0.25, "the queue did not fill up"
        assert worst < 0.1, worst


@pytest.mark.parametrize("groups", [257, 1024])
@pytest.mark.parametrize("most,tile", [(3, 0), (3, 64), (40, 0), (40, 128), (40, 512)])
def test_grouped_product_of_as_many_groups_as_the_c_entry_takes(ops, L, groups, most, tile):
    rng = np.random.default_rng(groups + most)
    counts = rng.integers(0, most + 1, groups).astype(np.int32)
    counts[-1] = most
    cu = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    rows, n, k = int(cu[-1]), 264, 144
    x, sx = codes(rows, k, 1)
    g = torch.Generator().manual_seed(5)
    w = (torch.randn((groups, n, k), generator=g) * 8).to(E4M3).cuda()
    sw = torch.rand((groups, blocks(n), blocks(k)), generator=g).cuda()
    assert L.b200_nvfp4_fp8_set_tile(tile, 0) == 0
    args = (x, w, torch.from_numpy(counts).cuda(), torch.from_numpy(cu).cuda(), sx, sw)
    out = ops.fp8_grouped_gemm(*args, out_dtype=torch.float32)
    for e in range(groups):
        lo, hi = cu[e], cu[e + 1]
        if hi > lo:
            want, total = reference(x[lo:hi], sx[lo:hi], w[e], sw[e])
            check(out[lo:hi], want, total, k)
    with pytest.raises(RuntimeError):
        ops.fp8_grouped_gemm(x, w.new_empty((1025, 8, 16)), args[2], args[3], sx, sw)
