"""Balance loss, per-expert counts and the router's gradient, against 64-bit references.

Tolerances. A score is 1 / (1 + e^-z): __expf is off by at most 2 + 1.173 |z| units of 2^-23, the sum and
the quotient by three more, so its relative error is at most d(z) = (5 + 1.2 |z|) 2^-23; a probability
carries that of its score, of the sum (the largest of the row) and of one quotient and product. The loss
is a sum of positive terms: the same relative error plus the additions of a chunk (2^-16 for up to 256
of them, taken as worst case). A gradient term p (1 - s) (slope - dot) is off by these errors relative to
the terms before the subtraction."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    import sm120_nvfp4_b200 as pkg
    return pkg


def case(t, e, k, seqs, seed, dtype=torch.float32, masked=0.1, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    z = (torch.randn((t, e), generator=g) * spread).to(dtype)
    ids = z.float().topk(k, dim=1).indices.to(torch.int32)
    ids[torch.rand((t, k), generator=g) < masked / 2] = -1        # empty slots
    ids[torch.rand(t, generator=g) < masked] = -1                 # masked tokens
    cu = None
    if seqs:
        inner = torch.sort(torch.randint(0, t + 1, (seqs + 1,), generator=g)).values
        cu = inner.to(torch.int32)
    gw = torch.randn((t, k), generator=g)
    return z, ids, cu, gw


def probabilities(z, scoring):
    z = z.double()
    if scoring == "softmax":
        p = torch.softmax(z, 1)
        return torch.nan_to_num(p) if torch.isinf(z).any() else p, torch.zeros_like(z)
    s = torch.sigmoid(z)
    logs = torch.nn.functional.logsigmoid(z)
    return torch.nan_to_num(torch.softmax(logs, 1)), s


def reference(z, ids, cu, scoring, alpha):
    """(loss, counts, slope, live, sequence of each token) in FP64, token by token."""
    t, e = z.shape
    k = ids.shape[1]
    bounds = [0, t] if cu is None else cu.tolist()
    s_count = len(bounds) - 1
    p, _ = probabilities(z, scoring)
    valid = (ids >= 0) & (ids < e)
    live = valid.any(1)
    seq = torch.full((t,), -1)
    counts = torch.zeros((s_count, e), dtype=torch.int64)
    total = torch.zeros((s_count, e), dtype=torch.float64)
    tokens = torch.zeros(s_count, dtype=torch.float64)
    for s in range(s_count):
        for i in range(bounds[s], bounds[s + 1]):
            seq[i] = s
            if live[i]:
                tokens[s] += 1
                total[s] += p[i]
                for j in range(k):
                    if valid[i, j]:
                        counts[s, ids[i, j]] += 1
    live &= seq >= 0
    filled = max(1, int((tokens > 0).sum()))
    slope = alpha * e * counts.double() / (k * tokens.clamp(min=1).unsqueeze(1) ** 2 * filled)
    return (slope * total).sum(), counts, slope, live, seq


def score_error(z):
    """d(z) of the row: a bound over its finite logits, as a column."""
    a = torch.where(torch.isfinite(z), z.double().abs(), 0.0).clamp(max=100).amax(1, keepdim=True)
    return (5 + 1.2 * a) * 2.0 ** -23


def reference_grad(z, ids, w, gw, cu, slope, g, scoring, live, seq):
    """Gradient in FP64 and the size its rounding errors are relative to."""
    t, e = z.shape
    p, s = probabilities(z, scoring)
    rest = 1 - s
    grad, size = torch.zeros((t, e), dtype=torch.float64), torch.zeros((t, e), dtype=torch.float64)
    if slope is not None:
        d = slope.double()[seq.clamp(min=0)] * live.unsqueeze(1)
        dot = (d * p).sum(1, keepdim=True)
        grad += g * p * rest * (d - dot) * live.unsqueeze(1)
        size += abs(g) * p * rest * (d + dot)
    if gw is not None:
        zs = torch.sigmoid(z.double())
        for i in range(t):
            ok = [j for j in range(ids.shape[1]) if 0 <= ids[i, j] < e]
            mean = sum(float(gw[i, j]) * float(w[i, j]) for j in ok)
            for j in ok:
                x = int(ids[i, j])
                grad[i, x] += float(w[i, j]) * (1 - zs[i, x]) * (float(gw[i, j]) - mean)
                size[i, x] += float(w[i, j]) * (1 - zs[i, x]) * (abs(float(gw[i, j])) + sum(abs(float(gw[i, n]) * float(w[i, n])) for n in ok))
    return grad, size


def weights_of(z, ids):
    s = torch.sigmoid(z.float()).gather(1, ids.clamp(min=0, max=z.shape[1] - 1).long()) * ((ids >= 0) & (ids < z.shape[1]))
    return s / s.sum(1, keepdim=True).clamp(min=1e-30)


def compare_grad(got, want, size, z):
    # four rounded factors and a dot product of E terms (pairwise over 32 lanes: E/32 + 5 additions)
    tol = (6 * score_error(z) + (z.shape[1] / 32 + 16) * 2.0 ** -23) * size + torch.finfo(got.dtype).eps / 2 * want.abs()
    tol = tol + torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps / 2 + 2.0 ** -126       # steps of subnormal results, underflow
    bad = (got.cpu().double() - want).abs() > tol
    assert not bad.any(), float(((got.cpu().double() - want).abs() / tol).max())


CASES = [(1, 1, 1, 0), (1, 8, 2, 1), (37, 13, 5, 4), (120, 64, 6, 3), (300, 160, 6, 0), (515, 256, 8, 9), (77, 100, 16, 30),
         (64, 384, 8, 2), (50, 513, 4, 3), (40, 1030, 33, 2), (21, 4096, 8, 2)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
@pytest.mark.parametrize("t,e,k,seqs", CASES)
def test_loss_counts_and_gradient(ops, t, e, k, seqs, scoring, dtype):
    z, ids, cu, gw = case(t, e, k, seqs, t + e, dtype)
    w = weights_of(z, ids)
    dev = lambda x: None if x is None else x.cuda()  # noqa: E731
    loss, counts, slope = ops.router_balance_loss(dev(z), dev(ids), cu_seqlens=dev(cu), scoring=scoring, alpha=0.5)
    wl, wc, ws, live, seq = reference(z, ids, cu, scoring, 0.5)
    assert torch.equal(counts.cpu().long(), wc)
    assert ((slope.cpu().double() - ws).abs() <= 2.0 ** -23 * ws).all()
    assert abs(float(loss) - float(wl)) <= float(wl) * (2.0 ** -16 + 4 * float(score_error(z).max()))
    g = torch.tensor(1.7)
    for with_weights, with_loss in ((True, True), (True, False), (False, True)):
        got = ops.router_backward(dev(z), dev(ids), topk_weights=dev(w) if with_weights else None,
                                  grad_weights=dev(gw) if with_weights else None, slope=slope if with_loss else None,
                                  grad_loss=dev(g) if with_loss else None, cu_seqlens=dev(cu), scoring=scoring)
        want, size = reference_grad(z, ids, w, gw if with_weights else None, cu, ws if with_loss else None, float(g), scoring, live, seq)
        assert got.dtype == dtype
        compare_grad(got, want, size, z)


def test_results_are_reproducible_and_chunks_cross_sequences(ops):
    t, e, k = 20011, 96, 4
    z, ids, cu, gw = case(t, e, k, 50, 3)
    args = (z.cuda(), ids.cuda())
    first = ops.router_balance_loss(*args, cu_seqlens=cu.cuda())
    for _ in range(3):
        again = ops.router_balance_loss(*args, cu_seqlens=cu.cuda())
        assert all(torch.equal(a, b) for a, b in zip(first, again))
    wl, wc, ws, _, _ = reference(z, ids, cu, "sigmoid", 1.0)
    assert torch.equal(first[1].cpu().long(), wc)
    assert abs(float(first[0]) - float(wl)) <= float(wl) * 2.0 ** -15


def test_masked_and_extreme_logits(ops):
    low = torch.finfo(torch.float32).min
    z = torch.zeros((8, 12))
    z[0] = -200.0 + torch.arange(12) * 0.5            # every sigmoid underflows
    z[1, :6] = float("-inf")                          # half of the experts masked
    z[2, :6] = low
    z[3] = 90.0
    z[4, 3] = 80.0
    z[5] = -60.0
    z[6] = low
    z[7] = float("-inf")                              # nothing left: no probability, no gradient
    ids = torch.tensor([[1, 2], [7, 8], [7, 7], [0, 11], [3, 12], [-5, 4], [0, 1], [-1, -1]], dtype=torch.int32)
    w, gw = weights_of(z, ids), torch.linspace(-1, 1, 16).view(8, 2)
    w[0], w[5], w[6] = 0.5, torch.tensor([0.0, 1.0]), 0.5
    for scoring in ("sigmoid", "softmax"):
        loss, counts, slope = ops.router_balance_loss(z.cuda(), ids.cuda(), scoring=scoring)
        wl, wc, ws, live, seq = reference(z, ids, None, scoring, 1.0)
        assert torch.equal(counts.cpu().long(), wc) and int(counts.sum()) == 12
        assert abs(float(loss) - float(wl)) <= float(wl) * 2.0 ** -15
        got = ops.router_backward(z.cuda(), ids.cuda(), topk_weights=w.cuda(), grad_weights=gw.cuda(), slope=slope,
                                  grad_loss=torch.ones((), device="cuda"), scoring=scoring)
        want, size = reference_grad(z, ids, w, gw, None, ws, 1.0, scoring, live, seq)
        compare_grad(got, want, size, z)
        assert (got[7] == 0).all()


def test_nan_reaches_its_own_row_and_sequence_only(ops):
    z, ids, _, gw = case(40, 20, 3, 0, 1, masked=0.0)
    cu = torch.tensor([0, 10, 30, 40], dtype=torch.int32).cuda()
    z[35, 4] = float("nan")
    loss, counts, slope = ops.router_balance_loss(z.cuda(), ids.cuda(), cu_seqlens=cu)
    assert torch.isnan(loss) and torch.isfinite(slope).all() and int(counts.sum()) == 120
    grad = ops.router_backward(z.cuda(), ids.cuda(), slope=slope, grad_loss=torch.ones((), device="cuda"), cu_seqlens=cu)
    assert torch.isnan(grad[35]).any() and torch.isfinite(grad[:35]).all() and torch.isfinite(grad[36:]).all()


def test_the_same_expert_twice_in_a_token(ops):
    z, _, _, gw = case(9, 16, 4, 0, 2)
    ids = torch.tensor([[3, 3, 3, 1], [0, 0, 1, 1], [5, -1, 5, 5]] * 3, dtype=torch.int32)
    w = torch.rand((9, 4))
    loss, counts, slope = ops.router_balance_loss(z.cuda(), ids.cuda())
    assert counts[0].tolist()[:6] == [6, 9, 0, 9, 0, 9]
    got = ops.router_backward(z.cuda(), ids.cuda(), topk_weights=w.cuda(), grad_weights=gw.cuda())
    want, size = reference_grad(z, ids, w, gw, None, None, 0.0, "sigmoid", None, None)
    compare_grad(got, want, size, z)
    assert torch.equal(got, ops.router_backward(z.cuda(), ids.cuda(), topk_weights=w.cuda(), grad_weights=gw.cuda()))


def test_no_tokens_and_empty_sequences(ops):
    z = torch.empty((0, 32), device="cuda")
    ids = torch.empty((0, 4), dtype=torch.int32, device="cuda")
    cu = torch.zeros(4, dtype=torch.int32, device="cuda")
    loss, counts, slope = ops.router_balance_loss(z, ids, cu_seqlens=cu)
    assert float(loss) == 0 and int(counts.sum()) == 0 and float(slope.abs().sum()) == 0
    grad = ops.router_backward(z, ids, slope=slope, grad_loss=torch.ones((), device="cuda"), cu_seqlens=cu)
    assert grad.shape == (0, 32)
    z, ids, _, _ = case(6, 8, 2, 0, 1, masked=0.0)
    cu = torch.tensor([3, 3, 3], dtype=torch.int32).cuda()                 # sequences, but none holds a token
    loss, counts, slope = ops.router_balance_loss(z.cuda(), ids.cuda(), cu_seqlens=cu)
    assert float(loss) == 0 and int(counts.sum()) == 0
    grad = ops.router_backward(z.cuda(), ids.cuda(), slope=slope, grad_loss=torch.ones((), device="cuda"), cu_seqlens=cu)
    assert (grad == 0).all()


def test_more_sequences_than_tokens_and_unaligned_rows(ops):
    z, ids, cu, gw = case(30, 24, 3, 200, 4)
    store = torch.zeros(30 * 24 + 1)
    store[1:] = z.flatten()
    off = store.cuda()[1:].view(30, 24)                                    # rows start 4 bytes off a 16-byte boundary
    loss, counts, slope = ops.router_balance_loss(off, ids.cuda(), cu_seqlens=cu.cuda())
    wl, wc, ws, live, seq = reference(z, ids, cu, "sigmoid", 1.0)
    assert torch.equal(counts.cpu().long(), wc) and abs(float(loss) - float(wl)) <= float(wl) * 2.0 ** -15
    got = ops.router_backward(off, ids.cuda(), slope=slope, grad_loss=torch.ones((), device="cuda"), cu_seqlens=cu.cuda())
    want, size = reference_grad(z, ids, None, None, cu, ws, 1.0, "sigmoid", live, seq)
    compare_grad(got, want, size, z)


def test_autograd_of_the_balanced_router(ops):
    t, e, k = 90, 48, 4
    z, _, cu, gw = case(t, e, k, 5, 8)
    leaf = z.cuda().requires_grad_()
    ids, weights, loss, counts = ops.router_topk_balanced(leaf, k, cu_seqlens=cu.cuda(), alpha=0.01)
    plain_ids, plain_weights = ops.router_topk(z.cuda(), k)
    assert torch.equal(ids, plain_ids) and torch.equal(weights, plain_weights)
    assert not ids.requires_grad and not counts.requires_grad
    ((weights * gw.cuda()).sum() + 3.0 * loss).backward()
    _, _, ws, live, seq = reference(z, ids.cpu(), cu, "sigmoid", 0.01)
    want, size = reference_grad(z, ids.cpu(), weights.detach().cpu(), gw, cu, ws, 3.0, "sigmoid", live, seq)
    compare_grad(leaf.grad, want, size, z)
    # the parts alone
    for part in ("weights", "loss", "none"):
        leaf.grad = None
        ids, weights, loss, counts = ops.router_topk_balanced(leaf, k, cu_seqlens=cu.cuda(), alpha=0.01)
        if part == "weights":
            (weights * gw.cuda()).sum().backward()
        elif part == "loss":
            loss.backward()
        else:
            (weights.detach().sum() + leaf.sum() * 0).backward()
        g = {"weights": (gw, None), "loss": (None, ws), "none": (None, None)}[part]
        want, size = reference_grad(z, ids.cpu(), weights.detach().cpu(), g[0], cu, g[1], 1.0, "sigmoid", live, seq)
        compare_grad(leaf.grad, want, size, z)
    # and the loss of a given routing, in half precision
    half = z.to(torch.bfloat16).cuda().requires_grad_()
    loss, _, slope = ops.router_balance_loss(half, ids, cu_seqlens=cu.cuda())
    loss.backward()
    assert half.grad.dtype == torch.bfloat16 and torch.equal(
        half.grad, ops.router_backward(half.detach(), ids, slope=slope, grad_loss=torch.ones((), device="cuda"), cu_seqlens=cu.cuda()))


def test_gradient_against_differences(ops):
    """Central differences of the FP64 loss and weights along random directions (step 1e-5: truncation and
    rounding both below 1e-8 relative to the terms)."""
    t, e, k = 12, 10, 3
    z, _, cu, gw = case(t, e, k, 2, 5, masked=0.0)
    cu = torch.tensor([0, 5, 12], dtype=torch.int32)
    leaf = z.cuda().requires_grad_()
    ids, weights, loss, _ = ops.router_topk_balanced(leaf, k, cu_seqlens=cu.cuda())
    ((weights * gw.cuda()).sum() + loss).backward()
    grad, at = leaf.grad.cpu().double(), ids.cpu().long()

    def value(x):
        picked = torch.sigmoid(x).gather(1, at)
        return float(((picked / picked.sum(1, keepdim=True)) * gw.double()).sum() + reference(x, ids.cpu(), cu, "sigmoid", 1.0)[0])

    g = torch.Generator().manual_seed(1)
    for _ in range(5):
        d = torch.randn((t, e), generator=g, dtype=torch.float64)
        slope = (value(z.double() + 1e-5 * d) - value(z.double() - 1e-5 * d)) / 2e-5
        # the FP32 gradient of 120 entries of size about 0.3: 2^-18 of the sum of their absolute values
        assert abs(float((grad * d).sum()) - slope) <= 2.0 ** -18 * float((grad.abs() * d.abs()).sum()) + 1e-7


def test_captured_and_on_another_stream(ops):
    t, e, k = 500, 128, 8
    z, ids, cu, gw = case(t, e, k, 7, 6)
    z, ids, cu, gw = z.cuda(), ids.cuda(), cu.cuda(), gw.cuda()
    w = weights_of(z.cpu(), ids.cpu()).cuda()
    one = torch.ones((), device="cuda")

    def step():
        loss, counts, slope = ops.router_balance_loss(z, ids, cu_seqlens=cu)
        return loss, counts, slope, ops.router_backward(z, ids, topk_weights=w, grad_weights=gw, slope=slope, grad_loss=one, cu_seqlens=cu)

    eager = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(eager, other))
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = step()
        graphs.append((graph, held))
    z.mul_(0.5)
    for graph, _ in graphs + graphs:
        graph.replay()
    torch.cuda.synchronize()
    eager = step()
    for _, held in graphs:
        assert all(torch.equal(a, b) for a, b in zip(eager, held))


def test_nan_in_masked_and_unselected_places(ops):
    """NaN and infinite logits of masked tokens, of tokens behind the last sequence and (through the
    weights alone) of experts that were not selected change nothing."""
    t, e, k = 40, 24, 3
    z, ids, _, gw = case(t, e, k, 0, 11, masked=0.0)
    cu = torch.tensor([2, 20, 30], dtype=torch.int32)
    ids[5] = -1
    w = weights_of(z, ids).nan_to_num()
    clean = z.clone()
    z[5], z[0], z[35] = float("nan"), float("inf"), float("nan")
    gw[5] = float("nan")                                           # its slots are empty
    one = torch.ones((), device="cuda")
    loss, counts, slope = ops.router_balance_loss(z.cuda(), ids.cuda(), cu_seqlens=cu.cuda())
    want = ops.router_balance_loss(clean.cuda(), ids.cuda(), cu_seqlens=cu.cuda())
    assert all(torch.equal(a, b) for a, b in zip((loss, counts, slope), want)) and torch.isfinite(loss)
    grad = ops.router_backward(z.cuda(), ids.cuda(), slope=slope, grad_loss=one, cu_seqlens=cu.cuda())
    assert torch.equal(grad, ops.router_backward(clean.cuda(), ids.cuda(), slope=slope, grad_loss=one, cu_seqlens=cu.cuda()))
    assert (grad[[0, 1, 5, 30, 35, 39]] == 0).all()
    both = ops.router_backward(z.cuda(), ids.cuda(), topk_weights=w.cuda(), grad_weights=gw.cuda(), slope=slope, grad_loss=one,
                               cu_seqlens=cu.cuda())
    assert (both[5] == 0).all()
    row = clean.clone()
    unselected = [x for x in range(e) if x not in ids[7].tolist()]
    row[7, unselected[0]] = float("nan")
    got = ops.router_backward(row.cuda(), ids.cuda(), topk_weights=w.cuda(), grad_weights=gw.cuda())
    assert torch.equal(got, ops.router_backward(clean.cuda(), ids.cuda(), topk_weights=w.cuda(), grad_weights=gw.cuda()))
    assert (got[7, unselected] == 0).all()


def test_autograd_captured_into_a_graph(ops):
    t, e, k = 200, 64, 4
    z, _, cu, gw = case(t, e, k, 3, 12)
    leaf, cu, gw = z.cuda().requires_grad_(), cu.cuda(), gw.cuda()

    def step():
        _, weights, loss, _ = ops.router_topk_balanced(leaf, k, cu_seqlens=cu)
        return torch.autograd.grad((weights * gw).sum() + loss, leaf)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(held, eager)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,e,k", [(70, 179, 5), (33, 255, 8), (9, 101, 7), (600, 63, 2), (19, 387, 4), (11, 777, 3)])
@pytest.mark.parametrize("offset", [0, 1, 3])
def test_rows_of_any_alignment(ops, t, e, k, offset, dtype):
    """Odd numbers of experts, and matrices that start off a 16-byte boundary with NaN on both sides."""
    z, ids, cu, gw = case(t, e, k, 2, t + e + offset, dtype)
    store = torch.full((t * e + 32,), float("nan"), dtype=dtype)
    store[offset:offset + t * e] = z.flatten()
    off = store.cuda()[offset:offset + t * e].view(t, e)
    w = weights_of(z, ids)
    loss, counts, slope = ops.router_balance_loss(off, ids.cuda(), cu_seqlens=cu.cuda())
    wl, wc, ws, live, seq = reference(z, ids, cu, "sigmoid", 1.0)
    assert torch.equal(counts.cpu().long(), wc) and abs(float(loss) - float(wl)) <= float(wl) * 2.0 ** -15
    got = ops.router_backward(off, ids.cuda(), topk_weights=w.cuda(), grad_weights=gw.cuda(), slope=slope,
                              grad_loss=torch.ones((), device="cuda"), cu_seqlens=cu.cuda())
    want, size = reference_grad(z, ids, w, gw, cu, ws, 1.0, "sigmoid", live, seq)
    compare_grad(got, want, size, z)


def test_offsets_beyond_32_bits(ops):
    # logits of more than 2^31 elements: all tokens but the last eight are indifferent between the experts
    t, e, k, ends = (1 << 19) + 7, 4096, 2, 8
    gen = torch.Generator().manual_seed(5)
    z = torch.zeros((t, e), dtype=torch.bfloat16, device="cuda")
    z[-ends:] = torch.randn((ends, e), generator=gen).to(torch.bfloat16).cuda()
    ids = (torch.arange(2 * t, dtype=torch.int32, device="cuda") % e).view(t, k)
    cu = torch.tensor([0, t - 3, t], dtype=torch.int32, device="cuda")
    loss, counts, slope = ops.router_balance_loss(z, ids, cu_seqlens=cu)
    want = torch.stack([torch.bincount(ids[:t - 3].flatten().long(), minlength=e), torch.bincount(ids[t - 3:].flatten().long(), minlength=e)])
    assert torch.equal(counts.long(), want)
    p = torch.sigmoid(z[-ends:].double())
    p /= p.sum(1, keepdim=True)
    tokens = torch.tensor([[t - 3.0], [3.0]], dtype=torch.float64, device="cuda")
    total = torch.stack([(t - ends) / e + p[:-3].sum(0), p[-3:].sum(0)])
    exact = float((e * want.double() / (k * tokens ** 2 * 2) * total).sum())
    # score error as above with |z| < 6, and a chunk's additions: 296 chunks, one thread per column each
    assert abs(float(loss) - exact) <= exact * ((5 + 1.2 * 6) * 2.0 ** -23 + (t / 290 + 32) * 2.0 ** -24)
    gw = torch.randn((ends, k), generator=gen).cuda()
    w = weights_of(z[-ends:].cpu(), ids[-ends:].cpu()).cuda()
    one = torch.ones((), device="cuda")
    every_w, every_g = torch.zeros((t, k), device="cuda"), torch.zeros((t, k), device="cuda")
    every_w[-ends:], every_g[-ends:] = w, gw
    grad = ops.router_backward(z, ids, topk_weights=every_w, grad_weights=every_g, slope=slope, grad_loss=one, cu_seqlens=cu)
    near = torch.tensor([0, ends - 3, ends], dtype=torch.int32, device="cuda")
    part = ops.router_backward(z[-ends:].contiguous(), ids[-ends:].contiguous(), topk_weights=w, grad_weights=gw, slope=slope, grad_loss=one,
                               cu_seqlens=near)
    assert torch.equal(grad[-ends:], part)


@pytest.mark.parametrize("t,seqs", [(700, 5), (150, 3)])
def test_launches_that_overlap_keep_their_order(ops, t, seqs):
    # loss, its second kernel (the smaller case has none) and the gradient may start while their predecessors drain; ids, sequences and logits
    # are written right before, over buffers used again at once
    e, k = 64, 6
    cases = [case(t, e, k, seqs, i) for i in range(8)]
    cases = [(z.cuda(), ids.cuda(), cu.cuda(), gw.cuda(), weights_of(z, ids).cuda()) for z, ids, cu, gw in cases]
    one = torch.ones((), device="cuda")

    def step(z, ids, cu, gw, w, wait):
        loss, counts, slope = ops.router_balance_loss(z, ids, cu_seqlens=cu)
        if wait:
            torch.cuda.synchronize()
        return loss, counts, slope, ops.router_backward(z, ids, topk_weights=w, grad_weights=gw, slope=slope, grad_loss=one, cu_seqlens=cu)

    want = [step(*c, True) for c in cases]
    buffers = [torch.empty_like(x) for x in cases[0]]

    def all_cases():
        got = []
        for c in cases:
            for to, x in zip(buffers, c):
                to.copy_(x)
            got.append([x.clone() for x in step(*buffers, False)])
        return got

    for _ in range(10):
        for a, w in zip(all_cases(), want):
            assert all(torch.equal(x, y) for x, y in zip(a, w))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = all_cases()
    for _ in range(10):
        graph.replay()
    torch.cuda.synchronize()
    for a, w in zip(held, want):
        assert all(torch.equal(x, y) for x, y in zip(a, w))


@pytest.mark.parametrize("t,e,k,seqs", [(64 * 7, 64, 4, 1), (64 * 7 + 1, 64, 4, 1), (32 * 4 + 1, 128, 8, 4), (64, 60, 3, 7), (65, 60, 3, 7),
                                        (30, 64, 2, 8), (224, 512, 8, 1), (225, 512, 8, 1), (9, 5, 2, 6), (448, 600, 4, 2)])
def test_around_what_one_launch_takes(ops, t, e, k, seqs):
    z, ids, cu, gw = case(t, e, k, seqs, t + e + seqs)
    loss, counts, slope = ops.router_balance_loss(z.cuda(), ids.cuda(), cu_seqlens=cu.cuda())
    wl, wc, ws, live, seq = reference(z, ids, cu, "sigmoid", 1.0)
    assert torch.equal(counts.cpu().long(), wc)
    assert ((slope.cpu().double() - ws).abs() <= ws * 2.0 ** -23).all()
    # a sum of positive terms: the score's error, and at most 64 additions of a block's rows and 16 + 8 of partial rows
    assert abs(float(loss) - float(wl)) <= float(wl) * (float(score_error(z).max()) * 2 + 96 * 2.0 ** -24)
    again = ops.router_balance_loss(z.cuda(), ids.cuda(), cu_seqlens=cu.cuda())
    assert all(torch.equal(a, b) for a, b in zip((loss, counts, slope), again))


@pytest.mark.parametrize("t,e", [(1 << 26, 7), (1 << 24, 13), (1 << 24, 100), (1 << 23, 200), (1 << 22, 520), (1 << 21, 1000), (1 << 20, 3000)])
def test_sums_of_equal_probabilities_do_not_drift(ops, t, e):
    """An indifferent router: every probability is 1 / E, whose roundings all go the same way, and the loss is 1 however
    the slots fall. In units of 2^-24: a row's sum 20 additions of a thread, 5 and 8 of the group's; its reciprocal and the
    quotient of the softmax 4 each at most; a run of 16 additions in FP32; the rest in FP64, the loss rounded once.
    (Beyond 512 experts a thread has 16 columns and a run 32 additions, the i-th of them off by i / 32 of the run's last
    unit: 16.5 in all.) Nothing of it grows with the tokens."""
    z = torch.full((t, e), 0.3, dtype=torch.bfloat16, device="cuda")
    ids = (torch.arange(t, dtype=torch.int32, device="cuda") % e).view(t, 1)
    for scoring in ("sigmoid", "softmax"):
        loss, counts, slope = ops.router_balance_loss(z, ids, scoring=scoring)
        assert abs(float(loss) - 1.0) <= (20 + 5 + 8 + 4 + 16 + 1) * 2.0 ** -24
        want = torch.full((1, e), t // e, dtype=torch.int32, device="cuda")
        want[0, :t % e] += 1
        assert torch.equal(counts, want)


@pytest.mark.parametrize("t,e,k,seqs", [(900, 24, 3, 256), (900, 24, 3, 257), (2500, 40, 3, 3000), (700, 130, 4, 1500), (400, 600, 2, 500),
                                        (1000, 5, 2, 65536)])
def test_many_sequences(ops, t, e, k, seqs):
    z, ids, cu, gw = case(t, e, k, seqs, t + seqs)
    loss, counts, slope = ops.router_balance_loss(z.cuda(), ids.cuda(), cu_seqlens=cu.cuda())
    wl, wc, ws, live, seq = reference(z, ids, cu, "sigmoid", 1.0)
    assert torch.equal(counts.cpu().long(), wc)
    assert ((slope.cpu().double() - ws).abs() <= ws * 2.0 ** -23).all()
    # positive terms: the score's error, and runs of 16 FP32 additions
    assert abs(float(loss) - float(wl)) <= float(wl) * (float(score_error(z).max()) * 2 + 32 * 2.0 ** -24)
    again = ops.router_balance_loss(z.cuda(), ids.cuda(), cu_seqlens=cu.cuda())
    assert all(torch.equal(a, b) for a, b in zip((loss, counts, slope), again))
    got = ops.router_backward(z.cuda(), ids.cuda(), slope=slope, grad_loss=torch.ones((), device="cuda"), cu_seqlens=cu.cuda())
    want, size = reference_grad(z, ids, None, None, cu, ws, 1.0, "sigmoid", live, seq)
    compare_grad(got, want, size, z)


def test_time_grows_with_the_sequences_and_not_with_their_square(ops):
    t, e = 65536, 64
    z = torch.randn((t, e), device="cuda")
    ids = z.topk(4).indices.to(torch.int32)

    def time(seqs):
        cu = torch.linspace(0, t, seqs + 1).to(torch.int32).cuda()
        times = []
        for _ in range(6):
            begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            begin.record()
            ops.router_balance_loss(z, ids, cu_seqlens=cu)
            end.record()
            torch.cuda.synchronize()
            times.append(begin.elapsed_time(end))
        return sorted(times)[2]

    few, many = time(4096), time(32768)
    assert many < 24 * few, (few, many)        # eight times the sequences; their square would be 64


def test_many_sequences_captured_and_written_right_before(ops):
    t, e, k, seqs = 600, 32, 4, 700
    cases = [case(t, e, k, seqs, i) for i in range(6)]
    cases = [(z.cuda(), ids.cuda(), cu.cuda()) for z, ids, cu, _ in cases]
    want = []
    for z, ids, cu in cases:
        want.append(ops.router_balance_loss(z, ids, cu_seqlens=cu))
        torch.cuda.synchronize()
    buffers = [torch.empty_like(x) for x in cases[0]]

    def all_cases():
        got = []
        for c in cases:
            for to, x in zip(buffers, c):
                to.copy_(x)
            got.append([x.clone() for x in ops.router_balance_loss(buffers[0], buffers[1], cu_seqlens=buffers[2])])
        return got

    for _ in range(10):
        for a, w in zip(all_cases(), want):
            assert all(torch.equal(x, y) for x, y in zip(a, w))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = all_cases()
    for _ in range(10):
        graph.replay()
    torch.cuda.synchronize()
    for a, w in zip(held, want):
        assert all(torch.equal(x, y) for x, y in zip(a, w))


@pytest.mark.parametrize("seqs", [0, 4])
def test_balanced_router_without_tokens(ops, seqs):
    # a rank that no token reaches takes part in the step all the same
    leaf = torch.empty((0, 32), device="cuda", requires_grad=True)
    cu = torch.zeros(seqs + 1, dtype=torch.int32, device="cuda") if seqs else None
    ids, weights, loss, counts = ops.router_topk_balanced(leaf, 4, cu_seqlens=cu, alpha=0.5)
    assert ids.shape == (0, 4) and ids.dtype == torch.int32 and weights.shape == (0, 4) and weights.dtype == torch.float32
    assert counts.shape == (max(seqs, 1), 32) and int(counts.abs().sum()) == 0 and float(loss.detach()) == 0
    (loss + weights.sum()).backward()
    assert leaf.grad.shape == (0, 32)
    for k in (0, 33):
        with pytest.raises(RuntimeError):
            ops.router_topk_balanced(leaf, k)


def test_transformations_without_a_rule_are_refused(ops):
    """Forward-mode derivatives and batched calls do not exist: they are refused, and nothing gets lost on the way."""
    z, ids, _, _ = case(12, 16, 3, 0, 1, masked=0.0)
    z, ids = z.cuda(), ids.cuda()
    ahead = torch.autograd.forward_ad
    loss = lambda x: ops.router_balance_loss(x, ids)[0]  # noqa: E731
    step = lambda x: ops.router_topk_balanced(x, 3)[2]  # noqa: E731
    for call in (loss, step):
        with ahead.dual_level():
            for x in (z, z.clone().requires_grad_()):
                with pytest.raises(RuntimeError):
                    call(ahead.make_dual(x, torch.ones_like(z)))
            with torch.no_grad(), pytest.raises(RuntimeError):
                call(ahead.make_dual(z, torch.ones_like(z)))
            assert torch.isfinite(call(z))                              # an ordinary tensor beside dual ones
        with pytest.raises(RuntimeError):
            torch.func.jvp(call, (z,), (torch.ones_like(z),))
        with pytest.raises(RuntimeError):
            torch.vmap(call)(torch.stack((z, z)))
    assert torch.isfinite(loss(z))


def test_padding_of_empty_sequences(ops):
    """cu_seqlens of a fixed length, its rest filled with the end of the last sequence and tokens behind that: same results, and
    nobody walks through the empty sequences one by one (of 65536, that took five hundred times as long as the kernel)."""
    t, e, k, used = 20000, 64, 4, 30
    z, ids, _, gw = case(t, e, k, 0, 9)
    z, ids = z.cuda(), ids.cuda()
    ends = torch.linspace(0, t - 37, used + 1).to(torch.int32)
    one = torch.ones((), device="cuda")
    results, times = [], []
    for seqs in (used, 65536):
        cu = torch.cat([ends[:12], ends[11].repeat((seqs - used) // 2), ends[12:], ends[-1].repeat(seqs - used - (seqs - used) // 2)]).cuda()
        assert cu.numel() == seqs + 1
        loss, counts, slope = ops.router_balance_loss(z, ids, cu_seqlens=cu)
        grad = ops.router_backward(z, ids, slope=slope, grad_loss=one, cu_seqlens=cu)
        results.append((loss, counts[counts.sum(1) > 0], slope[slope.sum(1) > 0], grad))
        spent = []
        for _ in range(7):
            begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            torch.cuda.synchronize()
            begin.record()
            for _ in range(10):
                ops.router_backward(z, ids, slope=slope, grad_loss=one, cu_seqlens=cu)
            end.record()
            torch.cuda.synchronize()
            spent.append(begin.elapsed_time(end))
        times.append(sorted(spent)[3])
    # chunks of tokens, and with them the order of the sums, go by the number of sequences: at most a unit of the loss
    assert abs(float(results[0][0]) - float(results[1][0])) <= 2.0 ** -23 * float(results[0][0])
    assert torch.equal(results[0][1], results[1][1]) and torch.equal(results[0][2], results[1][2])
    assert torch.equal(results[0][3], results[1][3])
    assert times[1] < 4 * times[0], times
