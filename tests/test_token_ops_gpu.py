"""The token operators (include/ebr_tokens.h, ebr_b200.token_ops) on the B200 against plain float64 implementations.

Tolerances, derived before any run. u is the unit roundoff of the output type (2^-24, 2^-11, 2^-8 for float32, float16,
bfloat16) and e = 2^-24 that of the float32 arithmetic:
* a lookup is one float32 product and one rounding: (u + 2 e) |ref|;
* a sum of m products in any order: (m + 2) e times the sum of the terms' magnitudes, and u |ref| for the rounding;
* a row's loss and gradient: the exponentials have relative error 2^-22 (ex2.approx) plus |x| e for their argument x, and
  the row's sum adds at most V / 32 terms in one lane and a tree of ten levels over the lanes: with arguments that count
  (x > -30, smaller terms are below 1e-9) a relative error r = 2^-22 + 30 e + (V / 32 + 10) e of every probability, and
  that much absolute error of every log q, beside |s - m| / tau * 2 e. The loss may be off by
  tau^2 (2 r + 4 e max |log terms|); a gradient element by |c| tau (2 r (q + p) + 4 e) + u |ref|, where float16 adds half its
  smallest subnormal number (2^-25).
"""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
TYPES = [torch.float32, torch.float16, torch.bfloat16]
U = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
TINY = {torch.float32: 0.0, torch.float16: 2.0**-25, torch.bfloat16: 0.0}
E = 2.0**-24


@pytest.fixture(autouse=True)
def _no_device_error():
    """No bounded wait of a kernel ran out during the test."""
    yield
    from ebr_b200 import _native

    _native.device_status()


def rand(*shape, seed=0, dtype=torch.float32):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(*shape, generator=g, device=DEV).to(dtype)


def randint(lo, hi, shape, seed=0, dtype=torch.int64):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randint(lo, hi, shape, generator=g, device=DEV).to(dtype)


def assert_within(got, ref, bound):
    off = (got.double() - ref).abs()
    assert bool((off <= bound).all()), f"off by {float((off - bound).max())} more than allowed"


# ---------------------------------------------------------------------------------------------------- embedding


def plain_embed(tokens, weight, scale):
    v = weight.shape[0]
    ok = (tokens >= 0) & (tokens < v)
    return weight.double()[torch.where(ok, tokens, 0).long()] * scale * ok.unsqueeze(-1)


def plain_embed_grad(tokens, g, scale, v):
    """(dW, sum of |terms|, terms) per table row in float64."""
    ok = (tokens >= 0) & (tokens < v)
    at = torch.where(ok, tokens, v).reshape(-1).long()
    g = g.double().reshape(-1, g.shape[-1])
    out = torch.zeros(v + 1, g.shape[1], device=DEV, dtype=torch.float64).index_add_(0, at, g)
    mag = torch.zeros_like(out).index_add_(0, at, g.abs())
    count = torch.bincount(at, minlength=v + 1).double().unsqueeze(1)
    return out[:v] * scale, mag[:v] * abs(scale), count[:v]


@pytest.mark.parametrize("wtype,otype", [(a, b) for a in TYPES for b in TYPES])
@pytest.mark.parametrize("n,v,c", [(1, 1, 1), (81, 10, 512), (200, 7, 3), (1000, 1023, 64), (1003, 1024, 771), (40, 5000, 2056)])
def test_embedding_lookup(n, v, c, wtype, otype):
    from ebr_b200.token_ops import scaled_embedding

    for idtype in (torch.int32, torch.int64):
        tokens = randint(-1, v + 1, (n,), seed=n, dtype=idtype)
        w = rand(v, c, seed=1, dtype=wtype)
        out = scaled_embedding(tokens, w, 1.7, otype)
        assert out.dtype == otype and out.shape == (n, c)
        ref = plain_embed(tokens, w, 1.7)
        assert_within(out, ref, (U[otype] + 2 * E) * ref.abs() + TINY[otype])


@pytest.mark.parametrize("gtype,wtype", [(a, b) for a in TYPES for b in TYPES])
@pytest.mark.parametrize("n,v,c", [(1, 1, 1), (81, 10, 512), (128, 2, 33), (512, 3, 520), (513, 3, 520), (100, 3001, 771), (129, 3001, 771), (3000, 2, 33), (1000, 1023, 64), (1003, 1024, 771),
                                   (6000, 5000, 72)])
def test_embedding_gradient(n, v, c, gtype, wtype):
    from ebr_b200.token_ops import scaled_embedding

    tokens = randint(-1, v + 1, (n,), seed=n)
    w = rand(v, c, seed=1, dtype=wtype).requires_grad_(True)
    g = rand(n, c, seed=2, dtype=gtype)
    dw = [torch.autograd.grad(scaled_embedding(tokens, w, 0.3, gtype), w, g)[0] for _ in range(2)]
    assert dw[0].dtype == wtype and torch.equal(dw[0], dw[1])  # the same bits each time
    ref, mag, count = plain_embed_grad(tokens, g, 0.3, v)
    assert_within(dw[0], ref, (count + 2) * E * mag + U[wtype] * ref.abs() + TINY[wtype])


@pytest.mark.parametrize("n,v,c,kind", [
    (62208, 10, 512, "skew"),      # runs of thousands of tokens, one of them most of the batch: the whole-block join
    (40000, 3, 130, "one"),        # a single run over every chunk
    (33000, 3000, 40, "even"),     # the whole-GPU sort, two passes
    (70000, 1 << 17, 24, "even"),  # a table of 6 MB that is zeroed beside the sort
    (20000, 1 << 20, 24, "even"),  # one of 100 MB: the cluster sort, three digits
    (300000, 9, 16, "even"),       # more tokens than a cluster sorts
    (600000, 40000, 8, "even"),    # more tiles than the placing blocks add up themselves
    (5000, 4, 64, "padding"),      # nothing but padding ids
])  # fmt: skip
def test_embedding_gradient_sort_paths(n, v, c, kind):
    from ebr_b200.token_ops import scaled_embedding

    if kind == "skew":
        tokens = torch.where(rand(n, seed=3) < 0.5, 0, randint(0, v, (n,), seed=4))
    elif kind == "one":
        tokens = torch.full((n,), 1, device=DEV)
    elif kind == "padding":
        tokens = torch.where(rand(n, seed=3) < 0, -1, v + 5)
    else:
        tokens = randint(-1, v + 1, (n,), seed=4)
    w = torch.zeros(v, c, device=DEV, requires_grad=True)
    g = rand(n, c, seed=5, dtype=torch.bfloat16)
    (dw,) = torch.autograd.grad(scaled_embedding(tokens, w, 2.0, torch.bfloat16), w, g)
    ref, mag, count = plain_embed_grad(tokens, g, 2.0, v)
    assert_within(dw, ref, (count + 2) * E * mag + U[torch.float32] * ref.abs())


def test_embedding_gradient_of_a_large_table_replays_as_a_cuda_graph():
    """The zeroing that runs beside the sort keeps its order in a graph: other tokens, the same buffers, several replays."""
    from ebr_b200.token_ops import scaled_embedding

    v, c, n = 1 << 20, 24, 20000
    tokens, g = randint(-1, v, (n,), seed=1), rand(n, c, seed=2)
    w = torch.zeros(v, c, device=DEV, requires_grad=True)

    def step():
        return torch.autograd.grad(scaled_embedding(tokens, w), w, g)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dw = step()
    for seed in (3, 4, 5):
        tokens.copy_(randint(-1, v, (n,), seed=seed))
        graph.replay()
        assert torch.equal(dw, step())


def test_embedding_ids_far_outside_the_table_and_empty_inputs():
    from ebr_b200.token_ops import scaled_embedding

    w = rand(10, 16).requires_grad_(True)
    tokens = torch.tensor([[-(2**40), 3, 2**40], [2**31, 9, -1]], device=DEV)  # ids that would wrap to small ones too
    out = scaled_embedding(tokens, w, 2.0)
    assert out.shape == (2, 3, 16)
    assert torch.equal(out[0, 1], w.detach()[3] * 2) and torch.equal(out[1, 1], w.detach()[9] * 2)
    assert not out[0, 0].any() and not out[0, 2].any() and not out[1, 0].any() and not out[1, 2].any()
    (dw,) = torch.autograd.grad(out, w, torch.ones_like(out))
    expect = torch.zeros_like(dw)
    expect[3] = expect[9] = 2
    assert torch.equal(dw, expect)
    empty = scaled_embedding(torch.empty(0, 5, dtype=torch.int64, device=DEV), w)
    assert empty.shape == (0, 5, 16)
    (dw,) = torch.autograd.grad(empty, w, torch.empty_like(empty))
    assert not dw.any()


def test_embedding_strided_inputs_and_non_finite_rows():
    from ebr_b200.token_ops import scaled_embedding

    big = rand(12, 40, seed=6)
    w = big[:, 3:35]  # row stride 40, first element not on a 16-byte boundary
    tokens = randint(0, 12, (9, 6), seed=7)
    out = scaled_embedding(tokens.t(), w, 1.0)
    assert torch.equal(out, w[tokens.t()])
    ww = w.detach().clone().requires_grad_(True)
    g = rand(32, 6, 9, seed=8).permute(1, 2, 0)  # a transposed upstream gradient
    (dw,) = torch.autograd.grad(scaled_embedding(tokens.t(), ww), ww, g)
    ref, mag, count = plain_embed_grad(tokens.t().reshape(-1), g.reshape(54, 32), 1.0, 12)
    assert_within(dw, ref, (count + 2) * E * mag + E * ref.abs())
    g2 = torch.ones(3, 4, device=DEV)
    g2[1] = float("nan")
    w3 = torch.zeros(5, 4, device=DEV, requires_grad=True)
    (dw,) = torch.autograd.grad(scaled_embedding(torch.tensor([1, 2, 4], device=DEV), w3), w3, g2)
    assert dw[2].isnan().all() and not dw[[0, 1, 3, 4]].isnan().any()
    (dw,) = torch.autograd.grad(scaled_embedding(torch.tensor([1, -1, 4], device=DEV), w3), w3, g2)
    assert not dw.isnan().any()  # a padding id's gradient goes nowhere


def test_embedding_is_differentiable_twice_and_by_differences():
    from ebr_b200.token_ops import scaled_embedding

    tokens = randint(-1, 6, (50,), seed=9)
    w = rand(6, 8, seed=10).requires_grad_(True)
    g = rand(50, 8, seed=11).requires_grad_(True)
    (dw,) = torch.autograd.grad(scaled_embedding(tokens, w, 1.5), w, g, create_graph=True)
    t = rand(6, 8, seed=12)
    (gg,) = torch.autograd.grad(dw, g, t)
    assert_within(gg, plain_embed(tokens, t, 1.5), 4 * E * plain_embed(tokens, t, 1.5).abs())
    # linear in w: a central difference is exact up to rounding, whatever the step
    with torch.no_grad():
        f = lambda a: (scaled_embedding(tokens, a, 1.5).double() * g.double()).sum()  # noqa: E731
        diff = (f(w + 2 * t) - f(w - 2 * t)) / 4
        scale = (plain_embed(tokens, w.abs() + 2 * t.abs(), 1.5) * g.abs()).sum()
    assert abs(float(diff) - (dw.detach().double() * t).sum().item()) <= float(100 * E * scale)


def test_embedding_offsets_past_32_bits():
    """A table of 2.3e9 elements: the last rows and their gradient."""
    from ebr_b200.token_ops import scaled_embedding

    v, c = (1 << 21) + 77, 1100
    w = torch.zeros(v, c, device=DEV, dtype=torch.bfloat16)
    w[-1], w[v - 50] = 3.0, 5.0
    w.requires_grad_(True)
    tokens = torch.tensor([v - 1, 0, v - 50, v - 1], device=DEV)
    out = scaled_embedding(tokens, w)
    assert out[:, 0].tolist() == [3.0, 0.0, 5.0, 3.0] and out[:, -1].tolist() == [3.0, 0.0, 5.0, 3.0]
    (dw,) = torch.autograd.grad(out, w, torch.ones_like(out))
    assert dw[v - 1].eq(2).all() and dw[v - 50].eq(1).all() and dw[0].eq(1).all()
    assert float(dw.float().sum()) == 4 * c


def test_embedding_refusals():
    from ebr_b200.token_ops import scaled_embedding

    w, t = rand(4, 8), torch.zeros(3, dtype=torch.int64, device=DEV)
    with pytest.raises(RuntimeError, match="only on CUDA"):
        scaled_embedding(t, w.cpu())
    with pytest.raises(RuntimeError, match="only on CUDA"):
        scaled_embedding(t.cpu(), w)
    with pytest.raises(TypeError):
        scaled_embedding(t, w.double())
    with pytest.raises(TypeError):
        scaled_embedding(t.float(), w)
    with pytest.raises(TypeError):
        scaled_embedding(t, w, 1.0, torch.float64)
    with pytest.raises(ValueError):
        scaled_embedding(t, w[0])


# ---------------------------------------------------------------------------------------------------- experts


def plain_route(ids, experts, capacity):
    """(row_of, slot_of, offsets) from the definition, one expert after another, on the host."""
    flat = ids.reshape(-1).cpu()
    n = flat.numel()
    rows = n if capacity is None else experts * capacity
    row_of, slot_of, offsets = torch.full((n,), -1), torch.full((rows,), -1), [0]
    for e in range(experts):
        mine = (flat == e).nonzero().squeeze(1)
        kept = mine if capacity is None else mine[:capacity]
        at = torch.arange(len(kept)) + (offsets[-1] if capacity is None else e * capacity)
        row_of[kept] = at
        slot_of[at] = kept
        offsets.append(offsets[-1] + len(mine))
    return row_of.view(ids.shape), slot_of, torch.tensor(offsets)


@pytest.mark.parametrize("idtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("t,k,e,capacity", [
    (1, 1, 1, None), (81, 2, 8, None), (81, 2, 8, 7), (0, 2, 5, None), (0, 2, 5, 3), (50, 33, 60, None), (700, 3, 1024, 2),
    (2049, 8, 1000, None), (17000, 2, 60, 400), (40000, 2, 7, None), (530000, 1, 33, None),
])  # fmt: skip
def test_expert_route(t, k, e, capacity, idtype):
    from ebr_b200.token_ops import expert_route

    ids = randint(-1, e + 1, (t, k), seed=t + k, dtype=idtype)
    r = expert_route(ids, e, capacity)
    row_of, slot_of, offsets = plain_route(ids, e, capacity)
    assert torch.equal(r.row_of.cpu().long(), row_of)
    assert torch.equal(r.slot_of.cpu().long(), slot_of)
    assert torch.equal(r.offsets.cpu().long(), offsets)
    assert r.rows == slot_of.numel() and r.top_k == k


@pytest.mark.parametrize("ids", ["one expert", "none valid"])
@pytest.mark.parametrize("capacity", [None, 5])
def test_expert_route_of_one_expert_and_of_none(ids, capacity):
    from ebr_b200.token_ops import expert_combine, expert_dispatch, expert_route

    choice = torch.full((33, 2), 3 if ids == "one expert" else -7, device=DEV)
    r = expert_route(choice, 4, capacity)
    for got, ref in zip((r.row_of, r.slot_of, r.offsets), plain_route(choice, 4, capacity)):
        assert torch.equal(got.cpu().long(), ref)
    x = rand(33, 24)
    rows = expert_dispatch(x, r)
    live = r.slot_of >= 0
    assert not rows[~live].any() and torch.equal(rows[live], x[(r.slot_of[live] // 2).long()])
    y = expert_combine(torch.full((r.rows, 24), float("nan"), device=DEV), r)
    dropped = (r.row_of < 0).all(1)
    assert not y[dropped].any() and y[~dropped].isnan().all()


def plain_dispatch(x, r, w=None):
    out = torch.zeros(r.rows, x.shape[-1], device=DEV, dtype=torch.float64)
    live = r.slot_of >= 0
    slot = r.slot_of[live].long()
    rows = x.double().reshape(-1, x.shape[-1])[slot // r.top_k]
    out[live] = rows if w is None else rows * w.double().reshape(-1)[slot].unsqueeze(1)
    return out


def plain_combine(rows, r, w=None):
    """(y, sum of |terms|)"""
    ok = (r.row_of >= 0).reshape(-1)
    got = rows.double()[r.row_of.reshape(-1).clamp(min=0).long()] * ok.unsqueeze(1)
    if w is not None:
        got = got * torch.where(ok, w.double().reshape(-1), 0).unsqueeze(1)
    got = got.view(*r.row_of.shape, -1)
    return got.sum(-2), got.abs().sum(-2)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("t,k,e,c,capacity", [
    (1, 1, 1, 1, None), (81, 2, 8, 512, None), (60, 3, 5, 999, 20), (40, 33, 50, 100, None), (37, 2, 4, 6, 30),
    (300, 4, 9, 2056, None), (2500, 2, 6, 64, 700),
])  # fmt: skip
def test_expert_dispatch_and_combine(t, k, e, c, capacity, dtype):
    from ebr_b200.token_ops import expert_combine, expert_dispatch, expert_route

    r = expert_route(randint(-1, e, (t, k), seed=t), e, capacity)
    x = rand(t, c, seed=1, dtype=dtype).requires_grad_(True)
    rows = rand(r.rows, c, seed=2, dtype=dtype).requires_grad_(True)
    gx, gy = rand(r.rows, c, seed=3, dtype=dtype), rand(t, c, seed=4, dtype=dtype)
    sent = expert_dispatch(x, r)
    assert torch.equal(sent.double(), plain_dispatch(x, r))
    for wtype in {torch.float32, dtype}:
        w = rand(t, k, seed=5, dtype=wtype).requires_grad_(True)
        y = expert_combine(rows, r, w)
        ref, mag = plain_combine(rows, r, w)
        assert_within(y, ref, (k + 2) * E * mag + U[dtype] * ref.abs() + TINY[dtype])
        dx, drows, dw = torch.autograd.grad([sent, y], [x, rows, w], [gx, gy], retain_graph=True)
        ref, mag = plain_combine(gx, r)
        assert_within(dx, ref, (k + 2) * E * mag + U[dtype] * ref.abs() + TINY[dtype])
        ref = plain_dispatch(gy, r, w)
        assert_within(drows, ref, (U[dtype] + 2 * E) * ref.abs() + TINY[dtype])
        terms = rows.double()[r.row_of.clamp(min=0).long()] * gy.double().unsqueeze(1) * (r.row_of >= 0).unsqueeze(-1)
        ref, mag = terms.sum(-1), terms.abs().sum(-1)
        assert dw.dtype == wtype
        assert_within(dw, ref, (c + 2) * E * mag + U[wtype] * ref.abs() + TINY[wtype])


def test_expert_dropped_slots_take_nothing_and_give_nothing():
    from ebr_b200.token_ops import expert_combine, expert_dispatch, expert_route

    ids = torch.tensor([[0, 1], [0, -1], [0, 1]], device=DEV)
    r = expert_route(ids, 2, capacity=1)  # token 0 keeps both; the others lose everything
    assert r.row_of.tolist() == [[0, 1], [-1, -1], [-1, -1]]
    w = torch.tensor([[0.5, 2.0], [float("nan"), float("inf")], [float("nan"), 1.0]], device=DEV, requires_grad=True)
    rows = torch.ones(2, 8, device=DEV, requires_grad=True)
    y = expert_combine(rows, r, w)
    assert y[0].eq(2.5).all() and not y[1:].any()
    g = torch.full((3, 8), float("inf"), device=DEV)
    g[0] = 1
    drows, dw = torch.autograd.grad(y, [rows, w], g)
    assert drows[0].eq(0.5).all() and drows[1].eq(2).all()
    assert dw.tolist() == [[8, 8], [0, 0], [0, 0]]
    x = torch.tensor([[1.0], [float("nan")], [3.0]], device=DEV)
    assert expert_dispatch(x, r).tolist() == [[1.0], [1.0]]


def test_expert_strides_leading_shapes_and_streams():
    from ebr_b200.token_ops import expert_combine, expert_dispatch, expert_route

    ids = randint(0, 5, (4, 6, 3), seed=1)
    r = expert_route(ids.transpose(0, 1), 5)  # [6, 4, 3], not contiguous
    x = rand(24, 70, seed=2)[:, 5:69]  # row stride 70
    flat = expert_route(ids.transpose(0, 1).reshape(24, 3), 5)
    assert torch.equal(expert_dispatch(x, flat).double(), plain_dispatch(x, flat))
    xs = x.reshape(6, 4, 64)
    assert torch.equal(expert_dispatch(xs, r), expert_dispatch(x, flat))
    rows = rand(72, 80, seed=3)[:, 8:72]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = expert_combine(rows, r)
    torch.cuda.current_stream().wait_stream(side)
    assert y.shape == (6, 4, 64)
    assert torch.equal(y, expert_combine(rows.contiguous(), r))


def test_expert_second_order_matches_plain_autograd():
    """d<dE/dx, u> for E = sum of (combine of squared dispatched rows), against the same built from indexing in float64."""
    from ebr_b200.token_ops import expert_combine, expert_dispatch, expert_route

    t, k, e, c = 19, 3, 5, 12
    r = expert_route(randint(-1, e, (t, k), seed=3), e)
    x0, w0, u = rand(t, c, seed=4), rand(t, k, seed=5), rand(t, c, seed=6)

    def hess(x, w, u, dispatch, combine):
        y = combine(dispatch(x).tanh(), w)
        (g,) = torch.autograd.grad((y * y).sum(), x, create_graph=True)
        return torch.autograd.grad((g * u).sum(), [x, w])

    got = hess(x0.clone().requires_grad_(True), w0.clone().requires_grad_(True), u,
               lambda x: expert_dispatch(x, r), lambda rows, w: expert_combine(rows, r, w))  # fmt: skip
    live, at = (r.row_of >= 0), r.row_of.clamp(min=0).long()
    tok = (r.slot_of.clamp(min=0) // k).long()
    ref = hess(x0.double().requires_grad_(True), w0.double().requires_grad_(True), u.double(),
               lambda x: x[tok] * (r.slot_of >= 0).unsqueeze(1),
               lambda rows, w: (rows[at] * (w * live).unsqueeze(-1)).sum(1))  # fmt: skip
    for a, b in zip(got, ref):  # some hundred float32 operations of order one to ten: 2e-5 of the largest
        assert float((a.double() - b).abs().max()) <= 2e-5 * float(b.abs().max())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("capacity", [None, 9])
def test_expert_second_order_of_each_type_with_dropped_slots(dtype, capacity):
    """The derivatives of <d rows, a> + <d w, b> + <d x, d>, where d rows, d w and d x are the gradients of the combine and
    the dispatch: products and sums over slots again, one rounding each and one for a sum of two."""
    from ebr_b200.token_ops import expert_combine, expert_dispatch, expert_route

    t, k, e, c = 40, 3, 7, 72
    r = expert_route(randint(-1, e, (t, k), seed=3), e, capacity)
    assert bool((r.row_of < 0).any())
    live = (r.row_of >= 0).unsqueeze(-1)
    for wtype in {torch.float32, dtype}:
        rows, gy, a = rand(r.rows, c, seed=1, dtype=dtype), rand(t, c, seed=2, dtype=dtype), rand(r.rows, c, seed=4, dtype=dtype)
        w, b = rand(t, k, seed=5, dtype=wtype), rand(t, k, seed=6, dtype=wtype)
        rows, gy, w = (v.requires_grad_(True) for v in (rows, gy, w))
        grows, gw = torch.autograd.grad(expert_combine(rows, r, w), [rows, w], gy, create_graph=True)
        drows, dw, dgy = torch.autograd.grad([grows, gw], [rows, w, gy], [a, b])
        assert drows.dtype == dgy.dtype == dtype and dw.dtype == wtype
        slack = 2 * E + U[dtype]
        ref = plain_dispatch(gy.detach(), r, b)
        assert_within(drows, ref, slack * ref.abs() + TINY[dtype])
        terms = a.double()[r.row_of.clamp(min=0).long()] * gy.detach().double().unsqueeze(1) * live
        assert_within(dw, terms.sum(-1), (c + 2) * E * terms.abs().sum(-1) + U[wtype] * terms.sum(-1).abs() + TINY[wtype])
        (one, m1), (two, m2) = plain_combine(a, r, w.detach()), plain_combine(rows.detach(), r, b)
        bound = (k + 2) * E * (m1 + m2) + U[dtype] * (one.abs() + two.abs() + (1 + U[dtype]) * (one + two).abs()) * 1.01
        assert_within(dgy, one + two, bound + 3 * TINY[dtype])
        x, gs = rand(t, c, seed=7, dtype=dtype).requires_grad_(True), rand(r.rows, c, seed=8, dtype=dtype).requires_grad_(True)
        d = rand(t, c, seed=9, dtype=dtype)
        (gx,) = torch.autograd.grad(expert_dispatch(x, r), x, gs, create_graph=True)
        assert torch.equal(torch.autograd.grad(gx, gs, d)[0].double(), plain_dispatch(d, r))


def test_expert_gradients_by_differences():
    """The combine is bilinear: central differences are exact up to rounding, whatever the step."""
    from ebr_b200.token_ops import expert_combine, expert_route

    t, k, e, c = 30, 2, 4, 16
    r = expert_route(randint(-1, e, (t, k), seed=3), e, 14)
    rows, w, g = rand(r.rows, c, seed=4), rand(t, k, seed=5), rand(t, c, seed=6)
    rr, ww = rows.clone().requires_grad_(True), w.clone().requires_grad_(True)
    drows, dw = torch.autograd.grad(expert_combine(rr, r, ww), [rr, ww], g)
    a, b = rand(r.rows, c, seed=7), rand(t, k, seed=8)
    f = lambda p, q: float((expert_combine(p, r, q).double() * g).sum())  # noqa: E731
    scale = float((plain_combine(rows.abs() + a.abs(), r, w.abs() + b.abs())[0] * g.abs()).sum())
    assert abs((f(rows + a, w) - f(rows - a, w)) / 2 - float((drows.double() * a).sum())) <= 50 * E * scale
    assert abs((f(rows, w + b) - f(rows, w - b)) / 2 - float((dw.double() * b).sum())) <= 50 * E * scale


def test_expert_layer_replays_as_a_cuda_graph():
    from ebr_b200.token_ops import expert_combine, expert_dispatch, expert_route

    ids, x = randint(0, 6, (200, 2), seed=1), rand(200, 64, seed=2)

    def layer():
        r = expert_route(ids, 6, 50)
        return expert_combine(expert_dispatch(x, r) * 2, r)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer()
    for seed in (5, 6):
        ids.copy_(randint(0, 6, (200, 2), seed=seed))
        x.copy_(rand(200, 64, seed=seed))
        graph.replay()
        assert torch.equal(out, layer())


def test_expert_route_from_several_threads():
    """Routes of different numbers of experts (of the sort's shared memory, that is) from threads of their own."""
    import threading

    from ebr_b200.token_ops import expert_route

    failures = []

    def work(experts):
        try:
            ids = randint(0, experts, (40000, 1), seed=experts)
            with torch.cuda.stream(torch.cuda.Stream()):
                first = expert_route(ids, experts)
                for _ in range(6000):
                    last = expert_route(ids, experts)
                if not (torch.equal(first.row_of, last.row_of) and torch.equal(first.offsets, last.offsets)):
                    failures.append(f"{experts} experts: another route")
        except Exception as e:  # noqa: BLE001
            failures.append(f"{experts} experts: {e}")

    threads = [threading.Thread(target=work, args=(e,)) for e in (1024, 700, 1000, 800)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures, failures


def test_expert_refusals():
    from ebr_b200.token_ops import expert_combine, expert_dispatch, expert_route

    ids = torch.zeros(4, 2, dtype=torch.int64, device=DEV)
    for bad in (0, 1025):
        with pytest.raises(ValueError):
            expert_route(ids, bad)
    with pytest.raises(ValueError):
        expert_route(ids, 4, 0)
    with pytest.raises(TypeError):
        expert_route(ids.float(), 4)
    with pytest.raises(RuntimeError, match="only on CUDA"):
        expert_route(ids.cpu(), 4)
    r = expert_route(ids, 4)
    with pytest.raises(ValueError):
        expert_dispatch(rand(5, 8), r)
    with pytest.raises(TypeError):
        expert_dispatch(rand(4, 8).double(), r)
    with pytest.raises(ValueError):
        expert_combine(rand(7, 8), r)
    with pytest.raises(ValueError):
        expert_combine(rand(8, 8), r, rand(4, 3))


# ---------------------------------------------------------------------------------------------------- distillation


def plain_distill(logits, ids, top, tau, weight=None):
    """(rows' losses, d loss / d logits per row, q, mass, largest |log term|) in float64."""
    v = logits.shape[-1]
    s, t = logits.double() / tau, top.double() / tau
    ok = (ids >= 0) & (ids < v)
    t = torch.where(ok, t, -math.inf)
    counts = (t > -math.inf).any(-1)
    if weight is not None:
        counts = counts & (weight != 0)
    s = torch.where(counts.unsqueeze(-1), s, 0.0)
    t = torch.where(counts.unsqueeze(-1), t, 0.0)
    logp, logq = torch.log_softmax(t, -1), torch.log_softmax(s, -1)
    p = logp.exp() * counts.unsqueeze(-1) * ok
    at = torch.where(ok, ids, 0).long()
    mine = logq.gather(-1, at)
    terms = torch.where(p > 0, p * (logp - mine), 0.0)
    q = logq.exp() * counts.unsqueeze(-1)
    mass = torch.zeros_like(q).scatter_add_(-1, at, p)
    w = torch.ones_like(q[..., 0]) if weight is None else torch.where(counts, weight.double(), 0.0)
    used = torch.where((p > 0) & torch.isfinite(mine), mine.abs() + logp.abs(), 0.0)
    return w * tau**2 * terms.sum(-1), w.unsqueeze(-1) * tau * (q - mass), q, mass, float(used.max()) if used.numel() else 0.0


def relative(v):
    return 2.0**-22 + 30 * E + (v / 32 + 10) * E


def check_distill(logits, ids, top, tau, weight=None):
    from ebr_b200.token_ops import topk_distill_loss

    v, dtype = logits.shape[-1], logits.dtype
    r = relative(v)
    ref, grad, q, mass, largest = plain_distill(logits, ids, top, tau, weight)
    w = 1.0 if weight is None else weight.abs().double()
    bound = w * tau**2 * (2 * r + 4 * E * (1 + largest))
    x = logits.detach().requires_grad_(True)
    rows = topk_distill_loss(x, ids, top, tau, row_weight=weight, reduction="none")
    assert rows.dtype == torch.float32 and rows.shape == logits.shape[:-1]
    finite = torch.isfinite(ref)
    assert torch.equal(torch.isfinite(rows), finite)
    assert_within(rows[finite], ref[finite], (bound + E * ref.abs())[finite])
    up = torch.rand(rows.shape, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV) + 0.5

    def within(got, c):
        c = torch.as_tensor(c, dtype=torch.float64, device=DEV).expand(rows.shape).unsqueeze(-1)
        ww = 1.0 if weight is None else weight.abs().double().unsqueeze(-1)
        assert got.dtype == dtype and got.shape == logits.shape
        assert_within(got, c * grad, c * ww * tau * (2 * r * (q + mass) + 4 * E * (q + mass)) + U[dtype] * (c * grad).abs()
                      + TINY[dtype] + 1e-38)  # fmt: skip

    within(torch.autograd.grad(rows, x, up)[0], up)
    n = rows.numel()
    for how, c in (("sum", 1.0), ("mean", 1.0 / max(n, 1))):
        total = topk_distill_loss(x, ids, top, tau, row_weight=weight, reduction=how)
        if bool(finite.all()):
            off = c * float((bound + E * ref.abs()).sum()) if n else 0.0
            assert abs(total.item() - c * float(ref.sum())) <= off + (n / 32 + 40) * E * c * float(ref.abs().sum()) + 1e-30
        first = torch.autograd.grad(total, x, retain_graph=True)[0]
        within(first, c)
        kept = first.clone()
        within(torch.autograd.grad(total, x, torch.tensor(0.37, device=DEV), retain_graph=True)[0], 0.37 * c)
        assert torch.equal(first, kept)  # a later backward has a gradient of its own
        again = topk_distill_loss(x, ids, top, tau, row_weight=weight, reduction=how)
        within(torch.autograd.grad(again * 3, x)[0], 3 * c)  # the first backward, an upstream that is not 1
    with torch.no_grad():
        assert torch.equal(topk_distill_loss(x, ids, top, tau, row_weight=weight, reduction="none"), rows.detach())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,v,k", [
    (1, 1, 1), (3, 2, 1), (81, 10, 4), (65, 32, 32), (9, 33, 5), (50, 10, 40), (20, 1000, 64), (7, 4099, 300), (5, 8192, 17),
    (4, 9001, 1024), (260, 15003, 9), (130, 20011, 8), (3, 50021, 20), (300, 33000, 3), (2, 131073, 64), (310, 70001, 5),
])  # fmt: skip
def test_distillation_against_float64(n, v, k, dtype):
    """Every kernel: four lanes a row, a warp, rings of both sizes, one CTA a row and clusters of up to 16."""
    ids = randint(-1, v, (n, k), seed=n)  # repeated ids wherever k is not far below v, and rows cut short
    logits = rand(n, v, seed=1) * 3
    logits.scatter_add_(1, ids.clamp(min=0), rand(n, k, seed=2).abs())
    check_distill(logits.to(dtype), ids, (rand(n, k, seed=3) * 2 + 3).to(dtype), 1.7)


@pytest.mark.parametrize("n,v,dtype", [
    (2700, 17000, torch.bfloat16),  # rings of 8 KB chunks, 888 CTAs: three and four rows each
    (900, 70001, torch.bfloat16),   # rings of 24 KB chunks, 296 CTAs: three and four rows each
    (200, 131073, torch.float32),   # clusters of two, 148 of them: a second row for some
])  # fmt: skip
def test_distillation_of_several_rows_to_a_ring(n, v, dtype):
    """Rows that do not count among those that do: the first of a CTA, several in a row, the last; and the others' values."""
    ids, top = randint(-1, v, (n, 6), seed=1), rand(n, 6, seed=2)
    logits = (rand(n, v, seed=3) * 2).to(dtype)
    weight = rand(n, seed=4).abs() + 0.25
    ids[[0, 1, 2, 148, 149, 297, n - 1] if n > 297 else [0, 1, 2, 148, 149, n - 1]] = -1
    weight[[1, 3, 4, 150, 151, n // 2, n - 2]] = 0
    logits[[0, 3, 150]] = math.nan
    check_distill(logits, ids, top, 1.3, weight)


def test_distillation_of_long_rows_repeats_bit_for_bit_on_another_stream():
    from ebr_b200.token_ops import topk_distill_loss

    for n, v in ((1000, 33000), (400, 70001)):
        x = rand(n, v, seed=1, dtype=torch.bfloat16).requires_grad_(True)
        ids, top = randint(-1, v, (n, 12), seed=2), rand(n, 12, seed=3)
        a = topk_distill_loss(x, ids, top)
        (ga,) = torch.autograd.grad(a, x)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            b = topk_distill_loss(x, ids, top)
            (gb,) = torch.autograd.grad(b, x)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(a, b) and torch.equal(ga, gb)


@pytest.mark.parametrize("v", [10, 700, 20000, 70000])
def test_distillation_masks(v):
    """Vocabulary masks of -inf and of the lowest value, rows that are all the lowest value, rows and weights that leave
    nothing, NaN and infinities in rows that do not count, entries of -inf, huge entries."""
    n, k = 12, 3
    ids, top = randint(0, v // 2, (n, k), seed=1, dtype=torch.int32), rand(n, k, seed=2)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        x = (rand(n, v, seed=3) * 2).to(dtype)
        x[:, v // 2 :] = -math.inf
        x[1, v // 2 :] = torch.finfo(dtype).min
        x[2] = torch.finfo(dtype).min
        x[3] = math.nan
        x[4] = -math.inf
        x[5, 0] = math.inf
        i, t = ids.clone(), top.clone()
        i[3:6] = -1  # rows without entries: whatever they hold
        i[6, 1:] = v + 3
        t[7, 0] = -math.inf
        t[8] = 1e30
        weight = torch.ones(n, device=DEV)
        weight[9] = 0
        x[9, 1] = math.nan
        weight[10] = -2.5
        check_distill(x, i, t, 1.3, weight)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("tau,share", [(1e-37, 1.0), (1e-30, 1.0), (1e-12, 1.0), (2.5e19, 0.01), (1e21, 1e-6)])
@pytest.mark.parametrize("n,v,k", [(4, 10, 9), (4, 700, 60), (4, 40001, 900)])
def test_distillation_at_extreme_temperatures(n, v, k, tau, share, dtype):
    """Losses that float32 holds, at temperatures whose square or inverse it does not. Beside the tolerances above, the
    rounding of the temperature and of the products with it and with the weight: 16 e of the loss, 8 e of the gradient."""
    from ebr_b200.token_ops import topk_distill_loss

    logits, ids, top = (rand(n, v, seed=1) * 3).to(dtype), randint(0, v, (n, k), seed=2), rand(n, k, seed=3)
    weight = torch.full((n,), share, device=DEV)
    ref, grad, q, mass, largest = plain_distill(logits, ids, top, tau, weight)
    assert float(ref.abs().max()) < 3e38
    r = relative(v)
    x = logits.clone().requires_grad_(True)
    rows = topk_distill_loss(x, ids, top, tau, row_weight=weight, reduction="none")
    assert_within(rows, ref, share * tau**2 * (2 * r + 4 * E * (1 + largest)) + 16 * E * ref.abs() + 1e-44)
    bound = share * tau * (2 * r + 4 * E) * (q + mass) + (U[dtype] + 8 * E) * grad.abs() + 1e-38
    assert_within(torch.autograd.grad(rows, x, torch.ones_like(rows))[0], grad, bound)
    total = topk_distill_loss(x, ids, top, tau, row_weight=weight)
    assert_within(torch.autograd.grad(total, x)[0], grad / n, bound / n + 1e-38)


@pytest.mark.parametrize("n,v", [(9, 10), (9, 700), (9, 40001), (900, 33001)])
def test_distillation_of_a_teacher_that_is_masked_out(n, v):
    """Entries of -inf alone are no entries: loss 0 and gradient 0, even of NaN logits; the other rows do not notice."""
    x, ids, top = rand(n, v, seed=1), randint(0, v, (n, 3), seed=2), rand(n, 3, seed=3)
    top[[0, 4, 5, n - 1]] = -math.inf
    ids[5, 1] = -1
    x[4] = math.nan
    check_distill(x.to(torch.bfloat16), ids, top, 1.4)


def test_distillation_of_an_entry_at_the_lowest_value():
    """A masked logit that the teacher names: tau p 3.4e38, which float32 holds at tau = 0.5."""
    from ebr_b200.token_ops import topk_distill_loss

    for dtype in (torch.float32, torch.bfloat16):
        for v in (12, 600, 40000):
            x = rand(3, v, seed=1).to(dtype)
            x[1, 5] = torch.finfo(dtype).min
            x.requires_grad_(True)
            ids, top = torch.tensor([[5, 6]] * 3, device=DEV), torch.zeros(3, 2, device=DEV)
            ref, grad, *_ = plain_distill(x.detach(), ids, top, 0.5)
            rows = topk_distill_loss(x, ids, top, 0.5, reduction="none")
            assert float(ref[1]) > 8e37 and abs(float(rows.detach()[1]) / float(ref[1]) - 1) < 1e-5
            (g,) = torch.autograd.grad(rows, x, torch.ones_like(rows))
            assert float((g.double() - grad).abs().max()) <= 2 * U[dtype] + 1e-5


def test_distillation_of_a_masked_entry_and_non_finite_rows():
    from ebr_b200.token_ops import topk_distill_loss

    for v in (12, 600, 30000):
        x = rand(4, v, seed=1)
        x[0, 5] = -math.inf  # the student gives the teacher's entry nothing: an infinite loss, a finite gradient
        x[1, 3] = math.nan
        x[2] = -math.inf
        x.requires_grad_(True)
        ids = torch.tensor([[5, 6]] * 4, device=DEV)
        rows = topk_distill_loss(x, ids, torch.zeros(4, 2, device=DEV), reduction="none")
        assert math.isinf(rows[0]) and math.isnan(rows[1]) and math.isnan(rows[2]) and math.isfinite(rows[3])
        (g,) = torch.autograd.grad(rows, x, torch.ones_like(rows))
        assert g[0].isfinite().all() and abs(float(g[0, 5]) + 0.5) < 1e-5
        assert g[1].isnan().all() and g[2].isnan().all() and g[3].isfinite().all()


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("n,v,k", [(70, 20, 5), (70, 10, 40), (300, 700, 5), (6, 40001, 5), (6, 40001, 70), (900, 33001, 5)])
def test_distillation_of_a_non_finite_teacher_beside_padding(n, v, k, bad):
    """A teacher's logit of NaN or infinity makes its own row's loss NaN, and the gradient of the logits that the row
    names; padding entries of the same row name nothing and are read nowhere. Every kernel; the logits are an interior view."""
    from ebr_b200.token_ops import topk_distill_loss

    full = rand(n + 2, v + 16, seed=1, dtype=torch.bfloat16)
    ids, good = randint(0, v, (n, k), seed=2), rand(n, k, seed=3)
    hit = torch.zeros(n, dtype=torch.bool, device=DEV)
    hit[[0, n // 2, n - 1]] = True
    ids[:, 1] = -1
    ids[hit, k // 2 :] = v + 3
    top = good.clone()
    top[hit, 0] = bad
    top[:, 1] = bad  # of a padding entry: nothing
    named = torch.zeros(n, v + 1, dtype=torch.bool, device=DEV)
    named.scatter_(1, torch.where((ids >= 0) & (ids < v), ids, v), True)
    named = named[:, :v] & hit.unsqueeze(1)
    for how in ("none", "mean"):
        results = []
        for teacher in (good, top):
            x = full[1:-1, 8 : v + 8].detach().requires_grad_(True)
            loss = topk_distill_loss(x, ids, teacher, 1.5, reduction=how)
            up = torch.ones_like(loss) if how == "none" else torch.tensor(0.5, device=DEV)
            first = torch.autograd.grad(loss, x, torch.ones_like(loss), retain_graph=True)[0]
            results.append((loss, first, torch.autograd.grad(loss, x, up)[0]))
        (a, *ga), (b, *gb) = results
        assert torch.equal(a[~hit], b[~hit]) and b[hit].isnan().all() if how == "none" else b.isnan()
        for p, q in zip(ga, gb):
            assert torch.equal(q.isnan(), named) and p.isfinite().all()
            assert torch.equal(p[~named], q[~named])
    with torch.no_grad():
        rows = topk_distill_loss(full[1:-1, 8 : v + 8], ids, top, 1.5, reduction="none")
    assert torch.equal(rows.isnan(), hit)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("v,wide", [(1000, 1024), (30001, 30016), (40001, 40960), (70003, 70005)])
def test_distillation_of_strided_logits(v, wide, dtype):
    """A view of a padded vocabulary, a view that starts at an odd element, and expanded upstream gradients."""
    from ebr_b200.token_ops import topk_distill_loss

    ids, top = randint(-1, v, (7, 9), seed=1), rand(7, 9, seed=2)
    full = (rand(7, wide + 3, seed=3) * 2).to(dtype)
    for view in (full[:, :v], full[:, 3 : v + 3]):
        check_distill(view, ids, top, 2.0)
    leaf = full.clone().requires_grad_(True)
    loss = topk_distill_loss(leaf[:, :v], ids, top, 2.0, reduction="none").mean()
    loss.backward()
    assert not leaf.grad[:, v:].any()
    ref = plain_distill(full[:, :v], ids, top, 2.0)[1] / 7
    assert float((leaf.grad[:, :v].double() - ref).norm()) <= (2 * U[dtype] + 1e-5) * float(ref.norm())
    check_distill(full[:, :v].reshape(1, 7, v), ids.view(1, 7, 9), top.view(1, 7, 9), 2.0)  # leading dimensions


@pytest.mark.parametrize("v,wide", [(1001, 1024), (20001, 20016), (40001, 40960)])
def test_distillation_of_a_padded_vocabulary_in_batches(v, wide):
    """[B, L, :V] of [B, L, W]: the values, and no copy of the logits (the peak of the loss alone stays far below one)."""
    from ebr_b200.token_ops import topk_distill_loss

    full = (rand(3, 50, wide, seed=1) * 2).to(torch.bfloat16)
    ids, top = randint(-1, v, (3, 50, 4), seed=2), rand(3, 50, 4, seed=3)
    view = full[:, :, :v]
    for logits in (view, view[:, ::2], view[1:2].transpose(0, 1), view[:, :1].expand(3, 50, v)):  # ... and strides that combine
        i = ids[:, : logits.shape[1]] if logits.shape[0] == 3 else ids[1:2].transpose(0, 1)
        t = top[:, : logits.shape[1]] if logits.shape[0] == 3 else top[1:2].transpose(0, 1)
        check_distill(logits, i, t, 1.5)
    x = view.detach().requires_grad_(True)
    topk_distill_loss(x, ids, top, reduction="none")
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    held = torch.cuda.memory_allocated()
    with torch.no_grad():
        topk_distill_loss(x, ids, top, reduction="none")
    assert torch.cuda.max_memory_allocated() - held < view.numel() // 2
    loss = topk_distill_loss(x, ids, top)  # and its gradient, made in the forward pass
    torch.autograd.grad(loss, x)
    assert torch.cuda.max_memory_allocated() - held < 3 * full.numel()  # bytes: one gradient is two an element


@pytest.mark.parametrize("how", ["none", "mean"])
def test_distillation_copies_logits_without_a_row_stride_once(how):
    """logits[:, :-1] of [B, L, V] has no one row stride: its copy is the forward's, and the backward makes none."""
    from ebr_b200.token_ops import topk_distill_loss

    full = rand(3, 51, 20000, seed=1, dtype=torch.bfloat16)
    view = full[:, :-1]
    ids, top = randint(-1, 20000, (3, 50, 4), seed=2), rand(3, 50, 4, seed=3)
    check_distill(view, ids, top, 1.5)
    for up in (1.0, 2.0):
        x = view.detach().requires_grad_(True)
        loss = topk_distill_loss(x, ids, top, reduction=how)
        upstream = torch.full_like(loss, up)
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        held = torch.cuda.memory_allocated()
        torch.autograd.grad(loss, x, upstream)
        gradient = 2 * view.numel() if how == "none" else 0  # bytes; a reduced loss holds it already
        assert torch.cuda.max_memory_allocated() - held <= gradient + (1 << 20)


def test_rows_of_batched_views_are_read_in_place():
    """Views whose leading dimensions share one row stride, and those that have none: the same values as their copies."""
    from ebr_b200.token_ops import expert_combine, expert_dispatch, expert_route, scaled_embedding

    big = rand(4, 6, 40, seed=1)
    r = expert_route(randint(0, 5, (4, 6, 2), seed=2), 5)
    w = rand(10, 34, seed=3).requires_grad_(True)
    tokens = randint(0, 10, (4, 6), seed=4)
    for view in (big[:, :, 3:37], big.transpose(0, 1)[:, :, :34].transpose(0, 1), rand(6, 4, 34, seed=5).transpose(0, 1),
                 big[:1, :, :34].expand(4, 6, 34), big[:, :1, :34].expand(4, 6, 34), big[:1, :1, :34].expand(4, 6, 34),
                 rand(34, 4, 6, seed=6).permute(1, 2, 0), rand(4, 6, 1, seed=7).expand(4, 6, 34)):  # fmt: skip
        assert torch.equal(expert_dispatch(view, r), expert_dispatch(view.contiguous(), r))
        x = torch.zeros(r.rows, 34, device=DEV, requires_grad=True)
        a, b = (torch.autograd.grad(expert_combine(x, r), x, g)[0] for g in (view, view.contiguous()))
        assert torch.equal(a, b)
        a, b = (torch.autograd.grad(scaled_embedding(tokens, w), w, g)[0] for g in (view, view.contiguous()))
        assert torch.equal(a, b)


def test_distillation_repeats_bit_for_bit_on_other_streams_and_for_many_rows():
    from ebr_b200.token_ops import topk_distill_loss

    for n, v in ((5000, 37), (900, 9000)):
        x = rand(n, v, seed=1, dtype=torch.bfloat16).requires_grad_(True)
        ids, top = randint(-1, v, (n, 12), seed=2), rand(n, 12, seed=3)
        a = topk_distill_loss(x, ids, top)
        (ga,) = torch.autograd.grad(a, x)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            b = topk_distill_loss(x, ids, top)
            (gb,) = torch.autograd.grad(b, x)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(a, b) and torch.equal(ga, gb)


def test_distillation_gradient_by_differences():
    from ebr_b200.token_ops import topk_distill_loss

    x, ids, top = rand(6, 40, seed=1), randint(0, 40, (6, 5), seed=2), rand(6, 5, seed=3)
    d = rand(6, 40, seed=4)
    leaf = x.clone().requires_grad_(True)
    (g,) = torch.autograd.grad(topk_distill_loss(leaf, ids, top, 1.5, reduction="sum"), leaf)
    h = 2.0**-5  # third derivatives of order one: h^2 / 6 of the size of |d|^3, and 40 roundings of a loss near 20 over h
    f = lambda a: topk_distill_loss(a, ids, top, 1.5, reduction="none").double().sum().item()  # noqa: E731
    diff = (f(x + h * d) - f(x - h * d)) / (2 * h)
    assert abs(diff - float((g.double() * d).sum())) <= h * h * float(d.abs().pow(3).sum()) / 6 + 40 * E * 20 / h


def test_distillation_empty_batches_and_refusals():
    from ebr_b200.token_ops import topk_distill_loss

    x = torch.empty(0, 10, device=DEV, requires_grad=True)
    i, t = torch.empty(0, 3, dtype=torch.int64, device=DEV), torch.empty(0, 3, device=DEV)
    assert topk_distill_loss(x, i, t, reduction="none").shape == (0,)
    total = topk_distill_loss(x, i, t, reduction="sum")
    assert total.item() == 0 and torch.autograd.grad(total, x)[0].shape == (0, 10)
    x, i, t = rand(2, 10), torch.zeros(2, 3, dtype=torch.int64, device=DEV), rand(2, 3)
    for bad in (
        lambda: topk_distill_loss(x, i[:1], t),
        lambda: topk_distill_loss(x, i, t[:, :2]),
        lambda: topk_distill_loss(x, i, t, 0.0),
        lambda: topk_distill_loss(x, i, t, reduction="max"),
        lambda: topk_distill_loss(x, i, t, row_weight=rand(3)),
        lambda: topk_distill_loss(x, i, t.clone().requires_grad_(True)),
        lambda: topk_distill_loss(x, i[:, :1].expand(2, 1025), t[:, :1].expand(2, 1025)),
        lambda: topk_distill_loss(rand(1, (1 << 19) + 1), i[:1], t[:1]),
    ):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        topk_distill_loss(x.double(), i, t)
    with pytest.raises(RuntimeError, match="only on CUDA"):
        topk_distill_loss(x.cpu(), i, t)
    leaf = x.clone().requires_grad_(True)
    (g,) = torch.autograd.grad(topk_distill_loss(leaf, i, t), leaf, create_graph=True)
    with pytest.raises(RuntimeError):  # differentiable once
        torch.autograd.grad(g.sum(), leaf)


# ---------------------------------------------------------------------------------------------------- together


def _plain_experts(net, blk, h):
    """The sparse MLP from indexing and matmul, as the definition has it (no expert over its capacity here)."""
    s = net.shape
    flat = h.reshape(-1, h.shape[-1])
    best, ids = (flat @ blk.router.t()).topk(s.experts_per_cell, dim=-1)
    w = best.softmax(-1)
    out = torch.zeros_like(flat)
    for k in range(s.experts_per_cell):
        gate, up = torch.einsum("nc,nwc->nw", flat, blk.expert_gate_up[ids[:, k]]).chunk(2, -1)
        act = torch.nn.functional.silu(gate) * up
        out = out + w[:, k : k + 1] * torch.einsum("nw,ncw->nc", act, blk.expert_down[ids[:, k]])
    return out.view(h.shape)


def test_forward_mode_is_refused():
    """A forward-mode tangent of any input, or of an upstream gradient, is an error and not a derivative of zero."""
    from torch.autograd import forward_ad

    from ebr_b200.token_ops import expert_combine, expert_dispatch, expert_route, scaled_embedding, topk_distill_loss

    tokens, w, x = randint(0, 6, (9,), seed=1), rand(6, 8, seed=2), rand(9, 8, seed=3)
    r = expert_route(randint(0, 4, (9, 2), seed=4), 4)
    rows, wt = rand(r.rows, 8, seed=5), rand(9, 2, seed=6)
    ids, top, weight = randint(0, 8, (9, 3), seed=7), rand(9, 3, seed=8), rand(9, seed=9).abs()
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (
            lambda: scaled_embedding(tokens, dual(w)),
            lambda: expert_dispatch(dual(x), r),
            lambda: expert_combine(dual(rows), r, wt),
            lambda: expert_combine(rows, r, dual(wt)),
            lambda: topk_distill_loss(dual(x), ids, top),
            lambda: topk_distill_loss(x, ids, dual(top)),
            lambda: topk_distill_loss(x, ids, top, row_weight=dual(weight), reduction="none"),
        ):
            with pytest.raises(NotImplementedError):
                call()
            with torch.no_grad(), pytest.raises(NotImplementedError):
                call()
        leaves = [t.clone().requires_grad_(True) for t in (w, x, rows, wt)]
        ww, xx, rr, ll = leaves
        for out, wrt in (
            (scaled_embedding(tokens, ww), [ww]),
            (expert_dispatch(xx, r), [xx]),
            (expert_combine(rr, r, ll), [rr, ll]),
            (topk_distill_loss(xx, ids, top, reduction="none"), [xx]),
        ):
            with pytest.raises(NotImplementedError):
                torch.autograd.grad((out * dual(torch.ones_like(out))).sum(), wrt)
        assert torch.equal(scaled_embedding(tokens, w), w[tokens])  # tensors without a tangent are as ever


def test_compiled_callers_get_the_same_results():
    """torch.compile breaks its graph at the operators and runs them as they are."""
    from ebr_b200.token_ops import expert_combine, expert_dispatch, expert_route, scaled_embedding, topk_distill_loss

    def f(tokens, w, experts, weights, ids, top):
        h = scaled_embedding(tokens, w, 2.0).tanh()
        r = expert_route(experts, 4, 12)
        return topk_distill_loss(expert_combine(expert_dispatch(h, r) * 2, r, weights) + h, ids, top, 1.5)

    args = [randint(0, 6, (20,), seed=1), rand(6, 32, seed=2).requires_grad_(True), randint(0, 4, (20, 2), seed=3),
            rand(20, 2, seed=4).requires_grad_(True), randint(-1, 32, (20, 3), seed=5), rand(20, 3, seed=6)]  # fmt: skip
    results = []
    for call in (f, torch.compile(f, backend="eager")):
        loss = call(*args)
        results.append((loss, *torch.autograd.grad(loss, [args[1], args[3]])))
    for a, b in zip(*results):
        assert torch.equal(a, b)


def test_expert_network_matches_plain_experts_to_second_order():
    """E, dE/dv and d<dE/dv, u>/d(v, weights) of the float32 network against the same network with a plain sparse MLP:
    1e-4 of the norms, the bar of the dense float32 network's fixtures."""
    from ebr_b200.expert_net import ExpertEnergyNet, ExpertShape

    shape = ExpertShape(board=(3, 3), hidden=64, heads=2, layers=2, dtype=torch.float32, experts=4, capacity_factor=4.0)
    net = ExpertEnergyNet(shape, generator=torch.Generator().manual_seed(0)).to(DEV)
    tokens, v, u = randint(-1, 10, (5, 9), seed=1), rand(5, 9, 64, seed=2), rand(5, 9, 64, seed=3)
    prev = torch.backends.cuda.matmul.allow_tf32
    torch.backends.cuda.matmul.allow_tf32 = False
    results = []
    try:
        for plain in (False, True):
            if plain:
                net._experts = lambda blk, h: _plain_experts(net, blk, h)
            x = net.embed(tokens)
            vv = v.clone().requires_grad_(True)
            e, g = net.energy_and_grad(vv, x, create_graph=True)
            blk = net.blocks[0]
            wrt = [vv, net.embedding, blk.router, blk.expert_gate_up, blk.expert_down]
            results.append([e, g, *torch.autograd.grad((g * u).sum(), wrt)])
    finally:
        torch.backends.cuda.matmul.allow_tf32 = prev
    for a, b in zip(*results):
        assert float((a.double() - b.double()).norm()) <= 1e-4 * float(b.double().norm())


def test_expert_network_routes_by_float32_scores(monkeypatch):
    """The bfloat16 network's choices are those of the float64 product of its activations with the bfloat16 router, wherever
    the scores of the chosen and of the others differ by more than the float32 product's rounding."""
    from ebr_b200 import expert_net
    from ebr_b200.expert_net import ExpertEnergyNet, ExpertShape

    net = ExpertEnergyNet(ExpertShape(layers=1), generator=torch.Generator().manual_seed(0)).to(DEV)
    seen, route = [], expert_net.expert_route
    monkeypatch.setattr(expert_net, "expert_route", lambda ids, *a: (seen.append(ids), route(ids, *a))[1])
    h = rand(40, 81, 512, seed=1, dtype=torch.bfloat16)
    router = net.blocks[0].router.detach().bfloat16()
    with torch.no_grad():
        out = net._experts(net.blocks[0], h)
    assert out.dtype == torch.bfloat16
    exact = h.double() @ router.double().t()
    magnitude = h.double().abs() @ router.double().abs().t()
    best, ids = exact.topk(net.shape.experts_per_cell + 1, dim=-1)
    clear = ((best[..., :-1] - best[..., 1:]) > 2 * 514 * E * magnitude.max(-1, keepdim=True).values).all(-1)
    assert float(clear.double().mean()) > 0.95
    assert torch.equal(seen[0][clear], ids[..., :-1][clear])


@pytest.mark.parametrize("sparse", [False, True])
def test_distillation_segment_embeds_as_the_network_does(sparse):
    """The segment's input is the one that the network sees in use, bit for bit, and the embedding is trained through it."""
    from ebr_b200.energy import LatentEnergyNet, NetShape
    from ebr_b200.expert_net import ExpertEnergyNet, ExpertShape, distill_segment_loss

    gen = torch.Generator().manual_seed(0)
    net = ExpertEnergyNet(ExpertShape(layers=1), generator=gen) if sparse else LatentEnergyNet(NetShape(layers=1), generator=gen)
    net = net.to(DEV)
    tokens = randint(0, 10, (4, 81), seed=1)
    ids, top = randint(0, 10, (4, 81, 3), seed=2), rand(4, 81, 3, seed=3)
    seen, step = [], net.microstep
    net.microstep = lambda z, x, **k: (seen.append(x.detach()), step(z, x, **k))[1]
    distill_segment_loss(net, net.fresh_states(4), tokens, ids, top, prefix=0, graded=1).backward()
    assert len(seen) == 1 and torch.equal(seen[0], net.embed(tokens))
    assert net.embedding.grad.isfinite().all() and net.embedding.grad.any()


def test_distillation_example_runs_and_learns():
    import importlib.util
    from pathlib import Path

    path = Path(__file__).resolve().parent.parent / "examples" / "distill_experts.py"
    spec = importlib.util.spec_from_file_location("distill_experts", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    losses = example.run(steps=12, n=16, experts=4, entries=3, layers=1)
    assert all(math.isfinite(x) for x in losses)
    assert min(losses[-3:]) < losses[0]
