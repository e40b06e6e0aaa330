"""The C ABI of include/ebr_tokens.h on the CPU host: every declared symbol is exported and bound, bad arguments are refused
with the documented codes before a device is touched, and scratch sizes are what the kernels need. The Python operators
refuse CPU tensors; the measured cases' plain forms agree with their float64 forms."""

from __future__ import annotations

import importlib.util
import random
from pathlib import Path

import pytest
import torch

from ebr_b200 import _native
from ebr_b200.build import build

from test_capi import declared_functions

ROOT = Path(__file__).resolve().parent.parent
HEADER = ROOT / "include" / "ebr_tokens.h"
P = 0x1000  # a pointer that no refused call follows
F32, F16, BF16, F64 = _native.FLOAT32, _native.FLOAT16, _native.BFLOAT16, _native.FLOAT64


@pytest.fixture(scope="module")
def lib():
    build()
    return _native.lib()


def test_every_declared_symbol_is_exported_and_bound(lib):
    names = declared_functions(HEADER)
    assert set(names) == set(_native.EXPORTED_TOKENS)
    for n in names:
        assert hasattr(lib, n), n


def test_embedding_refusals(lib):
    f = lambda **k: lib.ebr_scaled_embedding(*{**dict(w=F32, o=BF16, i=1, n=4, V=10, C=8, s=1.0, ids=P, p=P, ws=8, out=P,
                                                      st=None), **k}.values())  # fmt: skip
    assert f(w=F64) == _native.ERR_DTYPE and f(o=9) == _native.ERR_DTYPE and f(i=2) == _native.ERR_DTYPE
    assert f(V=0) == _native.ERR_SHAPE and f(C=0) == _native.ERR_SHAPE and f(n=-1) == _native.ERR_SHAPE
    assert f(n=1 << 30) == _native.ERR_SHAPE and f(V=1 << 30) == _native.ERR_SHAPE
    assert f(ws=-8) == _native.ERR_STRIDE and f(ids=P + 4) == _native.ERR_STRIDE
    assert f(ids=None) == _native.ERR_NULL and f(p=None) == _native.ERR_NULL and f(out=None) == _native.ERR_NULL
    assert f(n=0, ids=None, p=None, out=None) == _native.OK
    size = lib.ebr_scaled_embedding_grad_scratch_bytes
    assert size(0, 10, 8) == 0 and size(4, 0, 8) == 0
    assert size(4, 10, 8) == 0  # few tokens: one launch that keeps nothing
    assert size(512, 10, 8) == 0 and size(512, 4000, 8) > 0 and size(128, 4000, 8) == 0
    assert size(4000, 10, 8) >= 2 * 16000 + 2 * 8 * 4  # sorted keys and positions, two partial sums
    assert size(1 << 20, 1 << 17, 64) >= 4 * (1 << 22)  # two passes: both pairs of arrays
    g = lambda **k: lib.ebr_scaled_embedding_grad(*{**dict(g=BF16, w=F32, i=1, n=4000, V=10, C=8, s=1.0, ids=P, p=P, gs=8,
                                                           dw=P, sc=P, b=1 << 20, st=None), **k}.values())  # fmt: skip
    assert g(b=0) == _native.ERR_SCRATCH and g(sc=None) == _native.ERR_SCRATCH and g(sc=P + 4) == _native.ERR_SCRATCH
    assert g(dw=P + 4) == _native.ERR_STRIDE and g(dw=None) == _native.ERR_NULL and g(p=None) == _native.ERR_NULL
    assert g(g=F64) == _native.ERR_DTYPE and g(V=0) == _native.ERR_SHAPE


def test_expert_refusals(lib):
    f = lambda **k: lib.ebr_expert_route(*{**dict(i=0, T=4, K=2, E=8, c=0, ids=P, r=P, s=P, o=P, sc=None, b=0, st=None),
                                           **k}.values())  # fmt: skip
    assert f(i=5) == _native.ERR_DTYPE
    for bad in (dict(E=0), dict(E=1025), dict(K=0), dict(T=-1), dict(c=-1), dict(T=1 << 29, K=4), dict(E=1024, c=1 << 25)):
        assert f(**bad) == _native.ERR_SHAPE, bad
    for bad in (dict(ids=None), dict(r=None), dict(s=None), dict(o=None)):
        assert f(**bad) == _native.ERR_NULL, bad
    assert lib.ebr_expert_route_scratch_bytes(100, 2, 8) == 0  # one cluster, nothing spilled
    need = lib.ebr_expert_route_scratch_bytes(100000, 2, 8)
    assert need > 0 and f(T=100000, sc=P, b=need - 1) == _native.ERR_SCRATCH
    s = lambda **k: lib.ebr_expert_scatter(*{**dict(d=BF16, w=F32, T=4, K=2, C=8, R=8, x=P, xs=8, r=P, s=P, wt=None,
                                                    i=None, o=P, dots=None, st=None), **k}.values())  # fmt: skip
    assert s(d=F64) == _native.ERR_DTYPE and s(w=F16) == _native.ERR_DTYPE
    assert s(K=0) == _native.ERR_SHAPE and s(C=0) == _native.ERR_SHAPE and s(R=-1) == _native.ERR_SHAPE
    assert s(xs=-1) == _native.ERR_STRIDE
    assert s(o=None) == _native.ERR_NULL and s(dots=P) == _native.ERR_NULL and s(i=P) == _native.ERR_NULL
    assert s(x=None) == _native.ERR_NULL and s(s=None) == _native.ERR_NULL
    c = lambda **k: lib.ebr_expert_combine(*{**dict(d=BF16, w=F32, T=4, K=2, C=8, i=P, rs=8, r=P, wt=None, y=P, st=None),
                                             **k}.values())  # fmt: skip
    assert c(w=F16) == _native.ERR_DTYPE and c(T=-1) == _native.ERR_SHAPE and c(rs=-1) == _native.ERR_STRIDE
    assert c(y=None) == _native.ERR_NULL and c(r=None) == _native.ERR_NULL and c(i=None) == _native.ERR_NULL
    assert c(T=0, y=None, r=None, i=None) == _native.OK


def test_distillation_refusals(lib):
    f = lambda **k: lib.ebr_topk_distill(*{**dict(d=BF16, i=1, t=F32, N=4, V=100, K=3, tau=1.0, f=1.0, x=P, xs=100, ids=P,
                                                  top=P, rw=None, l=P, s=P, tot=None, g=None, gs=0, st=None),
                                           **k}.values())  # fmt: skip
    assert f(d=F64) == _native.ERR_DTYPE and f(t=F64) == _native.ERR_DTYPE and f(i=3) == _native.ERR_DTYPE
    for bad in (dict(V=0), dict(K=0), dict(K=1025), dict(V=(1 << 19) + 1), dict(N=1 << 31), dict(tau=0.0),
                dict(tau=float("nan")), dict(N=-1)):  # fmt: skip
        assert f(**bad) == _native.ERR_SHAPE, bad
    assert f(xs=-1) == _native.ERR_STRIDE and f(g=P, gs=99) == _native.ERR_STRIDE
    assert f(ids=P + 4) == _native.ERR_STRIDE and f(s=P + 4) == _native.ERR_STRIDE
    for bad in (dict(x=None), dict(ids=None), dict(top=None), dict(l=None), dict(s=None)):
        assert f(**bad) == _native.ERR_NULL, bad
    assert f(N=0, x=None, ids=None, top=None, l=None, s=None) == _native.OK
    g = lambda **k: lib.ebr_topk_distill_grad(*{**dict(d=BF16, i=1, t=F32, N=4, V=100, K=3, tau=1.0, f=1.0, x=P, xs=100,
                                                       ids=P, top=P, rw=None, s=P, u=P, us=0, one=0, g=P, gs=100, st=None),
                                                **k}.values())  # fmt: skip
    assert g(us=2) == _native.ERR_STRIDE and g(gs=10) == _native.ERR_STRIDE
    assert g(u=None) == _native.ERR_NULL and g(g=None) == _native.ERR_NULL and g(s=None) == _native.ERR_NULL
    assert g(N=0, x=None) == _native.OK


def test_distillation_temperatures(lib):
    args = lambda tau, x: (BF16, 1, F32, 4, 100, 3, tau, 1.0, x, 100, P, P, None, P, P, None, None, 0, None)  # noqa: E731
    for bad in (0.0, -1.0, 1e-39, 1.1e30, float("inf"), float("nan")):
        assert lib.ebr_topk_distill(*args(bad, None)) == _native.ERR_SHAPE, bad
    for good in (2.0**-126, 1.0, 1e30):
        assert lib.ebr_topk_distill(*args(good, None)) == _native.ERR_NULL, good  # accepted; the logits are missing


def test_distillation_rows(lib):
    """The number of rows leaves room for the last step of a kernel's row counter, an int."""
    args = lambda n: (BF16, 1, F32, n, 100, 3, 1.0, 1.0, None, 100, P, P, None, P, P, None, None, 0, None)  # noqa: E731
    for n in ((1 << 31) - 1, (1 << 31) - 148 * 6, (1 << 31) - (1 << 16)):
        assert lib.ebr_topk_distill(*args(n)) == _native.ERR_SHAPE, n
    assert lib.ebr_topk_distill(*args((1 << 31) - (1 << 16) - 1)) == _native.ERR_NULL  # accepted; the logits are missing


def test_arrays_that_start_inside_an_element_are_refused(lib):
    """A 16-bit array at an odd address and a 32-bit one at an address of 2 mod 4, in every place that takes one."""
    one = dict(n=4, V=10, C=8)
    lookup = dict(w=F32, o=BF16, i=1, **one, s=1.0, ids=P, p=P, ws=8, out=P, st=None)
    grad = dict(g=BF16, w=F32, i=1, **one, s=1.0, ids=P, p=P, gs=8, dw=P, sc=None, b=0, st=None)
    route = dict(i=0, T=4, K=2, E=8, c=0, ids=P, r=P, s=P, o=P, sc=None, b=0, st=None)
    scatter = dict(d=BF16, w=F32, T=4, K=2, C=8, R=8, x=P, xs=8, r=P, s=P, wt=P, i=P, o=P, dots=P, st=None)
    combine = dict(d=BF16, w=F32, T=4, K=2, C=8, i=P, rs=8, r=P, wt=P, y=P, st=None)
    sizes = dict(N=4, V=100, K=3, tau=1.0, f=1.0)
    distill = dict(d=BF16, i=1, t=F32, **sizes, x=P, xs=100, ids=P, top=P, rw=P, l=P, s=P, tot=P, g=P, gs=100, st=None)
    back = dict(d=BF16, i=1, t=F32, **sizes, x=P, xs=100, ids=P, top=P, rw=P, s=P, u=P, us=0, one=0, g=P, gs=100, st=None)
    for name, args, halves, words in (
        ("ebr_scaled_embedding", lookup, ("out",), ("p",)),
        ("ebr_scaled_embedding_grad", grad, ("p",), ("dw",)),
        ("ebr_expert_route", route, (), ("ids", "r", "s", "o")),
        ("ebr_expert_scatter", scatter, ("x", "i", "o"), ("r", "s", "wt", "dots")),
        ("ebr_expert_combine", combine, ("i", "y"), ("r", "wt")),
        ("ebr_topk_distill", distill, ("x", "g"), ("ids", "top", "rw", "l", "s", "tot")),
        ("ebr_topk_distill_grad", back, ("x", "g"), ("ids", "top", "rw", "s", "u")),
    ):
        for place, off in [(a, 1) for a in halves] + [(a, 2) for a in words]:
            assert getattr(lib, name)(*{**args, place: P + off}.values()) == _native.ERR_STRIDE, (name, place)


def test_python_operators_refuse_cpu_tensors():
    from ebr_b200 import token_ops as tk

    ids = torch.zeros(3, 2, dtype=torch.int64)
    for call in (
        lambda: tk.scaled_embedding(ids, torch.zeros(4, 8)),
        lambda: tk.expert_route(ids, 4),
        lambda: tk.topk_distill_loss(torch.zeros(3, 8), ids, torch.zeros(3, 2)),
    ):
        with pytest.raises(RuntimeError, match="only on CUDA"):
            call()


def test_measured_cases_agree_with_their_float64_forms(monkeypatch):
    """perf/operators.py on the CPU at small sizes: the plain forms against the definitions in float64, within their types'
    rounding (bfloat16 2^-8, float16 2^-11, float32 sums 1e-5, all relative to the norm)."""
    spec = importlib.util.spec_from_file_location("operators", ROOT / "perf" / "operators.py")
    ops = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ops)
    monkeypatch.setattr(ops, "DEV", "cpu")
    rng = random.Random(3)
    for case in ops.listed() + [ops.draw(rng) for _ in range(12)]:
        case = {**case, **{k: min(case[k], 50) for k in ("n", "tokens", "rows") if k in case}}
        if "vocab" in case:
            case["vocab"] = min(case["vocab"], 400)
        if "topk" in case and "vocab" in case:
            case["topk"] = min(case["topk"], case["vocab"])
        case["dim"] = min(case.get("dim", 1), 70)
        if case.get("capacity"):
            case["capacity"] = 4
        assert ops.work(case)["bytes"] > 0
        got, exact = ops.run(ops.prepare(case, 5)), ops.exact(case, 5)
        for a, b in zip(got, exact):
            if b is None:
                continue
            tol = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}.get(a.dtype, 1e-5)
            assert float((a.double() - b).norm()) <= tol * float(b.norm()) + 1e-6, case
