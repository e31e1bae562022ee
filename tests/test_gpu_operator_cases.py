"""Every case of perf/operators.py, and some that it draws, through the framework's calls: against its 64-bit definitions, and
the experts' numbers against its plain form."""

import importlib.util
import math
import os
import random

import pytest

from conftest import load_package

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def load():
    spec = importlib.util.spec_from_file_location("operator_cases", os.path.join(ROOT, "perf", "operators.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def cases():
    module = load()
    rng = random.Random(7)
    return [(c["name"], c) for c in module.listed()] + [(f"drawn_{i}", module.draw(rng)) for i in range(12)]


@pytest.fixture(scope="module")
def operators():
    import torch

    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    load_package()
    module = load()
    module.own = True
    yield module
    module._framework()[1].close()


def bound(module, case, state, exact):
    """How far a result of this type may be off, each element (or all)."""
    if case["op"] == "router":  # double arithmetic on both sides, rounded once: that, and a rounding that falls the other way
        return exact.abs() * 2.0 ** -23 + 1e-45
    if case["op"] != "attention":
        return exact * 0.0  # rows are rounded once, and the definitions are of the values that the cache holds
    # A score's error: q has 22 bits, D / 16 accumulations are rounded to float32 and three products more, each at most 2^-23 of
    # |q| |k|. The exponentials, the weight's 22 bits (and its product's with a scale) and the division are below 2^-19, and the
    # longest chain of additions is a quarter of the pieces of 16 and the partial results.
    size = [0.0, 0.0]
    for which in (0, 1):
        for a in range(0, state["views"][which].shape[0], 512):
            x = state["views"][which][a : a + 512]
            x = module._values(x, state["views"][2 + which][a : a + 512]) if case["cache"] == "q8_0" else x.float()
            size[which] = max(size[which], float(x.norm(dim=-1).amax() if which == 0 else x.abs().amax()))
    delta = state["scale"] * size[0] * float(state["q"].norm(dim=-1).amax()) * (case["dim"] / 16 + 4) * 2.0 ** -23
    return size[1] * (math.expm1(2 * delta) + 2.0 ** -19 + (case["max_len"] / 64 + 34) * 2.0 ** -24)


@pytest.mark.parametrize("case", [pytest.param(c, id=name) for name, c in cases()])
def test_case(operators, case):
    import torch

    torch.cuda.empty_cache()
    want = operators.exact(dict(case), 3)
    state = operators.prepare(dict(case), 3)
    got = operators.run(state)
    ids = None
    if case["op"] == "router":
        operators.own = False
        ids = operators.run(state)[0]
        operators.own = True
        assert torch.equal(got[0], ids)
    if want is None:
        pytest.skip("no 64-bit form of this size")
    pairs = [(g, w) for g, w in (zip(got, want) if isinstance(got, (list, tuple)) else [(got, want)]) if w is not None]
    assert pairs
    for g, w in pairs:
        assert g.shape == w.shape and (ids is not None or torch.isfinite(g).all())
        if case["op"] in ("write", "read"):  # the 64-bit form rounded to the result's type
            assert torch.equal(g.to(torch.float64), w.to(g.dtype).to(torch.float64))
        else:
            assert ((g.double() - w).abs() <= bound(operators, case, state, w)).all()
