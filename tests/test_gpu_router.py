"""The expert router on the GPU against a plain 64-bit restatement (tests/kv_reference.py): the same experts in the same
order, weights rounded to float32 once; and a decoder layer's step with the paged cache, the router and the experts."""

import numpy as np
import pytest

import kv_reference as ref
from conftest import load_package

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def b200():
    import torch

    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return load_package()


@pytest.fixture(scope="module")
def ctx(b200):
    c = b200.Context(0)
    yield c
    c.close()


def cu(a):
    import torch

    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def check(ctx, logits, top_k, bias=None, **how):
    ids, w = ctx.moe_router(cu(logits), top_k, bias=None if bias is None else cu(bias), **how)
    ctx.synchronize()
    want_ids, want_w = ref.route(logits, top_k, bias, **how)
    assert np.array_equal(ids.cpu().numpy(), want_ids)
    # the double arithmetic of both sides (an exponential within 2^-52 of the size of its argument, a sum of 1024 terms)
    # differs by far less than half a float32 step: one rounding, and a rounding that falls the other way
    assert (np.abs(w.cpu().numpy() - want_w) <= np.abs(want_w) * 2.0 ** -23 + 1e-45).all()


def test_refusals(b200, ctx):
    import torch

    x = torch.zeros(2, 64, device="cuda")
    for how in (dict(top_k=0), dict(top_k=65), dict(top_k=33), dict(top_k=8, n_group=3), dict(top_k=8, n_group=64), dict(top_k=8, n_group=8, topk_group=9),
                dict(top_k=8, n_group=8, topk_group=0), dict(top_k=9, n_group=8, topk_group=1), dict(top_k=1, n_group=2, group_top=3),
                dict(top_k=1, n_group=0)):
        with pytest.raises(b200.B200Error):
            ctx.moe_router(x, **how)
    with pytest.raises(b200.B200Error, match="UNSUPPORTED"):
        ctx.moe_router(torch.zeros(1, 1025, device="cuda"), 8)
    with pytest.raises(ValueError):
        ctx.moe_router(x, 8, bias=torch.zeros(63, device="cuda"))
    with pytest.raises(ValueError):
        ctx.moe_router(x.half(), 8)
    with pytest.raises(ValueError):
        ctx.moe_router(x.t(), 2)
    with pytest.raises(ValueError):
        ctx.moe_router(x, 8, ids=torch.zeros(2, 8, dtype=torch.int64, device="cuda"))
    ids, w = ctx.moe_router(x[:0], 8)
    assert ids.shape == (0, 8) and w.shape == (0, 8)
    ctx.synchronize()


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("T,E,k,groups", [
    (1, 128, 8, {}), (37, 256, 8, {}), (5, 1, 1, {}), (9, 7, 7, {}), (33, 32, 32, {}), (3, 1024, 32, {}), (4, 1000, 6, {}), (130, 60, 4, {}),
    (64, 256, 8, dict(n_group=8, topk_group=4, group_top=2)), (20, 64, 6, dict(n_group=8, topk_group=3, group_top=1)),
    (11, 160, 6, dict(n_group=32, topk_group=32, group_top=2)), (7, 8, 2, dict(n_group=8, topk_group=2, group_top=2)), (6, 513, 5, dict(n_group=3, topk_group=1)),
])
def test_router(ctx, score, biased, T, E, k, groups):
    rng = np.random.default_rng(T + E)
    logits = (rng.normal(0, 2, (T, E))).astype(np.float32)
    bias = rng.normal(0, 0.1, E).astype(np.float32) if biased else None
    for renorm, scale in ((True, 1.0), (False, 2.5)):
        check(ctx, logits, k, bias, score=score, renorm=renorm, scale=scale, **groups)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups", [{}, dict(n_group=4, topk_group=2, group_top=2)])
def test_ties_go_to_the_lowest_index(ctx, score, groups):
    rng = np.random.default_rng(1)
    logits = rng.integers(-2, 3, (50, 64)).astype(np.float32)
    logits[0] = 0.0
    logits[1] = -0.0
    logits[1, 5] = 0.0  # equal to -0
    check(ctx, logits, 8, score=score, **groups)
    check(ctx, logits, 8, np.zeros(64, np.float32), score=score, **groups)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_scores_that_float32_cannot_tell_apart(ctx, score):
    """Biased scores that differ by less than a float32 step of their sum are still ordered."""
    rng = np.random.default_rng(2)
    logits = (rng.normal(0, 1, (64, 1)) + rng.integers(-3, 4, (64, 128)) * 2.0 ** -22).astype(np.float32)
    check(ctx, logits, 8, np.full(128, 1.0, np.float32), score=score)
    check(ctx, logits, 8, np.full(128, -0.5, np.float32), score=score, n_group=8, topk_group=2, group_top=2)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("n_group,size,group_top", [(8, 32, 2), (8, 32, 1), (4, 5, 2), (32, 1, 2), (16, 64, 2)])
@pytest.mark.parametrize("steps", [1.0, 2.0 ** -22])
def test_groups_that_float32_cannot_tell_apart(ctx, score, n_group, size, group_top, steps):
    """Each group has the same logits in another order, and biases that only double precision sees: their sums decide between
    the groups. With logits that are `steps` apart a few experts of each group count, or all of them."""
    rng = np.random.default_rng(5)
    base = (rng.normal(0, 1, (40, 1)) + np.arange(size) * steps).astype(np.float32)
    logits = np.concatenate([base[:, rng.permutation(size)] for _ in range(n_group)], 1)
    bias = (rng.integers(-200, 200, n_group * size) * 2.0 ** -40).astype(np.float32)
    check(ctx, logits, min(4, n_group // 2 * size), bias, score=score, n_group=n_group, topk_group=n_group // 2, group_top=group_top)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("groups", [{}, dict(n_group=4, topk_group=2, group_top=2)])
def test_infinities_nan_and_the_types_ends(ctx, score, biased, groups):
    rng = np.random.default_rng(3)
    big = np.finfo(np.float32).max
    logits = rng.normal(0, 1, (12, 64)).astype(np.float32)
    logits[0] = -np.inf                       # nothing is left
    logits[1, :60] = -np.inf                  # fewer than are chosen
    logits[2, 3] = np.nan
    logits[3] = np.nan
    logits[4, [5, 40]] = np.inf
    logits[5] = -big                          # a mask of the type's lowest value
    logits[6, ::2] = -big
    logits[7] = rng.choice([-big, big], 64)
    logits[8, :32] = [-np.inf, np.nan] * 16
    logits[9] *= 1e-40
    logits[10] *= 100
    bias = rng.normal(0, 0.1, 64).astype(np.float32) if biased else None
    if biased:
        bias[[1, 17]] = -np.inf               # experts that are switched off
        bias[33] = np.nan
    for renorm in (True, False):
        check(ctx, logits, 8, bias, score=score, renorm=renorm, **groups)


@pytest.mark.parametrize("T,E,k,score,groups", [
    (5003, 64, 4, "sigmoid", dict(n_group=8, topk_group=3, group_top=2)), (20001, 16, 1, "softmax", {}), (9000, 40, 3, "softmax", dict(n_group=5, topk_group=2)),
    (2369, 32, 20, "sigmoid", {}),
])
def test_any_number_of_rows_per_warp(ctx, T, E, k, score, groups):
    """A warp takes 1 to 32 / (a power of two from k) rows: three of eight, nine of 32, four of eight, one of one."""
    rng = np.random.default_rng(T)
    check(ctx, rng.normal(0, 2, (T, E)).astype(np.float32), k, rng.normal(0, 0.1, E).astype(np.float32), score=score, **groups)


def test_many_rows_and_a_captured_call(ctx):
    import torch

    rng = np.random.default_rng(4)
    logits = rng.normal(0, 2, (5001, 128)).astype(np.float32)
    check(ctx, logits, 8)
    x = cu(logits)
    ids, w = torch.zeros(5001, 8, dtype=torch.int32, device="cuda"), torch.zeros(5001, 8, device="cuda")
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        ctx.moe_router(x, 8, score="sigmoid", ids=ids, w=w)
    x.copy_(cu(logits[::-1]))
    g.replay()
    torch.cuda.synchronize()
    want = ctx.moe_router(x, 8, score="sigmoid")
    assert torch.equal(ids, want[0]) and torch.equal(w, want[1])


@pytest.mark.parametrize("qname", ["F16", "Q8_0"])
def test_steps_of_a_decoder_layer_with_experts(b200, ctx, oracle, qname):
    """Four steps of three requests through one layer: the fused q|k|v product, its rows written to the paged cache and
    attended to, the o product, the router's scores and the routed experts. Each piece is held against its own reference on
    the inputs that it had."""
    import torch

    rng = np.random.default_rng(5)
    hidden, H, Hkv, D, E, F, k, page, S = 256, 8, 2, 64, 16, 256, 4, 16, 3
    def quant(n_out, n_in, n=1):
        return oracle.quantize(b200.Q8_0, rng.normal(0, 0.05, (n * n_out, n_in)).astype(np.float32))
    qkv = ctx.weight(b200.Q8_0, hidden, (H + 2 * Hkv) * D, data=quant((H + 2 * Hkv) * D, hidden))
    o = ctx.weight(b200.Q8_0, H * D, hidden, data=quant(hidden, H * D))
    gate_up = ctx.weight(b200.Q8_0, hidden, 2 * F, E, data=quant(2 * F, hidden, E))
    down = ctx.weight(b200.Q8_0, F, hidden, E, data=quant(hidden, F, E))
    gate = cu(rng.normal(0, 0.1, (E, hidden)).astype(np.float32))
    cache = ctx.kv_cache(getattr(b200, qname), Hkv, D, page, 12)
    table = cu(rng.permutation(12).reshape(S, 4).astype(np.int32))
    lens = cu(np.array([0, 14, 31], np.int32))
    past = [torch.randn(S, 31, Hkv, D, device="cuda") for _ in range(2)]
    ctx.kv_write(cache, *past, table, lens)
    x = cu(rng.normal(0, 1, (S, hidden)).astype(np.float32))
    for _ in range(4):
        lens += 1
        rows = ctx.mul_mat(qkv, x).view(S, 1, H + 2 * Hkv, D)
        q, kk, vv = rows[:, :, :H], rows[:, :, H:H + Hkv], rows[:, :, H + Hkv:]
        ctx.kv_write(cache, kk, vv, table, lens)
        a = ctx.kv_attention(cache, q, table, lens, D ** -0.5)
        y = x + ctx.mul_mat(o, a.view(S, H * D))
        logits = y @ gate.t()
        ids, w = ctx.moe_router(logits, k)
        out = ctx.moe_ffn(gate_up, down, y, ids, w)
        ck, cv = ctx.kv_read(cache, table, lens, n_tok=64)
        ctx.synchronize()
        sizes = lens.tolist()
        want, tol = ref.attention(q.cpu().numpy(), [t[:n].cpu().numpy() for t, n in zip(ck, sizes)], [t[:n].cpu().numpy() for t, n in zip(cv, sizes)],
                                  sizes, D ** -0.5)
        assert (np.abs(a.cpu().numpy() - want) <= tol).all()
        for got, row in ((ck, kk), (cv, vv)):  # the newest row is the one that was written, within its type's half step
            new = torch.stack([got[s, n - 1] for s, n in enumerate(sizes)])
            step = row[:, 0].unflatten(-1, (-1, 32)).abs().amax(-1, keepdim=True) * (2.0 ** -11 if qname == "F16" else 0.51 / 127 + 2.0 ** -11)
            assert ((new - row[:, 0]).unflatten(-1, (-1, 32)).abs() <= step).all()
        want_ids, want_w = ref.route(logits.cpu().numpy(), k)
        assert np.array_equal(ids.cpu().numpy(), want_ids) and np.allclose(w.cpu().numpy(), want_w, rtol=2.0 ** -23, atol=0)
        again = ctx.moe_ffn(gate_up, down, y, cu(want_ids), cu(want_w.astype(np.float32)))
        assert torch.allclose(out, again, rtol=1e-5, atol=1e-6 * float(again.abs().max()))
        x = y + out
    for t in (qkv, o, gate_up, down):
        ctx.free_weight(t)
    cache.close()
