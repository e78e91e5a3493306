"""The dense-head operators where they are easily wrong: rows far from zero, statistics at the edge of the floats' range,
what inference and partly frozen layers leave out, roundings counted exactly and what a call allocates.  Definitions,
tolerances and helpers are tests/test_gpu_dense.py's."""
from __future__ import annotations

import math
import sys
import weakref

import numpy as np
import pytest
import torch

from tests.conftest import load_pkg
from tests.test_gpu_dense import (F64, SUM, TYPES, act8_inputs, act8_ref, check_logp, close, gen, half_step, least, logp_inputs,
                                  logp_ref, norm_ref, randn)
from tests.test_gpu_layers import small_model

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def pkg():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return load_pkg()


@pytest.fixture(scope="module")
def K(pkg):
    return sys.modules[pkg.__name__ + ".kernels"]


# ---------------------------------------------------------------------------------------------------- log probabilities
def check_far(K, s, items, scale, k=0):
    """Against the definition, with no allowance for where the row lies: the differences z to the row's maximum are exact
    in 32 bits here, an exponent is off by 2^-22 of |z| (the difference times scale and log2 e), sums by SUM."""
    n, c = s.shape
    dlogp, dent = torch.ones(n, items.shape[1], device=DEV), torch.ones(n, device=DEV)
    r = K.log_prob_fwd(s, items, k=k, scale=scale)
    ref = logp_ref(s, items, k, scale, dlogp, dent)
    hmax = ref["entropy"].abs() + math.log(c)
    low = 2.0 ** -21 * hmax + SUM * (1 + hmax)
    close(r.logp, ref["logp"], low[:, None] + 2.0 ** -22 * ref["logp"].abs(), "logp")
    close(r.entropy, ref["entropy"], low, "entropy")
    close(r.lse, ref["lse"], low + 2.0 ** -22 * ref["lse"].abs(), "lse")
    if k:
        assert torch.equal(r.top_items, ref["top_items"])
        close(r.top_logp, ref["top_logp"], low[:, None] + 2.0 ** -22 * ref["top_logp"].abs(), "top")
    ds = K.log_prob_bwd(s, items, r.stats, dlogp, dent, scale=scale)
    close(ds, ref["dscores"], ref["size"] * (4 * low[:, None] + 2.0 ** -20 * (1 + low[:, None])) * 4 +
          half_step(s.dtype) * ref["dscores"].abs() + least(s.dtype), "dscores")


@pytest.mark.parametrize("scale", [1.0, 0.37])
@pytest.mark.parametrize("c", [40, 3000, 9000, 40001])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_log_prob_rows_of_one_mask_value(K, dtype, c, scale):
    """A row of nothing but a mask's finite value (-1e10, -1e30, ...) is uniform, as one of zeros is."""
    values = [v * sign for v in (1e5, 7e5, 1e7, 1e9, 1e10, 3e10, 1e12, 1e15, 1e20, 1e30, 1e36, 3e37) for sign in (1, -1)]
    s = torch.tensor(values, dtype=torch.float64, device=DEV).to(dtype)[:, None].expand(-1, c).contiguous()
    items = torch.tensor([0, c // 2, c - 1], device=DEV).expand(len(values), 3).contiguous()
    check_far(K, s, items, scale, k=20)


@pytest.mark.parametrize("c", [64, 3000, 9000, 40001])
def test_log_prob_rows_far_from_zero(K, c):
    """Scores a few steps apart, far from zero: the running maximum rises along the row, falls, and jumps about, over
    values at which its product with log2 e passes a power of two."""
    bases = [0.0, 5e4, 726817.0, -726817.0, 2.0 ** 19, 2.0 ** 20, -(2.0 ** 20), 1453635.0]
    steps = torch.arange(c, device=DEV).to(torch.float64).mul(64 / c).floor() / 16 - 2
    rows = []
    for b in bases:
        rows += [b + steps, b + steps.flip(0), b + steps[torch.randperm(c, device=DEV, generator=gen(c))]]
    s = torch.stack(rows).float()
    items = torch.tensor([0, c // 2, c - 1], device=DEV).expand(len(rows), 3).contiguous()
    check_far(K, s, items, 1.0)


@pytest.mark.parametrize("n,c", [(5, 3000), (300, 1100)])
def test_log_prob_of_1024_items_a_row(K, n, c):
    """The most given items a row, many of them more than once (the gradients of equal items are summed)."""
    s, items, dlogp, dent = logp_inputs(n, c, 1024, torch.float32, n)
    check_logp(K, s, items, 0, 1.0, dlogp, dent)


def test_log_prob_large_entropy_gradients(K):
    """A loss scale on the entropy term: masked columns get 0, the others what they get without it, scaled."""
    s, items, dlogp, dent = logp_inputs(6, 700, 2, torch.float32, 3, masked=0.3)
    r = K.log_prob_fwd(s, items)
    big = K.log_prob_bwd(s, items, r.stats, dlogp * 2.0 ** 30, dent * 2.0 ** 30)
    one = K.log_prob_bwd(s, items, r.stats, dlogp, dent)
    assert torch.isfinite(one).all() and torch.equal(big, one * 2.0 ** 30)  # powers of two: the same bits


# ---------------------------------------------------------------------------------------------------- layer norm
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,d", [(50, 96), (300, 3), (40, 257), (7, 1021), (5, 5000), (9, 9001), (3, 16399), (2, 70001)])
def test_layer_norm_rows_far_from_zero(K, n, d, dtype):
    """Rows of spread about 1 around a far mean.  The deviations from a rounded mean are exact or off by 2^-24 of
    themselves, and their own mean (off by SUM of the mean deviation) corrects the rest: nothing in y grows with the mean.
    The saved mean is off by its one rounding, which the backward's xhat sees as 2^-24 |mean| / sd."""
    at = 4096 if dtype == torch.float32 else 60
    x = (randn(gen(d), n, d) + at).to(dtype)
    dy = randn(gen(d + 1), n, d, dtype=dtype)
    y, mean, rstd = K.layer_norm_fwd(x, stats=True)
    ry, rmean, rrstd, xhat, g, rdx, rdw, rdb = norm_ref(x, None, None, 1e-5, dy)
    dev = (x.to(F64) - rmean[:, None]).abs().mean(1)
    close(mean, rmean, 2.0 ** -24 * rmean.abs() + 2 * SUM * dev, "mean")
    close(rstd, rrstd, 4 * SUM * rrstd, "rstd")
    close(y, ry, half_step(dtype) * ry.abs() + 4 * SUM * (1 + xhat.abs()) + least(dtype), "y")
    dx, dw, db = K.layer_norm_bwd(dy, x, mean, rstd)
    spread = (2.0 ** -24 * rmean.abs() * rrstd + 4 * SUM)[:, None]  # xhat's error
    ga, gx = g.abs().mean(1, keepdim=True), (g * xhat).abs().mean(1, keepdim=True)
    # dx = rstd (g - mean g - xhat mean(g xhat)): xhat's error in both places, the sums' and rstd's
    off = rrstd[:, None] * (spread * (gx + (xhat.abs() + 1) * ga) + 8 * SUM * (g.abs() + ga + (xhat.abs() + 1) * gx))
    close(dx, rdx, half_step(dtype) * rdx.abs() + off + least(dtype), "dx")
    close(dw, rdw, (dy.to(F64).abs() * (spread + SUM * xhat.abs())).sum(0) + 2.0 ** -24 * rdw.abs(), "dweight")


@pytest.mark.parametrize("d", [3, 40, 1021, 5000, 16399, 70001])
def test_layer_norm_constant_rows(K, d):
    """A constant row is its bias wherever it lies.  With D = x - mean, at most 2^-18 |x|, its correction is within
    (SUM + 2^-23) of D, and 1 / sqrt(eps) = 317 multiplies what is left."""
    x = torch.tensor([1000.1, -77.7, 0.3, 12345.6], device=DEV)[:, None].expand(4, d).contiguous()
    b = randn(gen(d), d)
    y, mean, rstd = K.layer_norm_fwd(x, None, b, 1e-5, stats=True)
    left = x[:, :1].to(F64).abs() * 2.0 ** -18 * (SUM + 2.0 ** -23) * 317
    close(y, b.to(F64).expand(4, d), left + 2.0 ** -24 * b.to(F64).abs(), "y")
    close(mean, x[:, 0], 2.0 ** -24 * x[:, 0].to(F64).abs(), "mean")
    # rstd, relative: half of var's error over eps, both of its terms being D^2 to 1.5 SUM; eps, the sum, the root and the
    # quotient are a rounding of 2^-24 each
    off = 1.5 * SUM * (x[:, 0].to(F64) * 2.0 ** -18).square() / 1e-5 + 2.0 ** -22
    close(rstd, torch.full((4,), 1e-5 ** -0.5, dtype=F64, device=DEV), 317 * off, "rstd")


def test_layer_norm_rows_of_huge_spread(K):
    """A row whose squares pass the floats' range has an infinite variance: rstd 0, y the bias, no NaN; its neighbours
    keep theirs."""
    x, b = randn(gen(1), 3, 1000), randn(gen(2), 1000)
    x[1] *= 1e27
    y, mean, rstd = K.layer_norm_fwd(x, None, b, stats=True)
    assert torch.equal(y[1], b) and rstd[1] == 0 and (rstd[[0, 2]] > 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d", [5, 8, 33, 1021, 9001, 16399])
def test_layer_norm_backward_of_a_large_constant_row(K, d, dtype):
    """mean times rstd is beyond the floats' range, xhat is 0: dx = rstd (g - mean g), at widths that end inside a vector
    too.  (2^100: the row's sums are exact.)"""
    x = torch.full((3, d), 2.0 ** 100, device=DEV, dtype=dtype)
    x[1] = randn(gen(d), d).to(dtype)
    dy = randn(gen(d + 1), 3, d, dtype=dtype)
    _, mean, rstd = K.layer_norm_fwd(x, eps=1e-20, stats=True)
    dx, dw, db = K.layer_norm_bwd(dy, x, mean, rstd)
    assert torch.isfinite(dw).all() and torch.isfinite(db).all()
    g = dy.to(F64)[[0, 2]]
    want = (g - g.mean(1, keepdim=True)) * 1e10
    # rstd = 1 / sqrt(1e-20 in 32 bits): a rounding of eps, of the root and of the quotient
    close(dx[[0, 2]], want, half_step(dtype) * want.abs() + 1e10 * SUM * (g.abs() + g.abs().mean(1, keepdim=True)), "dx")
    assert torch.isfinite(dx[1]).all()


# ---------------------------------------------------------------------------------------------------- layers
@pytest.mark.parametrize("mode", [torch.no_grad, torch.inference_mode])
def test_inference_keeps_nothing_for_a_backward(pkg, K, monkeypatch, mode):
    """Without gradients a linear layer packs no input and a norm writes no statistics; the outputs are the same bits, and
    what is refused stays refused."""
    x = randn(gen(1), 30, 64)
    norm, lin = pkg.layers.LayerNorm(64).to(DEV), pkg.layers.LinearAct8(64, 32).to(DEV)
    calls = []
    pack, fwd = K.act8_pack, K.layer_norm_fwd
    monkeypatch.setattr(K, "act8_pack", lambda t: calls.append("pack") or pack(t))

    def norm_fwd(*a, stats=False):
        calls.append("stats" if stats else "norm")
        return fwd(*a, stats=stats)

    monkeypatch.setattr(K, "layer_norm_fwd", norm_fwd)
    with_grad = lin(norm(x))
    assert with_grad.requires_grad and calls == ["stats", "pack"]
    calls.clear()
    with mode():
        got = lin(norm(x))
        for bad in (lambda: lin(x[:, :60]), lambda: lin(x.double()), lambda: norm(x.double()), lambda: lin(x.cpu()),
                    lambda: pkg.layers.linear_act8(x, lin.weight, lin.bias[:4]),
                    lambda: pkg.layers.linear_act8(x[:, :0], torch.nn.Parameter(lin.weight[:, :0]))):
            with pytest.raises(ValueError):
                bad()
    assert not got.requires_grad and torch.equal(got, with_grad.detach())
    assert "pack" not in calls and "stats" not in calls


def test_no_gradient_asked_for_keeps_nothing(pkg, K, monkeypatch):
    x, w = randn(gen(1), 30, 64), randn(gen(2), 8, 64)
    monkeypatch.setattr(K, "act8_pack", lambda t: pytest.fail("packed"))
    assert not pkg.layers.linear_act8(x, w).requires_grad
    b = randn(gen(3), 8).requires_grad_(True)
    pkg.layers.linear_act8(x, w, b).sum().backward()  # a bias alone needs no input
    assert torch.equal(b.grad, torch.full((8,), 30.0, device=DEV))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,d,o", [(70, 64, 96), (33, 40, 3), (1, 128, 64), (300, 33, 17)])
def test_linear_act8_rounds_once(pkg, dtype, n, d, o):
    """16-bit outputs: the product's 32-bit sum (d terms and the bias, 2^-23 of their size a term at the worst), rounded
    once; a product that nearly cancels the bias keeps its digits."""
    g = gen(n + d)
    x, w = randn(g, n, d, dtype=dtype), (randn(g, o, d) * 0.5).to(dtype)
    b = (randn(g, o) * 4).to(dtype)
    want = x.to(F64) @ w.to(F64).t() + b.to(F64)
    size = x.to(F64).abs() @ w.to(F64).abs().t() + b.to(F64).abs()
    for grad in (False, True):
        y = pkg.layers.linear_act8(x, w.clone().requires_grad_(grad), b).detach()
        close(y, want, half_step(dtype) * want.abs() + (d + 1) * 2.0 ** -23 * size + least(dtype), f"y, grad {grad}")
    assert pkg.layers.linear_act8(x.view(1, n, d), w, b).shape == (1, n, o)
    assert pkg.layers.linear_act8(x[0], w, b).shape == (o,)
    assert pkg.layers.linear_act8(x[:0], w, b).shape == (0, o)


def test_linear_act8_16_bit_step_in_a_captured_graph(pkg):
    """Forward and every gradient of a 16-bit layer, replayed on new inputs with eager work between."""
    g = gen(8)
    x, dy = randn(g, 500, 64, dtype=torch.bfloat16).requires_grad_(True), randn(g, 500, 48, dtype=torch.bfloat16)
    w, b = randn(g, 48, 64).requires_grad_(True), randn(g, 48).requires_grad_(True)

    def step():
        y = pkg.layers.linear_act8(x, w, b)
        return [y.detach(), *torch.autograd.grad(y, (x, w, b), dy)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for turn in range(4):
        with torch.no_grad():
            x.copy_(randn(g, 500, 64))
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in got]
        assert all(torch.equal(p, q) for p, q in zip(kept, step())), turn


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,o", [(100003, 131), (70001, 8), (257, 4096)])
def test_bias_alone_in_a_captured_graph(pkg, n, o, dtype):
    """A trained bias beside a frozen weight: the captured backward, replayed on new gradients with eager work between,
    gives the eager bits, and those are dy's column sums."""
    g = gen(n)
    x, w = randn(g, n, 8, dtype=dtype), randn(g, o, 8, dtype=dtype)
    b, dy = randn(g, o).requires_grad_(True), randn(g, n, o, dtype=dtype)

    def step():
        return torch.autograd.grad(pkg.layers.linear_act8(x, w, b), b, dy)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for turn in range(4):
        dy.copy_(randn(g, n, o))
        graph.replay()
        torch.cuda.synchronize()
        kept = got.clone()
        assert torch.equal(kept, step()), turn
        close(kept, dy.to(F64).sum(0), SUM * dy.to(F64).abs().sum(0), f"db, turn {turn}")


def test_log_probs_takes_two_dimensions(pkg):
    """The one layer that does: its items belong to the rows."""
    for bad in (lambda: pkg.layers.log_probs(torch.zeros(2, 3, 40, device=DEV), torch.zeros(6, 1, dtype=torch.int64, device=DEV)),
                lambda: pkg.layers.log_probs(torch.zeros(40, device=DEV), torch.zeros(1, 1, dtype=torch.int64, device=DEV))):
        with pytest.raises(ValueError):
            bad()


# ---------------------------------------------------------------------------------------------------- KGAT's checkpoints
@pytest.mark.parametrize("direct", [False, True])
@pytest.mark.parametrize("dim,layers", [(64, [64, 32, 16]), (256, [256, 128])])
def test_checkpoint_sides_are_let_go_once_read(pkg, K, monkeypatch, dim, layers, direct):
    """The backward holds one layer's sums in full, and no checkpoint of a layer that it is done with."""
    m, U, E = small_model(pkg, dim, layers)
    m.train()
    m.direct_backward, m.checkpoint_sides = direct, True
    rng = np.random.default_rng(2)
    ids = [torch.from_numpy(rng.integers(0, hi, 64)).to(DEV) for hi in (U, int(E * 0.1), int(E * 0.1))]
    kept, alive = [], []
    pack, unpack = K.act8_pack, K.act8_unpack

    def packed(t):
        a = pack(t)
        kept.append(weakref.ref(a.q))
        return a

    def unpacked(a, *more, **named):
        alive.append(sum(r() is not None for r in kept))
        return unpack(a, *more, **named)

    monkeypatch.setattr(K, "act8_pack", packed)
    monkeypatch.setattr(K, "act8_unpack", unpacked)
    m(*ids, mode=pkg.KGATMode.TRAIN_CF).backward()
    assert alive == list(range(len(layers), 0, -1))
    assert not any(r() is not None for r in kept)


# ---------------------------------------------------------------------------------------------------- 8-bit checkpoints
@pytest.mark.parametrize("dtype", TYPES)
def test_act8_wgrad_of_one_share_allocates_its_results_alone(K, dtype):
    """Where the rows are not shared out there are no parts to keep: the call's memory is dW and db."""
    x, dy = randn(gen(1), 64, 1024, dtype=dtype), randn(gen(2), 64, 1000, dtype=dtype)
    a = K.act8_pack(x)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    # bytes asked for: a cached block of which less than 1 MiB would be left is handed out, and counted as allocated, whole
    before = torch.cuda.memory_stats()["requested_bytes.all.current"]
    dW, db = K.act8_wgrad(dy, a)
    assert torch.cuda.memory_stats()["requested_bytes.all.peak"] - before == 4 * 1000 * 1025
    val, _ = act8_ref(x)
    size = dy.to(F64).abs().t() @ val.abs()
    close(dW, dy.to(F64).t() @ val, (8 * math.sqrt(3 * 64) + 32) * 2.0 ** -24 * size, "dW")
    close(db, dy.to(F64).sum(0), SUM * dy.to(F64).abs().sum(0), "db")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("o", [1, 2, 3])
@pytest.mark.parametrize("n,d", [(70, 5000), (3000, 5000), (5, 70001)])
def test_act8_wgrad_of_narrow_outputs_and_wide_inputs(K, n, d, o, dtype):
    """Every column of dW is written (tolerance: see test_act8_wgrad)."""
    x, dy = act8_inputs(n, d, dtype, n), randn(gen(n + o), n, o, dtype=dtype)
    torch.full((o * d + 64,), float("nan"), device=DEV)  # what an unwritten column would show
    dW, db = K.act8_wgrad(dy, K.act8_pack(x))
    val, _ = act8_ref(x)
    few = min(8 * math.sqrt(3 * n) + 32, 3 * n + 1) * 2.0 ** -24
    close(dW, dy.to(F64).t() @ val, few * (dy.to(F64).abs().t() @ val.abs()) + 2.0 ** -140, "dW")
    close(db, dy.to(F64).sum(0), SUM * dy.to(F64).abs().sum(0), "db")


@pytest.mark.parametrize("dtype", TYPES)
def test_act8_error_bound(K, dtype):
    """Within 2^-7 of the block's largest everywhere, clipped values too: a block's largest lies in [64, 128) steps,
    rounding costs at most half a step of 64, clipping a to 127 costs (a - 127) / a < 1 / 128."""
    g = gen(3)
    x = randn(g, 500, 320) * torch.exp2(torch.randint(-8, 8, (500, 1), device=DEV, generator=g).float())
    x[::2, ::32] = torch.linspace(126.5, 127.999, 250, device=DEV)[:, None]  # the topmost steps of a power of two
    x[::2, 1::32] = -x[::2, ::32]
    x = x.to(dtype)
    val = K.act8_unpack(K.act8_pack(x), torch.float32).to(F64)
    top = x.to(F64).abs().view(500, -1, 32).amax(2).repeat_interleave(32, 1)
    assert ((val - x.to(F64)).abs() <= top * 2.0 ** -7 + 2.0 ** -127).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_act8_wgrad_of_tiny_gradients(K, dtype):
    """dy down to its type's smallest numbers: 16-bit types keep every digit, a float's third bf16 term ends at 2^-133."""
    x = randn(gen(1), 64, 40) * 2.0 ** 60
    a = K.act8_pack(x)
    val, _ = act8_ref(x)
    for e in (-8, -14, -20, -24) if dtype == torch.float16 else (-60, -109, -118, -126, -130, -133):
        dy = (torch.randn(64, 48, device=DEV, dtype=F64, generator=gen(-e)) * 2.0 ** e).float().to(dtype)
        dW, db = K.act8_wgrad(dy, a)
        lost = 2.0 ** -133 * val.abs().sum(0) if dtype == torch.float32 else 0.0
        close(dW, dy.to(F64).t() @ val, (8 * math.sqrt(3 * 64) + 32) * 2.0 ** -24 * (dy.to(F64).abs().t() @ val.abs()) + lost, f"dW {e}")
        close(db, dy.to(F64).sum(0), SUM * dy.to(F64).abs().sum(0), f"db {e}")
