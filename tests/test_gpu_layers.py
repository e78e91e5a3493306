"""The dense-head operators as a user has them: the differentiable layers (layers.py), a run of them together, the
held-out likelihood of an evaluation and KGAT's 8-bit side checkpoints.  Tolerances count roundings as
tests/test_gpu_dense.py does."""
from __future__ import annotations

import sys

import numpy as np
import pytest
import torch
import torch.nn.functional as F

from tests.conftest import load_pkg
from tests.test_gpu_dense import SUM, close, gen, half_step, randn

pytestmark = pytest.mark.gpu
DEV = "cuda"
F64 = torch.float64


@pytest.fixture(scope="module")
def pkg():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return load_pkg()


@pytest.fixture(scope="module")
def K(pkg):
    return sys.modules[pkg.__name__ + ".kernels"]


def leaf(t):
    return t.detach().clone().requires_grad_(True)


def double(t):
    return t.detach().to(F64).requires_grad_(True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(7, 40), (3, 5, 64), (130,)])
def test_layer_norm_gradients(pkg, shape, dtype):
    """Against torch's layer norm in 64 bits, any leading dimensions; 2^-17 is what 32-bit statistics of rows of spread
    about 1 are off by (a few SUM), beside the type's own rounding."""
    g = gen(len(shape))
    x, w, b = randn(g, *shape, dtype=dtype), 1 + 0.1 * randn(g, shape[-1]), 0.1 * randn(g, shape[-1])
    dy = randn(g, *shape, dtype=dtype)
    a = [leaf(t) for t in (x, w, b)]
    y = pkg.layers.layer_norm(*a, 1e-5)
    assert y.shape == x.shape and y.dtype == dtype
    y.backward(dy)
    r = [double(t) for t in (x, w, b)]
    ry = F.layer_norm(r[0], shape[-1:], r[1], r[2], 1e-5)
    ry.backward(dy.to(F64))
    tol = 2.0 ** -17
    close(y.detach(), ry.detach(), half_step(dtype) * ry.detach().abs() + tol * 4, "y")
    rows = max(1, x.numel() // shape[-1])
    close(a[0].grad, r[0].grad, half_step(dtype) * r[0].grad.abs() + tol * 16, "dx")
    close(a[1].grad, r[1].grad, tol * 16 * rows, "dw")
    close(a[2].grad, r[2].grad, tol * 4 * rows, "db")


def test_layer_norm_module_and_partial_gradients(pkg):
    m, ref = pkg.layers.LayerNorm(48).to(DEV), torch.nn.LayerNorm(48).to(DEV)
    assert m.state_dict().keys() == ref.state_dict().keys()
    ref.load_state_dict(m.state_dict())
    x = randn(gen(1), 20, 48)
    close(m(x).detach(), ref(x).detach(), 2.0 ** -17 * 4, "module")
    m(x).sum().backward()  # an upstream gradient of stride 0, and no gradient into x
    close(m.bias.grad, torch.full((48,), 20.0, device=DEV), 1e-6, "db")
    xs = leaf(x)
    m.requires_grad_(False)
    m(xs).sum().backward()
    assert xs.grad is not None
    assert pkg.layers.LayerNorm(48, elementwise_affine=False).to(DEV)(x).shape == x.shape
    with torch.no_grad():
        assert not m(x).requires_grad
    for bad in (lambda: pkg.layers.LayerNorm((4, 8)), lambda: m(x[:, :40]), lambda: pkg.layers.layer_norm(x.cpu())):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("dtype,d,o", [(torch.float32, 64, 96), (torch.float32, 33, 17), (torch.bfloat16, 128, 64),
                                       (torch.float16, 40, 3)])
def test_linear_act8(pkg, K, dtype, d, o):
    """Output and input gradient are the exact layer's; the weight's is the product with the checkpoint's values."""
    g = gen(d)
    x, w, b, dy = randn(g, 70, d, dtype=dtype), randn(g, o, d) * 0.2, randn(g, o), randn(g, 70, o, dtype=dtype)
    a = [leaf(t) for t in (x, w, b)]
    y = pkg.layers.linear_act8(*a)
    y.backward(dy)
    wt = w.to(dtype).to(F64)
    ry = x.to(F64) @ wt.t() + b.to(dtype).to(F64)
    size = x.to(F64).abs() @ wt.abs().t() + b.abs()
    # a product of 70 terms summed in 32 bits and rounded, then the bias added and rounded again
    close(y.detach(), ry, 2 * half_step(dtype) * (ry.abs() + b.to(F64).abs()) + d * 2.0 ** -23 * size, "y")
    rdx = dy.to(F64) @ wt
    close(a[0].grad, rdx, half_step(dtype) * rdx.abs() + o * 2.0 ** -23 * (dy.to(F64).abs() @ wt.abs()), "dx")
    x8 = K.act8_unpack(K.act8_pack(x), torch.float32).to(F64)
    close(a[1].grad, dy.to(F64).t() @ x8, SUM * (dy.to(F64).abs().t() @ x8.abs()), "dW")
    close(a[2].grad, dy.to(F64).sum(0), SUM * dy.to(F64).abs().sum(0), "db")
    # parts left out; a module with the plain layer's parameters; leading dimensions
    c = leaf(x)
    pkg.layers.linear_act8(c, w, b).backward(dy)
    assert torch.equal(c.grad, a[0].grad)
    c = leaf(b)
    pkg.layers.linear_act8(x, w, c).backward(dy)
    close(c.grad, a[2].grad, 2 * SUM * dy.to(F64).abs().sum(0), "db alone")
    m = pkg.layers.LinearAct8(d, o).to(DEV)
    assert m.state_dict().keys() == torch.nn.Linear(d, o).state_dict().keys()
    assert m(x.view(7, 10, d)).shape == (7, 10, o)
    for bad in (lambda: pkg.layers.linear_act8(x, w[:, 1:]), lambda: pkg.layers.linear_act8(x, w, b[1:])):
        with pytest.raises(ValueError):
            bad()


def logp_loss(lp, items, weight):
    z = lp
    l = z - torch.logsumexp(z, 1, keepdim=True)
    given = torch.where(items < 0, 0.0, l.gather(1, items.clamp(min=0)))
    p = l.exp()
    return (given * weight).sum() - 0.3 * torch.special.entr(p).sum()


def test_log_probs_gradients(pkg):
    g = gen(4)
    s = randn(g, 6, 300) * 2
    items = torch.randint(0, 300, (6, 3), device=DEV, generator=g)
    items[2, 1], items[3, 2] = -1, items[3, 0]
    weight = randn(g, 6, 3)
    a, r = leaf(s), double(s)
    out = pkg.layers.log_probs(a, items, k=5, scale=0.5)
    assert not out.lse.requires_grad and not out.top_logp.requires_grad
    loss = (out.logp * weight).sum() - 0.3 * out.entropy.sum()
    loss.backward()
    ref = logp_loss(r * 0.5, items, weight.to(F64))
    ref.backward()
    close(loss.detach(), ref.detach(), 1e-5 * (1 + ref.detach().abs()), "loss")
    close(a.grad, r.grad, 2.0 ** -18, "ds")
    # one result alone, and a score row that is a view
    for pick in ("logp", "entropy"):
        a, r = leaf(s), double(s)
        getattr(pkg.layers.log_probs(a.t().contiguous().t(), items), pick).sum().backward()
        l = r - torch.logsumexp(r, 1, keepdim=True)
        if pick == "logp":
            torch.where(items < 0, 0.0, l.gather(1, items.clamp(min=0))).sum().backward()
        else:
            torch.special.entr(l.exp()).sum().backward()
        close(a.grad, r.grad, 2.0 ** -17, pick)
    with torch.no_grad():
        assert pkg.layers.log_probs(s, items).logp.shape == (6, 3)


class Head(torch.nn.Module):
    """User vectors through a normalised hidden layer onto the catalogue's vectors."""

    def __init__(self, layers, d, hidden):
        super().__init__()
        self.layers = layers
        self.norm0, self.norm1 = layers.LayerNorm(d), layers.LayerNorm(hidden)
        self.lin = layers.LinearAct8(d, hidden)

    def forward(self, users, items):
        x = self.norm0(users)
        return self.norm1(torch.relu(self.lin(x))) @ items.t(), x


def test_layers_together(pkg, K):
    """One training step of a listwise loss over the catalogue, every gradient against autograd in 64 bits with the
    checkpoint's values in the linear layer's weight gradient."""
    torch.manual_seed(3)
    g = gen(12)
    B, d, hidden, C = 37, 64, 48, 1100
    head = Head(pkg.layers, d, hidden).to(DEV)
    users, items = leaf(randn(g, B, d)), leaf(randn(g, C, hidden) * 0.5)
    held = torch.randint(0, C, (B, 2), device=DEV, generator=g)
    held[5, 1] = -1
    scores, x = head(users, items)
    out = pkg.layers.log_probs(scores, held, k=4)
    loss = -(out.logp.sum() + 0.1 * out.entropy.sum()) / B
    loss.backward()

    p = {k: double(v) for k, v in head.named_parameters()}
    u, v = double(users), double(items)
    x8 = K.act8_unpack(K.act8_pack(x.detach())).to(F64)
    h0 = F.layer_norm(u, (d,), p["norm0.weight"], p["norm0.bias"])
    W = p["lin.weight"]
    lin = h0 @ W.detach().t() + x8 @ (W - W.detach()).t() + p["lin.bias"]
    h = F.layer_norm(torch.relu(lin), (hidden,), p["norm1.weight"], p["norm1.bias"])
    z = h @ v.t()
    l = z - torch.logsumexp(z, 1, keepdim=True)
    ref = -(torch.where(held < 0, 0.0, l.gather(1, held.clamp(min=0))).sum() + 0.1 * torch.special.entr(l.exp()).sum()) / B
    ref.backward()
    close(loss.detach(), ref.detach(), 1e-5 * (1 + ref.detach().abs()), "loss")
    assert torch.equal(out.top_items, torch.topk(scores.detach(), 4, dim=1)[1])
    # a dozen 32-bit operations between the loss and each gradient, of sums of up to 1100 terms
    for name, a, r in [("users", users, u), ("items", items, v)] + [(k, q, p[k]) for k, q in head.named_parameters()]:
        close(a.grad, r.grad, 2.0 ** -16 * (r.grad.abs() + r.grad.abs().mean() * 4), name)


def test_layers_step_in_a_captured_graph(pkg):
    """The whole step captured (warmed up on the capture's stream, no eager graph alive) and replayed on new inputs."""
    torch.manual_seed(5)
    g = gen(2)
    head = Head(pkg.layers, 64, 32).to(DEV)
    items = randn(g, 500, 32)
    users, held = randn(g, 16, 64), torch.randint(0, 500, (16, 1), device=DEV, generator=g)
    params = list(head.parameters())

    def step():
        scores, _ = head(users, items)
        grads = torch.autograd.grad(-pkg.layers.log_probs(scores, held).logp.mean(), params)
        return [q.detach() for q in grads]

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
        users.copy_(randn(g, 16, 64))
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in got]
        assert all(torch.equal(a, b) for a, b in zip(kept, step())), turn


def small_model(pkg, dim, layers, seed=5):
    graph = sys.modules[pkg.__name__ + ".graph"]
    U, E, inter, trip = graph.synthetic_ckg(6000, 60000, seed=seed)
    lay = graph.build_layout(U, E, inter, trip)
    torch.manual_seed(31)
    m = pkg.KGAT(pkg.KGATArgs(user_num=U, entity_num=E, relation_num=len(lay.rel_order), layer_size=layers,
                              cf_embedding_dim=dim, kg_embedding_dim=dim, message_dropout=[0.1] * len(layers)))
    m.attach_graph(lay, DEV)
    m.build_optimizer(cf_lr=1e-3, kg_lr=1e-4)
    return m, U, E


@pytest.mark.parametrize("direct", [False, True])
@pytest.mark.parametrize("dim,layers", [(64, [64, 32]), (64, [64, 32, 16]), (128, [128, 64, 32]), (256, [256, 128])])
def test_checkpoint_sides(pkg, K, dim, layers, direct, monkeypatch):
    """KGAT.checkpoint_sides: the same loss bits, and the gradients of a step whose backward is handed the checkpoint's
    values, bit for bit; the frontier forward keeps its rows whole."""
    m, U, E = small_model(pkg, dim, layers)
    m.train()
    m.direct_backward = direct
    rng = np.random.default_rng(2)
    ids = [torch.from_numpy(rng.integers(0, hi, 64)).to(DEV) for hi in (U, int(E * 0.1), int(E * 0.1))]

    def step():
        torch.manual_seed(8)
        m.zero_grad(set_to_none=True)
        loss = m(*ids, mode=pkg.KGATMode.TRAIN_CF)
        loss.backward()
        return loss.detach().clone(), [p.grad.clone() for p in m.parameters() if p.grad is not None]

    exact = step()
    m.checkpoint_sides = True
    packs = []
    real = K.act8_pack
    monkeypatch.setattr(K, "act8_pack", lambda t: packs.append(t.shape) or real(t))
    got = step()
    assert len(packs) == len(layers)
    m.checkpoint_sides = False
    model = sys.modules[pkg.__name__ + ".model"]
    monkeypatch.setattr(model, "_side", lambda sides, l: K.act8_unpack(real(sides[l])))
    want = step()
    assert torch.equal(got[0], exact[0]) and torch.equal(got[0], want[0])
    assert len(got[1]) == len(want[1]) == len(exact[1])
    assert all(torch.equal(a, b) for a, b in zip(got[1], want[1]))
    assert not all(torch.equal(a, b) for a, b in zip(got[1], exact[1]))
    for a, b in zip(got[1], exact[1]):  # and near the exact sums' gradients
        assert (a - b).norm() <= 2.0 ** -5 * b.norm()
    monkeypatch.undo()
    m.checkpoint_sides = True
    with torch.no_grad():
        assert torch.isfinite(m(*ids, mode=pkg.KGATMode.TRAIN_CF))


@pytest.mark.parametrize("many", [False, True])
def test_log_likelihood(pkg, many):
    """evaluation.log_likelihood against the softmax of the model's masked scores in 64 bits; ``many``: more held-out
    items than one call takes."""
    m, U, E = small_model(pkg, 64, [64, 32])
    n_items = 1500
    rng = np.random.default_rng(7)
    users = [3, 9, 4, 77, 100]
    train = {u: rng.choice(n_items, 20, replace=False).tolist() for u in users}
    held = {u: [i for i in rng.choice(n_items, 1200 if many and u == 9 else 5, replace=False).tolist() if i not in train[u]]
            for u in users}
    held[4] = []
    res, per = pkg.evaluation.log_likelihood(m, train, held, n_items, scale=2.0, batch_size=2, return_per_user=True)
    kern = sys.modules[pkg.__name__ + ".kernels"]
    sc = kern.scores(m.propagate(), torch.tensor(users, device=DEV), torch.arange(n_items, device=DEV)).to(F64) * 2.0
    want_l, want_e = [], []
    for r, u in enumerate(users):
        sc[r, train[u]] = -float("inf")
        l = sc[r] - torch.logsumexp(sc[r], 0)
        want_e.append(torch.special.entr(l.exp()).sum().item())
        want_l.append(l[held[u]].mean().item() if held[u] else float("nan"))
    np.testing.assert_allclose(per["log_likelihood"], want_l, rtol=1e-5)
    np.testing.assert_allclose(per["entropy"], want_e, rtol=1e-5)
    mean = np.nanmean(want_l)
    np.testing.assert_allclose(res["log_likelihood"], mean, rtol=1e-5)
    np.testing.assert_allclose(res["perplexity"], np.exp(-mean), rtol=1e-4)
    np.testing.assert_allclose(res["entropy"], np.mean(want_e), rtol=1e-5)
    with pytest.raises(IndexError):
        pkg.evaluation.log_likelihood(m, train, {3: [n_items]}, n_items)
    empty = pkg.evaluation.log_likelihood(m, {}, {}, n_items)
    assert np.isnan(empty["log_likelihood"]) and np.isnan(empty["entropy"])


def test_linear_act8_types_and_refusals(pkg):
    """Autocast leaves the types alone; the wrong device or type is refused with and without a gradient."""
    x = torch.randn(6, 7, device="cuda", requires_grad=True)
    w, b = torch.randn(5, 7, device="cuda", requires_grad=True), torch.randn(5, device="cuda")
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = pkg.layers.linear_act8(x, w, b)
    assert y.dtype is torch.float32
    y.sum().backward()
    # sums of 5 products of O(1) numbers: 5 roundings of at most 2^-24 of the terms' sum each, on both sides
    want = w.detach().double().sum(0).expand(6, 7)
    assert ((x.grad.double() - want).abs() <= 10 * 2.0 ** -24 * w.detach().double().abs().sum(0)).all()
    for grad in (False, True):
        with torch.set_grad_enabled(grad):
            for bad in (lambda: pkg.layers.linear_act8(x.cpu(), w, b), lambda: pkg.layers.linear_act8(x, w.cpu(), b),
                        lambda: pkg.layers.linear_act8(x, w, b.cpu()), lambda: pkg.layers.linear_act8(x.double(), w, b),
                        lambda: pkg.layers.linear_act8(x, w[:, :6], b), lambda: pkg.layers.linear_act8(x, w, b[:4])):
                with pytest.raises(ValueError):
                    bad()
