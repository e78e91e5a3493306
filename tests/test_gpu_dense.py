"""The dense-head operators (csrc/layer_norm.hip, act8.hip, log_prob.hip) against their definitions in 64 bits.

Tolerances.  A result rounded to a type is off by at most half a step, eps(t) / 2 of its value; 32-bit sums of m terms
by at most about log2(m) + 8 roundings of 2^-24 of the sum of the terms' absolute values where threads sum trees of
short runs (HALF below counts 32 of them: 2^-19), and an exponential's argument x by 2^-24 |x|, which its power
carries as a relative error."""
from __future__ import annotations

import math

import pytest
import torch

from tests.conftest import load_pkg

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float32, torch.bfloat16, torch.float16]
SUM = 2.0 ** -19  # 32 roundings of 2^-24
F64 = torch.float64


@pytest.fixture(scope="module")
def K():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return __import__(load_pkg().__name__ + ".kernels", fromlist=["kernels"])


def half_step(t):
    return torch.finfo(t).eps / 2


def least(t):
    """What is lost below a type's normal numbers: fp16 keeps its subnormal steps, the others may go to zero."""
    f = torch.finfo(t)
    return f.smallest_normal * (f.eps if t == torch.float16 else 1)


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, device=DEV, generator=g).to(dtype)


def strided(x, extra=3, offset=1):
    """The same rows, at an odd offset and leading dimension."""
    n, d = x.shape
    big = torch.full((n, d + extra), float("nan"), dtype=x.dtype, device=x.device)
    big[:, offset:offset + d] = x
    return big[:, offset:offset + d]


def close(got, want, tol, what=""):
    """|got - want| <= tol (a tensor or a number) everywhere; NaN and infinities where the other has them."""
    got, want = got.to(F64), want.to(F64)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)]), what
    tol = torch.as_tensor(tol, dtype=F64, device=got.device).expand(want.shape)
    bad = ((got - want).abs() > tol) & fine
    if bad.any():
        i = tuple(x.item() for x in bad.nonzero()[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {i}: {got[i].item()} against "
                             f"{want[i].item()}, allowed {tol[i].item()}")


# ---------------------------------------------------------------------------------------------------- layer norm
def norm_ref(x, w, b, eps, dy=None):
    x = x.to(F64)
    mean = x.mean(1, keepdim=True)
    xc = x - mean
    rstd = 1 / (xc.square().mean(1, keepdim=True) + eps).sqrt()
    xhat = xc * rstd
    y = xhat * (1 if w is None else w.to(F64)) + (0 if b is None else b.to(F64))
    if dy is None:
        return y, mean[:, 0], rstd[:, 0], xhat
    dy = dy.to(F64)
    g = dy * (1 if w is None else w.to(F64))
    dx = rstd * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
    return y, mean[:, 0], rstd[:, 0], xhat, g, dx, (dy * xhat).sum(0), dy.sum(0)


def norm_inputs(n, d, dtype, w_dtype, seed):
    g = gen(seed)
    x = (randn(g, n, d) * (0.5 + torch.rand(n, 1, device=DEV, generator=g)) + 0.5).to(dtype)
    w = None if w_dtype is None else (1 + 0.2 * randn(g, d)).to(w_dtype)
    b = None if w_dtype is None else (0.1 * randn(g, d)).to(w_dtype)
    return x, w, b, randn(g, n, d, dtype=dtype)


NORM_SHAPES = [(1, 1), (1, 64), (3, 2), (5, 7), (17, 33), (2, 64), (129, 63), (300, 65), (1000, 128), (37, 255),
               (64, 257), (33, 511), (9, 1021), (20, 1024), (7, 2047), (6, 2049), (5, 4096), (3, 4100), (3, 8191),
               (2, 8193), (2, 16384), (3, 16399), (2, 32769), (2, 70001), (4099, 16), (20011, 8),
               # several rows a block with the sums in LDS, and wider rows in shares
               (600, 9001), (515, 16384), (70, 16399), (37, 20000)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,d", NORM_SHAPES)
def test_layer_norm(K, n, d, dtype):
    """Forward and backward; the values' error counts the type's last rounding, and 32-bit statistics: mean and var
    carry SUM of the row's mean |x| and mean square, which xhat sees divided by the row's spread."""
    w_dtype = [torch.float32, dtype, None][(n + d) % 3]
    x, w, b, dy = norm_inputs(n, d, dtype, w_dtype, n * 31 + d)
    eps = 1e-5
    y, mean, rstd = K.layer_norm_fwd(x, w, b, eps, stats=True)
    assert torch.equal(y, K.layer_norm_fwd(x, w, b, eps)) or d == 0
    ry, rmean, rrstd, xhat, g, rdx, rdw, rdb = norm_ref(x, w, b, eps, dy)
    xd = x.to(F64)
    big = xd.abs().mean(1)
    close(mean, rmean, SUM * big, "mean")
    spread = SUM * (1 + big * rrstd)  # relative error of xc / sd: the mean's, and var's
    close(rstd, rrstd, spread * rrstd, "rstd")
    wa = torch.ones(d, device=DEV, dtype=F64) if w is None else w.to(F64).abs()
    off = spread[:, None] * (xhat.abs() + 1)
    close(y, ry, half_step(dtype) * ry.abs() + off * wa + SUM * ry.abs() + least(dtype), "y")
    dx, dw, db = K.layer_norm_bwd(dy, x, mean, rstd, w)
    ga = g.abs().mean(1, keepdim=True)
    gx = (g * xhat).abs().mean(1, keepdim=True)
    off = (g.abs() + ga + (xhat.abs() + 1) * gx) * rrstd[:, None] * 4 * spread[:, None]
    close(dx, rdx, half_step(dtype) * rdx.abs() + off + least(dtype), "dx")
    wt = torch.float32 if w is None else w.dtype
    dya = dy.to(F64).abs()
    off = (dya * (xhat.abs() + 1) * 2 * spread[:, None]).sum(0) + SUM * (dya * xhat.abs()).sum(0)
    close(dw, rdw, off + half_step(wt) * rdw.abs(), "dweight")
    close(db, rdb, SUM * dya.sum(0) + half_step(wt) * rdb.abs(), "dbias")
    # the same bits again, from views at odd offsets and leading dimensions, and with parts left out
    y2, m2, r2 = K.layer_norm_fwd(strided(x), w, b, eps, stats=True)
    assert torch.equal(y, y2) and torch.equal(mean, m2) and torch.equal(rstd, r2)
    dx2, dw2, db2 = K.layer_norm_bwd(strided(dy, 5, 3), strided(x), mean, rstd, w)
    assert torch.equal(dx, dx2) and torch.equal(dw, dw2) and torch.equal(db, db2)
    a = K.layer_norm_bwd(dy, x, mean, rstd, w, need_dweight=False, need_dbias=False)
    assert torch.equal(a[0], dx) and a[1] is None and a[2] is None
    a = K.layer_norm_bwd(dy, x, mean, rstd, w, need_dx=False, need_dbias=False)
    assert a[0] is None and torch.equal(a[1], dw) and a[2] is None
    a = K.layer_norm_bwd(dy, x, mean, rstd, w, need_dx=False, need_dweight=False)
    assert a[1] is None and torch.equal(a[2], db)


def test_layer_norm_weight_alone_or_bias_alone(K):
    x, w, b, _ = norm_inputs(9, 70, torch.float32, torch.float32, 3)
    one, zero = torch.ones(70, device=DEV), torch.zeros(70, device=DEV)
    assert torch.equal(K.layer_norm_fwd(x, w, None), K.layer_norm_fwd(x, w, zero))
    close(K.layer_norm_fwd(x, None, b), K.layer_norm_fwd(x, one, b), 2.0 ** -24 * 8, "bias alone")


def test_layer_norm_long_reduction(K):
    """dweight / dbias over 300,001 rows."""
    x, w, b, dy = norm_inputs(300001, 24, torch.float32, torch.float32, 8)
    _, mean, rstd = K.layer_norm_fwd(x, w, b, stats=True)
    _, dw, db = K.layer_norm_bwd(dy, x, mean, rstd, w)
    *_, xhat, g, rdx, rdw, rdb = norm_ref(x, w, b, 1e-5, dy)
    dya = dy.to(F64).abs()
    close(dw, rdw, SUM * (dya * (xhat.abs() + 1)).sum(0) * 4, "dweight")
    close(db, rdb, SUM * dya.sum(0), "dbias")


def test_layer_norm_degenerate_rows(K):
    """A constant row has variance 0 (y = bias); an infinity or a NaN spoils its own row alone; no rows at all."""
    x = torch.full((4, 40), 3.0, device=DEV)
    x[1] = torch.arange(40, device=DEV)
    x[2, 7] = float("inf")
    x[3, 39] = float("nan")
    w, b = torch.full((40,), 2.0, device=DEV), torch.full((40,), 0.25, device=DEV)
    y, mean, rstd = K.layer_norm_fwd(x, w, b, 1e-5, stats=True)
    assert torch.equal(y[0], b) and torch.isnan(y[2:]).all() and torch.isfinite(y[1]).all()
    dy = torch.ones_like(x)
    dx, _, db = K.layer_norm_bwd(dy, x, mean, rstd, w)
    assert torch.isfinite(dx[:2]).all() and torch.isnan(dx[2:]).all() and torch.equal(db, torch.full_like(b, 4.0))
    e = torch.empty(0, 40, device=DEV)
    y, mean, rstd = K.layer_norm_fwd(e, w, b, stats=True)
    dx, dw, db = K.layer_norm_bwd(e, e, mean, rstd, w)
    assert y.shape == dx.shape == (0, 40) and not dw.any() and not db.any()


def test_layer_norm_offset_rows_keep_their_digits(K):
    """Rows far from zero: the deviations are taken from the mean, not from a difference of squares."""
    g = gen(5)
    x = randn(g, 50, 96) + 4096
    y = K.layer_norm_fwd(x)
    ry, *_ = norm_ref(x, None, None, 1e-5)
    # the mean is within 8 roundings of 2^-24 of 4096, and that shifts xhat (spread about 1) by as much
    close(y, ry, 8 * 2.0 ** -24 * 4096 + SUM * 5, "y")


def test_layer_norm_broadcast_inputs(K):
    """One row shown n times (stride 0)."""
    x, w, b, dy = norm_inputs(1, 77, torch.bfloat16, torch.float32, 4)
    xs, dys = x.expand(50, 77), dy.expand(50, 77)
    y, mean, rstd = K.layer_norm_fwd(xs, w, b, stats=True)
    assert torch.equal(y, K.layer_norm_fwd(x, w, b).expand(50, 77))
    a = K.layer_norm_bwd(dys, xs, mean, rstd, w)
    c = K.layer_norm_bwd(dys.contiguous(), xs.contiguous(), mean, rstd, w)
    assert all(torch.equal(p, q) for p, q in zip(a, c))


# ---------------------------------------------------------------------------------------------------- 8-bit checkpoints
def act8_ref(x):
    """(values in float64, codes) of the checkpoint's definition."""
    n, d = x.shape
    pad = -d % 32
    v = torch.nn.functional.pad(x.to(F64), (0, pad)).view(n, -1, 32)
    top = v.abs().amax(2, keepdim=True)
    bad = ~torch.isfinite(v).all(2, keepdim=True)
    e = (torch.frexp(torch.where(bad, 1.0, top))[1] - 7).clamp(min=-126)
    e = torch.where(top == 0, -126, e)  # frexp gives 0 the exponent 0, its logarithm is -infinity
    q = torch.round(v / torch.exp2(e.to(F64))).clamp(-127, 127)
    val = torch.where(bad, float("nan"), q * torch.exp2(e.to(F64)))
    return val.view(n, -1)[:, :d], torch.where(bad, 255, e + 127)[:, :, 0].to(torch.uint8)


def act8_inputs(n, d, dtype, seed):
    g = gen(seed)
    x = randn(g, n, d) * torch.exp2(torch.randint(-12, 8, (n, 1), device=DEV, generator=g).float())
    x[::3, ::5] = 0
    return x.to(dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,d", [(1, 1), (1, 32), (2, 31), (3, 33), (7, 64), (100, 65), (257, 129), (64, 1000), (5, 4096),
                                 (3, 5001), (2049, 16), (1, 100001)])
def test_act8_pack_unpack(K, n, d, dtype):
    """Every value to the bit (float and bf16 hold it; fp16 to half a step, or of its smallest normal's)."""
    x = act8_inputs(n, d, dtype, n + d)
    a = K.act8_pack(x)
    val, code = act8_ref(x)
    assert torch.equal(a.e, code)
    assert a.q.shape == (n, -(-d // 32) * 32) and not a.q[:, d:].any()
    assert torch.equal(K.act8_unpack(a, torch.float32).to(F64), val)
    assert torch.equal(K.act8_unpack(a, torch.bfloat16).to(F64), val)
    assert torch.equal(K.act8_unpack(a, torch.float16), val.to(torch.float16))
    assert K.act8_unpack(a).dtype == dtype
    b = K.act8_pack(strided(x))
    assert torch.equal(a.q, b.q) and torch.equal(a.e, b.e)
    out = torch.full((n, d + 5), 9.0, dtype=torch.float32, device=DEV)
    K.act8_unpack(a, out=out[:, 2:2 + d])
    assert torch.equal(out[:, 2:2 + d].to(F64), val) and (out[:, :2] == 9).all() and (out[:, 2 + d:] == 9).all()
    # the promise: within 2^-7 of the block's largest, 2^-6 in its topmost 1/255
    top = torch.nn.functional.pad(x.to(F64).abs(), (0, -d % 32)).view(n, -1, 32).amax(2).repeat_interleave(32, 1)[:, :d]
    err = (val - x.to(F64)).abs()
    assert (err <= top * 2.0 ** -6 + 2.0 ** -127).all()
    assert (err <= top * 2.0 ** -7 + 2.0 ** -127)[x.to(F64).abs() < top * 254 / 255].all()


def test_act8_borders(K):
    """The largest and smallest floats, values that round up to the next power, ties, zeros, infinities and NaN."""
    big = torch.finfo(torch.float32).max
    tiny = 2.0 ** -149
    rows = torch.zeros(10, 64, device=DEV)
    rows[0, :3] = torch.tensor([big, -big, big / 300])
    rows[1, :3] = torch.tensor([tiny, -tiny, 2.0 ** -126])
    rows[2, :4] = torch.tensor([127.75, 127.5, -127.75, 0.5])       # clipped at 127
    rows[3, :6] = torch.tensor([64.0, 0.5, 1.5, 2.5, -0.5, -1.5])   # ties to even
    rows[4, 5] = float("inf")
    rows[5, 33] = float("nan")
    rows[6, 31], rows[6, 32] = 1.0, -float("inf")
    rows[7, :2] = torch.tensor([2.0 ** -120, 2.0 ** -127])
    rows[8, :] = -1.0
    a = K.act8_pack(rows)
    val, code = act8_ref(rows)
    assert torch.equal(a.e, code)
    got = K.act8_unpack(a).to(F64)
    assert torch.equal(torch.isnan(got), torch.isnan(val))
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(val))
    assert (a.e[9] == 1).all() and not a.q[9].any()
    h = torch.zeros(1, 32, dtype=torch.float16, device=DEV)
    h[0, 0], h[0, 1] = 65504, 2.0 ** -24
    assert torch.equal(K.act8_unpack(K.act8_pack(h)).to(F64), act8_ref(h)[0])


WGRAD_SHAPES = [(1, 1, 1), (1, 64, 64), (2, 3, 5), (63, 17, 33), (64, 128, 128), (65, 129, 127), (513, 64, 257),
                (1000, 131, 67), (2048, 64, 64), (4099, 200, 96), (30011, 33, 40), (700, 300, 520), (1025, 513, 260),
                # tiles of 256, whole and in shares
                (333, 4001, 3999), (20000, 2000, 2041)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,o,d", WGRAD_SHAPES)
def test_act8_wgrad(K, n, o, d, dtype):
    """The products are exact, so only 32-bit sums of n terms are off: 2^-24 a term at the worst, and rounding errors of
    independent signs leave a few square roots of n of them (8 sqrt(n) + 32 are allowed)."""
    g = gen(n + 7 * o + d)
    x = act8_inputs(n, d, dtype, n * d)
    dy = randn(g, n, o) * torch.exp2(torch.randint(-6, 3, (n, 1), device=DEV, generator=g).float())
    dy = dy.to(dtype)
    a = K.act8_pack(x)
    dW, db = K.act8_wgrad(dy, a)
    val, _ = act8_ref(x)
    r = dy.to(F64).t() @ val
    size = dy.to(F64).abs().t() @ val.abs()
    terms = 3 * n  # a float dy goes in as three
    few = min(8 * math.sqrt(terms) + 32, terms + 1) * 2.0 ** -24
    close(dW, r, few * size + 2.0 ** -140, "dW")
    close(db, dy.to(F64).sum(0), SUM * dy.to(F64).abs().sum(0), "db")
    dW2, db2 = K.act8_wgrad(strided(dy), a)
    assert torch.equal(dW, dW2) and torch.equal(db, db2)
    dW3, none = K.act8_wgrad(dy, a, bias=False)
    assert none is None and torch.equal(dW, dW3)


@pytest.mark.parametrize("dtype", TYPES)
def test_act8_wgrad_products_are_exact(K, dtype):
    """One row: dW is a single product of dy and x, each with all its bits, so the result is its one rounding."""
    g = gen(11)
    x = act8_inputs(1, 200, torch.float32, 5)
    dy = randn(g, 1, 150, dtype=dtype)
    dW, db = K.act8_wgrad(dy, K.act8_pack(x))
    val, _ = act8_ref(x)
    # three terms of a float are summed in 32 bits: two roundings more than the product's own
    close(dW, dy.to(F64).t() @ val, (dy.to(F64).abs().t() @ val.abs()) * 3 * 2.0 ** -24, "dW")
    assert torch.equal(db, dy[0].float())


@pytest.mark.parametrize("x_type,dy_type", [(a, b) for a in TYPES for b in TYPES if a is not b])
@pytest.mark.parametrize("n,o,d", [(70, 3, 33), (900, 64, 70), (3000, 257, 130), (200, 1500, 1400)])
def test_act8_wgrad_mixed_types(K, n, o, d, x_type, dy_type):
    """x packed from one type and dy of another (tolerance: see test_act8_wgrad)."""
    g = gen(n + o)
    x = act8_inputs(n, d, x_type, n)
    dy = randn(g, n, o).to(dy_type)
    dW, db = K.act8_wgrad(dy, K.act8_pack(x))
    val, _ = act8_ref(x)
    few = min(8 * math.sqrt(3 * n) + 32, 3 * n + 1) * 2.0 ** -24
    close(dW, dy.to(F64).t() @ val, few * (dy.to(F64).abs().t() @ val.abs()) + 2.0 ** -140, "dW")
    close(db, dy.to(F64).sum(0), SUM * dy.to(F64).abs().sum(0), "db")


def test_act8_of_fp16_is_fp16(K):
    """Every finite fp16 number as a block's largest, beside smaller ones of every size: the values are fp16 numbers, and
    products with the smallest of them are not lost."""
    bits = torch.arange(1, 0x7C00, device=DEV, dtype=torch.int32).to(torch.int16)
    top = bits.view(torch.float16)
    scale = torch.exp2(-torch.arange(32, device=DEV, dtype=torch.float32))
    x = (top.float()[:, None] * scale * (1 - 2 * (torch.arange(32, device=DEV) % 2))).half()
    a = K.act8_pack(x)
    v = K.act8_unpack(a, torch.float32)
    assert torch.equal(v.half().float(), v)
    assert torch.equal(K.act8_unpack(a).float(), v)
    # one row at a time: a product's only rounding is to 32 bits; 2^-24 is fp16's smallest number
    for i in (0, 1, 5, 1022, 1023, 1024, 5000, 20000, 31742):
        for dy in (torch.tensor([[1.0, 2.0 ** -24, -3 * 2.0 ** -24, 65504.0, 2.0 ** -14]], device=DEV).half(),):
            dW, db = K.act8_wgrad(dy, K.act8_pack(x[i:i + 1]))
            want = dy.to(F64).t() @ v[i:i + 1].to(F64)
            assert torch.equal(dW.to(F64), want), i  # 11 + 7 bits: exact in 32
            assert torch.equal(db, dy[0].float())


def test_act8_wgrad_not_a_number(K):
    """A NaN block of x spoils its 32 columns of dW, a NaN or an infinity in dy its row of dW; no row spoils others."""
    g = gen(2)
    x, dy = randn(g, 300, 100), randn(g, 300, 70)
    x[7, 40] = float("nan")
    dy[9, 3], dy[200, 5] = float("inf"), float("nan")
    dW, db = K.act8_wgrad(dy, K.act8_pack(x))
    bad = torch.zeros(70, 100, dtype=torch.bool, device=DEV)
    bad[:, 32:64] = True
    bad[3], bad[5] = True, True
    assert torch.equal(torch.isnan(dW), bad)
    assert torch.isnan(db[5]) and torch.isinf(db[3]) and torch.isfinite(db[[0, 1, 2, 4, 6]]).all()


def test_act8_wgrad_no_rows(K):
    a = K.act8_pack(torch.empty(0, 40, device=DEV))
    dW, db = K.act8_wgrad(torch.empty(0, 30, device=DEV), a)
    assert dW.shape == (30, 40) and not dW.any() and not db.any()
    assert K.act8_unpack(a).shape == (0, 40)


# ---------------------------------------------------------------------------------------------------- log probabilities
def logp_ref(s, items, k, scale, dlogp=None, dent=None):
    z, c = s.to(F64), s.shape[1]
    bad = torch.isnan(z).any(1) | torch.isposinf(z).any(1)
    top = z.amax(1, keepdim=True)
    none = torch.isneginf(top[:, 0])
    top = torch.where(torch.isfinite(top), top, 0.0)
    z = (z - top) * scale  # the difference first: far from zero a logarithm of a few is lost in the sum, in 64 bits too
    lse = torch.logsumexp(z, 1)
    lp = z - torch.where(none, 0.0, lse)[:, None]
    lse = lse + top[:, 0] * scale
    p = lp.exp()
    h = torch.special.entr(p).sum(1)
    logp = lp.gather(1, items.clamp(0, c - 1))
    logp = torch.where(items < 0, 0.0, torch.where(bad[:, None] | (items >= c), float("nan"), logp))
    out = {"logp": logp, "lse": torch.where(bad, float("nan"), lse), "entropy": torch.where(bad, float("nan"), h)}
    if k:
        key = s.float() + 0.0
        top = torch.sort(torch.nan_to_num(key, nan=0.0, posinf=float("inf"), neginf=-float("inf")), dim=1, descending=True,
                         stable=True)[1][:, :k]
        out["top_items"] = torch.where(bad[:, None], -1, top)
        out["top_logp"] = torch.where(bad[:, None], float("nan"), lp.gather(1, top))
    if dlogp is not None:
        g = torch.where(items < 0, 0.0, torch.where(items >= c, float("nan"), dlogp.to(F64)))
        e = torch.zeros_like(z) if dent is None else dent.to(F64)[:, None] * (torch.xlogy(p, p) + p * h[:, None])
        own = torch.zeros_like(z).scatter_add_(1, items.clamp(0, c - 1), torch.where(items < 0, 0.0, torch.nan_to_num(g)))
        ds = scale * (own - p * g.sum(1, keepdim=True) - e)
        out["dscores"] = torch.where(bad[:, None], float("nan"), torch.where(none[:, None], 0.0, ds))
        out["size"] = scale * (own.abs() + p * (torch.nan_to_num(g).abs().sum(1, keepdim=True) + (
            0 if dent is None else dent.to(F64).abs()[:, None] * (torch.nan_to_num(lp, neginf=0.0).abs() + h[:, None]))))
    return out


def logp_inputs(n, c, t, dtype, seed, masked=0.2, spread=3.0):
    g = gen(seed)
    s = randn(g, n, c) * spread
    s[torch.rand(n, c, device=DEV, generator=g) < masked] = -float("inf")
    if n:
        s[:, 0] = torch.where(torch.isneginf(s[:, 0]), 0.5, s[:, 0])  # something is left
    items = torch.randint(0, c, (n, t), device=DEV, generator=g)
    items[torch.rand(n, t, device=DEV, generator=g) < 0.1] = -1
    if t > 2 and n:
        items[:, 2] = items[:, 1]  # the same item twice
    dlogp = randn(g, n, t)
    return s.to(dtype), items, dlogp, randn(g, n)


def check_logp(K, s, items, k, scale, dlogp, dent):
    r = K.log_prob_fwd(s, items, k=k, scale=scale)
    ref = logp_ref(s, items, k, scale, dlogp, dent)
    # an argument t = (s - max) scale is off by 2 roundings (difference, product), exp2's by 2^-22 |t| with the factor
    # log2 e, sums by SUM: log S by SUM + 2^-21 of the weighted mean |t|, which the entropy is (+ log S)
    z = torch.nan_to_num(s.to(F64) * scale, nan=0.0, posinf=0.0, neginf=0.0)
    size = z.abs().amax(1)
    hmax = ref["entropy"].nan_to_num().abs() + math.log(max(2, s.shape[1]))
    low = 2.0 ** -21 * (size + hmax) + SUM * (1 + hmax)
    near = torch.nan_to_num(ref["logp"], neginf=0.0).abs()
    close(r.logp, ref["logp"], low[:, None] + 2.0 ** -22 * near, "logp")
    close(r.lse, ref["lse"], low, "lse")
    close(r.entropy, ref["entropy"], low, "entropy")
    assert (r.top_items is None) == (k == 0)
    if k:
        assert torch.equal(r.top_items, ref["top_items"])
        close(r.top_logp, ref["top_logp"], low[:, None] + 2.0 ** -22 * ref["top_logp"].nan_to_num(neginf=0.0).abs(), "top")
    ds = K.log_prob_bwd(s, items, r.stats, dlogp, dent, scale=scale)
    # p is off by its argument's error, relative
    off = ref["size"] * (4 * low[:, None] + 2.0 ** -21 * (1 + torch.nan_to_num(z - ref["lse"].nan_to_num(neginf=0.0)[:, None]).abs()))
    close(ds, ref["dscores"], off + half_step(s.dtype) * ref["dscores"].nan_to_num().abs() +
          least(s.dtype), "dscores")
    return r, ds


LOGP_SHAPES = [(1, 1, 1, 1), (1, 2, 1, 2), (3, 5, 2, 5), (4, 63, 1, 63), (2, 64, 3, 64), (5, 65, 4, 65), (7, 127, 1, 100),
               (2, 128, 20, 128), (9, 257, 1, 1), (33, 1000, 3, 20), (300, 1021, 5, 7), (1, 4097, 4, 128),
               (3, 9500, 20, 100), (600, 4100, 1, 0), (1, 16385, 1, 20), (2, 50001, 6, 64), (3, 100003, 2, 128),
               (1, 300007, 1024, 0), (70, 20000, 4, 33), (1100, 300, 1, 0)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,c,t,k", LOGP_SHAPES)
def test_log_prob(K, n, c, t, k, dtype):
    s, items, dlogp, dent = logp_inputs(n, c, t, dtype, n + c + k)
    scale = [1.0, 0.37][n % 2]
    r, ds = check_logp(K, s, items, k, scale, dlogp, dent)
    # views, the same bits again, one output alone, and the gradient in the scores' place
    r2 = K.log_prob_fwd(strided(s), items, k=k, scale=scale)
    for a, b in zip(r, r2):
        assert (a is None and b is None) or torch.equal(a, b)
    assert torch.equal(ds, K.log_prob_bwd(strided(s), items, r.stats, dlogp, dent, scale=scale))
    place = s.clone()
    assert K.log_prob_bwd(place, items, r.stats, dlogp, dent, scale=scale, out=place) is place
    assert torch.equal(place, ds)
    check_logp(K, s, items, 0, scale, dlogp, None)


def test_log_prob_without_items(K):
    s, items, dlogp, dent = logp_inputs(5, 700, 0, torch.float32, 1)
    r, ds = check_logp(K, s, items, 10, 1.0, dlogp, dent)
    assert r.logp.shape == (5, 0)
    e = torch.empty(0, 700, device=DEV)
    r = K.log_prob_fwd(e, torch.empty(0, 3, dtype=torch.int64, device=DEV), k=4)
    assert r.logp.shape == (0, 3) and r.top_items.shape == (0, 4) and r.entropy.shape == (0,)


@pytest.mark.parametrize("c", [40, 3000, 20001])
@pytest.mark.parametrize("dtype", TYPES)
def test_log_prob_borders(K, c, dtype):
    """Rows masked whole, masked but one, of the type's lowest value alone, constant, with it as a mask, with NaN and
    infinities, +0 against -0, and items beyond the catalogue or negative."""
    low = torch.finfo(dtype).min
    s = torch.zeros(12, c, dtype=dtype, device=DEV)
    s[0] = -float("inf")
    s[1] = -float("inf")
    s[1, c // 2] = 3
    s[2] = low
    s[3] = 2.5
    s[4] = torch.linspace(-4, 4, c, device=DEV).to(dtype)
    s[4, ::3] = low
    s[5] = torch.linspace(4, -4, c, device=DEV).to(dtype)
    s[5, c - 1] = float("nan")
    s[6] = torch.linspace(-1, 1, c, device=DEV).to(dtype)
    s[6, 3] = float("inf")
    s[7, ::2] = -0.0
    s[8] = -float("inf")
    s[8, [1, c - 1]] = torch.tensor([low, low], dtype=dtype, device=DEV)
    s[9] = torch.finfo(dtype).max
    s[10] = (torch.arange(c, device=DEV) % 3).to(dtype)
    s[11] = -torch.finfo(dtype).max
    s[11, 5] = torch.finfo(dtype).max
    items = torch.stack([torch.tensor([0, c // 2, 5, -1]) for _ in range(12)]).to(DEV)
    items[3, 1] = c          # beyond
    items[4, 1] = 2 ** 40
    items[10, 3] = -2 ** 40  # padding too
    r = K.log_prob_fwd(s, items, k=16)
    ref = logp_ref(s, items, 16, 1.0)
    assert torch.equal(r.top_items, ref["top_items"])
    for name in ("logp", "top_logp", "entropy"):
        want = ref[name].float()  # row 11's difference of twice the largest number is -inf in 32 bits
        close(getattr(r, name), want, 1e-5 * (1 + torch.nan_to_num(want, neginf=0.0).abs()), name)
    dlogp, dent = torch.ones(12, 4, device=DEV), torch.ones(12, device=DEV)
    ds = K.log_prob_bwd(s, items, r.stats, dlogp, dent).float()
    assert not ds[0].any()
    nan_rows = [3, 4, 5, 6]
    assert torch.isnan(ds[nan_rows]).all()
    ok = [i for i in range(12) if i not in nan_rows]
    assert torch.isfinite(ds[ok]).all()
    for i in (2, 9, 7):  # uniform: p = 1 / c, no slope of the entropy
        want = torch.full((c,), -3.0 / c, dtype=F64, device=DEV)
        for j in (0, c // 2, 5):
            want[j] += 1
        close(ds[i], want, half_step(dtype) * want.abs() + 1e-5, f"row {i}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("k", [1, 20, 64, 65, 128])
def test_log_prob_ties_and_sorted_rows(K, k, dtype):
    """Scores from few values (ties across lanes, waves and shares), rising and falling rows, the best at the ends."""
    c = 40003
    g = gen(k)
    s = torch.randint(-3, 3, (5, c), device=DEV, generator=g).to(dtype)
    s[1] = torch.arange(c, device=DEV).float().mul(1e-3).to(dtype)
    s[2] = torch.arange(c, 0, -1, device=DEV).float().mul(1e-3).to(dtype)
    s[3] = 0
    s[4] = -float("inf")
    s[4, -k // 2:] = 1
    items = torch.zeros(5, 1, dtype=torch.int64, device=DEV)
    r = K.log_prob_fwd(s, items, k=k)
    assert torch.equal(r.top_items, logp_ref(s, items, k, 1.0)["top_items"])
    small = s[:, :9000].contiguous()
    r = K.log_prob_fwd(small, items, k=k)
    assert torch.equal(r.top_items, logp_ref(small, items, k, 1.0)["top_items"])


@pytest.mark.parametrize("k", [20, 40, 128])
def test_log_prob_ties_over_many_shares(K, k):
    """More equal scores than the pool that joins the shares holds."""
    s = torch.zeros(4, 300007, device=DEV)
    s[1] = torch.randint(0, 2, (300007,), device=DEV, generator=gen(k)).float()
    s[2, ::2] = -float("inf")
    s[3, 150000:] = torch.arange(150007, device=DEV).float().div(64).floor()
    items = torch.zeros(4, 1, dtype=torch.int64, device=DEV)
    r = K.log_prob_fwd(s, items, k=k)
    assert torch.equal(r.top_items, logp_ref(s, items, k, 1.0)["top_items"])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("c", [1, 2, 63, 65, 255, 257, 1023, 1025, 2047, 2049, 2056, 9000, 16385, 24577, 24600])
def test_log_prob_best_items_of_few_columns(K, c, dtype):
    """Columns about as many as the groups that the floor comes from, in a row's only step and in its last share."""
    for n, k in ((3, 1), (3, 48), (3, 49), (3, 128), (600, 20), (600, 100)):
        k = min(k, c)
        s = torch.randn(n, c, device=DEV).to(dtype)
        r = K.log_prob_fwd(s, torch.zeros(n, 1, dtype=torch.int64, device=DEV), k=k)
        value, index = torch.sort(s.float(), dim=1, descending=True, stable=True)
        assert torch.equal(r.top_items, index[:, :k]), (n, k)


def test_log_prob_against_differences(K):
    """The gradient against central differences of the kernels' own forward, taken in 64 bits of its definition."""
    s, items, dlogp, dent = logp_inputs(3, 50, 3, torch.float32, 9, masked=0.0, spread=1.0)
    r = K.log_prob_fwd(s, items, scale=0.7)
    ds = K.log_prob_bwd(s, items, r.stats, dlogp, dent, scale=0.7)
    h = 1e-4

    def total(x):
        z = x * 0.7
        lp = z - torch.logsumexp(z, 1, keepdim=True)
        given = torch.where(items < 0, 0.0, lp.gather(1, items.clamp(min=0)))
        return (given * dlogp.to(F64)).sum(1) - dent.to(F64) * (lp.exp() * lp).sum(1)

    for j in range(0, 50, 7):
        up, down = s.to(F64).clone(), s.to(F64).clone()
        up[:, j] += h
        down[:, j] -= h
        close(ds[:, j], (total(up) - total(down)) / (2 * h), 1e-5, f"column {j}")


def test_layer_norm_against_differences(K):
    x, w, b, dy = norm_inputs(4, 30, torch.float32, torch.float32, 6)
    _, mean, rstd = K.layer_norm_fwd(x, w, b, stats=True)
    dx, dw, db = K.layer_norm_bwd(dy, x, mean, rstd, w)
    h = 1e-4

    def total(xx, ww, bb):
        return (norm_ref(xx, ww, bb, 1e-5)[0] * dy.to(F64)).sum(1)

    x64, w64, b64 = x.to(F64), w.to(F64), b.to(F64)
    for j in range(0, 30, 7):
        e = torch.zeros(30, dtype=F64, device=DEV)
        e[j] = h
        close(dx[:, j], (total(x64 + e, w64, b64) - total(x64 - e, w64, b64)) / (2 * h), 2e-5, "dx")
        close(dw[j], ((total(x64, w64 + e, b64) - total(x64, w64 - e, b64)) / (2 * h)).sum(), 2e-5, "dw")
        close(db[j], ((total(x64, w64, b64 + e) - total(x64, w64, b64 - e)) / (2 * h)).sum(), 2e-5, "db")


# ---------------------------------------------------------------------------------------------------- the calls around them
def test_refusals(K):
    x = torch.zeros(4, 40, device=DEV)
    w = torch.ones(40, device=DEV)
    y, mean, rstd = K.layer_norm_fwd(x, stats=True)
    items = torch.zeros(4, 2, dtype=torch.int64, device=DEV)
    a = K.act8_pack(x)
    r = K.log_prob_fwd(x, items)
    g = torch.zeros(4, 2, device=DEV)
    wide = torch.zeros(5, 48, device=DEV)
    bad = [
        lambda: K.layer_norm_fwd(x.double()),
        lambda: K.layer_norm_fwd(x.cpu()),
        lambda: K.layer_norm_fwd(x[0]),
        lambda: K.layer_norm_fwd(x.t()),
        lambda: K.layer_norm_fwd(x[:, :0]),
        lambda: K.layer_norm_fwd(x, eps=-1.0),
        lambda: K.layer_norm_fwd(x, eps=float("nan")),
        lambda: K.layer_norm_fwd(x, w[:39]),
        lambda: K.layer_norm_fwd(x, w.half()),
        lambda: K.layer_norm_fwd(x.half(), w, w.half()),
        lambda: K.layer_norm_fwd(x, w.cpu()),
        lambda: K.layer_norm_fwd(x, torch.ones(80, device=DEV)[::2]),
        lambda: K.layer_norm_bwd(x[:3], x, mean, rstd),
        lambda: K.layer_norm_bwd(x.half(), x, mean, rstd),
        lambda: K.layer_norm_bwd(x, x, mean[:3], rstd),
        lambda: K.layer_norm_bwd(x, x, mean, rstd.double()),
        lambda: K.act8_pack(x.int()),
        lambda: K.act8_pack(x.t()),
        lambda: K.act8_unpack(x),
        lambda: K.act8_unpack(a, torch.float64),
        lambda: K.act8_unpack(a, out=torch.zeros(4, 39, device=DEV)),
        lambda: K.act8_unpack(a, out=torch.zeros(1, 40, device=DEV).expand(4, 40)),
        lambda: K.act8_unpack(a, torch.float16, out=torch.zeros(4, 40, device=DEV)),
        lambda: K.act8_unpack(K.Act8(a.q[:, :32], a.e, (4, 40), torch.float32)),
        lambda: K.act8_wgrad(x[:3], a),
        lambda: K.act8_wgrad(x[:, :0], a),
        lambda: K.act8_wgrad(x.double(), a),
        lambda: K.log_prob_fwd(x, items[:3]),
        lambda: K.log_prob_fwd(x, items.int()),
        lambda: K.log_prob_fwd(x, items.t().contiguous().t()),
        lambda: K.log_prob_fwd(x, items, k=41),
        lambda: K.log_prob_fwd(x, items, k=-1),
        lambda: K.log_prob_fwd(torch.zeros(4, 200, device=DEV), items, k=129),
        lambda: K.log_prob_fwd(x, items, scale=0.0),
        lambda: K.log_prob_fwd(x, items, scale=-1.0),
        lambda: K.log_prob_fwd(x, items, scale=float("nan")),
        lambda: K.log_prob_fwd(x, torch.zeros(4, 1025, dtype=torch.int64, device=DEV)),
        lambda: K.log_prob_fwd(x[:, :0], items),
        lambda: K.log_prob_bwd(x, items, r.stats[:3], g),
        lambda: K.log_prob_bwd(x, items, r.stats, g[:, :1]),
        lambda: K.log_prob_bwd(x, items, r.stats, g, torch.zeros(3, device=DEV)),
        lambda: K.log_prob_bwd(x, items, r.stats, g, out=torch.zeros(4, 41, device=DEV)),
        lambda: K.log_prob_bwd(x, items, r.stats, g, out=x.half()),
        lambda: K.log_prob_bwd(wide[:4, :40], items, r.stats, g, out=wide[:4, 1:41]),
        lambda: K.log_prob_bwd(wide[:4, :40], items, r.stats, g, out=wide[1:5, :40]),
        lambda: K.log_prob_bwd(x, items, r.stats, g, out=torch.zeros(1, 40, device=DEV).expand(4, 40)),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            print("not refused:", i)


def all_calls(K, s):
    y, mean, rstd = K.layer_norm_fwd(s["x"], s["w"], s["b"], stats=True)
    dx, dw, db = K.layer_norm_bwd(s["dy"], s["x"], mean, rstd, s["w"])
    a = K.act8_pack(y)
    dW, dB = K.act8_wgrad(s["dy"], a)
    r = K.log_prob_fwd(s["scores"], s["items"], k=20)
    ds = K.log_prob_bwd(s["scores"], s["items"], r.stats, s["dlogp"], s["dent"])
    return [y, mean, rstd, dx, dw, db, a.q, a.e, K.act8_unpack(a), dW, dB, r.logp, r.stats, r.top_items, r.top_logp, ds]


def call_state(seed):
    x, w, b, dy = norm_inputs(2000, 260, torch.float32, torch.float32, seed)
    scores, items, dlogp, dent = logp_inputs(4, 60000, 3, torch.float32, seed + 1)
    return {"x": x, "w": w, "b": b, "dy": dy, "scores": scores, "items": items, "dlogp": dlogp, "dent": dent}


def test_streams_and_captured_graphs(K):
    """The same bits on another stream, and from two graphs replayed in turn with eager work between them."""
    states = [call_state(1), call_state(2)]
    want = [all_calls(K, s) for s in states]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = all_calls(K, states[0])
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want[0]))
    graphs, outs = [], []
    for s in states:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(all_calls(K, s))
        graphs.append(g)
    for turn in range(4):
        for o in outs:
            for t in o:
                t.zero_()
        graphs[0].replay()
        eager = all_calls(K, states[turn % 2])
        graphs[1].replay()
        torch.cuda.synchronize()
        for o, w in ((outs[0], want[0]), (outs[1], want[1]), (eager, want[turn % 2])):
            assert all(torch.equal(a, b) for a, b in zip(o, w)), turn
    # new inputs in the captured buffers
    for key, v in states[1].items():
        states[0][key].copy_(v)
    graphs[0].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs[0], want[1]))


def test_outputs_stay_in_their_bounds(K):
    """Nothing behind an output's rows is written (outputs as views into a larger buffer)."""
    x, w, b, dy = norm_inputs(5, 45, torch.bfloat16, torch.float32, 1)
    s, items, dlogp, dent = logp_inputs(5, 999, 2, torch.bfloat16, 3)
    r = K.log_prob_fwd(s, items)
    big = torch.full((5, 1010), 7.0, dtype=torch.bfloat16, device=DEV)
    K.log_prob_bwd(s, items, r.stats, dlogp, dent, out=big[:, 3:1002])
    assert (big[:, :3] == 7).all() and (big[:, 1002:] == 7).all()
    assert torch.equal(big[:, 3:1002], K.log_prob_bwd(s, items, r.stats, dlogp, dent))


def test_more_rows_than_a_launch(K):
    """Rows of several launches: the last ones and the borders' are those of a call on them alone."""
    n = (1 << 23) + 5
    s = torch.randn(n, 3, device=DEV).to(torch.bfloat16)
    items = torch.arange(n, device=DEV).remainder(4).sub(1)[:, None].contiguous()
    g, h = torch.randn(n, 1, device=DEV), torch.randn(n, device=DEV)
    r = K.log_prob_fwd(s, items, k=2)
    ds = K.log_prob_bwd(s, items, r.stats, g, h)
    for part in (slice(0, 9), slice((1 << 23) - 4, n)):
        w = K.log_prob_fwd(s[part], items[part], k=2)
        for name in ("logp", "entropy", "lse", "top_items", "top_logp"):
            assert torch.equal(getattr(r, name)[part], getattr(w, name)), name
        assert torch.equal(ds[part], K.log_prob_bwd(s[part], items[part], w.stats, g[part], h[part]))
    n = (1 << 28) + 5
    x = torch.randn(n, 1, device=DEV)
    a = K.act8_pack(x)
    back = K.act8_unpack(a)
    for part in (slice(0, 9), slice((1 << 28) - 4, n)):
        w = K.act8_pack(x[part])
        assert torch.equal(a.q[part], w.q) and torch.equal(a.e[part], w.e)
        assert torch.equal(back[part], K.act8_unpack(w))


def test_a_row_of_2_to_30_scores(K):
    """Offsets of more than 32 bits, and shares of more columns.  The scores are 0 but for one of log 2^30 = 20.79 (in
    bf16 20.75): p = e^20.75 / (e^20.75 + c - 1)."""
    c = (1 << 30) + 77
    s = torch.zeros(1, c, dtype=torch.bfloat16, device=DEV)
    best = c - 2
    s[0, best] = 20.75
    items = torch.tensor([[best, 5, -1]], device=DEV)
    top = math.exp(20.75)
    lse = math.log(top + c - 1)
    want = torch.tensor([[20.75 - lse, -lse, 0.0]], dtype=torch.float64)
    r = K.log_prob_fwd(s, items, k=3)
    # S: a chain of at most 4200 additions (a share's 2^20 columns over 256 threads, and the joins), each off by 2^-24 of
    # the sum; a term's power off by 2^-22; lse about 21.5, off by some roundings of its size
    tol = 4200 * 2.0 ** -24 + 24 * 2.0 ** -22
    assert (r.logp.double().cpu() - want).abs().max() <= tol
    assert abs(r.lse.item() - lse) <= tol
    assert r.top_items.tolist() == [[best, 0, 1]]
    g = torch.tensor([[1.0, 0.0, 3.0]], device=DEV)
    ds = K.log_prob_bwd(s, items, r.stats, g)
    p, q = top / (top + c - 1), 1 / (top + c - 1)
    # exp of a logp off by tol, and bf16's rounding
    assert abs(ds[0, best].item() - (1 - p)) <= p * 2 * tol + (1 - p) * 2.0 ** -8
    others = ds[0, [0, 4, 5, 6, 16383, 16384, 1 << 29, c - 3, c - 1]].double().cpu()
    assert (others + q).abs().max() <= q * (2 * tol + 2.0 ** -8)
