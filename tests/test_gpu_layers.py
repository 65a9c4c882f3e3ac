"""The layer operators on the GPU (ops.group_norm, ops.gemm_bias_act, their backward passes and layers.*) against plain formulas in
64 bits on the same (already rounded) inputs.

Tolerances.  u = 2^-24 is half a step of fp32 arithmetic, h(t) = finfo(t).eps / 2 half a step of an output type, and an output below
the type's normal range is off by at most half its smallest step.
 * a sum of k products in fp32, in any order: k u sum |terms| (first order), doubled;
 * variance: at most 64 fp32 operations one after another on any path (rows of a thread, threads of a block; the rest is fp64): 64 u
   relative, half of that for rstd; the mean: 64 u of the largest |x|;
 * activations: slope at most 1.13; fp32 evaluation 16 u (1 + z^2 / 2) relative (the argument of exp is rounded), 16-bit types
   4e-5 relative on top (their erfc fit 1.8e-5, exp2 and reciprocal a few u)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
ACTS = ["none", "relu", "silu", "gelu"]


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available()
    return torch.device("cuda:0")


@pytest.fixture(scope="module")
def ops():
    from optimaltextures_amd import ops
    return ops


def half(t):
    return torch.finfo(t).eps / 2


def least(t):
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def act64(z, act):
    return {"none": lambda: z, "relu": lambda: z.clamp_min(0), "silu": lambda: z * torch.sigmoid(z),
            "gelu": lambda: z * torch.special.ndtr(z)}[act]()


def slope64(z, act):
    if act == "none":
        return torch.ones_like(z)
    if act == "relu":
        return (z > 0).double()
    if act == "silu":
        s = torch.sigmoid(z)
        return s * (1 + z * (1 - s))
    return torch.special.ndtr(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)


def act_rel(z, t, act):
    """relative error of an activation's evaluation (of |z| rather than of its value: the slope formulas add terms up to |z|)"""
    if act in ("none", "relu"):
        return torch.zeros_like(z)
    return 16 * U * (1 + z * z / 2).clamp_max(100) + (0 if t == torch.float32 else 4e-5)


def check(got, want, tol, what=""):
    got = got.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = (got - want).abs() - tol
    assert not torch.isnan(got).any() or torch.isnan(want).any(), what
    assert bool((off <= 0).all()), f"{what}: worst excess {float(off.max()):.3g}, at {int(off.argmax())}, tol {float(tol.reshape(-1)[off.argmax()]):.3g}"


# ------------------------------------------------------------------------------------------------ group norm
def norm64(x, groups, w, b, eps, act, mean=None, rstd=None):
    s, c = x.shape[0], x.shape[-1]
    v = x.double().reshape(s, -1, groups, c // groups)
    if mean is None:
        mean = v.mean(dim=(1, 3))
        rstd = ((v - mean.view(s, 1, groups, 1)) ** 2).mean(dim=(1, 3)).add(eps).rsqrt()
    xh = (v - mean.double().view(s, 1, groups, 1)) * rstd.double().view(s, 1, groups, 1)
    wv = torch.ones(1, 1, groups, c // groups, dtype=torch.float64, device=x.device) if w is None else w.double().view(-1, 1, groups, c // groups)
    bv = torch.zeros_like(wv) if b is None else b.double().view(-1, 1, groups, c // groups)
    return xh, wv, bv, xh * wv + bv, mean, rstd


def norm_input(dev, t, shape, groups, per_image=False, affine=True, seed=0, level=0.7, atype=None):
    g = torch.Generator(device=dev).manual_seed(seed)
    c = shape[-1]
    x = (torch.randn(shape, generator=g, device=dev) * (torch.rand(c, generator=g, device=dev) + 0.3)
         + level * torch.randn(c, generator=g, device=dev)).to(t)
    if not affine:
        return x, None, None
    ps = (shape[0], c) if per_image else (c,)
    w = (1 + 0.3 * torch.randn(ps, generator=g, device=dev)).to(atype or t)
    b = (0.3 * torch.randn(ps, generator=g, device=dev)).to(atype or t)
    return x, w, b


def norm_z_tol(x, groups, xh, w, b, rstd):
    s, c = x.shape[0], x.shape[-1]
    big = x.double().abs().reshape(s, -1, groups, c // groups).amax(dim=(1, 3), keepdim=True)
    r = rstd.view(s, 1, groups, 1).double()
    return w.abs() * r * 64 * U * big + (32 + 8) * U * (xh * w).abs() + 4 * U * b.abs() + 4 * U * (xh * w + b).abs()


def check_norm(ops, x, groups, w, b, eps, act, y, mean, rstd):
    t = x.dtype
    xh, wv, bv, z, mean64, rstd64 = norm64(x, groups, w, b, eps, act)
    s, c = x.shape[0], x.shape[-1]
    big = x.double().abs().reshape(s, -1, groups, c // groups).amax(dim=(1, 3))
    if mean is not None:
        check(mean, mean64, 64 * U * big + 1e-38, "mean")
        # the mean of a thread's rows is off by 8 u of the largest value, which a squared deviation sees squared
        check(rstd, rstd64, rstd64 * (33 * U + 0.5 * (8 * U * big * rstd64) ** 2), "rstd")
    zt = norm_z_tol(x, groups, xh, wv, bv, rstd64)
    y64 = act64(z, act)
    tol = 1.13 * zt + act_rel(z, t, act) * z.abs() + (half(t) + 4 * U) * y64.abs() + least(t)
    check(y, y64.reshape(x.shape), tol.reshape(x.shape), "y")


NORM_SHAPES = [
    ((1, 1, 1, 8), 8), ((1, 1, 1, 8), 1), ((2, 1, 1, 6), 3), ((1, 2, 1, 1), 1), ((1, 16, 16, 64), 8), ((2, 5, 7, 59), 1),
    ((2, 5, 7, 60), 5), ((3, 37, 53, 96), 6), ((1, 9, 1, 2056), 8), ((2, 3, 4, 2304), 32), ((1, 130, 129, 32), 32), ((5, 8, 8, 512), 32),
    ((1, 3, 3, 264), 33), ((70, 1, 3, 16), 2), ((2, 64, 64, 256), 32), ((1, 200, 210, 3), 1), ((3, 6, 6, 40), 10), ((1, 24, 24, 1), 1),
]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("shape,groups", NORM_SHAPES)
def test_group_norm(dev, ops, t, shape, groups):
    for k, act in enumerate(ACTS):
        per = k == 2
        x, w, b = norm_input(dev, t, shape, groups, per_image=per, affine=k != 1, seed=k, atype=torch.float32 if k == 3 else None)
        y, mean, rstd = ops.group_norm(x, groups, w, b, eps=1e-5, act=act, want_stats=True)
        check_norm(ops, x, groups, w, b, 1e-5, act, y, mean, rstd)
        assert torch.equal(ops.group_norm(x, groups, w, b, eps=1e-5, act=act), y)      # the same bits without the statistics


def norm_grad64(dy, x, groups, w, b, act, mean, rstd, per_image):
    s, c = x.shape[0], x.shape[-1]
    xh, wv, bv, z, _, _ = norm64(x, groups, w, b, 0, act, mean, rstd)
    d = dy.double().reshape(z.shape)
    dz = d * slope64(z, act)
    r = rstd.double().view(s, 1, groups, 1)
    e = dz * wv
    count = z.shape[1] * z.shape[3]
    s1, s2 = e.sum(dim=(1, 3), keepdim=True) / count, (e * xh).sum(dim=(1, 3), keepdim=True) / count
    dx = r * (e - s1 - xh * s2)
    over = 1 if per_image else (0, 1)
    return dict(dx=dx.reshape(x.shape), dw=(dz * xh).sum(dim=over).reshape(-1, c) if per_image else (dz * xh).sum(dim=over).reshape(c),
                db=dz.sum(dim=over).reshape(-1, c) if per_image else dz.sum(dim=over).reshape(c), xh=xh, z=z, dz=dz, d=d, e=e, r=r, wv=wv,
                over=over, count=count)


def check_norm_grad(ops, dy, x, groups, w, b, act, mean, rstd, dx, dw, db):
    t, c = x.dtype, x.shape[-1]
    per = w is not None and w.dim() == 2
    o = norm_grad64(dy, x, groups, w, b, act, mean, rstd, per)
    # dz: its argument z is off by a few u of its terms, act' has slope at most 1.13 too, its evaluation act_rel
    zerr = 8 * U * ((o["xh"] * o["wv"]).abs() + o["z"].abs() + 1)
    dzt = o["d"].abs() * (1.13 * zerr + act_rel(o["z"], t, act) * (1 + o["z"].abs()) + 4 * U)
    if act == "relu":   # a z that is zero to within its error may fall on either side
        dzt = dzt + o["d"].abs() * (o["z"].abs() <= zerr).double()
    xt = 6 * U * o["xh"].abs()
    rows = o["z"].shape[1]
    if w is not None:
        terms, tt = (o["dz"] * o["xh"]).abs(), dzt * o["xh"].abs() + o["dz"].abs() * xt
        k = 2 * (64 + rows / 64) * U      # rows of a thread one after another, the block's tree, the rest in fp64
        tol = (tt + k * terms).sum(dim=o["over"]).reshape(dw.shape)
        check(dw, o["dw"], tol + (half(dw.dtype) + 2 * U) * o["dw"].abs() + least(dw.dtype), "dw")
        tol = (dzt + k * o["dz"].abs()).sum(dim=o["over"]).reshape(db.shape)
        check(db, o["db"], tol + (half(db.dtype) + 2 * U) * o["db"].abs() + least(db.dtype), "db")
    et = dzt * o["wv"].abs() + 2 * U * o["e"].abs()
    k = 2 * (64 + rows / 64) * U
    s1t = (et + k * o["e"].abs()).sum(dim=(1, 3), keepdim=True) / o["count"]
    s2t = ((et + k * o["e"].abs()) * o["xh"].abs() + o["e"].abs() * xt).sum(dim=(1, 3), keepdim=True) / o["count"]
    s1, s2 = o["e"].abs().sum(dim=(1, 3), keepdim=True) / o["count"], (o["e"] * o["xh"]).abs().sum(dim=(1, 3), keepdim=True) / o["count"]
    tol = o["r"] * (et + s1t + o["xh"].abs() * s2t + 8 * U * (o["e"].abs() + s1 + o["xh"].abs() * s2))
    check(dx, o["dx"], tol.reshape(x.shape) + half(t) * o["dx"].abs() + least(t), "dx")


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("shape,groups", NORM_SHAPES)
def test_group_norm_backward(dev, ops, t, shape, groups):
    for k, act in enumerate(ACTS):
        x, w, b = norm_input(dev, t, shape, groups, per_image=k == 2, affine=k != 1, seed=10 + k, atype=torch.float32 if k == 3 else None)
        dy = torch.randn(shape, generator=torch.Generator(device=dev).manual_seed(k), device=dev).to(t)
        _, mean, rstd = ops.group_norm(x, groups, w, b, act=act, want_stats=True)
        dx, dw, db = ops.group_norm_backward(dy, x, mean, rstd, groups, w, b, act=act)
        assert (dw is None) == (w is None) and (db is None) == (b is None)
        check_norm_grad(ops, dy, x, groups, w, b, act, mean, rstd, dx, dw, db)


def test_group_norm_gradient_against_differences(dev, ops):
    """d(sum c y) by central differences of the 64-bit forward formula, in random directions, against <dx, direction>"""
    g = torch.Generator(device=dev).manual_seed(3)
    shape, groups = (2, 6, 5, 24), 4
    for act in ACTS:
        x, w, b = norm_input(dev, torch.float32, shape, groups, seed=4)
        cvec = torch.randn(shape, generator=g, device=dev, dtype=torch.float64)
        _, mean, rstd = ops.group_norm(x, groups, w, b, act=act, want_stats=True)
        grads = ops.group_norm_backward(cvec.float(), x, mean, rstd, groups, w, b, act=act)
        cvec = cvec.float().double()

        def loss(*a):
            _, _, _, z, _, _ = norm64(a[0], groups, a[1], a[2], 1e-5, act)
            return float((act64(z, act).reshape(shape) * cvec).sum())
        at = [x.double(), w.double(), b.double()]
        for which in range(3):
            v = torch.randn(at[which].shape, generator=g, device=dev, dtype=torch.float64)
            step = 1e-6
            lo, hi = [a.clone() for a in at], [a.clone() for a in at]
            lo[which] -= step * v
            hi[which] += step * v
            want = (loss(*hi) - loss(*lo)) / (2 * step)
            got = float((grads[which].double() * v).sum())
            # differences: 1e-12-ish curvature, 1e-16 / 1e-6 rounding of a loss of ~ 40; relu: a kink within the step is off by
            # less than step * |terms|; gradients: fp32 sums
            assert abs(got - want) <= 2e-5 * float(grads[which].double().norm() * v.norm()) + 1e-6, (act, which, got, want)


@pytest.mark.parametrize("t", TYPES)
def test_group_norm_strides_alignment_and_in_place(dev, ops, t):
    big, w, b = norm_input(dev, t, (3, 10, 11, 48), 4, seed=1)
    for view in (big[..., 8:40], big[..., 3:35], big[:, 2:7, :, :32], big[1:, :, :, 16:], big[:, :, :, 5:6]):
        c = view.shape[-1]
        groups = 4 if c % 4 == 0 else 1
        wv, bv = w[:c].contiguous(), b[:c].contiguous()
        want, mean, rstd = ops.group_norm(view.contiguous(), groups, wv, bv, act="silu", want_stats=True)
        got = ops.group_norm(view, groups, wv, bv, act="silu")
        # the same sums, if in another order where the access width differs: within the rounding of y
        assert torch.allclose(got.float(), want.float(), rtol=4 * half(t), atol=4 * half(t) if t != torch.float32 else 1e-5)
        check_norm(ops, view, groups, wv, bv, 1e-5, "silu", got, None, None)
        # into a slice of a larger map, whose other channels stay as they are
        frame = torch.full(view.shape[:-1] + (c + 9,), 7.0, dtype=t, device=dev)
        ops.group_norm(view, groups, wv, bv, act="silu", out=frame[..., 4:4 + c])
        check_norm(ops, view, groups, wv, bv, 1e-5, "silu", frame[..., 4:4 + c], None, None)
        assert bool((frame[..., :4] == 7).all()) and bool((frame[..., 4 + c:] == 7).all())
        same = view.contiguous()
        ops.group_norm(same, groups, wv, bv, act="silu", out=same)
        assert torch.equal(same, want)
        dy = torch.randn(view.shape, device=dev).to(t)
        dx, dw, db = ops.group_norm_backward(dy, view, mean, rstd, groups, wv, bv, act="silu")
        check_norm_grad(ops, dy, view, groups, wv, bv, "silu", mean, rstd, dx, dw, db)
        dyv = torch.randn(view.shape[:-1] + (c + 3,), device=dev).to(t)[..., 1:1 + c]
        dx, dw, db = ops.group_norm_backward(dyv, view, mean, rstd, groups, wv, bv, act="silu")
        check_norm_grad(ops, dyv, view, groups, wv, bv, "silu", mean, rstd, dx, dw, db)


def test_group_norm_levels_far_from_zero(dev, ops):
    """a mean a thousand spreads away: the variance keeps its digits (no uncentred squares)"""
    for shape, groups in (((2, 40, 40, 32), 8), ((1, 128, 128, 64), 1), ((1, 8, 8, 8), 8)):
        x = (torch.randn(shape, generator=torch.Generator(device=dev).manual_seed(0), device=dev) + 1000.0)
        y, mean, rstd = ops.group_norm(x, groups, eps=0.0, want_stats=True)
        check_norm(ops, x, groups, None, None, 0.0, "none", y, mean, rstd)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("shape,groups", [((8, 16, 16, 512), 32), ((4, 64, 64, 256), 8)])
def test_group_norm_means_near_zero(dev, ops, t, shape, groups):
    """means much smaller than the spread keep their digits.  In norm: a group of N values of spread 1 has a mean of about N^-1/2; its
    fp32 sum of terms of either sign passes through values up to about N^1/2, each of some 24 additions on a path rounding by
    u / 2 of that at most: 12 u N^1/2 / N, that is 12 u = 7e-7 of the mean, and u for its own rounding"""
    x = torch.randn(shape, generator=torch.Generator(device=dev).manual_seed(11), device=dev).to(t)
    _, mean, rstd = ops.group_norm(x, groups, want_stats=True)
    _, _, _, _, mean64, rstd64 = norm64(x, groups, None, None, 1e-5, "none")
    assert float((mean.double() - mean64).norm() / mean64.norm()) <= 1e-6
    assert float((rstd.double() - rstd64).norm() / rstd64.norm()) <= 1e-6


def test_group_norm_constant_and_nonfinite_groups(dev, ops):
    x = torch.randn(2, 6, 6, 32, device=dev)
    x[0, ..., 8:16] = 3.25                      # variance 0: rstd = eps^-1/2, y = bias
    x[1, 2, 3, 17] = float("inf")
    x[1, 0, 0, 31] = float("nan")
    x[0, 1, 1, 20] = 1e30                       # squares beyond fp32
    w, b = torch.randn(32, device=dev), torch.randn(32, device=dev)
    for act in ACTS:
        y, mean, rstd = ops.group_norm(x, 4, w, b, act=act, want_stats=True)
        assert torch.equal(y[0, ..., 8:16], act_t(b[8:16], act).expand(6, 6, 8)) or torch.allclose(y[0, ..., 8:16], act_t(b[8:16], act).expand(6, 6, 8), rtol=1e-6, atol=1e-7)
        assert abs(float(rstd[0, 1]) * math.sqrt(1e-5) - 1) < 1e-6 and float(mean[0, 1]) == 3.25
        assert bool(torch.isnan(y[1, ..., 16:]).all()) and not bool(torch.isnan(y[1, ..., :16]).any())
        assert not bool(torch.isnan(y[0, ..., :16]).any()) and not bool(torch.isnan(y[0, ..., 24:]).any())


def act_t(z, act):
    return act64(z.double(), act).float()


def test_group_norm_empty(dev, ops):
    for shape in ((0, 4, 4, 8), (2, 0, 4, 8)):
        x = torch.empty(shape, device=dev)
        w = torch.ones(8, device=dev)
        assert ops.group_norm(x, 2, w, w).shape == x.shape
        stats = torch.zeros(shape[0], 2, device=dev)
        dx, dw, db = ops.group_norm_backward(x, x, stats, stats, 2, w, w)
        assert dx.shape == x.shape and not bool(dw.any()) and not bool(db.any())
        w2 = torch.ones(shape[0], 8, device=dev, dtype=torch.float32)
        dx, dw, db = ops.group_norm_backward(x, x, stats, stats, 2, w2, w2)
        assert dw.shape == w2.shape and not bool(dw.any()) and not bool(db.any())


# ------------------------------------------------------------------------------------------------ product
def ints(dev, t, shape, seed, most=3):
    g = torch.Generator(device=dev).manual_seed(seed)
    return torch.randint(-most, most + 1, shape, generator=g, device=dev).to(t)


PRODUCT_SIZES = [  # rows n, inner K, outer M
    (1, 1, 1), (1, 8, 1), (1, 512, 2048), (2, 64, 64), (3, 7, 5), (5, 200, 331), (7, 4096, 64), (8, 72, 264), (15, 33, 17), (16, 2048, 512),
    (17, 256, 48), (31, 96, 4096), (33, 1000, 40), (63, 64, 65), (64, 64, 64), (65, 128, 63), (127, 40, 130), (128, 256, 256), (129, 136, 257),
    (200, 3, 3), (255, 32, 512), (257, 520, 136), (300, 256, 1), (512, 1, 70), (1000, 130, 514), (1237, 201, 331), (2049, 64, 128),
    (4097, 24, 8), (5000, 512, 130), (70000, 16, 24), (16384, 256, 512), (640, 2048, 1024), (256, 4104, 1032),
]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("n,k,m", PRODUCT_SIZES)
def test_gemm_bias_act_exact_on_integers(dev, ops, t, n, k, m):
    """small whole numbers: every product and sum is exact in fp32, the outputs are the exact sums rounded once"""
    x, w, b, r = ints(dev, t, (n, k), 1), ints(dev, t, (m, k), 2), ints(dev, t, (m,), 3), ints(dev, t, (n, m), 4)
    s = x.double() @ w.double().t().contiguous()
    assert torch.equal(ops.gemm_bias_act(x, w), s.to(t))
    y, pre = ops.gemm_bias_act(x, w, b, act="relu", residual=r, want_pre=True)
    assert torch.equal(pre, (s + b.double()).to(t))
    assert torch.equal(y, ((s + b.double()).clamp_min(0) + r.double()).to(t))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("n,k,m", PRODUCT_SIZES)
def test_gemm_bias_act_backward_exact_on_integers(dev, ops, t, n, k, m):
    x, w, d, pre = ints(dev, t, (n, k), 1), ints(dev, t, (m, k), 2), ints(dev, t, (n, m), 3), ints(dev, t, (n, m), 4)
    if n * 9 >= 1 << 24:
        pytest.skip("sums beyond 2^24 are not exact")
    for act in ("none", "relu"):
        e = d.double() * (1 if act == "none" else (pre > 0).double())
        dx, dw, db = ops.gemm_bias_act_backward(d, x, w, pre, act=act)
        assert torch.equal(dx, (e @ w.double()).to(t))
        assert torch.equal(dw, (e.t().contiguous() @ x.double()).to(t))
        assert torch.equal(db, e.sum(dim=0).to(t))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("n,k,m", [(65560, 72, 264), (65560, 264, 72), (65560, 1000, 1016), (65560, 128, 1000), (16400, 392, 72)])
def test_products_of_many_tiles_exact_on_integers(dev, ops, t, n, k, m):
    """sizes that take the larger tiles, with ragged ends, in every direction; long sums in pieces (dW)"""
    x, w, d = ints(dev, t, (n, k), 1), ints(dev, t, (m, k), 2), ints(dev, t, (n, m), 3)
    b, r = ints(dev, t, (m,), 4), ints(dev, t, (n, m), 5)
    assert torch.equal(ops.gemm_bias_act(x, w, b, act="relu", residual=r),
                       ((x.double() @ w.double().t().contiguous() + b.double()).clamp_min(0) + r.double()).to(t))
    dx, dw, db = ops.gemm_bias_act_backward(d, x, w, r, act="relu")
    e = d.double() * (r > 0)
    assert torch.equal(dx, (e @ w.double()).to(t))
    assert torch.equal(dw, (e.t().contiguous() @ x.double()).to(t))
    assert torch.equal(db, e.sum(dim=0).to(t))


def test_large_products_in_a_replayed_graph(dev, ops):
    """the tiles that need more than 64 KiB of LDS, and split sums, captured and replayed between eager calls"""
    x, w, d = (torch.randn(s, device=dev).bfloat16() for s in ((65536, 512), (1024, 512), (65536, 1024)))

    def step():
        return (ops.gemm_bias_act(x, w, act="gelu"), *ops.gemm_bias_act_backward(d, x, w))
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(3):
        x.copy_(torch.randn(x.shape, generator=torch.Generator(device=dev).manual_seed(seed), device=dev))
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b)


def product_input(dev, t, n, k, m, seed=0, btype=None):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(n, k, generator=g, device=dev).to(t), (torch.randn(m, k, generator=g, device=dev) / math.sqrt(k)).to(t),
            (0.3 * torch.randn(m, generator=g, device=dev)).to(btype or t), torch.randn(n, m, generator=g, device=dev).to(t))


def check_product(x, w, b, r, act, y, pre=None):
    t, k = x.dtype, x.shape[-1]
    xd, wd = x.double().reshape(-1, k), w.double()
    z, terms = xd @ wd.t().contiguous(), xd.abs() @ wd.abs().t().contiguous()
    if b is not None:
        z, terms = z + b.double(), terms + b.double().abs()
    zt = 2 * (k + 2) * U * terms
    if pre is not None:
        check(pre.reshape(z.shape), z, zt + half(t) * z.abs() + least(t), "pre")
    v = act64(z, act)
    tol = 1.13 * zt + act_rel(z, t, act) * z.abs()
    if r is not None:
        v = v + r.double().reshape(v.shape)
    check(y.reshape(v.shape), v, tol + (half(t) + 2 * U) * v.abs() + 2 * U * tol + least(t), "y")


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("n,k,m", [(1, 512, 2048), (3, 37, 50), (16, 2048, 512), (100, 64, 200), (1237, 201, 331), (4096, 256, 256), (700, 1024, 640)])
def test_gemm_bias_act(dev, ops, t, n, k, m):
    for i, act in enumerate(ACTS):
        x, w, b, r = product_input(dev, t, n, k, m, seed=i, btype=torch.float32 if i == 2 else None)
        y, pre = ops.gemm_bias_act(x, w, b, act=act, residual=r, want_pre=True)
        check_product(x, w, b, r, act, y, pre)
        assert torch.equal(ops.gemm_bias_act(x, w, b, act=act, residual=r), y)
        check_product(x, w, None, None, act, ops.gemm_bias_act(x, w, act=act))
        again = r.clone()
        assert ops.gemm_bias_act(x, w, b, act=act, residual=again, out=again) is again and torch.equal(again, y)


def check_product_grad(dy, x, w, pre, act, dx, dw, db):
    t, k = x.dtype, x.shape[-1]
    xd, wd, d = x.double().reshape(-1, k), w.double(), dy.double().reshape(-1, w.shape[0])
    if act != "none":
        z = pre.double().reshape(d.shape)
        e = d * slope64(z, act)
        et = d.abs() * (act_rel(z, t, act) * (1 + z.abs()) + 4 * U)
    else:
        e, et = d, torch.zeros_like(d)
    ed = et + (half(t) * e.abs() + least(t) if act != "none" else 0)      # as an operand: rounded to the type
    n, m = e.shape
    v = e @ wd
    check(dx.reshape(v.shape), v, ed @ wd.abs() + 2 * (m + 2) * U * (e.abs() @ wd.abs()) + half(t) * v.abs() + least(t), "dx")
    v = e.t().contiguous() @ xd
    check(dw, v, ed.t().contiguous() @ xd.abs() + 2 * (n + 2) * U * (e.abs().t().contiguous() @ xd.abs()) + half(t) * v.abs() + least(t), "dw")
    if db is not None:
        v = e.sum(dim=0)
        tol = et.sum(dim=0) + 2 * (1024 + 2) * U * e.abs().sum(dim=0)
        check(db, v, tol + half(db.dtype) * v.abs() + least(db.dtype), "db")


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("n,k,m", [(1, 512, 2048), (3, 37, 50), (16, 2048, 512), (100, 64, 200), (1237, 201, 331), (8192, 256, 256), (700, 1024, 640)])
def test_gemm_bias_act_backward(dev, ops, t, n, k, m):
    for i, act in enumerate(ACTS):
        x, w, b, dy = product_input(dev, t, n, k, m, seed=i)
        _, pre = ops.gemm_bias_act(x, w, b, act=act, want_pre=True)
        dx, dw, db = ops.gemm_bias_act_backward(dy, x, w, pre, act=act, bias_dtype=torch.float32 if i == 1 else None)
        check_product_grad(dy, x, w, pre, act, dx, dw, db)
        only = ops.gemm_bias_act_backward(dy, x, w, pre, act=act, want_x=False, want_bias=False)
        assert only[0] is None and only[2] is None and torch.equal(only[1], dw)
        only = ops.gemm_bias_act_backward(dy, x, w, pre, act=act, want_w=False, want_bias=False)
        assert only[1] is None and torch.equal(only[0], dx)
        only = ops.gemm_bias_act_backward(dy, x, w, pre, act=act, want_x=False, want_w=False)
        assert torch.equal(only[2], db if i != 1 else db.to(t))


def test_gemm_bias_act_gradient_against_differences(dev, ops):
    g = torch.Generator(device=dev).manual_seed(5)
    for act in ACTS:
        x, w, b, c = product_input(dev, torch.float32, 40, 24, 56, seed=6)
        _, pre = ops.gemm_bias_act(x, w, b, act=act, want_pre=True)
        grads = ops.gemm_bias_act_backward(c, x, w, pre, act=act)
        at = [x.double(), w.double(), b.double()]

        def loss(a):
            return float((act64(a[0] @ a[1].t().contiguous() + a[2], act) * c.double()).sum())
        for which in range(3):
            v = torch.randn(at[which].shape, generator=g, device=dev, dtype=torch.float64)
            lo, hi = [a.clone() for a in at], [a.clone() for a in at]
            lo[which] -= 1e-6 * v
            hi[which] += 1e-6 * v
            want, got = (loss(hi) - loss(lo)) / 2e-6, float((grads[which].double() * v).sum())
            assert abs(got - want) <= 2e-5 * float(grads[which].double().norm() * v.norm()) + 1e-6, (act, which, got, want)


@pytest.mark.parametrize("t", TYPES)
def test_gemm_bias_act_strides_and_alignment(dev, ops, t):
    xb, wb, rb = ints(dev, t, (300, 96), 1), ints(dev, t, (200, 104), 2), ints(dev, t, (300, 208), 3)
    b = ints(dev, t, (200,), 4)
    for (x0, kk), (w0, mm), r0 in (((0, 64), (0, 128), 0), ((8, 64), (16, 128), 8), ((3, 64), (5, 100), 1), ((0, 70), (1, 64), 2), ((16, 80), (8, 200), 8)):
        x, w, r = xb[:, x0:x0 + kk], wb[:mm, w0:w0 + kk], rb[:, r0:r0 + mm]
        assert not x.is_contiguous() and not w.is_contiguous() and not r.is_contiguous()
        s = x.double() @ w.double().t().contiguous() + b[:mm].double()
        want = (s.clamp_min(0) + r.double()).to(t)
        assert torch.equal(ops.gemm_bias_act(x, w, b[:mm], act="relu", residual=r), want)
        frame = torch.full((300, mm + 13), 5.0, dtype=t, device=dev)
        ops.gemm_bias_act(x, w, b[:mm], act="relu", residual=r, out=frame[:, 6:6 + mm])
        assert torch.equal(frame[:, 6:6 + mm], want) and bool((frame[:, :6] == 5).all()) and bool((frame[:, 6 + mm:] == 5).all())
        dx, dw, db = ops.gemm_bias_act_backward(r, x, w)
        assert torch.equal(dx, (r.double() @ w.double()).to(t)) and torch.equal(dw, (r.double().t().contiguous() @ x.double()).to(t))
        assert torch.equal(db, r.double().sum(dim=0).to(t))


@pytest.mark.parametrize("t", TYPES)
def test_gemm_bias_act_nonfinite_rows_stay_in_their_rows(dev, ops, t):
    """an infinite or NaN row reaches its own outputs only; tails beyond K and n bring nothing in"""
    for n, k, m in ((37, 50, 70), (130, 64, 128), (300, 264, 136), (4, 520, 64)):
        x, w, b, _ = product_input(dev, t, n, k, m)
        y0 = ops.gemm_bias_act(x, w, b, act="silu")
        x[1, 3], x[2, k - 1] = float("inf"), float("nan")
        y = ops.gemm_bias_act(x, w, b, act="silu")
        assert torch.equal(y[0], y0[0]) and torch.equal(y[3:], y0[3:])
        assert bool(torch.isnan(y[2]).all())
        want = x[1].double() @ w.double().t().contiguous()
        assert bool((torch.isinf(y[1]) | torch.isnan(y[1])).logical_or(want < 0).all())


def test_gemm_bias_act_empty(dev, ops):
    for t in TYPES:
        w, b = torch.ones(6, 4, dtype=t, device=dev), torch.ones(6, dtype=t, device=dev)
        x = torch.empty(0, 4, dtype=t, device=dev)
        assert ops.gemm_bias_act(x, w, b, act="gelu").shape == (0, 6)
        dx, dw, db = ops.gemm_bias_act_backward(torch.empty(0, 6, dtype=t, device=dev), x, w, torch.empty(0, 6, dtype=t, device=dev), act="gelu")
        assert dx.shape == (0, 4) and not bool(dw.any()) and not bool(db.any())
        x, w = torch.empty(5, 0, dtype=t, device=dev), torch.empty(6, 0, dtype=t, device=dev)     # K = 0: act(bias) + residual
        r = torch.ones(5, 6, dtype=t, device=dev)
        assert torch.equal(ops.gemm_bias_act(x, w, b, act="relu", residual=r), r + r)
        dx, dw, db = ops.gemm_bias_act_backward(r, x, w)
        assert dx.shape == (5, 0) and dw.shape == (6, 0) and torch.equal(db, 5 * b)
        x, w = torch.ones(5, 4, dtype=t, device=dev), torch.empty(0, 4, dtype=t, device=dev)
        assert ops.gemm_bias_act(x, w).shape == (5, 0)
        dx, dw, db = ops.gemm_bias_act_backward(torch.empty(5, 0, dtype=t, device=dev), x, w)
        assert not bool(dx.any()) and dw.shape == (0, 4) and db.shape == (0,)


def test_gemm_bias_act_offsets_beyond_32_bits(dev, ops):
    """rows whose byte offsets pass 2^32: the last rows of a long map"""
    n, k = (1 << 31) // 1000, 2048 + 8
    x = torch.zeros(n, k, dtype=torch.bfloat16, device=dev)[:, :64]
    tail = ints(dev, torch.bfloat16, (300, 64), 1)
    x[-300:] = tail
    x[:300] = tail
    w = ints(dev, torch.bfloat16, (128, 64), 2)
    want = (tail.double() @ w.double().t().contiguous()).to(torch.bfloat16)
    y = ops.gemm_bias_act(x, w)
    assert torch.equal(y[-300:], want) and torch.equal(y[:300], want) and not bool(y[300:-300].any())
    d = torch.zeros(n, 128, dtype=torch.bfloat16, device=dev)
    d[-300:] = want.clamp(-3, 3)
    dx, dw, db = ops.gemm_bias_act_backward(d, x, w)
    e = d[-300:].double()
    assert torch.equal(dw, (e.t().contiguous() @ tail.double()).to(torch.bfloat16)) and torch.equal(dx[-300:], (e @ w.double()).to(torch.bfloat16))


def test_group_norm_offsets_beyond_32_bits(dev, ops):
    n, ld = 1 << 20, 2056
    base = torch.zeros(2, n, ld, dtype=torch.bfloat16, device=dev)
    x = base[..., 8:72]
    v = torch.randn(2, n, 64, generator=torch.Generator(device=dev).manual_seed(0), device=dev).bfloat16()
    x.copy_(v)
    y, mean, rstd = ops.group_norm(x, 4, act="relu", want_stats=True)
    want, mean0, rstd0 = ops.group_norm(v, 4, act="relu", want_stats=True)
    assert torch.equal(mean, mean0) and torch.equal(rstd, rstd0) and torch.equal(y, want)
    ops.group_norm(x, 4, act="relu", out=x)
    assert torch.equal(x, want) and not bool(base[..., :8].any()) and not bool(base[:, -1, 72:].any())


# ------------------------------------------------------------------------------------------------ streams, graphs, gradients together
def block(layers, x, p, groups):
    """a residual block: norm, silu, widen, gelu, narrow onto the residual stream"""
    h = layers.group_norm_act(x, groups, p["gw"], p["gb"], act="silu")
    h = layers.linear_act(h, p["w1"], p["b1"], act="gelu")
    return layers.linear_act(h, p["w2"], p["b2"], residual=x)


def block64(x, p, groups):
    s, c = x.shape[0], x.shape[-1]
    _, _, _, z, _, _ = norm64_grad(x, groups, p["gw"], p["gb"])
    h = act64(z, "silu").reshape(x.shape)
    h = act64(h @ p["w1"].t() + p["b1"], "gelu")
    return h @ p["w2"].t() + p["b2"] + x


def norm64_grad(x, groups, w, b):
    s, c = x.shape[0], x.shape[-1]
    v = x.reshape(s, -1, groups, c // groups)
    m = v.mean(dim=(1, 3), keepdim=True)
    r = ((v - m) ** 2).mean(dim=(1, 3), keepdim=True).add(1e-5).rsqrt()
    return None, None, None, (v - m) * r * w.view(1, 1, groups, -1) + b.view(1, 1, groups, -1), m, r


def block_params(dev, t, c, wide, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    return dict(gw=(1 + 0.2 * r(c)).to(t), gb=(0.2 * r(c)).to(t), w1=(r(wide, c) / math.sqrt(c)).to(t), b1=(0.1 * r(wide)).to(t),
                w2=(r(c, wide) / math.sqrt(wide)).to(t), b2=(0.1 * r(c)).to(t))


@pytest.mark.parametrize("t,rel", [(torch.float32, 2e-5), (torch.bfloat16, 2e-2), (torch.float16, 2.5e-3)])
def test_block_of_the_operators_and_its_gradients(dev, t, rel):
    """norm -> product -> product with residual, twice, as a user chains them; gradients by torch's autograd in 64 bits.  In norms: about
    ten tensors in a row are rounded to the type (each half a step at worst, a third of that in the mean square), fp32 sums besides"""
    from optimaltextures_amd import layers
    c, wide, groups = 96, 200, 6
    x = torch.randn(2, 9, 11, c, generator=torch.Generator(device=dev).manual_seed(1), device=dev).to(t)
    ps = [block_params(dev, t, c, wide, seed=s) for s in (0, 1)]
    leaves = [x.clone().requires_grad_()] + [v.clone().requires_grad_() for p in ps for v in p.values()]
    names = list(ps[0])
    take = lambda ls: [dict(zip(names, ls[1 + 6 * i:7 + 6 * i])) for i in range(2)]  # noqa: E731
    y = leaves[0]
    for p in take(leaves):
        y = block(layers, y, p, groups)
    dy = torch.randn(y.shape, generator=torch.Generator(device=dev).manual_seed(2), device=dev).to(t)
    grads = torch.autograd.grad(y, leaves, dy)
    l64 = [v.detach().double().cpu().requires_grad_() for v in leaves]
    y64 = l64[0]
    for p in take(l64):
        y64 = block64(y64, p, groups)
    g64 = torch.autograd.grad(y64, l64, dy.double().cpu())
    for got, want in zip([y, *grads], [y64, *g64]):
        assert got.dtype == t and float((got.detach().double().cpu() - want.detach()).norm() / want.detach().norm()) <= rel
    with torch.no_grad():
        z = x
        for p in ps:
            z = block(layers, z, p, groups)
        assert torch.equal(z, y)        # serving: the same bits


def test_layers_refuse_a_gradient_of_a_gradient(dev):
    from optimaltextures_amd import layers
    x = torch.randn(2, 4, 4, 8, device=dev, requires_grad=True)
    w = torch.randn(8, 8, device=dev, requires_grad=True)
    for y in (layers.group_norm_act(x, 2, act="silu"), layers.linear_act(x, w, act="silu")):
        g, = torch.autograd.grad(y.sum(), x, create_graph=True)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(g.sum(), x)


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
def test_layers_in_a_replayed_graph(dev, ops, t):
    """forward and backward of a block captured together and replayed on new inputs, with eager work between the replays"""
    from optimaltextures_amd import layers
    c, wide, groups = 64, 192, 8
    p = {k: v.requires_grad_() for k, v in block_params(dev, t, c, wide).items()}
    x = torch.randn(3, 16, 16, c, device=dev).to(t).requires_grad_()
    dy = torch.randn(3, 16, 16, c, device=dev).to(t)

    def step():
        y = block(layers, x, p, groups)
        return (y.detach(), *torch.autograd.grad(y, [x, *p.values()], dy))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(4):
        g = torch.Generator(device=dev).manual_seed(seed)
        with torch.no_grad():
            x.copy_(torch.randn(x.shape, generator=g, device=dev))
            dy.copy_(torch.randn(x.shape, generator=g, device=dev))
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b)
        ops.gemm_bias_act(torch.randn(999, 77, device=dev), torch.randn(55, 77, device=dev))


def test_capture_over_a_living_eager_graph_is_refused(dev):
    from optimaltextures_amd import layers
    x = torch.randn(2, 8, 8, 16, device=dev, requires_grad=True)
    w = torch.randn(16, 16, device=dev, requires_grad=True)
    eager = layers.linear_act(x, w)           # its graph holds the leaves' accumulation nodes
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="eager graph of the same leaf"):
        with torch.cuda.graph(graph):
            layers.linear_act(x, w, act="relu")
    del eager
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layers.linear_act(x, w, act="relu")
    graph.replay()
    with torch.no_grad():
        assert torch.equal(y, layers.linear_act(x, w, act="relu"))


def test_layers_on_another_stream_and_two_at_once(dev, ops):
    """calls on two side streams at the same time, each with its own scratch: the bits of the calls alone"""
    shapes = [(3, 37, 53, 96), (2, 64, 64, 128)]
    xs = [torch.randn(s, device=dev).bfloat16() for s in shapes]
    ws = [torch.randn(200, s[-1], device=dev).bfloat16() for s in shapes]
    want = [(ops.group_norm(x, 4, act="silu"), ops.gemm_bias_act(x, w, act="gelu"),
             *ops.gemm_bias_act_backward(ops.gemm_bias_act(x, w), x, w)) for x, w in zip(xs, ws)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = [None, None]
    for _ in range(5):
        for i, (st, x, w) in enumerate(zip(streams, xs, ws)):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                got[i] = (ops.group_norm(x, 4, act="silu"), ops.gemm_bias_act(x, w, act="gelu"),
                          *ops.gemm_bias_act_backward(ops.gemm_bias_act(x, w), x, w))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            for u, v in zip(a, b):
                assert torch.equal(u, v)


def test_layers_refuse_bad_calls(dev, ops):
    from optimaltextures_amd import layers
    x, w, b = torch.randn(2, 4, 4, 8, device=dev), torch.randn(16, 8, device=dev), torch.randn(16, device=dev)
    bad = [lambda: ops.group_norm(x, 3), lambda: ops.group_norm(x, 0), lambda: ops.group_norm(x.double(), 2), lambda: ops.group_norm(x[0, 0, 0], 2),
           lambda: ops.group_norm(x, 2, b), lambda: ops.group_norm(x, 2, b[:8].half()), lambda: ops.group_norm(x, 2, b[:8].cpu()),
           lambda: ops.group_norm(x, 2, b[:8], torch.zeros(2, 8, device=dev)), lambda: ops.group_norm(x, 2, eps=-1.0),
           lambda: ops.group_norm(x, 2, out=x[:1]), lambda: ops.group_norm(x, 2, out=x.permute(0, 2, 1, 3)), lambda: ops.group_norm(x, 2, out=x.half()),
           lambda: ops.group_norm_backward(x[:1], x, b, b, 2), lambda: ops.group_norm_backward(x, x, b, b, 2),
           lambda: ops.gemm_bias_act(x, w.half()), lambda: ops.gemm_bias_act(x, w.t()), lambda: ops.gemm_bias_act(x, w, b[:8]),
           lambda: ops.gemm_bias_act(x, w, residual=x), lambda: ops.gemm_bias_act(x, w, out=x), lambda: ops.gemm_bias_act(x, w.cpu()),
           lambda: ops.gemm_bias_act(x, w, b.half()), lambda: ops.gemm_bias_act(x, w[0]), lambda: ops.gemm_bias_act(x, w[:8], out=x),
           lambda: ops.gemm_bias_act_backward(x, x, w), lambda: ops.gemm_bias_act_backward(x, x, w[:8], act="silu"),
           lambda: ops.gemm_bias_act_backward(x, x, w[:8], bias_dtype=torch.float16)]
    for f in bad:
        with pytest.raises(RuntimeError):
            f()
    for f in (lambda: ops.group_norm(x, 2, act="tanh"), lambda: layers.linear_act(x, w, act="swish")):
        with pytest.raises(ValueError):
            f()
