"""Layer norm (forward with residual sum, backward with the reductions of the weight's and bias's gradients) against the
formulas in 64 bits.  Bounds: one rounding of the result to its type (half a step, finfo.eps / 2 relative) plus 32-bit
arithmetic, counted as OPS roundings of 2^-24 on the sum of the magnitudes that enter (a thread adds at most 32 elements one
after the other, then at most 8 levels of a tree; the rest are single operations)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from pacednegatives_amd import kernels as K  # noqa: E402

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
U32, OPS = 2.0 ** -24, 64
SHAPES = [(1, 1), (1, 768), (3, 8), (17, 64), (5, 100), (33, 128), (300, 136), (4, 511), (70, 513), (129, 768), (40, 1023), (21, 1024),
          (9, 2048), (6, 2056), (5, 4100), (3, 8191), (2, 8192), (5000, 72)]


def half_step(t):
    return torch.finfo(t).eps / 2


def make(M, d, dtype, seed, shift=0.5):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(M, d, generator=g) * torch.exp(0.5 * torch.randn(d, generator=g)) + shift * torch.randn(M, 1, generator=g)
    res, dy, dres = (torch.randn(M, d, generator=g) for _ in range(3))
    w, b = 1 + 0.3 * torch.randn(d, generator=g), 0.2 * torch.randn(d, generator=g)
    return [t.to("cuda").to(dtype) for t in (x, res, dy, dres, w, b)]


def stats64(s, eps):
    s = s.to(F64)
    mean = s.mean(1, keepdim=True)
    rstd = ((s - mean).square().mean(1, keepdim=True) + eps).rsqrt()
    return s, mean, rstd, (s - mean) * rstd


def check_fwd(y, s, w, b, eps):
    s, mean, rstd, xh = stats64(s, eps)
    want = xh * w.to(F64) + b.to(F64)
    # an error e of the mean moves xh by e rstd; the variance's relative error (its sum of squares, and the mean's error
    # against the deviation) moves it by half of that
    entering = (xh.abs() + s.abs().mean(1, keepdim=True) * rstd * (1 + xh.abs())) * w.to(F64).abs() + b.to(F64).abs()
    assert ((y.to(F64) - want).abs() <= half_step(y.dtype) * want.abs() * (1 + 2 ** -7) + OPS * U32 * entering).all()


def check_bwd(dx, dw, db, dy, s, w, dres, eps, dw0=0.0, db0=0.0):
    s, mean, rstd, xh = stats64(s, eps)
    dy, w = dy.to(F64), w.to(F64)
    g = dy * w
    want = rstd * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    slack = s.abs().mean(1, keepdim=True) * rstd * (1 + xh.abs())          # of xh, as in check_fwd
    entering = rstd * (g.abs() + g.abs().mean(1, keepdim=True) + (xh.abs() + slack) * (g * xh).abs().mean(1, keepdim=True)
                       + xh.abs() * (g.abs() * slack).mean(1, keepdim=True)) * (1 + slack)
    if dres is not None:
        want = want + dres.to(F64)
        entering = entering + dres.to(F64).abs()
    assert ((dx.to(F64) - want).abs() <= half_step(dx.dtype) * want.abs() * (1 + 2 ** -7) + OPS * U32 * entering).all()
    # columns: a thread adds at most ceil(M / 512) rows of its team, then 6 levels of a wave and a workgroup, then 64 of 512
    # partial rows and 8 levels
    ops = OPS + s.shape[0] // 512 + 1 + 6 + 64 + 8
    if dw is not None:
        assert ((dw.to(F64) - dw0 - (dy * xh).sum(0)).abs() <= ops * U32 * ((dy.abs() * (xh.abs() + slack)).sum(0) + abs(dw0))).all()
    if db is not None:
        assert ((db.to(F64) - db0 - dy.sum(0)).abs() <= ops * U32 * (dy.abs().sum(0) + abs(db0))).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("M,d", SHAPES)
@pytest.mark.parametrize("residual", [False, True])
def test_forward_and_backward(M, d, dtype, residual):
    x, res, dy, dres, w, b = make(M, d, dtype, M * 10007 + d)
    y, mean, rstd = torch.empty_like(x), torch.empty(M, device="cuda"), torch.empty(M, device="cuda")
    xsum = torch.empty_like(x) if residual else None
    K.layernorm_fwd(x, w, b, y, mean, rstd, eps=1e-5, res=res if residual else None, xsum=xsum)
    s = x
    if residual:
        s = (x.float() + res.float()).to(dtype)          # one 32-bit addition, one rounding: exactly this
        assert torch.equal(xsum, s)
    check_fwd(y, s, w, b, 1e-5)
    dx, dw, db = torch.empty_like(x), torch.full((d,), 0.5, device="cuda"), torch.full((d,), -0.25, device="cuda")
    K.layernorm_bwd(dy, s, w, mean, rstd, dx, dres=dres if residual else None, dw=dw, db=db)
    check_bwd(dx, dw, db, dy, s, w, dres if residual else None, 1e-5, 0.5, -0.25)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("d,pad", [(64, 8), (64, 3), (768, 8), (768, 1), (999, 5)])
def test_rows_with_strides_and_offsets(d, pad, dtype):
    M = 37
    buf = [torch.full((M + 1, 2 * d + 2 * pad), 7.0, device="cuda", dtype=dtype) for _ in range(5)]
    x, res, dy, dres, w, b = make(M, d, dtype, d + pad)
    views = [t[:M, pad:pad + d] for t in buf]
    for v, t in zip(views, (x, res, dy, dres)):
        v.copy_(t)
    xv, rv, dyv, drv, yv = views
    mean, rstd, xs = torch.empty(M, device="cuda"), torch.empty(M, device="cuda"), torch.empty_like(x)
    K.layernorm_fwd(xv, w, b, yv, mean, rstd, res=rv, xsum=xs)
    check_fwd(yv, xs, w, b, 1e-5)
    for t in buf:                                          # nothing outside the rows is touched
        assert (t[:, :pad] == 7).all() and (t[:, pad + d:] == 7).all() and (t[M] == 7).all()
    K.layernorm_bwd(dyv, xs, w, mean, rstd, yv, dres=drv)
    check_bwd(yv, None, None, dy, xs, w, dres, 1e-5)
    for t in buf:
        assert (t[:, :pad] == 7).all() and (t[:, pad + d:] == 7).all() and (t[M] == 7).all()


def test_outputs_in_the_place_of_inputs():
    x, res, dy, dres, w, b = make(50, 768, BF16, 3)
    y, xs, mean, rstd = torch.empty_like(x), torch.empty_like(x), torch.empty(50, device="cuda"), torch.empty(50, device="cuda")
    K.layernorm_fwd(x, w, b, y, mean, rstd, res=res, xsum=xs)
    dx = torch.empty_like(x)
    K.layernorm_bwd(dy, xs, w, mean, rstd, dx, dres=dres)
    x2, r2 = x.clone(), res.clone()
    K.layernorm_fwd(x2, w, b, x2, res=r2, xsum=r2)
    assert torch.equal(x2, y) and torch.equal(r2, xs)
    d2 = dres.clone()
    K.layernorm_bwd(dy, xs, w, mean, rstd, d2, dres=d2)
    assert torch.equal(d2, dx)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("d", [3, 9, 127, 250, 767, 1001, 1535, 2049, 4093, 8190])
def test_rows_that_end_inside_a_piece_in_the_place_of_inputs(d, dtype):
    """(every team's width, rows whose last piece is read from the one before it)"""
    M = 70
    x, res, dy, dres, w, b = make(M, d, dtype, d)
    y, mean, rstd = torch.empty_like(x), torch.empty(M, device="cuda"), torch.empty(M, device="cuda")
    s = (x.float() + res.float()).to(dtype)
    r2 = res.clone()
    K.layernorm_fwd(x, w, b, y, mean, rstd, res=r2, xsum=r2)
    assert torch.equal(r2, s)
    check_fwd(y, s, w, b, 1e-5)
    x2, r3 = x.clone(), res.clone()
    K.layernorm_fwd(x2, w, b, x2, res=r3, xsum=r3)
    assert torch.equal(x2, y) and torch.equal(r3, s)
    dx, dw, db = torch.empty_like(x), torch.full((d,), 0.5, device="cuda"), torch.full((d,), -0.25, device="cuda")
    K.layernorm_bwd(dy, s, w, mean, rstd, dx, dres=dres, dw=dw, db=db)
    check_bwd(dx, dw, db, dy, s, w, dres, 1e-5, 0.5, -0.25)
    d2 = dy.clone()
    K.layernorm_bwd(d2, s, w, mean, rstd, d2, dres=dres)
    assert torch.equal(d2, dx)


def test_gradients_are_the_same_bits_every_time_and_each_is_optional():
    x, _, dy, _, w, b = make(4000, 768, BF16, 8)
    y, mean, rstd, dx = torch.empty_like(x), torch.empty(4000, device="cuda"), torch.empty(4000, device="cuda"), torch.empty_like(x)
    K.layernorm_fwd(x, w, b, y, mean, rstd)
    first = None
    for _ in range(3):
        dw, db = torch.zeros(768, device="cuda"), torch.zeros(768, device="cuda")
        K.layernorm_bwd(dy, x, w, mean, rstd, dx, dw=dw, db=db)
        first = first or (dw, db)
        assert torch.equal(dw, first[0]) and torch.equal(db, first[1])
    only = torch.zeros(768, device="cuda")
    K.layernorm_bwd(dy, x, w, mean, rstd, dx, dw=only)
    assert torch.equal(only, first[0])
    only.zero_()
    K.layernorm_bwd(dy, x, w, mean, rstd, dx, db=only)
    assert torch.equal(only, first[1])


def test_directional_derivative():
    """(L(x + h v) - L(x - h v)) / 2h against <dx, v> in fp32, L = sum dy y.  With h = 2^-5 and xh of order one the
    truncation is of order h^2 = 1e-3 of the terms; rounding 2^-24 |dy||y| sqrt(n) / h is below 1e-4 of them."""
    x, _, dy, _, w, b = make(8, 256, F32, 11, shift=0.0)
    v = torch.randn(8, 256, device="cuda", generator=torch.Generator("cuda").manual_seed(5))
    h, L = 2.0 ** -5, []
    mean, rstd, y = torch.empty(8, device="cuda"), torch.empty(8, device="cuda"), torch.empty_like(x)
    for k in (h, -h):
        K.layernorm_fwd(x + k * v, w, b, y, mean, rstd)
        L.append((y.double() * dy.double()).sum(1))
    K.layernorm_fwd(x, w, b, y, mean, rstd)
    dx = torch.empty_like(x)
    K.layernorm_bwd(dy, x, w, mean, rstd, dx)
    got, want = (L[0] - L[1]) / (2 * h), (dx.double() * v.double()).sum(1)
    scale = (dx.double().square().sum(1) * v.double().square().sum(1)).sqrt()
    assert ((got - want).abs() <= 4e-3 * scale).all()


def test_constant_rows_infinities_and_nan_stay_in_their_rows():
    x, _, dy, _, w, b = make(6, 256, BF16, 4)
    x[1] = 3.0                            # variance zero: rstd = 1 / sqrt(eps), y = b
    x[2, 7], x[3, 9] = float("inf"), float("nan")
    y, mean, rstd = torch.empty_like(x), torch.empty(6, device="cuda"), torch.empty(6, device="cuda")
    K.layernorm_fwd(x, w, b, y, mean, rstd)
    assert torch.equal(y[1], b) and not y[2].isfinite().any() and y[3].isnan().all()
    keep = [0, 1, 4, 5]
    check_fwd(y[keep], x[keep], w, b, 1e-5)
    dx = torch.empty_like(x)
    K.layernorm_bwd(dy, x, w, mean, rstd, dx)
    assert dx[keep].isfinite().all() and dx[3].isnan().all()


def test_no_rows():
    w, b = torch.ones(64, device="cuda"), torch.zeros(64, device="cuda")
    e, s = torch.empty(0, 64, device="cuda"), torch.empty(0, device="cuda")
    dw = torch.full((64,), 2.0, device="cuda")
    K.layernorm_fwd(e, w, b, torch.empty_like(e), s, s)
    K.layernorm_bwd(e, e, w, s, s, torch.empty_like(e), dw=dw)
    assert (dw == 2).all()


def test_captured_and_replayed_beside_eager_calls():
    x, res, dy, dres, w, b = make(500, 768, BF16, 12)
    bufs = [torch.empty_like(x) for _ in range(3)]
    mean, rstd, dw, db = torch.empty(500, device="cuda"), torch.empty(500, device="cuda"), torch.zeros(768, device="cuda"), torch.zeros(768, device="cuda")

    def step():
        dw.zero_(); db.zero_()
        K.layernorm_fwd(x, w, b, bufs[0], mean, rstd, res=res, xsum=bufs[1])
        K.layernorm_bwd(dy, bufs[1], w, mean, rstd, bufs[2], dres=dres, dw=dw, db=db)
    step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for k in range(3):
        x.copy_(make(500, 768, BF16, 20 + k)[0])
        step()
        want = [t.clone() for t in (*bufs, dw, db)]
        for t in bufs:
            t.fill_(9)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip((*bufs, dw, db), want))


def test_refusals():
    x = torch.zeros(4, 64, device="cuda", dtype=BF16)
    w, b, s = torch.ones(64, device="cuda", dtype=BF16), torch.zeros(64, device="cuda", dtype=BF16), torch.empty(4, device="cuda")
    y = torch.empty_like(x)
    for kw, words in ((dict(w=w.float()), "w must be"), (dict(b=b[:32]), "b must hold"), (dict(y=y.float()), "y must be"), (dict(y=y[:3]), "y must have shape"),
                      (dict(res=x), "go together"), (dict(mean=s.double()), "mean must be"), (dict(x=x.half()), "bf16 or fp32"), (dict(x=x.cpu()), "device tensor"),
                      (dict(x=x.t().contiguous().t()), "unit inner stride"), (dict(x=x[:1].expand(4, 64)), "rows overlap")):
        args = dict(x=x, w=w, b=b, y=y, mean=None, res=None) | kw
        with pytest.raises(ValueError, match=words):
            K.layernorm_fwd(args["x"], args["w"], args["b"], args["y"], args["mean"], res=args["res"])
    with pytest.raises(ValueError, match="dw must be"):
        K.layernorm_bwd(x, x, w, s, s, y, dw=w)
    with pytest.raises(ValueError, match="workspace must be"):
        K.layernorm_bwd(x, x, w, s, s, y, dw=torch.zeros(64, device="cuda"), workspace=torch.empty(1 << 20, device="cuda"))
    wide = torch.zeros(2, 8200, device="cuda")
    from pacednegatives_amd._lib import PacedHipError
    with pytest.raises(PacedHipError, match="8192"):
        K.layernorm_fwd(wide, wide[0].clone(), wide[0].clone(), torch.empty_like(wide))
