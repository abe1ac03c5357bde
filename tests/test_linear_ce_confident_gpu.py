"""Gradients of the linear-head loss on confident rows, entry by entry relative to the entry itself.

Every row has a label of its own: w is 4 times a unit vector for the first entries and zero for the others, h_r = a_r e_r with
label r, so z is 4 a_r at the label (exactly, also in the MFMA's sums) and 0 elsewhere, and
    loss = log(1 + (V - 1) exp(-4 a_r)),    the label's entry c_r = g_r expm1(-loss_r),
    dh[r][r] = 4 c_r,    dw[r][r] = c_r a_r  (no other row and no other entry reaches those elements).
Bound: 4 a_r <= 24 goes through a change of base (35 units, off by 2^-24 of it twice) into a power: 24 * 2^-23 relative; another
2^-20 for the power, the sums, log1p and expm1 in 32 bits; together below 2^-17.  Then half a bf16 step, 2^-8, for dh and for the
entry of P that dw is made of; up to 64 rows dw takes the entry's second part as well, which leaves 2^-8 2^-8.
An element of dw that several rows share is a sum in 32 bits: 2^-23 for each addend."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from pacednegatives_amd import kernels as K  # noqa: E402

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64


@pytest.mark.parametrize("R,V,d,tile", [(1, 1000, 64, 0), (48, 1000, 64, 0), (64, 40, 64, 0), (65, 1000, 128, 0), (130, 777, 192, 128), (300, 1000, 512, 0), (300, 1000, 512, 256),
                                        (1100, 13000, 1152, 0), (600, 66000, 640, 0), (20000, 7001, 64, 0)])
@pytest.mark.parametrize("f32", [False, True])
def test_small_losses_keep_their_gradients_digits(R, V, d, tile, f32):
    g = torch.Generator("cuda").manual_seed(R)
    a = (4 + torch.randint(0, 65, (R,), generator=g, device="cuda") / 32).to(BF16)         # 4 .. 6: losses of 1e-4 down to 1e-9
    a[0] = 6
    at = torch.arange(R, device="cuda")
    h, w = torch.zeros(R, d, device="cuda", dtype=BF16), torch.zeros(V, d, device="cuda", dtype=BF16)
    own = at % min(V, d)                                                                    # (64 x 40: rows beyond 40 share features and labels)
    h[at, own] = a
    w[torch.arange(min(V, d), device="cuda"), torch.arange(min(V, d), device="cuda")] = 4
    gl = 0.5 + torch.rand(R, generator=g, device="cuda")
    loss, lse = torch.empty(R, device="cuda"), torch.empty(R, device="cuda")
    dh, dw = torch.empty_like(h), torch.zeros(V, d, device="cuda", dtype=F32 if f32 else BF16)
    K.gemm_set_tile(tile)
    try:
        K.linear_ce_fwd(h, w, own, loss, lse)
        K.linear_ce_bwd(h, w, own, lse, gl, dh, dw, loss=loss)
    finally:
        K.gemm_set_tile(0)
    want = torch.log1p((V - 1) * torch.exp(-4 * a.to(F64)))
    assert want.min() < 1e-5             # (V - 1) exp(-24): 2.5e-6 for 66000 entries, under 1e-6 for the others
    assert ((loss.to(F64) - want).abs() <= 2.0 ** -17 * want).all()
    c = gl.to(F64) * torch.expm1(-want)
    assert ((dh[at, own].to(F64) - 4 * c).abs() <= (2.0 ** -8 + 2.0 ** -17) * (4 * c).abs()).all()
    shared = torch.zeros(V, dtype=F64, device="cuda").index_add_(0, own, c * a.to(F64))
    size = torch.zeros(V, dtype=F64, device="cuda").index_add_(0, own, (c * a.to(F64)).abs())
    k = torch.arange(min(V, d, R), device="cuda")
    tol = 2.0 ** -17 + (2.0 ** -16 if R <= 64 else 2.0 ** -8) + (0 if f32 else 2.0 ** -8 * (1 + 2.0 ** -7)) + 2.0 ** -23 * (R // min(V, d) + 64)
    assert ((dw[k, k].to(F64) - shared[k]).abs() <= tol * size[k]).all()


def test_both_ways_agree_where_losses_are_not_small_and_ignored_rows_stay_out():
    """Losses of order one: the two forms of the label's entry differ by 2^-21 (|lse| + |z|), and by the bf16 neighbour."""
    g = torch.Generator("cuda").manual_seed(2)
    h, w = (torch.randn(200, 128, generator=g, device="cuda") * 0.1).to(BF16), torch.randn(900, 128, generator=g, device="cuda").to(BF16)
    labels = torch.randint(0, 900, (200,), generator=g, device="cuda")
    labels[::9] = -100
    gl = torch.rand(200, generator=g, device="cuda")
    loss, lse = torch.empty(200, device="cuda"), torch.empty(200, device="cuda")
    K.linear_ce_fwd(h, w, labels, loss, lse)
    out = []
    for kw in ({}, {"loss": loss}):
        dh, dw = torch.empty_like(h), torch.zeros(900, 128, device="cuda")
        K.linear_ce_bwd(h, w, labels, lse, gl, dh, dw, **kw)
        assert (dh[::9] == 0).all()
        out.append((dh.double(), dw.double()))
    # one entry of a row in 900 moves, by a bf16 step at most
    assert (out[0][0] - out[1][0]).norm() <= 2.0 ** -7 * out[0][0].norm() and (out[0][1] - out[1][1]).norm() <= 2.0 ** -7 * out[0][1].norm()


def test_refusals():
    h, w, labels, v = torch.zeros(8, 64, device="cuda", dtype=BF16), torch.zeros(9, 64, device="cuda", dtype=BF16), torch.zeros(8, dtype=torch.int64, device="cuda"), torch.zeros(8, device="cuda")
    for loss, words in ((v[:4], "loss must hold"), (v.double(), "loss must be"), (v.cpu(), "device tensor")):
        with pytest.raises(ValueError, match=words):
            K.linear_ce_bwd(h, w, labels, v, v, torch.empty_like(h), loss=loss)


@pytest.mark.parametrize("R,V,d", [(65, 5000, 256), (300, 1000, 512), (1088, 6401, 256)])
@pytest.mark.parametrize("f32", [False, True])
def test_beyond_64_rows_dw_loses_half_a_step_of_p_and_no_more(R, V, d, f32):
    """Rows with labels of their own, so that one addend is most of an element, and rows that share one.  P's entries are off by
    a uniform error of at most 2^-8 of themselves, 2^-8 / sqrt(3) in the root mean square: by that much of the root of the sum of
    P^2 h^2 as a whole (a tenth more for chance), by 2^-8 of the sum of |P h| element by element (and 2^-11 for logits
    off by D < 2^-13 twice and sums of up to 1088 addends in 32 bits); dw's own rounding adds the same of dw."""
    from test_linear_ce_gpu import make, oracle
    h, w, labels, gl = make(R, V, d, R, ignored=0.0, size=1.0)
    labels[:R // 2] = torch.arange(R // 2, device="cuda")
    labels[R // 2:R // 2 + 9] = V - 1
    o = oracle(h, w, labels, gl, 1.0)
    assert o["D"].max() < 2.0 ** -13
    loss, lse = torch.empty(R, device="cuda"), torch.empty(R, device="cuda")
    dw = torch.zeros(V, d, device="cuda", dtype=F32 if f32 else BF16)
    K.linear_ce_fwd(h, w, labels, loss, lse)
    K.linear_ce_bwd(h, w, labels, lse, gl, None, dw, loss=loss)
    want, half = o["P"].t() @ o["h"], 2.0 ** -8
    err = dw.to(F64) - want
    root = (o["P"].square().t() @ o["h"].square()).sum().sqrt()
    own = 0.0 if f32 else half / 3 ** 0.5 * want.norm()
    assert err.norm() <= 1.1 * ((half / 3 ** 0.5 * root) ** 2 + own ** 2) ** 0.5
    size = o["P"].abs().t() @ o["h"].abs()
    assert (err.abs() <= (half + 2.0 ** -11) * size + (0 if f32 else half * (1 + half) * want.abs() + 2.0 ** -133)).all()
