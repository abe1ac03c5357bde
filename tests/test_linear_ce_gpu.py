"""Cross entropy of a linear head without its logits, and its gradients, against the definition in 64 bits.

Bounds.  A logit is a sum of d products in 32 bits: off by D = 8 2^-23 sqrt(d) (root of the sum of squared products), eight
deviations of a sum of random signs whose partial sums may be truncated, plus 2^-22 of its size for the change of base.  The
loss moves by at most (1 - exp(-loss)) 2 D, and by 2^-20 relative through exp, log and the sums.  The gradients use P rounded
to bf16 (half a step: 2^-8 relative to each entry) with exp off by 2 D, are sums in 32 bits (one rounding or truncation,
2^-23, for each addend), and are rounded to bf16 where that is their type."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from pacednegatives_amd import kernels as K  # noqa: E402

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
HALF = torch.finfo(BF16).eps / 2
IGN = -100


def make(R, V, d, seed, ignored=0.1, size=3.0):
    g = torch.Generator("cuda").manual_seed(seed)
    h = (size * d ** -0.5 * torch.randn(R, d, generator=g, device="cuda")).to(BF16)
    w = torch.randn(V, d, generator=g, device="cuda").to(BF16)
    labels = torch.randint(0, V, (R,), generator=g, device="cuda")
    if ignored:
        labels[torch.rand(R, generator=g, device="cuda") < ignored] = IGN
    return h, w, labels, (0.5 + torch.rand(R, generator=g, device="cuda")) / max(R, 1)


def oracle(h, w, labels, gl, scale, ignore=IGN):
    h, w, gl = h.to(F64), w.to(F64), gl.to(F64)
    V, d = w.shape
    z = scale * (h @ w.t())
    lse = torch.logsumexp(z, 1)
    kept = (labels != ignore) & (labels >= 0) & (labels < V)
    at = torch.where(kept, labels, torch.zeros_like(labels))[:, None]
    others = z.scatter(1, at, float("-inf"))
    rest = torch.logsumexp(others, 1)
    own = z.gather(1, at).squeeze(1)
    loss = torch.where(kept, torch.nn.functional.softplus(rest - own, threshold=1e9), torch.zeros_like(lse))
    p = torch.exp(z - lse[:, None]) * kept[:, None]
    P = p.scatter_add(1, at, -kept.to(F64)[:, None]) * gl[:, None]
    D = abs(scale) * 8 * 2.0 ** -23 * d ** 0.5 * (h.square() @ w.square().t()).amax(1).sqrt() + 2.0 ** -22 * z.abs().amax(1)
    return dict(loss=loss, lse=lse, P=P, p=p * gl.abs()[:, None], D=D, h=h, w=w, scale=scale)


def check_loss(o, loss, lse):
    assert ((loss.to(F64) - o["loss"]).abs() <= (1 - torch.exp(-o["loss"])) * 2 * o["D"] + 2.0 ** -20 * o["loss"]).all()
    assert ((lse.to(F64) - o["lse"]).abs() <= 2 * o["D"] + 2.0 ** -20 * o["lse"].abs() + 2.0 ** -20).all()


def check_grads(o, dh, dw, dw0=None):
    s = abs(o["scale"])
    dP = HALF * o["P"].abs() + 2 * (1 + HALF) * o["D"][:, None] * o["p"]
    for got, want, err, entering, n in ((dh, o["scale"] * o["P"] @ o["w"], s * dP @ o["w"].abs(), s * o["P"].abs() @ o["w"].abs(), o["P"].shape[1]),
                                        (dw, o["scale"] * o["P"].t() @ o["h"], s * dP.t() @ o["h"].abs(), s * o["P"].abs().t() @ o["h"].abs(), o["P"].shape[0])):
        if got is None:
            continue
        base = torch.zeros_like(want) if got is dh or dw0 is None else dw0.to(F64)
        # (each of n addends, up to 64 slabs or pieces, and the sum with what was there)
        tol = err + 2.0 ** -23 * (n + 64) * entering + 2.0 ** -23 * base.abs()
        if got.dtype == BF16:
            tol = tol * (1 + HALF) + HALF * want.abs() + 2.0 ** -133
        assert ((got.to(F64) - want - base).abs() <= tol).all()


def run(h, w, labels, gl, scale=1.0, f32=False, **kw):
    R, V = h.shape[0], w.shape[0]
    loss, lse = torch.full((R,), float("nan"), device="cuda"), torch.full((R,), float("nan"), device="cuda")
    K.linear_ce_fwd(h, w, labels, loss, lse, scale=scale, **kw)
    dh = torch.full((R, h.shape[1]), float("nan"), device="cuda", dtype=BF16)
    dw = torch.full((V, h.shape[1]), 0.25 if f32 else float("nan"), device="cuda", dtype=F32 if f32 else BF16)
    K.linear_ce_bwd(h, w, labels, lse, gl, dh, dw, scale=scale, **kw)
    return loss, lse, dh, dw


@pytest.fixture(params=[0, 64, 128, 256])
def tile(request):
    K.gemm_set_tile(request.param)
    yield request.param
    K.gemm_set_tile(0)


@pytest.mark.parametrize("R,V,d", [(1, 1, 64), (1, 7, 64), (2, 100, 64), (3, 64, 128), (16, 6401, 768), (33, 65, 64), (300, 1000, 128), (257, 511, 192), (130, 257, 1024)])
@pytest.mark.parametrize("f32", [False, True])
def test_loss_and_gradients(R, V, d, f32, tile):
    h, w, labels, gl = make(R, V, d, R + V + d, ignored=0.2 if R > 3 else 0.0)
    o = oracle(h, w, labels, gl, 1.0)
    loss, lse, dh, dw = run(h, w, labels, gl, f32=f32)
    check_loss(o, loss, lse)
    check_grads(o, dh, dw, torch.full_like(dw, 0.25) if f32 else None)
    assert (loss[labels == IGN] == 0).all() and (dh[labels == IGN] == 0).all()


@pytest.mark.parametrize("R,V,d", [(777, 6401, 512), (1088, 4096, 768), (2100, 9000, 256), (64, 32128, 512)])
def test_sizes_that_choose_their_own_tiles(R, V, d):
    h, w, labels, gl = make(R, V, d, R)
    o = oracle(h, w, labels, gl, 1.0)
    loss, lse, dh, dw = run(h, w, labels, gl)
    check_loss(o, loss, lse)
    check_grads(o, dh, dw)
    again = run(h, w, labels, gl)
    assert all(torch.equal(a, b) for a, b in zip((loss, lse, dh, dw), again))


@pytest.mark.parametrize("R,V,d,f32", [(1000, 17001, 512, False), (600, 33000, 512, False), (1500, 33000, 768, True), (1088, 32128, 256, False)])
def test_products_in_two_launches(R, V, d, f32):
    """(columns or rows that fill whole rounds of tiles, and the rest)"""
    h, w, labels, gl = make(R, V, d, 12)
    labels[:5] = torch.tensor([V - 1, V - 2, 16383, 16384, 32], device="cuda")
    o = oracle(h, w, labels, gl, 1.0)
    loss, lse, dh, dw = run(h, w, labels, gl, f32=f32)
    check_loss(o, loss, lse)
    check_grads(o, dh, dw, torch.full_like(dw, 0.25) if f32 else None)


@pytest.mark.parametrize("size", [64, 128, 256])
def test_a_forced_tile_where_both_widths_of_statistics_could_meet(size):
    K.gemm_set_tile(size)
    try:
        h, w, labels, gl = make(1100, 13000, 64, 13)
        o = oracle(h, w, labels, gl, 1.0)
        loss, lse, dh, dw = run(h, w, labels, gl)
    finally:
        K.gemm_set_tile(0)
    check_loss(o, loss, lse)
    check_grads(o, dh, dw)


@pytest.mark.parametrize("R,V", [(2816, 2900), (4300, 2561), (2561, 5000)])
def test_more_than_eight_tiles_each_way(R, V):
    """(11 x 12, 17 x 11 and 11 x 20 tiles of 256: bands of unequal width, the last one of a tile's single row or column)"""
    K.gemm_set_tile(256)
    try:
        h, w, labels, gl = make(R, V, 64, 11)
        o = oracle(h, w, labels, gl, 1.0)
        loss, lse, dh, dw = run(h, w, labels, gl)
    finally:
        K.gemm_set_tile(0)
    check_loss(o, loss, lse)
    check_grads(o, dh, dw)


@pytest.mark.parametrize("R,V,d,f32", [(20000, 7001, 64, False), (9000, 20001, 256, True)])
def test_vocabulary_in_several_pieces(R, V, d, f32):
    h, w, labels, gl = make(R, V, d, 5)
    o = oracle(h, w, labels, gl, 1.0)
    loss, lse, dh, dw = run(h, w, labels, gl, f32=f32)
    check_loss(o, loss, lse)
    check_grads(o, dh, dw, torch.full_like(dw, 0.25) if f32 else None)


@pytest.mark.parametrize("scale", [20.0, 0.05, -1.0])
def test_scale_and_confident_rows(scale):
    g = torch.Generator("cuda").manual_seed(3)
    w = torch.nn.functional.normalize(torch.randn(900, 256, generator=g, device="cuda"), dim=1)
    labels = torch.randint(0, 900, (200,), generator=g, device="cuda")
    h = torch.nn.functional.normalize(w[labels] + 0.3 * torch.nn.functional.normalize(torch.randn(200, 256, generator=g, device="cuda"), dim=1), dim=1)
    h, w, gl = h.to(BF16), w.to(BF16), torch.full((200,), 1 / 200, device="cuda")
    o = oracle(h, w, labels, gl, scale)
    loss, lse, dh, dw = run(h, w, labels, gl, scale)
    if scale == 20.0:
        assert o["loss"].min() < 1e-4
    check_loss(o, loss, lse)
    check_grads(o, dh, dw)


def test_agrees_with_the_kernel_on_stored_logits():
    h, w, labels, gl = make(96, 6400, 128, 9)
    logits, l0, loss = torch.empty(96, 6400, device="cuda"), torch.empty(96, device="cuda"), torch.empty(96, device="cuda")
    K.gemm(h, w, logits, epilogue=K.EPI_F32)
    K.cross_entropy(logits, labels, l0)
    K.linear_ce_fwd(h, w, labels, loss)
    D = oracle(h, w, labels, gl, 1.0)["D"]
    assert ((loss - l0).abs() <= 4 * D + 2.0 ** -18 * l0).all()


def test_labels_outside_the_vocabulary_and_garbage_in_ignored_rows():
    h, w, labels, gl = make(40, 300, 64, 2, ignored=0)
    labels[3], labels[4], labels[5], labels[6] = 300, -1, 2 ** 40, 7
    h2 = h.clone()
    h2[3], h2[4] = float("nan"), float("inf")
    for hh in (h, h2):
        loss, lse, dh = torch.empty(40, device="cuda"), torch.empty(40, device="cuda"), torch.empty_like(h)
        K.linear_ce_fwd(hh, w, labels, loss, lse, ignore_index=7)
        K.linear_ce_bwd(hh, w, labels, lse, gl, dh, None, ignore_index=7)
        assert (loss[3:7] == 0).all() and (dh[3:7] == 0).all()
        o = oracle(h, w, labels, gl, 1.0, ignore=7)
        keep = torch.tensor([i for i in range(40) if i not in (3, 4, 5, 6)], device="cuda")
        check_loss({k: v[keep] if k in ("loss", "lse", "D") else v for k, v in o.items()}, loss[keep], lse[keep])
        check_grads(o, dh, None)


def test_all_rows_ignored_and_no_rows():
    h, w, labels, gl = make(20, 130, 64, 1)
    labels.fill_(IGN)
    loss, lse, dh, dw = run(h, w, labels, gl)
    assert (loss == 0).all() and (dh == 0).all() and (dw == 0).all()
    for f32 in (False, True):
        loss, lse, dh, dw = run(h[:0], w, labels[:0], gl[:0], f32=f32)
        assert loss.numel() == 0 and (dw == (0.25 if f32 else 0)).all()


def test_infinite_and_nan_logits_stay_in_their_rows():
    h, w, labels, gl = make(10, 200, 64, 6, ignored=0)
    h[2, 5], h[7, 1] = float("nan"), float("inf")
    loss, lse, dh = torch.empty(10, device="cuda"), torch.empty(10, device="cuda"), torch.empty_like(h)
    K.linear_ce_fwd(h, w, labels, loss, lse)
    K.linear_ce_bwd(h, w, labels, lse, gl, dh)
    ok = torch.tensor([i not in (2, 7) for i in range(10)], device="cuda")
    assert loss[ok].isfinite().all() and dh[ok].isfinite().all()
    assert not loss[~ok].isfinite().any() and dh[~ok].isnan().any(1).all()


def test_strided_rows_and_single_outputs():
    R, V, d = 70, 333, 128
    h, w, labels, gl = make(R, V, d, 4)
    loss, lse, dh, dw = run(h, w, labels, gl)
    hb, wb = torch.zeros(R, d + 40, device="cuda", dtype=BF16), torch.zeros(V, 2 * d, device="cuda", dtype=BF16)
    hb[:, 8:8 + d], wb[:, d:] = h, w
    ob, ow = torch.full((R, d + 16), 3.0, device="cuda", dtype=BF16), torch.full((V, d + 8), 3.0, device="cuda", dtype=BF16)
    l2, e2 = torch.empty(R, device="cuda"), torch.empty(R, device="cuda")
    K.linear_ce_fwd(hb[:, 8:8 + d], wb[:, d:], labels, l2, e2)
    assert torch.equal(l2, loss) and torch.equal(e2, lse)
    K.linear_ce_bwd(hb[:, 8:8 + d], wb[:, d:], labels, lse, gl, ob[:, 8:8 + d], None)
    K.linear_ce_bwd(hb[:, 8:8 + d], wb[:, d:], labels, lse, gl, None, ow[:, :d])
    assert torch.equal(ob[:, 8:8 + d], dh) and torch.equal(ow[:, :d], dw)
    assert (ob[:, :8] == 3).all() and (ob[:, 8 + d:] == 3).all() and (ow[:, d:] == 3).all()


def test_directional_derivative():
    """(L(h + t v) - L(h - t v)) / 2t against <dh, v>, with h, v and t such that h +- t v are bf16 values exactly.  Truncation
    is t^2 / 6 of a third derivative, of order |v w|^3 with v w of order one: below 1e-2 for t = 1/4; dh is bf16 (2^-8)."""
    g = torch.Generator("cuda").manual_seed(8)
    R, V, d, t = 12, 500, 64, 0.25
    h = (torch.randint(-16, 17, (R, d), generator=g, device="cuda") / 16).to(BF16)
    v = (torch.randint(-1, 2, (R, d), generator=g, device="cuda") / 4).to(BF16)
    w = (torch.randn(V, d, generator=g, device="cuda") * 0.3).to(BF16)
    labels, gl = torch.randint(0, V, (R,), generator=g, device="cuda"), torch.ones(R, device="cuda")
    L = [torch.empty(R, device="cuda") for _ in range(3)]
    lse, dh = torch.empty(R, device="cuda"), torch.empty(R, d, device="cuda", dtype=BF16)
    K.linear_ce_fwd(h + t * v, w, labels, L[0])
    K.linear_ce_fwd(h - t * v, w, labels, L[1])
    K.linear_ce_fwd(h, w, labels, L[2], lse)
    K.linear_ce_bwd(h, w, labels, lse, gl, dh)
    got, want = (L[0].double() - L[1].double()) / (2 * t), (dh.double() * v.double()).sum(1)
    scale = (dh.double().square().sum(1) * v.double().square().sum(1)).sqrt()
    assert ((got - want).abs() <= 0.02 * scale + 0.01).all()


def test_captured_and_replayed_beside_eager_calls():
    R, V, d = 300, 3000, 256
    h, w, labels, gl = make(R, V, d, 1)
    loss, lse, dh, dw = torch.empty(R, device="cuda"), torch.empty(R, device="cuda"), torch.empty_like(h), torch.empty_like(w)

    def step():
        K.linear_ce_fwd(h, w, labels, loss, lse)
        K.linear_ce_bwd(h, w, labels, lse, gl, dh, dw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for k in range(3):
        h.copy_(make(R, V, d, 10 + k)[0])
        step()
        want = [t.clone() for t in (loss, lse, dh, dw)]
        for t in (loss, lse, dh, dw):
            t.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((loss, lse, dh, dw), want))


def test_refusals():
    h, w, labels, gl = make(8, 100, 64, 1)
    loss, lse = torch.empty(8, device="cuda"), torch.empty(8, device="cuda")
    for call, words in ((lambda: K.linear_ce_fwd(h[:, :32], w[:, :32], labels, loss), "multiple of 64"), (lambda: K.linear_ce_fwd(h, w, labels.int(), loss), "labels must be"),
                        (lambda: K.linear_ce_fwd(h, w, labels[:4], loss), "labels must hold"), (lambda: K.linear_ce_fwd(h.float(), w, labels, loss), "h must be"),
                        (lambda: K.linear_ce_fwd(h, w, labels, loss[:4]), "loss must hold"), (lambda: K.linear_ce_fwd(h, w[:0], labels, loss), "h must be"),
                        (lambda: K.linear_ce_fwd(h, w.cpu(), labels, loss), "device tensor"), (lambda: K.linear_ce_bwd(h, w, labels, lse, gl, h.float()), "dh must be"),
                        (lambda: K.linear_ce_bwd(h, w, labels, lse, gl, None, w.half()), "dw must be"), (lambda: K.linear_ce_bwd(h, w, labels, lse, gl.double()), "grad_loss must be"),
                        (lambda: K.linear_ce_fwd(h, w, labels, loss, workspace=loss), "workspace must be")):
        with pytest.raises(ValueError, match=words):
            call()
    from pacednegatives_amd._lib import PacedHipError
    buf = torch.zeros(8, 70, device="cuda", dtype=BF16)
    with pytest.raises(PacedHipError, match="multiples of 8"):
        K.linear_ce_fwd(buf[:, :64], w, labels, loss)


@pytest.mark.parametrize("R,V,d", [(1, 8000, 448), (9, 433, 384), (64, 5000, 256), (65, 5000, 256)])
@pytest.mark.parametrize("f32", [False, True])
def test_few_rows_lose_nothing_to_the_rounding_between_the_products(R, V, d, f32):
    """dh gets back what the label's entry lost; up to 64 rows dw is made of both parts of P.  What is left is the result's own
    rounding, half a step 2^-8 at most and uniform: 2^-8 / sqrt(3) of the norm; with fp32 sums dw has P's low part's, 2^-16.
    (dh's other entries, each off by 2^-8 / sqrt(3) of itself, weigh sqrt(sum p^2) against 1 - p: under a third here.)"""
    h, w, labels, gl = make(R, V, d, 77 + R, ignored=0.0, size=1.0)
    o = oracle(h, w, labels, gl, 1.0)
    _, _, dh, dw = run(h, w, labels, gl, f32=f32)
    rel = lambda got, want: ((got.double() - want).norm() / want.norm()).item()  # noqa: E731
    assert rel(dh, o["P"] @ o["w"]) < 1.1 * HALF / 3 ** 0.5
    want = o["P"].t() @ o["h"]
    if R <= 64:
        if f32:       # the sum with 1/4 rounds to 2^-24 of it
            assert (dw.double() - 0.25 - want).norm() <= 2.0 ** -15 * want.norm() + 2.0 ** -25 * dw.numel() ** 0.5
        else:
            assert rel(dw, want) < HALF / 3 ** 0.5
