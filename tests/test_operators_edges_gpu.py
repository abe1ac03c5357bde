"""Layer norm, 8-bit checkpoints and the linear-head loss where calls meet: several streams at once, workspaces of the caller's,
tensors whose offsets pass 32 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from pacednegatives_amd import _lib, kernels as K  # noqa: E402

BF16, F32, U8 = torch.bfloat16, torch.float32, torch.uint8


def rn(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator("cuda").manual_seed(seed), device="cuda")


def all_operators(seed):
    """One pass through everything; returns the closure that runs it and its outputs."""
    R, V, d, T = 900, 5000, 256, 3000
    h, w = (rn(seed, R, d) * 0.1).to(BF16), rn(seed + 1, V, d).to(BF16)
    labels = torch.randint(0, V, (R,), generator=torch.Generator("cuda").manual_seed(seed), device="cuda")
    gl = rn(seed + 2, R).abs()
    x, dy = rn(seed + 3, T, d).to(BF16), rn(seed + 4, T, 512).to(BF16)
    n, b = rn(seed + 5, d).to(BF16), rn(seed + 6, d).to(BF16)

    def run():
        e = lambda *s: torch.empty(*s, device="cuda")  # noqa: E731
        loss, lse, dh, dw = e(R), e(R), torch.empty_like(h), torch.empty_like(w)
        K.linear_ce_fwd(h, w, labels, loss, lse)
        K.linear_ce_bwd(h, w, labels, lse, gl, dh, dw)
        y, mean, rstd, dx, dn, db = torch.empty_like(x), e(T), e(T), torch.empty_like(x), torch.zeros(d, device="cuda"), torch.zeros(d, device="cuda")
        K.layernorm_fwd(x, n, b, y, mean, rstd)
        q, s = K.act8_quantize(y)
        dw8 = e(512, d)
        K.act8_dweight(dy, q, s, dw8, accumulate=False)
        K.layernorm_bwd(y, x, n, mean, rstd, dx, dw=dn, db=db)
        return [loss, lse, dh, dw, y, q, s, dw8, dx, dn, db]
    return run


def test_calls_on_several_streams_at_once():
    runs = [all_operators(100 * k) for k in range(3)]
    want = [[t.clone() for t in r()] for r in runs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in runs]
    got = [None] * 3
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        for k, (r, s) in enumerate(zip(runs, streams)):
            with torch.cuda.stream(s):
                got[k] = r()
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_workspaces_of_the_callers():
    """A workspace that is large enough is used up to the size asked for and not beyond; a smaller one is not used at all."""
    lib = _lib.load()
    R, V, d, T = 300, 1000, 128, 4000
    h, w, gl = (rn(1, R, d) * 0.1).to(BF16), rn(2, V, d).to(BF16), rn(3, R).abs()
    labels = torch.arange(R, device="cuda")
    x, dy, n = rn(4, T, d).to(BF16), rn(5, T, 64).to(BF16), torch.ones(d, device="cuda", dtype=BF16)
    e = lambda *s: torch.empty(*s, device="cuda")  # noqa: E731
    loss, lse, dh, dw, y, mean, rstd, dx = e(R), e(R), torch.empty_like(h), torch.empty_like(w), torch.empty_like(x), e(T), e(T), torch.empty_like(x)
    q, s = K.act8_quantize(x)
    K.layernorm_fwd(x, n, n, y, mean, rstd)
    dn, dw8 = e(d), e(64, d)

    def calls(ws):
        dn.zero_()
        K.linear_ce_fwd(h, w, labels, loss, lse, workspace=ws(lib.paced_linear_ce_fwd_workspace_bytes(R, V)))
        K.linear_ce_bwd(h, w, labels, lse, gl, dh, dw, workspace=ws(lib.paced_linear_ce_bwd_workspace_bytes(R, V, d)))
        K.layernorm_bwd(y, x, n, mean, rstd, dx, dw=dn, workspace=ws(lib.paced_layernorm_workspace_bytes(T, d)))
        K.act8_dweight(dy, q, s, dw8, accumulate=False, workspace=ws(lib.paced_act8_dweight_workspace_bytes(T, 64, d)))
        return [t.clone() for t in (loss, lse, dh, dw, dx, dn, dw8)]
    want = calls(lambda need: None)
    given = []

    def exact(need):
        given.append((need, torch.full((need + 4096,), 171, dtype=U8, device="cuda")))
        return given[-1][1]
    assert all(torch.equal(a, b) for a, b in zip(calls(exact), want))
    for need, t in given:
        assert need > 0 and (t[need:] == 171).all() and (t[:need] != 171).any()
    small = torch.full((64,), 171, dtype=U8, device="cuda")
    assert all(torch.equal(a, b) for a, b in zip(calls(lambda need: small), want)) and (small == 171).all()


def test_layer_norm_past_32_bit_offsets():
    M, d = 270_000, 8192                                 # 2.2e9 elements
    x = torch.zeros(M, d, device="cuda", dtype=BF16)
    rows = torch.tensor([0, 1, M // 2, 262_144, M - 1], device="cuda")       # 262144 * 8192 = 2^31
    x[rows] = rn(1, 5, d).to(BF16)
    w, b = rn(2, d).to(BF16), rn(3, d).to(BF16)
    mean, rstd = torch.empty(M, device="cuda"), torch.empty(M, device="cuda")
    few = x[rows].clone()
    y5, m5, r5 = torch.empty_like(few), torch.empty(5, device="cuda"), torch.empty(5, device="cuda")
    K.layernorm_fwd(few, w, b, y5, m5, r5)
    K.layernorm_fwd(x, w, b, x, mean, rstd)              # in place
    assert torch.equal(x[rows], y5) and torch.equal(mean[rows], m5) and torch.equal(rstd[rows], r5)
    assert torch.equal(x[262_143], b)                    # a row of zeros
    x.zero_()
    x[rows] = few
    dw, dw5, dx5 = torch.zeros(d, device="cuda"), torch.zeros(d, device="cuda"), torch.empty_like(few)
    K.layernorm_bwd(few, few, w, m5, r5, dx5, dw=dw5)
    mean.zero_()
    rstd.zero_()
    mean[rows], rstd[rows] = m5, r5
    K.layernorm_bwd(x, x, w, mean, rstd, x, dw=dw)
    assert torch.equal(x[rows], dx5) and (x[262_143] == 0).all()
    assert torch.allclose(dw, dw5, rtol=1e-5, atol=1e-4)  # five addends of order one in another order


def test_checkpoints_past_32_bit_offsets():
    T, n = 1_100_000, 2048                               # 2.25e9 elements
    x = torch.zeros(T, n, device="cuda", dtype=BF16)
    at = [0, 31, 1_048_575, 1_048_576, T - 1]            # 1048576 * 2048 = 2^31
    for k, r in enumerate(at):
        x[r] = float(k + 1)
    q, s = K.act8_quantize(x)
    K.act8_dequantize(q, s, x)                           # whole numbers up to 5: exact
    for k, r in enumerate(at):
        assert (x[r] == k + 1).all()
    assert x[1_048_574].abs().max() == 0 and x[T - 2].abs().max() == 0
    dy = torch.zeros(T, 8, device="cuda", dtype=BF16)
    dy[:, 1] = 1
    dy[1_048_576:, 2] = 1
    dw = torch.empty(8, n, device="cuda")
    K.act8_dweight(dy, q, s, dw, accumulate=False)
    assert (dw[1] == 15).all() and (dw[2] == 9).all() and (dw[0] == 0).all()


def test_linear_loss_past_32_bit_offsets():
    V, d, R = 2_200_000, 1024, 16                        # 2.25e9 weights; 2097152 * 1024 = 2^31
    w = torch.zeros(V, d, device="cuda", dtype=BF16)
    w[V - 1] = 1
    h = torch.full((R, d), 2.0 ** -8, device="cuda", dtype=BF16)             # z = 4 for the last entry, 0 for the others
    labels = torch.tensor([V - 1, 2_097_152, 0, 5] * 4, device="cuda")
    loss, lse, dh, dw, gl = torch.empty(R, device="cuda"), torch.empty(R, device="cuda"), torch.empty_like(h), torch.empty_like(w), torch.ones(R, device="cuda")
    K.linear_ce_fwd(h, w, labels, loss, lse)
    L = math.log(V - 1 + math.exp(4.0))
    want = torch.tensor([L - 4, L, L, L] * 4, device="cuda")
    assert torch.allclose(lse, torch.full_like(lse, L), rtol=2 ** -20) and torch.allclose(loss, want, rtol=2 ** -20)
    K.linear_ce_bwd(h, w, labels, lse, gl, dh, dw)
    p = math.exp(4 - L)
    tol = 3 * 2 ** -8                                    # P, the result, and P's sum in bf16
    assert torch.allclose(dh[0].float(), torch.full((d,), p - 1, device="cuda"), rtol=tol) and torch.allclose(dh[1].float(), torch.full((d,), p, device="cuda"), rtol=tol)
    q = math.exp(-L)
    for row, val in ((V - 1, 16 * p - 4), (2_097_152, 16 * q - 4), (5, 16 * q - 4), (7, 16 * q), (2_097_153, 16 * q), (V - 2, 16 * q)):
        assert torch.allclose(dw[row].float(), torch.full((d,), val * 2.0 ** -8, device="cuda"), rtol=tol), row
