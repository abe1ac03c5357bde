"""The loss's gradients where the vocabulary goes by in pieces because of w's row stride, against the definition in 64 bits (bounds
as in test_linear_ce_gpu.py: the number of pieces is among a sum's addends there)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from pacednegatives_amd import kernels as K  # noqa: E402
from test_linear_ce_gpu import IGN, check_grads, check_loss, make, oracle  # noqa: E402

BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("R,V,d,far", [(20, 1000, 64, 1 << 22), (70, 1100, 128, 1 << 22), (300, 2049, 64, 1 << 21), (600, 5000, 256, 3 << 18)])
@pytest.mark.parametrize("f32", [False, True])
def test_rows_of_w_far_apart(R, V, d, far, f32):
    h, w, labels, gl = make(R, V, d, R)
    labels[:6] = torch.tensor([V - 1, 0, 255, 256, 511, IGN], device="cuda")
    buf = torch.empty((V - 1) * far + d, device="cuda", dtype=BF16).as_strided((V, d), (far, 1))
    buf.copy_(w)
    assert V * far >= 2 ** 31
    o = oracle(h, w, labels, gl, 1.0)
    loss, lse, dh = torch.empty(R, device="cuda"), torch.empty(R, device="cuda"), torch.full_like(h, float("nan"))
    dw = torch.full((V, d), 0.25 if f32 else float("nan"), device="cuda", dtype=F32 if f32 else BF16)
    K.linear_ce_fwd(h, buf, labels, loss, lse)
    K.linear_ce_bwd(h, buf, labels, lse, gl, dh, dw, loss=loss)
    check_loss(o, loss, lse)
    check_grads(o, dh, dw, torch.full_like(dw, 0.25) if f32 else None)
    assert (dh[labels == IGN] == 0).all()
    again, dw2 = torch.empty_like(dh), torch.full_like(dw, 0.25)
    K.linear_ce_bwd(h, buf, labels, lse, gl, again, dw2, loss=loss)
    assert torch.equal(again, dh) and torch.equal(dw2, dw)
