"""Ordinary products take the kernel of their own rule, whatever calls of the linear-head loss (which choose a tile for each of
their products) came before them on the same thread."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from pacednegatives_amd import _lib, kernels as K  # noqa: E402

BF16, F32 = torch.bfloat16, torch.float32


def rn(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator("cuda").manual_seed(seed), device="cuda").to(BF16)


def loss_and_gradients(R, V, d):
    h, w, labels = rn(1, R, d), rn(2, V, d), torch.arange(R, device="cuda") % V
    loss, lse, dh, dw = torch.empty(R, device="cuda"), torch.empty(R, device="cuda"), torch.empty_like(h), torch.zeros(V, d, device="cuda")
    K.linear_ce_fwd(h, w, labels, loss, lse)
    K.linear_ce_bwd(h, w, labels, lse, torch.ones(R, device="cuda"), dh, dw)


@pytest.mark.parametrize("R,V,d", [(16, 500, 64), (300, 1000, 128), (1000, 17001, 512)])        # 64, 128 and 256 wide tiles
def test_products_after_calls_of_the_loss(R, V, d):
    last = _lib.load().paced_gemm_last_kernel
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    small, wide = (rn(3, 100, 256), rn(4, 128, 256)), (rn(5, 256 * 20, 128), rn(6, 256 * 20, 128))
    x, dy = rn(7, 512, 256), rn(8, 512, 256)
    middle = (rn(9, 2048, 128), rn(10, 1536, 128))
    assert 16 * 12 >= cus // 2 and 20 * 20 >= 200
    for _ in range(2):
        loss_and_gradients(R, V, d)
        c = torch.empty(100, 128, device="cuda", dtype=BF16)
        K.gemm(*small, c)
        assert last() == 65                                     # few tiles: 64x64, ring
        loss_and_gradients(R, V, d)
        g = torch.zeros(256, 256, device="cuda")
        K.gemm(dy, x, g, trans_a=True, trans_b=True, epilogue=K.EPI_ATOMIC_F32, splits=0)
        assert last() == 65                                     # a short contraction's weight gradient
        loss_and_gradients(R, V, d)
        m = torch.empty(2048, 1536, device="cuda", dtype=BF16)
        K.gemm(*middle, m)
        assert last() == 128
        loss_and_gradients(R, V, d)
        bits = K.sign_bits_buffer(256 * 20, 256 * 20, "cuda")
        assert bits.dim() == 1
        b = torch.empty(256 * 20, 256 * 20, device="cuda", dtype=BF16)
        K.gemm(*wide, b, epilogue=K.EPI_RELU_DROP, aux=bits)
        assert last() == 256                                    # (a tile-ordered bit matrix is refused by any other)
    for got, (p, q) in ((c, small), (m, middle)):
        want = p.double() @ q.double().t()
        assert ((got.double() - want).abs() <= 2 ** -8 * want.abs() + 2.0 ** -23 * 256 * (p.double().abs() @ q.double().abs().t())).all()
    want = dy.double().t() @ x.double()
    assert ((g.double() - want).abs() <= 2.0 ** -23 * 520 * (dy.double().abs().t() @ x.double().abs())).all()
