"""Weight gradients from checkpoints whose tokens span more bytes than one slice's 32-bit offsets reach: wide layers, operands with
far apart rows or heads.  Whole numbers (dy in [-3, 3], values in [-8, 8] times 1, 2 or 4), every sum below 2^24: exact in any order."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from pacednegatives_amd import kernels as K  # noqa: E402

BF16, F32 = torch.bfloat16, torch.float32


def whole(T, n, lo, hi, seed):
    return torch.randint(lo, hi + 1, (T, n), generator=torch.Generator("cuda").manual_seed(seed), dtype=torch.int8, device="cuda")


def checkpoint(T, N, seed):
    x = whole(T, N, -8, 8, seed).to(BF16)
    x *= torch.tensor([1, 2, 4], device="cuda", dtype=BF16)[torch.arange(N, device="cuda") % 3]
    return x, *K.act8_quantize(x)


@pytest.mark.parametrize("T,M,N", [(139264, 8192, 2048), (139264, 4096, 16384)])      # dy, or the codes, of all tokens: over 2 GiB
def test_wide_layers_of_a_long_batch(T, M, N):
    x, q, scale = checkpoint(T, N, 1)
    dy = whole(T, M, -3, 3, 2).to(BF16)
    assert 2 * T * M >= 2 ** 31 or T * N >= 2 ** 31
    rows, cols = torch.tensor([0, 1, 255, 256, 2047, M - 257, M - 1], device="cuda"), torch.tensor([0, 15, 16, 255, 1000, N - 1], device="cuda")
    want = dy[:, rows].float().t() @ x[:, cols].float()
    assert (dy[:, rows].float().abs().t() @ x[:, cols].float().abs()).max() < 2 ** 24
    dw = torch.full((M, N), float("nan"), device="cuda")
    K.act8_dweight(dy, q, scale, dw, accumulate=False)
    assert torch.equal(dw[rows][:, cols], want) and dw.isfinite().all()
    # every element: a row of ones times dw times ones is the sum over tokens of (sum of dy) (sum of x), whole numbers in 64 bits
    assert dw.double().sum() == (dy.sum(1, dtype=torch.float64) * x.sum(1, dtype=torch.float64)).sum()
    K.act8_dweight(dy, q, scale, dw)
    assert torch.equal(dw[rows][:, cols], 2 * want)


@pytest.mark.parametrize("T", [64, 65, 300])
@pytest.mark.parametrize("M,N", [(72, 48), (264, 528)])
@pytest.mark.parametrize("far", [1 << 23, (1 << 24) - 72])
def test_rows_far_apart(T, M, N, far):
    """(slices of one K step: 2^23 elements are 16 MiB, 64 rows of them 1 GiB)"""
    x, q, scale = checkpoint(T, N, 3)
    dy = whole(T, M, -3, 3, 4).to(BF16)
    buf = torch.empty((T - 1) * far + M, device="cuda", dtype=BF16).as_strided((T, M), (far, 1))
    buf.copy_(dy)
    want = dy.float().t() @ x.float()
    dw = torch.full((M, N), float("nan"), device="cuda")
    K.act8_dweight(buf, q, scale, dw, accumulate=False)
    assert torch.equal(dw, want)
    K.act8_dweight(buf, q, scale, dw)
    assert torch.equal(dw, 2 * want)


@pytest.mark.parametrize("T,N", [(64, 64), (200, 80)])
def test_heads_far_apart(T, N):
    far, H = (1 << 28) - 1032, 5
    x, q, scale = checkpoint(T, N, 5)
    dy = whole(T, 64 * H, -3, 3, 6).to(BF16)
    buf = torch.empty((H - 1) * far + (T + 63) // 64 * 64 * 64, device="cuda", dtype=BF16)
    heads = buf.as_strided((H, T, 64), (far, 64, 1))
    buf.as_strided((H, (T + 63) // 64 * 64, 64), (far, 64, 1)).zero_()
    heads.copy_(dy.view(T, H, 64).permute(1, 0, 2))
    dw = torch.full((64 * H, N), float("nan"), device="cuda")
    K.act8_dweight(heads, q, scale, dw, accumulate=False)
    assert torch.equal(dw, dy.float().t() @ x.float())


def test_what_no_slice_reaches_is_refused():
    from pacednegatives_amd._lib import PacedHipError
    x, q, scale = checkpoint(70, 32, 7)
    dw = torch.zeros(8, 32, device="cuda")
    far = 1 << 24
    dy = torch.empty(69 * far + 8, device="cuda", dtype=BF16).as_strided((70, 8), (far, 1))
    with pytest.raises(PacedHipError, match="2 GiB"):
        K.act8_dweight(dy, q, scale, dw)
    assert (dw == 0).all()
