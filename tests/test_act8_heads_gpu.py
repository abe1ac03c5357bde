"""The weight gradient that training with 8-bit checkpoints asks for most: head-major dy (q, k and v side by side) through the
256x256 kernel, in the engine's own sizes and in ragged ones.  Whole numbers (dy in [-3, 3], values in [-8, 8] times 1, 2 or 4; sums
below 2^24): exact in any order."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from pacednegatives_amd import _lib, kernels as K  # noqa: E402

BF16 = torch.bfloat16


def operands(T, H, N, gap, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    x = torch.randint(-8, 9, (T, N), generator=g, dtype=torch.int8, device="cuda").to(BF16)
    x *= torch.tensor([1, 2, 4], device="cuda", dtype=BF16)[torch.arange(N, device="cuda") % 3]
    dy = torch.randint(-3, 4, (T, 64 * H), generator=g, dtype=torch.int8, device="cuda").to(BF16)
    # rows behind the last token up to a multiple of 64 are read and have to be finite; behind those nothing is
    rows = (T + 63) // 64 * 64
    buf = torch.full((H, rows + gap, 64), float("nan"), device="cuda", dtype=BF16)
    buf[:, :rows] = 3
    buf[:, :T] = dy.view(T, H, 64).permute(1, 0, 2)
    return x, dy, buf[:, :T]


def exact(dy, x):
    assert dy.shape[0] * 3 * 32 < 2 ** 24
    return dy.float().t() @ x.float()


@pytest.mark.parametrize("T,H,N,gap,tile", [
    (139264, 36, 768, 0, 256),        # q, k, v of t5-base's encoder, 32 tuples of 17 documents of 256 tokens
    (139264 - 47, 36, 768, 64, 256),    # ragged last step, heads further apart than their rows
    (139264, 12, 768, 0, 256),        # one of the three
    (70001, 5, 784, 128, 256),        # 320 features: a tile of 256 and a part of one; 784 inputs likewise
    (40000 + 1, 9, 272, 0, 64),       # (45 tiles of 64 in 17 slices of 37 steps: 34 us by the plan's estimate; 6 of 256 in 42 of 15: 41)
])
def test_head_major_through_the_large_tiles(T, H, N, gap, tile):
    x, dy, heads = operands(T, H, N, gap, T + H)
    q, s = K.act8_quantize(x)
    want = exact(dy, x)
    dw = torch.full((64 * H, N), float("nan"), device="cuda")
    K.act8_dweight(heads, q, s, dw, accumulate=False)
    assert _lib.load().paced_act8_last_tile() == tile
    assert torch.equal(dw, want)
    K.act8_dweight(heads, q, s, dw)                   # what the engine calls: added to
    assert torch.equal(dw, 2 * want)
    rows = torch.empty_like(dw)                       # and the same bits from rows
    K.act8_dweight(dy, q, s, rows, accumulate=False)
    assert torch.equal(rows, want)


@pytest.mark.parametrize("T,H,N", [(600, 64, 4096), (577, 64, 4096)])
def test_one_slice_adds_to_dw_itself(T, H, N):
    x, dy, heads = operands(T, H, N, 64, T)
    q, s = K.act8_quantize(x)
    want = exact(dy, x)
    assert _lib.load().paced_act8_dweight_workspace_bytes(T, 64 * H, N) == 0
    dw = torch.full((64 * H, N + 4), 5.0, device="cuda")
    K.act8_dweight(heads, q, s, dw[:, :N], accumulate=False)
    assert _lib.load().paced_act8_last_tile() == 256
    K.act8_dweight(heads, q, s, dw[:, :N])
    assert torch.equal(dw[:, :N], 2 * want) and (dw[:, N:] == 5).all()


def test_the_small_kernel_reports_itself():
    x, dy, heads = operands(100, 2, 64, 0, 1)
    q, s = K.act8_quantize(x)
    dw = torch.zeros(128, 64, device="cuda")
    K.act8_dweight(heads, q, s, dw)
    assert _lib.load().paced_act8_last_tile() == 64 and torch.equal(dw, exact(dy, x))
