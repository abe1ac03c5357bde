"""8-bit activation checkpoints: codes and scales equal to the definition bit for bit, reading back exact, the weight gradient
exact on whole numbers and within the bound of 32-bit sums otherwise."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from pacednegatives_amd import kernels as K  # noqa: E402

BF16, F64 = torch.bfloat16, torch.float64
# magnitudes of the e4m3 codes 0..126
TABLE = torch.tensor([(m / 512 if e == 0 else (8 + m) * 2.0 ** (e - 10)) for e in range(16) for m in range(8)][:127], dtype=F64)


def definition(x):
    """(codes, scale bytes) of a bf16 [T, n] CPU tensor, in 64 bits by search in the table of all codes."""
    T, n = x.shape
    blocks = (T + 31) // 32
    v = torch.zeros(blocks * 32, n, dtype=F64)
    v[:T] = x.to(F64)
    v = v.view(blocks, 32, n)
    top = v.abs().amax(1)
    bad = ~v.isfinite().all(1)
    reach = torch.tensor([448.0 * 2.0 ** k for k in range(-117, 121)], dtype=F64)
    pick = torch.searchsorted(reach, torch.where(bad, torch.zeros_like(top), top))
    scale = reach[pick] / 448
    a = torch.nan_to_num(v).abs() / scale[:, None]
    hi = torch.searchsorted(TABLE, a).clamp(1, 126)
    lo = hi - 1
    below, above = a - TABLE[lo], TABLE[hi] - a
    code = torch.where((below < above) | ((below == above) & (lo % 2 == 0)), lo, hi)
    code = torch.where((pick == 237)[:, None], code.clamp(max=119), code)
    code = code + 128 * (torch.signbit(v)).to(torch.int64)
    code = torch.where(bad[:, None], torch.full_like(code, -1), code)        # any NaN code
    byte = torch.where(bad, torch.full_like(pick, 255), pick + 10)
    return code.view(blocks * 32, n)[:T], byte


def check_codes(x, q, scale):
    want, byte = definition(x.cpu())
    assert torch.equal(scale.cpu().long(), byte)
    got = q.cpu().long()
    assert torch.equal(torch.where(want < 0, torch.full_like(got, 127), got & 127), torch.where(want < 0, torch.full_like(want, 127), want & 127))
    assert torch.equal(torch.where(want < 0, torch.zeros_like(got), got >> 7), torch.where(want < 0, torch.zeros_like(want), want >> 7))
    assert ((got & 127) == 127)[want < 0].all()


def values(q, scale):
    c, s = q.cpu().long(), scale.cpu().long()
    v = torch.cat([TABLE, torch.tensor([float("nan")], dtype=F64)])[c & 127] * torch.where(c >= 128, -1.0, 1.0)
    return v * torch.exp2((s - 127).to(F64)).repeat_interleave(32, 0)[:q.shape[0]]


def random_x(T, n, seed, wide=False):
    g = torch.Generator().manual_seed(seed)
    if wide:                               # every kind of finite bf16: random bits, blocks of different reach
        bits = torch.randint(0, 65536, (T, n), generator=g)
        x = bits.to(torch.int32).to(torch.int16).view(BF16).double()
        x = torch.where(x.isfinite(), x, torch.zeros_like(x))
        lim = torch.exp2(torch.randint(-130, 128, (1, n), generator=g).double())
        return torch.where(x.abs() < lim, x, x.sign() * lim * torch.rand(T, n, generator=g)).to(BF16).cuda()
    return (torch.randn(T, n, generator=g) * torch.exp(torch.randn(n, generator=g))).to(BF16).cuda()


@pytest.mark.parametrize("T", [1, 7, 31, 32, 33, 64, 300])
@pytest.mark.parametrize("n", [16, 48, 512])
@pytest.mark.parametrize("wide", [False, True])
def test_codes_scales_and_reading_back(T, n, wide):
    x = random_x(T, n, T * 1000 + n, wide)
    q, scale = K.act8_quantize(x)
    check_codes(x, q, scale)
    y = torch.full_like(x, 5)
    K.act8_dequantize(q, scale, y)
    assert torch.equal(y.double().cpu(), values(q, scale))


def test_borders():
    """Largest magnitudes at and about 448 2^k, the largest bf16, subnormals, zeros of both signs, one value in a block."""
    n = 16
    x = torch.zeros(32 * 12, n, dtype=torch.float64)
    for i, top in enumerate((448.0, 450.0, 446.0, 464.0, 2.0 ** -109, 2.0 ** -133, 448 * 2.0 ** -117, 450 * 2.0 ** -117, 3.3895313892515355e38, 2.0 ** 127, 1.75 * 2.0 ** 127, 1.0)):
        x[32 * i] = top
        x[32 * i + 1] = -top
        x[32 * i + 2:32 * i + 31] = top * torch.linspace(-1, 1, 29, dtype=torch.float64)[:, None]
        x[32 * i + 31] = -0.0
    x = x.to(BF16).cuda()
    assert x.isfinite().all()
    q, scale = K.act8_quantize(x)
    check_codes(x, q, scale)
    y = torch.empty_like(x)
    K.act8_dequantize(q, scale, y)
    assert y.isfinite().all() and torch.equal(y.double().cpu(), values(q, scale))


def test_a_block_with_a_nan_or_an_infinity_reads_back_as_nan():
    x = random_x(96, 32, 4)
    x[40, 3], x[70, 8], x[71, 8] = float("nan"), float("inf"), float("-inf")
    q, scale = K.act8_quantize(x)
    check_codes(x, q, scale)
    y = torch.empty_like(x)
    K.act8_dequantize(q, scale, y)
    want = torch.zeros(96, 32, dtype=torch.bool)
    want[32:64, 3] = want[64:96, 8] = True
    assert torch.equal(y.isnan().cpu(), want)
    dw = torch.empty(8, 32, device="cuda")
    K.act8_dweight(torch.ones(96, 8, device="cuda", dtype=BF16), q, scale, dw, accumulate=False)
    assert torch.equal(dw.isnan().cpu(), want.any(0).expand(8, 32))


def test_strided_rows_and_their_surroundings():
    buf = torch.full((70, 96), 3.0, device="cuda", dtype=BF16)
    x = random_x(69, 48, 9)
    buf[:69, 16:64] = x
    q, scale = K.act8_quantize(buf[:69, 16:64])
    q0, s0 = K.act8_quantize(x)
    assert torch.equal(q, q0) and torch.equal(scale, s0)
    K.act8_dequantize(q, scale, buf[:69, 16:64])
    assert (buf[:, :16] == 3).all() and (buf[:, 64:] == 3).all() and (buf[69] == 3).all()
    assert torch.equal(buf[:69, 16:64].double().cpu(), values(q, scale))


def whole(T, M, N, seed, heads=False):
    """Whole numbers: dy in [-3, 3], checkpoint values in [-8, 8] times 1, 2 or 4: sums below 2^24 in any order."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randint(-8, 9, (T, N), generator=g).double() * torch.exp2(torch.randint(0, 3, (N,), generator=g).double())
    dy = torch.randint(-3, 4, (T, M), generator=g).double()
    q, scale = K.act8_quantize(x.to(BF16).cuda())
    assert torch.equal(values(q, scale), x)               # representable: four significant bits
    return dy, x, dy.to(BF16).cuda(), q, scale


@pytest.mark.parametrize("T", [1, 31, 63, 64, 65, 200, 1000, 4096 + 17])
@pytest.mark.parametrize("M,N", [(8, 16), (64, 64), (72, 80), (264, 16), (8, 528), (520, 272)])
def test_weight_gradient_is_exact_on_whole_numbers(T, M, N):
    dy, x, dyd, q, scale = whole(T, M, N, T + M + N)
    want = (dy.t() @ x).float()
    dw = torch.full((M, N), float("nan"), device="cuda")
    K.act8_dweight(dyd, q, scale, dw, accumulate=False)
    assert torch.equal(dw.cpu(), want)
    K.act8_dweight(dyd, q, scale, dw)
    assert torch.equal(dw.cpu(), 2 * want)


@pytest.mark.parametrize("T,M,N", [(300, 512, 512), (5000, 768, 768), (20000, 1024, 512), (70, 2048, 1024), (3000, 2304, 768)])
def test_weight_gradient_exact_at_sizes_that_take_large_tiles(T, M, N):
    dy, x, dyd, q, scale = whole(T, M, N, T + M)
    want = (dy.cuda().t() @ x.cuda()).float()
    dw = torch.full((M, N), float("nan"), device="cuda")
    K.act8_dweight(dyd, q, scale, dw, accumulate=False)
    assert torch.equal(dw, want)


@pytest.mark.parametrize("T,M,N", [(600, 4096, 4096), (9000, 2312, 784), (40000, 768, 768)])
def test_weight_gradient_of_256_tiles_is_written_and_added_to(T, M, N):
    """(one slice, which writes or adds itself; edges inside a tile; many slices)"""
    dy, x, dyd, q, scale = whole(T, M, N, T + M)
    want = (dy.cuda().t() @ x.cuda()).float()
    dw = torch.full((M + 1, N), float("nan"), device="cuda")
    dw[M] = 5
    K.act8_dweight(dyd, q, scale, dw[:M], accumulate=False)
    assert torch.equal(dw[:M], want) and (dw[M] == 5).all()
    K.act8_dweight(dyd, q, scale, dw[:M])
    assert torch.equal(dw[:M], 2 * want) and (dw[M] == 5).all()


@pytest.mark.parametrize("T", [65, 1000])
@pytest.mark.parametrize("H,N", [(1, 64), (3, 80), (12, 768)])
def test_weight_gradient_of_head_major_and_strided_dy(T, H, N):
    M = 64 * H
    dy, x, dyd, q, scale = whole(T, M, N, T + H)
    want = (dy.t() @ x).float().cuda()
    buf = torch.zeros(H, (T + 63) // 64 * 64 + 64, 64, device="cuda", dtype=BF16)
    buf[:, :T] = dyd.view(T, H, 64).permute(1, 0, 2)
    dw = torch.full((M, N), float("nan"), device="cuda")
    K.act8_dweight(buf[:, :T], q, scale, dw, accumulate=False)
    assert torch.equal(dw, want)
    wide = torch.full((T, M + 24), float("nan"), device="cuda", dtype=BF16)
    wide[:, 8:8 + M] = dyd
    out = torch.full((M, N + 12), 5.0, device="cuda")
    K.act8_dweight(wide[:, 8:8 + M], q, scale, out[:, 4:4 + N], accumulate=False)
    assert torch.equal(out[:, 4:4 + N], want) and (out[:, :4] == 5).all() and (out[:, 4 + N:] == 5).all()


@pytest.mark.parametrize("T,M,N", [(777, 128, 144), (30000, 256, 512)])
def test_weight_gradient_within_the_bound_of_32_bit_sums_and_reproducible(T, M, N):
    g = torch.Generator().manual_seed(T)
    x = random_x(T, N, T)
    dy = (torch.randn(T, M, generator=g) * 0.1).to(BF16).cuda()
    q, scale = K.act8_quantize(x)
    dw = torch.empty(M, N, device="cuda")
    K.act8_dweight(dy, q, scale, dw, accumulate=False)
    v = values(q, scale).cuda()
    want, entering = dy.double().t() @ v, dy.double().abs().t() @ v.abs()
    # at most one rounding (or truncation, 2^-23) for each addend
    assert ((dw.double() - want).abs() <= 2.0 ** -23 * (T + 64) * entering).all()
    # and as close as sums of random signs are: 2^-23 sqrt(T) of the root of the sum of squares, 8 deviations
    assert ((dw.double() - want).abs() <= 8 * 2.0 ** -23 * T ** 0.5 * (dy.double().square().t() @ v.square()).sqrt()).all()
    again = torch.empty_like(dw)
    K.act8_dweight(dy, q, scale, again, accumulate=False)
    assert torch.equal(dw, again)


def test_no_tokens():
    x = torch.empty(0, 32, device="cuda", dtype=BF16)
    q, scale = K.act8_quantize(x)
    assert q.shape == (0, 32) and scale.shape == (0, 32)
    K.act8_dequantize(q, scale, x)
    dw = torch.full((8, 32), 3.0, device="cuda")
    K.act8_dweight(torch.empty(0, 8, device="cuda", dtype=BF16), q, scale, dw)
    assert (dw == 3).all()
    K.act8_dweight(torch.empty(0, 8, device="cuda", dtype=BF16), q, scale, dw, accumulate=False)
    assert (dw == 0).all()


def test_captured_and_replayed_beside_eager_calls():
    T, M, N = 2000, 128, 256
    x, dy = random_x(T, N, 1), random_x(T, M, 2)
    q, scale, dw, y = torch.empty(T, N, dtype=torch.uint8, device="cuda"), torch.empty((T + 31) // 32, N, dtype=torch.uint8, device="cuda"), torch.empty(M, N, device="cuda"), torch.empty_like(x)

    def step():
        K.act8_quantize(x, q, scale)
        K.act8_dweight(dy, q, scale, dw, accumulate=False)
        K.act8_dweight(dy, q, scale, dw)
        K.act8_dequantize(q, scale, y)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for k in range(3):
        x.copy_(random_x(T, N, 10 + k))
        step()
        want = [t.clone() for t in (q, scale, dw, y)]
        dw.fill_(1); q.fill_(1)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((q, scale, dw, y), want))


def test_refusals():
    x = random_x(64, 32, 3)
    q, scale = K.act8_quantize(x)
    dy, dw = random_x(64, 16, 4), torch.zeros(16, 32, device="cuda")
    for call, words in ((lambda: K.act8_quantize(x[:, :24]), "multiple of 16"), (lambda: K.act8_quantize(x.float()), "x must be"), (lambda: K.act8_quantize(x, q[:32]), "q must hold"),
                        (lambda: K.act8_quantize(x.cpu()), "device tensor"), (lambda: K.act8_dequantize(q, scale[:1], x), "scale must be"),
                        (lambda: K.act8_dequantize(q, scale, x.float()), "y must be"), (lambda: K.act8_dweight(dy[:63], q, scale, dw), "dy must have shape"),
                        (lambda: K.act8_dweight(dy, q, scale, dw.to(BF16)), "dw must be"), (lambda: K.act8_dweight(dy, q, scale, dw[:8]), "dw must have shape"),
                        (lambda: K.act8_dweight(dy.t(), q, scale, dw), "dy must have shape")):
        with pytest.raises(ValueError, match=words):
            call()
    from pacednegatives_amd._lib import PacedHipError
    with pytest.raises(PacedHipError, match="multiple of 8"):
        K.act8_dweight(random_x(64, 12, 4)[:, :12], q, scale, torch.zeros(12, 32, device="cuda"))
    odd = torch.zeros(64, 40, device="cuda", dtype=BF16)
    with pytest.raises(PacedHipError, match="aligned"):
        K.act8_quantize(odd[:, 1:33])
