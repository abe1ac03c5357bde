"""The loss in a workspace of exactly the bytes it asks for, behind it guards that stay as they are: sizes that take every tile."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from pacednegatives_amd import _lib, kernels as K  # noqa: E402
from test_linear_ce_gpu import check_loss, make, oracle  # noqa: E402


@pytest.mark.parametrize("R,V,d", [(1, 1, 64), (16, 6401, 768), (64, 5000, 64), (65, 333, 64), (130, 4097, 64), (300, 1000, 128), (777, 6401, 512), (600, 33000, 512), (1088, 32128, 768),
                                   (2101, 17001, 512), (4100, 129, 64)])
@pytest.mark.parametrize("tile", [0, 64, 128, 256])
def test_exact_workspace(R, V, d, tile):
    h, w, labels, gl = make(R, V, d, R + V)
    loss, lse = torch.empty(R, device="cuda"), torch.empty(R, device="cuda")
    K.gemm_set_tile(tile)
    try:
        need = _lib.load().paced_linear_ce_fwd_workspace_bytes_for(R, V, d)
        ws = torch.full((need + 65536,), 171, dtype=torch.uint8, device="cuda")
        K.linear_ce_fwd(h, w, labels, loss, lse, workspace=ws)
        assert (ws[need:] == 171).all() and (ws[:need] != 171).any()
    finally:
        K.gemm_set_tile(0)
    check_loss(oracle(h, w, labels, gl, 1.0), loss, lse)


@pytest.mark.parametrize("R,V,d", [(20, 500, 64), (300, 1000, 128), (1088, 32128, 768)])
def test_the_entry_points_without_options_give_the_same_bits(R, V, d):
    """paced_linear_ce_fwd and _bwd, with the workspace that is enough for any d, against the wrappers' calls."""
    lib = _lib.load()
    h, w, labels, gl = make(R, V, d, 3)
    out = []
    for plain in (False, True):
        loss, lse, dh, dw = torch.empty(R, device="cuda"), torch.empty(R, device="cuda"), torch.empty_like(h), torch.empty_like(w)
        if plain:
            fb, bb = lib.paced_linear_ce_fwd_workspace_bytes(R, V), lib.paced_linear_ce_bwd_workspace_bytes(R, V, d)
            ws, s = torch.empty(max(fb, bb), dtype=torch.uint8, device="cuda"), torch.cuda.current_stream().cuda_stream
            p = lambda t: t.data_ptr()  # noqa: E731
            _lib.check(lib.paced_linear_ce_fwd(p(h), d, p(w), d, p(labels), p(loss), p(lse), R, V, d, -100, 1.0, p(ws), fb, s), "paced_linear_ce_fwd")
            _lib.check(lib.paced_linear_ce_bwd(p(h), d, p(w), d, p(labels), p(lse), p(gl), p(dh), d, p(dw), d, 0, R, V, d, -100, 1.0, p(ws), bb, s), "paced_linear_ce_bwd")
            torch.cuda.synchronize()
        else:
            K.linear_ce_fwd(h, w, labels, loss, lse)
            K.linear_ce_bwd(h, w, labels, lse, gl, dh, dw)
        out.append((loss, lse, dh, dw))
    assert all(torch.equal(a, b) for a, b in zip(*out))
