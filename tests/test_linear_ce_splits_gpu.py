"""Products of the linear-head loss that go out as two launches: which cuts are taken, and the values on both sides of each, against
the definition in 64 bits (bounds as in test_linear_ce_gpu.py)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from pacednegatives_amd import kernels as K  # noqa: E402
from test_linear_ce_gpu import IGN, check_grads, check_loss, make, oracle, run  # noqa: E402

SIZES = [(1000, 17001, 512), (600, 33000, 512), (1500, 33000, 768), (1088, 32128, 256), (1088, 32128, 768), (2101, 17001, 512), (4100, 32100, 256), (1300, 50001, 256)]


def cuts_of(R, V, d, f32, labels_at):
    """Runs one case with labels on both sides of every cut; (rows, columns of the forward pass, of the backward pass, rows of dw)."""
    h, w, labels, gl = make(R, V, d, R + V)
    labels[:len(labels_at)] = torch.tensor(labels_at, device="cuda")
    o = oracle(h, w, labels, gl, 1.0)
    loss, lse = torch.empty(R, device="cuda"), torch.empty(R, device="cuda")
    K.linear_ce_fwd(h, w, labels, loss, lse)
    fwd = K.linear_ce_last_split()[:2]
    loss, lse, dh, dw = run(h, w, labels, gl, f32=f32)
    rows, cols, dw_rows = K.linear_ce_last_split()
    check_loss(o, loss, lse)
    check_grads(o, dh, dw, torch.full_like(dw, 0.25) if f32 else None)
    assert (loss[labels == IGN] == 0).all() and (dh[labels == IGN] == 0).all()
    return fwd, (rows, cols), dw_rows


def test_every_kind_of_cut_is_taken_and_right():
    seen = {"rows": 0, "columns": 0, "rows of dw": 0, "none": 0}
    for k, (R, V, d) in enumerate(SIZES):
        f32 = k % 2 == 1
        fwd, (rows, cols), dw_rows = cuts_of(R, V, d, f32, [0, V - 1])
        edges = [e for c in (cols, fwd[1], dw_rows) if c for e in (c - 1, c, c + 1)]
        if edges:                                       # again, with labels beside the cuts
            assert cuts_of(R, V, d, f32, [e for e in edges if e < V] + [V - 1]) == (fwd, (rows, cols), dw_rows)
        print(f"{R} x {V} x {d}: logits {fwd} forward, {(rows, cols)} backward, dw {dw_rows}")
        for c in (rows, fwd[0]):
            assert c == 0 or (c % 256 == 0 and 0 < c < R)
        for c in (cols, fwd[1], dw_rows):
            assert c == 0 or (c % 256 == 0 and 0 < c < V)
        seen["rows"] += bool(rows and fwd[0])
        seen["columns"] += bool(cols and fwd[1])
        seen["rows of dw"] += bool(dw_rows)
        seen["none"] += not (rows or cols)
    assert all(seen.values()), seen


def test_a_single_launch_is_reported_as_one():
    h, w, labels, gl = make(40, 300, 64, 1)
    run(h, w, labels, gl)
    assert K.linear_ce_last_split()[:2] == (0, 0)
    K.gemm_set_tile(128)
    try:
        h, w, labels, gl = make(1088, 32128, 64, 1)
        run(h, w, labels, gl)
        assert K.linear_ce_last_split()[:2] == (0, 0)
    finally:
        K.gemm_set_tile(0)
