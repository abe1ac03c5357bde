"""What the lceT5 step asks of the linear-head loss: one call for each state's rows, and the no-grad forwards' launch limit."""
import warnings

import pytest
import torch

pytestmark = pytest.mark.gpu

from pacednegatives_amd import kernels as K  # noqa: E402

HP = {"model_name": "t5-tiny", "total_steps": 10, "eta": 35.0, "batch_size": 2, "lr": 1e-3, "meta_lr": 1e-2, "n": 3, "warmup_steps": 0,
      "use_mean": False, "ignore_index": -100, "dropout": 0.0, "seed": 0, "fused_loss": True}


@pytest.mark.parametrize("neg_len,rows", [(40, [16]), (24, [4, 12])])          # lengths agree: one packed state; else one each
def test_each_state_is_one_call_and_the_no_grad_pass_keeps_its_launch_limit(neg_len, rows, monkeypatch):
    from pacednegatives_amd.config import NAMED
    from pacednegatives_amd.lceT5 import LCEModel
    from pacednegatives_amd.synthetic import token_batch
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        m = LCEModel(HP | {"nograd_grid": 100})
    calls, inner = [], K.linear_ce_fwd

    def record(h, w, labels, loss, lse=None, **kw):
        calls.append((h.shape[0], lse is not None, kw.get("grid_limit")))
        return inner(h, w, labels, loss, lse, **kw)
    monkeypatch.setattr(K, "linear_ce_fwd", record)
    got = []
    for it in range(3):                       # (the first step runs in order, without a limit; the others beside each other)
        pos, neg = token_batch(2, 3, 40, NAMED["t5-tiny"].vocab_size, seed=50 + it)
        neg = {"input_ids": neg["input_ids"][:, :neg_len].contiguous(), "labels": neg["labels"]}
        got.append(m.training_step((pos, neg), it))
        torch.cuda.synchronize()
        saving, no_grad = [c for c in calls if c[1]], [c for c in calls if not c[1]]
        assert [c[0] for c in saving] == rows and [c[0] for c in no_grad] == rows
        assert all(c[2] is None for c in saving) and all(c[2] == (None if it == 0 else 100) for c in no_grad)
        calls.clear()
        # without dropout the two passes see the same parameters: the same rows, whatever the limit
        assert torch.equal(got[-1]["loss_rows"], got[-1]["main_loss_rows"])


def test_the_limit_limits_the_launch_and_leaves_the_bits():
    g = torch.Generator("cuda").manual_seed(1)
    R, V, d = 2048, 16384, 512                                                  # 512 tiles of 256x256
    h, w = (torch.randn(R, d, generator=g, device="cuda") * 0.1).to(torch.bfloat16), torch.randn(V, d, generator=g, device="cuda").to(torch.bfloat16)
    labels = torch.randint(0, V, (R,), generator=g, device="cuda")

    def run(limit):
        loss, lse = torch.empty(R, device="cuda"), torch.empty(R, device="cuda")
        best = 1e9
        for _ in range(5):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            K.linear_ce_fwd(h, w, labels, loss, lse, grid_limit=limit)
            b.record()
            b.synchronize()
            best = min(best, a.elapsed_time(b))
        return loss, lse, best
    free, few, half = run(None), run(8), run(128)
    for other in (few, half):
        assert torch.equal(free[0], other[0]) and torch.equal(free[1], other[1])
    assert few[2] > 5 * free[2]                                                 # 64 tiles for each of 8 workgroups instead of 2 for each of 256
    K.gemm_set_grid(8)
    try:
        assert run(None)[2] > 5 * free[2] and run(0)[2] < 2 * free[2]           # the process default, and a call that lifts it
    finally:
        K.gemm_set_grid(0)
