"""The operators as they are used together: in the lceT5 step (``fused_loss``, ``act8``) and as the head of an encoder language
model (residual sum and layer norm, product, 8-bit checkpoint of its input, loss over the vocabulary, backward through all)."""
import os
import subprocess
import sys
import warnings

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from pacednegatives_amd import kernels as K  # noqa: E402

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HP = {"model_name": "t5-tiny", "total_steps": 10, "eta": 35.0, "batch_size": 2, "lr": 1e-3, "meta_lr": 1e-2, "n": 3, "warmup_steps": 0,
      "use_mean": False, "ignore_index": -100, "dropout": 0.0, "seed": 0}


def step(neg_len=40, steps=1, **hp):
    """Rows, losses and summed gradients of training steps with the given options."""
    from pacednegatives_amd.config import NAMED
    from pacednegatives_amd.lceT5 import LCEModel
    from pacednegatives_amd.synthetic import token_batch
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        m = LCEModel(HP | hp)
    got = []
    m.on_gradients_ready = lambda m: got.append({k: m.model.params.grad(k).clone() for k in m.model.params.names()})
    out = []
    for it in range(steps):
        pos, neg = token_batch(2, 3, 40, NAMED["t5-tiny"].vocab_size, seed=50 + it)
        if neg_len != 40:
            neg = {"input_ids": neg["input_ids"][:, :neg_len].contiguous(), "labels": neg["labels"]}
        r = m.training_step((pos, neg), it)
        out.append((r["loss_rows"].clone(), r["main_loss_rows"].clone()))
    torch.cuda.synchronize()
    return out, got, m


def rel(a, b):
    return ((a.double() - b.double()).norm() / b.double().norm().clamp_min(1e-30)).item()


@pytest.mark.parametrize("neg_len", [40, 24])
def test_the_step_with_the_fused_loss_is_the_step(neg_len):
    """Same states; the loss rows differ by 32-bit summation order, d loss / d logits by the entries that round to the other
    bf16 neighbour for it, and every product behind rounds its operands to bf16 (half a step 2^-8): 2^-7 covers two."""
    want, gw, _ = step(neg_len)
    got, gg, _ = step(neg_len, fused_loss=True)
    for a, b in zip(got[0], want[0]):
        assert torch.allclose(a, b, rtol=2e-5, atol=0)
    for k in gw[0]:
        assert rel(gg[0][k], gw[0][k]) < 2 ** -7, k


def test_steps_with_the_fused_loss_side_streams_and_dropout_run_ahead():
    """Several overlapped steps: the fused and the stored-logits schedules draw the same masks and stay together."""
    want, _, _ = step(steps=3, dropout=0.1)
    got, _, m = step(steps=3, dropout=0.1, fused_loss=True)
    assert torch.allclose(got[0][1], want[0][1], rtol=2e-5)
    for a, b in zip(got, want):
        assert torch.allclose(a[1], b[1], rtol=2e-2)          # from the second step on the parameters differ by their updates
    assert m.model.params.g32.abs().max() == 0


@pytest.mark.parametrize("head_major", ["1", "0"])
def test_the_step_with_8_bit_checkpoints(head_major, monkeypatch):
    """Only the encoder's qkv, wi and wo gradients read checkpoints.  An e4m3 value is off by 2^-4 of itself at most, so
    |dw - dw'| <= 2^-4 |dy|^T |x| entry by entry and, the errors being independent of the signs, 2^-4 of the norm as a whole."""
    monkeypatch.setenv("PACED_HEAD_MAJOR", head_major)
    want, gw, _ = step()
    got, gg, m = step(act8=True)
    assert m.model.engine.act8
    assert all(torch.equal(a, b) for a, b in zip(got[0], want[0]))
    changed = 0
    for k in gw[0]:
        if k.startswith("enc.") and k.rsplit(".", 1)[1] in ("qkv", "wi", "wo"):
            assert 1e-4 < rel(gg[0][k], gw[0][k]) < 2 ** -4, k
            changed += 1
        else:
            assert rel(gg[0][k], gw[0][k]) < 1e-5, k           # fp32 atomics in another order
    assert changed == 6


def test_checkpoints_take_less_memory():
    from pacednegatives_amd.config import T5Dims
    from pacednegatives_amd.model import T5ForConditionalGenerationHIP
    dims = T5Dims(6400, 512, 64, 8, 2048, 4, 1)
    ids, lab = torch.randint(0, 6400, (8, 512)), torch.randint(0, 6400, (8, 2))
    held = []
    for on in (False, True):
        m = T5ForConditionalGenerationHIP(dims, device="cuda", seed=1)
        m.engine.act8 = on
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        st = m.engine.forward(ids, lab, save=True, want_logits=False)
        held.append(torch.cuda.memory_allocated() - before)
        m.engine.backward(st, dy=torch.zeros_like(st.y))
        del st
    # of xn, xn2 (d_model wide) and act (d_ff wide) 1 + 1/32 bytes are kept instead of 2
    saved = 4 * 8 * 512 * (512 * 2 + 2048) * (1 - 1 / 32)
    assert abs(held[0] - held[1] - saved) < 0.02 * saved


def test_the_training_command_takes_both(tmp_path):
    sys.path.insert(0, os.path.join(ROOT, "train"))
    import train_lce
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        model, trainer = train_lce.main(data="", dataset_name="", out_dir=str(tmp_path), total_steps=16, batch_size=2, n=2, num_workers=0, max_steps=2,
                                        model_name="t5-tiny", synthetic=8, eta=30.0, warmup_steps=2, fused_loss=True, act8=True)
    assert model.fused_loss and model.model.engine.act8 and model.global_step == 2
    assert os.path.exists(os.path.join(str(tmp_path), "finalmodel", "model.safetensors"))


def test_head_of_an_encoder_language_model():
    """x -> s = x + res, y = norm(s) -> t = y w1^T -> u = norm(t) -> loss over the vocabulary of u, and back to w1, both norms
    and x; y is kept in 8 bits for w1's gradient.  Reference: the same chain in 64 bits on the same bf16 operands, rounded
    where the chain stores (autograd through a straight-through rounding).  Each stored tensor is off by half a bf16 step and
    every later one inherits it: with five stores between the loss and x, 6 * 2^-8 of each gradient's norm; the checkpoint adds
    2^-4 to w1's."""
    R, d, V = 700, 256, 3001
    g = torch.Generator("cuda").manual_seed(4)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    x, res, w1, wv = rn(R, d).to(BF16), rn(R, d).to(BF16), (rn(d, d) / 16).to(BF16), (rn(V, d) * 0.5).to(BF16)
    n1, b1, n2, b2 = [(1 + 0.2 * rn(d)).to(BF16) if i % 2 == 0 else (0.2 * rn(d)).to(BF16) for i in range(4)]
    labels = torch.randint(0, V, (R,), generator=g, device="cuda")
    labels[::7] = -100
    gl = torch.full((R,), 1 / R, device="cuda")
    e = lambda *s: torch.empty(*s, device="cuda")  # noqa: E731
    s, y, t, u = [torch.empty_like(x) for _ in range(4)]
    m1, r1, m2, r2, loss, lse = e(R), e(R), e(R), e(R), e(R), e(R)
    K.layernorm_fwd(x, n1, b1, y, m1, r1, res=res, xsum=s)
    y8 = K.act8_quantize(y)
    K.gemm(y, w1, t)
    K.layernorm_fwd(t, n2, b2, u, m2, r2)
    K.linear_ce_fwd(u, wv, labels, loss, lse)
    du, dt, dy, dx, dwv = torch.empty_like(x), torch.empty_like(x), torch.empty_like(x), torch.empty_like(x), torch.empty_like(wv)
    dn1, db1, dn2, db2, dw1 = [torch.zeros(d, device="cuda") for _ in range(4)] + [torch.zeros(d, d, device="cuda")]
    K.linear_ce_bwd(u, wv, labels, lse, gl, du, dwv)
    K.layernorm_bwd(du, t, n2, m2, r2, dt, dw=dn2, db=db2)
    K.act8_dweight(dt, *y8, dw1)
    K.gemm(dt, w1, dy, trans_b=True)
    K.layernorm_bwd(dy, s, n1, m1, r1, dx, dw=dn1, db=db1)

    class Round(torch.autograd.Function):
        @staticmethod
        def forward(ctx, v):
            return v.to(BF16).to(F64)

        @staticmethod
        def backward(ctx, gv):
            return gv
    leaf = {k: v.to(F64).requires_grad_() for k, v in dict(x=x, w1=w1, wv=wv, n1=n1, b1=b1, n2=n2, b2=b2).items()}

    def norm(v, w, b):
        c = v - v.mean(1, keepdim=True)
        return c * (c.square().mean(1, keepdim=True) + 1e-5).rsqrt() * w + b
    h = Round.apply(norm(Round.apply(leaf["x"] + res.to(F64)), leaf["n1"], leaf["b1"]))
    h = Round.apply(norm(Round.apply(h @ leaf["w1"].t()), leaf["n2"], leaf["b2"]))
    want = torch.nn.functional.cross_entropy(h @ leaf["wv"].t(), labels, reduction="none")
    (want * gl.to(F64)).sum().backward()
    # u and what it is computed from may fall on the other side of a rounding: a logit moves by 2^-8 of its addends' root sum
    tol = 4 * 2 ** -8 * (u.double().square() @ wv.double().square().t()).amax(1).sqrt()
    assert ((loss.double() - want).abs() <= tol).all() and (loss[::7] == 0).all()
    for name, got, extra in (("wv", dwv, 0), ("n2", dn2, 0), ("b2", db2, 0), ("w1", dw1, 2 ** -4), ("n1", dn1, 0), ("b1", db1, 0), ("x", dx, 0)):
        r = rel(got, leaf[name].grad)
        print(f"{name}: {r:.2e}")
        assert r < 6 * 2 ** -8 + extra, name
