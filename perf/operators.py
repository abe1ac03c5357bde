"""Cases, plain forms and 64-bit values of the training operators that stand beside the T5 step's kernels:

* ``lm``   -- ``kernels.linear_ce_fwd`` / ``linear_ce_bwd``: cross entropy of a linear head over a large vocabulary (or of
  queries against a batch of documents) without the logits, and its gradients;
* ``ckpt`` -- ``kernels.act8_quantize`` / ``act8_dequantize``: an activation kept for the backward pass in 8 bits (e4m3 with
  one power-of-two scale for 32 tokens of a feature) and read back;
* ``dw``   -- ``kernels.act8_dweight``: a weight gradient from such a checkpoint;
* ``ln``   -- ``kernels.layernorm_fwd`` / ``layernorm_bwd``: layer norm with a residual sum, its gradients and the reduction
  of the weight's and the bias's.

``own`` false computes the plain forms with elementary torch operations in 32 bits, true calls the framework.
"""
import torch


own = False

BF16, F32 = torch.bfloat16, torch.float32
TYPES = {"bf16": BF16, "f32": F32}
IGNORE = -100


def _kernels():
    from pacednegatives_amd import kernels
    return kernels


# ------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # scoring of 8 (query, document) pairs: two target positions each, T5's vocabulary; a call's latency
        dict(name="lm_score_8_pairs", op="lm", rows=16, vocab=32128, d=768, train=False, scale=1.0, ignored=0.0),
        # one training step's target rows: 32 tuples of a query with 1 + 16 documents, two positions each
        dict(name="lm_train_32_tuples", op="lm", rows=1088, vocab=32128, d=768, train=True, scale=1.0, ignored=0.0),
        # a ragged batch over a vocabulary of odd size, padded positions among the labels
        dict(name="lm_train_odd_vocab", op="lm", rows=777, vocab=6401, d=512, train=True, scale=1.0, ignored=0.1),
        # contrastive training of a dense retriever: 512 queries against their batch's 17 documents each, temperature 0.05
        dict(name="lm_contrast_512", op="lm", rows=512, vocab=8704, d=768, train=True, scale=20.0, ignored=0.0),
        # language-model training of a large head: 8192 tokens, 50,001 entries
        dict(name="lm_train_8k_tokens", op="lm", rows=8192, vocab=50001, d=1024, train=True, scale=1.0, ignored=0.05),
        # the checkpoint of one short document batch
        dict(name="ckpt_300_tokens", op="ckpt", tokens=300, d=512, relu=False),
        # the checkpoint of one encoder layer's input: 32 tuples of 17 documents of 256 tokens
        dict(name="ckpt_139k_tokens", op="ckpt", tokens=139264, d=768, relu=False),
        # a small model's feed-forward gradient from a ragged batch, ReLU activations with dropout
        dict(name="dw_1001_tokens", op="dw", tokens=1001, d_out=512, d_in=2048, relu=True),
        # the fused q, k, v projection's gradient of one encoder layer, 32 tuples of 17 documents of 256 tokens
        dict(name="dw_139k_tokens", op="dw", tokens=139264, d_out=2304, d_in=768, relu=False),
        # one token's norm: latency
        dict(name="ln_one_token", op="ln", rows=1, d=768, dtype="bf16", train=False, residual=True),
        # a ragged 32-bit batch of an odd width, forward and backward
        dict(name="ln_train_odd_f32", op="ln", rows=5001, d=1023, dtype="f32", train=True, residual=False),
        # one layer's norm in training: 32 tuples of 17 documents of 256 tokens, with the residual sum
        dict(name="ln_train_139k_tokens", op="ln", rows=139264, d=768, dtype="bf16", train=True, residual=True),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    top = {c["op"]: max(_cost(x) for x in listed() if x["op"] == c["op"]) for c in listed()}
    while True:
        op = rng.choice(["lm", "lm", "ckpt", "dw", "ln", "ln"])
        if op == "lm":
            contrast = rng.random() < 0.25
            c = dict(op=op, rows=_log(rng, 1, 8192), vocab=_log(rng, 100, 64000), d=64 * rng.randint(1, 16), train=rng.random() < 0.7,
                     scale=20.0 if contrast else 1.0, ignored=rng.choice([0.0, 0.1]))
        elif op == "ckpt":
            c = dict(op=op, tokens=_log(rng, 1, 139264), d=16 * rng.randint(1, 128), relu=rng.random() < 0.5)
        elif op == "dw":
            c = dict(op=op, tokens=_log(rng, 1, 139264), d_out=8 * rng.randint(1, 288), d_in=16 * rng.randint(1, 128), relu=rng.random() < 0.5)
        else:
            c = dict(op=op, rows=_log(rng, 1, 139264), d=_log(rng, 8, 8192), dtype=rng.choice(["bf16", "bf16", "f32"]), train=rng.random() < 0.6,
                     residual=rng.random() < 0.5)
        if _cost(c) <= top[op]:
            return c


def work(case):
    if case["op"] == "lm":
        r, v, d = case["rows"], case["vocab"], case["d"]
        # logits once; with gradients the two products with the logits' gradient too
        one = 2 * r * v * d
        return {"bytes": (r + v) * d * 2 * (2 if case["train"] else 1) + r * 16, "flops": one * (3 if case["train"] else 1)}
    if case["op"] == "ckpt":
        n, blocks = case["tokens"] * case["d"], -(-case["tokens"] // 32) * case["d"]
        # the activation in, its codes and scales out and in again, the values out
        return {"bytes": n * (2 + 1 + 1 + 2) + 2 * blocks, "flops": 4 * n}
    if case["op"] == "dw":
        t, o, i = case["tokens"], case["d_out"], case["d_in"]
        return {"bytes": t * o * 2 + t * i + -(-t // 32) * i + o * i * 4, "flops": 2 * t * o * i}
    n, size = case["rows"] * case["d"], 2 if case["dtype"] == "bf16" else 4
    streams = 2 + (2 if case["residual"] else 0)           # x (and the residual and the sum), y
    if case["train"]:
        streams += 3 + (1 if case["residual"] else 0)      # dy, x, dx (and the residual stream's gradient)
    return {"bytes": n * size * streams + case["d"] * (2 * size + (8 if case["train"] else 0)), "flops": n * (20 if case["train"] else 8)}


def _cost(case):
    w = work(case)
    return w["flops"] if case["op"] in ("lm", "dw") else w["bytes"]


# ------------------------------------------------------------------------------------------------------------ inputs
def _rand(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFF)


def prepare(case, seed):
    g = _rand(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def uniform(*shape):
        return torch.rand(*shape, generator=g, device="cuda")

    if case["op"] == "lm":
        r, v, d = case["rows"], case["vocab"], case["d"]
        labels = torch.randint(0, v, (r,), generator=g, device="cuda")
        if case["scale"] != 1.0:      # unit vectors, a query near its own document
            w = torch.nn.functional.normalize(normal(v, d), dim=1)
            h = torch.nn.functional.normalize(w[labels] + 1.5 * torch.nn.functional.normalize(normal(r, d), dim=1), dim=1)
        else:                         # a normalised state against embeddings of unit variance: logits of deviation 3
            w = normal(v, d)
            h = 3.0 * d ** -0.5 * normal(r, d)
        if case["ignored"]:
            labels = torch.where(uniform(r) < case["ignored"], torch.full_like(labels, IGNORE), labels)
        weights = (0.5 + uniform(r)) / r      # what the loss rows are weighted with
        return dict(case=case, h=h.to(BF16), w=w.to(BF16), labels=labels, weights=weights)

    if case["op"] in ("ckpt", "dw"):
        t, d = case["tokens"], case["d" if case["op"] == "ckpt" else "d_in"]
        x = normal(t, d) * torch.exp(0.7 * normal(d))       # features of different size
        if case["relu"]:
            x = torch.relu(x) * (uniform(t, d) >= 0.1) / 0.9
        x = x.to(BF16)
        if case["op"] == "ckpt":
            return dict(case=case, x=x)
        values, scales = _quantised(x)
        codes = (values / scales.repeat_interleave(32, 0)[:t]).to(torch.float8_e4m3fn).view(torch.uint8)
        exponents = (torch.frexp(scales)[1] - 1 + 127).to(torch.uint8)
        dy = (normal(t, case["d_out"]) * 0.02).to(BF16)
        return dict(case=case, codes=codes, scales=exponents, dy=dy)

    r, d, dtype = case["rows"], case["d"], TYPES[case["dtype"]]
    spread = torch.exp(0.5 * normal(d))
    state = dict(case=case, x=(normal(r, d) * spread + 0.3 * normal(r, 1)).to(dtype), w=(1 + 0.2 * normal(d)).to(dtype), b=(0.1 * normal(d)).to(dtype))
    if case["residual"]:
        state["res"] = (normal(r, d) * spread).to(dtype)
    if case["train"]:
        state["dy"] = (0.05 * normal(r, d)).to(dtype)
        if case["residual"]:
            state["dres"] = (0.05 * normal(r, d)).to(dtype)
    return state


# ------------------------------------------------------------------------------------------------------- plain forms
def _power(e):
    """2^e in 32 bits, of whole numbers e from -126 to 127: exactly."""
    return ((e.int() + 127) << 23).view(F32)


def _quantised(x):
    """(values, scales) in 32 bits: of 32 tokens of a feature the scale is the smallest power of two (2^-117 at least) that
    brings the largest magnitude to 448 or less; e4m3 values, ties to even."""
    t, d = x.shape
    blocks = -(-t // 32)
    v = torch.zeros(blocks * 32, d, dtype=F32, device=x.device)
    v[:t] = x.float()
    v = v.view(blocks, 32, d)
    top = v.abs().amax(1)
    m, e = torch.frexp(top)                                  # top = m 2^e, m in [0.5, 1)
    e = torch.where(m > 0.875, e - 8, e - 9)                 # 448 = 0.875 * 2^9
    e = torch.where(top == 0, torch.full_like(e, -117), e).clamp_min(-117)
    scale = _power(e)
    u = v / scale.unsqueeze(1)
    u = torch.where((e == 120).unsqueeze(1), u.clamp(-240.0, 240.0), u)      # 256 * 2^120 would be infinite
    step = _power(torch.frexp(u)[1].clamp_min(-5) - 4)    # three bits behind the leading one, 2^-9 at least
    u = torch.round(u / step) * step
    return (u * scale.unsqueeze(1)).view(blocks * 32, d)[:t], scale


def _plain_lm(s):
    c = s["case"]
    h, w, labels = s["h"].float(), s["w"].float(), s["labels"]
    z = c["scale"] * (h @ w.t())
    kept = (labels != IGNORE).unsqueeze(1)
    at = labels.clamp_min(0).unsqueeze(1)
    # the entries beside the target's summed by themselves: a confident row's small loss keeps its digits
    t = z.gather(1, at)
    others = z.scatter(1, at, torch.where(kept, torch.full_like(t, float("-inf")), t))
    m = others.amax(1, keepdim=True)
    rest = torch.exp(others - m).sum(1, keepdim=True)
    loss = torch.where(t >= m, torch.log1p(rest * torch.exp(m - t)), (m - t) + torch.log(rest + torch.exp(t - m)))
    lse = torch.where(kept, t + loss, m + torch.log(rest))
    loss = torch.where(kept, loss, torch.zeros_like(loss))
    out = {"loss": loss.squeeze(1), "lse": lse.squeeze(1)}
    if c["train"]:
        g = torch.where(kept, s["weights"].unsqueeze(1), torch.zeros_like(loss))
        p = torch.exp(others - lse) * g
        p.scatter_add_(1, at, g * torch.expm1(-loss))
        out["dh"] = (c["scale"] * (p @ w)).to(BF16)
        out["dw"] = (c["scale"] * (p.t() @ h)).to(BF16)
    return out


def _plain_ln(s):
    c, dtype = s["case"], s["x"].dtype
    x = s["x"].float()
    out = {}
    if c["residual"]:
        out["xsum"] = (x + s["res"].float()).to(dtype)
        x = out["xsum"].float()
    w = s["w"].float()
    mean = x.mean(1, keepdim=True)
    xc = x - mean
    rstd = torch.rsqrt((xc * xc).mean(1, keepdim=True) + 1e-5)
    xh = xc * rstd
    out["y"] = (xh * w + s["b"].float()).to(dtype)
    if c["train"]:
        dy = s["dy"].float()
        g = dy * w
        dx = rstd * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
        if c["residual"]:
            dx = dx + s["dres"].float()
        out["dx"] = dx.to(dtype)
        out["dw"] = (dy * xh).sum(0, dtype=torch.float64).float()
        out["db"] = dy.sum(0, dtype=torch.float64).float()
    return out


def _plain(s):
    op = s["case"]["op"]
    if op == "lm":
        return _plain_lm(s)
    if op == "ckpt":
        values, scales = _quantised(s["x"])
        return {"values": values.to(BF16), "scales": scales}
    if op == "dw":
        t = s["codes"].shape[0]
        scales = _power(s["scales"].int() - 127)
        x = s["codes"].view(torch.float8_e4m3fn).float() * scales.repeat_interleave(32, 0)[:t]
        return {"dw": s["dy"].float().t() @ x}
    return _plain_ln(s)


# --------------------------------------------------------------------------------------------------------- framework
def _own_lm(s):
    K, c, h, w = _kernels(), s["case"], s["h"], s["w"]
    loss, lse = torch.empty(h.shape[0], device=h.device), torch.empty(h.shape[0], device=h.device)
    K.linear_ce_fwd(h, w, s["labels"], loss, lse, ignore_index=IGNORE, scale=c["scale"])
    out = {"loss": loss, "lse": lse}
    if c["train"]:
        out["dh"], out["dw"] = torch.empty_like(h), torch.empty_like(w)
        K.linear_ce_bwd(h, w, s["labels"], lse, s["weights"], out["dh"], out["dw"], ignore_index=IGNORE, scale=c["scale"])
    return out


def _own_ln(s):
    K, c, x = _kernels(), s["case"], s["x"]
    rows, d = x.shape
    out = {"y": torch.empty_like(x)}
    mean, rstd = (torch.empty(rows, device=x.device), torch.empty(rows, device=x.device)) if c["train"] else (None, None)
    if c["residual"]:
        out["xsum"] = torch.empty_like(x)
    K.layernorm_fwd(x, s["w"], s["b"], out["y"], mean, rstd, eps=1e-5, res=s.get("res"), xsum=out.get("xsum"))
    if c["train"]:
        out["dx"] = torch.empty_like(x)
        out["dw"], out["db"] = torch.zeros(d, device=x.device), torch.zeros(d, device=x.device)
        K.layernorm_bwd(s["dy"], out.get("xsum", x), s["w"], mean, rstd, out["dx"], dres=s.get("dres"), dw=out["dw"], db=out["db"])
    return out


def _own(s):
    K, op = _kernels(), s["case"]["op"]
    if op == "lm":
        return _own_lm(s)
    if op == "ckpt":
        x = s["x"]
        codes, scales = K.act8_quantize(x)
        values = torch.empty_like(x)
        K.act8_dequantize(codes, scales, values)
        return {"values": values, "scales": _power(scales.int() - 127)}
    if op == "dw":
        dw = torch.empty(s["dy"].shape[1], s["codes"].shape[1], device=s["dy"].device)
        K.act8_dweight(s["dy"], s["codes"], s["scales"], dw, accumulate=False)
        return {"dw": dw}
    return _own_ln(s)


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    f64 = torch.float64
    if case["op"] == "lm":
        h, w = s["h"].to(f64), s["w"].to(f64)
        keep = (s["labels"] >= 0).nonzero().squeeze(1)
        loss, lse = torch.zeros(h.shape[0], dtype=f64, device="cuda"), torch.empty(h.shape[0], dtype=f64, device="cuda")
        dh, dw = torch.zeros_like(h), torch.zeros_like(w)
        for rows in torch.arange(h.shape[0], device="cuda").split(2048):
            z = torch.mm(h[rows] * case["scale"], w.T)
            lse[rows] = torch.logsumexp(z, 1)
            mine = rows[torch.isin(rows, keep)]
            local, target = mine - rows[0], s["labels"][mine]
            loss[mine] = lse[mine] - z[local, target]
            if case["train"]:
                grad = torch.zeros_like(z)
                grad[local] = torch.softmax(z[local], 1)
                grad[local, target] -= 1.0
                grad[local] *= s["weights"][mine].to(f64).unsqueeze(1) * case["scale"]
                dh[rows] = grad @ w
                dw += grad.T @ h[rows]
        return {"loss": loss, "lse": lse, **({"dh": dh, "dw": dw} if case["train"] else {})}

    if case["op"] == "ckpt":
        # by search in the table of all magnitudes that the format has
        code = torch.arange(127, device="cuda")
        table = torch.where(code < 8, code.to(f64) / 512, (8 + code % 8).to(f64) * ((code // 8 - 10 + 1023) << 52).view(f64))
        x = s["x"].to(f64)
        out, scales = torch.empty_like(x), []
        for i in range(0, x.shape[0], 32 * 256):
            part = x[i:i + 32 * 256]
            rows = torch.arange(part.shape[0], device="cuda") // 32
            top = torch.zeros(int(rows[-1]) + 1, x.shape[1], dtype=f64, device="cuda").index_reduce_(0, rows, part.abs(), "amax")
            powers = (torch.arange(-117 + 1023, 121 + 1023, device="cuda") << 52).view(f64)
            pick = torch.searchsorted(448.0 * powers, top)            # the first whose reach is enough
            scale = powers[pick]
            a = part.abs() / scale[rows]
            hi = torch.searchsorted(table, a).clamp_(1, 126)
            lo = hi - 1
            below, above = a - table[lo], table[hi] - a
            near = torch.where((below < above) | ((below == above) & (lo % 2 == 0)), lo, hi)
            near = torch.where(pick[rows] == 237, near.clamp_max(119), near)      # 240 is code 119
            out[i:i + 32 * 256] = torch.copysign(table[near] * scale[rows], part)
            scales.append(scale)
        return {"values": out, "scales": torch.cat(scales)}

    if case["op"] == "dw":
        c = s["codes"].to(torch.int64)
        low, high = c & 7, (c >> 3) & 15
        a = torch.where(high == 0, low.to(f64) / 512, (8 + low).to(f64) * torch.exp2(high.to(f64) - 10))
        a = torch.where(c >= 128, -a, a)
        dw = torch.zeros(s["dy"].shape[1], c.shape[1], dtype=f64, device="cuda")
        for i in range(0, c.shape[0], 32 * 512):
            part = a[i:i + 32 * 512]
            f = torch.exp2(s["scales"][i // 32:i // 32 + 512].to(f64) - 127)
            part = part * f[torch.arange(part.shape[0], device="cuda") // 32]
            dw += s["dy"][i:i + 32 * 512].to(f64).T @ part
        return {"dw": dw}

    x, n = s["x"].to(f64), float(case["d"])
    out = {}
    if case["residual"]:
        out["xsum"] = x + s["res"].to(f64)
        x = out["xsum"].to(s["x"].dtype).to(f64)       # what is normalised is the sum as it is stored
    mean = x.sum(1) / n
    var = ((x - mean[:, None]) ** 2).sum(1) / n
    sd = torch.sqrt(var + 1e-5)
    xh = (x - mean[:, None]) / sd[:, None]
    out["y"] = xh * s["w"].to(f64) + s["b"].to(f64)
    if case["train"]:
        dy = s["dy"].to(f64)
        out["db"], out["dw"] = torch.ones(dy.shape[0], dtype=f64, device="cuda") @ dy, (dy * xh).sum(0)
        g = dy * s["w"].to(f64)
        dx = (g - (g.sum(1) / n)[:, None] - xh * ((g * xh).sum(1) / n)[:, None]) / sd[:, None]
        out["dx"] = dx + s["dres"].to(f64) if case["residual"] else dx
    return out
