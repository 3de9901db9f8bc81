"""What surrounds the optimizer step in a training program: layer norm, the products of a mixture of experts
and the clip of the gradients by their global norm, for timing and comparison.

A case is one call: a direction of layer norm, one of the three products of an expert layer (its output, the
gradient of its rows, the gradient of its weights) or one clip of a model's gradients.  With ``own`` the calls
go to this package; without it they are written out in elementary torch operations in 32 bits.
"""

import math

import torch

own = False

EPS = 1e-5
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32, "fp16": torch.float16}
ALIGN = 256                # bytes: every tensor of a flat buffer starts on such a boundary
MOST_ELEMENTS = 2 ** 26    # of a layer norm's input: the largest listed one
MOST_FLOPS = 2 * 16384 * 4096 * 14336
MOST_WEIGHTS = 8 * 4096 * 14336
MOST_GRADS = 4 * (2 * 4096 * 4096 + 2 * 1024 * 4096 + 3 * 14336 * 4096)


def _norm(way, rows, width, dtype, weights, bias=True):
    return dict(op="norm", way=way, rows=rows, width=width, dtype=dtype, weights=weights, bias=bias)


def _experts(way, experts, rows, inner, outer, dtype, spread=0.5, spare=0, grad="", shapes=0):
    """inner, outer: the widths of a layer's input and output rows.  spread: how unevenly the rows fall on the
    experts; spare: rows at the end that belong to none; grad: the type of the weights' gradient."""
    return dict(op="experts", way=way, experts=experts, rows=rows, inner=inner, outer=outer, dtype=dtype,
                spread=spread, spare=spare, grad=grad or dtype, shapes=shapes)


def _clip(model, dtype, out, active, order=2.0, **kw):
    """out: the type of the clipped copies, or "" to clip in place; active: whether the norm exceeds the bound."""
    c = dict(op="clip", model=model, dtype=dtype, out=out, active=active, order=order, layers=0, width=0, kv=0,
             ffn=0, vocab=0, context=0, count=0, shapes=0)
    c.update(kw)
    return c


def listed():
    return [
        # one decode step of GPT-2-small at batch 8: latency
        dict(_norm("forward", 8, 768, "bf16", "bf16"), name="norm_tokens"),
        # a batch of 16 sequences of 1024 through a block of Llama-3-8B's width
        dict(_norm("forward", 16384, 4096, "bf16", "bf16"), name="norm_forward"),
        # GPT-2-small's training batch, weights kept in fp32
        dict(_norm("backward", 16384, 768, "bf16", "fp32"), name="norm_backward"),
        # an fp32 model of odd width and an odd number of rows
        dict(_norm("backward", 4097, 1021, "fp32", "fp32"), name="norm_backward_odd"),
        # tokens of one decode step over many experts: the weights' bytes bound it
        dict(_experts("forward", 64, 48, 2048, 1024, "bf16", spread=1.0), name="experts_tokens"),
        # narrow experts in fp16, widths that are no multiple of 8
        dict(_experts("forward", 8, 4096, 500, 386, "fp16"), name="experts_odd"),
        # the up projection of eight experts of Llama-3-8B's block sizes
        dict(_experts("forward", 8, 16384, 4096, 14336, "bf16"), name="experts_forward"),
        # the rows' gradient of many unevenly used experts in a buffer with unused rows
        dict(_experts("rows_grad", 32, 8192, 4096, 2048, "bf16", spread=1.5, spare=320), name="experts_rows_grad"),
        # the weights' gradient, accumulated in fp32 as programs that clip in fp32 keep it
        dict(_experts("weight_grad", 16, 16384, 2048, 4096, "bf16", grad="fp32"), name="experts_weight_grad"),
        # a small MLP in fp32, its norm under the bound: launches and host time count
        dict(_clip("mlp", "fp32", "", False, layers=3, width=256, ffn=100), name="clip_mlp"),
        # 2,000 ragged bf16 tensors, the clipped copies in another buffer
        dict(_clip("ragged", "bf16", "bf16", True, count=2000, shapes=2), name="clip_ragged"),
        # fp32 accumulated grads of four Llama-3-8B layers, clipped into the parameters' type
        dict(_clip("llama", "fp32", "bf16", True, layers=4, width=4096, kv=1024, ffn=14336), name="clip_layers"),
    ]


def draw(rng):
    def logint(lo, hi, step=1):
        return max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))) // step * step)

    op = rng.choice(["norm", "experts", "experts", "clip"])
    if op == "norm":
        width = logint(16, 16384, rng.choice([1, 8, 64]))
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        return _norm(rng.choice(["forward", "backward"]), logint(1, min(65536, MOST_ELEMENTS // width)), width, dtype,
                     rng.choice([dtype, "fp32"]), rng.random() < 0.7)
    if op == "experts":
        step = rng.choice([1, 8, 8, 64, 128])
        inner, outer = logint(64, 8192, step), logint(64, 14336, step)
        experts = logint(1, max(1, min(128, MOST_WEIGHTS // (inner * outer))))
        rows = logint(1, min(65536, MOST_FLOPS // (2 * inner * outer), MOST_ELEMENTS * 4 // max(inner, outer)))
        way = rng.choice(["forward", "rows_grad", "weight_grad"])
        dtype = rng.choice(["bf16", "bf16", "fp16"])
        return _experts(way, experts, rows, inner, outer, dtype, spread=rng.choice([0.0, 0.5, 1.0, 2.0]),
                        spare=rng.choice([0, 0, logint(1, 512)]),
                        grad="fp32" if way == "weight_grad" and rng.random() < 0.5 else "", shapes=rng.randint(1, 999))
    dtype = rng.choice(["bf16", "fp32", "fp32", "fp16"])
    active = rng.random() < 0.7
    kw = dict(out=rng.choice([dtype, "bf16"]) if active else "", active=active,
              order=rng.choice([2.0, 2.0, 2.0, 1.0, math.inf]))
    model = rng.choice(["mlp", "gpt", "ragged", "llama"])
    if model == "mlp":
        return _clip("mlp", dtype, layers=rng.randint(2, 6), width=logint(24, 2000), ffn=logint(10, 1000), **kw)
    if model == "gpt":
        w = logint(96, 1280, 32)
        return _clip("gpt", dtype, layers=rng.randint(1, 12), width=w, ffn=4 * w, vocab=logint(1000, 50257),
                     context=logint(64, 2048), **kw)
    if model == "ragged":
        return _clip("ragged", dtype, count=logint(100, 4000), shapes=rng.randint(3, 999), **kw)
    w = logint(256, 4096, 64)
    f = logint(2 * w, int(3.5 * w), 8)
    kv = max(w // rng.choice([1, 4, 8]), 32)
    layer = 2 * w * w + 2 * kv * w + 3 * f * w
    return _clip("llama", dtype, layers=rng.randint(1, max(1, min(16, MOST_GRADS // layer))), width=w, kv=kv, ffn=f, **kw)


# ---------------------------------------------------------------------------- shapes
def _shapes(c):
    """The shapes of a clip's gradients, in the order that a model lists its parameters."""
    w, f = c["width"], c["ffn"]
    if c["model"] == "mlp":
        s = [(w, f), (w,)]
        for _ in range(c["layers"] - 2):
            s += [(w, w), (w,)]
        return s + [(10, w), (10,)]
    if c["model"] == "gpt":
        s = [(c["vocab"], w), (c["context"], w)]
        for _ in range(c["layers"]):
            s += [(w,), (w,), (w, 3 * w), (3 * w,), (w, w), (w,), (w,), (w,), (w, f), (f,), (f, w), (w,)]
        return s
    if c["model"] == "llama":
        return [(w, w), (c["kv"], w), (c["kv"], w), (w, w), (f, w), (f, w), (w, f), (w,), (w,)] * c["layers"]
    # ragged: element counts log-uniform in [64, 2^20]
    g = torch.Generator().manual_seed(c["shapes"])
    n = torch.exp(torch.rand(c["count"], generator=g, dtype=torch.float64) * math.log(2 ** 14) + math.log(64))
    return [(k,) for k in n.floor().long().tolist()]


def _offsets(sizes, itemsize):
    """Element offsets of tensors of these sizes in one flat buffer, and its length."""
    unit = ALIGN // itemsize
    at, out = 0, []
    for n in sizes:
        out.append(at)
        at += (n + unit - 1) // unit * unit
    return out, at


def _sizes(c):
    """Rows of each expert: multinomial with weights exp(spread x normal), so that some get none."""
    g = torch.Generator().manual_seed(1000 * c["shapes"] + c["experts"])
    p = torch.exp(c["spread"] * torch.randn(c["experts"], generator=g, dtype=torch.float64))
    picks = torch.multinomial(p, c["rows"], replacement=True, generator=g)
    return torch.bincount(picks, minlength=c["experts"]).tolist()


# ---------------------------------------------------------------------------- inputs
def prepare(case, seed):
    device = torch.device("cuda", 0)
    gen = torch.Generator(device=device).manual_seed(seed)

    def normal(shape, dtype, std=1.0, mean=0.0):
        return torch.empty(shape, dtype=dtype, device=device).normal_(mean, std, generator=gen)

    dt = DTYPES[case["dtype"]]
    if case["op"] == "norm":
        # rows of a residual stream: a mean and a scale of their own, weights near one
        rows, width, wdt = case["rows"], case["width"], DTYPES[case["weights"]]
        scale = normal((rows, 1), torch.float32).exp_()
        x = (normal((rows, width), torch.float32) + 0.5 * normal((rows, 1), torch.float32)).mul_(scale).to(dt)
        s = {"case": case, "x": x, "w": normal((width,), wdt, 0.2, 1.0),
             "b": normal((width,), wdt, 0.2) if case["bias"] else None}
        if case["way"] == "backward":
            # what the forward pass kept
            var, mean = torch.var_mean(x.double(), dim=1, correction=0)
            s.update(mean=mean.float(), rstd=(var + EPS).rsqrt().float(), dy=normal((rows, width), dt))
        return s
    if case["op"] == "experts":
        sizes = _sizes(case)
        total = case["rows"] + case["spare"]
        s = {"case": case, "sizes": sizes, "ends": torch.tensor(sizes).cumsum(0).to(torch.int32).to(device)}
        if case["way"] != "rows_grad":
            s["x"] = normal((total, case["inner"]), dt)
        if case["way"] != "forward":
            s["dy"] = normal((total, case["outer"]), dt)
        if case["way"] != "weight_grad":
            s["w"] = normal((case["experts"], case["outer"], case["inner"]), dt, case["inner"] ** -0.5)
        return s
    # gradients ~N(0, 1e-3) with a scale per tensor log-uniform in [0.1, 10], one in twenty all zero in the
    # ragged list, as views of a flat buffer; clipped copies in another one
    shapes = _shapes(case)
    n = [math.prod(q) for q in shapes]
    at, total = _offsets(n, dt.itemsize)
    host = torch.Generator().manual_seed(seed)
    flat = normal((total,), dt, 1e-3)
    scale = torch.exp((torch.rand(len(n), generator=host, dtype=torch.float64) * 2 - 1) * math.log(10.0))
    if case["model"] == "ragged":
        scale[torch.rand(len(n), generator=host) < 0.05] = 0.0
    rows = [flat[o:o + k] for k, o in zip(n, at)]
    torch._foreach_mul_(rows, scale.tolist())
    ends = [o + k for k, o in zip(n, at)]
    for a, b in zip(ends, at[1:] + [total]):
        if a < b:
            flat[a:b].zero_()
    s = {"case": case, "n": n, "flat": flat, "rows": rows, "grads": [r.view(q) for r, q in zip(rows, shapes)],
         "bound": _bound(case, rows), "out": None, "to": rows}
    if case["out"]:
        odt = DTYPES[case["out"]]
        oat, ototal = _offsets(n, odt.itemsize)
        s["flat"] = torch.zeros(ototal, dtype=odt, device=device)
        s["to"] = [s["flat"][o:o + k] for k, o in zip(n, oat)]
        s["out"] = [t.view(q) for t, q in zip(s["to"], shapes)]
    return s


def _bound(case, rows):
    """The norm that the gradients are clipped to: a fraction of what they have, or well over it."""
    order = case["order"]
    norms = torch.stack([n.double() for n in torch._foreach_norm(rows, order, dtype=torch.float32)])
    return float(torch.linalg.vector_norm(norms, order)) * (0.3 if case["active"] else 4.0)


# ---------------------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    if own:
        return _OWN[case["op"], case.get("way", "")](state)
    return _PLAIN[case["op"], case.get("way", "")](state)


def _own_norm_forward(s):
    import apexw_amd
    y, mean, rstd = apexw_amd.layer_norm_forward(s["x"], s["w"], s["b"], EPS)
    return {"y": y, "mean": mean, "rstd": rstd}


def _own_norm_backward(s):
    import apexw_amd
    dx, dw, db = apexw_amd.layer_norm_backward(s["dy"], s["x"], s["mean"], s["rstd"], s["w"], s["b"])
    return {"dx": dx, "dw": dw} if db is None else {"dx": dx, "dw": dw, "db": db}


def _own_experts_forward(s):
    import apexw_amd
    return apexw_amd.expert_matmul_forward(s["x"], s["w"], s["ends"])


def _own_experts_rows_grad(s):
    import apexw_amd
    return apexw_amd.expert_matmul_rows_grad(s["dy"], s["w"], s["ends"])


def _own_experts_weight_grad(s):
    import apexw_amd
    return apexw_amd.expert_matmul_weight_grad(s["dy"], s["x"], s["ends"], dtype=DTYPES[s["case"]["grad"]])


def _own_clip(s):
    import apexw_amd
    norm = apexw_amd.clip_grads(s["grads"], s["bound"], norm_type=s["case"]["order"], out=s["out"])
    return {"norm": norm, "grads": s["flat"]}


def _plain_norm_forward(s):
    x = s["x"].float()
    mean = x.mean(1)
    x = x - mean[:, None]
    rstd = (x.square().mean(1) + EPS).rsqrt()
    y = x * rstd[:, None] * s["w"].float()
    if s["b"] is not None:
        y = y + s["b"].float()
    return {"y": y.to(s["x"].dtype), "mean": mean, "rstd": rstd}


def _plain_norm_backward(s):
    dy, rstd = s["dy"].float(), s["rstd"][:, None]
    xh = (s["x"].float() - s["mean"][:, None]) * rstd
    g = dy * s["w"].float()
    dx = (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True)) * rstd
    out = {"dx": dx.to(s["x"].dtype), "dw": (dy * xh).sum(0).to(s["w"].dtype)}
    if s["b"] is not None:
        out["db"] = dy.sum(0).to(s["b"].dtype)
    return out


def _parts(t, s):
    """The rows of each expert in 32 bits, and the number of rows that belong to none."""
    return t[:s["case"]["rows"]].float().split(s["sizes"]), s["case"]["spare"]


def _plain_experts_forward(s):
    parts, spare = _parts(s["x"], s)
    y = torch.cat(list(map(torch.mm, parts, s["w"].float().transpose(1, 2)))).to(s["x"].dtype)
    return torch.cat([y, y.new_zeros(spare, y.shape[1])]) if spare else y


def _plain_experts_rows_grad(s):
    parts, spare = _parts(s["dy"], s)
    dx = torch.cat(list(map(torch.mm, parts, s["w"].float()))).to(s["dy"].dtype)
    return torch.cat([dx, dx.new_zeros(spare, dx.shape[1])]) if spare else dx


def _plain_experts_weight_grad(s):
    dy, x = _parts(s["dy"], s)[0], _parts(s["x"], s)[0]
    return torch.stack(list(map(torch.mm, map(torch.t, dy), x))).to(DTYPES[s["case"]["grad"]])


def _plain_clip(s):
    order = s["case"]["order"]
    rows = list(torch.empty(sum(s["n"]), dtype=torch.float32, device=s["flat"].device).split(s["n"]))
    torch._foreach_copy_(rows, s["rows"])
    norms = torch.stack(torch._foreach_norm(rows, order))
    norm = norms.max() if order == math.inf else norms.sum() if order == 1.0 else norms.square().sum().sqrt()
    torch._foreach_mul_(rows, (s["bound"] / (norm + 1e-6)).clamp(max=1.0))
    torch._foreach_copy_(s["to"], rows)
    return {"norm": norm, "grads": s["flat"]}


_OWN = {("norm", "forward"): _own_norm_forward, ("norm", "backward"): _own_norm_backward,
        ("experts", "forward"): _own_experts_forward, ("experts", "rows_grad"): _own_experts_rows_grad,
        ("experts", "weight_grad"): _own_experts_weight_grad, ("clip", ""): _own_clip}
_PLAIN = {("norm", "forward"): _plain_norm_forward, ("norm", "backward"): _plain_norm_backward,
          ("experts", "forward"): _plain_experts_forward, ("experts", "rows_grad"): _plain_experts_rows_grad,
          ("experts", "weight_grad"): _plain_experts_weight_grad, ("clip", ""): _plain_clip}


# ---------------------------------------------------------------------------- what a pass needs
def work(case):
    """Bytes: each input read once, each output written once, the weights of experts with rows only.  FLOPs: the
    multiplications and additions of the formulas."""
    size = DTYPES[case["dtype"]].itemsize
    if case["op"] == "norm":
        n, w = case["rows"] * case["width"], case["width"] * DTYPES[case["weights"]].itemsize
        if case["way"] == "forward":
            return {"bytes": 2 * n * size + 8 * case["rows"] + w * (1 + case["bias"]), "flops": 8 * n}
        return {"bytes": 3 * n * size + 8 * case["rows"] + w * (2 + case["bias"]), "flops": 14 * n}
    if case["op"] == "experts":
        rows, used = case["rows"], sum(k > 0 for k in _sizes(case))
        weights = case["inner"] * case["outer"]
        flops = 2 * rows * weights
        if case["way"] == "weight_grad":
            return {"bytes": rows * (case["inner"] + case["outer"]) * size
                    + case["experts"] * weights * DTYPES[case["grad"]].itemsize, "flops": flops}
        spare = case["spare"] * (case["outer"] if case["way"] == "forward" else case["inner"])
        return {"bytes": (rows * (case["inner"] + case["outer"]) + spare + used * weights) * size, "flops": flops}
    n = sum(math.prod(q) for q in _shapes(case))
    return {"bytes": n * (size + (DTYPES[case["out"]].itemsize if case["out"] else 0)), "flops": 3 * n}


# ---------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        x, w = s["x"].double(), s["w"].double()
        if case["way"] == "forward":
            var, mean = torch.var_mean(x, dim=1, correction=0)
            rstd = 1.0 / torch.sqrt(var + EPS)
            y = torch.addcmul(s["b"].double() if case["bias"] else torch.zeros_like(w), (x - mean[:, None]) * rstd[:, None], w)
            return {"y": y, "mean": mean, "rstd": rstd}
        dy, n = s["dy"].double(), case["width"]
        xh = (x - s["mean"].double()[:, None]) * s["rstd"].double()[:, None]
        g = dy * w
        dx = (n * g - g.sum(1, keepdim=True) - xh * (g * xh).sum(1, keepdim=True)) * (s["rstd"].double() / n)[:, None]
        out = {"dx": dx, "dw": torch.sum(dy * xh, 0)}
        if case["bias"]:
            out["db"] = torch.sum(dy, 0)
        return out
    if case["op"] == "experts":
        if 2 * case["rows"] * case["inner"] * case["outer"] > MOST_FLOPS:
            return None
        if case["way"] == "weight_grad":
            out = torch.zeros(case["experts"], case["outer"], case["inner"], dtype=torch.float64, device=s["dy"].device)
        else:
            out = torch.zeros(case["rows"] + case["spare"], case["outer" if case["way"] == "forward" else "inner"],
                              dtype=torch.float64, device=s["w"].device)
        a = 0
        for e, k in enumerate(s["sizes"]):
            b = a + k
            if k and case["way"] == "forward":
                out[a:b] = s["x"][a:b].double() @ s["w"][e].double().t()
            elif k and case["way"] == "rows_grad":
                out[a:b] = s["dy"][a:b].double() @ s["w"][e].double()
            elif k:
                out[e] = s["dy"][a:b].double().t() @ s["x"][a:b].double()
            a = b
        return out
    rows = [r.double() for r in s["rows"]]
    norms = torch.stack([torch.linalg.vector_norm(r, case["order"]) for r in rows])
    norm = torch.linalg.vector_norm(norms, case["order"])
    coef = min(s["bound"] / (float(norm) + 1e-6), 1.0)
    flat = torch.zeros(s["flat"].numel(), dtype=torch.float64, device=norm.device)
    for r, o in zip(rows, _offsets(s["n"], s["flat"].element_size())[0]):
        flat[o:o + r.numel()] = r * coef
    return {"norm": norm, "grads": flat}
