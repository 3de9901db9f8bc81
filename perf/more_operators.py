"""The two ends of a language model and the way between its experts, for timing and comparison: the embedding, the
tokens sorted by expert and back, and the cross entropy of the head over a large vocabulary.

A case is one call, or the two calls that belong together (the order of the tokens and their rows in it).  With
``own`` the calls go to this package; without it they are written out in elementary torch operations in 32 bits.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32, "fp16": torch.float16}
IGNORED = -100             # a target that counts for nothing
MOST_FLOPS = 2 * 8192 * 4096 * 128256
MOST_WEIGHTS = 4096 * 128256
MOST_ROWS = 65536 * 4096   # elements of the rows that a pass moves


def _head(way, rows, width, vocab, dtype, ignored=0.0):
    """ignored: the share of rows without a target (prompts, padding)."""
    return dict(op="head", way=way, rows=rows, width=width, vocab=vocab, dtype=dtype, ignored=ignored)


def _experts(way, tokens, k, experts, width, dtype, weights="fp32", spread=0.5, dropped=0.0):
    """spread: how unevenly the tokens choose; dropped: the share of choices that no expert takes."""
    return dict(op="experts", way=way, tokens=tokens, k=k, experts=experts, width=width, dtype=dtype, weights=weights,
                spread=spread, dropped=dropped)


def _embedding(way, tokens, width, vocab, dtype, scale=1.0, padded=0.0, grad=""):
    """padded: the share of tokens that are the padding's, the vocabulary's last; grad: the gradient's type."""
    return dict(op="embedding", way=way, tokens=tokens, width=width, vocab=vocab, dtype=dtype, scale=scale,
                padded=padded, grad=grad or dtype)


def listed():
    return [
        # the last tokens of 8 sequences scored against GPT-2-small's vocabulary: latency, the weights' bytes
        dict(_head("forward", 8, 768, 50257, "bf16"), name="head_tokens"),
        # 8 sequences of 1024 through Llama-3-8B's head
        dict(_head("forward", 8192, 4096, 128256, "bf16"), name="head_forward"),
        # GPT-2-small's training batch, a fifth of it prompts without a target
        dict(_head("backward", 16384, 768, 50257, "bf16", ignored=0.2), name="head_backward"),
        # a small fp16 model of odd sizes, half of the batch masked
        dict(_head("backward", 1001, 500, 10007, "fp16", ignored=0.5), name="head_backward_odd"),
        # one decode step of 16 sequences, two of 64 experts each: launches and host time count
        dict(_experts("dispatch", 16, 2, 64, 2048, "bf16"), name="dispatch_tokens"),
        # a training batch of Llama-3-8B's width on its way to two of eight experts
        dict(_experts("dispatch", 16384, 2, 8, 4096, "bf16"), name="dispatch_forward"),
        # the way back from eight of many narrow experts
        dict(_experts("combine", 8192, 8, 128, 2048, "bf16", spread=1.0), name="combine_forward"),
        # gradients of rows and weights in an fp32 model of odd width, choices over the experts' capacity dropped
        dict(_experts("combine_grad", 4097, 3, 17, 1021, "fp32", spread=1.0, dropped=0.05), name="combine_grad_odd"),
        # the tokens of one decode step
        dict(_embedding("forward", 8, 768, 50257, "bf16"), name="embedding_tokens"),
        # a training batch of Llama-3-8B's width, scaled by the root of the width
        dict(_embedding("forward", 16384, 4096, 128256, "bf16", scale=64.0), name="embedding_forward"),
        # GPT-2-small's training batch
        dict(_embedding("grad", 16384, 768, 50257, "bf16"), name="embedding_grad"),
        # a large padded batch of Llama-3-8B's width: one row of the gradient sums a tenth of the tokens
        dict(_embedding("grad", 65536, 4096, 128256, "bf16", scale=64.0, padded=0.1), name="embedding_grad_padded"),
    ]


def draw(rng):
    def logint(lo, hi, step=1):
        return max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))) // step * step)

    op = rng.choice(["head", "experts", "experts", "embedding"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    step = rng.choice([1, 8, 64, 64])
    if op == "head":
        way = rng.choice(["forward", "backward"])
        width = logint(64, 8192, rng.choice([8, 64, 64, 1]))
        vocab = logint(256, min(200000, MOST_WEIGHTS // width), step)
        most = MOST_FLOPS // ((2 if way == "forward" else 6) * width * vocab)
        return _head(way, logint(1, max(1, min(65536, most, MOST_ROWS // width))), width, vocab,
                     rng.choice(["bf16", "bf16", "fp16"]), ignored=rng.choice([0.0, 0.0, 0.2, 0.9]))
    if op == "experts":
        width, k = logint(32, 8192, step), rng.choice([1, 2, 2, 4, 6, 8])
        return _experts(rng.choice(["dispatch", "dispatch_grad", "combine", "combine_grad"]),
                        logint(1, min(65536, MOST_ROWS // (k * width))), k, logint(k, 256), width, dtype,
                        weights=rng.choice([dtype, "fp32"]), spread=rng.choice([0.0, 0.5, 1.0, 2.0]),
                        dropped=rng.choice([0.0, 0.0, 0.05, 0.5]))
    width = logint(32, 8192, step)
    vocab = logint(100, min(256000, MOST_WEIGHTS // width))
    return _embedding(rng.choice(["forward", "grad", "grad"]), logint(1, min(131072, MOST_ROWS // width)), width, vocab,
                      dtype, scale=rng.choice([1.0, width ** 0.5]), padded=rng.choice([0.0, 0.1, 0.6]),
                      grad=rng.choice([dtype, "fp32"]))


# ---------------------------------------------------------------------------- inputs
def prepare(case, seed):
    device = torch.device("cuda", 0)
    gen = torch.Generator(device=device).manual_seed(seed)

    def normal(shape, dtype, std=1.0):
        return torch.empty(shape, dtype=dtype, device=device).normal_(0.0, std, generator=gen)

    def uniform(shape):
        return torch.rand(shape, generator=gen, device=device)

    def words(n, vocab):
        # token ids of a vocabulary sorted by frequency: the logarithm of the rank evenly spread
        return torch.exp(uniform((n,)).double() * math.log(vocab + 1)).long().sub_(1).clamp_(0, vocab - 1)

    dt = DTYPES[case["dtype"]]
    s = {"case": case}
    if case["op"] == "head":
        # normed rows that lean towards their target's, so that probabilities run from near none to near one
        rows, width, vocab = case["rows"], case["width"], case["vocab"]
        target = words(rows, vocab)
        w = normal((vocab, width), dt, width ** -0.5)
        lean = uniform((rows, 1)) * 12.0
        x = (normal((rows, width), torch.float32) + lean * w[target].float()).to(dt)
        if case["ignored"]:
            target[uniform((rows,)) < case["ignored"]] = IGNORED
        s.update(x=x, w=w, target=target)
        if case["way"] == "backward":
            # what the forward pass kept, and the gradient of a mean over the rows that count; in fp16 of a loss
            # scaled by a power of two, as programs in fp16 keep their gradients out of the subnormal range
            kept = target != IGNORED
            count = max(int(kept.sum()), 1)
            scale = 2.0 ** round(math.log2(count)) if dt == torch.float16 else 1.0
            s["lse"] = torch.cat([torch.logsumexp(a.float() @ w.float().t(), 1) for a in x.split(4096)]) * kept
            s["dloss"] = torch.full((rows,), scale / count, device=device)
        return s
    if case["op"] == "experts":
        tokens, k, experts, width = case["tokens"], case["k"], case["experts"], case["width"]
        # k different experts a token, the likeliest of a router's noisy scores
        noise = -torch.log(-torch.log(uniform((tokens, experts)).clamp_(1e-7, 1 - 1e-7)))
        score, expert = torch.topk(case["spread"] * normal((experts,), torch.float32) + noise, k, dim=1)
        if case["dropped"]:
            expert = torch.where(uniform((tokens, k)) < case["dropped"], -1, expert)
        s["expert"] = expert.contiguous()
        if case["way"] == "dispatch":
            s["x"] = normal((tokens, width), dt)
            return s
        s["order"] = _plain_order(s["expert"], experts)
        rows = torch.where((s["order"][0] >= 0)[:, None], normal((tokens * k, width), torch.float32), 0.0).to(dt)
        if case["way"] == "dispatch_grad":
            s["drows"] = rows
            return s
        s.update(y=rows, w=torch.softmax(score, 1).to(DTYPES[case["weights"]]))
        if case["way"] == "combine_grad":
            s["dout"] = normal((tokens, width), dt)
        return s
    ids = words(case["tokens"], case["vocab"])
    if case["padded"]:
        ids[uniform((case["tokens"],)) < case["padded"]] = case["vocab"] - 1
    s["ids"] = ids
    if case["way"] == "forward":
        s["w"] = normal((case["vocab"], case["width"]), dt, 0.02)
    else:
        s["dy"] = normal((case["tokens"], case["width"]), dt)
    return s


# ---------------------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    return (_OWN if own else _PLAIN)[case["op"], case["way"]](state)


def _own_head_forward(s):
    import apexw_amd
    loss, lse = apexw_amd.linear_cross_entropy_forward(s["x"], s["w"], s["target"], ignore_index=IGNORED)
    return {"loss": loss, "lse": lse}


def _own_head_backward(s):
    import apexw_amd
    dx, dw = apexw_amd.linear_cross_entropy_backward(s["dloss"], s["x"], s["w"], s["target"], s["lse"],
                                                     ignore_index=IGNORED)
    return {"dx": dx, "dw": dw}


def _own_dispatch(s):
    import apexw_amd
    order = apexw_amd.expert_order(s["expert"], s["case"]["experts"])
    rows = apexw_amd.expert_dispatch_forward(s["x"], order)
    return {"rows": rows, "source": order.source, "place": order.place, "ends": order.ends}


def _own_dispatch_grad(s):
    import apexw_amd
    return apexw_amd.expert_dispatch_backward(s["drows"], apexw_amd.ExpertOrder(*s["order"]))


def _own_combine(s):
    import apexw_amd
    return apexw_amd.expert_combine_forward(s["y"], apexw_amd.ExpertOrder(*s["order"]), s["w"])


def _own_combine_grad(s):
    import apexw_amd
    dy, dw = apexw_amd.expert_combine_backward(s["dout"], s["y"], apexw_amd.ExpertOrder(*s["order"]), s["w"])
    return {"dy": dy, "dw": dw}


def _own_embedding(s):
    import apexw_amd
    return apexw_amd.embedding_forward(s["ids"], s["w"], s["case"]["scale"])


def _own_embedding_grad(s):
    import apexw_amd
    c = s["case"]
    return apexw_amd.embedding_weight_grad(s["dy"], s["ids"], c["vocab"], c["scale"], dtype=DTYPES[c["grad"]])


def _plain_head_forward(s):
    kept = s["target"] != IGNORED
    logits = s["x"].float() @ s["w"].float().t()
    top = logits.max(1, keepdim=True)[0]
    hit = logits.gather(1, s["target"].clamp(min=0)[:, None])[:, 0]
    lse = torch.log(torch.exp(logits - top).sum(1)) + top[:, 0]
    return {"loss": torch.where(kept, lse - hit, 0.0), "lse": torch.where(kept, lse, 0.0)}


def _plain_head_backward(s):
    x, w, target = s["x"].float(), s["w"].float(), s["target"]
    scale = torch.where(target != IGNORED, s["dloss"], 0.0)[:, None]
    g = torch.exp(x @ w.t() - s["lse"][:, None]) * scale
    g.scatter_add_(1, target.clamp(min=0)[:, None], -scale)
    return {"dx": (g @ w).to(s["x"].dtype), "dw": (g.t() @ x).to(s["w"].dtype)}


def _plain_order(expert, experts):
    """(the choice in each row, the row of each choice, one past each expert's last row); -1 for none."""
    flat = torch.where((expert < 0) | (expert >= experts), experts, expert).view(-1)
    choice = torch.sort(flat, stable=True)[1]
    place = torch.empty_like(choice)
    place[choice] = torch.arange(len(choice), device=choice.device)
    ends = torch.bincount(flat, minlength=experts + 1)[:experts].cumsum(0)
    source = torch.where(flat[choice] < experts, choice, -1)
    place = torch.where(flat < experts, place, -1)
    return source.int(), place.view(expert.shape).int(), ends.int()


def _plain_dispatch(s):
    source, place, ends = _plain_order(s["expert"], s["case"]["experts"])
    token = torch.div(source.clamp(min=0), s["case"]["k"], rounding_mode="floor")
    rows = torch.where((source >= 0)[:, None], s["x"][token], 0.0)
    return {"rows": rows, "source": source, "place": place, "ends": ends}


def _plain_dispatch_grad(s):
    place = s["order"][1]
    rows = torch.where((place >= 0)[..., None], s["drows"][place.clamp(min=0)].float(), 0.0)
    return rows.sum(1).to(s["drows"].dtype)


def _plain_combine(s):
    place = s["order"][1]
    rows = torch.where((place >= 0)[..., None], s["y"][place.clamp(min=0)].float() * s["w"].float()[..., None], 0.0)
    return rows.sum(1).to(s["y"].dtype)


def _plain_combine_grad(s):
    source, place, _ = s["order"]
    choice = source.clamp(min=0)
    token = torch.div(choice, s["case"]["k"], rounding_mode="floor")
    dout = s["dout"].float()
    dy = torch.where((source >= 0)[:, None], s["w"].float().view(-1)[choice][:, None] * dout[token], 0.0)
    dw = (s["y"][place.clamp(min=0)].float() * dout[:, None]).sum(2)
    return {"dy": dy.to(s["y"].dtype), "dw": torch.where(place >= 0, dw, 0.0).to(s["w"].dtype)}


def _plain_embedding(s):
    return (s["w"][s["ids"]].float() * s["case"]["scale"]).to(s["w"].dtype)


def _plain_embedding_grad(s):
    c = s["case"]
    dw = torch.zeros(c["vocab"], c["width"], dtype=torch.float32, device=s["dy"].device)
    dw.index_add_(0, s["ids"], s["dy"].float() * c["scale"])
    return dw.to(DTYPES[c["grad"]])


_OWN = {("head", "forward"): _own_head_forward, ("head", "backward"): _own_head_backward,
        ("experts", "dispatch"): _own_dispatch, ("experts", "dispatch_grad"): _own_dispatch_grad,
        ("experts", "combine"): _own_combine, ("experts", "combine_grad"): _own_combine_grad,
        ("embedding", "forward"): _own_embedding, ("embedding", "grad"): _own_embedding_grad}
_PLAIN = {("head", "forward"): _plain_head_forward, ("head", "backward"): _plain_head_backward,
          ("experts", "dispatch"): _plain_dispatch, ("experts", "dispatch_grad"): _plain_dispatch_grad,
          ("experts", "combine"): _plain_combine, ("experts", "combine_grad"): _plain_combine_grad,
          ("embedding", "forward"): _plain_embedding, ("embedding", "grad"): _plain_embedding_grad}


# ---------------------------------------------------------------------------- what a pass needs
def work(case):
    """Bytes: each input read once, each output written once, of a table's rows those that are looked up.  FLOPs:
    the multiplications and additions of the formulas over the rows that count."""
    size = DTYPES[case["dtype"]].itemsize
    if case["op"] == "head":
        rows, width, vocab = case["rows"], case["width"], case["vocab"]
        kept = rows - int(rows * case["ignored"])
        x, w = kept * width * size, vocab * width * size
        if case["way"] == "forward":
            return {"bytes": x + w + 16 * rows, "flops": 2 * kept * width * vocab}
        return {"bytes": x + rows * width * size + 2 * w + 16 * rows, "flops": 6 * kept * width * vocab}
    if case["op"] == "experts":
        tokens, choices, width = case["tokens"], case["tokens"] * case["k"], case["width"]
        weights = choices * DTYPES[case["weights"]].itemsize
        moved = (tokens + choices) * width * size
        if case["way"] == "dispatch":
            return {"bytes": moved + 16 * choices + 4 * case["experts"], "flops": choices}
        if case["way"] == "dispatch_grad":
            return {"bytes": moved + 4 * choices, "flops": choices * width}
        if case["way"] == "combine":
            return {"bytes": moved + 4 * choices + weights, "flops": 2 * choices * width}
        return {"bytes": moved + choices * width * size + 8 * choices + 2 * weights, "flops": 3 * choices * width}
    n = case["tokens"] * case["width"]
    if case["way"] == "forward":
        return {"bytes": 2 * n * size + 8 * case["tokens"], "flops": n}
    return {"bytes": n * size + 8 * case["tokens"] + case["vocab"] * case["width"] * DTYPES[case["grad"]].itemsize,
            "flops": n}


# ---------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "head":
        x, w = s["x"], s["w"].double()
        step = max(1, 2 ** 28 // case["vocab"])
        if case["way"] == "forward":
            out = {"loss": torch.zeros(case["rows"], dtype=torch.float64, device=x.device)}
            out["lse"] = torch.zeros_like(out["loss"])
            for a in range(0, case["rows"], step):
                logits, t = torch.mm(x[a:a + step].double(), w.t()), s["target"][a:a + step]
                at = torch.nonzero(t >= 0)[:, 0]
                lse = torch.logsumexp(logits[at], 1)
                out["lse"][a + at] = lse
                out["loss"][a + at] = lse - logits[at, t[at]]
            return out
        dx = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
        dw = torch.zeros_like(w)
        for a in range(0, case["rows"], step):
            rows, t = x[a:a + step].double(), s["target"][a:a + step]
            at = torch.nonzero(t >= 0)[:, 0]
            p = torch.exp(torch.mm(rows[at], w.t()) - s["lse"][a + at].double()[:, None])
            p[torch.arange(len(at), device=x.device), t[at]] -= 1.0
            p *= s["dloss"][a + at].double()[:, None]
            dx[a + at] = torch.mm(p, w)
            dw.addmm_(p.t(), rows[at])
        return {"dx": dx, "dw": dw}
    if case["op"] == "experts":
        k = case["k"]
        if case["way"] == "dispatch":
            flat = s["expert"].reshape(-1)
            lists = [torch.nonzero(flat == e)[:, 0] for e in range(case["experts"])]
            row = torch.cat(lists)
            source = torch.full((len(flat),), -1, device=flat.device)
            source[:len(row)] = row
            place = torch.full_like(flat, -1)
            place[row] = torch.arange(len(row), device=flat.device)
            rows = torch.zeros(len(flat), case["width"], dtype=torch.float64, device=flat.device)
            rows[:len(row)] = s["x"].double()[row // k]
            ends = torch.tensor([len(i) for i in lists], device=flat.device).cumsum(0)
            return {"rows": rows, "source": source.int(), "place": place.view_as(s["expert"]).int(), "ends": ends.int()}
        source, place, ends = s["order"]
        used = int(ends[-1])
        choice = source[:used].long()
        if case["way"] in ("dispatch_grad", "combine"):
            rows = (s["drows"] if case["way"] == "dispatch_grad" else s["y"])[:used].double()
            if case["way"] == "combine":
                rows = rows * s["w"].double().view(-1)[choice][:, None]
            out = torch.zeros(case["tokens"], case["width"], dtype=torch.float64, device=rows.device)
            return out.index_add_(0, choice // k, rows)
        dout, w = s["dout"].double()[choice // k], s["w"].double().view(-1)[choice]
        dy = torch.zeros(s["y"].shape, dtype=torch.float64, device=dout.device)
        dy[:used] = dout * w[:, None]
        dw = torch.zeros(case["tokens"] * k, dtype=torch.float64, device=dout.device)
        dw[choice] = torch.linalg.vecdot(s["y"][:used].double(), dout)
        return {"dy": dy, "dw": dw.view(case["tokens"], k)}
    if case["way"] == "forward":
        return torch.index_select(s["w"], 0, s["ids"]).double() * case["scale"]
    dw = torch.zeros(case["vocab"], case["width"], dtype=torch.float64, device=s["dy"].device)
    for a in range(0, case["tokens"], 8192):
        dw.index_add_(0, s["ids"][a:a + 8192], s["dy"][a:a + 8192].double())
    return dw * case["scale"]
