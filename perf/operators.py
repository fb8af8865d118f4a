"""Workloads of the operators at the two ends of a language model that shares one table between its input
embedding and its output head:

  loss        linear softmax cross entropy: logits = hidden @ weight^T, the loss of each token and of the batch, and the
              gradients of hidden and weight, without a teacher and without the [tokens, vocabulary] logits as a result
  embed       rows of the table picked by token id, times a scale
  embed_grad  its gradient: the rows of grad_out added up by token id, into zeros or on top of a gradient that is there

Each has its plain form in elementary torch operations (32-bit arithmetic, rounded once at the end) and the calls of
orda_b200.device.
"""
import math
import sys

import torch

own = False

IGNORE = -100
_context = None


def _device_context():
    """The handle a program keeps for all its calls."""
    global _context
    if _context is None:
        if "orda-cutile-rs_b200" not in sys.path:
            sys.path.insert(0, "orda-cutile-rs_b200")
        from orda_b200.device import DeviceContext

        _context = DeviceContext(torch.cuda.current_device())
    return _context


# ------------------------------------------------------------------ cases


def _loss(name, bt, h, v, grads=True, ignored=0.0, smoothing=0.0, mean=True, limit=0):
    return {"name": name, "op": "loss", "bt": bt, "h": h, "v": v, "grads": grads, "ignored": ignored,
            "smoothing": smoothing, "mean": mean, "limit": limit}


def _embed(name, n, h, v, dtype="bf16"):
    return {"name": name, "op": "embed", "n": n, "h": h, "v": v, "dtype": dtype}


def _embed_grad(name, n, h, v, dtype="bf16", out="bf16", accumulate=False):
    return {"name": name, "op": "embed_grad", "n": n, "h": h, "v": v, "dtype": dtype, "out": out,
            "accumulate": accumulate}


def listed():
    return [
        # the log-probability of one sampled token: the head's weights are read once
        _loss("loss of one token", 1, 4096, 131072, grads=False),
        # scoring the tokens of a few short prompts, odd count
        _loss("loss of 77 tokens", 77, 2048, 128256, grads=False),
        # a training step of a small model: launches and latency count
        _loss("train 256x512x8192", 256, 512, 8192),
        # the shape of the tied-teacher library example
        _loss("train 2048x4096x32000", 2048, 4096, 32000),
        # odd sizes, prompts masked out of the loss, label smoothing, summed losses
        _loss("train 1999x1000x100003", 1999, 1000, 100003, ignored=0.3, smoothing=0.1, mean=False),
        # memory-bound training: a workspace of 256 MiB, an eighth of the 16-bit logits
        _loss("train 8192x2048x128256 in 256 MiB", 8192, 2048, 128256, ignored=0.1, limit=256 << 20),
        # the headline shape of the repository's benchmark
        _loss("train 8192x4096x131072", 8192, 4096, 131072),
        # decoding: the embeddings of the next tokens of eight sequences
        _embed("embed 8", 8, 4096, 131072),
        # a prompt or a training batch
        _embed("embed 16384", 16384, 4096, 131072),
        # a training batch's gradient of the whole table
        _embed_grad("embed grad 8192", 8192, 4096, 131072),
        # shared table: the embedding's gradient on top of the head's fp32 gradient
        _embed_grad("embed grad 8192 on top", 8192, 4096, 131072, out="f32", accumulate=True),
        # odd sizes in fp32, few tokens that come up often
        _embed_grad("embed grad 5003x1001 f32", 5003, 1001, 997, dtype="f32", out="f32"),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["score", "train", "train", "embed", "embed_grad", "embed_grad"])
    if kind in ("score", "train"):
        v = _log_uniform(rng, 500, 131072)
        h = 8 * _log_uniform(rng, 8, 512)  # the tensor cores' operands start on 16-byte rows
        if kind == "score":
            case = _loss("", _log_uniform(rng, 1, 4096), h, v, grads=False, ignored=rng.choice([0.0, 0.0, 0.5]))
        else:
            case = _loss("", _log_uniform(rng, 1, 8192), h, v, ignored=rng.choice([0.0, 0.0, 0.1, 0.6]),
                         smoothing=rng.choice([0.0, 0.0, 0.1]), mean=rng.random() < 0.7,
                         limit=rng.choice([0, 0, 0, 64 << 20]))
    elif kind == "embed":
        case = _embed("", _log_uniform(rng, 1, 32768), _log_uniform(rng, 16, 8192), _log_uniform(rng, 500, 131072),
                      dtype=rng.choice(["bf16", "bf16", "f32"]))
    else:
        case = _embed_grad("", _log_uniform(rng, 1, 32768), _log_uniform(rng, 16, 4096),
                           _log_uniform(rng, 500, 131072), dtype=rng.choice(["bf16", "bf16", "f32"]),
                           out=rng.choice(["bf16", "f32"]))
        if case["out"] == "f32":
            case["accumulate"] = rng.random() < 0.5
    del case["name"]
    return case


# ------------------------------------------------------------------ inputs

_DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _token_ids(n, v, gen):
    """Token ids with the skew of text: the frequency of an id falls as its rank (log-uniform ids)."""
    u = torch.rand(n, generator=gen, device="cuda", dtype=torch.float64)
    return torch.exp(u * math.log(v + 1.0)).long().sub_(1).clamp_(0, v - 1)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32)

    v, h = case["v"], case["h"]
    if case["op"] == "loss":
        bt = case["bt"]
        weight = torch.empty(v, h, device="cuda", dtype=torch.bfloat16)
        weight.normal_(0.0, 0.02, generator=gen)
        labels = _token_ids(bt, v, gen)
        # hidden states that point towards their label as a model in training does: its logit stands up to
        # 12 above the others', more for some tokens than for others
        pull = torch.rand(bt, 1, generator=gen, device="cuda") * (12.0 / (0.02 * 0.02 * h))
        hidden = (randn(bt, h) + pull * weight[labels].float()).bfloat16()
        if case["ignored"] > 0:
            drop = torch.rand(bt, generator=gen, device="cuda") < case["ignored"]
            labels = torch.where(drop, torch.full_like(labels, IGNORE), labels)
        return {"case": dict(case), "hidden": hidden, "weight": weight, "labels": labels}
    n, dtype = case["n"], _DTYPES[case["dtype"]]
    ids = _token_ids(n, v, gen)
    state = {"case": dict(case), "ids": ids, "scale": math.sqrt(h)}
    if case["op"] == "embed":
        state["table"] = torch.empty(v, h, device="cuda", dtype=dtype).normal_(0.0, 0.02, generator=gen)
    else:
        state["grad_out"] = (randn(n, h) * 1e-3).to(dtype)
        if case["accumulate"]:
            state["grad"] = torch.empty(v, h, device="cuda", dtype=_DTYPES[case["out"]]).normal_(0.0, 1e-3,
                                                                                                 generator=gen)
    return state


# ------------------------------------------------------------------ plain forms


def _loss_plain(state):
    case, labels = state["case"], state["labels"]
    hidden, weight = state["hidden"].float(), state["weight"].float()
    v, a = case["v"], case["smoothing"]
    live = labels != IGNORE
    at = torch.where(live, labels, 0).unsqueeze(1)
    logits = hidden @ weight.T
    top = logits.amax(1, keepdim=True)
    picked = logits.gather(1, at)
    mean_logit = logits.mean(1, keepdim=True) if a > 0 else picked
    p = logits.sub_(top).exp_()
    total = p.sum(1, keepdim=True, dtype=torch.float64)
    lse = (top.double() + total.log())
    nll = torch.where(live, (lse - (1 - a) * picked - a * mean_logit).squeeze(1), 0.0)
    count = live.sum().clamp(min=1) if case["mean"] else torch.ones((), device=labels.device)
    out = {"loss": (nll.sum() / count).float(), "nll": nll.float(),
           "lse": torch.where(live, lse.squeeze(1), 0.0).float()}
    if case["grads"]:
        p.div_(total.float()).sub_(a / v)
        p.scatter_(1, at, p.gather(1, at) - (1 - a))
        p.mul_((live / count).float().unsqueeze(1))
        out["grad_hidden"] = (p @ weight).bfloat16()
        out["grad_weight"] = (p.T @ hidden).bfloat16()
    return out


def _embed_plain(state):
    table = state["table"]
    return {"out": (table[state["ids"]].float() * state["scale"]).to(table.dtype)}


def _embed_grad_plain(state):
    case = state["case"]
    rows = state["grad_out"].float() * state["scale"]
    if case["accumulate"]:
        state["grad"].index_add_(0, state["ids"], rows)
        return {"grad": state["grad"]}
    grad = torch.zeros(case["v"], case["h"], device=rows.device, dtype=torch.float32)
    return {"grad": grad.index_add_(0, state["ids"], rows).to(_DTYPES[case["out"]])}


# ------------------------------------------------------------------ one pass


def _run_own(state):
    from orda_b200 import Reduction
    from orda_b200 import device as dev

    ctx, case = _context or _device_context(), state["case"]
    if case["op"] == "loss":
        r = dev.linear_cross_entropy_device(
            ctx, state["hidden"], state["weight"], state["labels"], ignore_index=IGNORE,
            label_smoothing=case["smoothing"], reduction=Reduction.Mean if case["mean"] else Reduction.Sum,
            need_grad_hidden=case["grads"], need_grad_weight=case["grads"], grad_dtype=torch.bfloat16,
            piece_bytes=case["limit"])
        out = {"loss": r.loss, "nll": r.nll, "lse": r.lse}
        if case["grads"]:
            out["grad_hidden"], out["grad_weight"] = r.grad_hidden, r.grad_weight
        return out
    if case["op"] == "embed":
        return {"out": dev.embedding_device(ctx, state["table"], state["ids"], scale=state["scale"])}
    if case["accumulate"]:
        dev.embedding_grad_device(ctx, state["grad_out"], state["ids"], case["v"], scale=state["scale"],
                                  out=state["grad"], accumulate=True)
        return {"grad": state["grad"]}
    return {"grad": dev.embedding_grad_device(ctx, state["grad_out"], state["ids"], case["v"], scale=state["scale"],
                                              dtype=_DTYPES[case["out"]])}


def run(state):
    if own:
        _device_context()
        return _run_own(state)
    return {"loss": _loss_plain, "embed": _embed_plain, "embed_grad": _embed_grad_plain}[state["case"]["op"]](state)


# ------------------------------------------------------------------ floors


def _distinct(n, v):
    """Expected count of different ids among n of _token_ids."""
    k = torch.arange(1, v + 1, dtype=torch.float64)
    p = torch.log((k + 1) / k) / math.log(v + 1.0)
    return float((1 - (1 - p) ** n).sum())


def work(case):
    h, v = case["h"], case["v"]
    if case["op"] == "loss":
        bt = case["bt"]
        once = 2 * (bt + v) * h
        if not case["grads"]:
            return {"bytes": once + 16 * bt + 4, "flops": 2 * bt * v * h}
        return {"bytes": 2 * once + 16 * bt + 4, "flops": 6 * bt * v * h}
    n, size = case["n"], {"bf16": 2, "f32": 4}
    if case["op"] == "embed":
        return {"bytes": (n + _distinct(n, v)) * h * size[case["dtype"]] + 8 * n, "flops": n * h}
    rows = 2 * _distinct(n, v) if case["accumulate"] else v
    return {"bytes": n * h * size[case["dtype"]] + 8 * n + rows * h * size[case["out"]], "flops": n * h}


# ------------------------------------------------------------------ exact values


def _exact_loss(case, state):
    """64-bit values, a group of tokens at a time; the softmax through the differences to the label's logit."""
    w = state["weight"].double()
    bt, v, a = case["bt"], case["v"], case["smoothing"]
    labels = state["labels"]
    n_live = int((labels != IGNORE).sum())
    g = 1.0 / max(n_live, 1) if case["mean"] else 1.0
    nll = torch.zeros(bt, dtype=torch.float64, device="cuda")
    lse = torch.zeros_like(nll)
    grad_h = torch.zeros(bt, case["h"], dtype=torch.float64, device="cuda") if case["grads"] else None
    grad_w = torch.zeros(v, case["h"], dtype=torch.float64, device="cuda") if case["grads"] else None
    rows = torch.nonzero(labels != IGNORE).flatten()
    for part in rows.split(1024):
        x = state["hidden"][part].double()
        y = labels[part]
        z = x @ w.T
        lse[part] = torch.logsumexp(z, 1)
        own_logit = (x * w[y]).sum(1)
        nll[part] = (1 - a) * (lse[part] - own_logit) + (a * (lse[part].unsqueeze(1) - z).mean(1) if a > 0 else 0.0)
        if case["grads"]:
            target = torch.full_like(z, a / v)
            target[torch.arange(len(part), device="cuda"), y] += 1 - a
            d = (torch.exp(z - lse[part].unsqueeze(1)) - target) * g
            grad_h[part] = d @ w
            grad_w += d.T @ x
    out = {"loss": nll.sum() * g, "nll": nll, "lse": lse}
    if case["grads"]:
        out["grad_hidden"], out["grad_weight"] = grad_h, grad_w
    return out


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "loss":
        return _exact_loss(case, state)
    if case["op"] == "embed":
        return {"out": state["table"].double().index_select(0, state["ids"]) * state["scale"]}
    if case["accumulate"]:
        grad = state["grad"].double()
    else:
        grad = torch.zeros(case["v"], case["h"], dtype=torch.float64, device="cuda")
    grad.index_put_((state["ids"],), state["grad_out"].double() * state["scale"], accumulate=True)
    return {"grad": grad}
