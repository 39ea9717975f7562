"""Cases of the layer operators beside the protected GEMMs: real work over the
range that a training or serving program of this library calls them with.

Three operators:

* ``rotary``: norm of each query and key head and the rotation by position
  (``sdc_b200.layers.head_norm_rotary``), forward, and forward with backward;
* ``adapters``: low-rank adapters of many requests added to a shared
  projection's output (``sdc_b200.layers.low_rank_adapters``), forward, and
  forward with backward;
* ``distill``: distillation loss against a teacher's top logits
  (``sdc_b200.layers.distillation_loss`` and ``distillation_loss_and_grad``):
  the losses alone, losses and gradient in one call, and the mean loss with
  its backward pass through autograd.

``run`` computes a case in plain torch operations in fp32, or, with ``own``
set, through the library's public calls.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
TABLE = 32768  # positions of the rotation table (max_position_embeddings of the training workload)
EPS = 1e-6
ROPE_BASE = 1e6


# ------------------------------------------------------------------ cases ----

def _rotary(mode, tokens, sequence, heads, kv_heads, dim, rotary, dtype, interleaved=False, norm=True):
    return {"op": "rotary", "mode": mode, "tokens": tokens, "sequence": sequence, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "rotary": rotary, "dtype": dtype, "interleaved": interleaved,
            "norm": norm}


def _adapters(mode, tokens, requests, adapters, rank, k, n, dtype, without=0.0):
    return {"op": "adapters", "mode": mode, "tokens": tokens, "requests": requests, "adapters": adapters,
            "rank": rank, "k": k, "n": n, "dtype": dtype, "without": without}


def _distill(mode, rows, vocab, top, dtype, temperature=1.0, ragged=False):
    return {"op": "distill", "mode": mode, "rows": rows, "vocab": vocab, "top": top, "dtype": dtype,
            "temperature": temperature, "ragged": ragged}


def listed():
    return [
        # One decoded token of the 28 + 4 head, dim 128 attention: only latency counts.
        {"name": "rotary_decode_1", **_rotary("forward", 1, 1, 28, 4, 128, 128, "bf16")},
        # The prompt batch of the linear sweep (16384 tokens), views of the fused QKV projection.
        {"name": "rotary_prefill_16384", **_rotary("forward", 16384, 4096, 28, 4, 128, 128, "bf16")},
        # The training step's micro-batch (8 x 2048 tokens, 14 + 2 heads of dim 64), forward and backward.
        {"name": "rotary_train_16384", **_rotary("train", 16384, 2048, 14, 2, 64, 64, "bf16")},
        # An fp32 fine-tuning step on an odd number of tokens: half of an odd-sized head rotated, pairs interleaved.
        {"name": "rotary_train_fp32_odd", **_rotary("train", 1031, 347, 14, 2, 80, 40, "fp32", True)},
        # One decoded token with one adapter beside the output projection.
        {"name": "adapters_decode_1", **_adapters("forward", 1, 1, 1, 16, 3584, 3584, "bf16")},
        # A decoding batch beside the QKV projection: one token a request, few requests an adapter, some without one.
        {"name": "adapters_decode_192", **_adapters("forward", 192, 192, 48, 16, 3584, 4608, "bf16", 0.1)},
        # Prompts of odd lengths beside the gate/up projection, a rank that is not a power of two.
        {"name": "adapters_prefill_odd", **_adapters("forward", 8191, 23, 8, 24, 3584, 18944, "fp16", 0.1)},
        # Fine-tuning four adapters at once beside the output projection, forward and backward.
        {"name": "adapters_train_16384", **_adapters("train", 16384, 8, 4, 32, 3584, 3584, "bf16")},
        # One position's loss, as when candidates are scored one by one.
        {"name": "distill_score_1", **_distill("loss", 1, 151936, 20, "bf16")},
        # The held-out losses of a short sequence, position by position.
        {"name": "distill_eval_509", **_distill("loss", 509, 151936, 64, "bf16", 1.0, True)},
        # A training micro-batch's loss and logit gradient in one call (2 x 2048 tokens).
        {"name": "distill_step_4096", **_distill("grad", 4096, 151936, 64, "bf16", 2.0, True)},
        # fp32 logits of an odd vocabulary through autograd, lists of unequal length.
        {"name": "distill_train_fp32_odd", **_distill("train", 333, 50021, 100, "fp32", 1.5, True)},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["rotary", "adapters", "distill"])
    if op == "rotary":
        heads, kv = rng.choice([(28, 4), (14, 2), (14, 14), (7, 1), (1, 1)])
        dim = rng.choice([64, 80, 96, 128, 256])
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        tokens = _log(rng, 1, 16384 * 32 * 128 // ((heads + kv) * dim * (2 if dtype == "fp32" else 1)))
        tokens = min(tokens, 16384)
        return _rotary(rng.choice(["forward", "train"]), tokens, max(1, tokens // rng.randint(1, 8)), heads, kv, dim,
                       rng.choice([dim, dim, dim // 2]), dtype, rng.random() < 0.3, rng.random() < 0.8)
    if op == "adapters":
        k, n = rng.choice([(896, 896), (896, 4864), (4864, 896), (3584, 4608), (3584, 3584), (3584, 18944),
                           (18944, 3584), (1000, 1336)])
        rank = rng.choice([4, 8, 16, 32, 64, rng.randint(1, 64)])
        mode = rng.choice(["forward", "forward", "train"])
        tokens = _log(rng, 1, min(16384, 8191 * (3584 + 18944) // (k + n) // (2 if mode == "train" else 1)))
        requests = _log(rng, 1, min(tokens, 256))
        return _adapters(mode, tokens, requests, _log(rng, 1, 64), rank, k, n, rng.choice(["bf16", "bf16", "fp16"]),
                         rng.choice([0.0, 0.1, 0.5]))
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    vocab = rng.choice([151936, _log(rng, 1000, 151936), _log(rng, 1000, 151936)])
    rows = _log(rng, 1, min(8192, 4096 * 151936 // vocab // (2 if dtype == "fp32" else 1)))
    return _distill(rng.choice(["loss", "grad", "train"]), rows, vocab, _log(rng, 1, 256), dtype,
                    rng.choice([1.0, 1.0, 1.5, 2.0]), rng.random() < 0.5)


# ---------------------------------------------------------------- prepare ----

def _requests(case, seed):
    """Host lists that a scheduler has: the requests' lengths (their sum is the number of tokens) and adapters
    (-1: none)."""
    rng = np.random.default_rng(seed)
    tokens, requests = case["tokens"], case["requests"]
    cuts = np.sort(rng.choice(np.arange(1, tokens), requests - 1, replace=False)) if requests > 1 else []
    lengths = np.diff(np.concatenate([[0], cuts, [tokens]]).astype(np.int64))
    adapters = rng.integers(0, case["adapters"], requests)
    adapters[rng.random(requests) < case["without"]] = -1
    return lengths.tolist(), adapters.tolist()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    state = {"case": case}

    def normal(*shape, scale=1.0, dtype=dtype):
        return (torch.randn(*shape, device="cuda", generator=g, dtype=torch.float32) * scale).to(dtype)

    if case["op"] == "rotary":
        t, h, hk, d, r = (case[key] for key in ("tokens", "heads", "kv_heads", "dim", "rotary"))
        qkv = normal(t, (h + 2 * hk) * d, scale=1.5)
        state["q"] = qkv[:, :h * d].view(t, h, d)
        state["k"] = qkv[:, h * d:(h + hk) * d].view(t, hk, d)
        start = seed % 1000 if case["sequence"] > 1 else 17 + seed % (TABLE - 17)
        state["positions"] = (torch.arange(t, device="cuda") % case["sequence"]) + start
        angle = torch.arange(TABLE, device="cuda", dtype=torch.float64)[:, None] * \
            ROPE_BASE ** (-torch.arange(0, r, 2, device="cuda", dtype=torch.float64) / r)
        state["table"] = torch.cat((angle.cos(), angle.sin()), 1).float()
        state["q_weight"] = state["k_weight"] = None
        if case["norm"]:
            state["q_weight"] = (1 + normal(d, scale=0.2, dtype=torch.float32)).to(dtype)
            state["k_weight"] = (1 + normal(d, scale=0.2, dtype=torch.float32)).to(dtype)
        if case["mode"] == "train":
            state["dq"], state["dk"] = normal(t, h, d), normal(t, hk, d)
    elif case["op"] == "adapters":
        t, a, r, k, n = (case[key] for key in ("tokens", "adapters", "rank", "k", "n"))
        lengths, ids = _requests(case, seed)
        state["base"], state["x"] = normal(t, n), normal(t, k)
        state["a"] = normal(a, r, k, scale=k ** -0.5)
        state["b"] = normal(a, n, r, scale=r ** -0.5)
        state["scale"] = torch.rand(a, device="cuda", generator=g) + 0.5
        state["lengths"], state["ids"] = lengths, ids
        state["token_ids"] = torch.tensor(np.repeat(ids, lengths), device="cuda")
        if case["mode"] == "train":
            state["dy"] = normal(t, n)
        if own:
            # A serving or training step builds this once and uses it for every projection of every layer.
            from sdc_b200.layers import AdapterBatch
            state["batch"] = AdapterBatch(lengths, ids, a)
    else:
        rows, vocab, top = case["rows"], case["vocab"], min(case["top"], case["vocab"])
        logits = normal(rows, vocab, scale=2.5)
        state["logits"] = logits
        indices = torch.empty(rows, top, device="cuda", dtype=torch.int64)
        for i in range(0, rows, 1024):
            indices[i:i + 1024] = logits[i:i + 1024].topk(top, 1).indices
        # The teacher agrees on half of the list; the rest it took elsewhere (a stride over the vocabulary keeps
        # the indices of a row distinct). Its logits fall off along the list.
        shift = torch.arange(top, device="cuda") % 2 * (1 + seed % 7)
        indices = (indices + shift) % vocab
        srt, order = indices.sort(1)
        repeated = torch.zeros_like(srt, dtype=torch.bool)
        repeated[:, 1:] = srt[:, 1:] == srt[:, :-1]
        indices[torch.zeros_like(repeated).scatter(1, order, repeated)] = -1  # entries without a token
        teacher = 12 - 0.15 * torch.arange(top, device="cuda") + normal(rows, top, dtype=torch.float32)
        if case["ragged"]:
            lengths = torch.randint(1, top + 1, (rows, 1), device="cuda", generator=g)
            lengths[torch.rand(rows, 1, device="cuda", generator=g) < 0.05] = 0  # prompt positions: nothing to learn
            lengths[0] = top
            indices[torch.arange(top, device="cuda") >= lengths] = -1
        state["indices"], state["teacher"] = indices, teacher
        state["grad_loss"] = torch.full((), 1.0 / rows, device="cuda")
    return state


# -------------------------------------------------------------- plain forms ----

def _rotation(case, x, cos, sin, back=False):
    """Rotates the first ``rotary`` elements of each head of x [T, H, D] by the angles [T, 1, R/2]."""
    r = case["rotary"]
    sin = -sin if back else sin
    if case["interleaved"]:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., :r // 2], x[..., r // 2:r]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, x[..., r:]), -1)


def _plain_rotary(s):
    case = s["case"]
    half = case["rotary"] // 2
    angles = s["table"][s["positions"]][:, None, :]
    cos, sin = angles[..., :half], angles[..., half:]

    def forward(x, w):
        x = x.float()
        if w is not None:
            x = x * (x.square().mean(-1, keepdim=True) + EPS).rsqrt() * w.float()
        return _rotation(case, x, cos, sin)

    def backward(dy, x, w):
        dy = _rotation(case, dy.float(), cos, sin, True)
        if w is None:
            return dy, None
        x = x.float()
        rstd = (x.square().mean(-1, keepdim=True) + EPS).rsqrt()
        unit = x * rstd
        dunit = dy * w.float()
        return rstd * (dunit - unit * (dunit * unit).mean(-1, keepdim=True)), (dy * unit).sum((0, 1))

    out = {"q": forward(s["q"], s["q_weight"]), "k": forward(s["k"], s["k_weight"])}
    if case["mode"] == "train":
        out["dq"], out["dq_weight"] = backward(s["dq"], s["q"], s["q_weight"])
        out["dk"], out["dk_weight"] = backward(s["dk"], s["k"], s["k_weight"])
    return {name: value.to(s["q"].dtype) for name, value in out.items() if value is not None}


def _plain_adapters(s):
    case, dtype = s["case"], s["x"].dtype
    adapters, rank = case["adapters"], case["rank"]
    # All adapters' rows side by side; a token keeps its own adapter's products and zeros the others'.
    mine = (s["token_ids"][:, None] == torch.arange(adapters, device="cuda")) * s["scale"]
    mine = mine.repeat_interleave(rank, 1)
    a = s["a"].float().flatten(0, 1)
    b = s["b"].float().transpose(1, 2).flatten(0, 1)
    x = s["x"].float()
    low = (x @ a.T) * mine
    out = {"out": (s["base"].float() + low @ b).to(dtype)}
    if case["mode"] == "train":
        dy = s["dy"].float()
        dlow = (dy @ b.T) * mine
        out["dx"] = (dlow @ a).to(dtype)
        out["da"] = (dlow.T @ x).view(adapters, rank, -1).to(dtype)
        out["db"] = (low.T @ dy).view(adapters, rank, -1).transpose(1, 2).to(dtype)
    return out


def _plain_distill(s):
    case, dtype = s["case"], s["logits"].dtype
    t = case["temperature"]
    logits = s["logits"].float() / t
    top = logits.max(1, keepdim=True).values
    lse = top + (logits - top).exp().sum(1, keepdim=True).log()
    kept = s["indices"] >= 0
    some = kept.any(1, keepdim=True)
    at = s["indices"].clamp_min(0)
    teacher = (s["teacher"] / t).masked_fill(~kept, -math.inf)
    teacher = teacher - teacher.max(1, keepdim=True).values.masked_fill(~some, 0.0)
    p = teacher.exp()
    total = p.sum(1, keepdim=True).masked_fill(~some, 1.0)
    p = p / total
    log_ratio = (teacher - total.log()).masked_fill(~kept, 0.0) - (logits.gather(1, at) - lse)
    loss = t * t * (p * log_ratio).sum(1)
    valid = some.sum().clamp_min(1)
    if case["mode"] == "loss":
        return loss
    row = s["grad_loss"] if case["mode"] == "grad" else 1.0 / valid
    grad = (logits - lse).exp() * some
    grad = (grad.scatter_add(1, at, -p) * (row * t)).to(dtype)
    return {"loss": loss if case["mode"] == "grad" else loss.sum() / valid, "grad": grad}


# ------------------------------------------------------- the library's calls ----

def _own_rotary(s):
    from sdc_b200.layers import head_norm_rotary

    case = s["case"]
    if case["mode"] == "forward":
        q, k = head_norm_rotary(s["q"], s["k"], s["table"], s["positions"], s["q_weight"], s["k_weight"], EPS,
                                case["interleaved"])
        return {"q": q, "k": k}
    names = ["q", "k"] + (["q_weight", "k_weight"] if case["norm"] else [])
    inputs = [s[name].detach().requires_grad_() for name in names]
    q, k = head_norm_rotary(inputs[0], inputs[1], s["table"], s["positions"], *(inputs[2:] or (None, None)), EPS,
                            case["interleaved"])
    grads = torch.autograd.grad((q, k), inputs, (s["dq"], s["dk"]))
    out = {"q": q.detach(), "k": k.detach(), "dq": grads[0]}
    if case["norm"]:
        out.update(dq_weight=grads[2], dk=grads[1], dk_weight=grads[3])
    else:
        out.update(dk=grads[1])
    return out


def _own_adapters(s):
    from sdc_b200.layers import low_rank_adapters

    if s["case"]["mode"] == "forward":
        return {"out": low_rank_adapters(s["base"], s["x"], s["a"], s["b"], s["batch"], s["scale"])}
    x, a, b = (s[name].detach().requires_grad_() for name in ("x", "a", "b"))
    out = low_rank_adapters(s["base"], x, a, b, s["batch"], s["scale"])
    dx, da, db = torch.autograd.grad(out, (x, a, b), s["dy"])
    return {"out": out.detach(), "dx": dx, "da": da, "db": db}


def _own_distill(s):
    from sdc_b200.layers import distillation_loss, distillation_loss_and_grad

    case = s["case"]
    args = (s["indices"], s["teacher"], case["temperature"])
    if case["mode"] == "loss":
        return distillation_loss(s["logits"], *args, reduction="none")
    if case["mode"] == "grad":
        loss, grad = distillation_loss_and_grad(s["logits"], *args, grad_loss=s["grad_loss"])
        return {"loss": loss, "grad": grad}
    logits = s["logits"].detach().requires_grad_()
    loss = distillation_loss(logits, *args)
    return {"loss": loss.detach(), "grad": torch.autograd.grad(loss, logits)[0]}


PLAIN = {"rotary": _plain_rotary, "adapters": _plain_adapters, "distill": _plain_distill}
OWN = {"rotary": _own_rotary, "adapters": _own_adapters, "distill": _own_distill}


def run(state):
    return (OWN if own else PLAIN)[state["case"]["op"]](state)


# -------------------------------------------------------------------- work ----

def work(case):
    size = BYTES[case["dtype"]]
    if case["op"] == "rotary":
        values = case["tokens"] * (case["heads"] + case["kv_heads"]) * case["dim"]
        positions = min(case["tokens"], case["sequence"])
        small = positions * case["rotary"] * 4 + case["tokens"] * 8
        if case["mode"] == "forward":
            return {"bytes": 2 * values * size + small, "flops": 7 * values}
        return {"bytes": 4 * values * size + small, "flops": 20 * values}
    if case["op"] == "adapters":
        t, r, k, n = (case[key] for key in ("tokens", "rank", "k", "n"))
        weights = min(case["adapters"], case["requests"]) * r * (k + n)
        if case["mode"] == "forward":
            return {"bytes": (t * k + 2 * t * n + weights) * size, "flops": 2 * t * r * (k + n)}
        # x, base, out, dy and dx once each; the adapters' weights read and their gradients written.
        return {"bytes": (2 * t * k + 3 * t * n + weights + case["adapters"] * r * (k + n)) * size,
                "flops": 6 * t * r * (k + n)}
    values, pairs = case["rows"] * case["vocab"], case["rows"] * min(case["top"], case["vocab"])
    traffic = values * size + pairs * 12
    if case["mode"] == "loss":
        return {"bytes": traffic, "flops": 4 * values}
    return {"bytes": traffic + values * size, "flops": 8 * values}


# ------------------------------------------------------------------- exact ----

def _exact_rotary(s):
    case = s["case"]
    names = ["q", "k"] + (["q_weight", "k_weight"] if case["norm"] else [])
    leaves = {name: s[name].detach().double().requires_grad_(case["mode"] == "train") for name in names}
    half = case["rotary"] // 2
    angles = s["table"].double()[s["positions"]]
    turn = torch.complex(angles[:, :half], angles[:, half:])[:, None, :]
    out = {}
    for name in ("q", "k"):
        x = leaves[name]
        if case["norm"]:
            x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / case["dim"] + EPS) * leaves[name + "_weight"]
        head, rest = x[..., :case["rotary"]], x[..., case["rotary"]:]
        # A pair of elements is one complex number, the rotation a product with e^(i angle).
        pairs = head.unflatten(-1, (half, 2)) if case["interleaved"] else head.unflatten(-1, (2, half)).mT
        z = torch.complex(pairs[..., 0], pairs[..., 1]) * turn
        turned = torch.stack((z.real, z.imag), -1 if case["interleaved"] else -2).flatten(-2)
        out[name] = torch.cat((turned, rest), -1)
    if case["mode"] == "train":
        grads = torch.autograd.grad((out["q"], out["k"]), list(leaves.values()), (s["dq"].double(), s["dk"].double()))
        grads = dict(zip(leaves, grads))
        out = {"q": out["q"].detach(), "k": out["k"].detach()}
        for name in ("q", "k"):
            out["d" + name] = grads[name]
            if case["norm"]:
                out["d" + name + "_weight"] = grads[name + "_weight"]
    return out


def _exact_adapters(s):
    case = s["case"]
    train = case["mode"] == "train"
    out = {"out": s["base"].double()}
    if train:
        out["dx"] = torch.zeros(s["x"].shape, device="cuda", dtype=torch.float64)
        out["da"] = torch.zeros(s["a"].shape, device="cuda", dtype=torch.float64)
        out["db"] = torch.zeros(s["b"].shape, device="cuda", dtype=torch.float64)
    start = 0
    for length, adapter in zip(s["lengths"], s["ids"]):
        rows = slice(start, start + length)
        start += length
        if adapter < 0:
            continue
        a, b, scale = s["a"][adapter].double(), s["b"][adapter].double(), s["scale"][adapter].double()
        x = s["x"][rows].double()
        out["out"][rows] += scale * ((x @ a.T) @ b.T)
        if train:
            dy = s["dy"][rows].double()
            product = scale * (dy @ b)
            out["dx"][rows] = product @ a
            out["da"][adapter] += product.T @ x
            out["db"][adapter] += scale * (dy.T @ (x @ a.T))
    return out


def _exact_distill(s):
    case = s["case"]
    t, rows = case["temperature"], case["rows"]
    losses = torch.zeros(rows, device="cuda", dtype=torch.float64)
    valid = max(1, int((s["indices"] >= 0).any(1).sum()))
    upstream = s["grad_loss"].double() if case["mode"] == "grad" else 1.0 / valid
    grad = None if case["mode"] == "loss" else torch.zeros_like(s["logits"], dtype=torch.float64)
    for first in range(0, rows, 256):
        part = slice(first, min(rows, first + 256))
        logits, indices = s["logits"][part].double() / t, s["indices"][part]
        kept = indices >= 0
        log_q = torch.log_softmax(logits, 1)
        weight = torch.where(kept, torch.exp(s["teacher"][part].double() / t), 0.0)
        some = kept.any(1)
        p = torch.where(some[:, None], weight / weight.sum(1, keepdim=True), 0.0)
        row, column = kept.nonzero(as_tuple=True)
        term = p[row, column] * (p[row, column].log() - log_q[row, indices[row, column]])
        losses[part] = t * t * torch.zeros_like(losses[part]).index_add_(0, row, term)
        if grad is not None:
            slope = log_q.exp() * some[:, None]
            slope.index_put_((row, indices[row, column]), -p[row, column], accumulate=True)
            grad[part] = slope * (t * upstream)
    if case["mode"] == "loss":
        return losses
    return {"loss": losses if case["mode"] == "grad" else losses.sum() / valid, "grad": grad}


EXACT = {"rotary": _exact_rotary, "adapters": _exact_adapters, "distill": _exact_distill}


def exact(case, seed):
    return EXACT[case["op"]](prepare(case, seed))
