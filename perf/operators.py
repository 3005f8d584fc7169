"""Timed cases of the operators for token and feature models: layer normalisation, embedding
lookup and the distillation loss over a teacher's top logits, each with its gradient.

`listed()` names the cases and `draw(rng)` makes more of the same ranges.  `prepare` makes the
inputs on the GPU, `run` is one pass: in plain torch operations, or, where `own` is true, through
the `cuda` backend's methods on tensors that the backend holds.  `exact` is the same result in
64 bits and `work` the bytes and operations that a pass cannot do without.
"""
import math

import torch

own = False

EPSILON = 1e-5


# ---- cases ---------------------------------------------------------------------------------------
def listed():
    return [
        # one image's pooled feature vector in front of a classifier: a call that is all latency
        {"name": "layer_norm_one_vector", "kind": "layer_norm", "rows": 1, "width": 1024, "half": False, "stats": False},
        # 128 images of 14 x 14 pixels, 512 channels, 16-bit activation storage, a training forward pass
        {"name": "layer_norm_feature_maps_half", "kind": "layer_norm", "rows": 25088, "width": 512, "half": True, "stats": True},
        # the same maps normalised as a whole, 8 images: few rows and a long axis
        {"name": "layer_norm_whole_maps", "kind": "layer_norm", "rows": 8, "width": 100352, "half": False, "stats": True},
        # a training batch of 16 k tokens of a small text model
        {"name": "layer_norm_gradient_tokens", "kind": "layer_norm_backprop", "rows": 16384, "width": 1024, "half": False},
        # odd sizes: no row but the first starts on a 16-byte boundary
        {"name": "layer_norm_gradient_odd_half", "kind": "layer_norm_backprop", "rows": 3137, "width": 1001, "half": True},
        # the next token of 32 sequences
        {"name": "embedding_step_half", "kind": "embedding", "tokens": 32, "vocab": 32000, "width": 768, "storage": "float16"},
        # a long batch from a table that stays in the uint8 weight format
        {"name": "embedding_batch_uint8", "kind": "embedding", "tokens": 32768, "vocab": 50021, "width": 1024, "storage": "uint8"},
        # the table's gradient for a training batch whose tokens follow a Zipf law
        {"name": "embedding_gradient_batch", "kind": "embedding_backprop", "tokens": 16384, "vocab": 32000, "width": 768, "half": False},
        # few tokens, a large table, ragged sizes
        {"name": "embedding_gradient_ragged", "kind": "embedding_backprop", "tokens": 1021, "vocab": 100003, "width": 130, "half": True},
        # a batch of images, 1000 classes, the teacher's five best
        {"name": "distillation_classes", "kind": "distillation", "rows": 128, "classes": 1000, "top": 5, "half": False, "temperature": 2.0},
        # a batch of tokens over a vocabulary, 16-bit logits
        {"name": "distillation_tokens_half", "kind": "distillation", "rows": 8192, "classes": 32000, "top": 64, "half": True, "temperature": 1.0},
        # a handful of rows over a long odd vocabulary
        {"name": "distillation_long_rows", "kind": "distillation", "rows": 7, "classes": 131101, "top": 32, "half": False, "temperature": 4.0},
    ]


def _log_uniform(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def draw(rng):
    kind = rng.choice(["layer_norm", "layer_norm_backprop", "embedding", "embedding_backprop", "distillation"])
    if kind in ("layer_norm", "layer_norm_backprop"):
        width = _log_uniform(rng, 1, 120000)
        if rng.random() < 0.5:
            width = max(8, width // 8 * 8)
        case = {"kind": kind, "rows": _log_uniform(rng, 1, min(100000, (1 << 25) // width)), "width": width,
                "half": rng.random() < 0.4}
        return dict(case, stats=rng.random() < 0.5) if kind == "layer_norm" else case
    if kind in ("embedding", "embedding_backprop"):
        width = _log_uniform(rng, 4, 2048)
        if rng.random() < 0.6:
            width = max(8, width // 8 * 8)
        case = {"kind": kind, "tokens": _log_uniform(rng, 1, min(100000, (1 << 25) // width)),
                "vocab": _log_uniform(rng, 10, min(150000, (1 << 26) // width)), "width": width}
        if kind == "embedding":
            return dict(case, storage=rng.choice(["float32", "float16", "uint8"]))
        return dict(case, half=rng.random() < 0.3)
    classes = _log_uniform(rng, 2, 150000)
    if rng.random() < 0.5:
        classes = max(8, classes // 8 * 8)
    return {"kind": kind, "rows": _log_uniform(rng, 1, min(8192, (1 << 27) // classes)), "classes": classes,
            "top": _log_uniform(rng, 1, min(128, classes)), "half": rng.random() < 0.5,
            "temperature": rng.choice([1.0, 2.0, 4.0])}


# ---- inputs --------------------------------------------------------------------------------------
def _make(case, seed):
    """Every input of the case as a torch tensor on the GPU, from the seed alone."""
    g = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def uniform(*shape):
        return torch.rand(*shape, generator=g, device="cuda", dtype=torch.float64)

    kind = case["kind"]
    kept = torch.float16 if case.get("half") or case.get("storage") == "float16" else torch.float32
    if kind in ("layer_norm", "layer_norm_backprop"):
        rows, width = case["rows"], case["width"]
        x = (normal(rows, width) * 1.5 + normal(rows, 1)).to(kept)
        inputs = {"x": x, "gamma": 1 + 0.1 * normal(width)}
        if kind == "layer_norm":
            return dict(inputs, beta=0.1 * normal(width))
        x = x.double()
        mean = x.mean(-1, keepdim=True)
        rstd = ((x - mean).square().mean(-1, keepdim=True) + EPSILON).rsqrt()
        return dict(inputs, dy=normal(rows, width), stats=torch.cat([mean, rstd], -1).float())
    if kind in ("embedding", "embedding_backprop"):
        tokens, vocab, width = case["tokens"], case["vocab"], case["width"]
        # Zipf: the r-th token's share falls like 1 / r; the batch's last twentieth is padding
        indices = (torch.exp(uniform(tokens) * math.log(vocab)).long() - 1).clamp_(0, vocab - 1)
        indices = indices[torch.randperm(tokens, generator=g, device="cuda")].int()
        indices[tokens - tokens // 20:] = -1
        if kind == "embedding_backprop":
            return {"indices": indices, "dy": normal(tokens, width).to(kept)}
        if case["storage"] == "uint8":
            return {"indices": indices, "table": torch.randint(0, 256, (vocab, width), generator=g, device="cuda", dtype=torch.uint8)}
        return {"indices": indices, "table": normal(vocab, width).to(kept)}
    rows, classes, top = case["rows"], case["classes"], case["top"]
    # a teacher's list: distinct classes, logits in falling order; one row in eight has a shorter
    # list (-1 behind its end) and one row in 64 none at all
    first = (uniform(rows, 1) * classes).long()
    step = 1 + (uniform(rows, 1) * max(1, classes // top - 1)).long()
    indices = (first + step * torch.arange(top, device="cuda")) % classes
    length = torch.full((rows, 1), top, device="cuda", dtype=torch.long)
    length[7::8] = top // 2
    length[63::64] = 0
    indices = torch.where(torch.arange(top, device="cuda") < length, indices, -1).int()
    return {"logits": (2 * normal(rows, classes)).to(kept), "indices": indices,
            "teacher": (3 * normal(rows, top)).sort(-1, descending=True).values.to(kept),
            "dloss": (0.5 + uniform(rows)).float() / rows}


#: of the uint8 tables: w = byte * scale + min
QUANT_SCALE, QUANT_MIN = 0.0173, -2.2


class _Held:
    """The backend's tensors of one state; they go when the state goes."""

    def __init__(self, backend):
        self.backend, self.tensors, self.given = backend, {}, []

    def hold(self, name, x, storage=None):
        if storage == "uint8":
            t = self.backend.registerQuantized(list(x.shape), x.cpu().numpy(), QUANT_SCALE, QUANT_MIN)
        else:
            dtype = {torch.float32: "float32", torch.float16: "float16", torch.int32: "int32"}[x.dtype]
            t = self.backend.registerStored(list(x.shape), dtype)
            if x.numel():
                torch.as_tensor(self.backend.deviceArray(t), device="cuda").copy_(x)
        self.tensors[name] = t

    def give(self, outputs):
        """The results as torch views; those of the pass before are disposed."""
        for t in self.given:
            t.dispose()
        self.given = outputs
        return [torch.as_tensor(self.backend.deviceArray(t), device="cuda") for t in outputs]

    def __del__(self):
        for t in list(self.tensors.values()) + self.given:
            t.dispose()


def prepare(case, seed):
    inputs = _make(case, seed)
    state = {"case": case, "inputs": inputs}
    if own:
        # what a program of the backend has in hand: the same inputs as the backend's tensors
        import tfjs_core_b200 as tf
        if tf.ENGINE.backendName != "cuda":
            assert tf.set_backend("cuda")
        held = _Held(tf.ENGINE.backend)
        for name, x in inputs.items():
            held.hold(name, x, case.get("storage") if name == "table" else None)
        torch.cuda.synchronize()
        state = {"case": case, "held": held}
    return state


# ---- one pass ------------------------------------------------------------------------------------
def _plain_layer_norm(case, x, gamma, beta):
    v = x.float()
    mean = v.mean(-1, keepdim=True)
    centred = v - mean
    rstd = 1 / torch.sqrt((centred * centred).mean(-1, keepdim=True) + EPSILON)
    y = (centred * rstd * gamma + beta).to(x.dtype)
    return [y, torch.cat([mean, rstd], -1)] if case["stats"] else [y]


def _plain_layer_norm_backprop(case, x, gamma, dy, stats):
    mean, rstd = stats[:, :1], stats[:, 1:]
    normed = (x.float() - mean) * rstd
    scaled = dy * gamma
    dx = rstd * (scaled - scaled.mean(-1, keepdim=True) - normed * (scaled * normed).mean(-1, keepdim=True))
    return [dx, (dy * normed).sum(0), dy.sum(0)]


def _plain_embedding(case, indices, table):
    rows = table[indices.clamp(min=0).long()]
    if case["storage"] == "uint8":
        rows = (rows.double() * QUANT_SCALE + QUANT_MIN).float()
    rows = rows.float() * math.sqrt(case["width"])
    out = torch.where((indices >= 0)[:, None], rows, torch.zeros((), device="cuda"))
    return [out.half() if case["storage"] == "float16" else out]


def _plain_embedding_backprop(case, indices, dy):
    there = (indices >= 0)[:, None]
    scaled = torch.where(there, dy.float() * math.sqrt(case["width"]), torch.zeros((), device="cuda"))
    table = torch.zeros(case["vocab"], case["width"], device="cuda")
    return [table.index_add_(0, indices.clamp(min=0).long(), scaled)]


def _plain_distillation(case, logits, indices, teacher, dloss):
    t = case["temperature"]
    z = logits.float() / t
    top = z.max(-1, keepdim=True).values
    log_q = z - (top + (z - top).exp().sum(-1, keepdim=True).log())
    there, at = indices >= 0, indices.clamp(min=0).long()
    u = torch.where(there, teacher.float() / t, torch.full((), -torch.inf, device="cuda"))
    some = there.any(-1, keepdim=True)
    e = (u - torch.where(some, u.max(-1, keepdim=True).values, torch.zeros((), device="cuda"))).exp()
    p = torch.where(some, e / e.sum(-1, keepdim=True), torch.zeros((), device="cuda"))
    terms = torch.where(p > 0, p * (p.log() - log_q.gather(-1, at)), torch.zeros((), device="cuda"))
    loss = t * t * terms.sum(-1)
    difference = log_q.exp() * some
    difference.scatter_add_(-1, at, -p)
    return [loss, difference * (t * dloss)[:, None]]


def _own_layer_norm(bk, case, x, gamma, beta):
    y, stats = bk.layerNorm(x, gamma, beta, EPSILON, case["stats"], "float16" if case["half"] else "float32")
    return [y, stats] if case["stats"] else [y]


def _own_layer_norm_backprop(bk, case, x, gamma, dy, stats):
    return list(bk.layerNormBackprop(dy, x, gamma, stats))


def _own_embedding(bk, case, indices, table):
    return [bk.embeddingLookup(table, indices, math.sqrt(case["width"]),
                               "float16" if case["storage"] == "float16" else "float32")]


def _own_embedding_backprop(bk, case, indices, dy):
    return [bk.embeddingLookupBackprop(dy, indices, case["vocab"], math.sqrt(case["width"]))]


def _own_distillation(bk, case, logits, indices, teacher, dloss):
    loss, stats = bk.distillationLoss(logits, teacher, indices, case["temperature"])
    dlogits = bk.distillationLossBackprop(dloss, logits, teacher, indices, stats, case["temperature"])
    stats.dispose()
    return [loss, dlogits]


_PLAIN = {"layer_norm": _plain_layer_norm, "layer_norm_backprop": _plain_layer_norm_backprop,
          "embedding": _plain_embedding, "embedding_backprop": _plain_embedding_backprop,
          "distillation": _plain_distillation}
_OWN = {"layer_norm": _own_layer_norm, "layer_norm_backprop": _own_layer_norm_backprop,
        "embedding": _own_embedding, "embedding_backprop": _own_embedding_backprop,
        "distillation": _own_distillation}


def run(state):
    case = state["case"]
    if own:
        held = state["held"]
        return held.give(_OWN[case["kind"]](held.backend, case, **held.tensors))
    return _PLAIN[case["kind"]](case, **state["inputs"])


# ---- what a pass needs, and what it returns ------------------------------------------------------
def work(case):
    kind = case["kind"]
    if kind in ("layer_norm", "layer_norm_backprop"):
        rows, width = case["rows"], case["width"]
        size = 2 if case["half"] else 4
        if kind == "layer_norm":
            return {"bytes": 2 * rows * width * size + 8 * width + (8 * rows if case["stats"] else 0), "flops": 8 * rows * width}
        return {"bytes": rows * width * (4 + size + 4) + 12 * width + 8 * rows, "flops": 14 * rows * width}
    if kind == "embedding":
        size = {"float32": 4, "float16": 2, "uint8": 1}[case["storage"]]
        tokens, width = case["tokens"], case["width"]
        # the rows that the tokens name, each once (the expected number for the Zipf law); every output row
        share = math.log(case["vocab"])
        named = sum(-math.expm1(tokens * math.log1p(-min(0.999999, 1 / (share * r)))) for r in range(1, case["vocab"] + 1))
        return {"bytes": 4 * tokens + min(tokens, named) * width * size + tokens * width * (2 if size == 2 else 4),
                "flops": tokens * width}
    if kind == "embedding_backprop":
        tokens, width = case["tokens"], case["width"]
        return {"bytes": 4 * tokens + tokens * width * (2 if case["half"] else 4) + case["vocab"] * width * 4,
                "flops": tokens * width}
    rows, classes, top = case["rows"], case["classes"], case["top"]
    size = 2 if case["half"] else 4
    # the loss and its gradient are two calls: the first ends before the gradient's factor is there
    return {"bytes": rows * classes * (2 * size + 4) + 2 * rows * top * (size + 4) + 8 * rows, "flops": 8 * rows * classes}


def exact(case, seed):
    inputs = {k: v.double() if v.is_floating_point() else v.long() for k, v in _make(case, seed).items()}
    kind = case["kind"]
    if kind == "layer_norm":
        x = inputs["x"]
        var, mean = torch.var_mean(x, -1, correction=0)
        rstd = (var + EPSILON) ** -0.5
        y = torch.addcmul(inputs["beta"], (x - mean[:, None]) * rstd[:, None], inputs["gamma"])
        return [y, torch.stack([mean, rstd], 1)] if case["stats"] else [y]
    if kind == "layer_norm_backprop":
        x, dy, gamma, stats = (inputs[k] for k in ("x", "dy", "gamma", "stats"))
        normed = (x - stats[:, 0, None]) * stats[:, 1, None]
        a, n = dy * gamma, x.shape[1]
        along = torch.einsum("rw,rw->r", a, normed) / n
        dx = (a - a.sum(1, keepdim=True) / n - normed * along[:, None]) * stats[:, 1, None]
        return [dx, torch.einsum("rw,rw->w", dy, normed), torch.einsum("rw->w", dy)]
    if kind == "embedding":
        at, table = inputs["indices"], inputs["table"].double()
        if case["storage"] == "uint8":
            table = table * QUANT_SCALE + QUANT_MIN
        out = torch.zeros(case["tokens"], case["width"], device="cuda", dtype=torch.float64)
        named = at.ge(0).nonzero()[:, 0]
        out[named] = table.index_select(0, at[named]) * case["width"] ** 0.5
        return [out]
    if kind == "embedding_backprop":
        at = inputs["indices"]
        named = at.ge(0).nonzero()[:, 0]
        order = named[at[named].argsort(stable=True)]
        table = torch.zeros(case["vocab"], case["width"], device="cuda", dtype=torch.float64)
        return [table.index_put_((at[order],), inputs["dy"][order] * case["width"] ** 0.5, accumulate=True)]
    t, z, at, u, dloss = (case["temperature"], inputs["logits"], inputs["indices"], inputs["teacher"], inputs["dloss"])
    q = torch.softmax(z / t, -1)
    log_q = torch.log_softmax(z / t, -1)
    p = torch.zeros_like(u)
    some = at.ge(0).any(-1)
    p[some] = torch.softmax((u[some] / t).masked_fill(at[some] < 0, -torch.inf), -1)
    target = torch.zeros_like(q).scatter_add_(-1, at.clamp(min=0), p)
    loss = t * t * (torch.xlogy(p, p).sum(-1) - torch.einsum("rk,rk->r", p, log_q.gather(-1, at.clamp(min=0))))
    q[~some] = 0
    return [loss, (q - target) * (t * dloss)[:, None]]
