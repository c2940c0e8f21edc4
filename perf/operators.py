"""The operators around a GCN's aggregation, as calls with sizes: normalisation between layers, the scores
of the labels, the update of the weights.

``listed()`` names the cases, ``draw(rng)`` gives more of the same ranges, ``prepare`` makes what a program has
in hand before the call, ``run`` is one pass through the operator and ``exact`` the same from the definition in
64 bits.  Where ``own`` is false, ``run`` computes the operator in elementary torch operations.

A case's ``op`` is one of

* ``norm``    group norm with an activation over node features [nodes, channels], statistics per graph and
              group of channels (a batch holds its graphs end to end); with ``backward`` also the gradients of
              the features, the weight and the bias;
* ``labels``  log probability of each node's label, optionally the entropy of its distribution and the ``top``
              likeliest classes with theirs; with ``backward`` also the gradient of the logits;
* ``ortho``   a matrix (or ``batch`` of them) orthogonalised by five Newton-Schulz steps;
* ``muon``    one optimiser step over a list of weights: momentum, Newton-Schulz steps, decay and update.
"""
import torch

own = False

IGNORE = -100
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
NS_STEPS, NS_EPS = 5, 1e-7
NORM_EPS = 1e-5
LR, MOMENTUM, DECAY = 0.02, 0.95, 0.01
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}

# The largest sizes a drawn case may have: those of the largest listed case of its operator.
MOST_FEATURES = 232_965 * 128
MOST_LOGITS = 2_049 * 32_003
MOST_PRODUCTS = 2_048 ** 3


def norm_case(nodes, graphs, channels, groups, act, dtype, backward, name=None):
    c = {"op": "norm", "nodes": nodes, "graphs": graphs, "channels": channels, "groups": groups, "act": act,
         "dtype": dtype, "backward": backward}
    return c if name is None else {"name": name, **c}


def labels_case(rows, classes, dtype, top, entropy, backward, name=None):
    c = {"op": "labels", "rows": rows, "classes": classes, "dtype": dtype, "top": top, "entropy": entropy,
         "backward": backward}
    return c if name is None else {"name": name, **c}


def ortho_case(batch, rows, cols, dtype, name=None):
    c = {"op": "ortho", "batch": batch, "rows": rows, "cols": cols, "dtype": dtype}
    return c if name is None else {"name": name, **c}


def muon_case(weights, name=None):
    c = {"op": "muon", "weights": weights}
    return c if name is None else {"name": name, **c}


def listed():
    return [
        # between the layers of the 2-layer GCN on its 232,965-node graph, in training.  (The gradient of a ReLU
        # jumps at zero, where two roundings of one value differ, so the cases with gradients take a smooth one.)
        norm_case(232_965, 1, 128, 8, "silu", "float32", True, "norm full graph training"),
        # a batch of many small graphs (molecules, ego networks) in mixed precision, in training
        norm_case(100_000, 2_000, 256, 32, "silu", "bfloat16", True, "norm graph batch training"),
        # one small graph answered alone: the time to issue it is what counts
        norm_case(512, 1, 64, 4, "relu", "float32", False, "norm one small graph"),
        # the raw features, 602 wide, in groups of 43: nothing a vector load divides
        norm_case(24_001, 37, 602, 14, "none", "float16", True, "norm odd width training"),
        # the loss of the 2-layer GCN's training epoch: 41 classes, a third of the nodes without a label
        labels_case(232_965, 41, "float32", 0, False, True, "labels full graph training"),
        # answers for every node of the 12,000-node graph: the five likeliest classes and how sure they are
        labels_case(12_000, 41, "float32", 5, True, False, "labels answers"),
        # one node asked for its likeliest partners among all 100,000 nodes
        labels_case(1, 100_000, "float32", 10, True, False, "labels one wide query"),
        # a training step over a wide set of classes (an odd number of them), with an entropy term
        labels_case(2_049, 32_003, "bfloat16", 8, True, True, "labels wide training"),
        # the update of the 2-layer GCN's two weights
        muon_case("128x602,41x128", "muon gcn weights"),
        # the widest hidden layer of the reference's benchmark
        ortho_case(1, 2_048, 2_048, "float32", "ortho widest hidden"),
        # eight layers' gradients of one shape at once, in mixed precision
        ortho_case(8, 512, 1_024, "bfloat16", "ortho batch"),
        # a tall matrix with odd sides
        ortho_case(1, 1_001, 333, "float32", "ortho tall odd"),
    ]


def _log_int(rng, lo, hi):
    hi = max(lo, hi)
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(("norm", "labels", "ortho", "muon"))
    if op == "norm":
        groups = rng.choice((1, 2, 4, 8, 14, 16, 32))
        channels = groups * _log_int(rng, 1, min(86, 1_024 // groups))
        nodes = _log_int(rng, 50, min(232_965, MOST_FEATURES // channels))
        graphs = _log_int(rng, 1, max(1, min(2_000, nodes // 8)))
        backward = rng.random() < 0.6
        act = rng.choice(("none", "silu") if backward else ("none", "relu", "silu"))
        return norm_case(nodes, graphs, channels, groups, act, rng.choice(tuple(DTYPES)), backward)
    if op == "labels":
        classes = _log_int(rng, 2, 100_000)
        rows = _log_int(rng, 1, min(232_965, MOST_LOGITS // classes))
        top = min(classes, rng.choice((0, 0, 1, 5, 8, 10)))
        return labels_case(rows, classes, rng.choice(tuple(DTYPES)), top, rng.random() < 0.5, rng.random() < 0.5)
    if op == "ortho":
        rows, cols = _log_int(rng, 16, 2_048), _log_int(rng, 16, 2_048)
        batch = _log_int(rng, 1, min(8, MOST_PRODUCTS // (rows * cols * min(rows, cols))))
        return ortho_case(batch, rows, cols, rng.choice(tuple(DTYPES)))
    shapes = [(_log_int(rng, 16, 1_024), _log_int(rng, 16, 1_024)) for _ in range(rng.randint(1, 4))]
    return muon_case(",".join("%dx%d" % s for s in shapes))


def _shapes(case):
    return [tuple(int(v) for v in s.split("x")) for s in case["weights"].split(",")]


def work(case):
    """Every input read once, every output written once; the products of a Newton-Schulz step with the symmetric
    ones counted once: X X^T (rows^2 cols), its square (rows^3) and their sum times X (2 rows^2 cols)."""
    if case["op"] == "norm":
        size = case["nodes"] * case["channels"]
        e = torch.finfo(DTYPES[case["dtype"]]).bits // 8
        if not case["backward"]:
            return {"bytes": 2 * size * e + 8 * case["channels"], "flops": 8 * size}
        return {"bytes": 4 * size * e + 16 * case["channels"], "flops": 24 * size}
    if case["op"] == "labels":
        size, rows = case["rows"] * case["classes"], case["rows"]
        e = torch.finfo(DTYPES[case["dtype"]]).bits // 8
        per_row = 8 + 4 + (4 if case["entropy"] else 0) + 12 * case["top"]
        flops = 4 * size
        if case["backward"]:
            per_row += 4 + (4 if case["entropy"] else 0)
            flops += 6 * size
        return {"bytes": size * e * (2 if case["backward"] else 1) + rows * per_row, "flops": flops}
    if case["op"] == "ortho":
        shapes = [(case["rows"], case["cols"])] * case["batch"]
        moved = 2 * torch.finfo(DTYPES[case["dtype"]]).bits // 8
    else:
        shapes, moved = _shapes(case), 20                    # weight and momentum read and written, gradient read
    flops = 0
    for r, c in shapes:
        s, l = min(r, c), max(r, c)
        flops += NS_STEPS * (3 * s * s * l + s ** 3)
    return {"bytes": moved * sum(r * c for r, c in shapes), "flops": flops}


# ---------------------------------------------------------------------------------------- inputs
def _gradient_like(shape, g, dev):
    """A matrix as a layer's weight gradient is: a product over samples, on a floor of noise."""
    *lead, r, c = shape
    k = max(2, min(r, c) // 2)
    a = torch.randn((*lead, r, k), generator=g, device=dev) / k
    b = torch.randn((*lead, k, c), generator=g, device=dev)
    return 1e-3 * (torch.matmul(a, b) + 0.1 * torch.randn((*lead, r, c), generator=g, device=dev))


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev).manual_seed(int(seed))
    state = {"case": case}
    if case["op"] == "norm":
        n, b, ch = case["nodes"], case["graphs"], case["channels"]
        dt = DTYPES[case["dtype"]]
        # graph sizes around n / b: borders of a sorted random draw
        cut = torch.sort(torch.randint(0, n + 1, (b - 1,), generator=g, device=dev)).values
        ptr = torch.cat([cut.new_zeros(1), cut, cut.new_full((1,), n)])
        spread = 0.5 + torch.rand((ch,), generator=g, device=dev)
        centre = torch.randn((ch,), generator=g, device=dev)
        x = (torch.randn((n, ch), generator=g, device=dev) * spread + centre).to(dt)
        w = 1.0 + 0.1 * torch.randn((ch,), generator=g, device=dev)
        bias = 0.1 * torch.randn((ch,), generator=g, device=dev)
        state |= {"x": x, "w": w, "b": bias, "ptr": ptr, "batch": None if b == 1 else
                  torch.repeat_interleave(torch.arange(b, device=dev), ptr[1:] - ptr[:-1], output_size=n)}
        if case["backward"]:
            state["dy"] = torch.randn((n, ch), generator=g, device=dev).to(dt)
        if own:
            from cbm4gnn_amd.norm import GraphBatch
            state["graphs"] = None if b == 1 else GraphBatch(ptr, device=dev)
            for k in ("x", "w", "b"):
                state[k].requires_grad_(case["backward"])
    elif case["op"] == "labels":
        n, ch = case["rows"], case["classes"]
        labels = torch.randint(0, ch, (n,), generator=g, device=dev)
        z = 2.0 * torch.randn((n, ch), generator=g, device=dev)
        z.scatter_add_(1, labels[:, None], 4.0 * torch.rand((n, 1), generator=g, device=dev))
        if case["backward"]:
            labels = torch.where(torch.rand((n,), generator=g, device=dev) < 0.33, IGNORE, labels)
            state["g_logp"] = -(0.5 + torch.rand((n,), generator=g, device=dev)) / n
            state["g_entropy"] = 0.1 * torch.randn((n,), generator=g, device=dev) / n
        state |= {"logits": z.to(DTYPES[case["dtype"]]), "labels": labels}
        if own:
            state["logits"].requires_grad_(case["backward"])
    elif case["op"] == "ortho":
        shape = (case["rows"], case["cols"])
        shape = shape if case["batch"] == 1 else (case["batch"], *shape)
        state["grad"] = _gradient_like(shape, g, dev).to(DTYPES[case["dtype"]])
    else:
        shapes = _shapes(case)
        state["weights"] = [torch.randn(s, generator=g, device=dev) * (2.0 / sum(s)) ** 0.5 for s in shapes]
        state["grads"] = [_gradient_like(s, g, dev) for s in shapes]
        state["buffers"] = [5.0 * _gradient_like(s, g, dev) for s in shapes]
    return state


# ---------------------------------------------------------------------------------------- plain forms
def _per_graph(v, ptr):
    """Sums of the rows of v [nodes, groups] by graph, in 64 bits across rows: [graphs, groups]."""
    if ptr.numel() == 2:
        return v.double().sum(0, keepdim=True)
    upto = torch.cumsum(v.double().t().contiguous(), 1)       # along rows of memory: down the columns it is far slower
    upto = torch.cat([upto.new_zeros((v.size(1), 1)), upto], 1)[:, ptr]
    return (upto[:, 1:] - upto[:, :-1]).t()


def _to_rows(v, batch):
    return v.float()[:, :, None] if batch is None else v.float()[batch][:, :, None]


def _plain_norm(s):
    c = s["case"]
    n, groups, ptr, batch = c["nodes"], c["groups"], s["ptr"], s["batch"]
    x = s["x"].float().view(n, groups, -1)
    count = ((ptr[1:] - ptr[:-1]) * x.size(2)).clamp(min=1).double()[:, None]
    mean = _per_graph(x.sum(2), ptr) / count
    centred = x - _to_rows(mean, batch)
    rstd = torch.rsqrt(_per_graph((centred * centred).sum(2), ptr) / count + NORM_EPS)
    rstd = _to_rows(rstd, batch)
    xhat = centred * rstd
    w, b = s["w"].view(groups, -1), s["b"].view(groups, -1)
    pre = xhat * w + b
    sig = 1.0 / (1.0 + torch.exp(-pre)) if c["act"] == "silu" else None
    y = pre * sig if c["act"] == "silu" else pre.clamp(min=0) if c["act"] == "relu" else pre
    dt = s["x"].dtype
    if not c["backward"]:
        return {"y": y.reshape(n, -1).to(dt)}
    d = s["dy"].float().view(n, groups, -1)
    if c["act"] == "silu":
        d = d * (sig * (1.0 + pre * (1.0 - sig)))
    elif c["act"] == "relu":
        d = d * (pre > 0)
    dw, db = (d * xhat).sum(0).reshape(-1), d.sum(0).reshape(-1)
    dx = d * w
    s1 = _to_rows(_per_graph(dx.sum(2), ptr) / count, batch)
    s2 = _to_rows(_per_graph((dx * xhat).sum(2), ptr) / count, batch)
    dx = rstd * (dx - s1 - xhat * s2)
    return {"y": y.reshape(n, -1).to(dt), "dx": dx.reshape(n, -1).to(dt), "dw": dw, "db": db}


def _plain_top(z, k):
    """The k largest of each row and where they are, ties to the lowest index: the values' bits, made to order as
    whole numbers, above the index counted down, so that no two keys are equal."""
    bits = (z + 0.0).view(torch.int32)
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
    key = (order << 32) | (0xFFFFFFFF - torch.arange(z.size(1), device=z.device))
    index = 0xFFFFFFFF - (key.topk(k, dim=1).values & 0xFFFFFFFF)
    return z.gather(1, index), index


def _plain_labels(s):
    c = s["case"]
    z = s["logits"].float()
    known = s["labels"] != IGNORE
    at = torch.where(known, s["labels"], 0)[:, None]
    top = z.max(1, keepdim=True).values
    shifted = z - top
    e = torch.exp(shifted)
    total = e.sum(1, keepdim=True)
    log_total = torch.log(total)
    out = {"logp": torch.where(known, (shifted.gather(1, at) - log_total)[:, 0], 0.0)}
    p = e / total
    if c["entropy"]:
        entropy = log_total - (p * shifted).sum(1, keepdim=True)
        out["entropy"] = entropy[:, 0]
    if c["top"]:
        value, index = _plain_top(z, c["top"])
        out["top_logp"], out["top_index"] = value - top - log_total, index
    if c["backward"]:
        gl = torch.where(known, s["g_logp"], 0.0)[:, None]
        grad = -gl * p
        if c["entropy"]:
            grad -= s["g_entropy"][:, None] * p * (shifted - log_total + entropy)
        grad.scatter_add_(1, at, gl)
        out["grad"] = grad.to(s["logits"].dtype)
    return out


def _plain_ortho(g):
    x = g.float()
    tall = x.size(-2) > x.size(-1)
    if tall:
        x = x.transpose(-2, -1).contiguous()
    x = x / (torch.sqrt((x * x).sum((-2, -1), keepdim=True)) + NS_EPS)
    a, b, c = COEFFICIENTS
    for _ in range(NS_STEPS):
        gram = torch.matmul(x, x.transpose(-2, -1).contiguous())
        x = a * x + torch.matmul(b * gram + c * torch.matmul(gram, gram), x)
    return (x.transpose(-2, -1) if tall else x).to(g.dtype)


def _plain_muon(s):
    for w, g, buf in zip(s["weights"], s["grads"], s["buffers"]):
        buf.mul_(MOMENTUM).add_(g)
        step = _plain_ortho(g + MOMENTUM * buf)
        w.mul_(1.0 - LR * DECAY).add_(step, alpha=-LR * max(1.0, w.size(0) / w.size(1)) ** 0.5)
    return {"weights": s["weights"], "buffers": s["buffers"]}


# ---------------------------------------------------------------------------------------- the framework's calls
def _own_norm(s):
    from cbm4gnn_amd.norm import group_norm
    c = s["case"]
    y = group_norm(s["x"], c["groups"], s["w"], s["b"], graphs=s["graphs"], eps=NORM_EPS, activation=c["act"])
    if not c["backward"]:
        return {"y": y}
    dx, dw, db = torch.autograd.grad(y, (s["x"], s["w"], s["b"]), s["dy"])
    return {"y": y.detach(), "dx": dx, "dw": dw, "db": db}


def _own_labels(s):
    from cbm4gnn_amd.labels import label_log_probs
    c = s["case"]
    r = label_log_probs(s["logits"], s["labels"], entropy=c["entropy"], top=c["top"], ignore_index=IGNORE)
    out = {"logp": r.logp.detach()}
    if c["entropy"]:
        out["entropy"] = r.entropy.detach()
    if c["top"]:
        out["top_logp"], out["top_index"] = r.top_logp.detach(), r.top_index
    if c["backward"]:
        parts, grads = [r.logp], [s["g_logp"]]
        if c["entropy"]:
            parts.append(r.entropy)
            grads.append(s["g_entropy"])
        out["grad"], = torch.autograd.grad(parts, (s["logits"],), grads)
    return out


def _own_ortho(s):
    from cbm4gnn_amd.optim import orthogonalise
    return {"out": orthogonalise(s["grad"], steps=NS_STEPS, coefficients=COEFFICIENTS, eps=NS_EPS)}


def _own_muon(s):
    from cbm4gnn_amd.optim import muon_step
    muon_step(s["weights"], s["grads"], s["buffers"], lr=LR, momentum=MOMENTUM, weight_decay=DECAY, nesterov=True,
              steps=NS_STEPS, coefficients=COEFFICIENTS, eps=NS_EPS)
    return {"weights": s["weights"], "buffers": s["buffers"]}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"norm": _own_norm, "labels": _own_labels, "ortho": _own_ortho, "muon": _own_muon}[op](state)
    if op == "ortho":
        return {"out": _plain_ortho(state["grad"])}
    return {"norm": _plain_norm, "labels": _plain_labels, "muon": _plain_muon}[op](state)


# ---------------------------------------------------------------------------------------- from the definitions
def _exact_norm(s):
    """Graph by graph in 64 bits, the gradients by differentiating the forward form."""
    c = s["case"]
    x = s["x"].detach().double().requires_grad_(c["backward"])
    w = s["w"].detach().double().requires_grad_(c["backward"])
    b = s["b"].detach().double().requires_grad_(c["backward"])
    borders = s["ptr"].tolist()
    parts = []
    for lo, hi in zip(borders, borders[1:]):
        if hi > lo:
            v = x[lo:hi].reshape(hi - lo, c["groups"], -1)
            var, mean = torch.var_mean(v, (0, 2), correction=0, keepdim=True)
            parts.append(((v - mean) / torch.sqrt(var + NORM_EPS)).reshape(hi - lo, -1))
    y = torch.cat(parts) * w + b
    y = y * torch.sigmoid(y) if c["act"] == "silu" else torch.relu(y) if c["act"] == "relu" else y
    if not c["backward"]:
        return {"y": y}
    dx, dw, db = torch.autograd.grad(y, (x, w, b), s["dy"].double())
    return {"y": y.detach(), "dx": dx, "dw": dw, "db": db}


def _exact_labels(s):
    c = s["case"]
    z = s["logits"].detach().double().requires_grad_(c["backward"])
    logp = torch.log_softmax(z, 1)
    rows = torch.arange(c["rows"], device=z.device)
    known = (s["labels"] != IGNORE).double()
    out = {"logp": logp[rows, s["labels"].clamp(min=0)] * known}
    if c["entropy"]:
        out["entropy"] = -(logp.exp() * logp).sum(1)
    if c["top"]:
        order = torch.sort(s["logits"].detach().double(), dim=1, descending=True, stable=True).indices[:, :c["top"]]
        out["top_logp"], out["top_index"] = logp.detach().gather(1, order), order
    if c["backward"]:
        loss = (out["logp"] * s["g_logp"].double()).sum()
        if c["entropy"]:
            loss = loss + (out["entropy"] * s["g_entropy"].double()).sum()
        grad, = torch.autograd.grad(loss, (z,))
        out = {k: v.detach() for k, v in out.items()}
        out["grad"] = grad
    return out


def _exact_polynomial(m):
    """a X + b (X X^T) X + c (X X^T)^2 X, applied from the side that is longer, in 64 bits."""
    x = m.double()
    x = x / (torch.linalg.matrix_norm(x, keepdim=True) + NS_EPS)
    a, b, c = COEFFICIENTS
    wide = x.shape[-2] <= x.shape[-1]
    for _ in range(NS_STEPS):
        xt = x.mT.contiguous()
        if wide:
            once = (x @ xt) @ x
            x = a * x + b * once + c * ((x @ xt) @ once)
        else:
            once = x @ (xt @ x)
            x = a * x + b * once + c * (once @ (xt @ x))
    return x


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        return _exact_norm(s)
    if case["op"] == "labels":
        return _exact_labels(s)
    if case["op"] == "ortho":
        return {"out": _exact_polynomial(s["grad"])}
    weights, buffers = [], []
    for w, g, buf in zip(s["weights"], s["grads"], s["buffers"]):
        buf = MOMENTUM * buf.double() + g.double()
        step = _exact_polynomial(g.double() + MOMENTUM * buf)
        scale = max(1.0, w.shape[0] / w.shape[1]) ** 0.5
        weights.append((1.0 - LR * DECAY) * w.double() - LR * scale * step)
        buffers.append(buf)
    return {"weights": weights, "buffers": buffers}
