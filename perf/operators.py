"""What a node classifier needs around its aggregations: products grouped by node type, layer norm and the class log
probabilities, each with its gradients.

``listed()`` gives the cases, ``draw(rng)`` more of the same ranges, ``prepare`` a case's inputs and buffers, ``run`` one
pass, ``work`` what a pass has to move and compute, ``exact`` the outputs from the definitions in 64 bits.  ``run`` computes
the plain torch form unless ``own`` is set; then it makes the calls that a user makes of this package.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-5

# Bounds of a drawn case: no dearer than the largest listed one.
MAX_ROWS = 2_449_029
MAX_NORM = 100 * 2_449_029              # elements of a normalised matrix
MAX_LOGITS = 47 * 2_449_029             # elements of a logits matrix
MAX_GROUPED = 16_384 * 2048 * 2048      # rows * K * N
MAX_GROUPED_ROWS = 600_000 * 256        # rows * (K + N)
MAX_GROUPED_WEIGHTS = 16 * 2048 * 2048


def _norm(name, op, dtype, n, d, affine=True):
    return {"name": name, "op": op, "dtype": dtype, "n": n, "d": d, "affine": affine}


def _logprob(name, op, dtype, n, c, **more):
    return {"name": name, "op": op, "dtype": dtype, "n": n, "c": c, **more}


def _grouped(name, op, dtype, n, k, m, groups, skew, tail=0):
    return {"name": name, "op": op, "dtype": dtype, "n": n, "k": k, "m": m, "groups": groups, "skew": skew, "tail": tail}


def listed():
    return [
        # the input features of a full products-shaped graph, normalised before the first dense layer
        _norm("norm_forward_full_graph", "norm_forward", "f32", 2_449_029, 100),
        # one small batch of nodes served in 16 bits, at the odd width of Reddit-shaped features: latency
        _norm("norm_forward_small_batch", "norm_forward", "bf16", 97, 602),
        # training on the Reddit-shaped graph: every node's features, the gradient of weight and bias over all rows
        _norm("norm_backward_full_graph", "norm_backward", "f32", 232_965, 602),
        # training at a wide hidden state in 16 bits
        _norm("norm_backward_wide", "norm_backward", "bf16", 8192, 4096),
        # scoring every node of a products-shaped graph (47 classes), with five alternatives
        _logprob("logprob_forward_full_graph", "logprob_forward", "f32", 2_449_029, 47, top=5),
        # a few nodes against a very large label space: few rows, a long axis
        _logprob("logprob_forward_large_label_space", "logprob_forward", "bf16", 64, 100_000, top=8),
        # training on the Reddit-shaped graph (41 classes), two thirds of the nodes labelled
        _logprob("logprob_backward_full_graph", "logprob_backward", "f32", 232_965, 41, entropy=False),
        # training on a large label space in 16 bits with an entropy term
        _logprob("logprob_backward_large_label_space", "logprob_backward", "bf16", 2048, 32_768, entropy=True),
        # hidden update of a graph with four node types of very different sizes, fp32 as the rest of the model
        _grouped("grouped_forward_node_types", "grouped_forward", "f32", 600_000, 128, 128, 4, 1.0),
        # a handful of nodes of eight types through wide weights: every weight is read for a few rows
        _grouped("grouped_forward_few_rows", "grouped_forward", "bf16", 61, 2048, 2048, 8, 1.0),
        # training at odd widths (100 features, 47 classes), five types
        _grouped("grouped_backward_odd_widths", "grouped_backward", "f32", 200_003, 100, 47, 5, 1.0),
        # training at wide layers in 16 bits, sixteen types, some nearly empty
        _grouped("grouped_backward_wide", "grouped_backward", "bf16", 16_384, 2048, 2048, 16, 1.5),
    ]


def _log_uniform(rng, low, high):
    return low if high <= low else min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["norm_forward", "norm_backward", "logprob_forward", "logprob_backward", "grouped_forward", "grouped_backward"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    case = {"op": op, "dtype": dtype}
    if op.startswith("norm"):
        d = _log_uniform(rng, 1, 16_384)
        case.update(n=_log_uniform(rng, 1, min(MAX_ROWS, MAX_NORM // d)), d=d, affine=rng.random() < 0.8)
    elif op.startswith("logprob"):
        c = _log_uniform(rng, 1, 262_144)
        case.update(n=_log_uniform(rng, 1, min(MAX_ROWS, MAX_LOGITS // c)), c=c)
        if op == "logprob_forward":
            case["top"] = min(c, rng.choice([0, 1, 3, 5, 8, 16]))
        else:
            case["entropy"] = rng.random() < 0.5
    else:
        k, m = _log_uniform(rng, 1, 2048), _log_uniform(rng, 1, 2048)
        groups = _log_uniform(rng, 1, min(64, max(1, MAX_GROUPED_WEIGHTS // (k * m))))
        n = _log_uniform(rng, 1, min(600_000, MAX_GROUPED // (k * m), MAX_GROUPED_ROWS // (k + m)))
        case.update(n=n, k=k, m=m, groups=groups, skew=rng.choice([0.0, 0.7, 1.5]), tail=rng.choice([0, 0, min(n // 2, 37)]))
    return case


def _sizes(case, seed):
    """Rows of each type: shares that fall like 1 / rank^skew in a shuffled order, rounded down; what is left over goes to
    the largest.  With a strong skew and few rows some types have none."""
    rows, groups = case["n"] - case["tail"], case["groups"]
    share = (torch.arange(1, groups + 1, dtype=torch.float64)) ** -case["skew"]
    share = share[torch.randperm(groups, generator=torch.Generator().manual_seed(seed))]
    sizes = (share / share.sum() * rows).floor().long()
    sizes[share.argmax()] += rows - sizes.sum()
    return sizes.tolist()


def _logits(g, n, c, dtype):
    """Scores of spread 3 around a row's own offset; one class in 50 is masked out with -inf, but never class 0."""
    z = torch.randn(n, c, device="cuda", generator=g) * 3.0 + torch.randn(n, 1, device="cuda", generator=g) * 5.0
    if c > 1:
        z[:, 1:].masked_fill_(torch.rand(n, c - 1, device="cuda", generator=g) < 0.02, -math.inf)
    return z.to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t, n = DTYPES[case["dtype"]], case["n"]
    f32 = dict(device="cuda", dtype=torch.float32)
    s = {"op": case["op"]}
    if case["op"].startswith("norm"):
        d = case["d"]
        # features of different offsets and spreads; one row in 64 is all zeros (a node without any)
        x = torch.randn(n, d, generator=g, **f32) * (0.5 + torch.rand(n, 1, generator=g, **f32)) + torch.randn(n, 1, generator=g, **f32)
        x *= (torch.rand(n, 1, generator=g, **f32) >= 1 / 64).float()
        s["x"] = x.to(t)
        s["weight"] = 1.0 + 0.1 * torch.randn(d, generator=g, **f32) if case["affine"] else None
        s["bias"] = 0.1 * torch.randn(d, generator=g, **f32) if case["affine"] else None
        if case["op"] == "norm_forward":
            s.update(out=torch.empty_like(s["x"]), mean=torch.empty(n, **f32), rstd=torch.empty(n, **f32))
        else:
            s["dy"] = torch.randn(n, d, generator=g, **f32).to(t)
            x = s["x"].float()
            s["mean"] = x.mean(1)
            s["rstd"] = (x.var(1, unbiased=False) + EPS).rsqrt()
            s["dx"] = torch.empty_like(s["x"])
            s["dweight"] = torch.empty(d, **f32) if case["affine"] else None
            s["dbias"] = torch.empty(d, **f32) if case["affine"] else None
    elif case["op"].startswith("logprob"):
        c = case["c"]
        z = s["logits"] = _logits(g, n, c, t)
        s["labels"] = torch.randint(0, c, (n,), device="cuda", generator=g, dtype=torch.int32)
        s["labels"][torch.rand(n, generator=g, **f32) < 1 / 3] = -1          # nodes without a label
        if case["op"] == "logprob_forward":
            k = s["top"] = case["top"]
            s.update(logprob=torch.empty(n, **f32), stats=torch.empty(n, 2, **f32), entropy=torch.empty(n, **f32))
            s["top_ids"] = torch.empty(n, k, device="cuda", dtype=torch.int32) if k else None
            s["top_logprobs"] = torch.empty(n, k, **f32) if k else None
        else:
            m = z.float().amax(1, keepdim=True)
            e = (z.float() - m).exp()
            total = e.sum(1, keepdim=True)
            s["stats"] = torch.cat([m, total.log()], 1)
            s["dlogprob"] = -torch.rand(n, generator=g, **f32) / n             # what a weighted mean of -logprob hands back
            s["entropy"] = s["dentropy"] = None
            if case["entropy"]:
                s["entropy"] = (total.log() - (e * (z.float() - m).clamp(min=-1e30)).sum(1, keepdim=True) / total)[:, 0].contiguous()
                s["dentropy"] = 0.01 * torch.rand(n, generator=g, **f32) / n
            s["dlogits"] = torch.empty_like(z)
    else:
        k, m, groups = case["k"], case["m"], case["groups"]
        s["sizes"] = _sizes(case, seed)
        s["tail"] = case["tail"]
        s["group_ptr"] = torch.tensor([0] + s["sizes"]).cumsum(0).to(device="cuda", dtype=torch.int32)
        s["x"] = torch.randn(n, k, generator=g, **f32).to(t)
        s["w"] = (torch.randn(groups, k, m, generator=g, **f32) / math.sqrt(k)).to(t)
        if case["op"] == "grouped_forward":
            s["out"] = torch.zeros(n, m, device="cuda", dtype=t)
        else:
            s["dy"] = torch.randn(n, m, generator=g, **f32).to(t)
            s["dx"] = torch.zeros(n, k, device="cuda", dtype=t)
            s["dw"] = torch.empty(groups, k, m, **f32)
    return s


def _take(values, labels):
    """values[i, labels[i]], and 0 for a row without a label."""
    has = labels >= 0
    return torch.where(has, values.gather(1, labels.clamp(min=0).long()[:, None])[:, 0], 0.0)


def _top(z, k):
    """The k largest values' classes, largest first, equal values by class: unique keys of the value's order and the class."""
    bits = (z + 0.0).view(torch.int32)                                          # + 0.0: -0 counts as 0
    order = bits ^ ((bits >> 31) & 0x7FFFFFFF)
    key = (order.long() << 32) | (0xFFFFFFFF - torch.arange(z.shape[1], device=z.device))
    return (0xFFFFFFFF - (key.topk(k, dim=1).values & 0xFFFFFFFF)).int()


def _plain(s):
    op = s["op"]
    if op == "norm_forward":
        x = s["x"].float()
        mean = x.mean(1, keepdim=True)
        c = x - mean
        rstd = ((c * c).mean(1, keepdim=True) + EPS).rsqrt()
        y = c * rstd
        if s["weight"] is not None:
            y = y * s["weight"] + s["bias"]
        return {"out": y.to(s["x"].dtype), "mean": mean[:, 0], "rstd": rstd[:, 0]}
    if op == "norm_backward":
        dy = s["dy"].float()
        xhat = (s["x"].float() - s["mean"][:, None]) * s["rstd"][:, None]
        gr = dy * s["weight"] if s["weight"] is not None else dy
        dx = (gr - gr.mean(1, keepdim=True) - xhat * (gr * xhat).mean(1, keepdim=True)) * s["rstd"][:, None]
        out = {"dx": dx.to(s["x"].dtype)}
        if s["weight"] is not None:
            out.update(dweight=(dy * xhat).sum(0), dbias=dy.sum(0))
        return out
    if op == "logprob_forward":
        z = s["logits"].float()
        m = z.amax(1, keepdim=True)
        d = z - m
        e = d.exp()
        total = e.sum(1, keepdim=True)
        logsum = total.log()
        entropy = logsum - torch.where(e > 0, e * d, 0.0).sum(1, keepdim=True) / total
        out = {"logprob": _take(d - logsum, s["labels"]), "stats": torch.cat([m, logsum], 1), "entropy": entropy[:, 0]}
        if s["top"]:
            ids = _top(z, s["top"])
            out.update(top_ids=ids, top_logprobs=(d - logsum).gather(1, ids.long()))
        return out
    if op == "logprob_backward":
        logp = s["logits"].float() - s["stats"][:, :1] - s["stats"][:, 1:]
        p = logp.exp()
        has = s["labels"] >= 0
        up = torch.where(has, s["dlogprob"], 0.0)[:, None]
        dz = -up * p
        dz.scatter_add_(1, s["labels"].clamp(min=0).long()[:, None], up)
        if s["dentropy"] is not None:
            dz = dz - s["dentropy"][:, None] * p * torch.where(p > 0, logp + s["entropy"][:, None], 0.0)
        return {"dlogits": dz.to(s["logits"].dtype)}
    rows = s["sizes"] + [s["tail"]]
    t = s["x"].dtype
    x, w = s["x"].float(), s["w"].float()
    if op == "grouped_forward":
        parts = [a @ b for a, b in zip(x.split(rows), w)]
        return {"out": torch.cat(parts + [x.new_zeros(s["tail"], w.shape[2])]).to(t)}
    dy = s["dy"].float()
    dx = torch.cat([a @ b.T for a, b in zip(dy.split(rows), w)] + [x.new_zeros(s["tail"], w.shape[1])])
    return {"dx": dx.to(t), "dw": torch.stack([a.T @ b for a, b, _ in zip(x.split(rows), dy.split(rows), w)])}


def _framework(s):
    import mgg_osdi23_b200 as mgg
    op = s["op"]
    if op == "norm_forward":
        mgg.layer_norm_forward(s["out"], s["x"], s["weight"], s["bias"], EPS, mean=s["mean"], rstd=s["rstd"])
        return {k: s[k] for k in ("out", "mean", "rstd")}
    if op == "norm_backward":
        mgg.layer_norm_backward(s["dx"], s["dy"], s["x"], s["mean"], s["rstd"], s["weight"], dweight=s["dweight"], dbias=s["dbias"])
        return {k: s[k] for k in ("dx", "dweight", "dbias") if s[k] is not None}
    if op == "logprob_forward":
        mgg.class_logprob_forward(s["logprob"], s["logits"], s["labels"], stats=s["stats"], entropy=s["entropy"],
                                  top_ids=s["top_ids"], top_logprobs=s["top_logprobs"])
        return {k: s[k] for k in ("logprob", "stats", "entropy", "top_ids", "top_logprobs") if s[k] is not None}
    if op == "logprob_backward":
        mgg.class_logprob_backward(s["dlogits"], s["logits"], s["labels"], s["stats"], s["dlogprob"],
                                   entropy=s["entropy"], dentropy=s["dentropy"])
        return {"dlogits": s["dlogits"]}
    if op == "grouped_forward":
        mgg.grouped_dense_forward(s["out"], s["x"], s["w"], s["group_ptr"])
        return {"out": s["out"]}
    mgg.grouped_dense_backward(s["dx"], s["dw"], s["dy"], s["x"], s["w"], s["group_ptr"])
    return {"dx": s["dx"], "dw": s["dw"]}


def run(state):
    return _framework(state) if own else _plain(state)


def work(case):
    b, n = BYTES[case["dtype"]], case["n"]
    if case["op"].startswith("norm"):
        e = n * case["d"]
        if case["op"] == "norm_forward":
            return {"bytes": 2 * b * e + 8 * n + (8 * case["d"] if case["affine"] else 0), "flops": 8 * e}
        return {"bytes": 3 * b * e + 8 * n + (12 * case["d"] if case["affine"] else 0), "flops": 14 * e}
    if case["op"].startswith("logprob"):
        e = n * case["c"]
        if case["op"] == "logprob_forward":
            return {"bytes": b * e + 20 * n + 8 * n * case["top"], "flops": 6 * e}
        return {"bytes": 2 * b * e + 16 * n + (8 * n if case["entropy"] else 0), "flops": (8 if case["entropy"] else 5) * e}
    rows, k, m = n - case["tail"], case["k"], case["m"]
    weights = case["groups"] * k * m
    if case["op"] == "grouped_forward":
        return {"bytes": b * (rows * (k + m) + weights) + 4 * case["groups"] + 4, "flops": 2 * rows * k * m}
    return {"bytes": b * (rows * (2 * k + m) + weights) + 4 * weights + 4 * case["groups"] + 4, "flops": 4 * rows * k * m}


def exact(case, seed):
    s = prepare(case, seed)
    f64 = torch.float64
    if case["op"].startswith("norm"):
        x = s["x"].to(f64)
        one = torch.ones(case["d"], device="cuda", dtype=f64)
        w = s["weight"].to(f64) if case["affine"] else one
        if case["op"] == "norm_forward":
            var, mean = torch.var_mean(x, dim=1, correction=0)
            rstd = 1.0 / torch.sqrt(var + EPS)
            b = s["bias"].to(f64) if case["affine"] else 0.0 * one
            return {"out": torch.addcmul(b, (x - mean.unsqueeze(1)) / torch.sqrt(var + EPS).unsqueeze(1), w), "mean": mean, "rstd": rstd}
        # of the statistics that were handed in, as the gradient of y with mean and rstd functions of x
        dy, r = s["dy"].to(f64), s["rstd"].to(f64).unsqueeze(1)
        xhat = x.sub_(s["mean"].to(f64).unsqueeze(1)).mul_(r)
        out = {}
        if case["affine"]:
            out = {"dweight": torch.einsum("nd,nd->d", dy, xhat), "dbias": torch.einsum("nd->d", dy)}
        gr = dy.mul_(w)
        a = torch.einsum("nd->n", gr) / case["d"]
        c = torch.einsum("nd,nd->n", gr, xhat) / case["d"]
        return {"dx": gr.sub_(a.unsqueeze(1)).sub_(xhat.mul_(c.unsqueeze(1))).mul_(r), **out}
    if case["op"].startswith("logprob"):
        z = s["logits"].to(f64)
        rows = torch.arange(case["n"], device="cuda")
        y = s["labels"].long()
        if case["op"] == "logprob_forward":
            lse = torch.logsumexp(z, dim=1)
            lp = z - lse.unsqueeze(1)
            m = z.max(dim=1).values
            out = {"logprob": torch.where(y < 0, torch.zeros_like(m), lp[rows, y.clamp(min=0)]), "stats": torch.stack([m, lse - m], dim=1),
                   "entropy": torch.special.entr(lp.exp()).sum(dim=1)}
            if case["top"]:
                ids = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :case["top"]]
                out.update(top_ids=ids.int(), top_logprobs=torch.take_along_dim(lp, ids, dim=1))
            return out
        p = torch.softmax(z, dim=1)
        up = torch.where(y < 0, torch.zeros(1, device="cuda", dtype=f64), s["dlogprob"].to(f64))
        dz = p * -up.unsqueeze(1)
        dz[rows, y.clamp(min=0)] += up
        if case["entropy"]:
            h = torch.special.entr(p)
            # dH/dz_c = p_c (-log p_c) - p_c H
            dz += s["dentropy"].to(f64).unsqueeze(1) * (h - p * h.sum(dim=1, keepdim=True))
        return {"dlogits": dz}
    ends = s["group_ptr"].tolist()
    x, w = s["x"].to(f64), s["w"].to(f64)
    if case["op"] == "grouped_forward":
        out = torch.zeros(case["n"], case["m"], device="cuda", dtype=f64)
        for i in range(case["groups"]):
            out[ends[i]:ends[i + 1]] = torch.matmul(x[ends[i]:ends[i + 1]], w[i])
        return {"out": out}
    dy = s["dy"].to(f64)
    dx = torch.zeros(case["n"], case["k"], device="cuda", dtype=f64)
    dw = torch.zeros(case["groups"], case["k"], case["m"], device="cuda", dtype=f64)
    for i in range(case["groups"]):
        rows = slice(ends[i], ends[i + 1])
        dx[rows] = torch.einsum("nm,km->nk", dy[rows], w[i])
        dw[i] = torch.einsum("nk,nm->km", x[rows], dy[rows])
    return {"dx": dx, "dw": dw}
