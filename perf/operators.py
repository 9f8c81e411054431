"""Cases for measuring the fine-tune-and-serve operators of this package.

Four operators that one program uses together: the token rows of a table with a scale and their
gradient (`embedding_lookup`), the paired log-ratio preference loss (`preference_loss`), the global
gradient norm with clipping (`clip_grad_norm`), and the scores of a 4-bit document index
(`int4_scores`).  `run` computes each either in its plain form (elementary torch operations) or,
where `own` is true, through the package's entry points.
"""
import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------------------------------------
# cases
def listed():
    return [
        # one tokenised query against the 50k-row table, forward only: the latency of a single request
        {"name": "lookup one query", "op": "lookup", "V": 50_000, "E": 128, "B": 1, "L": 64, "dtype": "bf16",
         "ids": "int32", "scale": 1.0, "pad": 0, "train": False},
        # a training batch of queries at the 200k x 256 table: text-like (Zipf) ids, about half the
        # slots padding, forward and dense table gradient
        {"name": "lookup train batch", "op": "lookup", "V": 200_000, "E": 256, "B": 8192, "L": 64, "dtype": "fp32",
         "ids": "int64", "scale": 16.0, "pad": 0, "train": True},
        # an odd width, an odd batch, no padding id, half precision, as a last batch of an epoch has it
        {"name": "lookup ragged", "op": "lookup", "V": 30_011, "E": 100, "B": 37, "L": 29, "dtype": "fp16",
         "ids": "int32", "scale": 10.0, "pad": -1, "train": True},
        # the character tower's batch: 64 pairs of width 128, no reference model
        {"name": "preference small batch", "op": "preference", "B": 64, "H": 128, "K": 1, "dtype": "fp32", "ref": False,
         "mask": 0.0, "beta": 1.0, "temperature": 0.1, "smooth": 0.0, "kind": "sigmoid"},
        # the full training batch, one negative each, against a frozen reference model's margins
        {"name": "preference batch", "op": "preference", "B": 8192, "H": 256, "K": 1, "dtype": "fp32", "ref": True,
         "mask": 0.0, "beta": 0.5, "temperature": 0.1, "smooth": 0.1, "kind": "sigmoid"},
        # four negatives a query, some missing (ragged preference data), bf16 tower outputs
        {"name": "preference 4 negatives", "op": "preference", "B": 8192, "H": 256, "K": 4, "dtype": "bf16", "ref": True,
         "mask": 0.3, "beta": 0.5, "temperature": 0.1, "smooth": 0.0, "kind": "squared"},
        # the tied tower head's four gradients: the smallest clip of a step
        {"name": "clip tower head", "op": "clip", "sizes": "65536,256,65536,256", "dtype": "fp32", "out": "fp32",
         "max_norm": 1.0, "norm": 2.0},
        # the same with the dense gradient of the 200k x 256 table
        {"name": "clip table and head", "op": "clip", "sizes": "51200000,65536,256,65536,256", "dtype": "fp32",
         "out": "fp32", "max_norm": 1.0, "norm": 2.0},
        # many tensors of odd sizes and mixed types (accumulated half-precision gradients), clipped
        # into the fp32 gradients that the optimizer steps with
        {"name": "clip many mixed", "op": "clip", "sizes": "ragged 150 12000000 5", "dtype": "mixed", "out": "fp32",
         "max_norm": 1.0, "norm": 2.0},
        # one query over a million documents
        {"name": "index one query 1M", "op": "int4", "n": 1_000_000, "H": 256, "group": 32, "nq": 1, "qdtype": "fp32"},
        # a small batch of queries over 200k documents of the 128-wide tower
        {"name": "index 8 queries 200k", "op": "int4", "n": 200_000, "H": 128, "group": 64, "nq": 8, "qdtype": "fp32"},
        # an odd width whose last group is short, an odd number of documents, a larger query batch
        {"name": "index odd 33 queries", "op": "int4", "n": 28_834, "H": 100, "group": 64, "nq": 33, "qdtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["lookup", "preference", "clip", "int4"])
    if op == "lookup":
        E = rng.choice([rng.randint(1, 512), 8 * rng.randint(1, 64), rng.choice([64, 128, 256, 512])])
        V = _log(rng, 33, min(200_000, 50_000_000 // E))
        L = _log(rng, 1, 64)
        return {"op": op, "V": V, "E": E, "B": _log(rng, 1, max(2, min(8192, 100_000_000 // (E * L)))), "L": L,
                "dtype": rng.choice(list(DTYPES)), "ids": rng.choice(["int32", "int64"]),
                "scale": rng.choice([1.0, math.sqrt(E), rng.uniform(0.1, 4.0)]), "pad": rng.choice([0, -1]),
                "train": rng.random() < 0.7}
    if op == "preference":
        H = rng.choice([rng.randint(1, 512), 8 * rng.randint(1, 64), rng.choice([64, 128, 256])])
        K = rng.choice([1, 1, 2, 3, 4, rng.randint(5, 8)])
        return {"op": op, "B": _log(rng, 1, min(16384, 10_000_000 // (H * K))), "H": H, "K": K,
                "dtype": rng.choice(list(DTYPES)), "ref": rng.random() < 0.5, "mask": rng.choice([0.0, 0.3, 0.8]),
                "beta": rng.choice([0.1, 0.5, 1.0]), "temperature": rng.choice([0.05, 0.1, 1.0]),
                "smooth": rng.choice([0.0, 0.1]), "kind": rng.choice(["sigmoid", "squared"])}
    if op == "clip":
        count = _log(rng, 1, 200)
        total = _log(rng, 4 * count, 40_000_000)
        dtype = rng.choice(["fp32", "fp32", "bf16", "fp16", "mixed"])
        return {"op": op, "sizes": f"ragged {count} {total} {rng.randrange(1000)}", "dtype": dtype,
                "out": "fp32" if dtype == "mixed" else rng.choice([dtype, "fp32"]),
                "max_norm": rng.choice([0.1, 1.0, 1e5]), "norm": rng.choice([2.0, 2.0, math.inf])}
    H = rng.choice([rng.randint(1, 512), 32 * rng.randint(1, 32), rng.choice([64, 128, 256])])
    n = _log(rng, 1, 200_000_000 // max(H, 200))
    return {"op": op, "n": n, "H": H, "group": rng.choice([32, 64, 128]),
            "nq": _log(rng, 1, max(1, min(64, 16_000_000 // n))), "qdtype": rng.choice(list(DTYPES))}


def _sizes(case):
    text = case["sizes"]
    if not text.startswith("ragged"):
        return [int(s) for s in text.split(",")]
    count, total, seed = (int(s) for s in text.split()[1:])
    r = random.Random(seed)  # a few large tensors and many small ones
    share = [r.random() ** 4 + 1e-4 for _ in range(count)]
    whole = sum(share)
    return [max(1, int(total * s / whole)) for s in share]


def _clip_types(case):
    n = len(_sizes(case))
    kinds = ["bf16", "fp32", "fp16"] if case["dtype"] == "mixed" else [case["dtype"]]
    return [DTYPES[kinds[i % len(kinds)]] for i in range(n)]


# ------------------------------------------------------------------------------------------------
# inputs
def _inputs(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    def rand(*shape):
        return torch.rand(*shape, generator=g, device=DEV)

    op = case["op"]
    if op == "lookup":
        V, E, B, L, dt = case["V"], case["E"], case["B"], case["L"], DTYPES[case["dtype"]]
        ids = (float(V) ** rand(B, L)).long().clamp_(0, V - 1)  # p(id) ~ 1 / id: text-like
        if case["pad"] >= 0:  # sequences of 1..L tokens, the rest padding
            length = 1 + (rand(B, 1) * L).long()
            ids = torch.where(torch.arange(L, device=DEV) < length, ids, torch.full_like(ids, case["pad"]))
        s = {"weight": (randn(V, E) * E ** -0.5).to(dt), "ids": ids.to(getattr(torch, case["ids"]))}
        if case["train"]:
            s["dout"] = (randn(B, L, E) * 0.1).to(dt)
        return s
    if op == "preference":
        B, H, K, dt = case["B"], case["H"], case["K"], DTYPES[case["dtype"]]
        q, p, n = (torch.nn.functional.normalize(x, dim=-1) for x in (randn(B, H), randn(B, H), randn(B, K, H)))
        p = torch.nn.functional.normalize(p + 0.5 * q, dim=-1)  # positives lean to their queries
        s = {"q": q.to(dt), "p": p.to(dt), "n": n.to(dt), "ref": None, "mask": None}
        if case["ref"]:
            s["ref"] = randn(B, K) + 2.0
        if case["mask"]:
            s["mask"] = rand(B, K) >= case["mask"]
        return s
    if op == "clip":
        scale = torch.pow(10.0, -3.0 * rand(len(_sizes(case)))).tolist()
        return {"grads": [(randn(n) * a).to(dt) for n, a, dt in zip(_sizes(case), scale, _clip_types(case))]}
    n, H, group = case["n"], case["H"], case["group"]
    codes = (randn(n, H) * 2.5).round_().clamp_(-8, 7).to(torch.int8)
    scales = ((0.5 + rand(n, -(-H // group))) * (0.4 * H ** -0.5)).to(torch.bfloat16)
    q = torch.nn.functional.normalize(randn(case["nq"], H), dim=-1).to(DTYPES[case["qdtype"]])
    return {"codes": codes, "scales": scales, "q": q}


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    op = case["op"]
    if op == "lookup" and case["train"]:
        s["weight"].requires_grad_(True)
    elif op == "preference":
        for k in ("q", "p", "n"):
            s[k].requires_grad_(True)
    elif op == "clip":  # the optimizer's gradients: views of one flat buffer, in the parameters' order
        s["flat"] = torch.zeros(sum(_sizes(case)), dtype=DTYPES[case["out"]], device=DEV)
        s["out"] = list(torch.split(s["flat"], _sizes(case)))
    elif op == "int4":
        codes = s.pop("codes")
        if own:
            from twotower_amd import ops

            s["index"] = ops.Int4Rows.from_codes(codes, s.pop("scales"), case["group"])
        else:  # two codes to a byte, the even column low
            u = torch.nn.functional.pad((codes + 8).to(torch.uint8), (0, codes.shape[1] % 2))
            s["packed"] = u[:, 0::2] | (u[:, 1::2] << 4)
    return s


# ------------------------------------------------------------------------------------------------
# one pass
def run(state):
    return {"lookup": _lookup, "preference": _preference, "clip": _clip, "int4": _int4}[state["case"]["op"]](state)


def _lookup(s):
    c, w, ids = s["case"], s["weight"], s["ids"]
    pad = c["pad"] if c["pad"] >= 0 else None
    if own:
        from twotower_amd import ops

        out = ops.embedding_lookup(w, ids, scale=c["scale"], padding_idx=pad)
        return [out, torch.autograd.grad(out, w, s["dout"])[0]] if c["train"] else [out]
    w = w.detach()
    ids = ids.long()
    out = (w[ids].float() * c["scale"]).to(w.dtype)
    if not c["train"]:
        return [out]
    d = s["dout"].float() * c["scale"]
    if pad is not None:
        d = d * (ids != pad).unsqueeze(-1)
    grad = torch.zeros(w.shape, dtype=torch.float32, device=w.device).index_add_(0, ids.reshape(-1), d.reshape(-1, w.shape[1]))
    return [out, grad.to(w.dtype)]


def _preference(s):
    c = s["case"]
    if own:
        from twotower_amd import losses

        smooth = c["smooth"] if c["kind"] == "sigmoid" else 0.0  # (the squared loss has none, and refuses it)
        loss = losses.preference_loss(s["q"], s["p"], s["n"], ref_margin=s["ref"], mask=s["mask"], beta=c["beta"],
                                      temperature=c["temperature"], label_smoothing=smooth, loss_type=c["kind"])
        return [loss, *torch.autograd.grad(loss, (s["q"], s["p"], s["n"]))]
    q, p, n = (s[k].detach().float() for k in ("q", "p", "n"))
    h = ((q * p).sum(-1, keepdim=True) - (q.unsqueeze(1) * n).sum(-1)) / c["temperature"]
    if s["ref"] is not None:
        h = h - s["ref"]
    b = c["beta"]
    if c["kind"] == "sigmoid":
        e = c["smooth"]
        x = b * h
        tail = torch.log1p(torch.exp(-x.abs()))  # softplus(+-x) = max(+-x, 0) + tail
        row = (1 - e) * ((-x).clamp(min=0) + tail) + e * (x.clamp(min=0) + tail)
        g = b * (torch.sigmoid(x) - (1 - e))
    else:
        row = (h - 0.5 / b).square()
        g = 2 * (h - 0.5 / b)
    if s["mask"] is not None:
        count = s["mask"].sum().clamp(min=1)
        row, g = row * s["mask"], g * s["mask"]
    else:
        count = row.numel()
    g = g / (count * c["temperature"])
    dq = g.sum(1, keepdim=True) * p - (g.unsqueeze(-1) * n).sum(1)
    dp = g.sum(1, keepdim=True) * q
    dn = -g.unsqueeze(-1) * q.unsqueeze(1)
    return [row.sum() / count, *(t.to(s["q"].dtype) for t in (dq, dp, dn))]


def _clip(s):
    c = s["case"]
    if own:
        from twotower_amd import ops

        norm = ops.clip_grad_norm(s["grads"], c["max_norm"], norm_type=c["norm"], out=s["out"])
        return [norm, s["flat"]]
    if c["norm"] == 2.0:
        norm = torch.stack([g.float().square().sum() for g in s["grads"]]).sum().sqrt()
    else:
        norm = torch.stack([g.float().abs().max() for g in s["grads"]]).max()
    coef = (c["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    [o.copy_(g.float() * coef) for o, g in zip(s["out"], s["grads"])]
    return [norm, s["flat"]]


def _int4(s):
    c = s["case"]
    if own:
        from twotower_amd import ops

        return [ops.int4_scores(s["q"], s["index"])]
    u = torch.stack([s["packed"] & 15, s["packed"] >> 4], dim=-1).flatten(1)[:, :c["H"]]
    rows = (u.float() - 8.0) * s["scales"].float().repeat_interleave(c["group"], dim=1)[:, :c["H"]]
    return [s["q"].float() @ rows.t()]


# ------------------------------------------------------------------------------------------------
# what a pass cannot do without
def work(case):
    op = case["op"]
    if op == "lookup":
        e = 4 if case["dtype"] == "fp32" else 2
        tok, row = case["B"] * case["L"], case["E"] * e
        ids = tok * (4 if case["ids"] == "int32" else 8)
        b, f = ids + min(case["V"], tok) * row + tok * row, tok * case["E"]
        if case["train"]:
            b, f = b + tok * row + case["V"] * row, f + 2 * tok * case["E"]
        return {"bytes": b, "flops": f}
    if op == "preference":
        e = 4 if case["dtype"] == "fp32" else 2
        B, H, K = case["B"], case["H"], case["K"]
        b = 2 * B * (2 + K) * H * e + (B * K * 4 if case["ref"] else 0) + (B * K if case["mask"] else 0)
        return {"bytes": b, "flops": B * H * (2 + 5 * K + 2)}
    if op == "clip":
        o = 4 if case["out"] == "fp32" else 2
        b = sum(n * ((4 if t == torch.float32 else 2) + o) for n, t in zip(_sizes(case), _clip_types(case)))
        return {"bytes": b, "flops": 3 * sum(_sizes(case))}
    n, H, nq = case["n"], case["H"], case["nq"]
    b = n * (-(-H // 2) + 2 * -(-H // case["group"])) + nq * H * (4 if case["qdtype"] == "fp32" else 2) + n * nq * 4
    return {"bytes": b, "flops": 2 * n * H * nq}


# ------------------------------------------------------------------------------------------------
# the definitions in 64 bits
def exact(case, seed):
    s = _inputs(case, seed)
    op = case["op"]
    if op == "lookup":
        w, ids = s["weight"].double(), s["ids"].long().reshape(-1)
        out = torch.index_select(w, 0, ids).mul_(case["scale"]).reshape(*s["ids"].shape, -1)
        if not case["train"]:
            return [out]
        keep = ids != case["pad"]
        grad = torch.zeros_like(w).index_put_((ids[keep],), s["dout"].reshape(ids.numel(), -1)[keep].double(), accumulate=True)
        return [out, grad.mul_(case["scale"])]
    if op == "preference":
        q, p, n = (s[k].double().requires_grad_(True) for k in ("q", "p", "n"))
        h = torch.einsum("bkh,bh->bk", p.unsqueeze(1) - n, q) / case["temperature"]
        if s["ref"] is not None:
            h = h - s["ref"].double()
        if s["mask"] is not None:
            h = h[s["mask"]]
        h = h.reshape(-1)
        if case["kind"] == "sigmoid":
            f = torch.nn.functional.logsigmoid
            row = -(1 - case["smooth"]) * f(case["beta"] * h) - case["smooth"] * f(-case["beta"] * h)
        else:
            row = (h - 1 / (2 * case["beta"])) ** 2
        loss = row.sum() / max(1, row.numel())
        return [loss.detach(), *torch.autograd.grad(loss, (q, p, n))]
    if op == "clip":
        every = torch.cat([x.double() for x in s["grads"]])
        norm = every.abs().max() if case["norm"] == math.inf else torch.linalg.vector_norm(every)
        return [norm, every * min(1.0, case["max_norm"] / (norm.item() + 1e-6))]
    q, scores = s["q"].double(), []
    for a in range(0, case["n"], 1 << 17):
        rows = s["codes"][a:a + (1 << 17)].double()
        sc = s["scales"][a:a + (1 << 17)].double()
        col = torch.arange(case["H"], device=DEV) // case["group"]
        scores.append((rows * sc[:, col]) @ q.t())
    return [torch.cat(scores).t().contiguous()]
