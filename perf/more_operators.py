"""The two ends of a language model's training and scoring step as cases that can be timed and compared.

Six kinds, each one pass through an operator:

  embed      rows of the embedding table for given tokens, times a factor
  embed_bwd  the table's gradient: the rows of d_out summed by token, written as a whole table or added to a gradient that is there (tied weights)
  ln         layer norm of a stream without a residual's addition
  ln_bwd     the gradients of the layer norm: dx (which is the residual's too), dweight, dbias
  logp       log probabilities of given tokens with the log of the sum, the entropy and the largest alternatives
  logp_bwd   the gradient of these with respect to the logits

``run`` is either the calls of ``tyr_amd`` (``own``) or the same operators in elementary torch operations in 32 bits.
"""
from __future__ import annotations

import math

import torch

own = False

EPS = 1e-5
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # the tokens of one decode step of a batch: latency
        dict(name="embed_step", kind="embed", n=48, vocab=32768, d=4096, dtype="bf16", scale=1.0),
        # a training batch, embeddings times the root of their width
        dict(name="embed_batch", kind="embed", n=16384, vocab=65536, d=2048, dtype="bf16", scale=45.25),
        # fine-tuning on few ragged sequences: nearly all of the table's gradient is zero
        dict(name="embed_bwd_few", kind="embed_bwd", n=900, vocab=32768, d=1024, dtype="bf16", scale=1.0, into=False),
        # the gradient of a training batch
        dict(name="embed_bwd_train", kind="embed_bwd", n=32768, vocab=65536, d=2048, dtype="bf16", scale=45.25, into=False),
        # the table is the head's matrix too, whose gradient is there already; kept in f32
        dict(name="embed_bwd_tied", kind="embed_bwd", n=16384, vocab=50001, d=1024, dtype="f32", scale=1.0, into=True),
        # the norm in front of the head, a training batch
        dict(name="ln_train", kind="ln", rows=65536, d=1024, bias=True),
        # the gradients of few ragged sequences
        dict(name="ln_bwd_ragged", kind="ln_bwd", rows=2000, d=4096, resid=True),
        # the gradients of the training batch
        dict(name="ln_bwd_train", kind="ln_bwd", rows=65536, d=1024, resid=True),
        # the sampled tokens of one decode step, with the alternatives that a server answers with: latency
        dict(name="logp_step", kind="logp", rows=32, vocab=131072, width=131072, dtype="bf16", top=20, entropy=True),
        # scoring of given texts, an odd vocabulary whose rows are padded for the head's product
        dict(name="logp_score", kind="logp", rows=4096, vocab=50001, width=50008, dtype="bf16", top=5, entropy=True),
        # the gradient of a training batch's loss
        dict(name="logp_bwd_train", kind="logp_bwd", rows=4096, vocab=50001, width=50008, dtype="bf16", entropy=False),
        # policy training with an entropy term on f32 logits, rows that start anywhere
        dict(name="logp_bwd_policy", kind="logp_bwd", rows=777, vocab=50001, width=50001, dtype="f32", entropy=True),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("embed", "embed_bwd", "ln", "ln_bwd", "logp", "logp", "logp_bwd"))
    while True:
        if kind in ("embed", "embed_bwd"):
            c = dict(kind=kind, n=_log(rng, 1, 32768), vocab=_log(rng, 100, 131072), d=8 * _log(rng, 8, 512), dtype=rng.choice(("bf16", "bf16", "f32")),
                     scale=rng.choice((1.0, 1.0, 45.25)))
            if kind == "embed_bwd":
                c |= dict(into=rng.random() < 0.4)
            if (c["n"] + 2 * c["vocab"]) * c["d"] * (4 if c["dtype"] == "f32" else 2) <= 5 * 32768 * 2048 * 2:
                return c
        elif kind in ("ln", "ln_bwd"):
            c = dict(kind=kind, rows=_log(rng, 1, 65536), d=8 * _log(rng, 8, 1024))
            c |= dict(bias=rng.random() < 0.75) if kind == "ln" else dict(resid=rng.random() < 0.75)
            if c["rows"] * c["d"] <= 65536 * 1024:
                return c
        else:
            v = _log(rng, 100, 151000)
            c = dict(kind=kind, rows=_log(rng, 1, 4096), vocab=v, width=rng.choice((v, -(-v // 8) * 8, -(-v // 128) * 128)), dtype=rng.choice(("bf16", "bf16", "f32")),
                     entropy=rng.random() < 0.5)
            if kind == "logp":
                c |= dict(top=rng.choice((0, 0, 1, 5, 20, 50)))
            if c["rows"] * c["width"] * (4 if c["dtype"] == "f32" else 2) <= 4096 * 50001 * 2:
                return c


def _normal(g, *shape, std=1.0, dtype=torch.bfloat16):
    x = torch.randn(*shape, generator=g, device="cuda")
    return (x * std if std != 1.0 else x).to(dtype)


def _stream(g, rows, d):
    """Rows of a residual stream: a few channels are much larger than the others, and the rows have a mean."""
    loud = 1.0 + 15.0 * (torch.rand(d, generator=g, device="cuda") < 0.01)
    return (torch.randn(rows, d, generator=g, device="cuda") * loud + 0.3).to(torch.bfloat16)


def _tokens(g, n, vocab, none):
    """Tokens as texts have them: the k-th frequent one about 1/k as often as the first; some of them (-1) are padding."""
    ids = (torch.rand(n, generator=g, device="cuda", dtype=torch.float64) * math.log(vocab + 1)).exp().floor().long() - 1
    ids = ids.clamp(0, vocab - 1)
    return torch.where(torch.rand(n, generator=g, device="cuda") < none, -1, ids) if none else ids


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    kind = case["kind"]
    st = dict(case=case)
    if kind in ("embed", "embed_bwd"):
        n, vocab, d, dtype = case["n"], case["vocab"], case["d"], TYPES[case["dtype"]]
        st["ids"] = _tokens(g, n, vocab, 0.0 if kind == "embed" else 0.05)
        if kind == "embed":
            st["table"] = _normal(g, vocab, d, std=0.02, dtype=dtype)
        else:
            st["dout"] = _normal(g, n, d, dtype=dtype)
            st["grad"] = _normal(g, vocab, d, dtype=dtype) if case["into"] else None
        return st
    if kind in ("ln", "ln_bwd"):
        rows, d = case["rows"], case["d"]
        st["x"] = _stream(g, rows, d)
        st["w"] = (1.0 + _normal(g, d, std=0.2, dtype=torch.float32)).to(torch.bfloat16)
        if kind == "ln":
            st["b"] = _normal(g, d, std=0.2) if case["bias"] else None
        else:
            st["dy"] = _normal(g, rows, d)
            st["dres"] = _normal(g, rows, d) if case["resid"] else None
        return st
    rows, vocab, width = case["rows"], case["vocab"], case["width"]
    # rows of unlike sharpness; the given token is mostly a likely one; some positions (-1) are padding
    sharp = 0.5 + 3.0 * torch.rand(rows, 1, generator=g, device="cuda")
    x = torch.randn(rows, width, generator=g, device="cuda") * sharp
    st["targets"] = _tokens(g, rows, vocab, 0.05)
    x[torch.arange(rows, device="cuda"), st["targets"].clamp_min(0)] += 8.0
    st["x"] = x.to(TYPES[case["dtype"]])
    if kind == "logp_bwd":
        # what the forward pass left, and the gradients of its outputs
        st["lse"] = torch.empty(rows, device="cuda")
        st["ent"] = torch.empty(rows, device="cuda") if case["entropy"] else None
        for at in range(0, rows, 256):
            z = st["x"][at:at + 256, :vocab].double()
            top = z.amax(-1, keepdim=True)
            lse = top + (z - top).exp().sum(-1, keepdim=True).log()
            st["lse"][at:at + 256] = lse[:, 0].float()
            if case["entropy"]:
                st["ent"][at:at + 256] = -((z - lse).exp() * (z - lse)).sum(-1).float()
        st["dlogp"] = -(0.5 + torch.rand(rows, generator=g, device="cuda")) / rows
        st["dent"] = 0.01 * torch.rand(rows, generator=g, device="cuda") / rows if case["entropy"] else None
    return st


# ---- plain forms


def _plain_embed(st):
    return (st["table"][st["ids"]].float() * st["case"]["scale"]).to(st["table"].dtype)


def _plain_embed_bwd(st):
    case, ids = st["case"], st["ids"]
    real = ids >= 0
    add = torch.zeros(case["vocab"], case["d"], device="cuda").index_add_(0, ids.clamp_min(0), torch.where(real[:, None], st["dout"].float(), 0.0)) * case["scale"]
    if st["grad"] is None:
        return add.to(st["dout"].dtype)
    # in place, as the call: every pass adds once more
    return st["grad"].copy_((st["grad"].float() + add).to(st["dout"].dtype))


def _plain_ln(st):
    x = st["x"].float()
    c = x - x.mean(-1, keepdim=True)
    y = c * torch.rsqrt((c * c).mean(-1, keepdim=True) + EPS) * st["w"].float()
    return (y if st["b"] is None else y + st["b"].float()).to(torch.bfloat16)


def _plain_ln_bwd(st):
    x, dy = st["x"].float(), st["dy"].float()
    c = x - x.mean(-1, keepdim=True)
    rho = torch.rsqrt((c * c).mean(-1, keepdim=True) + EPS)
    n = c * rho
    g = dy * st["w"].float()
    dx = rho * (g - g.mean(-1, keepdim=True) - n * (g * n).mean(-1, keepdim=True))
    if st["dres"] is not None:
        dx = dx + st["dres"].float()
    return dx.to(torch.bfloat16), (dy * n).sum(0).to(torch.bfloat16), dy.sum(0).to(torch.bfloat16)


def _plain_logp(st):
    case, t = st["case"], st["targets"]
    x = st["x"][:, :case["vocab"]].float()
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(-1, keepdim=True)
    log = torch.log(total)
    given = (x.gather(1, t.clamp_min(0)[:, None]) - top - log)[:, 0]
    out = [torch.where(t >= 0, given, 0.0), (top + log)[:, 0]]
    if case["entropy"]:
        out.append((log - (e * (x - top)).sum(-1, keepdim=True) / total)[:, 0])
    if case["top"]:
        # by value, then by place: whole numbers that are all different
        b = (x + 0.0).view(torch.int32)
        b = (b ^ ((b >> 31) & 0x7fffffff)).long()
        at = ((b << 32) + (2 ** 32 - 1 - torch.arange(case["vocab"], device="cuda"))).topk(case["top"], dim=-1).values
        at = 2 ** 32 - 1 - (at & (2 ** 32 - 1))
        out += [x.gather(1, at) - top - log, at.int()]
    return out


def _plain_logp_bwd(st):
    case, t = st["case"], st["targets"]
    x = st["x"][:, :case["vocab"]].float()
    z = x - st["lse"][:, None]
    p = torch.exp(z)
    glp = torch.where(t >= 0, st["dlogp"], 0.0)[:, None]
    d = -glp * p
    if case["entropy"]:
        d = d - st["dent"][:, None] * p * (z + st["ent"][:, None])
    d.scatter_add_(1, t.clamp_min(0)[:, None], glp)
    out = torch.zeros(st["x"].shape, dtype=st["x"].dtype, device="cuda")
    out[:, :case["vocab"]] = d.to(out.dtype)
    return out


def run(st):
    case = st["case"]
    kind = case["kind"]
    if own:
        import tyr_amd

        if kind == "embed":
            return tyr_amd.embedding(st["ids"], st["table"], scale=case["scale"])
        if kind == "embed_bwd":
            return tyr_amd.embedding_bwd(st["dout"], st["ids"], case["vocab"], scale=case["scale"], into=st["grad"])
        if kind == "ln":
            return tyr_amd.layernorm_residual(st["x"], None, st["w"], st["b"], EPS)[0]
        if kind == "ln_bwd":
            return tyr_amd.layernorm_residual_bwd(st["dy"], st["x"], st["w"], EPS, d_resid=st["dres"])
        if kind == "logp":
            logp, lse, ent, top, at = tyr_amd.token_logprobs(st["x"], st["targets"], vocab=case["vocab"], top=case["top"], entropy=case["entropy"])
            return [logp, lse] + ([ent] if case["entropy"] else []) + ([top, at] if case["top"] else [])
        return tyr_amd.token_logprobs_bwd(st["dlogp"], st["x"], st["targets"], st["lse"], vocab=case["vocab"], entropy=st["ent"], d_entropy=st["dent"])
    return {"embed": _plain_embed, "embed_bwd": _plain_embed_bwd, "ln": _plain_ln, "ln_bwd": _plain_ln_bwd, "logp": _plain_logp,
            "logp_bwd": _plain_logp_bwd}[kind](st)


# ---- the operators' definitions in 64 bits


def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind == "embed":
        return torch.nn.functional.embedding(st["ids"], st["table"].double()) * case["scale"]
    if kind == "embed_bwd":
        keep = st["ids"] >= 0
        order = torch.argsort(st["ids"][keep], stable=True)
        ids, rows = st["ids"][keep][order], st["dout"][keep][order]
        out = torch.zeros(case["vocab"], case["d"], dtype=torch.float64, device="cuda") if st["grad"] is None else st["grad"].double()
        ends = torch.cat((torch.nonzero(ids[1:] != ids[:-1])[:, 0] + 1, torch.tensor([len(ids)], device="cuda"))).tolist()
        start = 0
        for end in ends if len(ids) else []:
            out[ids[start]] += rows[start:end].double().sum(0) * case["scale"]
            start = end
        return out
    if kind == "ln":
        return torch.nn.functional.layer_norm(st["x"].double(), (case["d"],), st["w"].double(), None if st["b"] is None else st["b"].double(), EPS)
    if kind == "ln_bwd":
        x, w = st["x"].double().requires_grad_(), st["w"].double().requires_grad_()
        b = torch.zeros_like(w).requires_grad_()
        y = torch.nn.functional.layer_norm(x, (case["d"],), w, b, EPS)
        loss = (y * st["dy"].double()).sum() + (0.0 if st["dres"] is None else (x * st["dres"].double()).sum())
        return torch.autograd.grad(loss, (x, w, b))
    if kind == "logp":
        parts = []
        for at in range(0, case["rows"], 256):
            z = torch.log_softmax(st["x"][at:at + 256, :case["vocab"]].double(), -1)
            t = st["targets"][at:at + 256]
            row = [torch.where(t >= 0, z[torch.arange(len(t), device="cuda"), t], 0.0), st["x"][at:at + 256, :case["vocab"]].double().logsumexp(-1)]
            if case["entropy"]:
                row.append(-(z * z.exp()).sum(-1))
            if case["top"]:
                row.append(z.sort(dim=-1, descending=True, stable=True).values[:, :case["top"]])
            parts.append(row)
        out = [torch.cat(p) for p in zip(*parts)]
        return out + [None] if case["top"] else out
    out = torch.zeros(st["x"].shape, dtype=torch.float64, device="cuda")
    for at in range(0, case["rows"], 256):
        x = st["x"][at:at + 256, :case["vocab"]].double().requires_grad_()
        z = torch.log_softmax(x, -1)
        t = st["targets"][at:at + 256]
        k = t >= 0
        loss = (z[k, t[k]] * st["dlogp"][at:at + 256][k].double()).sum()
        if case["entropy"]:
            loss = loss - ((z * z.exp()).sum(-1) * st["dent"][at:at + 256].double()).sum()
        out[at:at + 256, :case["vocab"]] = torch.autograd.grad(loss, x)[0] if loss.requires_grad else 0.0
    return out


def _distinct(case):
    """How many different tokens there are among n, in the mean (the padding left out of account)."""
    k = torch.arange(1, case["vocab"] + 1, dtype=torch.float64)
    share = torch.log1p(1.0 / k) / math.log(case["vocab"] + 1)
    return float((1.0 - (1.0 - share) ** case["n"]).sum())


def work(case):
    kind = case["kind"]
    if kind in ("embed", "embed_bwd"):
        e, n, d = 4 if case["dtype"] == "f32" else 2, case["n"], case["d"]
        if kind == "embed":
            return {"bytes": (_distinct(case) + n) * d * e + 8 * n, "flops": n * d}
        # 5 % is padding; of a gradient that is there only the tokens' rows are read and written
        return {"bytes": 0.95 * n * d * e + (2 * _distinct(case) if case["into"] else case["vocab"]) * d * e + 8 * n, "flops": n * d}
    if kind in ("ln", "ln_bwd"):
        n, d = case["rows"] * case["d"], case["d"]
        if kind == "ln":
            return {"bytes": 4 * n + 4 * d, "flops": 7 * n}
        return {"bytes": n * (8 if case["resid"] else 6) + 6 * d, "flops": 17 * n}
    e, rows, vocab = 4 if case["dtype"] == "f32" else 2, case["rows"], case["vocab"]
    if kind == "logp":
        return {"bytes": rows * (vocab * e + 8 + 8 + (4 if case["entropy"] else 0) + 8 * case["top"]), "flops": rows * vocab * (6 if case["entropy"] else 4)}
    return {"bytes": rows * ((vocab + case["width"]) * e + 16 + (8 if case["entropy"] else 0)), "flops": rows * vocab * (8 if case["entropy"] else 5)}
