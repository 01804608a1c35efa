"""The operators of a paged, quantised decoder layer as cases that can be timed and compared.

Five kinds, each one pass through an operator:

  norm     h = x + residual and its RMS norm, as bf16 (the layer of a bf16 model, the norm of q and k heads without a residual)
           or as e4m3 with a factor per row (the operand of the quantised projections)
  normbwd  the gradients of that norm: dx (which is the residual's too) and dweight
  append   rotate the new tokens' q and k, write k and v into the pages of the cache: one token a sequence, or a prompt's
  paged    attention of one new token over the pages: batches of equal or very unequal lengths, windows with sinks

``run`` is either the calls of ``tyr_amd`` (``own``) or the same operators in elementary torch operations in 32 bits.
"""
from __future__ import annotations

import math

import torch

own = False

HEADS = ((4, 4), (8, 2), (16, 16), (16, 4), (32, 8), (32, 32), (32, 1))
PAGES = (16, 16, 32, 48, 64, 128, 256)
EPS = 1e-6
BF16, E4M3 = torch.bfloat16, torch.float8_e4m3fn


def listed():
    return [
        # the quantised projections' operand for a batch of decoded tokens: latency
        dict(name="norm_fp8_decode", kind="norm", rows=32, d=4096, out="e4m3", residual=True),
        # the norm of the query heads of a prompt: many short rows, no residual
        dict(name="norm_heads_prompt", kind="norm", rows=1111 * 32, d=128, out="bf16", residual=False),
        # a prompt batch on its way into quantised projections
        dict(name="norm_fp8_prompt", kind="norm", rows=2222, d=4096, out="e4m3", residual=True),
        # a training batch
        dict(name="norm_train", kind="norm", rows=65536, d=1024, out="bf16", residual=True),
        # fine-tuning on few ragged sequences
        dict(name="norm_bwd_ragged", kind="normbwd", rows=2000, d=4096, resid=True),
        # the gradients of the training batch
        dict(name="norm_bwd_train", kind="normbwd", rows=65536, d=1024, resid=True),
        # one token of every sequence into the cache
        dict(name="append_decode", kind="append", B=32, T=1, Hq=32, Hkv=8, D=128, page=16, past=1500, cache="bf16"),
        # two prompts of unlike length into e4m3 pages
        dict(name="append_prompt", kind="append", B=2, T=1111, Hq=32, Hkv=8, D=128, page=16, past=0, cache="e4m3"),
        # interactive generation: one sequence
        dict(name="paged_single", kind="paged", B=1, Hq=32, Hkv=8, D=128, page=16, shortest=1500, longest=1500, window=0, sinks=0, cache="bf16"),
        # batched serving with long sequences (1 GiB of K and V)
        dict(name="paged_batch", kind="paged", B=32, Hq=32, Hkv=8, D=128, page=64, shortest=8192, longest=8192, window=0, sinks=0, cache="bf16"),
        # a server's mixture of short and long conversations, e4m3 cache
        dict(name="paged_ragged_e4m3", kind="paged", B=64, Hq=32, Hkv=8, D=128, page=16, shortest=37, longest=32768, window=0, sinks=0, cache="e4m3"),
        # long streams behind a window, the first tokens kept
        dict(name="paged_window_sinks", kind="paged", B=16, Hq=16, Hkv=4, D=64, page=32, shortest=20000, longest=32768, window=4096, sinks=4, cache="bf16"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("norm", "normbwd", "append", "paged", "paged"))
    while True:
        if kind in ("norm", "normbwd"):
            c = dict(kind=kind, rows=_log(rng, 1, 65536), d=8 * _log(rng, 8, 2048))
            if kind == "norm":
                c |= dict(out=rng.choice(("bf16", "e4m3")), residual=rng.random() < 0.75)
            else:
                c |= dict(resid=rng.random() < 0.75)
            if c["rows"] * c["d"] <= 65536 * 1024:
                return c
        elif kind == "append":
            hq, hkv = rng.choice(HEADS)
            t = 1 if rng.random() < 0.5 else _log(rng, 2, 2222)
            c = dict(kind=kind, B=_log(rng, 1, 128 if t == 1 else 8), T=t, Hq=hq, Hkv=hkv, D=rng.choice((64, 128, 128)), page=rng.choice(PAGES),
                     past=_log(rng, 1, 3000), cache=rng.choice(("bf16", "e4m3")))
            if c["B"] * t * (hq + 2 * hkv) * c["D"] <= 2222 * 48 * 128 and c["B"] * (t + c["past"]) * hkv * c["D"] <= 1 << 26:
                return c
        else:
            hq, hkv = rng.choice(HEADS)
            n = _log(rng, 1, 32768)
            c = dict(kind=kind, B=_log(rng, 1, 128), Hq=hq, Hkv=hkv, D=rng.choice((64, 128, 128)), page=rng.choice(PAGES),
                     shortest=n if rng.random() < 0.4 else _log(rng, 1, n), longest=n, window=0, sinks=0, cache=rng.choice(("bf16", "e4m3")))
            if rng.random() < 0.3:
                c |= dict(window=_log(rng, 1, 2 * n), sinks=rng.choice((0, 1, 4, 17, 64)))
            if c["B"] * hkv * n * c["D"] <= 32 * 8 * 8192 * 128:
                return c


def _lengths(case):
    """Cached rows of the sequences, evenly spaced in their logarithm."""
    B, lo, hi = case["B"], case["shortest"], case["longest"]
    return [hi if B == 1 else round(lo * (hi / lo) ** (i / (B - 1))) for i in range(B)]


def _new_tokens(case):
    """New tokens of the sequences: a prompt batch is padded to T."""
    B, T = case["B"], case["T"]
    return [max(1, T - i * T // (2 * B)) for i in range(B)]


def _normal(g, *shape, std=1.0, dtype=BF16):
    x = torch.randn(*shape, generator=g, device="cuda")
    return (x * std if std != 1.0 else x).to(dtype)


def _stream(g, rows, d):
    """Rows of a residual stream: a few channels are much larger than the others."""
    loud = 1.0 + 15.0 * (torch.rand(d, generator=g, device="cuda") < 0.01)
    return (torch.randn(rows, d, generator=g, device="cuda") * loud).to(BF16)


def _pool(g, pages, case):
    """Pages of K or V, and the kv heads' factors (e4m3)."""
    shape = (pages, case["Hkv"], case["page"], case["D"])
    if case["cache"] == "bf16":
        return _normal(g, *shape), None
    factor = (0.75 + 0.5 * torch.rand(case["Hkv"], generator=g, device="cuda")) * (4.5 / 448.0)
    values = torch.empty(shape, dtype=E4M3, device="cuda")
    for part in range(0, pages, 4096):
        n = min(4096, pages - part)
        values[part:part + n] = (_normal(g, n, *shape[1:], dtype=torch.float32) / factor[:, None, None]).clamp(-448.0, 448.0).to(E4M3)
    return values, factor


def _tables(g, rows, page):
    """Every sequence's pages, anywhere in the pool and in any order; -1 behind its last one.  -> table, pages in the pool"""
    need = [-(-r // page) for r in rows]
    total = sum(need) + 3
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(rows), max(need)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, total


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    kind = case["kind"]
    st = dict(case=case)
    if kind in ("norm", "normbwd"):
        rows, d = case["rows"], case["d"]
        st["x"] = _stream(g, rows, d)
        st["w"] = (1.0 + _normal(g, d, std=0.2, dtype=torch.float32)).to(BF16)
        st["res"] = _normal(g, rows, d) if kind == "norm" and case["residual"] else None
        if kind == "normbwd":
            st["dy"] = _normal(g, rows, d)
            st["dres"] = _normal(g, rows, d) if case["resid"] else None
        return st
    B, Hq, Hkv, D = (case[k] for k in ("B", "Hq", "Hkv", "D"))
    # which sequence of the batch has which length follows the seed
    order = torch.randperm(B, generator=g, device="cuda").tolist()
    if kind == "append":
        new, T, past = [_new_tokens(case)[i] for i in order], case["T"], case["past"]
        pos = [past * (i + 1) // B for i in order]
        table, pages = _tables(g, [p + n for p, n in zip(pos, new)], case["page"])
        st["q"] = _normal(g, B, T, Hq, D)
        st["kn"], st["vn"] = _normal(g, B, T, Hkv, D), _normal(g, B, T, Hkv, D)
        ang = torch.outer(torch.arange(past + T, device="cuda", dtype=torch.float64),
                          10000.0 ** (-torch.arange(0, D, 2, device="cuda", dtype=torch.float64) / D))
        st["cos"], st["sin"] = torch.cos(ang).float(), torch.sin(ang).float()
        st["pos"] = torch.tensor(pos, dtype=torch.int32, device="cuda")
        st["new"] = torch.tensor(new, dtype=torch.int32, device="cuda")
    else:
        lens = [_lengths(case)[i] for i in order]
        table, pages = _tables(g, lens, case["page"])
        st["q"] = _normal(g, B, Hq, 1, D)
        st["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    st["table"] = table
    st["k"], st["ks"] = _pool(g, pages, case)
    st["v"], st["vs"] = _pool(g, pages, case)
    return st


# ---- plain forms


def _plain_norm(st):
    h = st["x"] if st["res"] is None else (st["x"].float() + st["res"].float()).to(BF16)
    f = h.float()
    y = f * torch.rsqrt((f * f).mean(-1, keepdim=True) + EPS) * st["w"].float()
    if st["case"]["out"] == "bf16":
        return y.to(BF16), h
    top = y.abs().amax(-1)
    scale = torch.where(top < 2.0 ** -100, 1.0, top / 448.0)
    return (y / scale[:, None]).clamp(-448.0, 448.0).to(E4M3), scale, h


def _plain_normbwd(st):
    h, dy, w = st["x"].float(), st["dy"].float(), st["w"].float()
    d = h.shape[-1]
    rho = torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS)
    g = dy * w
    dx = rho * g - h * (rho ** 3 / d * (g * h).sum(-1, keepdim=True))
    if st["dres"] is not None:
        dx = dx + st["dres"].float()
    return dx.to(BF16), (dy * h * rho).sum(0).to(BF16)


def _rotate(x, c, s):
    a, b = x.float().chunk(2, -1)
    return torch.cat((a * c - b * s, a * s + b * c), -1)


def _plain_append(st):
    case = st["case"]
    B, T, page = case["B"], case["T"], case["page"]
    t = torch.arange(T, device="cuda")[None, :].expand(B, T)
    at = st["pos"].long()[:, None] + t
    c, s = st["cos"][at][:, :, None], st["sin"][at][:, :, None]
    q = _rotate(st["q"], c, s).to(BF16)
    k, v = _rotate(st["kn"], c, s), st["vn"].float()
    # tokens of the padding write what their sequence's first token writes
    real = (t < st["new"][:, None])
    at = torch.where(real, at, at[:, :1])
    where = (st["table"].long().gather(1, at // page), at % page)
    for new, pool, factor in ((k, st["k"], st["ks"]), (v, st["v"], st["vs"])):
        new = torch.where(real[:, :, None, None], new, new[:, :1])
        if factor is not None:
            new = (new / factor[:, None]).clamp(-448.0, 448.0)
        pool.view(torch.uint8 if factor is not None else torch.int16)[where[0], :, where[1]] = (
            new.to(E4M3).view(torch.uint8) if factor is not None else new.to(BF16).view(torch.int16))
    return q, st["k"], st["v"]


def _plain_paged(st):
    case = st["case"]
    B, Hq, Hkv, D = (case[k] for k in ("B", "Hq", "Hkv", "D"))
    table = st["table"].clamp_min(0).long()
    L = table.shape[1] * case["page"]

    def rows(pool, factor):
        x = pool[table].transpose(1, 2).reshape(B, Hkv, L, D).float()
        return x if factor is None else x * factor[:, None, None]

    j, n = torch.arange(L, device="cuda")[None, :], st["lens"].long()[:, None]
    seen = j < n
    if case["window"]:
        seen = seen & ((j >= n - case["window"]) | (j < case["sinks"]))
    q = st["q"].float().view(B, Hkv, Hq // Hkv, D) * D ** -0.5
    score = torch.matmul(rows(st["k"], st["ks"]), q.transpose(2, 3).contiguous())
    score = score.masked_fill(~seen[:, None, :, None], -math.inf)
    top = score.amax(2, keepdim=True)
    p = torch.exp(score - top)
    total = p.sum(2, keepdim=True)
    o = torch.matmul((p / total).transpose(2, 3).contiguous(), rows(st["v"], st["vs"]))
    return o.reshape(B, Hq, 1, D).to(BF16), (top + torch.log(total)).reshape(B, Hq)


def run(st):
    case = st["case"]
    kind = case["kind"]
    if own:
        import tyr_amd

        if kind == "norm":
            return (tyr_amd.rmsnorm_residual if case["out"] == "bf16" else tyr_amd.rmsnorm_residual_fp8)(st["x"], st["res"], st["w"], EPS)
        if kind == "normbwd":
            return tyr_amd.rmsnorm_residual_bwd(st["dy"], st["x"], st["w"], EPS, d_resid=st["dres"])
        if kind == "append":
            q = tyr_amd.paged_rope_append(st["q"], st["kn"], st["vn"], st["cos"], st["sin"], st["k"], st["v"], st["table"], st["pos"],
                                          new_lens=st["new"], k_scale=st["ks"], v_scale=st["vs"])
            return q, st["k"], st["v"]
        return tyr_amd.paged_decode(st["q"], st["k"], st["v"], st["table"], st["lens"], window=case["window"], sinks=case["sinks"],
                                    k_scale=st["ks"], v_scale=st["vs"])
    return {"norm": _plain_norm, "normbwd": _plain_normbwd, "append": _plain_append, "paged": _plain_paged}[kind](st)


# ---- the operators' definitions in 64 bits


def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind == "norm":
        # the statistics are those of the bf16 sum that the layer keeps
        h = (st["x"].double() if st["res"] is None else (st["x"].double() + st["res"].double()).to(BF16).double())
        y = h / torch.sqrt(h.pow(2).sum(-1, keepdim=True) / case["d"] + EPS) * st["w"].double()
        if case["out"] == "bf16":
            return y, h
        s = y.abs().max(-1).values / 448.0
        return y / s[:, None], s, h
    if kind == "normbwd":
        x, w = st["x"].double().requires_grad_(), st["w"].double().requires_grad_()
        y = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + EPS) * w
        loss = (y * st["dy"].double()).sum() + (0.0 if st["dres"] is None else (x * st["dres"].double()).sum())
        return torch.autograd.grad(loss, (x, w))
    if kind == "append":
        B, page, half = case["B"], case["page"], case["D"] // 2
        q, pools = st["q"].double(), [st["k"].double(), st["v"].double()]
        for b in range(B):
            first, n = int(st["pos"][b]), int(st["new"][b])
            z = torch.complex(st["cos"].double(), st["sin"].double())[first:first + case["T"], None]
            turned = []
            for x in (q[b], st["kn"][b].double()):
                y = torch.complex(x[..., :half], x[..., half:]) * z
                turned.append(torch.cat((y.real, y.imag), -1))
            q[b] = turned[0]
            ids = st["table"][b].tolist()
            for pool, new, factor in zip(pools, (turned[1], st["vn"][b].double()), (st["ks"], st["vs"])):
                new = new[:n] if factor is None else (new[:n] / factor.double()[:, None]).clamp(-448.0, 448.0)
                done = 0
                while done < n:
                    row = (first + done) % page
                    m = min(page - row, n - done)
                    pool[ids[(first + done) // page], :, row:row + m] = new[done:done + m].transpose(0, 1)
                    done += m
        return q, pools[0], pools[1]
    B, Hq, Hkv, D, page = (case[k] for k in ("B", "Hq", "Hkv", "D", "page"))
    o = torch.empty(B, Hq, 1, D, dtype=torch.float64, device="cuda")
    lse = torch.empty(B, Hq, dtype=torch.float64, device="cuda")
    for b in range(B):
        n = int(st["lens"][b])
        rows = torch.arange(n, device="cuda")
        if case["window"]:
            rows = rows[(rows < case["sinks"]) | (rows + case["window"] >= n)]
        ids = st["table"][b].long()[rows // page]
        k, v = (p[ids, :, rows % page].double().transpose(0, 1) for p in (st["k"], st["v"]))      # [Hkv, rows, D]
        if st["ks"] is not None:
            k, v = k * st["ks"].double()[:, None, None], v * st["vs"].double()[:, None, None]
        group = Hq // Hkv
        for h in range(Hkv):
            s = (k[h][None] * st["q"][b, h * group:(h + 1) * group].double()).sum(-1) / math.sqrt(D)     # [group, rows]
            lse[b, h * group:(h + 1) * group] = torch.logsumexp(s, -1)
            o[b, h * group:(h + 1) * group, 0] = torch.softmax(s, -1) @ v[h].contiguous()
    return o, lse


def work(case):
    kind = case["kind"]
    if kind in ("norm", "normbwd"):
        n, d = case["rows"] * case["d"], case["d"]
        if kind == "normbwd":
            return {"bytes": n * (8 if case["resid"] else 6) + 4 * d, "flops": 12 * n}
        moved = 2 * (2 if case["residual"] else 1) + (2 if case["residual"] else 0) + (2 if case["out"] == "bf16" else 1)
        return {"bytes": n * moved + 2 * d + (4 * case["rows"] if case["out"] == "e4m3" else 0), "flops": 5 * n}
    D, Hq, Hkv, e = case["D"], case["Hq"], case["Hkv"], 2 if case["cache"] == "bf16" else 1
    if kind == "append":
        new, padded = sum(_new_tokens(case)), case["B"] * case["T"]
        return {"bytes": 4 * padded * Hq * D + (4 + 2 * e) * new * Hkv * D + 4 * D * min(padded, case["past"] + case["T"]),
                "flops": 3 * D * (padded * Hq + new * Hkv)}
    seen = sum(n if not case["window"] else min(n, case["window"] + min(case["sinks"], max(0, n - case["window"]))) for n in _lengths(case))
    return {"bytes": 2 * e * seen * Hkv * D + 4 * case["B"] * Hq * D + 4 * case["B"] * Hq, "flops": 4 * D * Hq * seen}
