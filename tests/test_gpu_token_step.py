"""The operators at both ends of a language model together: a training step with tied weights, a scoring step, streams, captured graphs."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF16 = 2.0 ** -8


class Tied:
    """Embedding, blocks of norm and product with a residual, norm, product with the table: the parameters as f32 masters."""

    def __init__(self, vocab, d, blocks, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.vocab, self.d = vocab, d
        self.width = -(-vocab // 8) * 8                       # the product's columns
        self.master = {"table": torch.randn(vocab, d, generator=g, device="cuda") * 0.05}
        for i in range(blocks):
            self.master[f"p{i}"] = torch.randn(d, d, generator=g, device="cuda") * d ** -0.5 * 0.5
            self.master[f"w{i}"] = 1.0 + 0.1 * torch.randn(d, generator=g, device="cuda")
            self.master[f"b{i}"] = 0.1 * torch.randn(d, generator=g, device="cuda")
        self.blocks = blocks
        self.low = {k: v.bfloat16() for k, v in self.master.items()}

    def padded_table(self):
        t = torch.zeros(self.width, self.d, dtype=torch.bfloat16, device="cuda")
        t[:self.vocab] = self.low["table"]
        return t

    def gradients(self, ids, targets):
        """Mean loss over the real targets, and the gradient of every parameter, by the framework's calls alone."""
        import tyr_amd as T
        p, n = self.low, ids.numel()
        real = (targets >= 0) & (targets < self.vocab)
        scale = self.d ** 0.5
        h = T.embedding(ids, p["table"], scale=scale)
        kept = []
        y = None
        for i in range(self.blocks):
            out, h = T.layernorm_residual(h if y is None else y, None if y is None else h, p[f"w{i}"], p[f"b{i}"])
            y = T.gemm_bf16(out, p[f"p{i}"], trans_b=True)
            kept.append((out, h))
        last, h_last = T.layernorm_residual(y, h, torch.ones_like(p["w0"]), None)
        table = self.padded_table()
        logits = T.gemm_bf16(last, table, trans_b=True)
        logp, lse, _, _, _ = T.token_logprobs(logits, targets, vocab=self.vocab, entropy=False)
        count = real.sum()
        loss = -logp.sum() / count
        d_logits = T.token_logprobs_bwd((-1.0 / count).expand(n).contiguous(), logits, targets, lse, vocab=self.vocab, in_place=True)
        grads = {}
        d_table = T.gemm_bf16(d_logits.t().contiguous(), last)[:self.vocab].contiguous()
        d_last = T.gemm_bf16(d_logits, table)
        dh, _, _ = T.layernorm_residual_bwd(d_last, h_last, torch.ones_like(p["w0"]), bias=False)
        for i in reversed(range(self.blocks)):
            out, h = kept[i]
            grads[f"p{i}"] = T.gemm_bf16(dh.t().contiguous(), out)
            d_out = T.gemm_bf16(dh, p[f"p{i}"])
            dh, grads[f"w{i}"], grads[f"b{i}"] = T.layernorm_residual_bwd(d_out, h, p[f"w{i}"], d_resid=dh)
        grads["table"] = T.embedding_bwd(dh, ids, self.vocab, scale=scale, into=d_table)
        return loss, grads

    def reference(self, ids, targets):
        """The same by autograd in float64."""
        p = {k: v.double().requires_grad_() for k, v in self.low.items()}
        real = (targets >= 0) & (targets < self.vocab)
        inside = (ids >= 0) & (ids < self.vocab)
        h = p["table"][ids.clamp(0, self.vocab - 1)] * inside[:, None] * self.d ** 0.5
        F = torch.nn.functional
        for i in range(self.blocks):
            h = h + F.layer_norm(h, (self.d,), p[f"w{i}"], p[f"b{i}"], 1e-5) @ p[f"p{i}"].t()
        z = torch.log_softmax(F.layer_norm(h, (self.d,)) @ p["table"].t(), -1)
        loss = -z[real].gather(1, targets[real][:, None]).sum() / real.sum()
        names = list(p)
        return loss.detach(), dict(zip(names, torch.autograd.grad(loss, [p[k] for k in names])))


def _batch(n, vocab, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    ids = torch.randint(0, vocab, (n,), generator=g, device="cuda") % 40            # tokens repeat
    targets = torch.randint(0, vocab, (n,), generator=g, device="cuda")
    ids[-n // 8:], targets[-n // 8:] = -1, -1                                      # a padded batch
    return ids, targets


@pytest.mark.parametrize("vocab,d,blocks,n", [(1001, 128, 2, 96), (250, 64, 1, 64), (5003, 512, 2, 200)])
def test_training_step_with_tied_weights(vocab, d, blocks, n):
    """Gradients against float64.  Every activation and gradient between two calls is rounded to bf16, 2^-8 of its size: with b blocks some 4 b + 5
    such roundings lie on the way of a gradient, independent ones, each of at most 2^-8 / sqrt(3) in the root mean square; the norms and the softmax
    pass a relative error on at most about twofold: 2 sqrt(4 b + 5) 2^-8 of a gradient's norm."""
    import tyr_amd
    m = Tied(vocab, d, blocks, 1)
    ids, targets = _batch(n, vocab, 2)
    loss, grads = m.gradients(ids, targets)
    want_loss, want = m.reference(ids, targets)
    assert abs(float(loss) - float(want_loss)) <= 2.0 ** -6
    for k, g in grads.items():
        off = float((g.double() - want[k]).norm() / want[k].norm())
        assert off <= 2.0 * (4 * blocks + 5) ** 0.5 * BF16, (k, off)
    # the step: masters and their bf16 copies move against the gradient
    for k, g in grads.items():
        new, low = tyr_amd.sgd_step(m.master[k].contiguous(), g, 0.1)
        assert torch.equal(new, m.master[k] - g.float() * 0.1) and torch.equal(low, new.bfloat16())


def test_training_step_captured_and_replayed():
    """A step in a graph, replayed with other tokens and eager steps between: the bits of the eager step."""
    m = Tied(600, 128, 2, 3)
    ids, targets = _batch(80, 600, 4)
    static_ids, static_targets = ids.clone(), targets.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        m.gradients(static_ids, static_targets)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, grads = m.gradients(static_ids, static_targets)
    for k in range(4):
        ids, targets = _batch(80, 600, 10 + k)
        want_loss, want = m.gradients(ids, targets)
        static_ids.copy_(ids)
        static_targets.copy_(targets)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(loss, want_loss)
        for name in want:
            assert torch.equal(grads[name], want[name]), (k, name)


@pytest.mark.parametrize("n,vocab", [(300, 500), (9000, 1000)])
def test_large_and_small_sorts_captured_and_replayed(n, vocab):
    import tyr_amd
    g = torch.randn(n, 64, device="cuda").bfloat16()
    ids = torch.randint(-1, vocab, (n,), device="cuda")
    x = torch.randn(3, 100000, device="cuda").bfloat16()
    t = torch.randint(0, 100000, (3,), device="cuda")
    tyr_amd.embedding_bwd(g, ids, vocab)
    tyr_amd.token_logprobs(x, t, top=7)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = tyr_amd.embedding_bwd(g, ids, vocab)
        scored = tyr_amd.token_logprobs(x, t, top=7)
    for k in range(4):
        ids.copy_(torch.randint(-1, 2 if k == 1 else vocab, (n,), device="cuda"))
        x.copy_(torch.randn(3, 100000, device="cuda"))
        want, want_scored = tyr_amd.embedding_bwd(g, ids, vocab), tyr_amd.token_logprobs(x, t, top=7)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and all(torch.equal(a, b) for a, b in zip(scored, want_scored))


def test_calls_on_side_streams():
    """Two streams at once, given by argument and as the current one; scratch of each belongs to its stream."""
    import tyr_amd
    n, vocab = 9000, 300
    gs = [torch.randn(n, 512, device="cuda") for _ in range(2)]
    ids = [torch.randint(-1, vocab, (n,), device="cuda") for _ in range(2)]
    x, t = torch.randn(2, 200000, device="cuda"), torch.tensor([5, 7], device="cuda")
    h, w = torch.randn(3000, 1024, device="cuda").bfloat16(), torch.randn(1024, device="cuda").bfloat16()
    want = [tyr_amd.embedding_bwd(g, i, vocab) for g, i in zip(gs, ids)]
    scored, grads = tyr_amd.token_logprobs(x, t, top=9), tyr_amd.layernorm_residual_bwd(h, h, w)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(3):
        for k, s in enumerate(streams):
            got.append((k, tyr_amd.embedding_bwd(gs[k], ids[k], vocab, stream=s)))
            with torch.cuda.stream(s):
                got.append((2, tyr_amd.token_logprobs(x, t, top=9)))
                got.append((3, tyr_amd.layernorm_residual_bwd(h, h, w)))
    torch.cuda.synchronize()
    for k, out in got:
        if k < 2:
            assert torch.equal(out, want[k])
        else:
            assert all(torch.equal(a, b) for a, b in zip(out, scored if k == 2 else grads))


def test_scoring_step():
    """One token of every sequence: embedding, norm, the head's product, the sampled tokens' log probabilities and the alternatives."""
    import tyr_amd
    m = Tied(3001, 256, 1, 5)
    for batch in (1, 8, 33):
        ids = torch.randint(0, 3001, (batch,), device="cuda")
        h = tyr_amd.embedding(ids, m.low["table"], scale=16.0)
        out, _ = tyr_amd.layernorm_residual(h, None, m.low["w0"], m.low["b0"])
        logits = tyr_amd.gemm_bf16(out, m.padded_table(), trans_b=True)
        logp, lse, entropy, top_logp, top_ids = tyr_amd.token_logprobs(logits, ids, vocab=3001, top=10)
        z = torch.log_softmax(logits[:, :3001].double(), -1)
        # the tolerances of the operator alone: 2^-17 and 2^-23 of numbers below 64
        assert bool(((logp.double() - z.gather(1, ids[:, None])[:, 0]).abs() <= 2.0 ** -16).all())
        assert bool(((top_logp.double() - z.gather(1, top_ids.long())).abs() <= 2.0 ** -16).all())
        assert torch.equal(top_ids.long(), z.sort(dim=-1, descending=True, stable=True).indices[:, :10])
        assert bool(((entropy.double() + (z.exp() * z).sum(-1)).abs() <= 2.0 ** -13).all())
