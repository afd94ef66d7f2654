"""kv_append, kv_attn, verify_draft and token_logprobs as a server runs them: a ragged prompt in one
call, drafted tokens verified, single tokens, the whole step in a CUDA graph."""
import pytest
import torch

import test_kv_attn_gpu as A

pytestmark = pytest.mark.gpu

B, H, HEADS, D, V, BLOCK, PAGE = 3, 8, 2, 128, 1009, 16, 32


class Layer:
    """One attention layer over the per-head cache: token -> rows -> attention -> logits."""

    def __init__(self, seed=0, pages=40):
        g = torch.Generator(device="cuda").manual_seed(seed)
        rnd = lambda *s, scale: (torch.randn(*s, device="cuda", generator=g) * scale).bfloat16()  # noqa: E731
        self.embed, self.out = rnd(V, 256, scale=1.0), rnd(1024, H * D, scale=(H * D) ** -0.5)  # a padded vocabulary
        self.qkv = rnd((H + 2 * HEADS) * D, 256, scale=256 ** -0.5)
        code = lambda: torch.zeros(pages, HEADS, PAGE, D, dtype=torch.uint8, device="cuda").view(A.E4)  # noqa: E731
        scale = lambda: torch.zeros(pages, HEADS, PAGE // BLOCK, device="cuda")  # noqa: E731
        self.cache = [code(), scale(), code(), scale()]
        self.table = torch.randperm(pages, device="cuda", generator=g)[: B * 12].view(B, 12).int().contiguous()
        self.lens = torch.zeros(B, dtype=torch.int32, device="cuda")
        ang = torch.outer(torch.arange(12 * PAGE).double(), 10000.0 ** (-torch.arange(0, 64, 2).double() / 64))
        self.freqs = torch.stack([ang.cos(), ang.sin()], -1).float().cuda().contiguous()

    def step(self, tokens, n_new=None, positions=None, mask=None):
        """(queries, attended, logits) of T tokens per sequence; their rows are cached at lens .."""
        from kernelswift_b200 import ops

        rows = ops.proj_rope(self.embed[tokens].contiguous(), self.qkv).unflatten(-1, (H + 2 * HEADS, D))
        q, k, v = rows.split([H, HEADS, HEADS], 2)
        q = ops.kv_append(k, v, *self.cache, self.table, self.lens, freqs=self.freqs, positions=positions,
                          n_new=n_new, q=q)
        o = ops.kv_attn(q, *self.cache, self.table, self.lens, D ** -0.5, mask=mask, n_new=n_new)
        return q, o, ops.proj_rope(o.flatten(2), self.out)[..., :V]


def test_prompt_draft_and_single_tokens(cuda_ok):
    from kernelswift_b200 import ops

    m, g = Layer(), torch.Generator(device="cuda").manual_seed(1)
    # a prompt of 70, 33 and 1 tokens in one padded call
    new = torch.tensor([70, 33, 1], dtype=torch.int32, device="cuda")
    prompt = torch.randint(0, V, (B, 70), device="cuda", generator=g)
    q, o, logits = m.step(prompt, n_new=new)
    A.check(q, m.cache, m.table, m.lens, D ** -0.5, got=o, n_new=new)
    # token by token over the same cache: the other kernel, the same weights
    for t in (0, 17, 32):
        one = ops.kv_attn(q[:, t:t + 1].contiguous(), *m.cache, m.table, m.lens + t, D ** -0.5)
        for b in range(B):
            if t < int(new[b]):
                assert torch.allclose(one[b, 0].float(), o[b, t].float(), rtol=2.0 ** -6, atol=2.0 ** -6 * float(o[b, t].abs().max()))
    m.lens += new
    last = logits[torch.arange(B), new.long() - 1].float().argmax(-1)
    # five drafted tokens: a tree of two branches behind the newest token
    parents = torch.tensor([-1, 0, -1, 2, 2], device="cuda")
    drafted = torch.randint(0, V, (B, 5), device="cuda", generator=g)
    up = torch.eye(6, dtype=torch.bool, device="cuda")
    for i, par in enumerate(parents.tolist()):
        up[i + 1] |= up[par + 1]
    depth = up.sum(1) - 1
    mask = up[None].repeat(B, 1, 1).contiguous()
    tokens = torch.cat([last[:, None], drafted], 1)
    pos = (m.lens[:, None] + depth).int().contiguous()
    q, o, logits = m.step(tokens, positions=pos, mask=mask)
    A.check(q, m.cache, m.table, m.lens, D ** -0.5, got=o, mask=mask)
    p = torch.softmax(logits.float(), -1)
    u = torch.rand(B, 6, device="cuda", generator=g) * 0.02  # low: candidates often stand
    noise = torch.empty(B, V, device="cuda").exponential_(generator=g)
    out, stood, path = ops.verify_draft(p, drafted, u, noise, parents=parents.int().repeat(B, 1))
    # what the new tokens' log probabilities are: of the row that each was chosen from
    rows = torch.cat([torch.zeros(B, 1, dtype=torch.long, device="cuda"), path.long() + 1], 1).clamp_min(0)
    chosen = logits.gather(1, rows[..., None].expand(-1, -1, V)).contiguous()
    logp, entropy, top_logp, top_ids = ops.token_logprobs(chosen, out, top=3)
    want = torch.log_softmax(chosen.double(), -1)
    ref = torch.where(out < 0, 0.0, want.gather(2, out.clamp_min(0)[..., None])[..., 0])
    assert torch.allclose(logp.double(), ref, atol=2e-5) and (logp[out < 0] == 0).all() and (out < 0).any()
    assert torch.allclose(entropy.double(), -(want.exp() * want).sum(-1), atol=2e-5)
    assert torch.allclose(top_logp.double(), want.sort(-1, descending=True).values[..., :3], atol=2e-5)
    # the accepted path's rows once more, where the context goes on; then single tokens
    n = stood + 1
    way = torch.cat([last[:, None], out[:, :5]], 1)
    way = torch.where(torch.arange(6, device="cuda")[None] < n[:, None], way, 0).clamp_min(0)
    m.step(way, n_new=n.int())
    m.lens += n.int()
    last = out.gather(1, stood.long()[:, None])
    for _ in range(20):
        q, o, logits = m.step(last)
        A.check(q, m.cache, m.table, m.lens, D ** -0.5, got=o)
        m.lens += 1
        last = logits[:, 0].float().argmax(-1, keepdim=True)
    ops.device_status()


def test_a_captured_step_decodes_as_an_eager_one(cuda_ok):
    from kernelswift_b200 import ops

    def begin():
        m = Layer(seed=3)
        m.step(torch.arange(B * 20, device="cuda").view(B, 20))
        m.lens += 20
        return m, torch.arange(B, device="cuda")[:, None].contiguous()

    def decode(m, token, logp):
        _, _, logits = m.step(token)
        token.copy_(logits[:, 0].argmax(-1, keepdim=True))
        logp.copy_(ops.token_logprobs(logits, token)[0])
        m.lens += 1

    eager, token = begin()
    logp, want = torch.zeros(B, 1, device="cuda"), []
    for _ in range(30):
        decode(eager, token, logp)
        want.append((token.clone(), logp.clone()))
    m, token = begin()
    logp = torch.zeros(B, 1, device="cuda")
    start = [x.clone() for x in (*m.cache, m.lens, token)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):  # a pass before the capture, taken back below
        decode(m, token, logp)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        decode(m, token, logp)
    for x, y in zip((*m.cache, m.lens, token), start):
        x.copy_(y)
    for a, b in want:
        graph.replay()
        assert torch.equal(token, a) and torch.equal(logp, b)
    assert all(torch.equal(x, y) for x, y in zip(m.cache[1::2] + [m.lens], eager.cache[1::2] + [eager.lens]))
    ops.device_status()


def test_a_captured_step_leaves_the_cache_of_an_eager_one(cuda_ok):
    """Codes and scales, byte by byte, and the log probabilities' alternatives."""
    from kernelswift_b200 import ops

    def begin():
        m = Layer(seed=5)
        m.step(torch.arange(B * 20, device="cuda").view(B, 20))
        m.lens += 20
        return m, torch.arange(B, device="cuda")[:, None].contiguous()

    def decode(m, token, top):
        _, _, logits = m.step(token)
        token.copy_(logits[:, 0].argmax(-1, keepdim=True))
        for x, y in zip(top, ops.token_logprobs(logits, token, top=4)):
            x.copy_(y)
        m.lens += 1

    def outputs():
        at = (B, 1)
        return [torch.zeros(at, device="cuda"), torch.zeros(at, device="cuda"), torch.zeros(*at, 4, device="cuda"),
                torch.zeros(*at, 4, dtype=torch.int64, device="cuda")]

    (eager, token), top = begin(), outputs()
    want = []
    for _ in range(20):
        decode(eager, token, top)
        want.append([x.clone() for x in top])
    (m, token), top = begin(), outputs()
    start = [x.clone() for x in (*m.cache, m.lens, token)]
    decode(m, token, top)  # a pass before the capture, taken back below
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        decode(m, token, top)
    for x, y in zip((*m.cache, m.lens, token), start):
        x.copy_(y)
    for step in want:
        graph.replay()
        assert all(torch.equal(x, y) for x, y in zip(top, step))
    for x, y in zip((*m.cache, m.lens), (*eager.cache, eager.lens)):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    assert any(int((x.view(torch.uint8) != y.view(torch.uint8)).sum()) for x, y in zip(m.cache, start))
    ops.device_status()
