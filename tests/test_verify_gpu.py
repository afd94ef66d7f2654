"""verify_draft against the restatement (oracle/cache_oracle.py): tokens, counts and
paths have to be equal, since every decision is one rounded operation on the inputs."""
import numpy as np
import pytest
import torch

from oracle import cache_oracle as C

pytestmark = pytest.mark.gpu


def inputs(B, T, V, seed, spread=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    logits = spread * torch.randn(B, T + 1, V, device="cuda", generator=g)
    p = torch.softmax(logits, -1)
    u = torch.rand(B, T + 1, device="cuda", generator=g)
    noise = torch.empty(B, V, device="cuda").exponential_(generator=g).clamp_min_(1e-10)
    return g, logits, p, u, noise


def same(got, ref, tokens):
    out, n, path = (x.cpu().numpy() for x in got)
    B, T = tokens.shape
    for b in range(B):
        toks, way = ref(b)
        assert n[b] == len(way), b
        assert out[b].tolist() == toks + [-1] * (T + 1 - len(toks)), b
        assert path[b].tolist() == way + [-1] * (T - len(way)), b


@pytest.mark.parametrize("B,T,V", [(1, 1, 1), (1, 3, 32003), (5, 7, 1000), (3, 0, 77), (40, 4, 4099), (2, 12, 129280),
                                   (700, 2, 130), (17, 5, 65536)])
@pytest.mark.parametrize("dtype", [torch.int64, torch.int32])
def test_sampled_chain(cuda_ok, B, T, V, dtype):
    from kernelswift_b200 import ops

    g, logits, p, u, noise = inputs(B, T, V, B + V)
    q = torch.softmax(logits[:, :T] + 0.5 * torch.randn(B, T, V, device="cuda", generator=g), -1)
    tokens = torch.multinomial(q.view(-1, V), 1, generator=g).view(B, T) if T else torch.zeros(B, 0, device="cuda")
    tokens = tokens.to(dtype)
    got = ops.verify_draft(p, tokens, u, noise, q=q)
    ops.device_status()
    assert got[0].dtype == dtype
    pn, qn, tn, un, en = (x.cpu().numpy() for x in (p, q, tokens, u, noise))
    same(got, lambda b: C.verify_chain(pn[b], qn[b], tn[b].tolist(), un[b], en[b]), tokens)


def random_tree(g, B, T, deep):
    at = torch.arange(T, device="cuda")
    parents = torch.floor(torch.rand(B, T, device="cuda", generator=g) * (at + 1)).long() - 1
    follow = torch.rand(B, T, device="cuda", generator=g) < deep
    return torch.where(follow, at - 1, parents).int().contiguous()


@pytest.mark.parametrize("B,T,V,deep,kinds", [
    (1, 1, 1, 0.0, 1), (4, 9, 50, 0.5, 50), (3, 40, 129280, 0.5, 8), (64, 13, 1001, 0.3, 6),
    (2, 300, 5000, 0.2, 40), (1, 1024, 600, 0.1, 600), (5, 6, 32000, 1.0, 3), (9, 20, 64, 0.0, 5)])
def test_fixed_candidates(cuda_ok, B, T, V, deep, kinds):
    """Trees whose tokens come from the `kinds` likeliest: siblings repeat tokens too."""
    from kernelswift_b200 import ops

    g, _, p, u, noise = inputs(B, T, V, T + V, spread=6.0)
    parents = random_tree(g, B, T, deep)
    top = p.topk(min(kinds, V), -1).indices
    pick = torch.randint(0, min(kinds, V), (B, T), device="cuda", generator=g)
    rows = torch.arange(B, device="cuda")[:, None]
    tokens = top[rows, parents.long() + 1, pick].contiguous()
    got = ops.verify_draft(p, tokens, u, noise, parents=parents)
    ops.device_status()
    pn, tn, an, un, en = (x.cpu().numpy() for x in (p, tokens, parents, u, noise))
    same(got, lambda b: C.verify_tree(pn[b], tn[b].tolist(), an[b].tolist(), un[b], en[b]), tokens)


def test_chain_of_fixed_candidates_is_the_default(cuda_ok):
    from kernelswift_b200 import ops

    _, _, p, u, noise = inputs(6, 5, 300, 3, spread=8.0)
    tokens = p[:, :5].argmax(-1)
    chain = torch.arange(-1, 4, device="cuda").int().expand(6, 5).contiguous()
    a, b = ops.verify_draft(p, tokens, u, noise), ops.verify_draft(p, tokens, u, noise, parents=chain)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert int(a[1].max()) > 0


def test_edges_of_the_decisions(cuda_ok):
    """u = 0, probabilities of 0 and 1, equal rows, ties, a leaf at the end of the walk."""
    from kernelswift_b200 import ops

    V = 8
    one = torch.zeros(1, 3, V, device="cuda")
    one[0, :, 5] = 1.0
    noise, u = torch.ones(1, V, device="cuda"), torch.zeros(1, 3, device="cuda")
    tok = torch.tensor([[5, 5]], device="cuda")
    # p = q = certain: everything stands, the next token is certain too
    out, n, path = ops.verify_draft(one, tok, u, noise, q=one[:, :2].contiguous())
    assert out.tolist() == [[5, 5, 5]] and n.tolist() == [2] and path.tolist() == [[0, 1]]
    out, n, path = ops.verify_draft(one, tok, u, noise)
    assert out.tolist() == [[5, 5, 5]] and n.tolist() == [2] and path.tolist() == [[0, 1]]
    # a token of probability 0 falls even at u = 0; q > p nowhere: w = 0, so p's row decides
    out, n, _ = ops.verify_draft(one, torch.tensor([[2, 5]], device="cuda"), u, noise, q=one[:, :2].contiguous())
    assert out.tolist() == [[5, -1, -1]] and n.tolist() == [0]
    # ties go to the lowest token
    flat = torch.full((1, 1, V), 1 / V, device="cuda")
    out, n, path = ops.verify_draft(flat, torch.empty(1, 0, dtype=torch.int64, device="cuda"), u[:, :1].contiguous(), noise)
    assert out.tolist() == [[0]] and n.tolist() == [0] and path.shape == (1, 0)
    # every token is a rejected child: p's row takes the place of the empty rest
    p = torch.full((1, V + 1, V), 1 / V, device="cuda")
    p[0, 0, 0] = 0.0  # the children's stretches end at 7/8
    uu = torch.full((1, V + 1), 0.95, device="cuda")
    par = torch.full((1, V), -1, dtype=torch.int32, device="cuda")
    out, n, _ = ops.verify_draft(p, torch.arange(V, device="cuda")[None], uu, noise, parents=par)
    assert n.tolist() == [0] and out[0, 0].item() == 1


def test_invalid_tokens_and_parents_are_reported(cuda_ok):
    from kernelswift_b200 import ops

    _, _, p, u, noise = inputs(1, 3, 100, 5)
    u.zero_()  # everything valid of positive probability stands in a chain
    good = torch.tensor([[4, 5, 6]], device="cuda")
    assert ops.verify_draft(p, good, u, noise)[1].tolist() == [3]
    ops.device_status()
    for tok, par, n in (([4, 100, 6], [-1, 0, 1], 1), ([-1, 5, 6], [-1, 0, 1], 0), ([4, 5, 6], [-1, 1, 0], None),
                        ([4, 5, 6], [-2, 0, 1], 0), ([4, 5, 6], [-1, 0, 3], 2)):
        got = ops.verify_draft(p, torch.tensor([tok], device="cuda"), u, noise,
                               parents=torch.tensor([par], dtype=torch.int32, device="cuda"))
        with pytest.raises(RuntimeError, match="device status"):
            ops.device_status()
        if n is not None:
            assert got[1].tolist() == [n]


@pytest.mark.parametrize("kind", ["chain", "tree"])
def test_next_token_has_the_targets_distribution(cuda_ok, kind):
    """40000 sequences of one vocabulary of 6: the first emitted token is distributed as
    p's row 0, whatever was drafted.  Counts of a binomial are within 5 standard
    deviations (a chance of 6e-7 each)."""
    from kernelswift_b200 import ops

    B, V, T = 40000, 6, 3
    g = torch.Generator(device="cuda").manual_seed(11)
    p1 = torch.tensor([0.35, 0.05, 0.2, 0.1, 0.3, 0.0], device="cuda")
    q1 = torch.tensor([0.1, 0.3, 0.2, 0.2, 0.1, 0.1], device="cuda")
    p, q = p1.expand(B, T + 1, V).contiguous(), q1.expand(B, T, V).contiguous()
    u = torch.rand(B, T + 1, device="cuda", generator=g)
    noise = torch.empty(B, V, device="cuda").exponential_(generator=g)
    if kind == "chain":
        tok = torch.multinomial(q1.expand(B, V), T, replacement=True, generator=g)
        out = ops.verify_draft(p, tok, u, noise, q=q)[0]
    else:
        tok = torch.tensor([1, 4, 2], device="cuda").expand(B, T).contiguous()
        par = torch.tensor([-1, -1, 1], dtype=torch.int32, device="cuda").expand(B, T).contiguous()
        out = ops.verify_draft(p, tok, u, noise, parents=par)[0]
    counts = torch.bincount(out[:, 0], minlength=V).double().cpu().numpy()
    pp = p1.double().cpu().numpy()
    assert (np.abs(counts - B * pp) <= 5 * np.sqrt(B * pp * (1 - pp))).all(), counts


def test_refusals(cuda_ok):
    from kernelswift_b200 import ops

    _, _, p, u, noise = inputs(2, 3, 50, 1)
    tok, q = torch.zeros(2, 3, dtype=torch.int64, device="cuda"), p[:, :3].contiguous()
    par = torch.full((2, 3), -1, dtype=torch.int32, device="cuda")
    for call, why in [
        (lambda: ops.verify_draft(p.half(), tok, u, noise), "p must be"),
        (lambda: ops.verify_draft(p[:, :3].contiguous(), tok, u, noise), "p must be"),
        (lambda: ops.verify_draft(p, tok.float(), u, noise), "tokens"),
        (lambda: ops.verify_draft(p, tok, u[:, :3].contiguous(), noise), "u must be"),
        (lambda: ops.verify_draft(p, tok, u, noise[:, :9].contiguous()), "noise"),
        (lambda: ops.verify_draft(p, tok, u, noise, q=p), "q must be"),
        (lambda: ops.verify_draft(p, tok, u, noise, parents=par.long()), "parents"),
        (lambda: ops.verify_draft(p, tok, u, noise, q=q, parents=par), "exclude"),
        (lambda: ops.verify_draft(p.cpu(), tok, u, noise), "CUDA"),
        (lambda: ops.verify_draft(p.transpose(1, 2).contiguous().transpose(1, 2), tok, u, noise), "contiguous"),
    ]:
        with pytest.raises(RuntimeError, match=why):
            call()


def test_a_refused_call_leaves_the_next_alone(cuda_ok):
    """Whatever a large call is told, an ordinary one after it works."""
    from kernelswift_b200 import ops

    p, noise = torch.full((1, 2, 5_000_000), 1e-7, device="cuda"), torch.ones(1, 5_000_000, device="cuda")
    tok, u = torch.zeros(1, 1, dtype=torch.int64, device="cuda"), torch.full((1, 2), 0.5, device="cuda")
    for _ in range(2):
        try:
            ops.verify_draft(p, tok, u, noise)
        except RuntimeError:
            pass
        assert ops.verify_draft(p[..., :9].contiguous(), tok, u, noise[:, :9].contiguous())[1].tolist() == [0]
        ops.device_status()


@pytest.mark.parametrize("B,V", [(300, 1_400_000), (1, 20_000_003)])
def test_fixed_candidates_of_large_vocabularies(cuda_ok, B, V):
    """The batch does not limit the vocabulary.  Tokens at powers of two from a rejected
    child stay in the draw, the child does not."""
    from kernelswift_b200 import ops

    T = 3
    g = torch.Generator(device="cuda").manual_seed(5)
    p = torch.rand(B, T + 1, V, device="cuda", generator=g).mul_(1e-9)
    tokens = torch.randint(0, V // 2, (B, T), device="cuda", generator=g)
    at = torch.arange(B, device="cuda")
    other = tokens[:, 0] + 2 ** (14 + at % 6)
    p[at, 0, other] = 0.25
    p[at[:, None], 0, tokens] = 0.2       # the children of the root: likelier than all but `other`
    p[at, 1, V - 1] = 0.5
    u = torch.full((B, T + 1), 0.99, device="cuda")
    u[::3, 0] = 0.1                       # taken: the first child, whose own row then gives V - 1
    noise = torch.ones(B, V, device="cuda")
    parents = torch.full((B, T), -1, dtype=torch.int32, device="cuda")
    out, n, path = ops.verify_draft(p, tokens, u, noise, parents=parents)
    ops.device_status()
    took = at % 3 == 0
    alike = (tokens == other[:, None]).any(1)  # (then it is a child itself)
    assert torch.equal(n, took.int()) and torch.equal(path[:, 0], torch.where(took, 0, -1).int())
    assert (out[took, 0] == tokens[took, 0]).all() and (out[took, 1] == V - 1).all()
    fine = ~took & ~alike
    assert (out[fine, 0] == other[fine]).all()
    assert not (out[~took, :1] == tokens[~took]).any()


def test_many_siblings_of_a_large_vocabulary(cuda_ok):
    """1024 siblings that are the likeliest entries: the draw passes all of them over."""
    from kernelswift_b200 import ops

    V, T = 5_000_000, 1024
    p = torch.full((1, T + 1, V), 1e-9, device="cuda")
    tokens = (torch.arange(T, device="cuda") * 4801 + 17)[None].contiguous()
    p[0, 0, tokens[0]] = 0.0005
    p[0, 0, 3_000_000] = 2e-9
    par = torch.full((1, T), -1, dtype=torch.int32, device="cuda")
    u = torch.full((1, T + 1), 0.9, device="cuda")
    out, n, _ = ops.verify_draft(p, tokens, u, torch.ones(1, V, device="cuda"), parents=par)
    ops.device_status()
    assert n.tolist() == [0] and out[0, 0].item() == 3_000_000


@pytest.mark.parametrize("small", [3e-17, 1e-18, 7e-17])
@pytest.mark.parametrize("count", [1, 40, 300])
def test_stretches_leave_no_gap(cuda_ok, small, count):
    """Children too small for fp64 to tell their stretches' ends apart, and a u on the edge
    before them: u is below the children's sum, so exactly one child is taken, one whose
    stretch lies within the sum's rounding of u."""
    from kernelswift_b200 import ops

    T, V = count + 2, 400
    p = torch.zeros(1, T + 1, V, device="cuda")
    p[0, 0, 0], p[0, 0, 1 : count + 1], p[0, 0, count + 1] = 0.5, small, 0.25
    p[0, 1:, 399] = 1.0
    u = torch.full((1, T + 1), 0.5, device="cuda")
    par = torch.full((1, T), -1, dtype=torch.int32, device="cuda")
    for _ in range(3):
        out, n, path = ops.verify_draft(p, torch.arange(T, device="cuda")[None], u,
                                        torch.ones(1, V, device="cuda"), parents=par)
        assert n.tolist() == [1] and 1 <= path[0, 0].item() <= T - 1
        assert out[0, :2].tolist() == [path[0, 0].item(), 399]
