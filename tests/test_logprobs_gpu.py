"""token_logprobs against the 64-bit restatement (oracle/head_cache_oracle.py).

Tolerance: sums of V positive fp32 terms, each with a relative error of the exponential (its
argument (x - m) log2 e is rounded three times: at most 3 * 2^-24 * 200 / e-folding where
terms count, |x - m| < 30: 2^-17) and tree-summed: ln S is off by at most 2^-17 + 40 * 2^-24
< 1.1e-5, and x - m - ln S adds two roundings of at most max(|x - m|, |logp|) * 2^-24.  The
entropy has the same relative errors in sums of positive terms: 1.5e-5 of itself + 1.1e-5."""
import numpy as np
import pytest
import torch

from oracle import head_cache_oracle as O

pytestmark = pytest.mark.gpu


def check(logits, tokens, top):
    from kernelswift_b200 import ops

    logp, ent, tl, ti = ops.token_logprobs(logits, tokens, top=top)
    x = logits.double().cpu().numpy().reshape(-1, logits.shape[-1])
    tok = tokens.cpu().numpy().reshape(-1)
    for i in range(len(x)):
        a, b, c, d = O.logprobs(x[i], int(tok[i]), top)
        got = float(logp.view(-1)[i])
        lim = 1.1e-5 + 2.0 ** -23 * max(abs(a), np.abs(x[i]).max())
        assert (np.isnan(a) and np.isnan(got)) or got == a or abs(got - a) <= lim, (i, got, a)
        got = float(ent.view(-1)[i])
        assert (np.isnan(b) and np.isnan(got)) or abs(got - b) <= 1.1e-5 + 1.5e-5 * abs(b), (i, got, b)
        if top:
            assert ti.view(-1, top)[i].tolist() == d.tolist(), (i, ti.view(-1, top)[i].tolist(), d.tolist())
            np.testing.assert_allclose(tl.view(-1, top)[i].double().cpu().numpy(), c, rtol=2.0 ** -22,
                                       atol=1.1e-5 + 2.0 ** -23 * np.abs(x[i][np.isfinite(x[i])]).max(initial=0))
    if not top:
        assert tl is None and ti is None
    ops.device_status()
    return logp, ent, tl, ti


@pytest.mark.parametrize("N,V,top", [
    (1, 1, 1), (3, 2, 2), (2, 7, 0), (5, 33, 32), (1, 1000, 5), (7, 32003, 20), (2, 129280, 32), (300, 4099, 1),
    (1, 32768, 3), (1, 32769, 3), (3, 16385, 8), (1, 262145, 20), (1, 600011, 32),
])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("pad", [0, 3])
def test_values(cuda_ok, N, V, top, dtype, pad):
    g = torch.Generator(device="cuda").manual_seed(N * 7 + V)
    wide = (3 * torch.randn(N, V + pad, device="cuda", generator=g)).to(dtype)
    wide[:, V:] = 100.0
    tokens = torch.randint(0, V, (N,), device="cuda", generator=g)
    check(wide[:, :V], tokens, top)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_orders_that_are_hard_to_search(cuda_ok, dtype):
    """Sorted rows, equal values, few finite ones, zeros of both signs, steps: ties go to the
    lowest index."""
    V, top = 50001, 32
    at = torch.arange(V, device="cuda").float()
    x = torch.stack([at / V * 20, -at / V * 20, torch.zeros(V, device="cuda"), torch.full((V,), -3.0, device="cuda"),
                     torch.floor(at / 1000), -torch.floor(at / 1000), torch.where(at % 2 == 0, 0.0, -0.0),
                     torch.where(at % 7001 == 5, at / V, float("-inf")), torch.where(at == V - 1, 9.0, 0.0),
                     torch.where(at < 2000, 5.0, at % 5)]).to(dtype)
    check(x, torch.arange(10, device="cuda") * 13, top)
    check(x[:, : 50001 - 8].repeat(1, 14), torch.arange(10, device="cuda") * 13, top)  # several passes
    check(x, torch.arange(10, device="cuda").int(), 1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("low", [float("-inf"), -1e30, "min"])
@pytest.mark.parametrize("V", [300, 20011, 129280])
def test_masked_vocabularies(cuda_ok, dtype, low, V):
    """All but a few tokens at -inf, or at a value that stands for it."""
    g = torch.Generator(device="cuda").manual_seed(V)
    low = torch.finfo(dtype).min if low == "min" else low
    x = torch.full((6, V), low, device="cuda").to(dtype)
    for i, n in enumerate((0, 1, 3, 20, 31, 200)):
        at = torch.randperm(V, device="cuda", generator=g)[:n]
        x[i, at] = torch.randn(n, device="cuda", generator=g).to(dtype)
    if low == float("-inf"):
        x[0, V // 2] = 0
    check(x, torch.randint(0, V, (6,), device="cuda", generator=g), 20)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("big", [1e-30, 1.0, 3e4, 1e30])
def test_any_size(cuda_ok, dtype, big):
    g = torch.Generator(device="cuda").manual_seed(3)
    x = (torch.randn(6, 5003, device="cuda", generator=g) * big).to(dtype)
    x[1] -= 1e3
    x[2, 17] = 200.0
    check(x, torch.full((6,), 17, device="cuda"), 5)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("top", [0, 4])
@pytest.mark.parametrize("V", [9, 40000])
def test_rows_that_are_not_finite(cuda_ok, dtype, top, V):
    """NaN and infinities stay in their rows; masked tokens (-inf) have log probability -inf."""
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn(8, V, device="cuda", generator=g).to(dtype)
    inf, nan = float("inf"), float("nan")
    x[1, 3] = nan
    x[2, 3] = inf
    x[3] = -inf
    x[4, 2:] = -inf
    x[5] = -inf
    x[5, V - 1] = nan
    x[6, 1] = torch.finfo(dtype).min
    logp, ent, tl, ti = check(x, torch.tensor([0, 3, 3, 3, 3, 3, 1, 2], device="cuda"), top)
    assert logp.isnan().tolist() == [False, True, True, True, False, True, False, False]
    assert logp[4] == -inf and ent[4] > 0


def test_padding_and_tokens_outside_the_vocabulary(cuda_ok):
    from kernelswift_b200 import ops

    x = torch.randn(2, 3, 500, device="cuda")
    tokens = torch.tensor([[4, -1, 499], [0, -7, 2]], device="cuda")
    logp, ent, _, _ = check(x, tokens, 0)
    assert logp[0, 1] == 0 and logp[1, 1] == 0 and (ent > 0).all()
    tokens[1, 2] = 500
    logp, _, _, _ = ops.token_logprobs(x, tokens)
    assert logp[1, 2].isnan() and not logp[1, 0].isnan()
    with pytest.raises(RuntimeError, match="index"):
        ops.device_status()


def test_repeats_streams_and_graphs(cuda_ok):
    from kernelswift_b200 import ops

    g = torch.Generator(device="cuda").manual_seed(9)
    x = torch.randn(5, 70000, device="cuda", generator=g).bfloat16()
    tokens = torch.randint(0, 70000, (5,), device="cuda", generator=g).int()
    first = check(x, tokens, 20)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        second = ops.token_logprobs(x, tokens, top=20)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        third = ops.token_logprobs(x, tokens, top=20)
    graph.replay()
    for a, b, c in zip(first, second, third):
        assert torch.equal(a, b) and torch.equal(a, c)
    assert first[3].dtype == torch.int32
    x.copy_(x.flip(1))
    graph.replay()
    assert torch.equal(third[3], 69999 - first[3]) or not torch.equal(third[0], first[0])


def test_offsets_past_32_bits(cuda_ok):
    from kernelswift_b200 import ops

    N, V = 20000, 129280
    x = torch.zeros(N, V, dtype=torch.bfloat16, device="cuda")
    assert x.numel() > 2 ** 31
    x[-1, 77] = 5.0
    tokens = torch.full((N,), 77, device="cuda")
    logp, ent, tl, ti = ops.token_logprobs(x, tokens, top=1)
    ref = O.logprobs(x[-1].double().cpu().numpy(), 77, 1)
    assert abs(float(logp[-1]) - ref[0]) < 2e-5 and int(ti[-1]) == 77 and int(ti[-2]) == 0
    assert abs(float(logp[0]) + np.log(V)) < 2e-5


def test_no_rows(cuda_ok):
    from kernelswift_b200 import ops

    logp, ent, tl, ti = ops.token_logprobs(torch.empty(0, 100, device="cuda"), torch.empty(0, dtype=torch.int64, device="cuda"), top=3)
    assert logp.shape == (0,) and tl.shape == (0, 3) and ti.shape == (0, 3)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_replay_on_other_logits_gives_theirs(cuda_ok, dtype):
    """The captured call, replayed on other logits and tokens: all four outputs are those of a call of
    its own, which the restatement confirms."""
    from kernelswift_b200 import ops

    g = torch.Generator(device="cuda").manual_seed(19)
    x = torch.randn(5, 70000, device="cuda", generator=g).to(dtype)
    tokens = torch.randint(0, 70000, (5,), device="cuda", generator=g)
    graph = torch.cuda.CUDAGraph()
    ops.token_logprobs(x, tokens, top=20)
    with torch.cuda.graph(graph):
        got = ops.token_logprobs(x, tokens, top=20)
    for i in range(3):
        x.copy_(torch.randn(5, 70000, device="cuda", generator=g) * (i + 1))
        tokens.copy_(torch.randint(0, 70000, (5,), device="cuda", generator=g))
        for out in got:
            out.fill_(-7)
        graph.replay()
        for a, b in zip(got, check(x, tokens, 20)):
            assert torch.equal(a, b)
