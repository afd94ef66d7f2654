"""Refusals of the per-head cache's operators and of token_logprobs (no GPU needed), and the
restatement that their GPU tests compare with, against torch in 64 bits."""
import numpy as np
import pytest
import torch

from kernelswift_b200 import ops
from oracle import head_cache_oracle as O

E4 = torch.float8_e4m3fn


def cache(pages=4, heads=2, page=32, d=64, per=2):
    x8 = torch.zeros(pages, heads, page, d, dtype=torch.uint8).view(E4)
    return [x8, torch.zeros(pages, heads, per), x8.clone(), torch.zeros(pages, heads, per)]


def append_args():
    k = torch.zeros(1, 3, 2, 64, dtype=torch.bfloat16)
    return dict(k=k, v=k.clone(), **dict(zip(("k8", "k_scale", "v8", "v_scale"), cache())),
                page_table=torch.zeros(1, 4, dtype=torch.int32), lens=torch.zeros(1, dtype=torch.int32))


@pytest.mark.parametrize("change,why", [
    (dict(k=torch.zeros(1, 3, 2, 64)), "k must be bfloat16"),
    (dict(k=torch.zeros(3, 2, 64, dtype=torch.bfloat16)), "k must be bfloat16"),
    (dict(v=torch.zeros(1, 2, 2, 64, dtype=torch.bfloat16)), r"k and v must be \[b, t, 2, 64\]"),
    (dict(k=torch.zeros(1, 3, 2, 128, dtype=torch.bfloat16)[..., ::2]), "together"),
    (dict(v=torch.zeros(1, 3, 4, 64, dtype=torch.bfloat16)[:, :, ::2]), "together"),
    (dict(k8=torch.zeros(4, 2, 32, 64)), "k8 and v8"),
    (dict(k_scale=torch.zeros(4, 2, 2).double()), "k_scale and v_scale"),
    (dict(v_scale=torch.zeros(4, 2, 1)), "k_scale and v_scale"),
    (dict(k_scale=torch.zeros(4, 2, 5), v_scale=torch.zeros(4, 2, 5)), "blocks"),
    (dict(page_table=torch.zeros(2, 4, dtype=torch.int32)), "page_table"),
    (dict(page_table=torch.zeros(1, 4, dtype=torch.int64)), "page_table"),
    (dict(lens=torch.zeros(2, dtype=torch.int32)), "lens"),
    (dict(n_new=torch.zeros(1)), "n_new"),
    (dict(freqs=torch.zeros(10, 32)), "freqs"),
    (dict(positions=torch.zeros(1, 4, dtype=torch.int32)), "positions"),
    (dict(q=torch.zeros(1, 2, 4, 64, dtype=torch.bfloat16)), "tokens of k"),
    (dict(q=torch.zeros(1, 3, 4, 32, dtype=torch.bfloat16)), "q must be bfloat16"),
    (dict(), "CUDA"),
])
def test_append_refuses(change, why):
    with pytest.raises(RuntimeError, match=why):
        ops.kv_append(**{**append_args(), **change})


@pytest.mark.parametrize("change,why", [
    (dict(q=torch.zeros(1, 3, 4, 64)), "q must be bfloat16"),
    (dict(q=torch.zeros(1, 3, 3, 64, dtype=torch.bfloat16)), "multiple of 2"),
    (dict(q=torch.zeros(1, 3, 4, 128, dtype=torch.bfloat16)), r"q must be \[b, t, h, 64\]"),
    (dict(mask=torch.zeros(1, 3, 4, dtype=torch.bool)), "mask"),
    (dict(mask=torch.zeros(1, 3, 3)), "mask"),
    (dict(attn_sink=torch.zeros(2)), "attn_sink"),
    (dict(n_new=torch.zeros(2, dtype=torch.int32)), "n_new"),
    (dict(lens=torch.zeros(1)), "lens"),
    (dict(v_scale=torch.zeros(4, 2, 4)), "k_scale and v_scale"),
    (dict(), "CUDA"),
])
def test_attention_refuses(change, why):
    args = append_args()
    del args["k"], args["v"]
    args["q"] = torch.zeros(1, 3, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match=why):
        ops.kv_attn(**{**args, "softmax_scale": 0.1, **change})


@pytest.mark.parametrize("logits,tokens,why", [
    (torch.zeros(2, 5).half(), torch.zeros(2, dtype=torch.int64), "logits must be"),
    (torch.zeros(2, 5), torch.zeros(3, dtype=torch.int64), "one per row"),
    (torch.zeros(2, 5), torch.zeros(2), "tokens must be"),
    (torch.zeros(4, 2, 5).transpose(0, 1)[:, ::2], torch.zeros(2, 2, dtype=torch.int64), "constant stride"),
    (torch.zeros(2, 5), torch.zeros(2, dtype=torch.int64), "CUDA"),
])
def test_logprobs_refuses(logits, tokens, why):
    with pytest.raises(RuntimeError, match=why):
        ops.token_logprobs(logits, tokens)


@pytest.mark.parametrize("lens,n,block", [(0, 40, 16), (5, 1, 16), (13, 70, 32), (31, 2, 16)])
def test_appended_rows_read_back_within_half_a_step(lens, n, block):
    """4 significant bits: half a step is at most 2^-4 of the value, or 2^-10 of the scale
    (half of e4m3's smallest number); a row rounded again adds the same once more."""
    rng = np.random.default_rng(lens + n)
    heads, d, page = 2, 64, 32
    codes, scale = np.zeros((8, heads, page, d), np.uint8), np.zeros((8, heads, page // block))
    table = rng.permutation(8)
    x = rng.standard_normal((lens + n, heads, d)).astype(np.float32)
    if lens:
        O.append(x[:lens], codes, scale, table, 0, block)
    O.append(x[lens:], codes, scale, table, lens, block)
    back = O.head_rows(codes, scale, table, lens + n)
    pos = np.arange(lens + n)
    s = scale[table[pos // page], :, pos % page // block][..., None]
    once = pos[:, None, None] >= lens
    lim = np.where(once, 1.0, 2.0 + 2.0 ** -4) * np.maximum(np.abs(x) * 2.0 ** -4, s * 2.0 ** -10)
    assert (np.abs(back - x) <= lim).all()
    # power-of-two scales that the largest element needs
    top = np.abs(x[lens:]).max()
    assert (np.log2(scale[scale > 0]) % 1 == 0).all() and scale.max() <= 2 * np.abs(x).max() / 448 and top <= 448 * scale.max()


def test_rotation_keeps_lengths_and_turns_by_positions():
    rng = np.random.default_rng(0)
    x = rng.standard_normal((6, 2, 16))
    ang = np.outer(np.arange(9), [1.0, 0.1, 0.01])
    fr = np.stack([np.cos(ang), np.sin(ang)], -1)
    y = O.rotate(x, fr, np.array([0, 1, 2, 3, 8, 8]))
    assert np.array_equal(y[..., :10], x[..., :10].astype(np.float32)) and np.allclose(y[0], x[0])
    assert np.allclose((y[..., 10:] ** 2).sum(-1), (x[..., 10:] ** 2).sum(-1))
    # the product of two rotated rows depends on their distance alone
    a, b = x[:1].repeat(2, 0), x[1:2].repeat(2, 0)
    ra, rb = O.rotate(a, fr, np.array([2, 6])), O.rotate(b, fr, np.array([1, 5]))
    assert np.allclose((ra * rb).sum(-1)[0], (ra * rb).sum(-1)[1], atol=1e-5)


def test_logprob_restatement_agrees_with_torch():
    x = torch.randn(4, 300, dtype=torch.float64)
    x[1, 5:] = -float("inf")
    lp = torch.log_softmax(x, -1)
    for i in range(4):
        a, b, c, d = O.logprobs(x[i].numpy(), 3, 4)
        p = lp[i].exp()
        assert np.isclose(a, lp[i, 3]) and np.isclose(b, -(torch.where(p > 0, p * lp[i], 0.0)).sum())
        assert np.allclose(c, lp[i].topk(4).values) and d.tolist() == lp[i].topk(4).indices.tolist()


@pytest.mark.parametrize("first", [False, True])
def test_models_that_rotate_halves_permute_their_projections(first):
    """Rotation of halves (i, i + rd/2), of a head's last or first columns: with the columns of queries
    and keys permuted alike, the rotation of pairs at the end gives the same scores."""
    rng = np.random.default_rng(3)
    d, rd, n = 24, 16, 7
    q, k = rng.standard_normal((2, n, 1, d)).astype(np.float32)
    ang = np.outer(np.arange(n), 0.3 ** np.arange(rd // 2))
    fr = np.stack([np.cos(ang), np.sin(ang)], -1)
    at = 0 if first else d - rd

    def halves(x):
        y = x.astype(np.float64)
        a, b = x[..., at:at + rd // 2], x[..., at + rd // 2:at + rd]
        c, s = fr[:, None, :, 0], fr[:, None, :, 1]
        y[..., at:at + rd // 2], y[..., at + rd // 2:at + rd] = a * c - b * s, a * s + b * c
        return y[:, 0]

    rest = [i for i in range(d) if not at <= i < at + rd]
    order = rest + [at + i // 2 + (i % 2) * (rd // 2) for i in range(rd)]
    pairs = [O.rotate(x[..., order], fr, np.arange(n)).astype(np.float64)[:, 0] for x in (q, k)]
    # (fp32 rotation: 2^-22 of the sums' terms)
    assert np.allclose(pairs[0] @ pairs[1].T, halves(q) @ halves(k).T, atol=2.0 ** -22 * d * 20)
