"""The cache, tree attention and verification together, as examples/speculative_decode.py
runs them: the cache a speculative run leaves is the one that decoding the same tokens one
by one leaves, and a tree's probabilities are those of decoding along its path."""
import os
import sys

import pytest
import torch

from conftest import ROOT

sys.path.insert(0, os.path.join(ROOT, "examples"))
pytestmark = pytest.mark.gpu


def test_speculative_steps_leave_the_cache_of_plain_decoding(cuda_ok):
    import speculative_decode as S
    from kernelswift_b200 import ops

    model, g = S.ToyModel(), torch.Generator(device="cuda").manual_seed(3)
    B, n = 3, 40
    parents = torch.tensor([-1, -1, 0, 0, 1, 2, 2, 5])
    fast, slow = S.Cache(model, B, 200), S.Cache(model, B, 200)
    prompt = torch.randint(0, model.vocab, (B, n), device="cuda", generator=g)
    last = S.prefill(model, fast, prompt)
    tokens = [prompt[b].tolist() for b in range(B)]
    accepted = 0
    for _ in range(6):
        new, stood = S.step(model, fast, last, parents, g)
        for b in range(B):
            tokens[b] += new[b, : int(stood[b]) + 1].tolist()
        last = new.gather(1, stood.long()[:, None])[:, 0]
        accepted += int(stood.sum())
    assert accepted > 0                    # else no path was ever moved
    ops.device_status()
    assert fast.lens.tolist() == [len(t) - 1 for t in tokens]
    assert all(0 <= x < model.vocab for t in tokens for x in t)
    # the same tokens cached at once
    for b in range(B):
        seq = torch.tensor(tokens[b][:-1], device="cuda")[None].expand(B, -1).contiguous()
        pos = torch.arange(seq.shape[1], device="cuda").expand_as(seq)
        slow.write(model.queries_and_latents(seq, pos)[1], pos.contiguous())
        slow.lens = fast.lens[b].expand(B).contiguous()
        m = int(fast.lens[b])
        assert torch.equal(fast.rows()[b, :m], slow.rows()[b])


def test_tree_probabilities_are_those_of_decoding_along_each_path(cuda_ok):
    """Output columns and scores go through the same codes; what differs is how the weights
    are cut into tiles: bf16 results within one rounding, so logits within 2^-7 of their
    scale."""
    import speculative_decode as S

    model, g = S.ToyModel(seed=2), torch.Generator(device="cuda").manual_seed(5)
    prompt = torch.randint(0, model.vocab, (1, 30), device="cuda", generator=g)
    parents = torch.tensor([-1, 0, 0, 1, -1])
    drafted = torch.randint(0, model.vocab, (1, 5), device="cuda", generator=g)
    cache = S.Cache(model, 1, 100)
    last = S.prefill(model, cache, prompt)
    depth, mask = S.tree(torch.cat([torch.tensor([-1]), parents + 1]))
    toks = torch.cat([last[:, None], drafted], 1)
    n = cache.lens.long()[:, None]
    q, kv = model.queries_and_latents(toks, n + depth)
    cache.write(kv, n + torch.arange(6, device="cuda"))
    whole = cache.attend(q, model, mask[None].contiguous()).float()
    for node in range(6):
        way = mask[node].nonzero()[:, 0]
        one = S.Cache(model, 1, 100)
        S.prefill(model, one, prompt)
        one.write(kv[:, way].contiguous(), n + torch.arange(len(way), device="cuda"))
        alone = one.attend(q[:, way].contiguous(), model).float()[:, -1]
        diff = (whole[:, node] - alone).abs()
        assert (diff <= 2.0 ** -7 * alone.abs().amax()).all(), float(diff.max())
