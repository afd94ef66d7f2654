"""Serving over a per-head cache in 8 bits, as cases that can be timed and compared.

Three operators of a decoding step where keys and values are kept per head (grouped queries):

* ``kv_append``      rotates new keys (and queries) to their positions and quantises keys and
  values into a paged e4m3 cache with one power-of-two scale for each block of tokens and head;
* ``kv_attn``        attends from one token, a tree of drafted tokens or a chunk of a prompt over
  that cache;
* ``token_logprobs`` gives the log probabilities of chosen tokens, the entropy of their
  distributions and the likeliest alternatives.

The cache: k8 and v8 e4m3 [pages, heads, page, D], k_scale and v_scale fp32 [pages, heads,
page / block].  With ``own`` false, ``run`` computes each operator from elementary torch
operations in 32 bits; with ``own`` true it calls ``kernelswift_b200.ops``.
"""
import math

import torch

own = False

DEV = "cuda"
VOCAB = 129280  # ModelArgs.vocab_size of the indexer module


# ------------------------------------------------------------------------------ cases
def listed():
    return [
        # one decode step of eight ragged sequences, queries rotated in the same call: latency
        dict(name="append_decode", op="append", batch=8, t=1, h=32, hkv=8, d=128, rd=64, page=64,
             block=16, longest=4000, ragged=True, short=False, fused=False),
        # drafted tokens of many sequences, some with fewer than the call's five, blocks of 32
        dict(name="append_drafts", op="append", batch=37, t=5, h=0, hkv=3, d=64, rd=64, page=96,
             block=32, longest=2000, ragged=True, short=True, fused=False),
        # two prompts of 16384 tokens; keys, values and queries are slices of one projection
        dict(name="append_prefill", op="append", batch=2, t=16384, h=32, hkv=8, d=128, rd=128,
             page=64, block=16, longest=1, ragged=False, short=False, fused=True),
        # one new token of one sequence, short context: the smallest attention call
        dict(name="attn_single_short", op="attn", batch=1, t=1, h=16, hkv=2, d=128, page=64,
             block=16, longest=509, ragged=False, tree=False, sink=False, short=False),
        # one new token of one sequence, 64 heads in groups of eight, long context
        dict(name="attn_single_long", op="attn", batch=1, t=1, h=64, hkv=8, d=128, page=64,
             block=16, longest=131069, ragged=False, tree=False, sink=False, short=False),
        # a decode batch of ragged sequences with sinks, groups of five
        dict(name="attn_batch_ragged", op="attn", batch=48, t=1, h=40, hkv=8, d=128, page=64,
             block=64, longest=8000, ragged=True, tree=False, sink=True, short=False),
        # trees of 13 drafted tokens, 64 heads in groups of eight
        dict(name="attn_tree_ragged", op="attn", batch=16, t=13, h=64, hkv=8, d=128, page=32,
             block=32, longest=6001, ragged=True, tree=True, sink=True, short=False),
        # the ends of four prompts of different lengths, heads of 256 columns
        dict(name="attn_chunk_ragged", op="attn", batch=4, t=777, h=16, hkv=4, d=256, page=48,
             block=16, longest=4001, ragged=True, tree=False, sink=False, short=True),
        # a chunk of a long prompt: the tensor-bound end
        dict(name="attn_chunk_large", op="attn", batch=1, t=4096, h=64, hkv=8, d=128, page=64,
             block=16, longest=12288, ragged=False, tree=False, sink=False, short=False),
        # one token of eight sequences over the full vocabulary, five alternatives: latency
        dict(name="logprobs_decode", op="logprobs", rows=8, vocab=VOCAB, dtype="bf16", top=5, pad=0),
        # scoring given text, an odd vocabulary cut from a padded one, no alternatives
        dict(name="logprobs_score", op="logprobs", rows=4096, vocab=32003, dtype="fp32", top=0, pad=61),
        # a prompt's log probabilities with twenty alternatives over the full vocabulary
        dict(name="logprobs_prompt", op="logprobs", rows=2048, vocab=VOCAB, dtype="bf16", top=20, pad=0),
    ]


def _spread(rng, lo, hi):
    """A whole number from lo to hi, evenly over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "append", "attn", "attn", "attn", "attn", "logprobs", "logprobs"])
    if op == "logprobs":
        vocab = _spread(rng, 1000, VOCAB)
        return dict(op=op, rows=_spread(rng, 1, min(4096, int(2.6e8) // vocab)), vocab=vocab,
                    dtype=rng.choice(["bf16", "fp32"]), top=rng.choice([0, 1, 5, 20, 32]),
                    pad=rng.choice([0, 0, 1, 61]))
    d = rng.choice([64, 128, 128, 192, 256])
    block = rng.choice([16, 16, 32, 64, 128, 48])
    page = block * rng.choice([1, 2, 3, 4])
    hkv = rng.choice([1, 2, 3, 4, 8])
    h = hkv * rng.choice([1, 2, 4, 5, 7, 8, 16])
    if op == "append":
        batch = _spread(rng, 1, 64)
        return dict(op=op, batch=batch, t=_spread(rng, 1, max(1, 20000 // (batch * (1 + (h + 2 * hkv) // 48)))),
                    h=rng.choice([0, h]), hkv=hkv, d=d, rd=rng.choice([0, 32, 64, d]), page=page, block=block,
                    longest=_spread(rng, 1, 8000), ragged=rng.random() < 0.6, short=rng.random() < 0.4,
                    fused=rng.random() < 0.4)
    batch = _spread(rng, 1, 64)
    t = rng.choice([1, 1, _spread(rng, 2, 64), _spread(rng, 2, max(2, 2048 // batch))])
    # at most a third of the largest listed case's products, and a few GB of scores or cache at most
    most = min(131000, int(1.3e9 / (batch * t * h)), int(1.5e9 / (batch * hkv * d)), int(6.4e11 / (batch * t * h * d)))
    return dict(op=op, batch=batch, t=t, h=h, hkv=hkv, d=d, page=page, block=block,
                longest=_spread(rng, 1, max(2, most)), ragged=rng.random() < 0.6,
                tree=1 < t <= 64 and rng.random() < 0.6, sink=rng.random() < 0.4,
                short=t > 1 and rng.random() < 0.4)


# ------------------------------------------------------------------------------ inputs
def _lengths(case):
    """Cached tokens of each sequence: the case alone sets how many sequences have which."""
    n, batch = case["longest"], case["batch"]
    if not case["ragged"]:
        return [n] * batch
    return [max(0, int(n * (i + 1) / batch) - (i % 3)) for i in range(batch)]


def _counts(case):
    """New tokens of each sequence: all of the call's, or fewer for some."""
    t, batch = case["t"], case["batch"]
    if not case["short"]:
        return [t] * batch
    return [t - (i * t) // batch for i in range(batch)]


def _power(amax):
    """The smallest power of two >= max(amax, 1e-4) / 448."""
    mant, ex = torch.frexp(amax.clamp_min(1e-4) / 448.0)
    return torch.ldexp(torch.ones_like(amax), ex - (mant == 0.5).to(ex.dtype))


def _cache(g, pages, heads, page, block, d):
    """A filled cache: columns of N(0, 1), their sizes spread over the blocks."""
    x8 = torch.empty(pages, heads, page, d, dtype=torch.float8_e4m3fn, device=DEV)
    scale = torch.empty(pages, heads, page // block, device=DEV)
    step = max(1, (1 << 26) // (heads * page * d))
    for at in range(0, pages, step):
        n = min(step, pages - at)
        x = torch.randn(n, heads, page // block, block, d, device=DEV, generator=g)
        x *= torch.exp2(torch.randint(-1, 2, (n, heads, page // block, 1, 1), device=DEV, generator=g).float())
        s = _power(x.abs().amax((-1, -2)))
        x8[at:at + n].view(torch.uint8).copy_(
            (x / s[..., None, None]).to(torch.float8_e4m3fn).view(torch.uint8).view(n, heads, page, d))
        scale[at:at + n] = s
    return x8, scale


def _table(g, batch, each, spare=3):
    """Pages of every sequence, in no order, out of a pool with some pages to spare."""
    pool = batch * each + spare
    perm = torch.randperm(pool, device=DEV, generator=g)[: batch * each]
    return perm.view(batch, each).int().contiguous(), pool


def _tree(g, batch, t):
    """The ancestor mask of trees of t drafted tokens; half of the nodes follow their predecessor."""
    at = torch.arange(t, device=DEV)
    parents = torch.floor(torch.rand(batch, t, device=DEV, generator=g) * (at + 1)).long() - 1
    parents = torch.where(torch.rand(batch, t, device=DEV, generator=g) < 0.5, at - 1, parents)
    mask = torch.eye(t, dtype=torch.bool, device=DEV).repeat(batch, 1, 1)
    for i in range(1, t):
        p = parents[:, i].clamp_min(0)
        mask[:, i] |= mask[torch.arange(batch, device=DEV), p] & (parents[:, i] >= 0)[:, None]
    return mask


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    op = case["op"]
    if op == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        dtype = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
        wide = torch.empty(rows, vocab + case["pad"], dtype=dtype, device=DEV)
        step = max(1, (1 << 26) // vocab)
        for at in range(0, rows, step):
            n = min(step, rows - at)
            wide[at:at + n] = 2.5 * torch.randn(n, wide.shape[1], device=DEV, generator=g)
        logits = wide[:, :vocab]
        # half of the given tokens are likely ones
        best = torch.cat([logits[at:at + step].float().argmax(1) for at in range(0, rows, step)])
        some = torch.randint(0, vocab, (rows,), device=DEV, generator=g)
        tokens = torch.where(torch.rand(rows, device=DEV, generator=g) < 0.5, best, some)
        return dict(op=op, logits=logits, tokens=tokens, top=case["top"])
    b, t, h, hkv, d, page, block = (case[k] for k in ("batch", "t", "h", "hkv", "d", "page", "block"))
    order = torch.randperm(b, device=DEV, generator=g)
    lens = torch.tensor(_lengths(case), dtype=torch.int32, device=DEV)[order].contiguous()
    n_new = torch.tensor(_counts(case), dtype=torch.int32, device=DEV).contiguous() if case["short"] else None
    table, pool = _table(g, b, -(-(case["longest"] + t) // page))
    k8, k_scale = _cache(g, pool, hkv, page, block, d)
    v8, v_scale = _cache(g, pool, hkv, page, block, d)
    state = dict(op=op, k8=k8, k_scale=k_scale, v8=v8, v_scale=v_scale, table=table, lens=lens, n_new=n_new)
    if op == "append":
        # sizes spread over the tokens, so that some blocks' scales grow
        parts = [(x, torch.randn(b, t, x, d, device=DEV, generator=g)) for x in (hkv, hkv, h) if x]
        grow = torch.exp2(torch.randint(-2, 3, (b, t, 1, 1), device=DEV, generator=g).float())
        parts = [(x, (y * grow).bfloat16()) for x, y in parts]
        if case["fused"]:  # one projection's output, cut up
            wide = torch.cat([y.flatten(2) for _, y in parts], -1)
            cut = wide.split([x * d for x, _ in parts], -1)
            parts = [(x, y.unflatten(-1, (x, d))) for (x, _), y in zip(parts, cut)]
        state.update(k=parts[0][1], v=parts[1][1], q=parts[2][1] if h else None, freqs=None)
        if case["rd"]:
            pos = torch.arange(case["longest"] + t, device=DEV, dtype=torch.float64)
            ang = torch.outer(pos, 10000.0 ** (-torch.arange(0, case["rd"], 2, device=DEV, dtype=torch.float64) / case["rd"]))
            state["freqs"] = torch.stack([ang.cos(), ang.sin()], -1).float().contiguous()
        return state
    state["q"] = torch.randn(b, t, h, d, device=DEV, generator=g).bfloat16()
    state["mask"] = _tree(g, b, t) if case["tree"] else None
    state["sink"] = torch.randn(h, device=DEV, generator=g) if case["sink"] else None
    state["softmax_scale"] = d ** -0.5
    return state


# ------------------------------------------------------------------------------ one pass
def run(s):
    if own:
        from kernelswift_b200 import ops

        if s["op"] == "append":
            q = ops.kv_append(s["k"], s["v"], s["k8"], s["k_scale"], s["v8"], s["v_scale"], s["table"],
                              s["lens"], freqs=s["freqs"], n_new=s["n_new"], q=s["q"])
            return [x for x in (s["k8"], s["k_scale"], s["v8"], s["v_scale"], q) if x is not None]
        if s["op"] == "attn":
            return ops.kv_attn(s["q"], s["k8"], s["k_scale"], s["v8"], s["v_scale"], s["table"], s["lens"],
                               s["softmax_scale"], mask=s["mask"], attn_sink=s["sink"], n_new=s["n_new"])
        return [x for x in ops.token_logprobs(s["logits"], s["tokens"], top=s["top"]) if x is not None]
    return {"append": _plain_append, "attn": _plain_attn, "logprobs": _plain_logprobs}[s["op"]](s)


def _live(s, t):
    """[batch, t]: which of the call's tokens are there."""
    at = torch.arange(t, device=DEV)[None].expand(len(s["lens"]), t)
    return at >= 0 if s["n_new"] is None else at < s["n_new"][:, None]


def _rotate(x, freqs, pos):
    """The last columns of x [b, t, heads, d] in 32 bits, as pairs rotated by freqs[pos]."""
    x = x.float()
    if freqs is None:
        return x
    rd = 2 * freqs.shape[1]
    c, sn = freqs[pos.clamp_max(freqs.shape[0] - 1)][:, :, None].unbind(-1)
    a, b = x[..., x.shape[-1] - rd:].unflatten(-1, (rd // 2, 2)).unbind(-1)
    y = torch.stack([a * c - b * sn, a * sn + b * c], -1).flatten(-2)
    return torch.cat([x[..., : x.shape[-1] - rd], y], -1)


def _plain_append(s):
    b, t = s["k"].shape[:2]
    page, per = s["k8"].shape[2], s["k_scale"].shape[2]
    block = page // per
    lens = s["lens"].long()
    pos = lens[:, None] + torch.arange(t, device=DEV)
    live = _live(s, t)
    pages = s["table"].long().gather(1, (pos // page).clamp_max(s["table"].shape[1] - 1))
    place, row = pages[live], (pos % page)[live]
    # the block that a sequence's tokens so far end in
    there = (lens % block > 0) & live[:, 0]
    end = s["table"].long().gather(1, (lens // page).clamp_max(s["table"].shape[1] - 1)[:, None])[:, 0]
    end, first = end[there], (lens % page // block)[there]
    filled = (lens % block)[there]
    old_rows = first[:, None] * block + torch.arange(block, device=DEV)
    for x, x8, scale in ((_rotate(s["k"], s["freqs"], pos), s["k8"], s["k_scale"]),
                         (s["v"].float(), s["v8"], s["v_scale"])):
        heads, d = x.shape[2:]
        x = x[live]
        amax = torch.zeros(scale.shape[0], per, heads, device=DEV).view(-1, heads)
        amax.scatter_reduce_(0, (place * per + row // block)[:, None].expand(-1, heads), x.abs().amax(-1), "amax")
        new = _power(amax).view(-1, per, heads).transpose(1, 2)
        before = scale[end, :, first]
        after = torch.maximum(new[end, :, first], before)
        codes = x8.view(torch.uint8)
        old = codes[end[:, None], :, old_rows].view(torch.float8_e4m3fn).float()
        old = (old * (before / after)[:, None, :, None]).to(torch.float8_e4m3fn).view(torch.uint8)
        keep = torch.arange(block, device=DEV)[None] < filled[:, None]
        codes[end[:, None].expand_as(keep)[keep], :, old_rows[keep]] = old[keep]
        scale[place, :, row // block] = new[place, :, row // block]
        scale[end, :, first] = after
        x = (x / scale[place, :, row // block][..., None]).to(torch.float8_e4m3fn)
        codes[place, :, row] = x.view(torch.uint8)
    out = [s["k8"], s["k_scale"], s["v8"], s["v_scale"]]
    if s["q"] is not None:
        out.append(_rotate(s["q"], s["freqs"], pos).bfloat16())
    return out


def _values(x8, scale, table):
    """The pages of every sequence as fp32 [batch, heads, pages x page, d]."""
    at = table.long()
    x = x8.view(torch.uint8)[at].view(torch.float8_e4m3fn).float()  # [b, pages, heads, page, d]
    x = x.unflatten(3, (scale.shape[2], -1)) * scale[at][..., None, None]
    return x.flatten(3, 4).transpose(1, 2).flatten(2, 3)


def _allowed(s, t, n):
    """[batch, t, n]: what each new token may attend to; without a mask, a chain."""
    j = torch.arange(n, device=DEV)[None] - s["lens"][:, None].long()
    mask = s["mask"]
    if mask is None:
        mask = torch.ones(t, t, dtype=torch.bool, device=DEV).tril()[None].expand(len(j), t, t)
    drafted = mask.gather(2, j.clamp(0, t - 1)[:, None, :].expand(-1, t, -1))
    ok = (j < 0)[:, None] | (drafted & ((j >= 0) & (j < t))[:, None])
    return ok & _live(s, t)[..., None]


def _plain_attn(s):
    b, t, h, d = s["q"].shape
    k, v = _values(s["k8"], s["k_scale"], s["table"]), _values(s["v8"], s["v_scale"], s["table"])
    heads, n = k.shape[1:3]
    ok = _allowed(s, t, n)
    q = s["q"].float().view(b, t, heads, h // heads, d).permute(0, 2, 1, 3, 4)
    out = torch.empty(b, heads, t, h // heads, d, device=DEV)
    for g in range(heads):  # one head's scores at a time
        x = torch.matmul(q[:, g].flatten(1, 2), k[:, g].transpose(1, 2)).mul_(s["softmax_scale"])
        x = x.view(b, t, -1, n).masked_fill_(~ok[:, :, None], -math.inf)
        top = x.amax(-1, keepdim=True)
        if s["sink"] is not None:
            sink = s["sink"].view(heads, -1)[g][:, None]
            top = torch.maximum(top, sink)
        top = torch.where(top == -math.inf, 0.0, top)
        e = x.sub_(top).exp_()
        den = e.sum(-1, keepdim=True)
        if s["sink"] is not None:
            den = den + torch.exp(sink - top)
        o = torch.matmul(e.view(b, -1, n), v[:, g]).view(b, t, -1, d)
        out[:, g] = torch.where(den > 0, o / den, 0.0)
    out = out.permute(0, 2, 1, 3, 4).reshape(b, t, h, d)
    return torch.where(_live(s, t)[..., None, None], out, 0.0).bfloat16()


def _plain_logprobs(s):
    x = s["logits"].float()
    m = x.amax(1, keepdim=True)
    e = torch.exp(x - m)
    total = e.sum(1)
    lse = m[:, 0] + torch.log(total)
    logp = x.gather(1, s["tokens"][:, None])[:, 0] - lse
    entropy = torch.log(total) + (e * (m - x)).sum(1) / total
    if not s["top"]:
        return [logp, entropy]
    # the largest values, the lowest index first among equal ones: one whole number for both
    bits = (x + 0.0).view(torch.int32)
    bits = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
    at = torch.arange(x.shape[1], device=DEV)
    best = torch.topk(bits * (1 << 32) + (0xFFFFFFFF - at), s["top"], 1).values
    ids = 0xFFFFFFFF - (best & 0xFFFFFFFF)
    return [logp, entropy, x.gather(1, ids) - lse[:, None], ids]


# ------------------------------------------------------------------------------ floors and truth
def work(case):
    op = case["op"]
    if op == "logprobs":
        n = float(case["rows"] * case["vocab"])
        return dict(bytes=n * (2 if case["dtype"] == "bf16" else 4) + case["rows"] * (16.0 + 12 * case["top"]),
                    flops=5.0 * n)
    b, h, hkv, d = case["batch"], case["h"], case["hkv"], case["d"]
    lens, new = _lengths(case), _counts(case)
    if op == "append":
        # rows read in 16 bits, written in 8 (queries: 16), their blocks' scales
        rows = float(sum(new))
        return dict(bytes=rows * d * (hkv * 6 + h * 4) + rows * hkv * 8 / case["block"] + rows * case["rd"] * 4,
                    flops=rows * d * (hkv * 6 + h * 3))
    seen = sum(n + k for n, k in zip(lens, new))
    pairs = sum(n * k + k * (k + 1) / 2 for n, k in zip(lens, new))
    return dict(bytes=seen * hkv * (2.0 * d + 8 / case["block"]) + sum(new) * h * d * 2.0 + b * case["t"] * h * d * 2.0,
                flops=4.0 * h * d * pairs)


def exact(case, seed):
    s = prepare(case, seed)
    op = s["op"]
    if op == "logprobs":
        parts = []
        step = max(1, (1 << 26) // case["vocab"])
        for at in range(0, case["rows"], step):
            x = s["logits"][at:at + step].double()
            lse = torch.logsumexp(x, 1)
            lp = x - lse[:, None]
            out = [lp.gather(1, s["tokens"][at:at + step, None])[:, 0], -(lp.exp() * lp).sum(1)]
            if s["top"]:
                out.append(lp.sort(1, descending=True).values[:, : s["top"]])
            parts.append(out)
        outs = [torch.cat(x) for x in zip(*parts)]
        return outs + [None] if s["top"] else outs
    code = torch.arange(256, device=DEV)
    ex, man = (code >> 3) & 15, (code & 7).double()
    value = torch.where(ex == 0, man / 8 * 2.0 ** -6, (1 + man / 8) * torch.exp2((ex - 7).double()))
    value = torch.where(code >= 128, -value, value)
    page, per = s["k8"].shape[2], s["k_scale"].shape[2]
    block = page // per
    lens, table = s["lens"].tolist(), s["table"].tolist()
    new = s["n_new"].tolist() if s["n_new"] is not None else [case["t"]] * len(lens)
    if op == "append":
        def turned(x):  # complex products
            x = x.double()
            if s["freqs"] is None:
                return x
            rd, t = 2 * s["freqs"].shape[1], x.shape[1]
            z = torch.view_as_complex(x[..., x.shape[-1] - rd:].reshape(*x.shape[:3], rd // 2, 2).contiguous())
            f = torch.view_as_complex(s["freqs"].double())
            z = torch.stack([z[i] * f[n: n + t, None] for i, n in enumerate(lens)])
            return torch.cat([x[..., : x.shape[-1] - rd], torch.view_as_real(z).flatten(-2)], -1)

        if sum(-(-(n + k) // block) - n // block for n, k in zip(lens, new)) > 8000:
            return None  # block by block: too long
        outs = []
        for x, x8, scale in ((turned(s["k"]), s["k8"], s["k_scale"]), (s["v"].double(), s["v8"], s["v_scale"])):
            held, scale = value[x8.view(torch.uint8).long()], scale.double()
            for i, (n, k) in enumerate(zip(lens, new)):
                at = n
                while at < n + k:
                    stop = min(n + k, (at // block + 1) * block)
                    p, first = table[i][at // page], at % page // block
                    rows = x[i, at - n: stop - n].transpose(0, 1)  # [heads, tokens, d]
                    mant, e = torch.frexp(rows.abs().amax((1, 2)).clamp_min(1e-4) / 448)
                    sc = torch.ldexp(torch.ones_like(mant), torch.where(mant > 0.5, e, e - 1))
                    if at % block:
                        sc = torch.maximum(sc, scale[p, :, first])
                        held[p, :, first * block: at % page] *= (scale[p, :, first] / sc)[:, None, None]
                    held[p, :, at % page: at % page + stop - at] = rows / sc[:, None, None]
                    scale[p, :, first] = sc
                    at = stop
            outs += [held, scale]
        return outs + ([turned(s["q"])] if s["q"] is not None else [])
    b, t, h, d = s["q"].shape
    heads = s["k8"].shape[1]
    out = torch.zeros(b, t, h, d, dtype=torch.float64, device=DEV)
    for i in range(b):
        n = lens[i] + new[i]
        pg = torch.tensor(table[i][: -(-n // page)], device=DEV)
        tree = s["mask"][i] if s["mask"] is not None else torch.ones(t, t, device=DEV).tril().bool()
        for g in range(heads):
            k, v = (value[x8.view(torch.uint8)[pg, g].long()].view(len(pg), per, block, d)
                    * sc[pg, g].double()[..., None, None] for x8, sc in ((s["k8"], s["k_scale"]), (s["v8"], s["v_scale"])))
            k, v = k.reshape(-1, d)[:n], v.reshape(-1, d)[:n]
            hs = slice(g * (h // heads), (g + 1) * (h // heads))
            step = max(1, int(2.5e8) // (n * (h // heads)))
            for t0 in range(0, new[i], step):
                t1 = min(t0 + step, new[i])
                x = torch.einsum("thd,nd->thn", s["q"][i, t0:t1, hs].double(), k) * s["softmax_scale"]
                x[..., lens[i]:].masked_fill_(~tree[t0:t1, None, : new[i]], -math.inf)
                if s["sink"] is not None:
                    x = torch.cat([x, s["sink"][hs].double()[None, :, None].expand(t1 - t0, -1, 1)], -1)
                out[i, t0:t1, hs] = torch.softmax(x, -1)[..., :n] @ v
    return out
