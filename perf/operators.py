"""The serving operators over a quantised latent cache, as cases that can be timed and compared.

Four operators make one speculative decoding step of a sparse-attention model that keeps its
latent key-values in 8 bits:

* ``cache_write``  quantises new latent rows as they enter a paged cache;
* ``cache_read``   reads a stretch of every sequence back as bf16 rows (what ``sparse_attn`` takes);
* ``tree_attn``    attends from a tree (or chain) of drafted tokens over the cache;
* ``verify_draft`` accepts or rejects the drafted tokens with given random numbers.

A cached row is D = dq + dr wide: dq columns in e4m3 with one power-of-two scale per row, dr
columns (the rotary part) in bf16.  With ``own`` false, ``run`` computes each operator from
elementary torch operations in 32 bits; with ``own`` true it calls ``kernelswift_b200.ops``.
"""
import math

import torch

own = False

DEV = "cuda"
VOCAB = 129280  # ModelArgs.vocab_size of the indexer module


# ------------------------------------------------------------------------------ cases
def listed():
    return [
        # one decode step of eight sequences appends eight latent rows: launch latency
        dict(name="write_decode", op="write", rows=8, dq=512, dr=64, page=64, stride=576),
        # a prefill of two sequences of 32768 tokens fills the cache; the rows are a slice of a
        # wider projection output
        dict(name="write_prefill", op="write", rows=65536, dq=512, dr=64, page=64, stride=640),
        # an odd-sized stretch of FP8 index keys (128 columns, no rotary part) of three sequences
        dict(name="read_index_keys", op="read", batch=3, n=333, dq=128, dr=0, page=16),
        # chunked prefill: the cached prefix of four sequences as bf16 rows for the sparse attention
        dict(name="read_prefix", op="read", batch=4, n=16379, dq=512, dr=64, page=64),
        # one new token of one sequence, few heads, short context: the smallest attention call
        dict(name="attn_single_short", op="attn", batch=1, t=1, h=16, dq=128, dr=0, dv=128,
             longest=509, ragged=False, page=64, tree=False, sink=False),
        # one new token of one sequence with 128 heads over a long context: work split over the keys
        dict(name="attn_single_long", op="attn", batch=1, t=1, h=128, dq=512, dr=64, dv=512,
             longest=131069, ragged=False, page=64, tree=False, sink=False),
        # a decode batch of ragged sequences with 16 heads (one rank's share of the heads)
        dict(name="attn_batch_ragged", op="attn", batch=48, t=1, h=16, dq=512, dr=64, dv=512,
             longest=8000, ragged=True, page=64, tree=False, sink=True),
        # trees of 13 drafted tokens, 64 heads of 512 columns whose last 64 are rotary, sinks
        dict(name="attn_tree_ragged", op="attn", batch=16, t=13, h=64, dq=448, dr=64, dv=512,
             longest=6001, ragged=True, page=32, tree=True, sink=True),
        # large trees over long contexts: the tensor-bound end
        dict(name="attn_tree_large", op="attn", batch=8, t=32, h=128, dq=512, dr=64, dv=512,
             longest=8192, ragged=False, page=64, tree=True, sink=False),
        # one sequence, three drafted tokens, a small vocabulary: latency
        dict(name="verify_chain_small", op="verify", batch=1, t=3, vocab=32003, tree=False),
        # a batch of sampled chains of seven tokens over the full vocabulary
        dict(name="verify_chain", op="verify", batch=64, t=7, vocab=VOCAB, tree=False),
        # trees of 40 fixed candidates
        dict(name="verify_tree", op="verify", batch=16, t=40, vocab=VOCAB, tree=True),
    ]


def _spread(rng, lo, hi):
    """A whole number from lo to hi, evenly over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["write", "read", "attn", "attn", "attn", "verify", "verify"])
    dq, dr, dv = rng.choice([(512, 64, 512), (448, 64, 512), (512, 64, 512), (128, 0, 128),
                             (256, 64, 256), (192, 64, 192), (64, 64, 64)])
    page = rng.choice([1, 16, 32, 48, 64, 100, 256])
    if op == "write":
        return dict(op=op, rows=_spread(rng, 1, 60000), dq=dq, dr=dr, page=page,
                    stride=dq + dr + rng.choice([0, 0, 8, 64]))
    if op == "read":
        batch = _spread(rng, 1, 64)
        return dict(op=op, batch=batch, n=_spread(rng, 1, 60000 // batch), dq=dq, dr=dr, page=page)
    if op == "attn":
        h = rng.choice([1, 5, 16, 20, 32, 64, 128])
        t = rng.choice([1, 1, _spread(rng, 2, 64)])
        batch = _spread(rng, 1, 64)
        # at most half of the largest listed case's products, and a few GB of scores at most
        most = min(131000, 200000 // batch, int(1.3e8 / (batch * t * h)))
        return dict(op=op, batch=batch, t=t, h=h, dq=dq, dr=dr, dv=dv,
                    longest=_spread(rng, 1, max(2, most)), ragged=rng.random() < 0.6, page=page,
                    tree=t > 1 and rng.random() < 0.7, sink=rng.random() < 0.5)
    tree = rng.random() < 0.5
    t = rng.randint(1, 48) if tree else rng.randint(1, 12)
    vocab = _spread(rng, 1000, VOCAB)
    return dict(op=op, batch=_spread(rng, 1, max(1, min(64, 600 // t))), t=t, vocab=vocab, tree=tree)


# ------------------------------------------------------------------------------ inputs
def _lengths(case):
    """Cached tokens of each sequence: the case alone sets how many sequences have which."""
    n, batch = case["longest"], case["batch"]
    if not case["ragged"]:
        return [n] * batch
    return [max(0, int(n * (i + 1) / batch)) for i in range(batch)]


def _quantise(x):
    """Rows in e4m3 with one power-of-two scale per row, as the cache holds them."""
    amax = x.abs().amax(-1).clamp_min(1e-4)
    mant, ex = torch.frexp(amax / 448.0)
    scale = torch.ldexp(torch.ones_like(amax), ex - (mant == 0.5).to(ex.dtype))
    return (x / scale[..., None]).to(torch.float8_e4m3fn), scale


def _cache(g, pages, page, dq, dr):
    """A filled cache: latent rows of N(0, 1) columns, their sizes spread over rows."""
    rows = pages * page
    kv8 = torch.empty(pages, page, dq, dtype=torch.float8_e4m3fn, device=DEV)
    scale = torch.empty(pages, page, device=DEV)
    flat8, flats = kv8.view(rows, dq), scale.view(rows)
    step = 1 << 17
    for at in range(0, rows, step):
        n = min(step, rows - at)
        x = torch.randn(n, dq, device=DEV, generator=g)
        x *= torch.exp2(torch.randint(-1, 2, (n, 1), device=DEV, generator=g).float())
        q, s = _quantise(x.bfloat16().float())
        flat8.view(torch.uint8)[at:at + n] = q.view(torch.uint8)
        flats[at:at + n] = s
    tail = torch.randn(pages, page, dr, device=DEV, generator=g).bfloat16() if dr else None
    return kv8, scale, tail


def _table(g, batch, each, spare=3):
    """Pages of every sequence, in no order, out of a pool with some pages to spare."""
    pool = batch * each + spare
    perm = torch.randperm(pool, device=DEV, generator=g)[: batch * each]
    return perm.view(batch, each).int().contiguous(), pool


def _tree(g, batch, t):
    """Parents of each drafted token (-1: the last accepted one) and the ancestor mask."""
    r = torch.rand(batch, t, device=DEV, generator=g)
    at = torch.arange(t, device=DEV)
    parents = torch.floor(r * (at + 1)).long() - 1
    # deeper trees than uniform parents give: half of the nodes follow their predecessor
    deep = torch.rand(batch, t, device=DEV, generator=g) < 0.5
    parents = torch.where(deep, at - 1, parents)
    mask = torch.eye(t, dtype=torch.bool, device=DEV).repeat(batch, 1, 1)
    for i in range(1, t):
        p = parents[:, i].clamp_min(0)
        up = mask[torch.arange(batch, device=DEV), p]
        mask[:, i] |= up & (parents[:, i] >= 0)[:, None]
    return parents.int().contiguous(), mask


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    op = case["op"]
    if op == "write":
        rows, dq, dr, page = case["rows"], case["dq"], case["dr"], case["page"]
        pages = -(-rows // page) + 2
        wide = torch.randn(rows, case["stride"], device=DEV, generator=g)
        wide *= torch.exp2(torch.randint(-2, 3, (rows, 1), device=DEV, generator=g).float())
        kv = wide.bfloat16()[:, : dq + dr]
        kv8, scale, tail = _cache(g, pages, page, dq, dr)
        slots = torch.randperm(pages * page, device=DEV, generator=g)[:rows].contiguous()
        return dict(op=op, kv=kv, slots=slots, kv8=kv8, scale=scale, tail=tail)
    if op == "read":
        batch, n, page = case["batch"], case["n"], case["page"]
        table, pool = _table(g, batch, -(-n // page))
        kv8, scale, tail = _cache(g, pool, page, case["dq"], case["dr"])
        # the last sequence ends inside the stretch
        lens = torch.full((batch,), n, dtype=torch.int32, device=DEV)
        lens[-1] = n - n // 7
        return dict(op=op, kv8=kv8, scale=scale, tail=tail, table=table, lens=lens, n=n)
    if op == "attn":
        b, t, h, dq, dr, page = (case[k] for k in ("batch", "t", "h", "dq", "dr", "page"))
        lens = _lengths(case)
        order = torch.randperm(b, device=DEV, generator=g)
        lens = torch.tensor(lens, dtype=torch.int32, device=DEV)[order].contiguous()
        table, pool = _table(g, b, -(-(case["longest"] + t) // page))
        kv8, scale, tail = _cache(g, pool, page, dq, dr)
        q = torch.randn(b, t, h, dq + dr, device=DEV, generator=g).bfloat16()
        mask = _tree(g, b, t)[1] if case["tree"] else None
        sink = torch.randn(h, device=DEV, generator=g) if case["sink"] else None
        return dict(op=op, q=q, kv8=kv8, scale=scale, tail=tail, table=table, lens=lens, mask=mask,
                    sink=sink, softmax_scale=(dq + dr) ** -0.5, dv=case["dv"])
    b, t, vocab = case["batch"], case["t"], case["vocab"]
    logits = 3.0 * torch.randn(b, t + 1, vocab, device=DEV, generator=g)
    p = torch.softmax(logits, -1)
    u = torch.rand(b, t + 1, device=DEV, generator=g)
    noise = torch.empty(b, vocab, device=DEV).exponential_(generator=g).clamp_min_(1e-10)
    state = dict(op=op, p=p, u=u, noise=noise, q=None, parents=None, mask=None)
    if case["tree"]:
        # candidates: the likeliest tokens after each node, one per child
        parents, mask = _tree(g, b, t)
        rank = ((parents[:, :, None] == parents[:, None, :]).tril(-1)).sum(-1)
        top = p.topk(min(t, vocab), -1).indices
        rows = torch.arange(b, device=DEV)[:, None]
        state["tokens"] = top[rows, parents.long() + 1, rank.clamp_max(vocab - 1)].contiguous()
        state["parents"], state["mask"] = parents, mask
    else:
        # a draft whose distribution is near the target's, its tokens sampled from it
        q = torch.softmax(logits[:, :t] + 0.5 * torch.randn(b, t, vocab, device=DEV, generator=g), -1)
        e = torch.empty(b, t, vocab, device=DEV).exponential_(generator=g).clamp_min_(1e-10)
        state["tokens"], state["q"] = (q / e).argmax(-1), q
    return state


# ------------------------------------------------------------------------------ one pass
def run(s):
    if own:
        from kernelswift_b200 import ops

        if s["op"] == "write":
            ops.cache_write(s["kv"], s["slots"], s["kv8"], s["scale"], s["tail"])
            return [x for x in (s["kv8"], s["scale"], s["tail"]) if x is not None]
        if s["op"] == "read":
            return ops.cache_read(s["kv8"], s["scale"], s["tail"], s["table"], s["lens"], s["n"])
        if s["op"] == "attn":
            return ops.tree_attn(s["q"], s["kv8"], s["scale"], s["tail"], s["table"], s["lens"],
                                 s["softmax_scale"], dv=s["dv"], mask=s["mask"],
                                 attn_sink=s["sink"])
        return ops.verify_draft(s["p"], s["tokens"], s["u"], s["noise"], q=s["q"],
                                parents=s["parents"])
    return {"write": _plain_write, "read": _plain_read, "attn": _plain_attn,
            "verify": _plain_verify}[s["op"]](s)


def _plain_write(s):
    kv8, scale, tail = s["kv8"], s["scale"], s["tail"]
    dq = kv8.shape[-1]
    x8, sc = _quantise(s["kv"][:, :dq].float())
    kv8.view(torch.uint8).view(-1, dq)[s["slots"]] = x8.view(torch.uint8)
    scale.view(-1)[s["slots"]] = sc
    if tail is not None:
        tail.view(-1, tail.shape[-1])[s["slots"]] = s["kv"][:, dq:]
    return [x for x in (kv8, scale, tail) if x is not None]


def _rows32(s):
    """The pages of every sequence as fp32 rows [batch, pages x page, D]."""
    at = s["table"].long()
    x = s["kv8"].view(torch.uint8)[at].view(torch.float8_e4m3fn).float() * s["scale"][at][..., None]
    if s["tail"] is not None:
        x = torch.cat([x, s["tail"][at].float()], -1)
    return x.flatten(1, 2)


def _plain_read(s):
    x = _rows32(s)[:, : s["n"]]
    inside = torch.arange(s["n"], device=DEV)[None] < s["lens"][:, None]
    return torch.where(inside[..., None], x, 0.0).bfloat16()


def _allowed(lens, t, n, mask):
    """[batch, t, n]: what each drafted token may attend to; without a mask, a chain."""
    pos = torch.arange(n, device=DEV)
    j = pos[None] - lens[:, None].long()
    if mask is None:
        mask = torch.ones(t, t, dtype=torch.bool, device=DEV).tril()[None].expand(len(lens), t, t)
    drafted = mask.gather(2, j.clamp(0, t - 1)[:, None, :].expand(-1, t, -1))
    return (j < 0)[:, None] | (drafted & ((j >= 0) & (j < t))[:, None])


def _plain_attn(s):
    q = s["q"].float()
    b, t, h, d = q.shape
    k = _rows32(s)
    ok = _allowed(s["lens"], t, k.shape[1], s["mask"])
    x = torch.matmul(q.view(b, t * h, d), k.transpose(1, 2)).view(b, t, h, -1) * s["softmax_scale"]
    x = torch.where(ok[:, :, None], x, -math.inf)
    top = x.amax(-1, keepdim=True)
    if s["sink"] is not None:
        top = torch.maximum(top, s["sink"][:, None])
    top = torch.where(top == -math.inf, 0.0, top)
    e = torch.exp(x - top)
    den = e.sum(-1, keepdim=True)
    if s["sink"] is not None:
        den = den + torch.exp(s["sink"][:, None] - top)
    o = torch.matmul(e.view(b, t * h, -1), k[..., : s["dv"]]).view(b, t, h, -1)
    return torch.where(den > 0, o / den, 0.0).bfloat16()


def _plain_verify(s):
    p, tokens, u, noise, q = s["p"], s["tokens"], s["u"], s["noise"], s["q"]
    b, t = tokens.shape
    at, rows = torch.arange(t, device=DEV), torch.arange(b, device=DEV)
    if q is not None:  # sampled chain: token i stands with probability min(1, p / q)
        px = p[:, :t].gather(2, tokens[..., None])[..., 0]
        qx = q.gather(2, tokens[..., None])[..., 0]
        ok = (u[:, :t] * qx < px).long().cumprod(1).bool()
        n = ok.sum(1)
        last = p[rows, n]
        left = torch.where((n < t)[:, None], (last - q[rows, n.clamp_max(t - 1)]).clamp_min(0.0), last)
    else:  # fixed candidates: u of the parent's row falls into the stretch of one child, or of none
        row = s["parents"].long() + 1
        px = p[rows[:, None], row, tokens].double()
        older = (row[:, :, None] == row[:, None, :]).tril(-1)
        px = torch.where((older & (tokens[:, :, None] == tokens[:, None, :])).any(-1), 0.0, px)
        lo = torch.where(older, px[:, None, :], 0.0).sum(-1)
        ux = u[rows[:, None], row].double()
        ok = (((lo <= ux) & (ux < lo + px))[:, None, :] | ~s["mask"]).all(-1)
        n = ok.sum(1)
        end = torch.where(ok, at + 1, 0).amax(1)
        last = p[rows, end]
        gone = torch.where(row == end[:, None], tokens, p.shape[2])
        keep = torch.ones(b, p.shape[2] + 1, device=DEV).scatter_(1, gone, 0.0)[:, :-1]
        left = last * keep
    left = torch.where((left > 0).any(1, keepdim=True), left, last)
    new = (left / noise).argmax(1)
    path = torch.where(ok, at, t).sort(1).values
    seen = torch.cat([tokens, new[:, None]], 1).gather(1, torch.cat([path, path[:, :1] * 0 + t], 1))
    place = torch.arange(t + 1, device=DEV)[None]
    out = torch.where(place < n[:, None], seen, torch.where(place == n[:, None], new[:, None], -1))
    return out, n.int(), torch.where(path < t, path, -1).int()


# ------------------------------------------------------------------------------ floors and truth
def work(case):
    op = case["op"]
    if op == "verify":
        # the row where the draft ends: target, noise, and for sampled chains the draft's row
        row = 4.0 * case["vocab"] * case["batch"]
        return dict(bytes=row * (2 if case["tree"] else 3) + 40.0 * case["batch"] * case["t"],
                    flops=3.0 * case["vocab"] * case["batch"])
    dq, dr = case["dq"], case["dr"]
    held = dq + 2 * dr + 4
    if op == "write":
        return dict(bytes=case["rows"] * (2.0 * (dq + dr) + 8 + held), flops=3.0 * case["rows"] * dq)
    if op == "read":
        n = case["n"] * case["batch"]
        there = n - case["n"] // 7
        return dict(bytes=there * float(held) + 2.0 * n * (dq + dr), flops=1.0 * there * dq)
    b, t, h, d, dv = case["batch"], case["t"], case["h"], dq + dr, case["dv"]
    keys = float(sum(_lengths(case)))
    return dict(bytes=(keys + b * t) * held + 2.0 * b * t * h * (d + dv),
                flops=2.0 * h * (d + dv) * (t * keys + b * t * (t + 1) / 2))


def exact(case, seed):
    s = prepare(case, seed)
    op = s["op"]
    if op == "verify":
        return None
    code = torch.arange(256, device=DEV)
    ex, man = (code >> 3) & 15, (code & 7).double()
    value = torch.where(ex == 0, man / 8 * 2.0 ** -6, (1 + man / 8) * torch.exp2((ex - 7).double()))
    value = torch.where(code >= 128, -value, value)
    if op == "write":
        dq = s["kv8"].shape[-1]
        x = s["kv"].double()
        amax = x[:, :dq].abs().amax(-1).clamp_min(1e-4)
        mant, ex = torch.frexp(amax / 448)
        sc = torch.ldexp(torch.ones_like(amax), torch.where(mant > 0.5, ex, ex - 1))
        held = value[s["kv8"].view(torch.uint8).long()]
        held.view(-1, dq)[s["slots"]] = x[:, :dq] / sc[:, None]
        scale = s["scale"].double()
        scale.view(-1)[s["slots"]] = sc
        if s["tail"] is None:
            return [held, scale]
        tail = s["tail"].double()
        tail.view(-1, tail.shape[-1])[s["slots"]] = x[:, dq:]
        return [held, scale, tail]
    lens, table = s["lens"].tolist(), s["table"].long()
    outs = []
    for b in range(len(lens)):
        k = value[s["kv8"].view(torch.uint8)[table[b]].long()] * s["scale"][table[b]].double()[..., None]
        if s["tail"] is not None:
            k = torch.cat([k, s["tail"][table[b]].double()], -1)
        k = k.flatten(0, 1)
        if op == "read":
            k = k[: s["n"]].clone()
            k[lens[b]:] = 0
            outs.append(k)
            continue
        q = s["q"][b].double()
        t, h, d = q.shape
        tree = s["mask"][b] if s["mask"] is not None else torch.ones(t, t, device=DEV).tril().bool()
        n = lens[b] + t
        rows = []
        step = max(1, int(2.5e8) // (h * n))
        for t0 in range(0, t, step):
            qt = q[t0:t0 + step]
            x = (qt.flatten(0, 1) @ k[:n].T).view(len(qt), h, n) * s["softmax_scale"]
            x[:, :, lens[b]:].masked_fill_(~tree[t0:t0 + step, None, :], -math.inf)
            if s["sink"] is not None:
                x = torch.cat([x, s["sink"].double()[None, :, None].expand(len(qt), h, 1)], -1)
            w = torch.softmax(x, -1)[..., :n]
            rows.append((w.reshape(-1, n) @ k[:n, : s["dv"]]).view(len(qt), h, -1))
        outs.append(torch.cat(rows))
    return torch.stack(outs)
