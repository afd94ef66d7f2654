"""kv_attn against a 64-bit restatement (torch on the device, pinned to
oracle/head_cache_oracle.py by the first test).

Tolerance, per output element: the result's rounding 2^-8 |o|; every weight's rounding to bf16,
at most 2^-8 of it: 2^-8 sum w |v|; a score is a sum of D products in fp32 and three more
roundings, so it is off by at most d = (D + 8) 2^-24 scale max_k sum |q| |k|, and numerator and
denominator move by that: 2 d sum w |v|; exponentials, sums and the joining of parts: 2^-16 of
sum w |v| (ex2.approx 2^-22, sums of at most 2^17 terms over 2^7 or more partial sums)."""
import math

import numpy as np
import pytest
import torch

from oracle import head_cache_oracle as O

pytestmark = pytest.mark.gpu

E4 = torch.float8_e4m3fn


def value_table():
    return torch.from_numpy(O.e4m3_values()).cuda()


def make(B, T, H, heads, d, page, block, lens, seed, spare=2, scale_bits=(-9, -6), codes=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    each = -(-(max(lens) + T) // page)
    pool = B * each + spare
    table = torch.randperm(pool, device="cuda", generator=g)[: B * each].view(B, each).int().contiguous()
    parts = []
    for _ in range(2):
        x = (torch.randn(pool, heads, page, d, device="cuda", generator=g) * 100).clamp(-448, 448).to(E4)
        s = torch.exp2(torch.randint(*scale_bits, (pool, heads, page // block), device="cuda", generator=g).float())
        parts += [x, s]
    q = torch.randn(B, T, H, d, device="cuda", generator=g).bfloat16()
    return g, q, parts, table, torch.tensor(lens, dtype=torch.int32, device="cuda")


def head_rows(x8, scale, pages, g, n):
    """float64 [n, D] of key head g."""
    page = x8.shape[2]
    block = page // scale.shape[2]
    at = torch.arange(n, device="cuda")
    p, r = pages.long()[at // page], at % page
    s = scale.view(torch.int32) & ~1  # without the mark
    return value_table()[x8.view(torch.uint8)[p, g, r].long()] * s.view(torch.float32)[p, g, r // block].double()[:, None]


def reference(q, parts, table, lens, sm, mask=None, sink=None, n_new=None):
    """(out, sum of w |v|, 2 d) in float64."""
    B, T, H, d = q.shape
    heads = parts[0].shape[1]
    G = H // heads
    out = torch.zeros(B, T, H, d, dtype=torch.float64, device="cuda")
    size, off = torch.zeros_like(out), torch.zeros(B, T, H, 1, dtype=torch.float64, device="cuda")
    for b in range(B):
        n, m = int(lens[b]), T if n_new is None else int(n_new[b])
        if m == 0:
            continue
        seen = torch.ones(m, n + m, dtype=torch.bool, device="cuda")
        seen[:, n:] = torch.ones(m, m, device="cuda").tril().bool() if mask is None else mask[b, :m, :m].bool()
        for g in range(heads):
            k, v = head_rows(parts[0], parts[1], table[b], g, n + m), head_rows(parts[2], parts[3], table[b], g, n + m)
            for t0 in range(0, m, max(1, (1 << 25) // (G * (n + m)))):
                t1 = min(m, t0 + max(1, (1 << 25) // (G * (n + m))))
                x = q[b, t0:t1, g * G:(g + 1) * G].double()
                s = (x.reshape(-1, d) @ k.T).view(t1 - t0, G, -1) * sm
                s = torch.where(seen[t0:t1, None], s, -math.inf)
                top = s.amax(-1, keepdim=True)
                if sink is not None:
                    sk = sink[g * G:(g + 1) * G].double()[None, :, None].expand_as(top)
                    top = torch.maximum(top, sk)
                top = torch.where(top == -math.inf, 0.0, top)
                e = torch.exp(s - top)
                den = e.sum(-1, keepdim=True)
                if sink is not None:
                    den = den + torch.exp(sk - top)
                w = torch.where(den == 0, 0.0, e / den)
                # keys that a row does not see have no part in it, whatever they hold
                bad = v.isnan()
                o = (w.reshape(-1, n + m) @ torch.where(bad, 0.0, v)).view(t1 - t0, G, d)
                if bad.any():
                    o = torch.where((seen[t0:t1].double() @ bad.double() > 0)[:, None], math.nan, o)
                out[b, t0:t1, g * G:(g + 1) * G] = o
                size[b, t0:t1, g * G:(g + 1) * G] = (w.reshape(-1, n + m) @ torch.where(bad, 0.0, v).abs()).view(t1 - t0, G, d)
                most = (x.reshape(-1, d).abs() @ torch.where(k.isnan(), 0.0, k).abs().T).view(t1 - t0, G, -1)
                most = torch.where(seen[t0:t1, None], most, 0.0).amax(-1, keepdim=True)
                off[b, t0:t1, g * G:(g + 1) * G] = 2 * (d + 8) * 2.0 ** -24 * abs(sm) * most
    return out, size, off


def check(q, parts, table, lens, sm, got=None, **kw):
    from kernelswift_b200 import ops

    if got is None:
        kw2 = {("attn_sink" if k == "sink" else k): v for k, v in kw.items()}
        got = ops.kv_attn(q, *parts, table, lens, sm, **kw2)
        ops.device_status()
    ref, size, off = reference(q, parts, table, lens, sm, **kw)
    g = got.double()
    assert torch.equal(g.isnan(), ref.isnan())
    lim = 2.0 ** -8 * ref.abs() + (2.0 ** -8 + 2.0 ** -16 + off) * size + 1e-30
    bad = ((g - ref).abs() > lim) & ~ref.isnan()
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist(), g[bad][:4].tolist(), ref[bad][:4].tolist())
    # weights and sums do not lean to one side: the mean error is far below a rounding
    fine = ~ref.isnan() & (size > 0)
    if int(fine.sum()) > 50000:
        assert float(((g - ref)[fine] / size[fine]).mean().abs()) < 2.0 ** -11
    return got


def tree_mask(g, B, T):
    return torch.rand(B, T, T, device="cuda", generator=g) < 0.5


def test_restatement(cuda_ok):
    g, q, parts, table, lens = make(2, 3, 4, 2, 64, 32, 16, [5, 40], 1)
    sink = torch.randn(4, device="cuda", generator=g)
    mask = tree_mask(g, 2, 3)
    out, size, _ = reference(q, parts, table, lens, 0.1, mask=mask, sink=sink)
    host = [x.view(torch.uint8).cpu().numpy() if x.dtype == E4 else x.double().cpu().numpy() for x in parts]
    for b in range(2):
        n = int(lens[b])
        k, v = (O.head_rows(host[i], host[i + 1], table[b].cpu().numpy(), n + 3) for i in (0, 2))
        for t in range(3):
            seen = np.concatenate([np.ones(n, bool), mask[b, t].cpu().numpy()])
            a, w = O.attn_token(q[b, t].double().cpu().numpy(), k, v, seen, 0.1, sink.double().cpu().numpy())
            assert np.allclose(out[b, t].cpu().numpy(), a, rtol=1e-10, atol=1e-12)
            assert np.allclose(size[b, t].cpu().numpy(), w, rtol=1e-10)


SHAPES = [
    (1, 1, 1, 1, 64, 16, 16, [0]), (1, 1, 16, 2, 128, 64, 16, [509]), (3, 1, 8, 8, 128, 64, 64, [0, 1, 127]),
    (2, 1, 10, 2, 64, 48, 48, [128, 1000]), (2, 1, 32, 2, 128, 32, 32, [255, 700]), (2, 5, 14, 2, 192, 16, 16, [3, 260]),
    (2, 4, 8, 4, 256, 128, 128, [1, 333]), (1, 3, 64, 1, 128, 80, 16, [500]), (4, 13, 64, 8, 128, 32, 32, [0, 17, 400, 901]),
    (2, 70, 6, 3, 64, 64, 16, [0, 90]), (1, 300, 4, 1, 128, 96, 32, [150]), (2, 130, 5, 5, 256, 64, 16, [100, 0]),
    (1, 129, 16, 2, 192, 112, 112, [64]), (3, 40, 16, 1, 128, 256, 128, [10, 700, 0]),
]


@pytest.mark.parametrize("B,T,H,heads,d,page,block,lens", SHAPES)
@pytest.mark.parametrize("kind", ["plain", "sink", "mask", "new"])
def test_shapes(cuda_ok, B, T, H, heads, d, page, block, lens, kind):
    g, q, parts, table, lens = make(B, T, H, heads, d, page, block, lens, B * 100 + T + d)
    kw = {}
    if kind != "plain":
        kw["sink"] = torch.randn(H, device="cuda", generator=g)
    if kind == "mask":
        kw["mask"] = tree_mask(g, B, T)
    if kind == "new":
        kw["n_new"] = torch.randint(0, T + 1, (B,), device="cuda", generator=g).int()
        kw["n_new"][0] = 0 if B > 1 else T
    got = check(q, parts, table, lens, d ** -0.5, **kw)
    if kind == "new":
        for b in range(B):
            assert not got[b, int(kw["n_new"][b]):].any()


@pytest.mark.parametrize("H,heads,T,n", [(8, 1, 1, 70001), (64, 8, 1, 20000), (4, 4, 1, 33000), (32, 2, 3, 9001), (128, 1, 2, 12345)])
def test_long_contexts_are_split_and_joined(cuda_ok, H, heads, T, n):
    g, q, parts, table, lens = make(1, T, H, heads, 128, 64, 16, [n], H + T)
    check(q, parts, table, lens, 128 ** -0.5)


@pytest.mark.parametrize("d", [64, 128, 192, 256])
@pytest.mark.parametrize("B,T,H,heads,n", [(4, 100, 32, 2, 3000), (1, 64, 64, 1, 10000), (3, 5, 20, 1, 50000), (20, 11, 24, 3, 2500),
                                           (2, 150, 6, 2, 1500)])
def test_stretches_of_many_tiles(cuda_ok, d, B, T, H, heads, n):
    """Every CTA walks several tiles of several row tiles, in every form of the kernels."""
    g, q, parts, table, lens = make(B, T, H, heads, d, 64, 16, [n - i for i in range(B)], d + T)
    check(q, parts, table, lens, d ** -0.5)


@pytest.mark.parametrize("B,T", [(200, 1), (64, 9), (700, 1)])
def test_many_ragged_sequences(cuda_ok, B, T):
    lens = [(i * 37) % 300 for i in range(B)]
    g, q, parts, table, lens = make(B, T, 6, 2, 64, 32, 32, lens, B)
    check(q, parts, table, lens, 0.125, sink=torch.randn(6, device="cuda", generator=g))


def test_a_table_wider_than_the_contexts(cuda_ok):
    g, q, parts, table, lens = make(3, 2, 8, 2, 128, 64, 16, [100, 7, 300], 4)
    wide = torch.full((3, 3000), 10 ** 8, dtype=torch.int32, device="cuda")
    wide[:, : table.shape[1]] = table
    a = check(q, parts, wide, lens, 0.1)
    assert torch.allclose(a.float(), check(q, parts, table, lens, 0.1).float(), rtol=2 ** -6, atol=1e-3)


@pytest.mark.parametrize("T", [1, 40])
def test_running_maximum_grows_late(cuda_ok, T):
    g, q, parts, table, lens = make(1, T, 8, 1, 128, 64, 16, [2000], 6)
    at = torch.arange(parts[0].shape[0], device="cuda")
    order = torch.zeros_like(at)
    order[table[0].long()] = torch.arange(table.shape[1], device="cuda")
    parts[1].copy_(torch.exp2((-12 + order // 3).float())[:, None, None].expand_as(parts[1]))
    check(q, parts, table, lens, 1.0)


@pytest.mark.parametrize("T", [1, 33])
def test_masks_that_leave_nothing(cuda_ok, T):
    g, q, parts, table, lens = make(3, T, 8, 2, 128, 64, 16, [0, 0, 50], 8)
    mask = tree_mask(g, 3, T)
    mask[0] = False
    mask[1, 0] = False
    got = check(q, parts, table, lens, 0.1, mask=mask)
    assert not got[0].any() and not got[1, 0].any()
    check(q, parts, table, lens, 0.1, mask=mask, sink=torch.randn(8, device="cuda", generator=g))


@pytest.mark.parametrize("T", [1, 3, 40, 200])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_hidden_rows_may_hold_anything(cuda_ok, T, d):
    """Stale codes (NaN among them) and scales (NaN, infinite) behind the last row, and pages
    that nobody may read."""
    g, q, parts, table, lens = make(2, T, 8, 2, d, 64, 16, [70, 5], 9, spare=3)
    new = torch.tensor([max(1, T - 3), T], dtype=torch.int32, device="cuda")
    want = check(q, parts, table, lens, 0.1, n_new=new)
    used = torch.zeros(parts[0].shape[0], 64, dtype=torch.bool, device="cuda")
    for b in range(2):
        at = torch.arange(int(lens[b] + new[b]), device="cuda")
        used[table[b].long()[at // 64], at % 64] = True
    for i in (0, 2):
        x = parts[i].view(torch.uint8)
        x.copy_(torch.where(used[:, None, :, None], x, 0x7F))
        blocks = used.view(-1, 4, 16).any(-1)[:, None]
        parts[i + 1].copy_(torch.where(blocks, parts[i + 1], math.nan if i else math.inf))
    got = check(q, parts, table, lens, 0.1, n_new=new)
    assert torch.equal(got, want)


@pytest.mark.parametrize("T", [1, 4, 150])
@pytest.mark.parametrize("d", [64, 128, 192, 256])
@pytest.mark.parametrize("n", [40, 1500])
def test_nan_elements_reach_only_what_sees_them(cuda_ok, T, d, n):
    """Appended NaN and infinities: a value's makes its column of the rows that see it NaN, a
    key's the whole row."""
    from kernelswift_b200 import ops

    heads, H = 2, 6
    g, q, parts, table, lens = make(2, T, H, heads, d, 32, 16, [n, n + 3], 10)
    k, v = (torch.randn(2, T, heads, d, device="cuda", generator=g).bfloat16() for _ in range(2))
    v[0, T // 2, 1, 5] = math.nan
    v[0, 0, 0, d - 1] = -math.inf
    k[1, T - 1, 0, 7] = math.inf
    ops.kv_append(k, v, *parts, table, lens)
    mask = torch.ones(2, T, T, device="cuda").tril().bool()
    mask[0, T - 1, 0] = False
    for kw in ({}, {"mask": mask}):
        got = check(q, parts, table, lens, 0.1, **kw)
        # (masked, a single token does not see its own row)
        assert got[0, :, 3:, 5].isnan().any() == (T > 1 or not kw)
        assert got[1, T - 1, :3].isnan().all() and not got[1, :, 3:].isnan().any()
        assert not got[0, :, :3, : d - 1].isnan().any()


def test_queries_that_are_not_finite_stay_in_their_rows(cuda_ok):
    from kernelswift_b200 import ops

    for T in (1, 40):
        g, q, parts, table, lens = make(1, T, 8, 2, 128, 64, 16, [300], 12)
        clean = ops.kv_attn(q, *parts, table, lens, 0.1)
        q2 = q.clone()
        q2[0, 0, 1, 3] = math.nan
        q2[0, T - 1, 6, 100] = math.inf
        got = ops.kv_attn(q2, *parts, table, lens, 0.1)
        rows = torch.ones(T, 8, dtype=torch.bool, device="cuda")
        rows[0, 1] = rows[T - 1, 6] = False
        assert got[0, 0, 1].isnan().all() and torch.equal(got[0][rows], clean[0][rows])


@pytest.mark.parametrize("T", [1, 40])
@pytest.mark.parametrize("bits", [-22, 0, 7, 8, 60, 110, 118])
def test_scales_over_the_whole_range(cuda_ok, T, bits):
    """Values up to the largest that bf16 holds (448 * 2^119 needs all its range: 2^118 here, the
    codes being below 448); keys as large with a softmax scale that brings them back."""
    g, q, parts, table, lens = make(2, T, 8, 2, 128, 64, 16, [300, 1000], 14)
    parts[3].mul_(2.0 ** (bits + 7) if bits < 118 else 2.0 ** 125)
    check(q, parts, table, lens, 0.1)
    parts[1].mul_(2.0 ** min(bits, 100))
    check(q, parts, table, lens, 0.1 * 2.0 ** -min(bits, 100))


@pytest.mark.parametrize("T", [1, 40])
@pytest.mark.parametrize("big", [2.0 ** 30, 2.0 ** 100])
def test_large_rows_without_weight(cuda_ok, T, big):
    """Hidden rows, and seen ones of no weight, of any size take no precision from the others."""
    g, q, parts, table, lens = make(1, T, 8, 1, 128, 64, 16, [500], 15)
    parts[3][table[0, 2].long()] *= big
    x = parts[0].view(torch.uint8)
    x[table[0, 2].long()] = 0  # scores of 0 ..
    sink = torch.full((8,), 200.0, device="cuda")  # .. with a weight of e^-200
    check(q, parts, table, lens, 0.1, sink=sink)
    check(q, parts, table, lens, 0.1)


@pytest.mark.parametrize("T", [1, 40])
@pytest.mark.parametrize("down", [5.0, 21.0, 24.0, 60.0])
def test_weights_far_below_the_largest(cuda_ok, T, down):
    """Rows whose largest weights meet zeros only: what shows is weights of e^-down.  Each may be
    off by 2^-32 of the largest, so an output by 2^-32 sum |v| more than elsewhere."""
    from kernelswift_b200 import ops

    g, q, parts, table, lens = make(1, T, 8, 2, 128, 64, 16, [200], 40)
    q.fill_(1.0)
    first = table[0, 0].long()
    parts[1].fill_(2.0 ** -7)
    parts[0].view(torch.uint8).fill_(0xB8)  # -1: scores of -128 * 2^-7 times the softmax scale
    for x in (parts[0], parts[2]):
        x.view(torch.uint8)[first] = 0  # 64 keys with scores of 0 and no values
    got = ops.kv_attn(q, *parts, table, lens, down).double()
    ops.device_status()
    ref, size, off = reference(q, parts, table, lens, down)
    most = sum(head_rows(parts[2], parts[3], table[0], h, 200 + T).abs().sum(0).max() for h in range(2))
    lim = 2.0 ** -8 * ref.abs() + (2.0 ** -8 + 2.0 ** -16 + off) * size + 2.0 ** -32 * most
    assert ((got - ref).abs() <= lim).all()


@pytest.mark.parametrize("T", [1, 2, 40])
@pytest.mark.parametrize("big,key", [(2.0 ** 20, 1), (2.0 ** 60, 0), (2.0 ** 100, 0), (2.0 ** 126, 0), (2.0 ** 40, 1), (2.0 ** -130, 1)])
def test_queries_of_any_size_within_a_row(cuda_ok, T, big, key):
    """Columns of a query that are far larger than the others, where the keys are zero (then the
    others make the score) or where they are not."""
    g, q, parts, table, lens = make(1, T, 8, 2, 128, 64, 16, [300], 30)
    q[..., ::2] *= big
    if not key:
        parts[0].view(torch.uint8)[..., ::2] = 0
    check(q, parts, table, lens, 0.1 if big < 1 or not key else 0.1 / big)
    q[..., 1::4] *= 2.0 ** -20
    check(q, parts, table, lens, 0.1 if big < 1 or not key else 0.1 / big)


@pytest.mark.parametrize("T", [1, 40])
@pytest.mark.parametrize("size", [2.0 ** -126, 2.0 ** -60, 2.0 ** 60, 2.0 ** 127])
def test_queries_of_any_size(cuda_ok, T, size):
    g, q, parts, table, lens = make(1, T, 8, 2, 64, 64, 16, [300], 31)
    q.copy_(q.clamp(-1, 1) * size)
    assert q.isfinite().all()
    # (scores are sums before the softmax scale: keys of 2^-6 keep them finite)
    parts[1].fill_(2.0 ** -14)
    check(q, parts, table, lens, 0.1 / size if size < 2.0 ** 100 else 2.0 ** -126)


@pytest.mark.parametrize("sm", [0.0, -0.07, 1e-30, 40.0])
def test_any_softmax_scale(cuda_ok, sm):
    for T in (1, 40):
        g, q, parts, table, lens = make(2, T, 8, 2, 64, 64, 16, [300, 20], 16)
        check(q, parts, table, lens, sm)


@pytest.mark.parametrize("n", [60, 3000])
def test_sinks_of_any_size(cuda_ok, n):
    for T in (1, 40):
        g, q, parts, table, lens = make(1, T, 8, 2, 128, 64, 16, [n], 17)
        sink = torch.tensor([-1e30, -300.0, -20, 0, 20, 300, 1e30, -math.inf], device="cuda")
        got = check(q, parts, table, lens, 0.1, sink=sink)
        assert not got[:, :, 6].any()


def test_bad_pages_and_lengths_are_reported(cuda_ok):
    from kernelswift_b200 import ops

    for T in (1, 40):
        g, q, parts, table, lens = make(2, T, 8, 2, 128, 64, 16, [200, 90], 18)
        good = ops.kv_attn(q, *parts, table, lens, 0.1)
        bad = table.clone()
        bad[0, 1], bad[0, 2] = -1, 10 ** 7
        got = ops.kv_attn(q, *parts, bad, lens, 0.1)
        with pytest.raises(RuntimeError, match="index"):
            ops.device_status()
        assert torch.equal(got[1], good[1]) and got[0].isfinite().all()
        got = ops.kv_attn(q, *parts, table, lens + 10 ** 6, 0.1)
        with pytest.raises(RuntimeError, match="index"):
            ops.device_status()
        assert got.isfinite().all()
        check(q, parts, table, lens, 0.1)


def test_repeats_streams_workspace_and_out(cuda_ok):
    from kernelswift_b200 import ops

    for T in (1, 30):
        g, q, parts, table, lens = make(3, T, 16, 2, 128, 64, 16, [5000, 3, 700], 20)
        first = check(q, parts, table, lens, 0.1)
        ws = torch.full((ops.kv_attn_workspace_size(T, 16, 2, 128),), 255, dtype=torch.uint8, device="cuda")
        out = torch.full_like(first, 7.0)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            assert ops.kv_attn(q, *parts, table, lens, 0.1, out=out, workspace=ws) is out
        torch.cuda.current_stream().wait_stream(s)
        assert torch.equal(out, first)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            third = ops.kv_attn(q, *parts, table, lens, 0.1)
        graph.replay()
        assert torch.equal(third, first)
        lens.copy_(torch.tensor([17, 4900, 0], device="cuda"))  # other lengths, the same graph
        graph.replay()
        check(q, parts, table, lens, 0.1, got=third)
        with pytest.raises(RuntimeError, match="workspace"):
            ops.kv_attn(q, *parts, table, lens, 0.1, workspace=ws[:-256])


def test_two_calls_at_once(cuda_ok):
    from kernelswift_b200 import ops

    a, b = (make(2, T, 16, 4, 128, 64, 16, [9000, 300], 21 + T)[1:] for T in (1, 20))
    want = [ops.kv_attn(x[0], *x[1], x[2], x[3], 0.1) for x in (a, b)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(5):
        for i, (s, x) in enumerate(zip(streams, (a, b))):
            with torch.cuda.stream(s):
                got[i].append(ops.kv_attn(x[0], *x[1], x[2], x[3], 0.1))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_offsets_past_32_bits(cuda_ok):
    for T in (1, 40):
        pages, heads, page, d = 140000, 4, 64, 128
        g = torch.Generator(device="cuda").manual_seed(1)
        x8 = torch.zeros(pages, heads, page, d, dtype=torch.uint8, device="cuda")
        assert x8.numel() > 2 ** 32
        scale = torch.full((pages, heads, 4), 2.0 ** -7, device="cuda")
        table = torch.tensor([[pages - 1, 5, pages - 2, pages - 70000]], dtype=torch.int32, device="cuda")
        for p in table[0].tolist():
            x8[p] = (torch.randn(heads, page, d, device="cuda", generator=g) * 100).clamp(-448, 448).to(E4).view(torch.uint8)
        q = torch.randn(1, T, 16, d, device="cuda", generator=g).bfloat16()
        lens = torch.tensor([190], dtype=torch.int32, device="cuda")
        check(q, [x8.view(E4), scale, x8.view(E4), scale], table, lens, 0.1)
        del x8


def test_empty_calls(cuda_ok):
    from kernelswift_b200 import ops

    g, q, parts, table, lens = make(2, 1, 8, 2, 128, 64, 16, [5, 6], 25)
    assert ops.kv_attn(q[:, :0], *parts, table, lens, 0.1).shape == (2, 0, 8, 128)
    assert ops.kv_attn(q[:0], *parts, table[:0], lens[:0], 0.1).shape == (0, 1, 8, 128)
    with pytest.raises(RuntimeError, match="64, 128, 192 or 256"):
        ops.kv_attn(q[..., :32].contiguous(), parts[0][..., :32].contiguous(), parts[1], parts[2][..., :32].contiguous(),
                    parts[3], table, lens, 0.1)


@pytest.mark.parametrize("d", [192, 256])
@pytest.mark.parametrize("T,longest", [(3, 40), (9, 300)])
def test_many_short_row_tiles_of_wide_heads(cuda_ok, d, T, longest):
    """Every CTA of the kernel for many rows goes through a dozen row tiles of one to three tiles each,
    call after call: its warpgroups stay in step, and no wait runs out."""
    from kernelswift_b200 import ops

    lens = [(i * 37) % longest for i in range(450)]
    g, q, parts, table, lens = make(450, T, 16, 4, d, 64, 16, lens, d + T)
    want = check(q, parts, table, lens, d ** -0.5)
    for _ in range(100):
        got = ops.kv_attn(q, *parts, table, lens, d ** -0.5)
    assert torch.equal(got, want)
    ops.device_status()


@pytest.mark.parametrize("T", [1, 4, 40])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("codes,bits", [(0x7F, 0x7F800000), (0xFF, 0x7FC00001), (0x7F, 0x3C000001)])
def test_missing_pages_are_not_seen_whatever_the_first_page_holds(cuda_ok, T, d, codes, bits):
    """Pages outside the pool: the result is that of the sequence without them.  The pool's first
    page is nobody's, all NaN codes, its scales infinite, NaN or marked."""
    from kernelswift_b200 import ops

    g, q, parts, table, lens = make(2, T, 8, 2, d, 64, 16, [200, 90], 44 + T + d)
    spare = next(p for p in range(parts[0].shape[0]) if p and not (table == p).any())
    table[table == 0] = spare
    for i in (0, 2):
        parts[i].view(torch.uint8)[0] = codes
        parts[i + 1].view(torch.int32)[0] = bits
    # the first sequence loses two pages in its middle, the second its last ones, its own tokens' among them
    bad, left = table.clone(), table.clone()
    bad[0, 1], bad[0, 2], bad[1, 1:] = -1, 10 ** 7, parts[0].shape[0]
    left[0, 1:-2] = table[0, 3:]
    mask = torch.ones(2, T, T, device="cuda").tril().bool()
    mask[1] = False
    got = ops.kv_attn(q, *parts, bad, lens, 0.1)
    with pytest.raises(RuntimeError, match="index"):
        ops.device_status()
    check(q, parts, left, torch.tensor([200 - 128, 64], device="cuda"), 0.1, got=got, mask=mask)


@pytest.mark.parametrize("T", [1, 4])
@pytest.mark.parametrize("top", [0, 14, 40, 97, 120])
@pytest.mark.parametrize("small", [112, 115, 118, 121, 124, 127, 130, 132])
def test_small_elements_of_a_query_count_once(cuda_ok, T, top, small):
    """Elements of 2^-small, down to bf16's least numbers, beside ones of 2^-top that meet zero keys, in
    every other head; the heads between have small ones alone.  The keys and the softmax scale
    bring the small ones back."""
    g, q, parts, table, lens = make(1, T, 8, 2, 64, 64, 16, [300], small * 100 + top)
    e = torch.full((8, 64), -float(small), dtype=torch.float64, device="cuda")
    e[::2, ::4] = -float(top)
    q = (q.double() * torch.exp2(e)).bfloat16()
    parts[0].view(torch.uint8)[..., ::4] = 0
    parts[1].mul_(2.0 ** 20)
    check(q, parts, table, lens, 2.0 ** (small - 22))


@pytest.mark.parametrize("T", [1, 4])
@pytest.mark.parametrize("d", [64, 256])
def test_rows_beside_a_widely_spread_one_lose_nothing(cuda_ok, T, d):
    """Every other head has elements of 2^120, which meet zero keys, and of 2^-130; the heads between have
    ordinary ones, and some of 2^-25."""
    g, q, parts, table, lens = make(1, T, 8, 2, d, 64, 16, [300], 45 + T)
    q[..., ::2, ::4] *= 2.0 ** 120
    q[..., ::2, 1::4] *= 2.0 ** -130
    q[..., 1::2, 2::4] *= 2.0 ** -25
    parts[0].view(torch.uint8)[..., ::4] = 0
    check(q, parts, table, lens, 0.1)


@pytest.mark.parametrize("d,T,H", [(64, 1, 16), (64, 2, 16), (128, 1, 16), (128, 2, 16), (192, 1, 16), (256, 1, 16)])
def test_weights_of_few_rows_are_good_to_half_a_step_of_fp16(cuda_ok, d, T, H):
    """Values that cancel, so that the weights' rounding shows: two keys, the second one's values the
    negative of the first one's.  Each weight is off by at most 2^-11 of itself (2^-32 of the largest
    where it is smaller than fp16's normal numbers), the sum of them by no rounding but fp32's."""
    from kernelswift_b200 import ops

    B = 64
    g, q, parts, table, lens = make(B, T, H, 2, d, 16, 16, [1] * B, 50 + d + T)
    codes = parts[2].view(torch.uint8)
    codes[:, :, 1] = codes[:, :, 0] ^ 0x80
    mask = torch.zeros(B, T, T, dtype=torch.bool, device="cuda")
    mask[:, :, 0] = True  # every token sees the cached row and the first new one
    got = ops.kv_attn(q, *parts, table, lens, d ** -0.5, mask=mask).double()
    ops.device_status()
    ref, size, off = reference(q, parts, table, lens, d ** -0.5, mask=mask)
    most = size.amax()
    lim = 2.0 ** -8 * ref.abs() + (2.0 ** -11 + 2.0 ** -16 + off) * size + 2.0 ** -32 * most
    assert ((got - ref).abs() <= lim).all()
    assert float((ref.abs() < 0.1 * size).double().mean()) > 0.05  # many do cancel
