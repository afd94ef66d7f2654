"""tree_attn against the 64-bit restatement (oracle/cache_oracle.py).

Tolerance, per element, A = sum w |v| (bf16 has 8 significant bits: a rounding is off by
at most 2^-8 of the value): the result is rounded to bf16, 2^-8 of |out| <= A; the
kernel rounds each weight before the product with v, to bf16 for v's bf16 columns (at most
2^-8 of A) and to three e5m2 parts for its e4m3 ones (2^-9); what is left is fp32 (scores of
size ~10 off by about 1e-5, sums of exponentials), for which 2^-12 of A is room.  |got - exact| <= (2^-8 + 2^-8 + 2^-12) A.
"""
import numpy as np
import pytest
import torch

from helpers import bits_from_bf16
from oracle import cache_oracle as C

pytestmark = pytest.mark.gpu
TOL = 2.0 ** -8 + 2.0 ** -8 + 2.0 ** -12


def build(B, T, H, dq, dr, page, lens, seed, spare=2, key_scale=None, q_scale=1.0):
    """Queries and a filled paged cache; the slots no sequence reaches hold NaN."""
    from kernelswift_b200 import ops

    g = torch.Generator(device="cuda").manual_seed(seed)
    each = max(1, -(-(max(lens) + T) // page))
    pages = B * each + spare
    table = torch.randperm(pages, device="cuda", generator=g)[:B * each].view(B, each).int().contiguous()
    kv8 = torch.full((pages, page, dq), 0x7F, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    scale = torch.full((pages, page), float("nan"), device="cuda")
    tail = torch.full((pages, page, dr), float("nan"), dtype=torch.bfloat16, device="cuda") if dr else None
    for b in range(B):
        n = lens[b] + T
        kv = torch.randn(n, dq + dr, device="cuda", generator=g)
        if key_scale is not None:
            kv *= key_scale(torch.arange(n, device="cuda").float())[:, None]
        pos = torch.arange(n, device="cuda")
        ops.cache_write(kv.bfloat16(), table[b].long()[pos // page] * page + pos % page, kv8, scale, tail)
    q = (q_scale * torch.randn(B, T, H, dq + dr, device="cuda", generator=g)).bfloat16()
    return g, q, kv8, scale, tail, table, torch.tensor(lens, dtype=torch.int32, device="cuda")


def check(q, kv8, scale, tail, table, lens, sm, dv, mask=None, sink=None, got=None, rows=None):
    """Compare every (or a sample of) drafted token's output; returns the output."""
    from kernelswift_b200 import ops

    if got is None:
        got = ops.tree_attn(q, kv8, scale, tail, table, lens, sm, dv=dv, mask=mask, attn_sink=sink)
        ops.device_status()
    B, T, H, D = q.shape
    codes = kv8.view(torch.uint8).cpu().numpy().reshape(-1, kv8.shape[-1])
    s = scale.double().cpu().numpy().reshape(-1)
    t = tail.double().cpu().numpy().reshape(-1, tail.shape[-1]) if tail is not None else None
    snk = sink.double().cpu().numpy() if sink is not None else None
    qn, gn = q.double().cpu().numpy(), got.double().cpu().numpy()
    assert got.shape == (B, T, H, dv) and got.dtype == torch.bfloat16
    for b in range(B):
        n = int(lens[b])
        r = C.sequence_rows(codes, s, t, (table[b].cpu().numpy(), kv8.shape[1]), n + T)
        for i in (range(T) if rows is None else rows):
            seen = np.ones(n + T, bool)
            seen[n:] = mask[b, i].cpu().numpy() if mask is not None else np.arange(T) <= i
            ref, size = C.tree_attn_row(qn[b, i], r, seen, sm, snk, dv)
            err = np.abs(gn[b, i] - ref)
            assert (err <= TOL * size + 1e-37).all(), (b, i, float((err / np.maximum(size, 1e-30)).max()))
    return got


def tree_mask(g, B, T, p=0.5):
    m = (torch.rand(B, T, T, device="cuda", generator=g) < p).tril()
    return m | torch.eye(T, dtype=torch.bool, device="cuda")


@pytest.mark.parametrize("B,T,H,dq,dr,dv,page,lens", [
    (1, 1, 16, 128, 0, 128, 64, [0]),
    (1, 1, 16, 128, 0, 128, 64, [1]),
    (4, 1, 16, 512, 64, 512, 64, [127, 128, 126, 255]),
    (3, 1, 128, 512, 64, 512, 64, [300, 0, 129]),
    (2, 5, 20, 448, 64, 512, 48, [200, 77]),
    (3, 13, 64, 448, 64, 448, 32, [60, 500, 1]),
    (2, 33, 5, 192, 64, 192, 100, [1000, 3]),
    (1, 64, 1, 64, 64, 64, 1, [90]),
    (5, 2, 7, 256, 64, 320, 256, [1, 2, 3, 700, 5]),
    (2, 3, 40, 64, 0, 64, 16, [130, 400]),
    (1, 130, 3, 320, 0, 256, 7, [20]),
    (2, 4, 32, 512, 0, 128, 64, [640, 641]),
    (1, 2, 200, 128, 64, 192, 64, [333]),
    (70, 1, 8, 128, 64, 128, 16, [3 * i for i in range(70)]),
])
@pytest.mark.parametrize("tree,sink", [(False, False), (True, True)])
def test_shapes(cuda_ok, B, T, H, dq, dr, dv, page, lens, tree, sink):
    g, *a = build(B, T, H, dq, dr, page, lens, seed=B * 100 + T * 10 + H)
    mask = tree_mask(g, B, T) if tree else None
    snk = torch.randn(H, device="cuda", generator=g) if sink else None
    check(*a, (dq + dr) ** -0.5, dv, mask, snk, rows=None if T < 20 else [0, 1, T // 2, T - 1])


@pytest.mark.parametrize("H,T,n", [(16, 1, 40000), (128, 1, 20000), (64, 8, 9001), (3, 2, 70001)])
def test_long_context_is_split_and_joined(cuda_ok, H, T, n):
    g, *a = build(1, T, H, 512, 64, 64, [n], seed=H)
    check(*a, 576 ** -0.5, 512, rows=[0, T - 1])


@pytest.mark.parametrize("B,T,H,n", [(1, 1, 16, 500), (3, 5, 24, 130), (40, 1, 16, 900), (9, 7, 64, 250)])
def test_short_contexts_in_short_and_wide_tables(cuda_ok, B, T, H, n):
    """A short table takes a CTA per row tile, a wide one (whose entries past the context are
    never looked at) is split: both are right."""
    g, q, kv8, scale, tail, table, lens = build(B, T, H, 448, 64, 32, [max(0, n - 31 * b) for b in range(B)], seed=n)
    sink = torch.randn(H, device="cuda", generator=g)
    mask = tree_mask(g, B, T)
    wide = torch.cat([table, torch.full((B, 300), -7, device="cuda", dtype=torch.int32)], 1)
    for t in (table, wide):
        check(q, kv8, scale, tail, t, lens, 512 ** -0.5, 512, mask, sink)


@pytest.mark.parametrize("dq,dr,dv", [(512, 64, 128), (512, 0, 384), (384, 64, 64), (256, 0, 128), (320, 64, 256)])
def test_values_narrower_than_the_codes(cuda_ok, dq, dr, dv):
    """Chunks of which only the scores read go back to the loads before the others."""
    from kernelswift_b200 import ops

    g, *a = build(4, 3, 40, dq, dr, 64, [5000, 1300, 1, 257], seed=dv)
    first = check(*a, (dq + dr) ** -0.5, dv)
    for _ in range(20):
        assert torch.equal(first, ops.tree_attn(*a, (dq + dr) ** -0.5, dv=dv))
    ops.device_status()


@pytest.mark.parametrize("tree", [False, True])
def test_rows_of_many_sequences_at_once(cuda_ok, tree):
    """More work items than CTAs, ragged, some sequences empty."""
    lens = [(37 * i) % 900 if i % 5 else 0 for i in range(180)]
    g, *a = build(180, 3, 32, 128, 64, 32, lens, seed=4)
    check(*a, 0.07, 192, tree_mask(g, 180, 3) if tree else None)


def test_running_maximum_grows_late(cuda_ok):
    """Scores that grow by hundreds along the keys, shrink, and spike at single keys."""
    for shape in (lambda x: 1 + x / 40, lambda x: torch.clamp(20 - x / 30, min=0.01),
                  lambda x: torch.where(x % 131 == 130, 30.0, 0.1)):
        g, *a = build(2, 3, 24, 512, 64, 64, [1500, 900], seed=9, key_scale=shape, q_scale=2.0)
        check(*a, 576 ** -0.5, 512)


def test_large_and_small_magnitudes(cuda_ok):
    """Rows whose scales are far from 1, in both directions, in one sequence."""
    g, *a = build(2, 2, 16, 448, 64, 64, [300, 200], seed=12, q_scale=2.0 ** -20,
                  key_scale=lambda x: torch.exp2((x % 41) - 20))
    check(*a, 1.0, 512)


@pytest.mark.parametrize("at", [0, 200, 399])
@pytest.mark.parametrize("dv", [128, 192])
def test_large_rows_without_weight_take_no_precision(cuda_ok, at, dv):
    """One row 2^24 times as large as the others whose score rules it out: the others are as
    exact as without it.  And the reverse: one small row that has nearly all the weight."""
    from kernelswift_b200 import ops

    g, q, kv8, scale, tail, table, lens = build(1, 1, 1, 128, 64, 32, [400], seed=31)
    slot = (table[0, at // 32].long() * 32 + at % 32).view(1)
    away = (-2.0 ** 24 * q.float().view(1, 192)).bfloat16()
    ops.cache_write(away, slot, kv8, scale, tail)
    check(q, kv8, scale, tail, table, lens, 192 ** -0.5, dv)
    strong = torch.full((1, 1, 1, 192), 2.0 ** 12, device="cuda").bfloat16()
    ops.cache_write((2.0 ** -9 * torch.ones(1, 192, device="cuda")).bfloat16(), slot, kv8, scale, tail)
    other = torch.arange(401, device="cuda")
    other = other[other != at]
    kv = torch.randn(400, 192, device="cuda", generator=g)
    kv -= kv.mean(1, keepdim=True) + 0.01     # scores of -0.01 * 192 * 2^12 against 2^-9 * 192 * 2^12
    ops.cache_write(kv.bfloat16(), table[0].long()[other // 32] * 32 + other % 32, kv8, scale, tail)
    check(strong, kv8, scale, tail, table, lens, 2.0 ** -8, dv)


@pytest.mark.parametrize("big", [2.0 ** -120, 2.0 ** 60])
def test_scales_at_the_ends_of_the_range(cuda_ok, big):
    """A cache filled by hand, its scales (powers of two) far from 1 and some of them 0."""
    g = torch.Generator(device="cuda").manual_seed(15)
    pages, page, n = 6, 64, 300
    code = torch.randint(0, 256, (pages, page, 192), device="cuda", generator=g)
    code = torch.where((code & 127) == 127, 0x38, code).to(torch.uint8)
    scale = big * torch.exp2(torch.randint(-3, 4, (pages, page), device="cuda", generator=g).float())
    scale[:, ::7] = 0
    q = (torch.randn(1, 2, 20, 192, device="cuda", generator=g) * 0.004 / big).bfloat16()
    table = torch.arange(pages, device="cuda").int()[None].contiguous()
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    check(q, code.view(torch.float8_e4m3fn), scale, None, table, lens, 0.07, 192)


def test_masks_that_leave_nothing(cuda_ok):
    """A token whose mask row is empty on an empty context gives zeros, with and without a
    sink; its neighbours are untouched."""
    from kernelswift_b200 import ops

    for sink in (None, torch.randn(16, device="cuda")):
        g, *a = build(3, 6, 16, 128, 64, 16, [0, 5, 0], seed=2)
        mask = tree_mask(g, 3, 6)
        mask[0, 2] = False
        mask[1, 3] = False
        mask[2] = False
        got = check(*a, 0.1, 128, mask, sink)
        assert (got[0, 2] == 0).all() and (got[2] == 0).all() and (got[1, 3] != 0).any()


def test_nan_rows_reach_only_the_tokens_that_see_them(cuda_ok):
    from kernelswift_b200 import ops

    B, T, H = 2, 5, 16
    g, q, kv8, scale, tail, table, lens = build(B, T, H, 128, 64, 32, [50, 70], seed=6)
    mask = tree_mask(g, B, T)
    mask[0, :, 2] = False
    mask[0, 2, 2] = mask[0, 4, 2] = True
    bad = torch.randn(1, 192, device="cuda").bfloat16()
    bad[0, 150] = float("inf")
    pos = 50 + 2
    slot = table[0, pos // 32].long() * 32 + pos % 32
    clean = ops.tree_attn(q, kv8, scale, tail, table, lens, 0.1, dv=192, mask=mask)
    ops.cache_write(bad, slot.view(1), kv8, scale, tail)
    got = ops.tree_attn(q, kv8, scale, tail, table, lens, 0.1, dv=192, mask=mask)
    ops.device_status()
    hit = torch.zeros(B, T, dtype=torch.bool, device="cuda")
    hit[0, 2] = hit[0, 4] = True
    assert got[hit].isnan().all()
    assert torch.equal(got[~hit], clean[~hit])
    # a marked row of the shared context reaches every token of its sequence, no other
    ops.cache_write(bad, (table[1, 0].long() * 32 + 3).view(1), kv8, scale, tail)
    got = ops.tree_attn(q, kv8, scale, tail, table, lens, 0.1, dv=192, mask=mask)
    assert got[1].isnan().all() and torch.equal(got[0][~hit[0]], clean[0][~hit[0]])


def test_infinite_queries_stay_in_their_rows(cuda_ok):
    from kernelswift_b200 import ops

    g, q, *rest = build(2, 3, 20, 128, 0, 32, [40, 300], seed=8)
    clean = ops.tree_attn(q, *rest, 0.1)
    q[0, 1, 3, 5] = float("inf")
    q[1, 2, 19, 0] = float("nan")
    got = ops.tree_attn(q, *rest, 0.1)
    hit = torch.zeros(2, 3, 20, dtype=torch.bool, device="cuda")
    hit[0, 1, 3] = hit[1, 2, 19] = True
    assert got[hit].isnan().all() and torch.equal(got[~hit], clean[~hit])


def test_one_token_equals_sparse_attention_over_the_same_rows(cuda_ok):
    """T = 1 against ops.sparse_attn on the rows read back (its own rounding of the
    weights: twice the tolerance apart)."""
    from kernelswift_b200 import ops

    g, q, kv8, scale, tail, table, lens = build(2, 1, 64, 512, 64, 64, [255, 255], seed=3)
    sink = torch.randn(64, device="cuda", generator=g)
    rows = ops.cache_read(kv8, scale, tail, table, lens + 1, 256)
    idx = torch.arange(256, device="cuda").int().expand(2, 1, 256).contiguous()
    a = ops.tree_attn(q, kv8, scale, tail, table, lens, 576 ** -0.5, dv=512, attn_sink=sink)
    b = ops.sparse_attn(q, rows, sink, idx, 576 ** -0.5, dv=512)
    size = ops.sparse_attn(q, rows.abs(), sink, idx, 0.0, dv=512).float().amax()
    assert (a.float() - b.float()).abs().max() <= 2 * TOL * 3 * size


def test_bad_pages_are_skipped_and_reported(cuda_ok):
    from kernelswift_b200 import ops

    g, q, kv8, scale, tail, table, lens = build(2, 2, 16, 128, 64, 32, [90, 90], seed=5)
    good = ops.tree_attn(q, kv8, scale, tail, table, lens, 0.1, dv=128)
    broken = table.clone()
    broken[1, 1] = kv8.shape[0]
    got = ops.tree_attn(q, kv8, scale, tail, broken, lens, 0.1, dv=128)
    with pytest.raises(RuntimeError, match="device status"):
        ops.device_status()
    assert torch.equal(got[0], good[0]) and torch.isfinite(got[1].float()).all()
    lens[0] = 10 ** 6  # longer than the table: the positions past it are skipped
    got = ops.tree_attn(q, kv8, scale, tail, table, lens, 0.1, dv=128)
    with pytest.raises(RuntimeError, match="device status"):
        ops.device_status()
    assert torch.equal(got[1], good[1])
    ops.device_status()


def test_repeats_streams_workspace_and_out(cuda_ok):
    from kernelswift_b200 import ops

    g, *a = build(3, 4, 48, 512, 64, 64, [5000, 100, 2500], seed=7)
    ref = ops.tree_attn(*a, 0.05, dv=512)
    need = ops.tree_attn_workspace_size(3, 4, 48, 512)
    ws = torch.full((need,), 0xFF, dtype=torch.uint8, device="cuda")
    out = torch.empty_like(ref)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(5):
            out.fill_(7)
            assert ops.tree_attn(*a, 0.05, dv=512, out=out, workspace=ws) is out
    side.synchronize()
    assert np.array_equal(bits_from_bf16(out), bits_from_bf16(ref))
    empty = a[0][:, :0].contiguous()
    assert ops.tree_attn(empty, *a[1:], 0.05, dv=512).shape == (3, 0, 48, 512)


def test_captured_in_a_graph(cuda_ok):
    """The lengths are read on the device: one captured call serves growing contexts."""
    from kernelswift_b200 import ops

    g, q, kv8, scale, tail, table, lens = build(2, 1, 16, 512, 64, 64, [700, 650], seed=10)
    lens0 = lens.clone()
    out = torch.empty(2, 1, 16, 512, dtype=torch.bfloat16, device="cuda")
    ws = torch.empty(ops.tree_attn_workspace_size(2, 1, 16, 512), dtype=torch.uint8, device="cuda")
    call = lambda: ops.tree_attn(q, kv8, scale, tail, table, lens, 0.04, dv=512, out=out, workspace=ws)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for n in (700, 3, 128):
        lens.copy_(torch.tensor([n, 650], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        check(q, kv8, scale, tail, table, lens, 0.04, 512, got=out)
    lens.copy_(lens0)


def test_offsets_past_32_bits(cuda_ok):
    from kernelswift_b200 import ops

    pages, page = 70000, 64
    kv8 = torch.zeros(pages, page, 512, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    scale, tail = torch.ones(pages, page, device="cuda"), torch.zeros(pages, page, 64, dtype=torch.bfloat16, device="cuda")
    g, q, k8, sc, tl, table, lens = build(1, 2, 16, 512, 64, 64, [300], seed=13)
    ref = ops.tree_attn(q, k8, sc, tl, table, lens, 0.04, dv=512)
    shift = pages - k8.shape[0]
    kv8.view(torch.uint8)[shift:], scale[shift:], tail[shift:] = k8.view(torch.uint8), sc, tl
    got = ops.tree_attn(q, kv8, scale, tail, table + shift, lens, 0.04, dv=512)
    ops.device_status()
    assert torch.equal(got, ref)


def test_refusals(cuda_ok):
    from kernelswift_b200 import ops

    g, q, kv8, scale, tail, table, lens = build(2, 2, 16, 128, 64, 32, [20, 20], seed=5)
    f = lambda *a, **k: (lambda: ops.tree_attn(*a, **k))  # noqa: E731
    mask = torch.ones(2, 2, 2, dtype=torch.bool, device="cuda")
    z = lambda *s: torch.zeros(*s, dtype=torch.uint8, device="cuda")  # noqa: E731
    zq = lambda d: torch.zeros(2, 2, 16, d, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    for call, why in [
        (f(q.half(), kv8, scale, tail, table, lens, 0.1), "bfloat16"),
        (f(q[..., :128].contiguous(), kv8, scale, tail, table, lens, 0.1), "128 columns"),
        (f(q, kv8, scale, tail, table[:1], lens, 0.1), "page_table"),
        (f(q, kv8, scale, tail, table, lens.long(), 0.1), "lens"),
        (f(q, kv8, scale, tail, table, lens, 0.1, dv=100), "dv=100"),
        (f(q, kv8, scale, tail, table, lens, 0.1, dv=256), "dv=256"),
        (f(q, kv8, scale, tail, table, lens, 0.1, mask=mask[:1]), "mask"),
        (f(q, kv8, scale, tail, table, lens, 0.1, mask=mask.float()), "mask"),
        (f(q, kv8, scale, tail, table, lens, 0.1, attn_sink=torch.zeros(15, device="cuda")), "attn_sink"),
        (f(q, kv8, scale, tail, table, lens, 0.1, workspace=z(16)), "bytes needed"),
        (f(q, kv8, scale, tail, table, lens, 0.1, out=torch.empty(2, 2, 16, 64, dtype=torch.bfloat16, device="cuda")), "shape"),
        (f(q.cpu(), kv8, scale, tail, table, lens, 0.1), "CUDA"),
        (f(q.transpose(1, 2), kv8, scale, tail, table, lens, 0.1), "contiguous|columns|lens|page"),
        (f(zq(96), z(2, 4, 96), torch.ones(2, 4, device="cuda"), None, table, lens, 0.1, dv=64), "dq=96"),
        (f(zq(640), z(2, 4, 640), torch.ones(2, 4, device="cuda"), None, table, lens, 0.1, dv=64), "dq=640"),
    ]:
        with pytest.raises(RuntimeError, match=why):
            call()
    ops.device_status()


# ---- range and precision, whatever the sizes of the rows and queries beside a token's own
def put(kv8, scale, tail, table, b, pos, rows):
    """Rows written at positions `pos` of sequence b."""
    from kernelswift_b200 import ops

    page = kv8.shape[1]
    pos = torch.as_tensor(pos, device="cuda")
    ops.cache_write(rows.bfloat16(), table[b].long()[pos // page] * page + pos % page, kv8, scale, tail)


@pytest.mark.parametrize("n", [40, 3000])
@pytest.mark.parametrize("dv", [128, 192])
@pytest.mark.parametrize("big", [2.0 ** 24, 2.0 ** 56, 2.0 ** 60, 2.0 ** 80, 2.0 ** 110])
def test_hidden_drafted_rows_of_any_size(cuda_ok, n, dv, big):
    """A drafted row that the mask hides takes nothing from the others, however much larger
    than they it is (n = 3000: nor through the join of parts)."""
    g, q, kv8, scale, tail, table, lens = build(2, 4, 8, 128, 64, 32, [n, n + 90], seed=41)
    for b in range(2):
        put(kv8, scale, tail, table, b, [int(lens[b]) + 1], big * torch.randn(1, 192, device="cuda", generator=g))
    mask = torch.eye(4, dtype=torch.bool, device="cuda").repeat(2, 1, 1)
    mask[:, :, 0] = True
    mask[:, 3, 2] = True
    mask[:, 1, 1] = False
    check(q, kv8, scale, tail, table, lens, 192 ** -0.5, dv, mask)


@pytest.mark.parametrize("at", [0, 200, 1999])
@pytest.mark.parametrize("dv", [128, 192])
@pytest.mark.parametrize("big", [2.0 ** 56, 2.0 ** 60, 2.0 ** 80, 2.0 ** 110])
def test_context_rows_of_any_size_without_weight(cuda_ok, at, dv, big):
    g, q, kv8, scale, tail, table, lens = build(1, 1, 1, 128, 64, 32, [2000], seed=42)
    put(kv8, scale, tail, table, 0, [at], -big * q.float().view(1, 192))
    check(q, kv8, scale, tail, table, lens, 192 ** -0.5, dv)


@pytest.mark.parametrize("n,at", [(300, 0), (300, 299), (4000, 5), (4000, 3990)])
@pytest.mark.parametrize("dv", [128, 192])
@pytest.mark.parametrize("bits", [30, 60, 80, 95])
def test_large_rows_whose_weight_makes_up_for_their_size(cuda_ok, n, at, dv, bits):
    """One row 2^bits as large as the others with about 2^-bits of their weight: both sides
    count.  Rotary column 0 alone sets the scores."""
    T, H = 2, 3
    g, q, kv8, scale, tail, table, lens = build(1, T, H, 128, 64, 64, [n], seed=43)
    q.zero_()
    q[..., 0] = q[..., 128] = 1.0
    rows = torch.randn(n + T, 192, device="cuda", generator=g)
    rows[:, 0] = rows[:, 128] = 0.0
    rows[at] *= 2.0 ** bits
    rows[at, 128] = -round(2 * bits * np.log(2)) / 2
    put(kv8, scale, tail, table, 0, list(range(n + T)), rows)
    check(q, kv8, scale, tail, table, lens, 1.0, dv)


@pytest.mark.parametrize("n", [300, 3000])
@pytest.mark.parametrize("dv", [128, 192])
@pytest.mark.parametrize("big", [2.0 ** 20, 2.0 ** 40, 2.0 ** 60, 2.0 ** 110])
def test_scores_of_any_size(cuda_ok, n, dv, big):
    """Large rows that are seen: scores of about `big` in either direction, so that one of
    them, or the rest of the context, has all the weight."""
    g, q, kv8, scale, tail, table, lens = build(2, 3, 12, 128, 64, 32, [n, n // 3], seed=49)
    for b in range(2):
        at = [n // 100, n // 5, int(lens[b]) + 1]
        put(kv8, scale, tail, table, b, at, big * torch.randn(3, 192, device="cuda", generator=g))
    check(q, kv8, scale, tail, table, lens, 192 ** -0.5, dv)


@pytest.mark.parametrize("n", [300, 3000])
@pytest.mark.parametrize("dq,dv", [(512, 512), (128, 128), (128, 192)])
def test_rows_at_the_top_of_the_range(cuda_ok, n, dq, dv):
    """Rows near the largest that the cache holds, queries so small that the scores are
    ordinary: no product on the way overflows."""
    g, *a = build(2, 2, 16, dq, 64, 64, [n, n // 2], seed=46, key_scale=lambda x: 0 * x + 2.0 ** 124,
                  q_scale=2.0 ** -119)
    check(*a, 2.0 ** -5 * (dq + 64) ** -0.5, dv)
    # and beside ordinary rows, to which ordinary queries give all the weight
    g, q, kv8, scale, tail, table, lens = build(1, 1, 1, dq, 64, 64, [n], seed=47)
    put(kv8, scale, tail, table, 0, [n // 2], -2.0 ** 122 * q.float().view(1, dq + 64))
    check(q, kv8, scale, tail, table, lens, (dq + 64) ** -0.5, dv)


@pytest.mark.parametrize("codes,rotary,keys,sm", [
    (0.0, 2.0 ** 14, 2.0 ** 14, 2.0 ** -31),      # a query of rotary columns alone
    (2.0 ** -110, 2.0 ** 14, 2.0 ** 14, 2.0 ** -31),
    (0.0, 2.0 ** 100, 2.0 ** -80, 2.0 ** -23),
    (1.0, 0.0, 1.0, 2.0 ** -4),
    (2.0 ** -20, 1.0, 1.0, 2.0 ** -4),
    (1.0, 2.0 ** -30, 1.0, 2.0 ** -4),
    (2.0 ** -118, 2.0 ** -118, 2.0 ** 100, 2.0 ** 14),  # small queries keep their bits
    (2.0 ** 110, 2.0 ** 110, 2.0 ** -10, 2.0 ** -104),
])
def test_queries_of_any_size_in_either_part(cuda_ok, codes, rotary, keys, sm):
    g, q, *rest = build(2, 2, 16, 128, 64, 32, [150, 60], seed=44, key_scale=lambda x: 0 * x + keys)
    q = torch.cat([q[..., :128].float() * codes, q[..., 128:].float() * rotary], -1).bfloat16()
    check(q, *rest, sm, 192)


@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("column", [3, 127, 128, 191])
def test_queries_that_are_not_finite_in_either_part(cuda_ok, value, column):
    from kernelswift_b200 import ops

    g, q, *rest = build(2, 3, 20, 128, 64, 32, [40, 300], seed=45)
    clean = ops.tree_attn(q, *rest, 0.1, dv=192)
    q[0, 1, 3, column] = q[1, 2, 19, column] = value
    got = ops.tree_attn(q, *rest, 0.1, dv=192)
    hit = torch.zeros(2, 3, 20, dtype=torch.bool, device="cuda")
    hit[0, 1, 3] = hit[1, 2, 19] = True
    assert got[hit].isnan().all() and torch.equal(got[~hit], clean[~hit])


@pytest.mark.parametrize("B,T,H,dq,dr,dv,lens", [(3, 1, 16, 512, 64, 512, [1, 127, 900]), (2, 5, 24, 448, 64, 448, [200, 77]),
                                                 (1, 2, 128, 128, 0, 128, [3000]), (2, 1, 5, 64, 64, 64, [2, 3])])
def test_weights_of_the_codes_within_the_stated_bound(cuda_ok, B, T, H, dq, dr, dv, lens):
    """Where v has no bf16 columns, the weights are off by at most 2^-11 of themselves (fp16,
    which three parts of 3 bits and a sign hold exactly): beside the output's rounding (2^-8)
    and fp32 work (2^-12) nothing else is allowed."""
    bound = 2.0 ** -8 + 2.0 ** -11 + 2.0 ** -12
    g, *a = build(B, T, H, dq, dr, 64, lens, seed=48)
    from kernelswift_b200 import ops

    q, kv8, scale, tail, table, n = a
    got = ops.tree_attn(*a, (dq + dr) ** -0.5, dv=dv).double().cpu().numpy()
    codes, s = kv8.view(torch.uint8).cpu().numpy().reshape(-1, dq), scale.double().cpu().numpy().reshape(-1)
    t = tail.double().cpu().numpy().reshape(-1, dr) if dr else None
    for b in range(B):
        rows = C.sequence_rows(codes, s, t, (table[b].cpu().numpy(), 64), lens[b] + T)
        for i in range(T):
            seen = np.arange(lens[b] + T) <= lens[b] + i
            ref, size = C.tree_attn_row(q[b, i].double().cpu().numpy(), rows, seen, (dq + dr) ** -0.5, None, dv)
            assert (np.abs(got[b, i] - ref) <= bound * size).all()


@pytest.mark.parametrize("n", [90, 3000])
@pytest.mark.parametrize("dv", [128, 192])
def test_a_key_with_all_the_weight_is_returned_exactly(cuda_ok, n, dv):
    """The weight that counts most is not rounded: a key 2^-30 and more ahead of the others
    comes out as it is cached, code times scale."""
    from kernelswift_b200 import ops

    g, q, kv8, scale, tail, table, lens = build(2, 3, 5, 128, 64, 32, [n, n // 3], seed=50)
    q = torch.randn(2, 3, 1, 192, device="cuda", generator=g).expand(2, 3, 5, 192).bfloat16().contiguous()
    at = [n // 9, 2, n // 3 - 1]
    for b in range(2):
        for i in range(3):  # each token's own favourite, its scores twice any other's or more
            put(kv8, scale, tail, table, b, [at[i]], 8 * q[b, i, :1].float())
    mask = torch.eye(3, dtype=torch.bool, device="cuda").repeat(2, 1, 1)
    got = ops.tree_attn(q, kv8, scale, tail, table, lens, 0.25, dv=dv, mask=mask)
    rows = ops.cache_read(kv8, scale, tail, table, lens, n)
    ops.device_status()
    for b in range(2):
        for i in range(3):
            s = (rows[b, : int(lens[b])].double() @ q[b, i, 0].double()) * 0.25
            assert s.topk(2).values.diff().item() < -25 and int(s.argmax()) == at[i]
            assert torch.equal(got[b, i], rows[b, at[i], :dv].expand(5, dv))


@pytest.mark.parametrize("sm", [0.0, -0.07, 2.0 ** -120, 1e-42, 40.0])
def test_any_softmax_scale(cuda_ok, sm):
    g, *a = build(2, 2, 20, 128, 64, 32, [300, 41], seed=51)
    check(*a, float(np.float32(sm)), 192)


@pytest.mark.parametrize("n", [60, 3000])
def test_sinks_of_any_size(cuda_ok, n):
    from kernelswift_b200 import ops

    g, *a = build(2, 1, 6, 128, 64, 32, [n, n // 3], seed=52)
    sink = torch.tensor([float("-inf"), -1e30, 0.0, 60.0, 1e30, float("inf")], device="cuda")
    got = ops.tree_attn(*a, 0.07, dv=192, attn_sink=sink)
    assert (got[:, :, 4:] == 0).all()
    q, *rest = a
    check(q[:, :, :4].contiguous(), *rest, 0.07, 192, None, sink[:4].contiguous(), got=got[:, :, :4])
