"""kv_append against the 64-bit restatement (oracle/head_cache_oracle.py).

Rotation (fp32, every operation rounded), scale and code are exact to specify: codes and scales
have to be equal, and rows that the call does not write have to stay as they were."""
import numpy as np
import pytest
import torch

from oracle import head_cache_oracle as O

pytestmark = pytest.mark.gpu

STALE = 0x7F  # what untouched rows hold: e4m3's NaN


def make(B, heads, d, page, block, lens, T, seed, spare=2, fill=False):
    """A cache of random codes (or STALE everywhere but below lens), tables in no order."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    each = -(-(max(lens) + T) // page)
    pool = B * each + spare
    table = torch.randperm(pool, device="cuda", generator=g)[: B * each].view(B, each).int()
    parts = []
    for _ in range(2):
        codes = torch.randint(0, 0x7F, (pool, heads, page, d), device="cuda", generator=g).to(torch.uint8)
        codes |= (torch.randint(0, 2, codes.shape, device="cuda", generator=g) << 7).to(torch.uint8)
        scale = torch.exp2(torch.randint(-9, -3, (pool, heads, page // block), device="cuda", generator=g).float())
        parts += [codes.view(torch.float8_e4m3fn), scale]
    return g, table.contiguous(), torch.tensor(lens, dtype=torch.int32, device="cuda"), parts


def rows(g, B, T, heads, d, spread=3):
    x = torch.randn(B, T, heads, d, device="cuda", generator=g)
    return (x * torch.exp2(torch.randint(-spread, spread + 1, (B, T, 1, 1), device="cuda", generator=g).float())).bfloat16()


def freq_table(n, rd):
    ang = torch.outer(torch.arange(n).double(), 10000.0 ** (-torch.arange(0, rd, 2).double() / max(rd, 1)))
    return torch.stack([ang.cos(), ang.sin()], -1).float().cuda().contiguous()


def host(t):
    return t.view(torch.uint8).cpu().numpy().copy() if t.dtype == torch.float8_e4m3fn else t.double().cpu().numpy()


def expect(k, v, parts, table, lens, freqs, positions=None, n_new=None):
    """Codes and scales that have to be there afterwards."""
    B, T = k.shape[:2]
    k8, ks, v8, vs = (host(x) for x in parts)
    page, block = k8.shape[2], k8.shape[2] // ks.shape[2]
    fr = None if freqs is None else freqs.cpu().numpy()
    for b in range(B):
        n = T if n_new is None else int(n_new[b])
        at = int(lens[b])
        pos = at + np.arange(n) if positions is None else positions[b, :n].cpu().numpy()
        tb = table[b].cpu().numpy()
        O.append(O.rotate(host(k[b, :n]), fr, pos), k8, ks, tb, at, block)
        O.append(np.asarray(host(v[b, :n]), np.float32), v8, vs, tb, at, block)
    return k8, ks, v8, vs


def same(parts, want):
    for name, got, ref in zip(("k8", "k_scale", "v8", "v_scale"), parts, want):
        got = host(got)
        if got.dtype == np.uint8:  # any NaN is one
            got, ref = (np.where((x & 0x7F) == 0x7F, 0x7F, x) for x in (got, ref))
            # -0 and 0 are told apart
        bad = np.argwhere(got != ref)
        assert not len(bad), (name, len(bad), bad[:3].tolist())


@pytest.mark.parametrize("B,T,heads,d,rd,page,block,lens", [
    (1, 1, 1, 64, 0, 16, 16, [0]), (3, 1, 2, 128, 64, 64, 16, [5, 16, 63]), (2, 5, 8, 128, 128, 96, 32, [31, 1000]),
    (2, 40, 3, 64, 64, 48, 48, [7, 95]), (1, 300, 2, 256, 32, 128, 128, [129]), (4, 17, 1, 192, 64, 64, 64, [0, 1, 62, 64]),
    (2, 131, 5, 64, 8, 16, 16, [15, 17]), (1, 1, 4, 256, 256, 80, 80, [79]), (2, 33, 2, 192, 192, 112, 112, [111, 3]),
])
def test_codes_and_scales_are_exact(cuda_ok, B, T, heads, d, rd, page, block, lens):
    from kernelswift_b200 import ops

    g, table, n, parts = make(B, heads, d, page, block, lens, T, B * 100 + T)
    k, v = rows(g, B, T, heads, d), rows(g, B, T, heads, d)
    v[0, -1] = 0
    freqs = freq_table(max(lens) + T, rd) if rd else None
    want = expect(k, v, parts, table, n, freqs)
    assert ops.kv_append(k, v, *parts, table, n, freqs=freqs) is None
    ops.device_status()
    same(parts, want)


def test_scales_grow_within_a_block_and_start_anew(cuda_ok):
    """Token by token: sizes that go up make the rows there be rounded again; the first row of
    a block forgets the scale that the page held."""
    from kernelswift_b200 import ops

    g, table, n, parts = make(2, 2, 64, 32, 16, [3, 14], 24, 5)
    for step in range(24):
        k, v = (rows(g, 2, 1, 2, 64, 0) * 2.0 ** ((step * 5) % 11 - 5) for _ in range(2))
        want = expect(k, v, parts, table, n, None)
        ops.kv_append(k, v, *parts, table, n)
        same(parts, want)
        n = n + 1


def test_rows_behind_and_pages_of_others_stay(cuda_ok):
    from kernelswift_b200 import ops

    g, table, n, parts = make(3, 2, 128, 64, 32, [10, 40, 0], 30, 7)
    for x in parts[::2]:
        x.view(torch.uint8).fill_(STALE)
    new = torch.tensor([0, 7, 30], dtype=torch.int32, device="cuda")
    k, v = rows(g, 3, 30, 2, 128), rows(g, 3, 30, 2, 128)
    want = expect(k, v, parts, table, n, None, n_new=new)
    ops.kv_append(k, v, *parts, table, n, n_new=new)
    ops.device_status()
    same(parts, want)
    assert int((parts[0].view(torch.uint8) != STALE).sum()) <= (7 + 30) * 2 * 128


@pytest.mark.parametrize("big", [2.0 ** -30, 2.0 ** 40, 2.0 ** 120, 3.3e38])
def test_sizes_at_the_ends_of_the_range(cuda_ok, big):
    from kernelswift_b200 import ops

    g, table, n, parts = make(1, 2, 64, 16, 16, [4], 9, 3)
    v = torch.randn(1, 9, 2, 64, device="cuda", generator=g).clamp(-1, 1)
    v[..., 0] = 1
    k, v = (v * big).bfloat16(), (-v * big).bfloat16()
    assert k.isfinite().all()
    want = expect(k, v, parts, table, n, None)
    ops.kv_append(k, v, *parts, table, n)
    same(parts, want)


def test_elements_that_are_not_finite_are_marked(cuda_ok):
    from kernelswift_b200 import ops

    g, table, n, parts = make(2, 2, 64, 32, 16, [5, 20], 36, 11)
    k, v = rows(g, 2, 30, 2, 64), rows(g, 2, 30, 2, 64)
    k[0, 3, 1, 5], k[1, 20, 0, 63], v[0, 0, 0, 0], v[1, 29, 1, 7] = (float(x) for x in ("nan", "inf", "-inf", "nan"))
    want = expect(k, v, parts, table, n, None)
    ops.kv_append(k, v, *parts, table, n)
    same(parts, want)
    assert (np.isnan(O.e4m3_values()[want[0]])).sum() == 2
    # the mark stays while the block is added to, and goes when it begins anew
    k2, v2 = rows(g, 2, 3, 2, 64), rows(g, 2, 3, 2, 64)
    for lens, marks in (([35, 50], 4), ([0, 0], 2)):  # the first sequence's block had one in either part
        n = torch.tensor(lens, dtype=torch.int32, device="cuda")
        want = expect(k2, v2, parts, table, n, None)
        ops.kv_append(k2, v2, *parts, table, n)
        same(parts, want)
        assert sum(int(O.unmarked(x)[1].sum()) for x in (want[1], want[3])) == marks


def test_strided_rows_positions_and_queries(cuda_ok):
    """Slices of one projection, a tree's depths as positions; rotated queries are the fp32
    rotation rounded once."""
    from kernelswift_b200 import ops

    B, T, H, heads, d, rd = 3, 6, 10, 2, 128, 64
    g, table, n, parts = make(B, heads, d, 64, 16, [30, 0, 100], T, 13)
    wide = rows(g, B, T + 2, H + 2 * heads, d)[:, 1:-1]
    q, k, v = wide[:, :, :H], wide[:, :, H:H + heads], wide[:, :, H + heads:]
    assert not k.is_contiguous()
    depth = torch.tensor([0, 1, 1, 2, 2, 3], device="cuda")
    pos = (n[:, None] + depth).int().contiguous()
    freqs = freq_table(120, rd)
    want = expect(k, v, parts, table, n, freqs, positions=pos)
    out = ops.kv_append(k, v, *parts, table, n, freqs=freqs, positions=pos, q=q)
    ops.device_status()
    same(parts, want)
    for b in range(B):
        ref = torch.from_numpy(O.rotate(host(q[b]), freqs.cpu().numpy(), pos[b].cpu().numpy())).bfloat16()
        assert torch.equal(out[b].cpu(), ref)
    q2 = wide[:, :, :H].contiguous()
    assert ops.kv_append(k, v, *parts, table, n, q=q2) is q2  # nothing to rotate


def test_bad_pages_positions_and_lengths_are_reported(cuda_ok):
    from kernelswift_b200 import ops

    def call(change, bad_rows):
        g, table, n, parts = make(2, 1, 64, 16, 16, [3, 3], 20, 17)
        k, v = rows(g, 2, 20, 1, 64), rows(g, 2, 20, 1, 64)
        freqs = freq_table(40, 64)
        before = [host(x) for x in parts]
        table, n, freqs = change(table.clone(), n.clone(), freqs)
        ops.kv_append(k, v, *parts, table, n, freqs=freqs)
        with pytest.raises(RuntimeError, match="index"):
            ops.device_status()
        ops.device_status()
        return k, v, parts, table, n, freqs, before

    def page(value):
        def f(table, n, freqs):
            table[0, 1] = value
            return table, n, freqs
        return f

    for value in (-1, 10 ** 6):
        k, v, parts, table, n, freqs, before = call(page(value), 1)
        new = torch.tensor([13, 20])  # sequence 0: the rows of its first page
        ref = [torch.from_numpy(x) for x in before]
        want = expect(k, v, [ref[0].view(torch.float8_e4m3fn), ref[1], ref[2].view(torch.float8_e4m3fn), ref[3]],
                      table, n, freqs, n_new=new)
        same(parts, want)
    call(lambda t, n, f: (t, n + 20, f), 1)                  # past the table
    call(lambda t, n, f: (t, n, f[:10].contiguous()), 1)     # past the rotation's rows


def test_offsets_past_32_bits(cuda_ok):
    """A cache of more than 2^32 bytes: the last pages."""
    from kernelswift_b200 import ops

    pages, heads, page, d = 140000, 4, 64, 128
    block = 64
    k8 = torch.zeros(pages, heads, page, d, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    scale = torch.zeros(pages, heads, page // block, device="cuda")
    v8, v_scale = k8.clone(), scale.clone()
    assert k8.numel() > 2 ** 32
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v = rows(g, 1, 3, heads, d), rows(g, 1, 3, heads, d)
    table = torch.tensor([[pages - 1]], dtype=torch.int32, device="cuda")
    n = torch.tensor([2], dtype=torch.int32, device="cuda")
    last = [k8[-1:].clone(), scale[-1:].clone(), v8[-1:].clone(), v_scale[-1:].clone()]
    ops.kv_append(k, v, k8, scale, v8, v_scale, table, n)
    want = expect(k, v, last, torch.zeros_like(table), n, None)
    same([k8[-1:], scale[-1:], v8[-1:], v_scale[-1:]], want)
    assert int((k8[:-1].view(torch.uint8).view(torch.int64) != 0).sum()) == 0


def test_streams_and_graphs(cuda_ok):
    from kernelswift_b200 import ops

    g, table, n, parts = make(2, 2, 128, 64, 16, [3, 60], 4, 19)
    k, v, q = rows(g, 2, 4, 2, 128), rows(g, 2, 4, 2, 128), rows(g, 2, 4, 6, 128)
    freqs = freq_table(80, 64)
    want = expect(k, v, parts, table, n, freqs)
    start = [x.clone() for x in parts]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        out = ops.kv_append(k, v, *parts, table, n, freqs=freqs, q=q)
    torch.cuda.current_stream().wait_stream(s)
    same(parts, want)
    for x, y in zip(parts, start):
        x.copy_(y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out2 = ops.kv_append(k, v, *parts, table, n, freqs=freqs, q=q)
    same(parts, [host(x) for x in start])
    graph.replay()
    same(parts, want)
    assert torch.equal(out, out2)
    graph.replay()  # the same rows again change nothing
    same(parts, want)


def test_queries_that_are_not_rotated_go_on_to_attention(cuda_ok):
    """Without freqs, slices of one projection: what comes back is what kv_attn takes."""
    from kernelswift_b200 import ops

    B, T, H, heads, d = 2, 3, 8, 2, 128
    g, table, n, parts = make(B, heads, d, 64, 16, [30, 7], T, 23)
    wide = rows(g, B, T, H + 2 * heads, d, 0)
    q, k, v = wide.split([H, heads, heads], 2)
    want = expect(k, v, parts, table, n, None)
    out = ops.kv_append(k, v, *parts, table, n, q=q)
    same(parts, want)
    assert out.is_contiguous() and torch.equal(out, q)
    whole = ops.kv_attn(out, *parts, table, n, d ** -0.5)
    assert torch.equal(whole, ops.kv_attn(q.clone(memory_format=torch.contiguous_format), *parts, table, n, d ** -0.5))
    assert ops.kv_append(k, v, *parts, table, n, q=out) is out
