"""cache_write / cache_read against the 64-bit restatement (oracle/cache_oracle.py).

Quantisation is exact to specify: codes and scales have to be equal, and reading back
(an e4m3 code times a power of two) has no rounding in bf16."""
import numpy as np
import pytest
import torch

from helpers import bits_from_bf16
from oracle import cache_oracle as C

pytestmark = pytest.mark.gpu

NAN_BYTES = 0x7F  # untouched slots hold this code before a write


def empty_cache(pages, page, dq, dr):
    kv8 = torch.full((pages, page, dq), NAN_BYTES, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    scale = torch.full((pages, page), -3.0, device="cuda")
    tail = torch.full((pages, page, dr), 7.0, dtype=torch.bfloat16, device="cuda") if dr else None
    return kv8, scale, tail


def f64(t):
    return t.double().cpu().numpy()


def codes_of(kv8):
    return kv8.view(torch.uint8).cpu().numpy().reshape(-1, kv8.shape[-1])


@pytest.mark.parametrize("R,dq,dr,page,pad", [
    (1, 512, 64, 64, 0), (7, 512, 64, 64, 64), (1000, 512, 64, 48, 8), (333, 128, 0, 16, 0),
    (65, 448, 64, 100, 0), (40, 16, 0, 1, 8), (129, 64, 64, 7, 0), (50, 1024, 8, 32, 0),
    (20, 528, 320, 16, 0), (31, 208, 72, 5, 16), (257, 256, 1024, 64, 0),
])
@pytest.mark.parametrize("slot_dtype", [torch.int32, torch.int64])
def test_write_bit_exact(cuda_ok, R, dq, dr, page, pad, slot_dtype):
    from kernelswift_b200 import ops

    g = torch.Generator(device="cuda").manual_seed(R * 1000 + dq)
    pages = -(-R // page) + 2
    wide = torch.randn(R, dq + dr + pad, device="cuda", generator=g)
    wide *= torch.exp2(torch.randint(-18, 18, (R, 1), device="cuda", generator=g).float())
    kv = wide.bfloat16()[:, :dq + dr]
    kv[0, :dq] = 0
    kv[-1, 0] = 448.0  # a maximum on the power-of-two edge of the scale
    kv[-1, 1:dq] = 0.5
    slots = torch.randperm(pages * page, device="cuda", generator=g)[:R]
    if R > 5:
        slots[3] = -1  # a padding row
    slots = slots.to(slot_dtype)
    kv8, scale, tail = empty_cache(pages, page, dq, dr)
    ops.cache_write(kv, slots, kv8, scale, tail)
    ops.device_status()
    codes, s = C.cache_rows(f64(kv), dq)
    ref8 = np.full((pages * page, dq), NAN_BYTES, np.uint8)
    refs = np.full(pages * page, -3.0)
    at = slots.cpu().numpy()
    ref8[at[at >= 0]], refs[at[at >= 0]] = codes[at >= 0], s[at >= 0]
    assert np.array_equal(codes_of(kv8), ref8)
    assert np.array_equal(f64(scale).reshape(-1), refs)
    if dr:
        reft = np.full((pages * page, dr), 7.0)
        reft[at[at >= 0]] = f64(kv)[at >= 0, dq:]
        assert np.array_equal(f64(tail).reshape(-1, dr), reft)


def test_write_marks_rows_that_are_not_finite(cuda_ok):
    from kernelswift_b200 import ops

    kv = torch.randn(8, 128 + 64, device="cuda").bfloat16()
    kv[1, 5], kv[2, 127], kv[3, 128], kv[4, 191] = float("nan"), float("inf"), float("-inf"), float("nan")
    kv[6] = torch.finfo(torch.bfloat16).max  # the largest finite rows stay finite
    kv8, scale, tail = empty_cache(1, 8, 128, 64)
    ops.cache_write(kv, torch.arange(8, device="cuda"), kv8, scale, tail)
    table, lens = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.tensor([8], dtype=torch.int32, device="cuda")
    back = ops.cache_read(kv8, scale, tail, table, lens, 8)[0]
    bad = torch.zeros(8, dtype=torch.bool)
    bad[1:5] = True
    assert torch.equal(scale[0].isnan().cpu(), bad)
    assert (codes_of(kv8)[1:5] == 0).all()
    assert torch.equal(back[:, :128].isnan().all(1).cpu(), bad)
    assert torch.equal(back[:, :128].isnan().any(1).cpu(), bad)
    assert torch.isfinite(back[6].float()).all()


def test_write_codes_equal_quant_fp8_rows(cuda_ok):
    """With no tail a page per sequence is what indexer_topk_fp8 takes."""
    from kernelswift_b200 import ops

    k = torch.randn(3, 40, 128, device="cuda").bfloat16()
    kv8, scale, _ = empty_cache(3, 40, 128, 0)
    ops.cache_write(k, torch.arange(120, device="cuda"), kv8, scale)
    k8, ks = ops.quant_fp8_rows(k)
    assert torch.equal(kv8.view(torch.uint8), k8.view(torch.uint8)) and torch.equal(scale, ks)


@pytest.mark.parametrize("B,n,start,dq,dr,page", [
    (1, 1, 0, 512, 64, 64), (3, 130, 0, 512, 64, 64), (2, 77, 51, 448, 64, 48), (5, 33, 0, 128, 0, 1),
    (2, 300, 7, 64, 64, 100), (1, 19, 3, 16, 8, 5), (2, 20, 0, 1024, 1024, 16), (4, 9, 0, 272, 40, 2),
])
def test_read_exact(cuda_ok, B, n, start, dq, dr, page):
    from kernelswift_b200 import ops

    g = torch.Generator(device="cuda").manual_seed(n)
    each = -(-(start + n) // page)
    table = torch.randperm(B * each + 3, device="cuda", generator=g)[:B * each].view(B, each).int().contiguous()
    pages = B * each + 3
    kv8, scale, tail = empty_cache(pages, page, dq, dr)
    kv = torch.randn(pages * page, dq + dr, device="cuda", generator=g)
    kv *= torch.exp2(torch.randint(-30, 30, (pages * page, 1), device="cuda", generator=g).float())
    ops.cache_write(kv.bfloat16(), torch.arange(pages * page, device="cuda"), kv8, scale, tail)
    lens = torch.tensor([(start + n, 0, start, start + n // 2, 10 ** 6)[b % 5] for b in range(B)],
                        dtype=torch.int32, device="cuda")
    got = ops.cache_read(kv8, scale, tail, table, lens, n, start)
    ops.device_status()
    codes, s = codes_of(kv8), f64(scale).reshape(-1)
    t = f64(tail).reshape(-1, dr) if dr else None
    for b in range(B):
        ref = C.sequence_rows(codes, s, t, (table[b].cpu().numpy(), page), start + n)[start:]
        ref[max(0, int(lens[b]) - start):] = 0
        assert np.array_equal(f64(got[b]), ref)
    out = torch.empty_like(got)
    assert ops.cache_read(kv8, scale, tail, table, lens, n, start, out=out) is out
    assert np.array_equal(bits_from_bf16(out), bits_from_bf16(got))


def test_read_feeds_sparse_attention(cuda_ok):
    """The rows read back are the kv of sparse_attn: same result as from the values."""
    from kernelswift_b200 import ops

    g = torch.Generator(device="cuda").manual_seed(1)
    kv = torch.randn(2, 100, 576, device="cuda", generator=g).bfloat16()
    kv8, scale, tail = empty_cache(10, 20, 512, 64)
    ops.cache_write(kv, torch.arange(200, device="cuda"), kv8, scale, tail)
    table = torch.arange(10, device="cuda").view(2, 5).int()
    lens = torch.full((2,), 100, dtype=torch.int32, device="cuda")
    back = ops.cache_read(kv8, scale, tail, table, lens, 100)
    ref = torch.cat([(kv8.float() * scale[..., None]).view(2, 100, 512), tail.float().view(2, 100, 64)], -1)
    assert torch.equal(back.float(), ref)
    q = torch.randn(2, 3, 16, 576, device="cuda", generator=g).bfloat16()
    idx = torch.randint(0, 100, (2, 3, 32), device="cuda", generator=g).int()
    sink = torch.zeros(16, device="cuda")
    assert torch.equal(ops.sparse_attn(q, back, sink, idx, 0.04, dv=512),
                       ops.sparse_attn(q, ref.bfloat16(), sink, idx, 0.04, dv=512))


def test_out_of_range_slots_and_pages_are_reported(cuda_ok):
    from kernelswift_b200 import ops

    kv = torch.randn(4, 128, device="cuda").bfloat16()
    kv8, scale, _ = empty_cache(2, 4, 128, 0)
    ops.cache_write(kv, torch.tensor([0, 8, 3, -5], device="cuda"), kv8, scale)
    with pytest.raises(RuntimeError, match="query row 1"):
        ops.device_status()
    assert (scale.view(-1)[[0, 3]] > 0).all() and (scale.view(-1)[[1, 2, 4, 5, 6, 7]] == -3).all()
    lens = torch.tensor([6], dtype=torch.int32, device="cuda")
    for table in ([[0, 2]], [[0, -1]], [[0]]):
        got = ops.cache_read(kv8, scale, None, torch.tensor(table, dtype=torch.int32, device="cuda"), lens, 6)
        with pytest.raises(RuntimeError, match="device status"):
            ops.device_status()
        assert (got[0, 4:] == 0).all() and torch.isfinite(got[0, 0].float()).all()
    ops.device_status()


def test_slots_past_32_bit_offsets(cuda_ok):
    """A pool of over 2^31 bytes of codes: the last slots hold what was written there."""
    from kernelswift_b200 import ops

    pages, page, dq = 70000, 64, 512  # 2.3e9 bytes
    kv8 = torch.zeros(pages, page, dq, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    scale = torch.zeros(pages, page, device="cuda")
    kv = torch.randn(70, dq, device="cuda").bfloat16()
    first = pages * page - 70
    ops.cache_write(kv, torch.arange(first, first + 70, device="cuda"), kv8, scale)
    codes, s = C.cache_rows(f64(kv), dq)
    assert np.array_equal(codes_of(kv8[-2:])[-70:], codes)
    table = torch.tensor([[pages - 1, pages - 2]], dtype=torch.int32, device="cuda")
    got = ops.cache_read(kv8, scale, None, table, torch.tensor([64], dtype=torch.int32, device="cuda"), 64)
    ops.device_status()
    assert np.array_equal(f64(got[0]), C.e4m3_values()[codes[-64:]] * s[-64:, None])


def test_empty_calls_and_streams(cuda_ok):
    from kernelswift_b200 import ops

    kv8, scale, tail = empty_cache(2, 4, 64, 64)
    ops.cache_write(torch.empty(0, 128, dtype=torch.bfloat16, device="cuda"),
                    torch.empty(0, dtype=torch.int64, device="cuda"), kv8, scale, tail)
    table, lens = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    assert ops.cache_read(kv8, scale, tail, table, lens, 0).shape == (1, 0, 128)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    kv = torch.randn(4, 128, device="cuda").bfloat16()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.cache_write(kv, torch.arange(4, device="cuda"), kv8, scale, tail)
        got = ops.cache_read(kv8, scale, tail, table, lens + 4, 4)
    side.synchronize()
    assert torch.equal(got[0, :, 64:], kv[:, 64:])


def test_refusals(cuda_ok):
    from kernelswift_b200 import ops

    kv8, scale, tail = empty_cache(2, 4, 64, 64)
    kv, slots = torch.zeros(3, 128, dtype=torch.bfloat16, device="cuda"), torch.arange(3, device="cuda")
    table, lens = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    bad = [
        (lambda: ops.cache_write(kv.float(), slots, kv8, scale, tail), "bfloat16"),
        (lambda: ops.cache_write(kv, slots.float(), kv8, scale, tail), "slots"),
        (lambda: ops.cache_write(kv, slots[:2], kv8, scale, tail), "2 slots"),
        (lambda: ops.cache_write(kv, slots, kv8, scale, None), "128 columns"),
        (lambda: ops.cache_write(kv, slots, kv8, scale.half(), tail), "kv_scale"),
        (lambda: ops.cache_write(kv, slots, kv8, scale[:1], tail), "kv_scale"),
        (lambda: ops.cache_write(kv, slots, kv8.float(), scale, tail), "kv8"),
        (lambda: ops.cache_write(kv, slots.cpu(), kv8, scale, tail), "CUDA"),
        (lambda: ops.cache_write(kv.cpu(), slots, kv8, scale, tail), "device"),
        (lambda: ops.cache_write(torch.zeros(3, 129, dtype=torch.bfloat16, device="cuda")[:, :128], slots, kv8, scale, tail), "16-byte"),
        (lambda: ops.cache_write(torch.zeros(256, 3, dtype=torch.bfloat16, device="cuda").t()[:, ::2], slots, kv8, scale, tail), "contiguous"),
        (lambda: ops.cache_write(torch.zeros(3, 40, dtype=torch.bfloat16, device="cuda"), slots,
                                 torch.zeros(2, 4, 40, dtype=torch.uint8, device="cuda"), scale), "dq=40"),
        (lambda: ops.cache_read(kv8, scale, tail, table.long(), lens, 1), "page_table"),
        (lambda: ops.cache_read(kv8, scale, tail, table, lens.long(), 1), "lens"),
        (lambda: ops.cache_read(kv8, scale, tail, table, lens, -1), "negative"),
        (lambda: ops.cache_read(kv8, scale, tail, table, lens, 2 ** 31), "2\\^31|memory"),
        (lambda: ops.cache_read(kv8, scale, tail, table, lens, 1, out=torch.empty(1, 1, 64, dtype=torch.bfloat16, device="cuda")), "shape"),
    ]
    for call, why in bad:
        with pytest.raises(RuntimeError, match=why):
            call()
    ops.device_status()


@pytest.mark.parametrize("dq,dr", [(128, 64), (16, 8), (512, 64), (272, 40), (64, 1024), (1024, 1024)])
def test_rows_that_are_not_finite_read_back_as_nan_whole(cuda_ok, dq, dr):
    """Wherever the NaN or the infinity was, no column of the row reads as a number."""
    from kernelswift_b200 import ops

    kv = torch.randn(9, dq + dr, device="cuda").bfloat16()
    kv[1, dq - 1], kv[2, dq], kv[4, dq + dr - 1], kv[7, 0] = float("nan"), float("inf"), float("nan"), float("-inf")
    kv8, scale, tail = empty_cache(3, 3, dq, dr)
    ops.cache_write(kv, torch.arange(9, device="cuda"), kv8, scale, tail)
    table = torch.arange(3, dtype=torch.int32, device="cuda")[None].contiguous()
    back = ops.cache_read(kv8, scale, tail, table, torch.tensor([9], dtype=torch.int32, device="cuda"), 9)[0]
    bad = torch.zeros(9, dtype=torch.bool, device="cuda")
    bad[[1, 2, 4, 7]] = True
    assert back[bad].isnan().all() and torch.isfinite(back[~bad].float()).all()
    assert torch.equal(back[~bad][:, dq:], kv[~bad][:, dq:])
