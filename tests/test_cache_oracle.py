"""The 64-bit restatement of the latent-cache operators (oracle/cache_oracle.py) against
independent statements of its parts, the host side of the operators, and a chain of them
on small numbers.  No GPU."""
import numpy as np
import pytest
import torch

from kernelswift_b200 import ops
from oracle import cache_oracle as C
from oracle import ks_oracle as O


def test_e4m3_values_and_codes_against_torch():
    codes = torch.arange(256, dtype=torch.uint8)
    ref = codes.view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(C.e4m3_values(), ref, equal_nan=True)
    rng = np.random.default_rng(0)
    x = np.concatenate([rng.standard_normal(20000) * 100, rng.standard_normal(20000) * 0.01,
                        C.e4m3_values()[:0x7F], -C.e4m3_values()[:0x7F],
                        (C.e4m3_values()[:0x7E] + C.e4m3_values()[1:0x7F]) / 2])  # ties
    x = x[np.abs(x) <= 448]
    got = torch.from_numpy(x).float().to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(C.e4m3_codes(x.astype(np.float32).astype(np.float64)), got)


def test_rows_equal_the_fp8_quantiser_restated():
    rng = np.random.default_rng(1)
    x = (rng.standard_normal((200, 64)) * np.exp(rng.uniform(-10, 10, (200, 1)))).astype(np.float32)
    bits = O.f32_to_bf16(x)
    codes, scale = C.cache_rows(O.bf16_to_f32(bits).astype(np.float64), 64)
    ref_codes, ref_scale = O.quant_fp8_rows(bits)
    assert np.array_equal(scale, ref_scale.astype(np.float64))
    assert np.array_equal(codes & 0x7F, ref_codes & 0x7F)  # (the sign of zero is not stated there)


def test_rows_that_are_not_finite_and_the_largest_scale():
    x = np.ones((4, 32))
    x[0, 3], x[1, 31], x[2] = np.nan, np.inf, 3.3895e38
    codes, scale = C.cache_rows(x, 16)
    assert np.isnan(scale[:2]).all() and (codes[:2] == 0).all()
    assert scale[2] == 2.0 ** 119 and (codes[2] == 0x7E).all()
    assert np.isfinite(np.float32(scale[2] * 448))


def test_tree_attention_restated():
    """Equal scores average the rows that are seen; a sink takes its share; nothing seen
    gives zeros."""
    rows = np.arange(12, dtype=np.float64).reshape(4, 3)
    q = np.zeros((2, 3))
    seen = np.array([True, False, True, True])
    out, size = C.tree_attn_row(q, rows, seen, 1.0, None, 2)
    assert np.allclose(out, rows[seen][:, :2].mean(0)) and np.allclose(size, out)
    out, _ = C.tree_attn_row(q, rows, seen, 1.0, np.array([0.0, -np.inf]), 2)
    assert np.allclose(out[0], rows[seen][:, :2].sum(0) / 4) and np.allclose(out[1], rows[seen][:, :2].mean(0))
    out, _ = C.tree_attn_row(q, rows, np.zeros(4, bool), 1.0, None, 2)
    assert (out == 0).all()


def test_verification_restated():
    p = np.array([[0.5, 0.3, 0.2], [0.1, 0.8, 0.1], [0.2, 0.2, 0.6]], np.float32)
    noise = np.ones(3, np.float32)
    # fixed candidates: u picks the stretch of one of the children 1 and 0 of the root
    par, tok = [-1, -1], [1, 0]
    assert C.verify_tree(p, tok, par, [0.29, 0, 0], noise) == ([1, 1], [0])
    assert C.verify_tree(p, tok, par, [0.31, 0, 0], noise) == ([0, 2], [1])
    assert C.verify_tree(p, tok, par, [0.85, 0, 0], noise) == ([2], [])
    # a sampled chain: u q < p, then the rest of p over q
    q = np.array([[0.9, 0.1, 0.0], [0.1, 0.8, 0.1]], np.float32)
    assert C.verify_chain(p, q, [0, 1], [0.5, 0.99], noise) == ([0, 1, 2], [0, 1])
    assert C.verify_chain(p, q, [0, 1], [0.6, 0.0], noise) == ([1], [])


def test_workspace_of_tree_attention_is_host_only(built_lib):
    n = ops.tree_attn_workspace_size(1, 1, 16, 512)
    assert n % 256 == 0 and n >= 148 * 2 * 16 * 512 * 4
    assert ops.tree_attn_workspace_size(64, 64, 128, 512) == ops.tree_attn_workspace_size(1, 1, 17, 512)


def test_ops_refuse_host_tensors_and_wrong_shapes():
    kv8, scale = torch.zeros(2, 4, 64, dtype=torch.uint8), torch.zeros(2, 4)
    kv = torch.zeros(3, 64, dtype=torch.bfloat16)
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    q = torch.zeros(1, 2, 4, 64, dtype=torch.bfloat16)
    p = torch.zeros(1, 3, 9)
    for call, why in [
        (lambda: ops.cache_write(kv, torch.arange(3), kv8, scale), "CUDA"),
        (lambda: ops.cache_write(kv, torch.arange(2), kv8, scale), "2 slots"),
        (lambda: ops.cache_write(kv, torch.arange(3), kv8[0], scale), "kv8"),
        (lambda: ops.cache_write(kv, torch.arange(3), kv8[:0], scale[:0]), "no pages"),
        (lambda: ops.cache_read(kv8, scale, None, i32(1, 2), i32(1), 5), "CUDA"),
        (lambda: ops.cache_read(kv8, scale, torch.zeros(2, 3, 8, dtype=torch.bfloat16), i32(1, 2), i32(1), 5), "kv_tail"),
        (lambda: ops.tree_attn(q, kv8, scale, None, i32(1, 2), i32(1), 1.0), "CUDA"),
        (lambda: ops.tree_attn(q, kv8, scale, None, i32(2, 2), i32(1), 1.0), "page_table"),
        (lambda: ops.tree_attn(q, kv8, scale, None, i32(1, 2), i32(1), 1.0, mask=torch.ones(1, 2, 3).bool()), "mask"),
        (lambda: ops.verify_draft(p, torch.zeros(1, 2).long(), torch.zeros(1, 3), torch.zeros(1, 9)), "CUDA"),
        (lambda: ops.verify_draft(p, torch.zeros(1, 3).long(), torch.zeros(1, 3), torch.zeros(1, 9)), "p must be"),
    ]:
        with pytest.raises(RuntimeError, match=why):
            call()


def test_three_e5m2_parts_hold_a_half_exactly():
    """The split of tree attention's weights, restated: parts rounded to nearest at fp16's
    high byte (an e5m2 number) add up to every fp16 number from 2^-3 to 55109 exactly, and to
    smaller ones within half of e5m2's smallest."""
    half = np.arange(0x7B00, dtype=np.uint16)
    w = half.view(np.float16).astype(np.float64)
    half, w = half[w <= 55109], w[w <= 55109]
    rest, parts = half.view(np.float16), 0.0
    for _ in range(3):
        part = ((rest.view(np.uint16).astype(np.uint32) + 0x80) & 0xFF00).astype(np.uint16).view(np.float16)
        assert np.isfinite(part).all()
        parts = parts + part.astype(np.float64)
        rest = rest - part
    assert (parts == w)[w >= 2.0 ** -3].all() and (np.abs(parts - w) <= 2.0 ** -17).all()
